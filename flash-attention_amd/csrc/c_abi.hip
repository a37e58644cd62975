// extern "C" surface of libmyfa_gfx950.so (declared in include/myfa.h).
//
// Replaces the argument checking / dispatch half of the reference's binding
// layer (csrc/api.cpp:110-192); output allocation stays with the caller.
#include "myfa_common.h"
#include "paged_common.h"
#include "tuning.h"
#include "window_attn_common.h"

#include <cstdarg>
#include <cstdio>
#include <cstring>
#include <string>

namespace myfa {

namespace {
thread_local char g_err[512] = "";
}

int fail(int code, const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_err, sizeof(g_err), fmt, ap);
    va_end(ap);
    return code;
}

thread_local hipError_t t_launch_err = hipSuccess;

int check_launch(const char* what) {
    const hipError_t e = t_launch_err;
    t_launch_err = hipSuccess;
    if (e != hipSuccess) return fail(MYFA_E_LAUNCH, "%s: launch failed: %s", what, hipGetErrorString(e));
    return MYFA_OK;
}

#ifdef MYFA_TUNING
Tuning& tuning() {
    static Tuning t{};
    return t;
}
#endif

// implemented in the kernel translation units
int softmax_f32(const float* in, float* out, int64_t h, int64_t w, hipStream_t s);
int softmax_rows(const void* in, void* out, int64_t h, int64_t w, int dtype, hipStream_t s);
int softmax_strided(const void* in, void* out, int64_t outer, int64_t len, int64_t inner, int dtype, hipStream_t s);
int softmax_strided_pro(const void* in, void* out, int64_t outer, int64_t len, int64_t inner, int dtype,
                        float scale, const float* mask, int64_t mask_outer, bool causal, hipStream_t s,
                        void* ws, size_t ws_bytes);
size_t softmax_strided_ws_bytes(int64_t outer, int64_t len, int64_t inner, int dtype);
int matmul_f32(const float* a, const float* b, float* c, int64_t m, int64_t k, int64_t n, hipStream_t s);
int attn_fwd_f32(const float* q, const float* k, const float* v, float* o, float* lse,
                 int64_t heads, int64_t N, int64_t d, int64_t k_key_stride, int64_t k_d_stride,
                 float scale, bool causal, hipStream_t s, float* ws, size_t ws_bytes);
size_t attn_fwd_f32_ws_bytes(int64_t heads, int64_t N, int64_t d);
int attn_fwd_mfma(const void* q, const void* k, const void* v, void* o, float* lse,
                  int64_t heads, int64_t N, int64_t d, float scale, int dtype, bool causal, hipStream_t s);
const char* attn_fwd_mfma_kernel_name(int64_t d, int dtype, bool causal);
int attn_bwd_mfma(const void* q, const void* k, const void* v, const void* o, const float* lse, const void* dout,
                  void* dq, void* dk, void* dv, float* delta, int64_t heads, int64_t N, int64_t d,
                  float scale, int dtype, bool causal, hipStream_t s);
int attn_bwd_mfma_static_ws(const void* q, const void* k, const void* v, const void* o, const float* lse, const void* dout,
                            void* dq, void* dk, void* dv, int64_t heads, int64_t N, int64_t d,
                            float scale, int dtype, bool causal, hipStream_t s);
int window_attn_fwd(const void* q, const void* k, const void* v, void* o, float* lse, const WindowShape& w, int dtype, hipStream_t s);
int64_t window_attn_bwd_ws_bytes(const WindowShape& w, int elem_size);
int window_attn_bwd(const void* q, const void* k, const void* v, const void* o, const float* lse, const void* dout,
                    void* dq, void* dk, void* dv, float* ws, const WindowShape& w, int dtype, hipStream_t s);
int paged_append(const void* k, const void* v, const PagedCache& c, const AppendShape& a, hipStream_t s);
int64_t paged_decode_ws_bytes(const DecodeShape& w, int64_t cap, bool weights);
int paged_decode(const void* q, const PagedCache& c, void* o, float* lse, float* weight_sum, float* ws, const DecodeShape& w,
                 int dtype, hipStream_t s);
int paged_evict(const PagedCache& c, const EvictShape& e, hipStream_t s);

namespace {

constexpr int64_t kMaxCount = 1 << 28;     // tokens of a sequence, and batch, heads, ... each: products of two fit 64 bits
// keys of a paged sequence: the kernels' 32-bit loops step up to 8192 keys past the last one
constexpr int64_t kMaxCapacity = (1ll << 31) - (1 << 16);

int elem_size(int dtype) { return dtype == MYFA_F32 ? 4 : 2; }
bool misaligned(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 != 0; }

// Element type and head dim of the window and paged operators.
int check_elem(const char* what, int64_t d, int dtype) {
    if (dtype != MYFA_F32 && dtype != MYFA_F16 && dtype != MYFA_BF16) return fail(MYFA_E_INVALID, "%s: unknown dtype tag %d", what, dtype);
    const int64_t step = dtype == MYFA_F32 ? 4 : 8, most = dtype == MYFA_F32 ? 128 : 256;
    if (d % step != 0 || d > most)
        return fail(MYFA_E_UNSUPPORTED, "%s: head dim %lld; multiples of %lld up to %lld are supported for this element type", what,
                    (long long)d, (long long)step, (long long)most);
    return MYFA_OK;
}

// n strides of a tensor: multiples of 16 bytes, below 2^40 elements
int check_strides(const char* what, const char* name, const int64_t* st, int n, int dtype) {
    if (!st) return fail(MYFA_E_INVALID, "%s: null strides of %s", what, name);
    for (int i = 0; i < n; ++i)
        if (st[i] * elem_size(dtype) % 16 != 0 || st[i] <= -(1ll << 40) || st[i] >= 1ll << 40)
            return fail(MYFA_E_INVALID, "%s: stride %lld of %s is not a multiple of 16 bytes", what, (long long)st[i], name);
    return MYFA_OK;
}

int window_shape(const char* what, WindowShape& w, const int32_t* seq_lens, int64_t B, int64_t H, int64_t Hkv, int64_t Nq, int64_t Nk,
                 int64_t d, int64_t window, int64_t sinks, float scale) {
    for (int64_t x : {B, H, Hkv, Nq, Nk, d, sinks})
        if (x < 0) return fail(MYFA_E_INVALID, "%s: negative size", what);
    for (int64_t x : {B, H, Hkv, Nq, Nk})
        if (x > kMaxCount) return fail(MYFA_E_UNSUPPORTED, "%s: size %lld beyond 2^28", what, (long long)x);
    if (B * H > kMaxCount || B * H * Nk > 1ll << 40) return fail(MYFA_E_UNSUPPORTED, "%s: too many rows", what);
    if (Nq > Nk) return fail(MYFA_E_INVALID, "%s: more queries (%lld) than keys (%lld)", what, (long long)Nq, (long long)Nk);
    if (H < 1 || Hkv < 1 || H % Hkv != 0)
        return fail(MYFA_E_INVALID, "%s: %lld query heads are not a multiple of %lld key/value heads", what, (long long)H, (long long)Hkv);
    if (window < 1) return fail(MYFA_E_INVALID, "%s: window %lld; a query sees at least itself", what, (long long)window);
    if (!(scale > 0.f) || scale > 3e38f) return fail(MYFA_E_INVALID, "%s: scale must be positive and finite", what);
    w.B = (int)B; w.H = (int)H; w.Hkv = (int)Hkv; w.Nq = (int)Nq; w.Nk = (int)Nk; w.d = (int)d;
    w.window = (int)(window < Nk ? window : Nk);
    w.sinks = (int)(sinks < Nk ? sinks : Nk);
    w.scale = scale;
    w.lens = seq_lens;
    return MYFA_OK;
}

int window_strides(const char* what, WindowShape& w, const int64_t* qs, const int64_t* ks, const int64_t* vs, int dtype) {
    const char* names[3] = {"q", "k", "v"};
    const int64_t* in[3] = {qs, ks, vs};
    int64_t* out[3] = {w.qs, w.ks, w.vs};
    for (int t = 0; t < 3; ++t) {
        if (int rc = check_strides(what, names[t], in[t], 3, dtype)) return rc;
        if (in[t][2] < 0 || in[t][2] * elem_size(dtype) >= 1 << 24)
            return fail(MYFA_E_UNSUPPORTED, "%s: row stride %lld of %s", what, (long long)in[t][2], names[t]);
        for (int i = 0; i < 3; ++i) out[t][i] = in[t][i];
    }
    return MYFA_OK;
}

// The cache part of a paged call; `table` may be null where the caller checks sizes only.
int paged_cache(const char* what, PagedCache& c, const void* k, const void* v, const int32_t* table, int64_t B, int64_t Hkv, int64_t d,
                int64_t num_pages, int64_t page, int64_t width, const int64_t* ks, const int64_t* vs, int dtype) {
    for (int64_t x : {B, Hkv, d, num_pages, width})
        if (x < 0) return fail(MYFA_E_INVALID, "%s: negative size", what);
    if (Hkv < 1) return fail(MYFA_E_INVALID, "%s: no heads", what);
    if (page < 1) return fail(MYFA_E_INVALID, "%s: page of %lld keys", what, (long long)page);
    for (int64_t x : {B, Hkv, num_pages, width, page})
        if (x > kMaxCount) return fail(MYFA_E_UNSUPPORTED, "%s: size %lld beyond 2^28", what, (long long)x);
    if (B * Hkv > kMaxCount) return fail(MYFA_E_UNSUPPORTED, "%s: %lld heads", what, (long long)(B * Hkv));
    if (width * page > kMaxCapacity) return fail(MYFA_E_UNSUPPORTED, "%s: capacity of %lld keys a sequence", what, (long long)(width * page));
    if (int rc = check_elem(what, d, dtype)) return rc;
    if (int rc = check_strides(what, "the key cache", ks, 3, dtype)) return rc;
    if (int rc = check_strides(what, "the value cache", vs, 3, dtype)) return rc;
    if (misaligned(k) || misaligned(v)) return fail(MYFA_E_INVALID, "%s: caches must be 16-byte aligned", what);
    c.k = static_cast<const char*>(k);
    c.v = static_cast<const char*>(v);
    for (int i = 0; i < 3; ++i) { c.kst[i] = ks[i] * elem_size(dtype); c.vst[i] = vs[i] * elem_size(dtype); }
    c.table = table;
    c.num_pages = (int)num_pages;
    c.width = (int)width;
    c.row_bytes = (int)d * elem_size(dtype);
    c.page = FastDiv((uint32_t)page);
    return MYFA_OK;
}

int check_workspace(const char* what, const void* ws, int64_t bytes, int64_t need) {
    if (bytes < need || (need > 0 && !ws) || misaligned(ws))
        return fail(MYFA_E_INVALID, "%s: the workspace needs %lld bytes, 16-byte aligned", what, (long long)need);
    return MYFA_OK;
}

}  // namespace

}  // namespace myfa

using namespace myfa;

extern "C" {

int myfa_abi_version(void) { return MYFA_ABI_VERSION; }

const char* myfa_last_error(void) { return g_err; }

int myfa_device_info(int device, int* cu_count, int* lds_bytes, int* wave_size, char* arch, int arch_len) {
    hipDeviceProp_t p;
    const hipError_t e = hipGetDeviceProperties(&p, device);
    if (e != hipSuccess) return fail(MYFA_E_DEVICE, "device %d: %s", device, hipGetErrorString(e));
    if (cu_count) *cu_count = p.multiProcessorCount;
    if (lds_bytes) *lds_bytes = (int)p.sharedMemPerBlock;
    if (wave_size) *wave_size = p.warpSize;
    if (arch && arch_len > 0) {
        std::strncpy(arch, p.gcnArchName, (size_t)arch_len - 1);
        arch[arch_len - 1] = '\0';
    }
    return MYFA_OK;
}

int myfa_softmax_f32(const float* in, float* out, int64_t h, int64_t w, void* stream) {
    return softmax_f32(in, out, h, w, static_cast<hipStream_t>(stream));
}

int myfa_softmax(const void* in, void* out, int64_t h, int64_t w, int dtype, void* stream) {
    return softmax_rows(in, out, h, w, dtype, static_cast<hipStream_t>(stream));
}

int myfa_softmax_nd(const void* in, void* out, int64_t outer, int64_t len, int64_t inner, int dtype, void* stream) {
    return softmax_strided(in, out, outer, len, inner, dtype, static_cast<hipStream_t>(stream));
}

int myfa_softmax_nd_ex(const void* in, void* out, int64_t outer, int64_t len, int64_t inner, int dtype,
                       float scale, const float* add_mask, int64_t mask_outer, int flags, void* stream) {
    if ((flags & ~MYFA_SOFTMAX_CAUSAL) != 0) return fail(MYFA_E_INVALID, "softmax: unknown flag bits 0x%x", flags);
    return softmax_strided_pro(in, out, outer, len, inner, dtype, scale, add_mask, mask_outer,
                               (flags & MYFA_SOFTMAX_CAUSAL) != 0, static_cast<hipStream_t>(stream), nullptr, 0);
}

int64_t myfa_softmax_nd_ws_bytes(int64_t outer, int64_t len, int64_t inner, int dtype) {
    return (int64_t)softmax_strided_ws_bytes(outer, len, inner, dtype);
}

int myfa_softmax_nd_ws(const void* in, void* out, int64_t outer, int64_t len, int64_t inner, int dtype,
                       float scale, const float* add_mask, int64_t mask_outer, int flags,
                       void* workspace, int64_t workspace_bytes, void* stream) {
    if ((flags & ~MYFA_SOFTMAX_CAUSAL) != 0) return fail(MYFA_E_INVALID, "softmax: unknown flag bits 0x%x", flags);
    if (workspace_bytes < 0 || (workspace == nullptr && workspace_bytes > 0) || reinterpret_cast<uintptr_t>(workspace) % 16 != 0)
        return fail(MYFA_E_INVALID, "softmax: workspace must be 16-byte aligned with a non-negative size");
    return softmax_strided_pro(in, out, outer, len, inner, dtype, scale, add_mask, mask_outer,
                               (flags & MYFA_SOFTMAX_CAUSAL) != 0, static_cast<hipStream_t>(stream),
                               workspace, (size_t)workspace_bytes);
}

int myfa_attn_fwd_f32(const float* q, const float* k_t, const float* v, float* o,
                      int64_t n, int64_t d, float scale, void* stream) {
    if (n < 0 || d < 0) return fail(MYFA_E_INVALID, "attention: negative size n=%lld d=%lld", (long long)n, (long long)d);
    if (n == 0 || d == 0) return MYFA_OK;
    if (!q || !k_t || !v || !o) return fail(MYFA_E_INVALID, "attention: null pointer");
    // K_t is [d, n]: key stride 1, dim stride n
    return attn_fwd_f32(q, k_t, v, o, nullptr, 1, n, d, 1, n, scale, false, static_cast<hipStream_t>(stream), nullptr, 0);
}

int64_t myfa_attn_fwd_f32_ws_bytes(int64_t n, int64_t d) { return (int64_t)attn_fwd_f32_ws_bytes(1, n, d); }

int myfa_attn_fwd_f32_ws(const float* q, const float* k_t, const float* v, float* o,
                         int64_t n, int64_t d, float scale, void* workspace, int64_t workspace_bytes, void* stream) {
    if (n < 0 || d < 0) return fail(MYFA_E_INVALID, "attention: negative size n=%lld d=%lld", (long long)n, (long long)d);
    if (n == 0 || d == 0) return MYFA_OK;
    if (!q || !k_t || !v || !o) return fail(MYFA_E_INVALID, "attention: null pointer");
    if (workspace_bytes < 0 || (workspace == nullptr && workspace_bytes > 0) || reinterpret_cast<uintptr_t>(workspace) % 16 != 0)
        return fail(MYFA_E_INVALID, "attention: workspace must be 16-byte aligned with a non-negative size");
    return attn_fwd_f32(q, k_t, v, o, nullptr, 1, n, d, 1, n, scale, false, static_cast<hipStream_t>(stream),
                        static_cast<float*>(workspace), (size_t)workspace_bytes);
}

int myfa_attn_fwd_bhnd(const void* q, const void* k, const void* v, void* o, float* lse,
                       int64_t B, int64_t H, int64_t N, int64_t d, float scale, int dtype, void* stream) {
    return myfa_attn_fwd_bhnd_ex(q, k, v, o, lse, B, H, N, d, scale, dtype, 0, stream);
}

int myfa_attn_fwd_bhnd_ex(const void* q, const void* k, const void* v, void* o, float* lse,
                          int64_t B, int64_t H, int64_t N, int64_t d, float scale, int dtype, int flags, void* stream) {
    if ((flags & ~MYFA_ATTN_CAUSAL) != 0) return fail(MYFA_E_INVALID, "attention: unknown flag bits 0x%x", flags);
    const bool causal = (flags & MYFA_ATTN_CAUSAL) != 0;
    if (B < 0 || H < 0 || N < 0 || d < 0)
        return fail(MYFA_E_INVALID, "attention: negative size B=%lld H=%lld N=%lld d=%lld",
                    (long long)B, (long long)H, (long long)N, (long long)d);
    if (B == 0 || H == 0 || N == 0 || d == 0) return MYFA_OK;
    if (!q || !k || !v || !o) return fail(MYFA_E_INVALID, "attention: null pointer");
    const int64_t heads = B * H;
    hipStream_t s = static_cast<hipStream_t>(stream);
    switch (dtype) {
        case MYFA_F32:
            // K is [N, d]: key stride d, dim stride 1
            return attn_fwd_f32(static_cast<const float*>(q), static_cast<const float*>(k),
                                static_cast<const float*>(v), static_cast<float*>(o), lse,
                                heads, N, d, d, 1, scale, causal, s, nullptr, 0);
        case MYFA_F16:
        case MYFA_BF16:
            if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) |
                 reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(o)) % 16 != 0)
                return fail(MYFA_E_INVALID, "attention (f16/bf16): tensors must be 16-byte aligned");
            return attn_fwd_mfma(q, k, v, o, lse, heads, N, d, scale, dtype, causal, s);
        default:
            return fail(MYFA_E_INVALID, "attention: unknown dtype tag %d", dtype);
    }
}

const char* myfa_attn_fwd_bhnd_kernel(int64_t d, int dtype, int flags) {
    if ((flags & ~MYFA_ATTN_CAUSAL) != 0 || d <= 0) return nullptr;
    if (dtype == MYFA_F32) return d <= 512 ? "attn_fwd_f32_kernel" : nullptr;
    if (dtype != MYFA_F16 && dtype != MYFA_BF16) return nullptr;
    return attn_fwd_mfma_kernel_name(d, dtype, (flags & MYFA_ATTN_CAUSAL) != 0);
}

int myfa_attn_bwd_bhnd(const void* q, const void* k, const void* v, const void* o, const float* lse,
                       const void* dout, void* dq, void* dk, void* dv, float* delta_ws,
                       int64_t B, int64_t H, int64_t N, int64_t d, float scale, int dtype, int flags, void* stream) {
    if (B < 0 || H < 0 || N < 0 || d < 0)
        return fail(MYFA_E_INVALID, "attention backward: negative size B=%lld H=%lld N=%lld d=%lld",
                    (long long)B, (long long)H, (long long)N, (long long)d);
    if ((flags & ~MYFA_ATTN_CAUSAL) != 0) return fail(MYFA_E_INVALID, "attention backward: unknown flag bits 0x%x", flags);
    if (B == 0 || H == 0 || N == 0 || d == 0) return MYFA_OK;
    if (!q || !k || !v || !o || !lse || !dout || !dq || !dk || !dv || !delta_ws)
        return fail(MYFA_E_INVALID, "attention backward: null pointer");
    if (dtype != MYFA_F16 && dtype != MYFA_BF16 && dtype != MYFA_F32)
        return fail(MYFA_E_UNSUPPORTED, "attention backward: float16, bfloat16 or float32 (dtype tag %d)", dtype);
    if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) |
         reinterpret_cast<uintptr_t>(o) | reinterpret_cast<uintptr_t>(dout) | reinterpret_cast<uintptr_t>(dq) |
         reinterpret_cast<uintptr_t>(dk) | reinterpret_cast<uintptr_t>(dv)) % 16 != 0)
        return fail(MYFA_E_INVALID, "attention backward: tensors must be 16-byte aligned");
    return attn_bwd_mfma(q, k, v, o, lse, dout, dq, dk, dv, delta_ws, B * H, N, d, scale, dtype,
                         (flags & MYFA_ATTN_CAUSAL) != 0, static_cast<hipStream_t>(stream));
}

int myfa_attn_bwd_bhnd_static_ws(const void* q, const void* k, const void* v, const void* o, const float* lse,
                                 const void* dout, void* dq, void* dk, void* dv,
                                 int64_t B, int64_t H, int64_t N, int64_t d, float scale, int dtype, int flags, void* stream) {
    if (B < 0 || H < 0 || N < 0 || d < 0)
        return fail(MYFA_E_INVALID, "attention backward: negative size B=%lld H=%lld N=%lld d=%lld",
                    (long long)B, (long long)H, (long long)N, (long long)d);
    if ((flags & ~MYFA_ATTN_CAUSAL) != 0) return fail(MYFA_E_INVALID, "attention backward: unknown flag bits 0x%x", flags);
    if (B == 0 || H == 0 || N == 0 || d == 0) return MYFA_OK;
    if (!q || !k || !v || !o || !lse || !dout || !dq || !dk || !dv)
        return fail(MYFA_E_INVALID, "attention backward: null pointer");
    if (dtype != MYFA_F16 && dtype != MYFA_BF16 && dtype != MYFA_F32)
        return fail(MYFA_E_UNSUPPORTED, "attention backward: float16, bfloat16 or float32 (dtype tag %d)", dtype);
    if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) |
         reinterpret_cast<uintptr_t>(o) | reinterpret_cast<uintptr_t>(dout) | reinterpret_cast<uintptr_t>(dq) |
         reinterpret_cast<uintptr_t>(dk) | reinterpret_cast<uintptr_t>(dv)) % 16 != 0)
        return fail(MYFA_E_INVALID, "attention backward: tensors must be 16-byte aligned");
    if (B > MYFA_BWD_STATIC_WS_ROWS || H > MYFA_BWD_STATIC_WS_ROWS || B * H > MYFA_BWD_STATIC_WS_ROWS)
        return fail(MYFA_E_UNSUPPORTED, "attention backward (static workspace): B*H*N exceeds %d rows", MYFA_BWD_STATIC_WS_ROWS);
    return attn_bwd_mfma_static_ws(q, k, v, o, lse, dout, dq, dk, dv, B * H, N, d, scale, dtype,
                                   (flags & MYFA_ATTN_CAUSAL) != 0, static_cast<hipStream_t>(stream));
}

int myfa_matmul_f32(const float* a, const float* b, float* c, int64_t m, int64_t k, int64_t n, void* stream) {
    return matmul_f32(a, b, c, m, k, n, static_cast<hipStream_t>(stream));
}

int myfa_window_attn_fwd(const void* q, const void* k, const void* v, void* o, float* lse, const int32_t* seq_lens,
                         int64_t B, int64_t H, int64_t Hkv, int64_t Nq, int64_t Nk, int64_t d,
                         const int64_t* q_strides, const int64_t* k_strides, const int64_t* v_strides,
                         int64_t window, int64_t sinks, float scale, int dtype, void* stream) {
    const char* what = "window attention";
    WindowShape w;
    if (int rc = window_shape(what, w, seq_lens, B, H, Hkv, Nq, Nk, d, window, sinks, scale)) return rc;
    if (int rc = check_elem(what, d, dtype)) return rc;
    if (d == 0 && lse) return fail(MYFA_E_UNSUPPORTED, "%s: head dim 0 has an output of no elements, but a log-sum-exp, which is not formed", what);
    if (B == 0 || Nq == 0 || d == 0) return MYFA_OK;
    if (!q || !k || !v || !o) return fail(MYFA_E_INVALID, "%s: null pointer", what);
    if (misaligned(q) || misaligned(k) || misaligned(v) || misaligned(o)) return fail(MYFA_E_INVALID, "%s: tensors must be 16-byte aligned", what);
    if (int rc = window_strides(what, w, q_strides, k_strides, v_strides, dtype)) return rc;
    return window_attn_fwd(q, k, v, o, lse, w, dtype, static_cast<hipStream_t>(stream));
}

int64_t myfa_window_attn_bwd_ws_bytes(int64_t B, int64_t H, int64_t Hkv, int64_t Nq, int64_t Nk, int64_t d, int64_t window, int64_t sinks, int dtype) {
    WindowShape w;
    if (window_shape("window attention backward", w, nullptr, B, H, Hkv, Nq, Nk, d, window, sinks, 1.f) != MYFA_OK || d > 256) return 0;
    if (B == 0 || Nk == 0 || d == 0) return 0;
    return window_attn_bwd_ws_bytes(w, elem_size(dtype));
}

int myfa_window_attn_bwd(const void* q, const void* k, const void* v, const void* o, const float* lse, const void* dout,
                         void* dq, void* dk, void* dv, const int32_t* seq_lens,
                         int64_t B, int64_t H, int64_t Hkv, int64_t Nq, int64_t Nk, int64_t d,
                         const int64_t* q_strides, const int64_t* k_strides, const int64_t* v_strides,
                         int64_t window, int64_t sinks, float scale, int dtype,
                         void* workspace, int64_t workspace_bytes, void* stream) {
    const char* what = "window attention backward";
    WindowShape w;
    if (int rc = window_shape(what, w, seq_lens, B, H, Hkv, Nq, Nk, d, window, sinks, scale)) return rc;
    if (int rc = check_elem(what, d, dtype)) return rc;
    if (B == 0 || Nk == 0 || d == 0) return MYFA_OK;
    // (no queries: the keys' gradients are still written, as zeros)
    if (!k || !v || !dk || !dv || (Nq > 0 && (!q || !o || !lse || !dout || !dq))) return fail(MYFA_E_INVALID, "%s: null pointer", what);
    for (const void* p : {q, k, v, o, dout, static_cast<const void*>(dq), static_cast<const void*>(dk), static_cast<const void*>(dv)})
        if (misaligned(p)) return fail(MYFA_E_INVALID, "%s: tensors must be 16-byte aligned", what);
    if (int rc = window_strides(what, w, q_strides, k_strides, v_strides, dtype)) return rc;
    if (int rc = check_workspace(what, workspace, workspace_bytes, window_attn_bwd_ws_bytes(w, elem_size(dtype)))) return rc;
    return window_attn_bwd(q, k, v, o, lse, dout, dq, dk, dv, static_cast<float*>(workspace), w, dtype, static_cast<hipStream_t>(stream));
}

int myfa_paged_append(const void* k, const void* v, void* k_cache, void* v_cache, const int32_t* block_table,
                      const int32_t* seq_lens, const int32_t* counts,
                      int64_t B, int64_t Hkv, int64_t n, int64_t d, int64_t num_pages, int64_t page, int64_t table_width,
                      const int64_t* k_strides, const int64_t* v_strides,
                      const int64_t* kc_strides, const int64_t* vc_strides, int dtype, void* stream) {
    const char* what = "paged append";
    PagedCache c;
    if (int rc = paged_cache(what, c, k_cache, v_cache, block_table, B, Hkv, d, num_pages, page, table_width, kc_strides, vc_strides, dtype)) return rc;
    if (n < 0) return fail(MYFA_E_INVALID, "%s: negative size", what);
    if (n > kMaxCount) return fail(MYFA_E_UNSUPPORTED, "%s: size %lld beyond 2^28", what, (long long)n);
    if (B == 0 || n == 0 || d == 0 || num_pages == 0 || table_width == 0) return MYFA_OK;
    if (!k || !v || !k_cache || !v_cache || !block_table || !seq_lens) return fail(MYFA_E_INVALID, "%s: null pointer", what);
    if (misaligned(k) || misaligned(v)) return fail(MYFA_E_INVALID, "%s: tensors must be 16-byte aligned", what);
    if (int rc = check_strides(what, "k", k_strides, 3, dtype)) return rc;
    if (int rc = check_strides(what, "v", v_strides, 3, dtype)) return rc;
    AppendShape a;
    a.B = (int)B; a.Hkv = (int)Hkv; a.n = (int)n;
    for (int i = 0; i < 3; ++i) { a.ks[i] = k_strides[i] * elem_size(dtype); a.vs[i] = v_strides[i] * elem_size(dtype); }
    a.lens = seq_lens;
    a.counts = counts;
    return paged_append(k, v, c, a, static_cast<hipStream_t>(stream));
}

namespace {
int decode_shape(const char* what, DecodeShape& w, int64_t B, int64_t H, int64_t Hkv, int64_t d, int64_t window, int64_t sinks, int64_t cap) {
    for (int64_t x : {B, H, Hkv, d, sinks})
        if (x < 0) return fail(MYFA_E_INVALID, "%s: negative size", what);
    for (int64_t x : {B, H, Hkv})
        if (x > kMaxCount) return fail(MYFA_E_UNSUPPORTED, "%s: size %lld beyond 2^28", what, (long long)x);
    if (B * H > kMaxCount) return fail(MYFA_E_UNSUPPORTED, "%s: %lld heads", what, (long long)(B * H));
    if (H < 1 || Hkv < 1 || H % Hkv != 0)
        return fail(MYFA_E_INVALID, "%s: %lld query heads are not a multiple of %lld key/value heads", what, (long long)H, (long long)Hkv);
    w.B = (int)B; w.H = (int)H; w.Hkv = (int)Hkv; w.d = (int)d;
    w.window = (int)(window >= 1 && window < cap ? window : cap);
    w.sinks = (int)(sinks < cap ? sinks : cap);
    return MYFA_OK;
}
}  // namespace

int64_t myfa_paged_attn_decode_ws_bytes(int64_t B, int64_t H, int64_t Hkv, int64_t d, int64_t page, int64_t table_width,
                                        int64_t window, int64_t sinks, int with_weights) {
    DecodeShape w;
    if (page < 1 || page > kMaxCount || table_width < 0 || table_width > kMaxCount || page * table_width > kMaxCapacity || d > 256) return 0;
    if (decode_shape("paged attention", w, B, H, Hkv, d, window, sinks, page * table_width) != MYFA_OK) return 0;
    if (B == 0 || d == 0) return 0;
    return paged_decode_ws_bytes(w, page * table_width, with_weights != 0);
}

int myfa_paged_attn_decode(const void* q, const void* k_cache, const void* v_cache, const int32_t* block_table,
                           const int32_t* seq_lens, void* o, float* lse, float* weight_sum,
                           int64_t B, int64_t H, int64_t Hkv, int64_t d, int64_t num_pages, int64_t page, int64_t table_width,
                           const int64_t* q_strides, const int64_t* kc_strides, const int64_t* vc_strides,
                           int64_t window, int64_t sinks, float scale, int dtype,
                           void* workspace, int64_t workspace_bytes, void* stream) {
    const char* what = "paged attention";
    PagedCache c;
    if (int rc = paged_cache(what, c, k_cache, v_cache, block_table, B, Hkv, d, num_pages, page, table_width, kc_strides, vc_strides, dtype)) return rc;
    DecodeShape w;
    if (int rc = decode_shape(what, w, B, H, Hkv, d, window, sinks, page * table_width)) return rc;
    if (!(scale > 0.f) || scale > 3e38f) return fail(MYFA_E_INVALID, "%s: scale must be positive and finite", what);
    if (d == 0 && (lse || weight_sum)) return fail(MYFA_E_UNSUPPORTED, "%s: head dim 0 has an output of no elements, but a log-sum-exp and weights, which are not formed", what);
    if (B == 0 || d == 0) return MYFA_OK;
    if (!q || !o || !seq_lens || (table_width > 0 && !block_table) || (num_pages > 0 && (!k_cache || !v_cache)))
        return fail(MYFA_E_INVALID, "%s: null pointer", what);
    if (misaligned(q) || misaligned(o)) return fail(MYFA_E_INVALID, "%s: tensors must be 16-byte aligned", what);
    if (int rc = check_strides(what, "q", q_strides, 2, dtype)) return rc;
    w.scale = scale;
    w.lens = seq_lens;
    w.qs[0] = q_strides[0];
    w.qs[1] = q_strides[1];
    if (int rc = check_workspace(what, workspace, workspace_bytes, paged_decode_ws_bytes(w, page * table_width, weight_sum != nullptr))) return rc;
    return paged_decode(q, c, o, lse, weight_sum, static_cast<float*>(workspace), w, dtype, static_cast<hipStream_t>(stream));
}

int myfa_paged_evict(void* k_cache, void* v_cache, const float* weight_sum, const int32_t* block_table,
                     const int32_t* seq_lens, const int32_t* new_block_table,
                     float* new_weight_sum, int32_t* new_lens, int32_t* kept,
                     int64_t B, int64_t Hkv, int64_t d, int64_t num_pages, int64_t page, int64_t table_width, int64_t new_width,
                     const int64_t* kc_strides, const int64_t* vc_strides,
                     int64_t budget, int64_t sinks, int64_t recent, int dtype, void* stream) {
    const char* what = "paged eviction";
    PagedCache c;
    if (int rc = paged_cache(what, c, k_cache, v_cache, block_table, B, Hkv, d, num_pages, page, table_width, kc_strides, vc_strides, dtype)) return rc;
    if (new_width < 0 || new_width > kMaxCount || new_width * page > kMaxCapacity) return fail(MYFA_E_UNSUPPORTED, "%s: new table of %lld pages", what, (long long)new_width);
    if (budget < 1 || sinks < 0 || recent < 0 || sinks > budget || recent > budget - sinks)
        return fail(MYFA_E_INVALID, "%s: budget %lld must be at least 1 and hold sinks (%lld) and recent (%lld)", what, (long long)budget,
                    (long long)sinks, (long long)recent);
    if (new_width * page < budget)
        return fail(MYFA_E_INVALID, "%s: the new table holds %lld keys, the budget is %lld", what, (long long)(new_width * page), (long long)budget);
    if (B == 0) return MYFA_OK;
    if (!seq_lens || !new_block_table || !new_weight_sum || !new_lens || !kept || (table_width > 0 && (!weight_sum || !block_table)) ||
        (num_pages > 0 && d > 0 && (!k_cache || !v_cache)))
        return fail(MYFA_E_INVALID, "%s: null pointer", what);
    EvictShape e;
    e.B = (int)B; e.Hkv = (int)Hkv; e.cap = (int)(table_width * page); e.new_cap = (int)(new_width * page);
    e.budget = (int)budget; e.sinks = (int)sinks; e.recent = (int)recent;
    e.lens = seq_lens; e.sums = weight_sum; e.new_sums = new_weight_sum; e.new_lens = new_lens; e.kept = kept;
    e.new_table = new_block_table;
    return paged_evict(c, e, static_cast<hipStream_t>(stream));
}

#ifdef MYFA_TUNING
// Exported by the tuning flavour only (not part of include/myfa.h).  Keys: attn_variant,
// attn_thr, attn_spec, attn_wgs, matmul_block, matmul_ksplit, softmax_tpr, softmax_v, softmax_map, softmax_nt, softmax_pad,
// softmax_split_wgs, reset (back to the defaults).  Returns 0, or 1 for an unknown key.
int myfa_tuning_set(const char* key, double value) {
    Tuning& t = tuning();
    const std::string k(key ? key : "");
    if (k == "reset") t = Tuning{};
    else if (k == "attn_variant") t.attn_variant = (int)value;
    else if (k == "attn_thr") t.attn_thr = (float)value;
    else if (k == "attn_spec") t.attn_spec = (int)value;
    else if (k == "attn_xflags") t.attn_xflags = (int)value;
    else if (k == "attn_wgs") t.attn_wgs = (int)value;
    else if (k == "attn_pre") t.attn_pre = (int)value;
    else if (k == "attn_occ") t.attn_occ = (int)value;
    else if (k == "attn_f32_wgs") t.attn_f32_wgs = (int)value;
    else if (k == "matmul_block") t.matmul_block = (int)value;
    else if (k == "matmul_ksplit") t.matmul_ksplit = (int)value;
    else if (k == "softmax_tpr") t.softmax_shape[0] = (int)value;
    else if (k == "softmax_v") t.softmax_shape[1] = (int)value;
    else if (k == "softmax_map") t.softmax_shape[2] = (int)value;
    else if (k == "softmax_nt") t.softmax_shape[3] = (int)value;
    else if (k == "softmax_pad") t.softmax_shape[4] = (int)value;
    else if (k == "softmax_split_wgs") t.softmax_split_wgs = (int)value;
    else if (k == "softmax_cols_big") t.softmax_cols_big = (int)value;
    else return fail(MYFA_E_INVALID, "tuning: unknown key '%s'", k.c_str());
    return MYFA_OK;
}
// attn_dbg: device buffer of 24 u64 per workgroup for the stamped attention build (NULL: off)
int myfa_tuning_set_ptr(const char* key, void* p) {
    const std::string k(key ? key : "");
    if (k == "attn_dbg") tuning().attn_dbg = static_cast<unsigned long long*>(p);
    else return fail(MYFA_E_INVALID, "tuning: unknown pointer key '%s'", k.c_str());
    return MYFA_OK;
}
#endif

}  // extern "C"
