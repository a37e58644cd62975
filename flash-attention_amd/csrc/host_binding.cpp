// Host layer of window attention and the paged cache: checks the arguments, allocates results and workspaces
// with torch's allocator and calls the C ABI (include/myfa.h) on the current stream of the tensors' device.
//
// These operators serve single tokens: a call's kernels take a few microseconds, and the same checks written in
// Python with a ctypes call of 20 arguments take 12 to 18 (measured on one MI355X host; here under 2).  The Python
// functions of window.py and paged.py hold the documentation and forward to these.
// Failures are RuntimeError (TORCH_CHECK), as everywhere in the package.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <optional>
#include <string>
#include <utility>
#include <vector>

#include "myfa.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

void* current_stream(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
void check(int status) { TORCH_CHECK(status == MYFA_OK, myfa_last_error()); }

int tag(const Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return MYFA_F32;
        case at::kHalf: return MYFA_F16;
        case at::kBFloat16: return MYFA_BF16;
        default: TORCH_CHECK(false, "unsupported dtype ", t.scalar_type());
    }
}

// An integer argument that is given as one (or as a float that is whole).
int64_t whole(py::handle x, const char* name) {
    if (PyLong_Check(x.ptr())) return x.cast<int64_t>();
    if (PyFloat_Check(x.ptr())) {
        const double v = PyFloat_AS_DOUBLE(x.ptr());
        TORCH_CHECK(v == (double)(int64_t)v, name, " must be an integer, got ", v);
        return (int64_t)v;
    }
    PyObject* i = PyNumber_Index(x.ptr());
    if (!i) throw py::error_already_set();
    return py::reinterpret_steal<py::object>(i).cast<int64_t>();
}

void check_gpu(const Tensor& t, const char* name) { TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor"); }
void check_same(const Tensor& t, const Tensor& ref, const char* name) {
    TORCH_CHECK(t.device() == ref.device(), name, " is on ", t.device(), ", expected ", ref.device(), ": all operands must be on one device");
}
void check_dense(const Tensor& t, const Tensor& ref, const char* name) {
    check_gpu(t, name);
    TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
    check_same(t, ref, name);
}
void check_ints(const Tensor& t, at::IntArrayRef shape, const Tensor& ref, const char* name) {
    check_dense(t, ref, name);
    TORCH_CHECK(t.scalar_type() == at::kInt && t.sizes() == shape, name, " must be an int32 tensor of shape ", shape, ", got ", t.scalar_type(), " ", t.sizes());
}
void check_sums(const Tensor& t, at::IntArrayRef shape, const Tensor& ref) {
    check_dense(t, ref, "weight_sum");
    TORCH_CHECK(t.scalar_type() == at::kFloat, "expected scalar type Float but found ", t.scalar_type(), " for weight_sum");
    TORCH_CHECK(t.sizes() == shape, "weight_sum must be ", shape, ", got ", t.sizes());
}

// Strides of all dimensions but the last, in elements (0 for a dimension of one element, whose stride means nothing);
// the last dimension is dense and rows begin at multiples of 16 bytes.
struct Strides {
    int64_t s[3] = {0, 0, 0};
    Strides(const Tensor& t, const char* name) {
        const int64_t n = t.dim() - 1;
        if (t.numel() == 0) return;
        const int64_t size = (int64_t)t.element_size();
        bool ok = (t.stride(n) == 1 || t.size(n) == 1) && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
        for (int64_t i = 0; i < n; ++i) {
            s[i] = t.size(i) > 1 ? t.stride(i) : 0;
            ok = ok && s[i] * size % 16 == 0;
        }
        TORCH_CHECK(ok, name, " must have a dense last dimension and rows that begin at multiples of 16 bytes");
    }
};

// A tensor that a call is going to write in place: no history to keep, and no element in the place of another (two workgroups
// would write there, in no order).  Sorted by stride, every dimension has to step over all that the smaller ones span, as
// slices and transposes of dense tensors do.
void check_target(const Tensor& t, const char* name) {
    TORCH_CHECK(!(t.requires_grad() && at::GradMode::is_enabled()), name, " requires grad, and the call writes it in place without a history");
    if (t.numel() == 0) return;
    std::vector<std::pair<int64_t, int64_t>> dims;
    for (int64_t i = 0; i < t.dim(); ++i)
        if (t.size(i) > 1) dims.emplace_back(t.stride(i), t.size(i));
    std::sort(dims.begin(), dims.end());
    int64_t span = 1;
    for (const auto& [stride, size] : dims) {
        TORCH_CHECK(stride >= span, name, " is written in place, but elements of it share memory (sizes ", t.sizes(), ", strides ", t.strides(), ")");
        span += (size - 1) * stride;
    }
}
// A tensor that a call has written in place, for the graphs that saved it.  (Tensors of inference mode have no version.)
void written(const Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

const int32_t* ints(const OptTensor& t) { return t.has_value() ? t->const_data_ptr<int32_t>() : nullptr; }

// ---------------------------------------------------------------- window attention

struct WindowSizes { int64_t B, H, G, nq, nk, d, window, sinks, pad; };

WindowSizes check_window(const Tensor& q, const Tensor& k, const Tensor& v, py::handle window, py::handle sinks, const OptTensor& lens, const char* what) {
    check_gpu(q, "q"); check_gpu(k, "k"); check_gpu(v, "v");
    check_same(k, q, "k"); check_same(v, q, "v");
    TORCH_CHECK(q.dim() == 4 && k.dim() == 4, what, " expects (B, H, N, d) tensors, got ", q.dim(), "-D and ", k.dim(), "-D");
    TORCH_CHECK(k.sizes() == v.sizes() && k.size(0) == q.size(0) && k.size(3) == q.size(3) && q.size(2) <= k.size(2), "Wrong sizes!");
    TORCH_CHECK(q.scalar_type() == k.scalar_type() && q.scalar_type() == v.scalar_type(), "Scalar type mismatch!");
    const bool f32 = tag(q) == MYFA_F32;
    WindowSizes w{q.size(0), q.size(1), k.size(1), q.size(2), k.size(2), q.size(3), whole(window, "window"), whole(sinks, "sinks"), 0};
    TORCH_CHECK(w.H >= 1 && w.G >= 1 && w.H % w.G == 0, w.H, " query heads are not a multiple of ", w.G, " key/value heads");
    const int64_t most = f32 ? 128 : 256;
    TORCH_CHECK(w.d <= most, what, " supports head dims up to ", most, " for ", q.scalar_type(), ", got ", w.d);
    TORCH_CHECK(w.window >= 1 && w.sinks >= 0, "window must be an integer of at least 1 and sinks one of at least 0, got ", w.window, " and ", w.sinks);
    if (lens.has_value()) check_ints(*lens, {w.B}, q, "seq_lens");
    // zero columns up to the next head dim whose rows are whole 16-byte chunks change nothing (no columns at all get some, too:
    // the logits are 0, and the log-sum-exp is that of as many zeros as a row sees)
    const int64_t step = f32 ? 4 : 8;
    w.pad = w.d == 0 ? step : (step - w.d % step) % step;
    return w;
}

Tensor padded(const Tensor& t, int64_t n) { return at::constant_pad_nd(t, {0, n}); }

std::pair<Tensor, Tensor> window_fwd(const Tensor& q, const Tensor& k, const Tensor& v, const WindowSizes& w, double scale, bool want_lse, const OptTensor& lens) {
    if (w.pad) {
        WindowSizes p = w;
        p.d += w.pad;
        p.pad = 0;
        auto r = window_fwd(padded(q, w.pad), padded(k, w.pad), padded(v, w.pad), p, scale, want_lse, lens);
        return {r.first.narrow(3, 0, w.d).contiguous(), r.second};
    }
    const Strides qs(q, "q"), ks(k, "k"), vs(v, "v");
    const c10::DeviceGuard guard(q.device());
    Tensor out = at::empty({w.B, w.H, w.nq, w.d}, q.options().memory_format(at::MemoryFormat::Contiguous)), lse;
    if (want_lse) lse = at::empty({w.B, w.H, w.nq}, q.options().dtype(at::kFloat).memory_format(at::MemoryFormat::Contiguous));
    check(myfa_window_attn_fwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), want_lse ? lse.data_ptr<float>() : nullptr, ints(lens),
                               w.B, w.H, w.G, w.nq, w.nk, w.d, qs.s, ks.s, vs.s, w.window, w.sinks, (float)scale, tag(q), current_stream(q)));
    return {out, lse};
}

py::object window_attn_fwd(const Tensor& q, const Tensor& k, const Tensor& v, py::handle window, py::handle sinks, double scale, bool want_lse, const OptTensor& lens) {
    const WindowSizes w = check_window(q, k, v, window, sinks, lens, "window_attn_fwd");
    auto r = window_fwd(q, k, v, w, scale, want_lse, lens);
    if (!want_lse) return py::cast(r.first);
    return py::make_tuple(r.first, r.second);
}

std::vector<Tensor> window_bwd(const Tensor& dout, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& out, const Tensor& lse, const WindowSizes& w,
                               double scale, const OptTensor& lens) {
    if (w.pad) {
        WindowSizes p = w;
        p.d += w.pad;
        p.pad = 0;
        auto g = window_bwd(padded(dout, w.pad), padded(q, w.pad), padded(k, w.pad), padded(v, w.pad), padded(out, w.pad), lse, p, scale, lens);
        for (Tensor& t : g) t = t.narrow(3, 0, w.d).contiguous();
        return g;
    }
    const Strides qs(q, "q"), ks(k, "k"), vs(v, "v");
    const c10::DeviceGuard guard(q.device());
    const auto opt = q.options().memory_format(at::MemoryFormat::Contiguous);
    Tensor dq = at::empty({w.B, w.H, w.nq, w.d}, opt), dk = at::empty({w.B, w.G, w.nk, w.d}, opt), dv = at::empty({w.B, w.G, w.nk, w.d}, opt);
    const int64_t bytes = myfa_window_attn_bwd_ws_bytes(w.B, w.H, w.G, w.nq, w.nk, w.d, w.window, w.sinks, tag(q));
    Tensor ws = at::empty({bytes}, opt.dtype(at::kByte));
    check(myfa_window_attn_bwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr<float>(), dout.data_ptr(), dq.data_ptr(), dk.data_ptr(),
                               dv.data_ptr(), ints(lens), w.B, w.H, w.G, w.nq, w.nk, w.d, qs.s, ks.s, vs.s, w.window, w.sinks, (float)scale, tag(q),
                               ws.data_ptr(), bytes, current_stream(q)));
    return {dq, dk, dv};
}

py::tuple window_attn_bwd(const Tensor& dout, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& out, const Tensor& lse, py::handle window,
                          py::handle sinks, double scale, const OptTensor& lens) {
    const WindowSizes w = check_window(q, k, v, window, sinks, lens, "window_attn_bwd");
    check_dense(dout, q, "dout"); check_dense(out, q, "out"); check_dense(lse, q, "lse");
    TORCH_CHECK(q.sizes() == out.sizes() && q.sizes() == dout.sizes(), "Wrong sizes!");
    TORCH_CHECK(q.scalar_type() == out.scalar_type() && q.scalar_type() == dout.scalar_type(), "Scalar type mismatch!");
    TORCH_CHECK(lse.scalar_type() == at::kFloat && lse.sizes() == q.sizes().slice(0, 3), "lse must be the float32 (B, H, Nq) tensor returned by window_attn_fwd");
    auto g = window_bwd(dout, q, k, v, out, lse, w, scale, lens);
    return py::make_tuple(g[0], g[1], g[2]);
}

// (A function of Python's took 85 us for a forward and backward whose kernels take 43, this one takes 66.)
struct WindowAttn : torch::autograd::Function<WindowAttn> {
    static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const WindowSizes& w, double scale,
                          const OptTensor& lens) {
        auto r = window_fwd(q, k, v, w, scale, true, lens);
        ctx->save_for_backward({q, k, v, r.first, r.second, lens.has_value() ? *lens : Tensor()});
        const int64_t sizes[] = {w.B, w.H, w.G, w.nq, w.nk, w.d, w.window, w.sinks, w.pad};
        ctx->saved_data["sizes"] = at::IntArrayRef(sizes);
        ctx->saved_data["scale"] = scale;
        return r.first;
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list douts) {
        const auto saved = ctx->get_saved_variables();
        const auto s = ctx->saved_data["sizes"].toIntVector();
        const WindowSizes w{s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7], s[8]};
        Tensor dout = douts[0].contiguous();
        if (reinterpret_cast<uintptr_t>(dout.data_ptr()) % 16 != 0) dout = dout.clone();
        auto g = window_bwd(dout, saved[0], saved[1], saved[2], saved[3], saved[4], w, ctx->saved_data["scale"].toDouble(),
                            saved[5].defined() ? OptTensor(saved[5]) : OptTensor());
        if (at::GradMode::is_enabled()) {                 // (create_graph: the gradients' own gradients are an error, not zero)
            for (Tensor& t : g) t = t.detach().set_requires_grad(true);
            auto once = std::make_shared<torch::autograd::DelayedError>("window_attn_func can be differentiated once only", (int64_t)g.size());
            g = (*once)(std::move(g));
        }
        return {g[0], g[1], g[2], Tensor(), Tensor(), Tensor()};
    }
};

Tensor window_attn_func(const Tensor& q, const Tensor& k, const Tensor& v, py::handle window, py::handle sinks, double scale, const OptTensor& lens) {
    return WindowAttn::apply(q, k, v, check_window(q, k, v, window, sinks, lens, "window_attn_func"), scale, lens);
}

// ---------------------------------------------------------------- the paged cache

struct Cache {
    int64_t pages, heads, page, d, B, width;
    Strides ks, vs;
};

Cache check_cache(const Tensor& k, const Tensor& v, const Tensor& table, const Tensor& lens) {
    check_gpu(k, "k_cache"); check_gpu(v, "v_cache");
    check_same(v, k, "v_cache");
    TORCH_CHECK(k.dim() == 4 && k.sizes() == v.sizes(), "k_cache and v_cache must be (pages, heads, page, d) tensors of one shape");
    TORCH_CHECK(k.scalar_type() == v.scalar_type(), "Scalar type mismatch!");
    tag(k);
    TORCH_CHECK(k.size(1) >= 1 && k.size(2) >= 1 && k.size(3) >= 1, "a page holds at least one key of one head, of at least one column");
    TORCH_CHECK(table.dim() == 2, "block_table must be an int32 (B, width) tensor");
    check_ints(table, table.sizes(), k, "block_table");
    check_ints(lens, {table.size(0)}, k, "seq_lens");
    return {k.size(0), k.size(1), k.size(2), k.size(3), table.size(0), table.size(1), Strides(k, "k_cache"), Strides(v, "v_cache")};
}

void paged_kv_append(const Tensor& k, const Tensor& v, const Tensor& kc, const Tensor& vc, const Tensor& table, const Tensor& lens, const OptTensor& counts) {
    const Cache c = check_cache(kc, vc, table, lens);
    check_gpu(k, "k"); check_gpu(v, "v");
    check_same(k, kc, "k"); check_same(v, kc, "v");
    TORCH_CHECK(k.dim() == 4 && k.sizes() == v.sizes() && k.size(0) == c.B && k.size(1) == c.heads && k.size(3) == c.d, "Wrong sizes!");
    TORCH_CHECK(k.scalar_type() == kc.scalar_type() && v.scalar_type() == kc.scalar_type(), "Scalar type mismatch!");
    if (counts.has_value()) check_ints(*counts, {c.B}, kc, "counts");
    check_target(kc, "k_cache"); check_target(vc, "v_cache");
    const Strides ks(k, "k"), vs(v, "v");
    const c10::DeviceGuard guard(kc.device());
    check(myfa_paged_append(k.data_ptr(), v.data_ptr(), kc.data_ptr(), vc.data_ptr(), table.const_data_ptr<int32_t>(), lens.const_data_ptr<int32_t>(), ints(counts),
                            c.B, c.heads, k.size(2), c.d, c.pages, c.page, c.width, ks.s, vs.s, c.ks.s, c.vs.s, tag(kc), current_stream(kc)));
    written(kc);
    written(vc);
}

py::object paged_attn_decode(const Tensor& q, const Tensor& kc, const Tensor& vc, const Tensor& table, const Tensor& lens, double scale, py::handle window_,
                             py::handle sinks_, const OptTensor& sums, bool want_lse) {
    const Cache c = check_cache(kc, vc, table, lens);
    check_gpu(q, "q");
    check_same(q, kc, "q");
    TORCH_CHECK(q.dim() == 3 && q.size(0) == c.B && q.size(2) == c.d, "Wrong sizes!");
    TORCH_CHECK(q.scalar_type() == kc.scalar_type(), "Scalar type mismatch!");
    const int64_t H = q.size(1), window = whole(window_, "window"), sinks = whole(sinks_, "sinks");
    TORCH_CHECK(H >= 1 && H % c.heads == 0, H, " query heads are not a multiple of ", c.heads, " key/value heads");
    TORCH_CHECK(window >= 0 && sinks >= 0, "window and sinks must be integers of at least 0, got ", window, " and ", sinks);
    if (sums.has_value()) {
        check_sums(*sums, {c.B, c.heads, c.width * c.page}, kc);
        check_target(*sums, "weight_sum");
    }
    const Strides qs(q, "q");
    const c10::DeviceGuard guard(kc.device());
    const auto opt = q.options().memory_format(at::MemoryFormat::Contiguous);
    Tensor out = at::empty({c.B, H, c.d}, opt), lse, ws;
    if (want_lse) lse = at::empty({c.B, H}, opt.dtype(at::kFloat));
    const int64_t bytes = myfa_paged_attn_decode_ws_bytes(c.B, H, c.heads, c.d, c.page, c.width, window, sinks, sums.has_value());
    if (bytes > 0) ws = at::empty({bytes}, opt.dtype(at::kByte));
    check(myfa_paged_attn_decode(q.data_ptr(), kc.data_ptr(), vc.data_ptr(), table.const_data_ptr<int32_t>(), lens.const_data_ptr<int32_t>(), out.data_ptr(),
                                 want_lse ? lse.data_ptr<float>() : nullptr, sums.has_value() ? sums->data_ptr<float>() : nullptr, c.B, H, c.heads, c.d,
                                 c.pages, c.page, c.width, qs.s, c.ks.s, c.vs.s, window, sinks, (float)scale, tag(q), bytes > 0 ? ws.data_ptr() : nullptr, bytes,
                                 current_stream(kc)));
    if (sums.has_value()) written(*sums);
    if (!want_lse) return py::cast(out);
    return py::make_tuple(out, lse);
}

py::tuple paged_kv_evict(const Tensor& kc, const Tensor& vc, const Tensor& sums, const Tensor& table, const Tensor& lens, const Tensor& new_table, py::handle budget_,
                         py::handle sinks_, py::handle recent_) {
    const Cache c = check_cache(kc, vc, table, lens);
    check_sums(sums, {c.B, c.heads, c.width * c.page}, kc);
    check_target(kc, "k_cache"); check_target(vc, "v_cache");
    TORCH_CHECK(new_table.dim() == 2, "new_block_table must be an int32 (B, width) tensor");
    check_ints(new_table, {c.B, new_table.size(1)}, kc, "new_block_table");
    const int64_t budget = whole(budget_, "budget"), sinks = whole(sinks_, "sinks"), recent = whole(recent_, "recent"), capacity = new_table.size(1) * c.page;
    TORCH_CHECK(budget >= 1 && sinks >= 0 && recent >= 0 && sinks <= budget && recent <= budget - sinks, "budget (", budget, ") must be at least 1 and hold sinks (", sinks,
                ") and recent (", recent, ")");
    TORCH_CHECK(capacity >= budget, "new_block_table holds ", capacity, " keys a sequence, the budget is ", budget);
    const c10::DeviceGuard guard(kc.device());
    const auto opt = sums.options().memory_format(at::MemoryFormat::Contiguous);
    Tensor new_sums = at::empty({c.B, c.heads, capacity}, opt), new_lens = at::empty({c.B}, opt.dtype(at::kInt)), kept = at::empty({c.B, c.heads, budget}, opt.dtype(at::kInt));
    check(myfa_paged_evict(kc.data_ptr(), vc.data_ptr(), sums.const_data_ptr<float>(), table.const_data_ptr<int32_t>(), lens.const_data_ptr<int32_t>(),
                           new_table.const_data_ptr<int32_t>(), new_sums.data_ptr<float>(), new_lens.data_ptr<int32_t>(), kept.data_ptr<int32_t>(), c.B, c.heads, c.d,
                           c.pages, c.page, c.width, new_table.size(1), c.ks.s, c.vs.s, budget, sinks, recent, tag(kc), current_stream(kc)));
    written(kc);
    written(vc);
    return py::make_tuple(new_sums, new_lens, kept);
}

}  // namespace

PYBIND11_MODULE(_host, m) {
    m.def("window_attn_fwd", &window_attn_fwd);
    m.def("window_attn_bwd", &window_attn_bwd);
    m.def("window_attn_func", &window_attn_func);
    m.def("paged_kv_append", &paged_kv_append);
    m.def("paged_attn_decode", &paged_attn_decode);
    m.def("paged_kv_evict", &paged_kv_evict);
}
