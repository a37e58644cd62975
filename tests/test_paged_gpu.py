"""The paged cache on the GPU: append, attention of one new token, eviction by accumulated weight, and a run of them
together, against their definitions (float64 on the CPU; whole numbers and copies exactly)."""
import pytest
import torch

import window_reference as ref

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def mfa():
    import my_flash_attn_cuda
    assert torch.cuda.is_available()
    return my_flash_attn_cuda


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class Cache:
    """A pool whose every unused place is NaN, tables in no order with -1 behind a sequence's pages."""

    def __init__(self, lens, G, page, d, dtype, seed=0, spare=3, width=None, fill=True):
        self.gen = torch.Generator().manual_seed(seed)
        self.lens, self.page, self.G, self.d, self.dtype = lens, page, G, d, dtype
        B, self.width = len(lens), width or max(1, max(-(-n // page) for n in lens))
        used = [-(-n // page) for n in lens]
        self.pages = sum(used) + spare
        ids = torch.randperm(self.pages, generator=self.gen).tolist()
        self.table = torch.full((B, self.width), -1, dtype=torch.int32)
        self.free = ids
        for b in range(B):
            for j in range(used[b]):
                self.table[b, j] = self.free.pop()
        self.k_pool, self.v_pool = (torch.full((self.pages, G, page, d), float("nan")).to(dtype) for _ in range(2))
        self.k, self.v = ([torch.randn(G, n, d, generator=self.gen).to(dtype) for n in lens] for _ in range(2))
        if fill:
            for b, n in enumerate(lens):
                for j in range(n):
                    self.k_pool[self.table[b, j // page], :, j % page] = self.k[b][:, j]
                    self.v_pool[self.table[b, j // page], :, j % page] = self.v[b][:, j]

    def gpu(self):
        return self.k_pool.cuda(), self.v_pool.cuda(), self.table.cuda(), _i32(self.lens)


def _decode_reference(c, q, scale, window, sinks):
    """Per sequence: the definition of a sequence's last row."""
    outs = []
    for b, n in enumerate(c.lens):
        if n == 0:
            H = q.shape[1]
            outs.append({"out": (torch.zeros(H, c.d, dtype=torch.float64),) * 2,
                         "lse": (torch.full((H,), float("-inf"), dtype=torch.float64), torch.zeros(H, dtype=torch.float64)), "p": None})
            continue
        vis = ref.seen(1, n, window or n, sinks, n)[None]
        r = ref.attention(q[b][None, :, None], c.k[b][None], c.v[b][None], vis, scale, c.dtype)
        outs.append({"out": tuple(t[0, :, 0] for t in r["out"]), "lse": tuple(t[0, :, 0] for t in r["lse"]),
                     "p": tuple(t[0, :, 0] for t in r["p"])})
    return outs


def _check_decode(mfa, lens, H, G, page, d, window, sinks, dtype, weights, seed=0, width=None):
    c = Cache(lens, G, page, d, dtype, seed, width=width)
    q = torch.randn(len(lens), H, d, generator=c.gen).to(dtype)
    k_pool, v_pool, table, L = c.gpu()
    cap = c.width * page
    before = torch.rand(len(lens), G, cap, generator=c.gen)
    sums = before.cuda() if weights else None
    out, lse = mfa.paged_attn_decode(q.cuda(), k_pool, v_pool, table, L, scale=d ** -0.5, window=window, sinks=sinks,
                                     weight_sum=sums, return_lse=True)
    want = _decode_reference(c, q, d ** -0.5, window, sinks)
    for b, w in enumerate(want):
        ref.check(f"out[{b}]", out[b], w["out"])
        ref.check(f"lse[{b}]", lse[b], w["lse"])
        if weights:
            value, bound = before[b].double(), torch.zeros(G, cap, dtype=torch.float64)
            if w["p"] is not None:
                p, bp = (t.reshape(G, H // G, -1).sum(1) for t in w["p"])
                value[:, :lens[b]] += p
                bound[:, :lens[b]] += bp + (H // G + 2) * ref.W * p + 2 * ref.W * value[:, :lens[b]] * (p > 0)
            ref.check(f"weights[{b}]", sums[b], (value, bound))
    return out


DECODE = [
    # lens, H, G, page, d, window, sinks
    ([1], 1, 1, 16, 64, 0, 0),
    ([33], 8, 2, 16, 128, 0, 0),
    ([500, 0, 1, 31, 32, 513], 8, 2, 16, 128, 0, 0),
    ([700, 65, 300], 6, 6, 24, 64, 0, 0),                # pages that end inside a tile, one head per head
    ([300, 129], 12, 3, 64, 80, 0, 0),
    ([40, 200], 40, 2, 32, 64, 0, 0),                    # twenty query heads share one
    ([777, 50, 100], 8, 4, 16, 128, 100, 4),
    ([777, 130, 3], 4, 1, 5, 64, 64, 70),                # odd pages, sinks over more than one tile
    ([400], 2, 1, 16, 16, 1, 0),                         # the token sees itself alone
    ([97, 64], 4, 2, 1, 64, 0, 0),                       # pages of one key
    ([90], 4, 2, 128, 64, 1000, 3),                      # a page longer than the sequence
]


@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("case", DECODE, ids=lambda c: "-".join(map(str, c)).replace(" ", ""))
def test_decode(mfa, case, dtype, weights):
    _check_decode(mfa, *case, dtype, weights)


@pytest.mark.parametrize("d", [136, 192, 256])
def test_decode_wide_heads(mfa, d):
    _check_decode(mfa, [300, 77], 4, 2, 16, d, 0, 0, BF16, True)


def test_decode_long_and_split(mfa):
    """One long sequence beside a short one: many shares, most of them empty for the short one."""
    _check_decode(mfa, [9000, 40], 4, 1, 32, 128, 0, 0, BF16, True)
    _check_decode(mfa, [9000, 40], 4, 1, 32, 128, 2000, 4, F16, False)


@pytest.mark.parametrize("B,weights", [(40, False), (64, True), (65, False)])
def test_decode_many_sequences_of_unlike_lengths(mfa, B, weights):
    """Batches large and long enough that the sequences go longest first, with equal lengths and empty ones among them; and one
    sequence too many for that."""
    lens = [(37 * b * b) % 300 for b in range(B)]
    lens[7], lens[B - 1], lens[3], lens[4] = 4300, 0, 120, 120
    _check_decode(mfa, lens, 32, 32, 16, 16, 0, 0, BF16, weights)


def test_decode_table_wider_than_needed(mfa):
    _check_decode(mfa, [100, 20], 4, 2, 16, 64, 0, 0, BF16, True, width=400)


def test_decode_sinks_are_inside_the_window(mfa):
    c = Cache([50], 1, 16, 64, BF16, 3)
    q = torch.randn(1, 4, 64, generator=c.gen).to(BF16).cuda()
    args = c.gpu()
    a = mfa.paged_attn_decode(q, *args, scale=0.125)
    assert torch.equal(a, mfa.paged_attn_decode(q, *args, scale=0.125, window=50, sinks=7))


def test_decode_far_pages(mfa):
    """Offsets beyond 2^32 bytes: the used pages stand at the end of a pool of more than 4 GiB."""
    page, G, d, pages = 64, 2, 128, 140000
    k_pool = torch.empty(pages, G, page, d, device="cuda", dtype=BF16)
    v_pool = torch.empty(pages, G, page, d, device="cuda", dtype=BF16)
    assert k_pool.numel() * 2 > 1 << 32
    c = Cache([150], G, page, d, BF16, 4)
    table = (c.table + pages - c.pages).cuda()
    table[c.table.cuda() < 0] = -1
    new = [torch.stack(t)[:, :, :].cuda() for t in (c.k, c.v)]
    mfa.paged_kv_append(*new, k_pool, v_pool, table, _i32([0]))
    q = torch.randn(1, 4, d, generator=c.gen).to(BF16)
    out = mfa.paged_attn_decode(q.cuda(), k_pool, v_pool, table, _i32([150]), scale=0.09)
    ref.check("out", out[0], _decode_reference(c, q, 0.09, 0, 0)[0]["out"])


def test_decode_bad_pages_and_lengths(mfa):
    """A page number outside the pool, or a length beyond the table, makes that sequence NaN and no other."""
    c = Cache([100, 100, 100, 100], 2, 16, 64, BF16, 5)
    q = torch.randn(4, 4, 64, generator=c.gen).to(BF16)
    k_pool, v_pool, table, _ = c.gpu()
    table[1, 3] = c.pages
    table[2, 0] = -5
    sums = torch.zeros(4, 2, c.width * 16, device="cuda")
    out = mfa.paged_attn_decode(q.cuda(), k_pool, v_pool, table, _i32([100, 100, 100, c.width * 16 + 1]), scale=0.125, weight_sum=sums)
    assert torch.isnan(out[1:]).all()
    ref.check("out", out[0], _decode_reference(c, q, 0.125, 0, 0)[0]["out"])
    assert torch.isfinite(sums[0]).all()
    # a bad page that nothing sees does not matter, nor does a negative length
    out = mfa.paged_attn_decode(q.cuda(), k_pool, v_pool, table, _i32([100, 100, 100, -3]), scale=0.125, window=20)
    assert torch.isfinite(out).all() and not out[3].any()


def test_decode_strided(mfa):
    """Caches of (pages, page, heads, d) order and of interleaved keys and values, q a slice: the same bits."""
    c = Cache([200, 90], 2, 16, 64, BF16, 6)
    q = torch.randn(2, 4, 64, generator=c.gen).to(BF16).cuda()
    k_pool, v_pool, table, L = c.gpu()
    want = mfa.paged_attn_decode(q, k_pool, v_pool, table, L, scale=0.125)
    kt, vt = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (k_pool, v_pool))
    both = torch.stack([k_pool, v_pool], 1)
    wide = torch.zeros(2, 12, 64, device="cuda", dtype=BF16)
    wide[:, 4:8] = q
    assert torch.equal(want, mfa.paged_attn_decode(q, kt, vt, table, L, scale=0.125))
    assert torch.equal(want, mfa.paged_attn_decode(wide[:, 4:8], both[:, 0], both[:, 1], table, L, scale=0.125))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("G,page,d,n", [(2, 16, 64, 1), (3, 24, 80, 37), (1, 5, 128, 200), (2, 1, 8, 3)])
def test_append(mfa, dtype, G, page, d, n):
    lens, counts = [0, 7, 30], [n, n - 1, 0]
    c = Cache([x + n for x in lens], G, page, d, dtype, 7, fill=False)
    k_pool, v_pool, table, _ = c.gpu()
    new = torch.randn(3, n, 2, G, d, generator=c.gen).to(dtype)
    k, v = new[:, :, 0].transpose(1, 2), new[:, :, 1].transpose(1, 2)                   # strided, (B, G, n, d)
    for cnt in (None, counts):
        want_k, want_v = c.k_pool.clone(), c.v_pool.clone()
        for b in range(3):
            for t in range(n if cnt is None else cnt[b]):
                at = lens[b] + t
                want_k[c.table[b, at // page], :, at % page] = k[b, :, t]
                want_v[c.table[b, at // page], :, at % page] = v[b, :, t]
        kp, vp = k_pool.clone(), v_pool.clone()
        gk = new.cuda()
        mfa.paged_kv_append(gk[:, :, 0].transpose(1, 2), gk[:, :, 1].transpose(1, 2), kp, vp, table, _i32(lens),
                            counts=None if cnt is None else _i32(cnt))
        # (the rest of the pool, NaN here, is left as it was)
        assert torch.equal(kp.cpu().nan_to_num(9.0), want_k.nan_to_num(9.0))
        assert torch.equal(vp.cpu().nan_to_num(9.0), want_v.nan_to_num(9.0))


def test_append_drops_what_has_no_place(mfa):
    c = Cache([16, 16, 16], 1, 8, 16, BF16, 8, fill=False)
    k_pool, v_pool, table, _ = c.gpu()
    table[1, 1] = c.pages + 7
    table[2, 0] = -1
    k = torch.ones(3, 1, 4, 16, device="cuda", dtype=BF16)
    mfa.paged_kv_append(k, k, k_pool, v_pool, table, _i32([14, 6, -2]))
    written = [(int(table[0, 1]), 6), (int(table[0, 1]), 7), (int(table[1, 0]), 6), (int(table[1, 0]), 7)]
    want = torch.full((c.pages, 8), False)
    for p, s in written:
        want[p, s] = True
    for pool in (k_pool, v_pool):
        assert torch.equal(torch.isfinite(pool).all(-1)[:, 0].cpu(), want)


def _evict_reference(sums, lens, budget, sinks, recent):
    kept = []
    for b, n in enumerate(lens):
        rows = []
        for g in range(sums.shape[1]):
            if n <= budget:
                rows.append(list(range(n)))
                continue
            order = sorted(range(sinks, n - recent), key=lambda j: (-float("inf") if sums[b, g, j] != sums[b, g, j] else -float(sums[b, g, j]),
                                                                    0 if sums[b, g, j] != sums[b, g, j] else 1, j))
            rows.append(sorted(list(range(sinks)) + order[:budget - sinks - recent] + list(range(n - recent, n))))
        kept.append(rows)
    return kept


EVICT = [
    # lens, G, page, d, budget, sinks, recent
    ([100], 1, 16, 64, 40, 4, 8),
    ([100, 30, 0, 41, 40], 2, 16, 64, 40, 4, 8),
    ([9000, 300], 2, 24, 16, 777, 1, 100),
    ([8192, 8191], 1, 16, 8, 3000, 0, 7),
    ([30000], 1, 32, 8, 1111, 4, 64),
    ([5000], 1, 32, 8, 4999, 0, 0),
    ([64, 200], 3, 16, 80, 16, 4, 12),                 # nothing is left for the weights
    ([300], 2, 7, 64, 1, 0, 0),
    ([300], 2, 16, 64, 50, 0, 50),
]


@pytest.mark.parametrize("kind", ["plain", "ties", "zeros", "odd"])
@pytest.mark.parametrize("case", EVICT, ids=lambda c: "-".join(map(str, c)).replace(" ", ""))
def test_evict(mfa, case, kind):
    lens, G, page, d, budget, sinks, recent = case
    dtype = {"plain": BF16, "ties": F16, "zeros": F32, "odd": BF16}[kind]
    new_width = -(-budget // page) + (kind == "ties")
    c = Cache(lens, G, page, d, dtype, 9, spare=len(lens) * new_width)
    B, cap = len(lens), c.width * page
    sums = torch.randn(B, G, cap, generator=c.gen).exp()
    if kind == "ties":
        sums = (sums * 3).floor()
    if kind == "zeros":
        sums = torch.where(torch.rand(sums.shape, generator=c.gen) < 0.5, 0.0, -0.0)
    if kind == "odd":                                   # negative sums, infinities, NaN
        sums = torch.randn(B, G, cap, generator=c.gen)
        pick = torch.rand(sums.shape, generator=c.gen)
        sums = torch.where(pick < 0.02, float("inf"), torch.where(pick < 0.04, float("-inf"), torch.where(pick < 0.05, float("nan"), sums)))
    new_table = torch.full((B, new_width), -1, dtype=torch.int32)
    for b, n in enumerate(lens):
        for j in range(-(-min(n, budget) // page)):
            new_table[b, j] = c.free.pop()
    k_pool, v_pool, table, L = c.gpu()
    new_sums, new_lens, kept = mfa.paged_kv_evict(k_pool, v_pool, sums.cuda(), table, L, new_table.cuda(), budget, sinks=sinks, recent=recent)
    want = _evict_reference(sums, lens, budget, sinks, recent)
    assert new_lens.cpu().tolist() == [min(n, budget) for n in lens]
    want_k, want_v = c.k_pool.clone(), c.v_pool.clone()
    for b in range(B):
        for g in range(G):
            rows = want[b][g]
            assert kept[b, g].cpu().tolist() == rows + [-1] * (budget - len(rows)), (b, g)
            moved = torch.zeros(new_width * page)
            moved[:len(rows)] = sums[b, g][rows]
            assert torch.equal(new_sums[b, g].cpu().nan_to_num(7.5), moved.nan_to_num(7.5))
            for i, j in enumerate(rows):
                p, s = int(new_table[b, i // page]), i % page
                want_k[p, g, s], want_v[p, g, s] = c.k[b][g, j], c.v[b][g, j]
    assert torch.equal(k_pool.cpu().nan_to_num(9.0), want_k.nan_to_num(9.0))
    assert torch.equal(v_pool.cpu().nan_to_num(9.0), want_v.nan_to_num(9.0))


def test_evict_bad_pages(mfa):
    c = Cache([64, 64], 1, 16, 16, BF16, 10, spare=4)
    k_pool, v_pool, table, L = c.gpu()
    new_table = torch.tensor([[c.free.pop(), c.pages + 3], [c.free.pop(), c.free.pop()]], dtype=torch.int32, device="cuda")
    table[1, 0] = -7
    sums = torch.zeros(2, 1, 64, device="cuda")
    before = k_pool.clone()
    _, lens, kept = mfa.paged_kv_evict(k_pool, v_pool, sums, table, L, new_table, 32, sinks=16, recent=16)
    assert lens.tolist() == [32, 32]
    assert torch.equal(k_pool[new_table[0, 0]].cpu()[0], c.k[0][0, :16])
    assert torch.isnan(k_pool[new_table[1, 0]]).all()
    assert torch.equal(v_pool[new_table[1, 1]].cpu()[0], c.v[1][0, 48:])
    same = torch.ones(c.pages, dtype=torch.bool, device="cuda")
    same[new_table[0, 0]] = same[new_table[1, 0]] = same[new_table[1, 1]] = False
    assert torch.equal(k_pool[same].nan_to_num(9.0), before[same].nan_to_num(9.0))


@pytest.mark.parametrize("case", [([5000, 40, 300], 2, 16, 16, 300, 4, 20), ([2048, 2049], 1, 16, 128, 128, 0, 0), ([2049], 1, 16, 128, 129, 1, 1),
                                  ([1000], 1, 10, 64, 256, 4, 32), ([1000], 1, 10, 64, 257, 4, 32)], ids=lambda c: "-".join(map(str, c)).replace(" ", ""))
@pytest.mark.parametrize("kind", ["plain", "ties"])
def test_evict_around_one_launch(mfa, case, kind):
    """Sizes on both sides of what the selection moves by itself."""
    test_evict(mfa, case, kind)


def test_evict_bad_pages_of_many_keys(mfa):
    """The same as test_evict_bad_pages where a second launch moves the keys."""
    c = Cache([640, 640], 1, 16, 128, BF16, 11, spare=40)
    k_pool, v_pool, table, L = c.gpu()
    new = [[c.free.pop() for _ in range(20)] for _ in range(2)]
    new[0][7] = c.pages + 3
    new_table = torch.tensor(new, dtype=torch.int32, device="cuda")
    table[1, 2] = -7
    before = k_pool.clone()
    mfa.paged_kv_evict(k_pool, v_pool, torch.zeros(2, 1, 640, device="cuda"), table, L, new_table, 320, sinks=160, recent=160)
    same = torch.ones(c.pages, dtype=torch.bool, device="cuda")
    for b in range(2):
        for i in range(20):
            if (b, i) == (0, 7):
                continue
            at = 16 * i if i < 10 else 640 - 320 + 16 * i
            same[new[b][i]] = False
            if (b, i) == (1, 2):
                assert torch.isnan(k_pool[new[b][i]]).all() and torch.isnan(v_pool[new[b][i]]).all()
            else:
                assert torch.equal(k_pool[new[b][i]].cpu()[0], c.k[b][0, at:at + 16]) and torch.equal(v_pool[new[b][i]].cpu()[0], c.v[b][0, at:at + 16])
    assert torch.equal(k_pool[same].nan_to_num(9.0), before[same].nan_to_num(9.0))


def test_prefill_append_decode_evict(mfa):
    """A padded batch of prompts through window attention into the cache, tokens decoded with the same window, the
    cache cut by the weights, and decoding on: every step against the definition on the keys it should see."""
    torch.manual_seed(0)
    H, G, d, page, window, sinks, scale = 4, 2, 64, 16, 24, 4, 0.125
    prompt, steps = [70, 33], 3
    B, N = 2, max(prompt)
    width = -(-(N + 8) // page)
    q, k, v = (torch.randn(B, n, N + 8, d).to(BF16) for n in (H, G, G))
    vis = torch.stack([ref.seen(N, N, window, sinks, n) for n in prompt])
    L = _i32(prompt)
    out = mfa.window_attn_fwd(*(t[:, :, :N].cuda() for t in (q, k, v)), window, sinks=sinks, scale=scale, seq_lens=L)
    ref.check("prefill", out, ref.attention(*(t[:, :, :N] for t in (q, k, v)), vis, scale, BF16)["out"])

    pool = torch.full((B * width * 2, 2, G, page, d), float("nan"), device="cuda", dtype=BF16)
    k_pool, v_pool = pool[:, 0], pool[:, 1]
    ids = torch.randperm(B * width * 2).to(torch.int32)
    table, new_table = ids[:B * width].view(B, width).cuda(), ids[B * width:].view(B, width).cuda()
    zero = torch.zeros_like(L)
    mfa.paged_kv_append(*(t[:, :, :N].cuda() for t in (k, v)), k_pool, v_pool, table, zero, counts=L)
    sums = torch.zeros(B, G, width * page, device="cuda")
    held = [{x: t[b, :, :prompt[b]] for x, t in (("k", k), ("v", v))} for b in range(B)]
    want_sums = torch.zeros(B, G, width * page, dtype=torch.float64)
    bound = torch.zeros_like(want_sums)

    def token(at, window, sinks):
        """One token per sequence, number `at` of each sequence's remaining rows; checks it."""
        nonlocal L
        kt, vt, qt = (torch.stack([t[b, :, prompt[b] + at] for b in range(B)]) for t in (k, v, q))
        mfa.paged_kv_append(kt[:, :, None].cuda(), vt[:, :, None].cuda(), k_pool, v_pool, table, L)
        L = L + 1
        out = mfa.paged_attn_decode(qt.cuda(), k_pool, v_pool, table, L, scale=scale, window=window, sinks=sinks, weight_sum=sums)
        for b in range(B):
            for x, t in (("k", kt), ("v", vt)):
                held[b][x] = torch.cat([held[b][x], t[b][:, None]], 1)
            n = held[b]["k"].shape[1]
            r = ref.attention(qt[b][None, :, None], held[b]["k"][None], held[b]["v"][None], ref.seen(1, n, window or n, sinks, n)[None], scale, BF16)
            ref.check(f"decode {at} of {b}", out[b], tuple(t[0, :, 0] for t in r["out"]))
            want_sums[b, :, :n] += r["p"][0][0, :, 0].reshape(G, H // G, n).sum(1)
            bound[b, :, :n] += r["p"][1][0, :, 0].reshape(G, H // G, n).sum(1) + 8 * ref.W
    for at in range(steps):
        token(at, window, sinks)
    ref.check("sums", sums, (want_sums, bound))
    for at in range(steps, steps + 2):
        token(at, 0, 0)
    old = [{x: t.clone() for x, t in h.items()} for h in held]
    budget = 40
    sums, L, kept = mfa.paged_kv_evict(k_pool, v_pool, sums, table, L, new_table, budget, sinks=4, recent=8)
    table = new_table
    assert L.tolist() == [budget, 38]
    for b in range(B):
        rows = kept[b].cpu().long()
        assert [r[:4].tolist() for r in rows] == [[0, 1, 2, 3]] * G
        for x in ("k", "v"):
            held[b][x] = torch.stack([old[b][x][g, rows[g][rows[g] >= 0]] for g in range(G)])
    want_sums = sums.cpu().double()
    for at in range(steps + 2, steps + 4):
        token(at, 0, 0)
    ref.check("sums", sums, (want_sums, bound * 0 + 64 * ref.W + want_sums * 4 * ref.W))


def test_decode_same_result_every_time_and_on_another_stream(mfa):
    c = Cache([3000, 1200], 2, 16, 128, BF16, 11)
    q = torch.randn(2, 8, 128, generator=c.gen).to(BF16).cuda()
    args = c.gpu()
    want, wsum = None, None
    torch.cuda.synchronize()
    for stream in (torch.cuda.current_stream(), torch.cuda.Stream(), torch.cuda.Stream()):
        with torch.cuda.stream(stream):
            sums = torch.zeros(2, 2, c.width * 16, device="cuda")
            out = mfa.paged_attn_decode(q, *args, scale=0.1, weight_sum=sums)
        stream.synchronize()
        if want is None:
            want, wsum = out, sums
        assert torch.equal(out, want) and torch.equal(sums, wsum)


def test_graph_replays(mfa):
    """Append, decode and evict captured together and replayed over new tokens, each replay against eager calls; a
    second graph of the same calls shares nothing with it."""
    c = Cache([300, 100], 2, 16, 64, BF16, 12, spare=8, width=20)
    B, H = 2, 4
    for b in range(B):                                   # room for the new token's page
        c.table[b, -(-c.lens[b] // 16)] = c.free.pop()
    new_table = torch.tensor([[c.free.pop(), c.free.pop()] for _ in range(B)], dtype=torch.int32, device="cuda")
    k_pool, v_pool, table, L = c.gpu()
    q, k, v = torch.zeros(B, H, 64, device="cuda", dtype=BF16), *(torch.zeros(B, 2, 1, 64, device="cuda", dtype=BF16) for _ in range(2))
    base = torch.rand(B, 2, 20 * 16, device="cuda")

    def step(kp, vp):
        sums = base.clone()
        mfa.paged_kv_append(k, v, kp, vp, table, L)
        out = mfa.paged_attn_decode(q, kp, vp, table, L + 1, scale=0.125, window=64, sinks=4, weight_sum=sums)
        return (out, sums, *mfa.paged_kv_evict(kp, vp, sums, table, L + 1, new_table, 32, sinks=2, recent=8))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(k_pool.clone(), v_pool.clone())
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        kp, vp, graph = k_pool.clone(), v_pool.clone(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = step(kp, vp)
        graphs.append((graph, held, kp, vp))
    for r in range(3):
        gen = torch.Generator().manual_seed(50 + r)
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=gen))
        for graph, *_ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        ek, ev = k_pool.clone(), v_pool.clone()
        want = (*step(ek, ev), ek, ev)
        for _, held, kp, vp in graphs:
            for a, b in zip((*held, kp, vp), want):
                assert torch.equal(a.float().nan_to_num(9.0), b.float().nan_to_num(9.0))


def test_refusals(mfa):
    c = Cache([40], 2, 16, 64, BF16, 13)
    k_pool, v_pool, table, L = c.gpu()
    q = torch.zeros(1, 4, 64, device="cuda", dtype=BF16)
    sums = torch.zeros(1, 2, c.width * 16, device="cuda")
    new = torch.zeros(1, 2, 1, 64, device="cuda", dtype=BF16)
    nt = torch.zeros(1, 2, device="cuda", dtype=torch.int32)
    dec, app, ev = mfa.paged_attn_decode, mfa.paged_kv_append, mfa.paged_kv_evict
    bad = [
        (lambda: dec(q[:, :3].contiguous(), k_pool, v_pool, table, L), "multiple"),
        (lambda: dec(q.half(), k_pool, v_pool, table, L), "Scalar type"),
        (lambda: dec(q[:, :, :32].contiguous(), k_pool, v_pool, table, L), "Wrong sizes"),
        (lambda: dec(q, k_pool, v_pool[:, :, :8].contiguous(), table, L), "one shape"),
        (lambda: dec(q, k_pool, v_pool, table.long(), L), "int32"),
        (lambda: dec(q, k_pool, v_pool, table[0], L), "block_table"),
        (lambda: dec(q, k_pool, v_pool, table, L.repeat(2)), "int32"),
        (lambda: dec(q, k_pool, v_pool, table, L.cpu()), "CUDA tensor"),
        (lambda: dec(q, k_pool, v_pool, table, L, window=-1), "window"),
        (lambda: dec(q, k_pool, v_pool, table, L, sinks=1.5), "sinks"),
        (lambda: dec(q, k_pool, v_pool, table, L, scale=-1.0), "scale"),
        (lambda: dec(q, k_pool, v_pool, table, L, scale=float("inf")), "scale"),
        (lambda: dec(q, k_pool, v_pool, table, L, weight_sum=sums[:, :, 1:].contiguous()), "weight_sum must"),
        (lambda: dec(q, k_pool, v_pool, table, L, weight_sum=sums.half()), "Float"),
        (lambda: dec(q, k_pool, v_pool, table, L, weight_sum=sums.transpose(1, 2).contiguous().transpose(1, 2)), "contiguous"),
        (lambda: dec(torch.zeros(1, 4, 60, device="cuda", dtype=BF16), k_pool[..., :60], v_pool[..., :60], table, L), "16 bytes|head dim"),
        (lambda: dec(q, k_pool.double(), v_pool.double(), table, L), "unsupported dtype"),
        (lambda: dec(*(torch.zeros(s, device="cuda") for s in ((1, 4, 256), (3, 2, 16, 256), (3, 2, 16, 256))), table, L), "head dim"),
        (lambda: app(new[:, :1], new[:, :1], k_pool, v_pool, table, L), "Wrong sizes"),
        (lambda: app(new, new.half(), k_pool, v_pool, table, L), "Scalar type"),
        (lambda: app(new, new, k_pool, v_pool, table, L, counts=L.long()), "int32"),
        (lambda: ev(k_pool, v_pool, sums, table, L, nt, 0), "budget"),
        (lambda: ev(k_pool, v_pool, sums, table, L, nt, 8, sinks=5, recent=4), "budget"),
        (lambda: ev(k_pool, v_pool, sums, table, L, nt, 33), "holds 32 keys"),
        (lambda: ev(k_pool, v_pool, sums, table, L, nt.repeat(2, 1), 16), "int32"),
        (lambda: ev(k_pool, v_pool, sums[0], table, L, nt, 16), "weight_sum must"),
    ]
    for call, match in bad:
        with pytest.raises(RuntimeError, match=match):
            call()


def test_empty_batch(mfa):
    k_pool = torch.zeros(4, 2, 16, 64, device="cuda", dtype=BF16)
    table, L = torch.zeros(0, 3, device="cuda", dtype=torch.int32), torch.zeros(0, device="cuda", dtype=torch.int32)
    assert mfa.paged_attn_decode(torch.zeros(0, 4, 64, device="cuda", dtype=BF16), k_pool, k_pool, table, L).shape == (0, 4, 64)
    mfa.paged_kv_append(*(torch.zeros(0, 2, 1, 64, device="cuda", dtype=BF16) for _ in range(2)), k_pool, k_pool, table, L)
    sums, lens, kept = mfa.paged_kv_evict(k_pool, k_pool, torch.zeros(0, 2, 48, device="cuda"), table, L,
                                          torch.zeros(0, 2, device="cuda", dtype=torch.int32), 20)
    assert sums.shape == (0, 2, 32) and lens.shape == (0,) and kept.shape == (0, 2, 20)


@pytest.mark.parametrize("weights", [False, True])
def test_decode_with_no_pages_at_all(mfa, weights):
    """A table of width 0 holds nothing: a length of 0 gives 0, any other lies beyond the capacity."""
    k_pool = torch.zeros(4, 2, 16, 64, device="cuda", dtype=BF16)
    q = torch.ones(3, 4, 64, device="cuda", dtype=BF16)
    sums = torch.zeros(3, 2, 0, device="cuda") if weights else None
    out, lse = mfa.paged_attn_decode(q, k_pool, k_pool, _i32([[], [], []]), _i32([0, 1, 40]), weight_sum=sums, return_lse=True)
    assert not out[0].any() and (lse[0] == float("-inf")).all()
    assert torch.isnan(out[1:]).all() and torch.isnan(lse[1:]).all()


def test_writes_in_place_are_seen_by_autograd(mfa):
    """What a call writes in place gets a new version, so that a graph that saved it is not run over other values."""
    c = Cache([100, 40], 2, 16, 64, BF16, 14, spare=8, width=10)
    for b in range(2):
        c.table[b, -(-c.lens[b] // 16)] = c.free.pop()
    new_table = torch.tensor([[c.free.pop(), c.free.pop()] for _ in range(2)], dtype=torch.int32, device="cuda")
    k_pool, v_pool, table, L = c.gpu()
    new = torch.ones(2, 2, 1, 64, device="cuda", dtype=BF16)
    sums = torch.zeros(2, 2, 160, device="cuda")
    calls = {
        "append": (lambda: mfa.paged_kv_append(new, new, k_pool, v_pool, table, L), (k_pool, v_pool)),
        "decode": (lambda: mfa.paged_attn_decode(new[:, :, 0], k_pool, v_pool, table, L, weight_sum=sums), (sums,)),
        "evict": (lambda: mfa.paged_kv_evict(k_pool, v_pool, sums, table, L, new_table, 32), (k_pool, v_pool)),
    }
    for name, (call, written) in calls.items():
        everything = (k_pool, v_pool, sums, table, L, new_table, new)
        before = [t._version for t in everything]
        call()
        for t, n in zip(everything, before):
            assert (t._version > n) == any(t is x for x in written), name
    w = torch.randn(k_pool.shape, device="cuda", dtype=BF16, requires_grad=True)
    saved = (w * v_pool).sum()
    mfa.paged_kv_append(new, new, k_pool, v_pool, table, L)
    with pytest.raises(RuntimeError, match="inplace"):
        saved.backward()
    # tensors of inference mode have no version
    with torch.inference_mode():
        pools = [t.clone() for t in (k_pool, v_pool)]
        mfa.paged_kv_append(new, new, *pools, table, L)
    mfa.paged_kv_append(new, new, *pools, table, L)
    assert torch.equal(pools[0].nan_to_num(9.0), k_pool.nan_to_num(9.0))


def test_writes_in_place_are_refused_where_they_cannot_be_made(mfa):
    """A cache whose places share memory, and a tensor whose history autograd would have to keep."""
    c = Cache([20, 20], 2, 16, 64, BF16, 15, spare=4)
    k_pool, v_pool, table, L = c.gpu()
    new = torch.ones(2, 2, 1, 64, device="cuda", dtype=BF16)
    nt = torch.tensor([[c.free.pop()], [c.free.pop()]], dtype=torch.int32, device="cuda")
    sums, q = torch.zeros(2, 2, 32, device="cuda"), torch.ones(2, 4, 64, device="cuda", dtype=BF16)
    shared = [k_pool[:, :1].expand(-1, 2, -1, -1),                                                 # one head for all
              k_pool[:1].expand(c.pages, -1, -1, -1),
              torch.zeros(c.pages * 4096, device="cuda", dtype=BF16).as_strided(k_pool.shape, (2048, 1024, 32, 1))]     # rows half over each other
    for x in shared:
        for pools in ((x, v_pool), (v_pool, x)):
            with pytest.raises(RuntimeError, match="share memory"):
                mfa.paged_kv_append(new, new, *pools, table, L)
            with pytest.raises(RuntimeError, match="share memory"):
                mfa.paged_kv_evict(*pools, sums, table, L, nt, 16)
        mfa.paged_attn_decode(q, x, x, table, L, weight_sum=sums)                                  # reads alone
    grad = v_pool.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="requires grad"):
        mfa.paged_kv_append(new, new, k_pool, grad, table, L)
    with pytest.raises(RuntimeError, match="requires grad"):
        mfa.paged_kv_evict(grad, k_pool, sums, table, L, nt, 16)
    with pytest.raises(RuntimeError, match="requires grad"):
        mfa.paged_attn_decode(q, k_pool, v_pool, table, L, weight_sum=sums.clone().requires_grad_())
    with torch.no_grad():
        mfa.paged_kv_append(new, new, k_pool, grad, table, L)
    # (pages, page, heads, d) pools, interleaved ones and slices hold every place once
    both = torch.zeros(c.pages, 16, 2, 2, 72, device="cuda", dtype=BF16)[..., :64]
    mfa.paged_kv_append(new, new, both[:, :, 0].transpose(1, 2), both[:, :, 1].transpose(1, 2), table, L)
    assert both.sum() == 2 * 2 * 2 * 64


def test_caches_of_no_columns_are_refused(mfa):
    pool, L, table = torch.zeros(2, 1, 16, 0, device="cuda", dtype=BF16), _i32([3]), _i32([[1]])
    sums = torch.zeros(1, 1, 16, device="cuda")
    for call in (lambda: mfa.paged_attn_decode(torch.zeros(1, 1, 0, device="cuda", dtype=BF16), pool, pool, table, L, weight_sum=sums, return_lse=True),
                 lambda: mfa.paged_kv_append(pool[:1], pool[:1], pool, pool, table, L), lambda: mfa.paged_kv_evict(pool, pool, sums, table, L, table, 4)):
        with pytest.raises(RuntimeError, match="at least one column"):
            call()


def test_results_do_not_depend_on_fresh_memory(mfa):
    """Outputs and workspaces filled with NaN (whole numbers with their largest) before the call change nothing: torch does that to fresh
    memory in its deterministic mode."""
    def calls():
        for lens, H, G, page, d, window, sinks, width in (([500, 0, 1, 31, 513], 8, 2, 16, 128, 0, 0, None), ([40, 200], 40, 2, 32, 64, 0, 0, 64),
                                                          ([5000, 40], 4, 1, 32, 80, 700, 4, None), ([3000, 90, 0], 4, 2, 24, 128, 0, 0, 400)):
            c = Cache(lens, G, page, d, BF16, 16, spare=8 * len(lens), width=width)
            q = torch.randn(len(lens), H, d, generator=c.gen).to(BF16).cuda()
            args = c.gpu()
            sums = torch.rand(len(lens), G, c.width * page, generator=c.gen).cuda()
            yield mfa.paged_attn_decode(q, *args, scale=0.1, window=window, sinks=sinks, return_lse=True)
            yield (*mfa.paged_attn_decode(q, *args, scale=0.1, window=window, sinks=sinks, weight_sum=sums, return_lse=True), sums)
            for budget in (17, 100):
                new_table = torch.full((len(lens), 8), -1, dtype=torch.int32)
                for b, n in enumerate(lens):
                    for j in range(-(-min(n, budget) // page)):
                        new_table[b, j] = c.free[8 * b + j]
                yield (*mfa.paged_kv_evict(*args[:2], sums, *args[2:], new_table.cuda(), budget, sinks=2, recent=5), *args[:2])
    want = [[t.clone() for t in x] for x in calls()]
    before = torch.are_deterministic_algorithms_enabled(), torch.utils.deterministic.fill_uninitialized_memory
    try:
        torch.use_deterministic_algorithms(True, warn_only=True)
        torch.utils.deterministic.fill_uninitialized_memory = True
        assert torch.isnan(torch.empty(5, device="cuda")).all()
        for x, y in zip(calls(), want):
            assert len(x) == len(y) and all(torch.equal(a.float().nan_to_num(9.0), b.float().nan_to_num(9.0)) for a, b in zip(x, y))
    finally:
        torch.use_deterministic_algorithms(before[0])
        torch.utils.deterministic.fill_uninitialized_memory = before[1]
