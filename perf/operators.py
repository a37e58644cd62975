"""The cases on which the serving and long-context operators are measured, with their plain forms.

Four operators that a language model with a sliding window and a paged cache runs together:

  window   attention in which a query sees the last `window` keys up to its own position and the first
           `sinks` keys; forward, and forward with gradients; grouped key/value heads, padded batches
  append   the keys and values of new tokens go into their places in a paged cache
  decode   attention of one new token per sequence over that cache, by choice with the same window and
           sinks, and by choice adding the weights it formed to a running sum per cached key
  evict    the cache is cut to `budget` keys per head: the first `sinks`, the last `recent` and of the rest
           those with the largest sums of weights (ties: the lowest index), copied to new pages in order

`listed()` has the measured cases, `draw()` more of the same ranges, `run()` one pass: elementary torch
operations in float32, or, with `own` set, the calls that a user makes of my_flash_attn_cuda.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _package():
    if "my_flash_attn_cuda" not in sys.modules:
        sys.path.insert(0, os.path.join(os.getcwd(), "flash-attention_amd"))
    import my_flash_attn_cuda
    return my_flash_attn_cuda


# ------------------------------------------------------------------ the cases

def listed():
    return [
        # a short prompt of one request: launches are what counts
        _window("window prompt", 1, 8, 8, 128, 128, 64, 64, 4, False, False, "f16"),
        # a long document in one piece
        _window("window document", 1, 16, 4, 16384, 16384, 128, 4096, 4, False, False, "bf16"),
        # the second piece of a padded batch of prompts whose first piece stands before it; odd sizes
        _window("window padded piece", 3, 6, 2, 777, 1500, 80, 300, 1, True, False, "f16"),
        # a training step of a layer with grouped heads
        _window("window step", 4, 32, 8, 4096, 4096, 128, 1024, 4, False, True, "bf16"),
        # the same in float32 on a small padded batch of odd length
        _window("window step padded", 2, 3, 3, 1025, 1025, 64, 200, 0, True, True, "f32"),
        # one new token of one request
        _decode("decode one request", 1, 32, 8, 128, 16, 1024, 0, 0, False, "bf16"),
        # one new token each of a full batch, with the weights summed for a later eviction
        _decode("decode batch, weights", 64, 32, 8, 128, 16, 4096, 0, 0, True, "bf16"),
        # a few requests with very long contexts
        _decode("decode long contexts", 8, 32, 8, 128, 64, 131072, 0, 0, False, "f16"),
        # the new token of every sequence in a batch
        _append("append tokens", 64, 8, 128, 16, 1, 4096, "bf16"),
        # the prompts of a batch
        _append("append prompts", 8, 8, 128, 16, 4096, 8192, "bf16"),
        # one request over its budget
        _evict("evict one request", 1, 8, 64, 16, 1024, 256, 4, 32, "f16"),
        # a batch of long requests over their budgets
        _evict("evict batch", 16, 8, 128, 16, 8192, 2048, 4, 512, "bf16"),
    ]


def _window(name, batch, heads, kv_heads, q_len, kv_len, dim, window, sinks, padded, train, dtype):
    return dict(name=name, op="window", batch=batch, heads=heads, kv_heads=kv_heads, q_len=q_len, kv_len=kv_len,
                dim=dim, window=window, sinks=sinks, padded=padded, train=train, dtype=dtype)


def _decode(name, batch, heads, kv_heads, dim, page, max_len, window, sinks, weights, dtype):
    return dict(name=name, op="decode", batch=batch, heads=heads, kv_heads=kv_heads, dim=dim, page=page,
                max_len=max_len, window=window, sinks=sinks, weights=weights, dtype=dtype)


def _append(name, batch, kv_heads, dim, page, tokens, max_len, dtype):
    return dict(name=name, op="append", batch=batch, kv_heads=kv_heads, dim=dim, page=page, tokens=tokens,
                max_len=max_len, dtype=dtype)


def _evict(name, batch, kv_heads, dim, page, max_len, budget, sinks, recent, dtype):
    return dict(name=name, op="evict", batch=batch, kv_heads=kv_heads, dim=dim, page=page, max_len=max_len,
                budget=budget, sinks=sinks, recent=recent, dtype=dtype)


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["window", "window", "decode", "decode", "append", "evict"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f16", "f32"])
    dim = rng.choice([64, 128, 128, rng.randrange(16, 129, 8)])
    kv_heads, group = rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 2, 3, 4, 8])
    if op == "window":
        train = rng.random() < 0.5
        kv_len = _log(rng, 64, 6000 if train else 12000)
        q_len = kv_len if train or rng.random() < 0.5 else rng.randrange(1, kv_len + 1)
        heads = min(kv_heads * group, 16) // kv_heads * kv_heads
        batch = rng.randrange(1, 5) if kv_len < 4000 else 1
        case = _window("", batch, heads, kv_heads, q_len, kv_len, dim, _log(rng, 16, kv_len + 1), rng.choice([0, 1, 4, 16]),
                       rng.random() < 0.4, train, "f32" if dtype == "f32" and kv_len < 2000 else "bf16" if dtype == "f32" else dtype)
    elif op == "decode":
        batch = _log(rng, 1, 64)
        most = 8 * 131072 * 8 // (batch * kv_heads) // (2 if dtype == "f32" else 1)
        max_len = _log(rng, 16, min(most, 100000))
        windowed = rng.random() < 0.4
        case = _decode("", batch, kv_heads * group, kv_heads, dim, rng.choice([16, 32, 64, 24]), max_len,
                       _log(rng, 16, max_len + 1) if windowed else 0, rng.choice([0, 4]) if windowed else 0,
                       rng.random() < 0.4, dtype)
    elif op == "append":
        tokens = rng.choice([1, _log(rng, 1, 2500)])
        case = _append("", _log(rng, 1, 48 if tokens == 1 else 8), kv_heads, dim, rng.choice([16, 32, 64, 24]), tokens,
                       tokens + _log(rng, 1, 3000), dtype)
    else:
        max_len = _log(rng, 64, 8000)
        budget = rng.randrange(24, max_len + 1)
        case = _evict("", _log(rng, 1, 16), kv_heads, dim, rng.choice([16, 32, 64, 24]), max_len, budget,
                      rng.choice([0, 4]), rng.randrange(0, budget - 8), dtype)
    del case["name"]
    return case


def _lengths(case):
    """Every sequence's length: the first is as long as the case allows, the others are spread from an eighth of that on."""
    b = np.arange(case["batch"])
    if case["op"] == "window":
        most = case["kv_len"]
        if not case["padded"]:
            return np.full(b.shape, most)
    else:
        most = case["max_len"]
    if case["op"] == "append":
        most -= case["tokens"]
    share = 1 - (b * 0.6180339887498949 % 1) * 0.875
    return np.maximum(np.minimum(1, most), np.rint(most * share)).astype(np.int64)


# ------------------------------------------------------------------ inputs

def _randn(gen, dtype, *shape):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)


def _pages(case):
    return -(-case["max_len"] // case["page"])


def _table(case, gen, lens, first, per, most):
    """Every sequence's pages, in no order, out of the `most` pages from `first` on; -1 behind its last."""
    ids = first + torch.randperm(most, generator=gen, device="cuda")[: case["batch"] * per]
    table = ids.reshape(case["batch"], per).to(torch.int32)
    used = (lens + case["page"] - 1) // case["page"]
    return torch.where(torch.arange(per, device="cuda") < used[:, None], table, -1)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    lens = torch.from_numpy(_lengths(case)).cuda()
    state = {"case": case, "lens": lens.to(torch.int32)}
    B, d, G = case["batch"], case["dim"], case["kv_heads"]
    if case["op"] == "window":
        state["q"] = _randn(gen, dtype, B, case["heads"], case["q_len"], d).requires_grad_(case["train"])
        state["k"] = _randn(gen, dtype, B, G, case["kv_len"], d).requires_grad_(case["train"])
        state["v"] = _randn(gen, dtype, B, G, case["kv_len"], d).requires_grad_(case["train"])
        if case["train"]:
            state["dout"] = _randn(gen, dtype, B, case["heads"], case["q_len"], d)
        return state
    per = _pages(case)
    full = lens + case.get("tokens", 0)
    target = -(-case.get("budget", 0) // case["page"])
    state["table"] = _table(case, gen, full, 0, per, B * per)
    state["k_cache"] = _randn(gen, dtype, B * (per + target), G, case["page"], d)
    state["v_cache"] = _randn(gen, dtype, B * (per + target), G, case["page"], d)
    if case["op"] == "append":
        state["k"] = _randn(gen, dtype, B, G, case["tokens"], d)
        state["v"] = _randn(gen, dtype, B, G, case["tokens"], d)
    if case["op"] == "decode":
        state["q"] = _randn(gen, dtype, B, case["heads"], d)
    if case["op"] == "evict" or case.get("weights"):
        # a few keys gather most of the weight; keys that nothing looked at yet tie at zero
        sums = torch.randn((B, G, per * case["page"]), generator=gen, device="cuda").mul(2).exp()
        sums = torch.where(torch.rand(sums.shape, generator=gen, device="cuda") < 0.1, 0.0, sums)
        state["sums"] = torch.where(torch.arange(per * case["page"], device="cuda") < lens[:, None, None], sums, 0.0)
    if case["op"] == "evict":
        kept = lens.clamp(max=case["budget"])
        state["new_table"] = _table(case, gen, kept, B * per, target, B * target)
    return state


# ------------------------------------------------------------------ one pass

def run(state):
    case = state["case"]
    return globals()[("_own_" if own else "_plain_") + case["op"]](state, case)


def _own_window(s, c):
    mfa = _package()
    lens = s["lens"] if c["padded"] else None
    scale = c["dim"] ** -0.5
    if not c["train"]:
        return mfa.window_attn_fwd(s["q"], s["k"], s["v"], c["window"], sinks=c["sinks"], scale=scale, seq_lens=lens)
    out = mfa.window_attn_func(s["q"], s["k"], s["v"], c["window"], sinks=c["sinks"], scale=scale, seq_lens=lens)
    return (out.detach(), *torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["dout"]))


def _own_append(s, c):
    _package().paged_kv_append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["table"], s["lens"])
    return s["k_cache"], s["v_cache"]


def _own_decode(s, c):
    out = _package().paged_attn_decode(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"], scale=c["dim"] ** -0.5,
                                       window=c["window"], sinks=c["sinks"], weight_sum=s.get("sums"))
    return (out, s["sums"]) if c["weights"] else out


def _own_evict(s, c):
    sums, lens, kept = _package().paged_kv_evict(s["k_cache"], s["v_cache"], s["sums"], s["table"], s["lens"], s["new_table"],
                                                 c["budget"], sinks=c["sinks"], recent=c["recent"])
    return s["k_cache"], s["v_cache"], sums, lens, kept


def _weights(scores, visible):
    """Softmax over the last axis of what is visible; rows that see nothing are zero."""
    scores = scores.masked_fill(~visible, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == float("-inf"), 0.0, top))
    total = p.sum(-1, keepdim=True)
    return p / torch.where(total == 0, 1.0, total)


def _plain_window(s, c):
    B, H, G, d = c["batch"], c["heads"], c["kv_heads"], c["dim"]
    Nq, Nk, scale = c["q_len"], c["kv_len"], d ** -0.5
    q, k, v = (s[n].detach().float() for n in "qkv")
    key = torch.arange(Nk, device="cuda")
    pos = torch.arange(Nk - Nq, Nk, device="cuda")[:, None]
    visible = (key <= pos) & ((pos - key < c["window"]) | (key < c["sinks"]))
    lens = s["lens"].view(B, 1, 1)
    visible = (visible & (key < lens) & (pos < lens)).view(B, 1, 1, Nq, Nk)
    q = q.reshape(B, G, H // G, Nq, d)
    kt, vt = k.transpose(-1, -2).contiguous().unsqueeze(2), v.transpose(-1, -2).contiguous().unsqueeze(2)
    k, v = k.unsqueeze(2), v.unsqueeze(2)
    p = _weights(torch.matmul(q, kt).mul_(scale), visible)
    out = torch.matmul(p, v)
    rounded = out.reshape(B, H, Nq, d).to(s["q"].dtype)
    if not c["train"]:
        return rounded
    dout = s["dout"].float().reshape(B, G, H // G, Nq, d)
    ds = torch.matmul(dout, vt)
    ds = ds.sub_((dout * out).sum(-1, keepdim=True)).mul_(p)
    dv = torch.matmul(p.transpose(-1, -2).contiguous(), dout).sum(2)
    dq = torch.matmul(ds, k).mul_(scale).reshape(B, H, Nq, d)
    dk = torch.matmul(ds.transpose(-1, -2).contiguous(), q).mul_(scale).sum(2)
    return rounded, dq.to(s["q"].dtype), dk.to(s["k"].dtype), dv.to(s["v"].dtype)


def _plain_append(s, c):
    at = s["lens"].long()[:, None] + torch.arange(c["tokens"], device="cuda")
    pages = torch.gather(s["table"].long(), 1, at // c["page"])
    s["k_cache"][pages, :, at % c["page"]] = s["k"].transpose(1, 2)
    s["v_cache"][pages, :, at % c["page"]] = s["v"].transpose(1, 2)
    return s["k_cache"], s["v_cache"]


def _gathered(cache, table):
    """[pages, heads, page, d] and [batch, pages a sequence] to [batch, heads, keys, d]."""
    x = cache[table.clamp(min=0).long()].transpose(1, 2)
    return x.reshape(x.shape[0], x.shape[1], -1, x.shape[-1])


def _plain_decode(s, c):
    B, H, G, d = c["batch"], c["heads"], c["kv_heads"], c["dim"]
    k = _gathered(s["k_cache"], s["table"]).float()
    v = _gathered(s["v_cache"], s["table"]).float()
    key, lens = torch.arange(k.shape[2], device="cuda"), s["lens"].view(B, 1, 1, 1)
    visible = key < lens
    if c["window"]:
        visible = visible & ((lens - 1 - key < c["window"]) | (key < c["sinks"]))
    q = s["q"].float().reshape(B, G, H // G, d)
    p = _weights((torch.matmul(q, k.transpose(-1, -2).contiguous())).mul_(d ** -0.5), visible)
    out = torch.matmul(p, v).reshape(B, H, d).to(s["q"].dtype)
    if not c["weights"]:
        return out
    s["sums"].add_(p.sum(2))
    return out, s["sums"]


def _plain_evict(s, c):
    B, G, page, budget = c["batch"], c["kv_heads"], c["page"], c["budget"]
    sums, lens = s["sums"], s["lens"].long()
    key = torch.arange(sums.shape[-1], device="cuda")
    behind, n = key >= lens.view(B, 1, 1), lens.view(B, 1, 1)
    always = (key < c["sinks"]) | (key >= n - c["recent"])
    rank = torch.where(behind, -2.0, torch.where(always, float("inf"), sums))
    order = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :budget]
    kept_lens = lens.clamp(max=budget)
    slot = torch.arange(budget, device="cuda")
    live = slot < kept_lens.view(B, 1, 1)
    # those that are chosen, in ascending order; behind them nothing
    kept = torch.where(live[..., : order.shape[-1]], order, sums.shape[-1]).sort(-1).values
    kept = torch.nn.functional.pad(kept, (0, budget - kept.shape[-1]), value=sums.shape[-1])
    live = live.expand(B, G, budget)
    source = torch.where(live, kept, 0)
    new_sums = torch.zeros((B, G, s["new_table"].shape[1] * page), device="cuda")
    new_sums[..., :budget] = torch.where(live, torch.gather(sums, 2, source), 0.0)
    b, g, i = torch.nonzero(live, as_tuple=True)
    j = source[b, g, i]
    old, new = s["table"].long()[b, j // page], s["new_table"].long()[b, i // page]
    s["k_cache"][new, g, i % page] = s["k_cache"][old, g, j % page]
    s["v_cache"][new, g, i % page] = s["v_cache"][old, g, j % page]
    return s["k_cache"], s["v_cache"], new_sums, kept_lens.int(), torch.where(live, kept, -1).int()


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    lens = _lengths(case).astype(np.float64)
    d, G, B = case["dim"], case["kv_heads"], case["batch"]
    if case["op"] == "window":
        pos = np.arange(case["kv_len"] - case["q_len"], case["kv_len"], dtype=np.float64)
        sees = np.minimum(pos + 1, case["window"]) + np.clip(pos + 1 - case["window"], 0, case["sinks"])
        pairs = sum(float(sees[pos < n].sum()) for n in lens) * case["heads"]
        q, kv = B * case["heads"] * case["q_len"] * d * size, B * G * case["kv_len"] * d * size
        if case["train"]:  # reads q, k, v, dout, writes out and the gradients
            return {"bytes": 4 * q + 4 * kv, "flops": 14 * d * pairs}
        return {"bytes": 2 * q + 2 * kv, "flops": 4 * d * pairs}
    if case["op"] == "decode":
        sees = lens
        if case["window"]:
            sees = np.minimum(lens, case["window"]) + np.clip(lens - case["window"], 0, case["sinks"])
        keys = float(sees.sum()) * G
        table = float(np.ceil(sees / case["page"]).sum()) * 4
        return {"bytes": 2 * keys * d * size + (8 * keys if case["weights"] else 0) + 2 * B * case["heads"] * d * size + table,
                "flops": 4 * d * keys * (case["heads"] // G)}
    if case["op"] == "append":
        return {"bytes": 4 * B * G * case["tokens"] * d * size, "flops": 0}
    kept = float(np.minimum(lens, case["budget"]).sum()) * G
    return {"bytes": 4 * kept * d * size + 4 * float(lens.sum()) * G + 4 * kept + 4 * B * G * case["budget"], "flops": 0}


# ------------------------------------------------------------------ the definition in 64 bits

def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "window":
        return _exact_window(case, state)
    if case["op"] == "decode":
        return _exact_decode(case, state)
    if case["op"] == "append":
        return _exact_append(case, state)
    return _exact_evict(case, state)


def _exact_window(c, s):
    B, H, G, Nq, Nk = c["batch"], c["heads"], c["kv_heads"], c["q_len"], c["kv_len"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    grads = [torch.zeros(s[n].shape, dtype=torch.float64, device="cuda") for n in "qkv"]
    step = 2048
    for b, n in enumerate(_lengths(c).tolist()):
        for h in range(H):
            g = h // (H // G)
            for i0 in range(0, max(0, min(Nq, n - (Nk - Nq))), step):
                rows = slice(i0, min(i0 + step, Nq, n - (Nk - Nq)))
                p0, p1 = rows.start + Nk - Nq, rows.stop + Nk - Nq
                # keys that some row of the piece sees
                low = max(0, p0 - c["window"] + 1)
                keys = torch.cat([torch.arange(0, min(c["sinks"], low)), torch.arange(low, p1)]).cuda()
                x = [s["q"][b, h, rows].detach().double(), s["k"][b, g].detach().double()[keys], s["v"][b, g].detach().double()[keys]]
                x = [t.requires_grad_(c["train"]) for t in x]
                gap = torch.arange(p0, p1, device="cuda")[:, None] - keys[None, :]
                hidden = (gap < 0) | ((gap >= c["window"]) & (keys >= c["sinks"])[None, :])
                logits = torch.matmul(x[0], x[1].t()) / math.sqrt(c["dim"])
                o = torch.matmul(torch.softmax(logits.masked_fill(hidden, float("-inf")), -1), x[2])
                out[b, h, rows] = o.detach()
                if c["train"]:
                    dq, dk, dv = torch.autograd.grad(o, x, s["dout"][b, h, rows].double())
                    grads[0][b, h, rows] = dq
                    grads[1][b, g].index_add_(0, keys, dk)
                    grads[2][b, g].index_add_(0, keys, dv)
    return (out, *grads) if c["train"] else out


def _keys_of(cache, table_row, n, page):
    """The first n keys of one sequence, [heads, n, d], in 64 bits."""
    x = cache[table_row[: -(-n // page)].long()].double()
    return x.permute(1, 0, 2, 3).reshape(cache.shape[1], -1, cache.shape[-1])[:, :n]


def _exact_decode(c, s):
    H, G, page = c["heads"], c["kv_heads"], c["page"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    sums = s["sums"].double() if c["weights"] else None
    for b, n in enumerate(_lengths(c).tolist()):
        k, v = (_keys_of(s[x], s["table"][b], n, page) for x in ("k_cache", "v_cache"))
        low = max(0, n - c["window"]) if c["window"] else 0
        seen = torch.cat([torch.arange(0, min(c["sinks"], low)), torch.arange(low, n)]).cuda()
        for g in range(G):
            q = s["q"][b, g * (H // G):(g + 1) * (H // G)].double()
            w = torch.softmax(torch.matmul(q, k[g, seen].t()) / math.sqrt(c["dim"]), -1)
            out[b, g * (H // G):(g + 1) * (H // G)] = torch.matmul(w, v[g, seen])
            if c["weights"]:
                sums[b, g, seen] += w.sum(0)
    return (out, sums) if c["weights"] else out


def _exact_append(c, s):
    for b, n in enumerate(_lengths(c).tolist()):
        done = 0
        while done < c["tokens"]:
            page, slot = divmod(n + done, c["page"])
            many = min(c["page"] - slot, c["tokens"] - done)
            at = int(s["table"][b, page])
            s["k_cache"][at, :, slot:slot + many] = s["k"][b, :, done:done + many]
            s["v_cache"][at, :, slot:slot + many] = s["v"][b, :, done:done + many]
            done += many
    return s["k_cache"].double(), s["v_cache"].double()


def _exact_evict(c, s):
    B, G, page, budget = c["batch"], c["kv_heads"], c["page"], c["budget"]
    sums = s["sums"].cpu().numpy()
    table, new_table = s["table"].cpu().numpy(), s["new_table"].cpu().numpy()
    new_sums = np.zeros((B, G, new_table.shape[1] * page))
    kept = np.full((B, G, budget), -1, np.int32)
    lens = _lengths(c)
    old_k, old_v = s["k_cache"].clone(), s["v_cache"].clone()
    for b, n in enumerate(lens.tolist()):
        for g in range(G):
            if n <= budget:
                chosen = np.arange(n)
            else:
                first, last = np.arange(min(c["sinks"], n)), np.arange(max(c["sinks"], n - c["recent"]), n)
                middle = np.arange(len(first), n - len(last))
                best = middle[np.lexsort((middle, -sums[b, g, middle].astype(np.float64)))]
                chosen = np.sort(np.concatenate([first, best[: budget - len(first) - len(last)], last]))
            m = len(chosen)
            kept[b, g, :m] = chosen
            new_sums[b, g, :m] = sums[b, g, chosen]
            at = np.arange(m)
            old, new = (torch.from_numpy(x.astype(np.int64)).cuda() for x in (table[b, chosen // page], new_table[b, at // page]))
            i, j = (torch.from_numpy(x % page).cuda() for x in (at, chosen))
            s["k_cache"][new, g, i] = old_k[old, g, j]
            s["v_cache"][new, g, i] = old_v[old, g, j]
    return (s["k_cache"].double(), s["v_cache"].double(), torch.from_numpy(new_sums).cuda(),
            torch.from_numpy(np.minimum(lens, budget).astype(np.int32)).cuda(), torch.from_numpy(kept).cuda())
