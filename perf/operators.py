"""Timed workloads of the 8-bit key/value cache: a decode step (append one token to each sequence and
attend), a prompt or a piece of one (append, attend), filling and reading back, and eviction by
accumulated attention weight; at the Gemma-3-270M attention shape (4 heads, 1 key/value head of 256)
and at generic grouped shapes.

The cache holds, for each sequence, key/value head and block of 32 positions, int8 codes with one
scale for the keys and one for the values; the positions of a block that is not full are held in
32 bits. Keys, values and queries are N(0, 1) with a few strong channels, as they leave a norm with
weights; attention weights accumulated so far are exponential, with many near zero.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

BLOCK = 32


def listed():
    return [
        # the first tokens of a chat: one sequence, one new token; latency is all there is
        {"name": "step_33", "kind": "step", "seqs": 1, "heads": 4, "kv": 1, "hd": 256, "lo": 33, "hi": 33, "window": 0,
         "cap": 0.0, "prefix": 0, "ring": False, "scored": False},
        # a full batch of the 270M shape, one global block: histories from one token to a document
        {"name": "step_64", "kind": "step", "seqs": 64, "heads": 4, "kv": 1, "hd": 256, "lo": 1, "hi": 8192, "window": 0,
         "cap": 0.0, "prefix": 0, "ring": False, "scored": False},
        # the same batch in a local block: a ring of 512 positions
        {"name": "step_window", "kind": "step", "seqs": 64, "heads": 4, "kv": 1, "hd": 256, "lo": 290, "hi": 4001, "window": 512,
         "cap": 0.0, "prefix": 0, "ring": True, "scored": False},
        # two very long conversations over grouped heads, capped scores
        {"name": "step_long", "kind": "step", "seqs": 2, "heads": 32, "kv": 8, "hd": 128, "lo": 100001, "hi": 131072,
         "window": 0, "cap": 50.0, "prefix": 0, "ring": False, "scored": False},
        # a service that evicts: every step accumulates the weight of each position
        {"name": "step_scored", "kind": "step", "seqs": 16, "heads": 8, "kv": 2, "hd": 96, "lo": 500, "hi": 16384, "window": 0,
         "cap": 0.0, "prefix": 0, "ring": False, "scored": True},
        # a prompt of the 270M shape in one call
        {"name": "prompt_4096", "kind": "prompt", "seqs": 1, "heads": 4, "kv": 1, "hd": 256, "hist": 0, "n": 4096, "window": 0,
         "cap": 0.0, "prefix": 0, "scored": False},
        # the next piece of two long documents: a prefix that all see, a window, capped scores, an odd length
        {"name": "prompt_piece", "kind": "prompt", "seqs": 2, "heads": 16, "kv": 4, "hd": 128, "hist": 8192, "n": 1001,
         "window": 4096, "cap": 30.0, "prefix": 700, "scored": False},
        # prompts whose weights are wanted for eviction
        {"name": "prompt_scored", "kind": "prompt", "seqs": 3, "heads": 8, "kv": 2, "hd": 64, "hist": 0, "n": 2048, "window": 0,
         "cap": 0.0, "prefix": 0, "scored": True},
        # the keys and values of short questions, of ragged lengths, into the cache and back
        {"name": "fill_short", "kind": "fill", "seqs": 48, "kv": 1, "hd": 256, "lo": 3, "hi": 70},
        # a document's keys and values into the cache and back
        {"name": "fill_8192", "kind": "fill", "seqs": 2, "kv": 8, "hd": 128, "lo": 8000, "hi": 8192},
        # a full batch at its limit: every sequence back to a quarter of it
        {"name": "evict_64", "kind": "evict", "seqs": 64, "kv": 1, "hd": 256, "lo": 4097, "hi": 8192, "keep": 2048, "recent": 256},
        # two long conversations cut to an odd number of positions
        {"name": "evict_long", "kind": "evict", "seqs": 2, "kv": 8, "hd": 128, "lo": 60001, "hi": 65536, "keep": 8190,
         "recent": 1000},
    ]


def _log(rng, lo, hi):
    """An integer between lo and hi, even over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["step", "step", "step", "prompt", "prompt", "fill", "evict"])
    hd = rng.choice([64, 80, 96, 128, 256, 4 * rng.randint(4, 64)])
    kv = rng.choice([1, 1, 2, 4, 8])
    heads = kv * rng.choice([1, 2, 3, 4, 8])
    if kind == "step":
        seqs = _log(rng, 1, 64)
        most = max(64, min(131072, 230_000_000 // (seqs * kv * hd)))   # positions: no more bytes than the longest listed case
        hi = _log(rng, 2, most)
        lo = rng.randint(1, hi)
        ring = rng.random() < 0.2
        window = _log(rng, 16, 2048) if ring or rng.random() < 0.2 else 0
        return {"kind": kind, "seqs": seqs, "heads": heads, "kv": kv, "hd": hd, "lo": lo, "hi": hi, "window": window,
                "cap": rng.choice([0.0, 0.0, 30.0, 50.0]), "prefix": 0 if ring else rng.choice([0, 0, _log(rng, 1, 64)]), "ring": ring,
                "scored": not ring and rng.random() < 0.3}
    if kind == "prompt":
        seqs = rng.choice([1, 1, 2, 4])
        hist = rng.choice([0, 0, BLOCK * _log(rng, 1, 128)])
        most = 4 * 256 * 4096 * 4096 // 2 / (heads * hd * seqs)   # pairs of a query and a key
        n = int(math.sqrt(hist * hist + 2 * most) - hist)
        n = _log(rng, 2, max(2, min(4096, n)))
        return {"kind": kind, "seqs": seqs, "heads": heads, "kv": kv, "hd": hd, "hist": hist, "n": n,
                "window": rng.choice([0, 0, _log(rng, 16, 4096)]), "cap": rng.choice([0.0, 0.0, 30.0]),
                "prefix": rng.choice([0, 0, _log(rng, 1, max(1, hist + n))]), "scored": rng.random() < 0.3}
    if kind == "fill":
        seqs = _log(rng, 1, 64)
        hi = _log(rng, 2, max(64, min(8192, 16_000_000 // (seqs * kv * hd))))
        return {"kind": kind, "seqs": seqs, "kv": kv, "hd": hd, "lo": rng.randint(1, hi), "hi": hi}
    seqs = _log(rng, 1, 64)
    hi = _log(rng, 64, max(128, min(65536, 33_000_000 // (seqs * kv * hd))))
    lo = rng.randint(hi // 2, hi)
    keep = rng.randint(1, lo)
    return {"kind": kind, "seqs": seqs, "kv": kv, "hd": hd, "lo": lo, "hi": hi, "keep": keep, "recent": rng.randint(0, keep)}


# ---- inputs ---------------------------------------------------------------------------------

def _lengths(case):
    """The sequences' lengths: spread over [lo, hi], the last one hi."""
    n, lo, hi = case["seqs"], case["lo"], case["hi"]
    return [hi if i == n - 1 else lo + int((hi - lo + 1) * ((i * 0.6180339887498949) % 1.0)) for i in range(n)]


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _values(g, rows, kv, hd):
    """[rows, kv, hd] N(0, 1), every 29th channel four times as strong."""
    x = torch.randn(rows, kv, hd, generator=g, device="cuda")
    x[:, :, 5::29] *= 4.0
    return x


def _inputs(case, seed):
    """Keys and values of every position, sequence after sequence, the queries, and the weights accumulated so far."""
    g = _generator(seed)
    kind = case["kind"]
    lens = [case["hist"] + case["n"]] * case["seqs"] if kind == "prompt" else _lengths(case)
    x = {"lens": lens, "k": _values(g, sum(lens), case["kv"], case["hd"]), "v": _values(g, sum(lens), case["kv"], case["hd"])}
    if kind in ("step", "prompt"):
        n = case.get("n", 1)
        x["q"] = torch.randn(case["seqs"] * n, case["heads"], case["hd"], generator=g, device="cuda")
    if kind == "evict" or case.get("scored"):
        u = torch.rand(case["seqs"], case["kv"], max(lens), generator=g, device="cuda")
        x["weights"] = u.pow(8).mul_(3.0)
        live = torch.arange(max(lens), device="cuda")[None, None, :] < torch.tensor(lens, device="cuda")[:, None, None]
        x["weights"] *= live
    return x


def _scale(case):
    return float(np.float32(1.0 / math.sqrt(case["hd"])))


def _padded(x, lens, fill=None):
    """[sum(lens), ...] rows as [sequences, max(lens), ...]; zeros past each length."""
    at = torch.arange(max(lens), device=x.device)
    n = torch.tensor(lens, device=x.device)
    first = torch.cumsum(n, 0) - n
    live = at[None, :] < n[:, None]
    rows = torch.where(live, first[:, None] + at[None, :], torch.zeros_like(at)[None, :])
    y = x[rows.reshape(-1)].view(len(lens), max(lens), *x.shape[1:])
    return y * live.view(*live.shape, *([1] * (x.dim() - 1)))


def _rows(seq_pos_n_prefix):
    return np.asarray(seq_pos_n_prefix, dtype=np.uint32).reshape(-1, 4)


def prepare(case, seed):
    x = _inputs(case, seed)
    kind, lens, S = case["kind"], x["lens"], case["seqs"]
    s = {"case": case, "lens": lens}
    n_new = [1 if kind == "step" else case["n"] if kind == "prompt" else n if kind == "fill" else 0 for n in lens]
    hist = [n - m for n, m in zip(lens, n_new)]
    starts = np.cumsum([0] + lens)
    new = torch.cat([torch.arange(int(starts[i]) + hist[i], int(starts[i]) + lens[i], device="cuda") for i in range(S)])
    for name in ("k", "v"):   # the call's own rows, packed
        if kind != "evict":
            s[name] = x[name][new].contiguous()
    for name in ("q", "weights"):
        if name in x:
            s[name] = x[name]
    if own:
        _prepare_own(case, s, x, hist, n_new, starts)
    else:
        _prepare_plain(case, s, x, hist)
    return s


# ---- the plain form ---------------------------------------------------------------------------

def _codes(x):
    """[..., 32, hd] values as int8 codes and one scale: the quotient in 64 bits, rounded once."""
    amax = x.abs().amax(dim=(-2, -1))
    scale = amax / torch.full_like(amax, 127.0)   # a quotient: by a plain number torch multiplies by its reciprocal
    q = torch.round(x.double() / scale.double().clamp_min(1e-300)[..., None, None])
    return q.clamp_(-127, 127).to(torch.int8), scale


def _blocks(x, lens):
    """Rows [sequences, L, kv, hd] as [sequences, kv, L / 32, 32, hd], the last block filled with zeros."""
    S, L, kv, hd = x.shape
    nb = -(-L // BLOCK)
    y = torch.zeros(S, nb * BLOCK, kv, hd, dtype=x.dtype, device=x.device)
    y[:, :L] = x
    return y.view(S, nb, BLOCK, kv, hd).permute(0, 3, 1, 2, 4).contiguous()


def _plain_cache(x, lens):
    """Codes and scales of the full blocks and the rows of the open one, of padded rows [S, L, kv, hd]."""
    b = _blocks(x, lens)
    codes, scale = _codes(b)
    n = torch.tensor(lens, device="cuda")
    last = torch.div(n, BLOCK, rounding_mode="floor")   # the open block, if the length leaves one
    pick = last.clamp_max(b.shape[2] - 1).view(-1, 1, 1, 1, 1).expand(-1, b.shape[1], 1, BLOCK, b.shape[4])
    return {"codes": codes, "scale": scale, "tail": b.gather(2, pick).squeeze(2)}


def _prepare_plain(case, s, x, hist):
    kind = case["kind"]
    for name in ("k", "v"):
        if kind == "fill":
            continue
        full = _padded(x[name], s["lens"])
        if kind != "evict":   # the call's own rows are not in the cache yet
            at = torch.arange(full.shape[1], device="cuda")
            full = full * (at[None, :] < torch.tensor(hist, device="cuda")[:, None])[:, :, None, None]
            s["cache_" + name] = _plain_cache(full, hist)
        else:
            s["cache_" + name] = _plain_cache(full, s["lens"])
    n = torch.tensor(s["lens"], device="cuda")
    s["n"] = n
    if kind == "step":
        s["block"] = torch.div(n - 1, BLOCK, rounding_mode="floor")
        s["slot"] = (n - 1) % BLOCK
        s["seq"] = torch.arange(case["seqs"], device="cuda")


def _plain_values(c, n):
    """The values that a cache stands for, [S, kv, L, hd]: codes times scale, and the open block's own."""
    x = c["codes"].float() * c["scale"][..., None, None]
    S, kv, nb, _, hd = x.shape
    block = torch.arange(nb, device="cuda")
    is_open = block[None, :] == torch.div(n, BLOCK, rounding_mode="floor")[:, None]
    x = torch.where(is_open[:, None, :, None, None], c["tail"][:, :, None], x)
    return x.reshape(S, kv, nb * BLOCK, hd)


def _plain_append_one(c, row, s):
    """One new row [S, kv, hd] of every sequence; a block that it fills gets its codes."""
    starts_block = (s["slot"] == 0)[:, None, None, None]
    tail = torch.where(starts_block, torch.zeros_like(c["tail"]), c["tail"])
    tail[s["seq"], :, s["slot"]] = row
    codes, scale = _codes(tail)
    full = (s["slot"] == BLOCK - 1)
    at = (s["seq"], slice(None), s["block"])
    all_codes, all_scale = c["codes"].clone(), c["scale"].clone()
    all_codes[at] = torch.where(full[:, None, None, None], codes, all_codes[at])
    all_scale[at] = torch.where(full[:, None], scale, all_scale[at])
    return {"codes": all_codes, "scale": all_scale, "tail": tail}


def _plain_append_many(c, rows, hist, n):
    """n new rows [S, n, kv, hd] of every sequence, from a position that starts a block."""
    b = _blocks(rows, None)
    codes, scale = _codes(b)
    first = hist // BLOCK
    all_codes, all_scale = c["codes"].clone(), c["scale"].clone()
    all_codes[:, :, first:first + b.shape[2]] = codes
    all_scale[:, :, first:first + b.shape[2]] = scale
    return {"codes": all_codes, "scale": all_scale, "tail": b[:, :, min(n // BLOCK, b.shape[2] - 1)]}


def _visible(case, n, nq, L):
    """[S, nq, L]: which positions the queries at n - nq .. n - 1 see."""
    i = (n[:, None] - nq + torch.arange(nq, device="cuda")[None, :])[:, :, None]
    j = torch.arange(L, device="cuda")[None, None, :]
    see = j <= i
    if case["window"]:
        see &= i - j < case["window"]
    see |= j < case["prefix"]
    return see & (j < n[:, None, None])


def _plain_attend(case, s, k, v):
    S, kv, L, hd = k.shape
    nq, H = case.get("n", 1), case["heads"]
    G = H // kv
    q = s["q"].view(S, nq, kv, G, hd).permute(0, 2, 3, 1, 4).reshape(S, kv, G * nq, hd)
    sc = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(_scale(case))
    if case["cap"]:
        sc = case["cap"] * torch.tanh(sc / case["cap"])
    see = _visible(case, s["n"], nq, L)[:, None, None]
    sc = sc.view(S, kv, G, nq, L).masked_fill_(~see, float("-inf"))
    p = torch.exp(sc - sc.amax(dim=-1, keepdim=True))
    p = p / p.sum(dim=-1, keepdim=True)
    o = torch.matmul(p.view(S, kv, G * nq, L), v).view(S, kv, G, nq, hd)
    out = {"out": o.permute(0, 3, 1, 2, 4).reshape(S * nq, H, hd)}
    if case["scored"]:
        w = s["weights"]
        Lw = w.shape[2]
        old = torch.arange(Lw, device="cuda")[None, :] < (s["n"] - nq)[:, None]
        out["weights"] = w * old[:, None] + p.sum(dim=(2, 3))[:, :, :Lw]
    return out


def _plain_evict(case, s):
    w, n, keep = s["weights"], s["n"], case["keep"]
    j = torch.arange(w.shape[2], device="cuda")[None, :]
    key = torch.where((j >= (n - case["recent"])[:, None])[:, None], torch.full_like(w, float("inf")), w)
    key = torch.where((j >= n[:, None])[:, None], torch.full_like(w, float("-inf")), key)
    at = torch.sort(key, dim=2, descending=True, stable=True)[1][:, :, :keep].sort(dim=2)[0]
    out = {"kept": at.to(torch.int32), "weights": w.gather(2, at)}
    for name in ("k", "v"):
        x = _plain_values(s["cache_" + name], n)
        x = x.gather(2, at[..., None].expand(-1, -1, -1, x.shape[3])).transpose(1, 2)
        lens = [keep] * case["seqs"]
        c = _plain_cache(x, lens)
        y = _plain_values(c, torch.tensor(lens, device="cuda"))
        out[name] = y[:, :, :keep].transpose(1, 2).contiguous()
    return out


def _plain_fill(case, s):
    lens, n = s["lens"], s["n"]
    at = torch.arange(max(lens), device="cuda")
    live = at[None, :] < n[:, None]
    out = {}
    for name in ("k", "v"):
        y = _plain_values(_plain_cache(_padded(s[name], lens), lens), n)
        out[name] = y[:, :, :max(lens)].transpose(1, 2)[live]
    return out


def run(s):
    case = s["case"]
    if own:
        return _run_own(case, s)
    kind = case["kind"]
    if kind == "fill":
        return _plain_fill(case, s)
    if kind == "evict":
        return _plain_evict(case, s)
    kv = []
    for name in ("k", "v"):
        c = s["cache_" + name]
        if kind == "step":
            c = _plain_append_one(c, s[name], s)
        else:
            c = _plain_append_many(c, s[name].view(case["seqs"], case["n"], case["kv"], case["hd"]), case["hist"], case["n"])
        kv.append(_plain_values(c, s["n"]))
    return _plain_attend(case, s, *kv)


# ---- the framework's calls ----------------------------------------------------------------------

_ctx = None


def _context():
    """The program's device context: one, as long as it runs."""
    global _ctx
    if _ctx is None:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vortex-rt_amd"))
        import vrt
        _ctx = vrt.Context("0")
    return _ctx


def _prepare_own(case, s, x, hist, n_new, starts):
    ctx = _context()
    import vrt
    kind, lens, S, kv, hd = case["kind"], s["lens"], case["seqs"], case["kv"], case["hd"]
    ring = case.get("ring", False)
    max_ctx = -(-case["window"] // BLOCK) * BLOCK if ring else max(lens)
    c = s["cache"] = vrt.Kv8Cache(ctx, 2 * S if kind == "evict" else S, max_ctx, kv, hd)
    torch.cuda.synchronize()
    for i in range(S):   # the history, a ring's in pieces that it holds
        step = max_ctx if ring else max(1, hist[i])
        for p in range(0, hist[i], step):
            m = min(step, hist[i] - p)
            o = (int(starts[i]) + p) * kv * hd * 4
            c.append(_rows([(i, p, m, 0)]), x["k"].data_ptr() + o, x["v"].data_ptr() + o)
    if kind == "evict":
        for i in range(S):
            o = int(starts[i]) * kv * hd * 4
            c.append(_rows([(i, 0, lens[i], 0)]), x["k"].data_ptr() + o, x["v"].data_ptr() + o)
        s["moves"] = np.asarray([(i, S + i, lens[i], case["keep"], case["recent"]) for i in range(S)], dtype=np.uint32)
        s["rows"] = _rows([(S + i, 0, case["keep"], 0) for i in range(S)])
        s["kept"] = torch.zeros(S, kv, case["keep"], dtype=torch.int32, device="cuda")
        w = torch.zeros(2 * S, kv, max_ctx, device="cuda")   # the cache's regions: sources, then destinations
        w[:S] = s["weights"]
        s["weights"] = w
        n_out = S * case["keep"]
    else:
        s["rows"] = _rows([(i, hist[i], n_new[i], case.get("prefix", 0)) for i in range(S)])
        n_out = sum(n_new)
    if kind in ("evict", "fill"):
        s["k_out"], s["v_out"] = (torch.empty(n_out, kv, hd, device="cuda") for _ in range(2))
    else:
        s["out"] = torch.empty_like(s["q"])
        if case["scored"]:
            s["weights_out"] = torch.zeros_like(s["weights"])
    torch.cuda.synchronize()
    ctx.sync()


def _run_own(case, s):
    kind, c = case["kind"], s["cache"]
    if kind == "evict":
        S, keep = case["seqs"], case["keep"]
        c.evict(s["moves"], s["weights"].data_ptr(), s["kept"].data_ptr(), keep)
        c.read(s["rows"], s["k_out"].data_ptr(), s["v_out"].data_ptr())
        shape = (S, keep, case["kv"], case["hd"])
        return {"kept": s["kept"], "weights": s["weights"][S:, :, :keep], "k": s["k_out"].view(shape), "v": s["v_out"].view(shape)}
    c.append(s["rows"], s["k"].data_ptr(), s["v"].data_ptr())
    if kind == "fill":
        c.read(s["rows"], s["k_out"].data_ptr(), s["v_out"].data_ptr())
        return {"k": s["k_out"], "v": s["v_out"]}
    if not case["scored"]:
        c.attend(s["rows"], s["q"].data_ptr(), s["out"].data_ptr(), case["heads"], _scale(case), softcap=case["cap"],
                 window=case["window"])
        return {"out": s["out"]}
    c.attend(s["rows"], s["q"].data_ptr(), s["out"].data_ptr(), case["heads"], _scale(case), softcap=case["cap"],
             window=case["window"], weights_in=s["weights"].data_ptr(), weights_out=s["weights_out"].data_ptr())
    return {"out": s["out"], "weights": s["weights_out"]}


# ---- what a pass cannot do without --------------------------------------------------------------

def _seen(case, n, nq):
    """Pairs of a query and a position that it sees, and the positions that any query of a sequence sees."""
    pairs, first = 0, n
    window = case["window"] or n
    for i in range(n - nq, n):
        lo = max(0, i + 1 - window)
        pre = min(case["prefix"], n)
        pairs += i + 1 - lo + min(pre, lo) + max(0, pre - i - 1)
        first = min(first, lo)
    return pairs, n - first + min(min(case["prefix"], n), first)


def work(case):
    kind, kv, hd = case["kind"], case["kv"], case["hd"]
    row = 2 * kv * hd   # keys and values of a position: bytes of codes, a quarter of the bytes in 32 bits
    if kind == "fill":
        n = sum(_lengths(case))
        return {"bytes": n * row * 9 + n // BLOCK * 8 * kv, "flops": n * row * 3}
    if kind == "evict":
        n, m = sum(_lengths(case)), case["seqs"] * case["keep"]
        return {"bytes": n * kv * 4 + m * (row * 6 + 8 * kv), "flops": m * row * 3 + n * kv}
    nq, H = case.get("n", 1), case["heads"]
    lens = [case["hist"] + nq] * case["seqs"] if kind == "prompt" else _lengths(case)
    some = {n: _seen(case, n, nq) for n in set(lens)}
    pairs, seen = sum(some[n][0] for n in lens), sum(some[n][1] for n in lens)
    q = nq * case["seqs"]
    by = seen * (row + kv / 4) + q * (row * 4 + 8 * H * hd)
    if kind == "prompt":   # the new positions' codes are written
        by += q * row
    if case["scored"]:
        by += 8 * kv * sum(lens)
    return {"bytes": by, "flops": 4 * H * hd * pairs}


# ---- the same in 64 bits ------------------------------------------------------------------------

def _stored(x, length):
    """What a cache holds of one sequence's rows x [length, kv, hd], in 64 bits: the full blocks of 32 rows as
    scale * round(x / scale), the scale and each product 32-bit numbers; the rows after them as they are."""
    full = length // BLOCK * BLOCK
    y = x.double()
    b = y[:full].reshape(full // BLOCK, BLOCK, *x.shape[1:])
    s = (b.abs().amax(dim=3).amax(dim=1) / 127.0).float().double()[:, None, :, None]
    q = torch.where(s > 0, torch.round(b / torch.where(s > 0, s, torch.ones_like(s))), torch.zeros_like(b))
    return torch.cat([(q.clamp(-127, 127) * s).float().double().reshape(full, *x.shape[1:]), y[full:]])


def exact(case, seed):
    x = _inputs(case, seed)
    kind, lens, S, kv = case["kind"], x["lens"], case["seqs"], case["kv"]
    starts = np.cumsum([0] + lens)
    part = lambda name, i: x[name][int(starts[i]):int(starts[i + 1])]  # noqa: E731
    if kind == "fill":
        return {n: torch.cat([_stored(part(n, i), lens[i]) for i in range(S)]) for n in ("k", "v")}
    if kind == "evict":
        keep, out = case["keep"], {"k": [], "v": [], "weights": []}
        for i in range(S):
            w = x["weights"][i, :, :lens[i]].double()
            old = lens[i] - case["recent"]
            at = torch.sort(-w[:, :old], dim=1, stable=True)[1][:, :keep - case["recent"]]
            at = torch.cat([at.sort(dim=1)[0], torch.arange(old, lens[i], device="cuda").expand(kv, -1)], dim=1)
            out["weights"].append(w.gather(1, at))
            for n in ("k", "v"):
                y = _stored(part(n, i), lens[i])
                y = torch.stack([y[at[h], h] for h in range(kv)], dim=1)
                out[n].append(_stored(y, keep))
        return {"kept": None, **{n: torch.stack(v) for n, v in out.items()}}
    nq, H, hd = case.get("n", 1), case["heads"], case["hd"]
    G = H // kv
    outs, ws = [], torch.zeros(S, kv, max(lens), dtype=torch.float64, device="cuda")
    for i in range(S):
        n = lens[i]
        k, v = (_stored(part(m, i), n) for m in ("k", "v"))
        q = x["q"][i * nq:(i + 1) * nq].double()
        qi, kj = torch.arange(n - nq, n, device="cuda")[:, None], torch.arange(n, device="cuda")[None, :]
        see = kj <= qi
        if case["window"]:
            see = see & (qi - kj < case["window"])
        see = see | (kj < case["prefix"])
        o = torch.empty(nq, H, hd, dtype=torch.float64, device="cuda")
        for h in range(H):
            sc = (q[:, h] @ k[:, h // G].t()) * _scale(case)
            if case["cap"]:
                sc = torch.tanh(sc / case["cap"]) * case["cap"]
            p = torch.softmax(torch.where(see, sc, torch.full_like(sc, -float("inf"))), dim=1)
            o[:, h] = p @ v[:, h // G]
            ws[i, h // G, :n] += p.sum(dim=0)
        outs.append(o)
        if case["scored"]:
            ws[i, :, :n - nq] += x["weights"][i, :, :n - nq].double()
    res = {"out": torch.cat(outs)}
    if case["scored"]:
        res["weights"] = ws
    return res
