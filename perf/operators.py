"""Window attention with sinks and the paged key/value cache, as cases that can be timed and compared.

Five operators on plain CUDA tensors in ``torch_mojo_backend_b200.raw``:

* ``window_fwd`` / ``window_bwd``: causal attention in which a query at position p sees the keys p - W + 1 .. p and the
  first N ones (the sinks), for training (kind "train") and for prompts ("prefill");
* ``paged_append``: new keys (rotated by position on the way) and values into the pages of a cache of 16 or 4 bits, and
  the rotated queries beside them ("append");
* ``paged_attention``: the newest tokens of every sequence against its pages, of 16 bits or of 4 ("attend");
* ``paged_gather``: sequences read back out of the pages as dense tensors ("gather", and behind every append of 4 bits,
  which is how the values that the codes stand for are seen).

A cache of 4 bits holds codes 0..15 of 32 elements each with a scale and a minimum of the cache's 16-bit type; an element
is code * scale + minimum.  The order of the codes in a row is `_k_order` / `_v_order` below.

Where ``own`` is false the same results are computed by elementary torch operations in 32 bits.
"""

from __future__ import annotations

import functools
import random

import numpy as np
import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_GROUP = 32   # elements that share a scale and a minimum


# --------------------------------------------------------------------------- cases
def _window(kind, B, Hq, Hkv, Sq, Sk, D, dtype, window, sinks, std=1.0):
    return {"kind": kind, "B": B, "Hq": Hq, "Hkv": Hkv, "Sq": Sq, "Sk": Sk, "D": D, "dtype": dtype, "window": window,
            "sinks": sinks, "std": std}


def _paged(kind, B, Hq, Hkv, S, D, dtype, bits, page, longest, *, spread=0.0, padded=False, window=0, sinks=0, rotary=0,
           interleaved=False):
    """`longest`: keys of the longest sequence, the new ones included; the shortest has (1 - spread) of them.  `padded`: the
    sequences have 1 to S new tokens, not S each."""
    return {"kind": kind, "B": B, "Hq": Hq, "Hkv": Hkv, "S": S, "D": D, "dtype": dtype, "bits": bits, "page": page,
            "longest": longest, "spread": spread, "padded": padded, "window": window, "sinks": sinks, "rotary": rotary,
            "interleaved": interleaved}


def listed():
    return [
        # training step of GPT-2-small's attention with a local window: a call of this size is mostly latency
        {"name": "gpt2-window-train-bf16", **_window("train", 2, 12, 12, 1024, 1024, 64, "bf16", 256, 4)},
        # Llama-style grouped-query training step on an 8k context, window of 1k
        {"name": "llama-window-train-bf16", **_window("train", 2, 32, 8, 8192, 8192, 128, "bf16", 1024, 4, 0.5)},
        # an fp32 run on sequences whose length fits no tile, sinks that end inside one
        {"name": "ragged-window-train-fp32", **_window("train", 3, 8, 4, 777, 777, 64, "fp32", 200, 3)},
        # the last 16k tokens of a 20001-token prompt, against what is already there
        {"name": "window-prefill-fp16", **_window("prefill", 1, 32, 8, 16384, 20001, 128, "fp16", 2048, 4)},
        # one decoding step of a large batch: the new token of every sequence rotated and appended
        {"name": "append-step-bf16", **_paged("append", 64, 32, 8, 1, 128, "bf16", 16, 16, 2048, spread=0.9, rotary=128)},
        # prompts of different lengths written to a 4-bit cache, then read back; half of each head rotated, in pairs
        {"name": "append-prompt-4bit-fp16", **_paged("append", 6, 16, 4, 1500, 64, "fp16", 4, 32, 1700, spread=0.1, padded=True,
                                                     rotary=32, interleaved=True)},
        # one decoding step of an ordinary chat: caches of about a thousand tokens
        {"name": "decode-chat-fp16", **_paged("attend", 4, 32, 8, 1, 128, "fp16", 16, 16, 1000, spread=0.3)},
        # one decoding step over long caches of very different lengths
        {"name": "decode-long-bf16", **_paged("attend", 8, 32, 8, 1, 128, "bf16", 16, 64, 32768, spread=0.6)},
        # a long-running stream per sequence: a window of the cache and its first tokens, drafted tokens verified at once
        {"name": "verify-window-bf16", **_paged("attend", 32, 32, 8, 4, 128, "bf16", 16, 32, 9000, spread=0.9, padded=True, window=1024,
                                                sinks=4)},
        # one decoding step over long caches of 4 bits
        {"name": "decode-long-4bit-bf16", **_paged("attend", 16, 32, 8, 1, 128, "bf16", 4, 64, 32768, spread=0.3)},
        # a chat's step over a 4-bit cache of small heads
        {"name": "decode-chat-4bit-fp16", **_paged("attend", 3, 12, 12, 1, 64, "fp16", 4, 16, 1100, spread=0.5)},
        # cached prompts made dense for a long next chunk
        {"name": "gather-bf16", **_paged("gather", 4, 32, 8, 1, 128, "bf16", 16, 64, 16896, spread=0.2)},
    ]


def _length(rng, lo, hi):
    """Spread over the logarithm of the range; a round number as often as not."""
    n = int(round(lo * (hi / lo) ** rng.random()))
    if rng.random() < 0.5 and n >= 128:
        n = n // 64 * 64
    return max(1, n)


_MOST_PAIRS = 2 * 32 * 8192 * 1024 * 128    # visible pairs x head dimension of the largest training case
_MOST_CACHE = 16 * 32768 * 8 * 128          # elements of K of the largest cache


def draw(rng):
    while True:
        kind = rng.choice(["train", "train", "prefill", "append", "append", "attend", "attend", "attend", "attend", "gather"])
        hkv = rng.choice([1, 2, 4, 6, 8, 12, 16])
        hq = hkv * rng.choice([1, 1, 2, 3, 4, 8])
        d = rng.choice([64, 128])
        if kind in ("train", "prefill"):
            dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
            sq = _length(rng, 32, 16384)
            sk = sq + (_length(rng, 1, 8192) if kind == "prefill" and rng.random() < 0.5 else 0)
            c = _window(kind, _length(rng, 1, 8), hq, hkv, sq, sk, d, dtype, _length(rng, 16, 4096), rng.choice([0, 0, 1, 4, 4, 130]),
                        rng.choice([0.5, 1.0]))
            heavy = c["B"] * c["Hq"] * _pairs(c) * d * (1 if dtype != "fp32" else 16)
            values = c["B"] * d * (hq * sq + 2 * hkv * sk)
            if heavy <= _MOST_PAIRS and values <= 1.5e8:
                return c
            continue
        dtype = rng.choice(["bf16", "fp16"])
        bits, page = rng.choice([16, 4]), rng.choice([16, 32, 64, 128])
        spread = rng.choice([0.0, 0.1, 0.5, 0.9])
        if kind == "append":
            s = rng.choice([1, 1, 3, _length(rng, 2, 4096)])
            half = rng.random() < 0.3
            c = _paged(kind, _length(rng, 1, 128), hq, hkv, s, d, dtype, bits, page, s + _length(rng, 1, 512), spread=0.0 if s > 8 else spread,
                       padded=rng.random() < 0.5, rotary=d // 2 if half else d, interleaved=rng.random() < 0.3)
            if c["B"] * c["longest"] * hkv * d <= 4e7:
                return c
            continue
        longest = _length(rng, 16, 65536)
        s = rng.choice([1, 1, 1, 2, 4, 7]) if kind == "attend" else 1
        windowed = kind == "attend" and rng.random() < 0.4
        c = _paged(kind, _length(rng, 1, 128), hq, hkv, s, d, dtype, bits, page, max(longest, s), spread=spread,
                   padded=s > 1 and rng.random() < 0.5, window=_length(rng, 16, 4096) if windowed else 0,
                   sinks=rng.choice([0, 1, 4, 20]) if windowed else 0)
        if c["B"] * c["longest"] * hkv * d <= (_MOST_CACHE if kind == "attend" else _MOST_CACHE // 4):
            return c


# --------------------------------------------------------------------------- what a case's sizes come to
def _pairs(c):
    """Visible (query, key) pairs of one head of one sequence."""
    pos = np.arange(c["Sq"], dtype=np.int64) + c["Sk"] - c["Sq"]
    near = np.minimum(pos + 1, c["window"])
    return int((near + np.minimum(pos + 1 - near, c["sinks"])).sum())


def _sequences(c):
    """(keys, new tokens) of every sequence, by the case alone."""
    B, S, longest = c["B"], c["S"], c["longest"]
    keys = [max(S, longest - int(c["spread"] * longest * b / B)) for b in range(B)]
    new = [1 + b * (S - 1) // max(1, B - 1) if c["padded"] else S for b in range(B)]
    return keys, new


def _attended(c):
    """Visible (query row, key) pairs of one head over all sequences, and the keys that have to be read."""
    pairs = read = 0
    for keys, new in zip(*_sequences(c)):
        pos = np.arange(keys - new, keys, dtype=np.int64)
        if c["window"]:
            near = np.minimum(pos + 1, c["window"])
            pairs += int((near + np.minimum(pos + 1 - near, c["sinks"])).sum())
            first = max(0, keys - new - c["window"] + 1)
            read += keys - first + min(first, c["sinks"])
        else:
            pairs += int((pos + 1).sum())
            read += keys
    return pairs, read


def _row_bytes(c):
    """Bytes of one key (or value) of one head in the cache."""
    return c["D"] * 2 if c["bits"] == 16 else c["D"] // 2 + c["D"] // _GROUP * 4


def work(c):
    B, Hq, Hkv, D = c["B"], c["Hq"], c["Hkv"], c["D"]
    if c["kind"] in ("train", "prefill"):
        size = 4 if c["dtype"] == "fp32" else 2
        q, kv = B * Hq * c["Sq"] * D * size, 2 * B * Hkv * c["Sk"] * D * size
        forward = 4 * B * Hq * _pairs(c) * D
        lse = 4 * B * Hq * c["Sq"]
        if c["kind"] == "train":
            return {"bytes": 4 * q + 2 * kv + lse, "flops": 3.5 * forward}
        return {"bytes": 2 * q + kv + lse, "flops": forward}
    keys, new = _sequences(c)
    if c["kind"] == "append":
        n = sum(new)
        moved = n * (2 * Hkv * (2 * D + _row_bytes(c)) + 2 * Hq * 2 * D + 4 * c["rotary"])
        if c["bits"] == 4:   # read back: codes and scales in, dense rows out
            moved += 2 * Hkv * (sum(keys) * _row_bytes(c) + B * c["longest"] * D * 2)
        return {"bytes": moved, "flops": n * (Hq + Hkv) * c["rotary"] * 3}
    if c["kind"] == "gather":
        return {"bytes": 2 * Hkv * (sum(keys) * _row_bytes(c) + B * c["longest"] * D * 2), "flops": 0}
    pairs, read = _attended(c)
    rows = sum(new) * Hq
    return {"bytes": 2 * Hkv * read * _row_bytes(c) + rows * (4 * D + 4), "flops": 4 * Hq * pairs * D}


# --------------------------------------------------------------------------- inputs
def _randn(gen, shape, std, dtype):
    t = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32 if dtype == torch.float32 else torch.float16)
    return t.mul_(std).to(dtype)


def _k_order(D):
    """Element of the row that the i-th code of a key's row stands for."""
    return np.arange(D).reshape(D // 32, 4, 8).transpose(1, 0, 2).reshape(-1)


def _v_order(D):
    """Element of the row that the i-th code of a value's row stands for."""
    return np.arange(D).reshape(D // 32, 8, 4).transpose(1, 0, 2).reshape(-1)


@functools.lru_cache(maxsize=None)
def _orders(D):
    """The two orders and their inverses, on the GPU."""
    k, v = _k_order(D), _v_order(D)
    return tuple(torch.from_numpy(np.ascontiguousarray(o)).cuda() for o in (k, v, np.argsort(k), np.argsort(v)))


def _quantise(x, order):
    """(codes of the last dimension's elements, two to a byte in the given order; scale and minimum of every group)."""
    D = x.shape[-1]
    g = x.float().unflatten(-1, (D // _GROUP, _GROUP))
    low = g.amin(-1)
    scale = ((g.amax(-1) - low) / 15).to(x.dtype)
    codes = ((g - low[..., None]) / scale.float()[..., None]).round().clamp(0, 15)
    codes = torch.where(scale[..., None] == 0, 0, codes).flatten(-2)[..., order].to(torch.uint8)
    return codes[..., 0::2] | codes[..., 1::2] << 4, torch.stack([scale, low.to(x.dtype)], -1)


def _values(codes, scales, inverse):
    """What codes and scales stand for, in 32 bits."""
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)[..., inverse].float()
    s = scales.float()
    return (c.unflatten(-1, (-1, _GROUP)) * s[..., :1] + s[..., 1:]).flatten(-2)


def _table(c, rng):
    """(block table with unused entries of -1, number of pages)."""
    keys, _ = _sequences(c)
    rng.shuffle(keys)
    pages = [-(-n // c["page"]) for n in keys]
    spare = 3
    order = list(range(sum(pages) + spare))
    rng.shuffle(order)
    table = np.full((c["B"], -(-c["longest"] // c["page"])), -1, dtype=np.int32)
    at = 0
    for b, n in enumerate(pages):
        table[b, :n] = order[at:at + n]
        at += n
    return table, keys, len(order)


def _rotation(c):
    """cos and sin of every position's angles, computed in 64 bits."""
    angle = np.arange(c["longest"], dtype=np.float64)[:, None] * 10000.0 ** (-np.arange(0, c["rotary"], 2) / c["rotary"])
    return tuple(torch.from_numpy(f(angle).astype(np.float32)).cuda() for f in (np.cos, np.sin))


def _prepare_paged(c, seed):
    B, Hq, Hkv, S, D = (c[n] for n in ("B", "Hq", "Hkv", "S", "D"))
    dtype, rng = _DTYPES[c["dtype"]], random.Random(seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    table, keys, n_pages = _table(c, rng)
    _, new = _sequences(c)
    state = {**c, "table": torch.from_numpy(table).cuda(), "lengths": torch.tensor(keys, dtype=torch.int32, device="cuda"),
             "new": torch.tensor(new, dtype=torch.int32, device="cuda") if c["padded"] else None, "scale": D ** -0.5}
    order_k, order_v, _, _ = _orders(D)
    shape = (n_pages, Hkv, c["page"], D)
    # keys have a few channels that stand out, as models' keys do
    stand_out = torch.ones(D, device="cuda")
    stand_out[:: D // 4] = 3.0
    state["pages"] = []
    scales = []
    for order, spread in ((order_k, stand_out), (order_v, 1.0)):
        x = (_randn(gen, shape, 1.0, dtype) * spread).to(dtype)
        if c["bits"] == 4:
            x, s = _quantise(x, order)
            scales.append(s)
        state["pages"].append(x.contiguous())
    state["pages"] += [s.contiguous() for s in scales]
    # queries, keys and values of the new tokens: views of one fused projection, as a transformer block makes them
    proj = _randn(gen, (B, S, (Hq + 2 * Hkv) * D), 1.0, dtype)
    state["q"], state["k"], state["v"] = (p.unflatten(2, (-1, D)).transpose(1, 2) for p in proj.split([Hq * D, Hkv * D, Hkv * D], 2))
    if c["kind"] == "append":
        state["cos"], state["sin"] = _rotation(c)
        state["q_out"] = torch.zeros((B, Hq, S, D), dtype=dtype, device="cuda")
    if c["kind"] == "attend":
        # rows behind a sequence's new tokens stay what they are
        state["out"] = torch.zeros((B, Hq, S, D), dtype=dtype, device="cuda")
        state["lse"] = torch.zeros((B, Hq, S), dtype=torch.float32, device="cuda")
    return state


def prepare(case, seed):
    if case["kind"] not in ("train", "prefill"):
        return _prepare_paged(case, seed)
    B, Hq, Hkv, Sq, Sk, D = (case[n] for n in ("B", "Hq", "Hkv", "Sq", "Sk", "D"))
    dtype, std = _DTYPES[case["dtype"]], case["std"]
    gen = torch.Generator(device="cuda").manual_seed(seed)
    state = {**case, "q": _randn(gen, (B, Hq, Sq, D), std, dtype), "k": _randn(gen, (B, Hkv, Sk, D), std, dtype),
             "v": _randn(gen, (B, Hkv, Sk, D), std, dtype), "scale": D ** -0.5}
    if case["kind"] == "train":
        state["grad"] = _randn(gen, (B, Hq, Sq, D), 1.0, dtype)
    return state


# --------------------------------------------------------------------------- the plain forms
_PLAIN_SCORES = 1 << 29   # scores in 32 bits held at a time


def _plain_window(st):
    """Query rows in chunks of what memory holds, each against the keys that it can see."""
    q, k, v, W, N = st["q"], st["k"], st["v"], st["window"], st["sinks"]
    (B, Hq, Sq, D), (Hkv, Sk) = q.shape, k.shape[1:3]
    group, off, scale = Hq // Hkv, Sk - Sq, st["scale"]
    train = "grad" in st
    res = {"out": torch.empty_like(q), "lse": torch.empty((B, Hq, Sq), device="cuda")}
    if train:
        res["dq"] = torch.empty_like(q)
        dk, dv = (torch.zeros(k.shape, device="cuda") for _ in range(2))
    kf, vf = k.float(), v.float()
    rows = max(64, min(Sq, _PLAIN_SCORES // (B * Hq * min(Sk, W + N + 1024)), 1024))
    for r0 in range(0, Sq, rows):
        r1 = min(Sq, r0 + rows)
        pos = torch.arange(r0, r1, device="cuda") + off
        first = max(N, r0 + off - W + 1)
        cols = torch.cat([torch.arange(min(N, r1 + off), device="cuda"), torch.arange(min(first, r1 + off), r1 + off, device="cuda")])
        kc, vc = kf[:, :, None, cols], vf[:, :, None, cols]
        qc = q[:, :, r0:r1].float().unflatten(1, (Hkv, group)) * scale
        s = qc @ kc.mT
        seen = (cols <= pos[:, None]) & ((cols > pos[:, None] - W) | (cols < N))
        s.masked_fill_(~seen, -torch.inf)
        top = s.amax(-1, keepdim=True)
        p = s.sub_(top).exp_()
        total = p.sum(-1, keepdim=True)
        p.div_(total)
        o = p @ vc
        res["out"][:, :, r0:r1] = o.flatten(1, 2)
        res["lse"][:, :, r0:r1] = (top + total.log()).flatten(1, 2)[..., 0]
        if train:
            g = st["grad"][:, :, r0:r1].float().unflatten(1, (Hkv, group))
            dv[:, :, cols] += (p.mT @ g).sum(2)
            ds = p.mul_((g @ vc.mT).sub_((g * o).sum(-1, keepdim=True)))
            res["dq"][:, :, r0:r1] = ((ds @ kc) * scale).flatten(1, 2)
            dk[:, :, cols] += (ds.mT @ qc).sum(2)
    if train:
        res["dk"], res["dv"] = dk.to(k.dtype), dv.to(v.dtype)
    return res


def _new_tokens(st):
    """How many of the S new tokens of each sequence there are."""
    return st["new"] if st["new"] is not None else torch.full_like(st["lengths"], st["S"])


def _plain_rotate(x, cos, sin, interleaved):
    """x (..., D) by the angles (..., R / 2) of its positions, in 32 bits."""
    R, x = 2 * cos.shape[-1], x.float()
    a, b = (x[..., 0:R:2], x[..., 1:R:2]) if interleaved else (x[..., :R // 2], x[..., R // 2:R])
    a, b = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
    return torch.cat([turned, x[..., R:]], -1)


def _plain_append(st):
    new, lengths, S, dtype = _new_tokens(st), st["lengths"], st["S"], st["q"].dtype
    step = torch.arange(S, device="cuda")
    there = step < new[:, None]                                                  # (B, S)
    pos = torch.where(there, (lengths - new)[:, None] + step, 0).long()
    cos, sin = st["cos"][pos][:, :, None], st["sin"][pos][:, :, None]            # (B, S, 1, R / 2)
    q, k, v = (st[n].transpose(1, 2) for n in ("q", "k", "v"))                   # (B, S, H, D)
    q = _plain_rotate(q, cos, sin, st["interleaved"]).to(dtype)
    k = _plain_rotate(k, cos, sin, st["interleaved"]).to(dtype)
    st["q_out"].copy_(torch.where(there[:, None, :, None], q.transpose(1, 2), st["q_out"]))
    seq, at = there.nonzero(as_tuple=True)
    page, slot = st["table"][seq, pos[seq, at] // st["page"]].long(), pos[seq, at] % st["page"]
    rows = [k[seq, at], v[seq, at]]
    if st["bits"] == 4:
        order_k, order_v, _, _ = _orders(st["D"])
        (ck, sk), (cv, sv) = _quantise(rows[0], order_k), _quantise(rows[1], order_v)
        rows = [ck, cv, sk, sv]
    for pages, row in zip(st["pages"], rows):
        pages[page, :, slot] = row
    if st["bits"] == 16:
        return {"q": st["q_out"], "k_pages": st["pages"][0], "v_pages": st["pages"][1]}
    return {"q": st["q_out"], **_plain_gather(st)}


def _plain_rows(st, pos):
    """k and v at positions (B, n) of the sequences, as (B, n, H, D) in 32 bits."""
    page, slot = st["table"].gather(1, pos // st["page"]).long().clamp_(min=0), pos % st["page"]
    got = [p[page, :, slot] for p in st["pages"]]
    if st["bits"] == 16:
        return got[0].float(), got[1].float()
    _, _, inverse_k, inverse_v = _orders(st["D"])
    return _values(got[0], got[2], inverse_k), _values(got[1], got[3], inverse_v)


def _plain_gather(st):
    pos = torch.arange(st["longest"], device="cuda").expand(st["B"], -1)
    there = pos < st["lengths"][:, None]
    k, v = _plain_rows(st, pos)
    return {n: torch.where(there[:, :, None, None], x, 0).to(st["q"].dtype).transpose(1, 2).contiguous() for n, x in (("k", k), ("v", v))}


def _plain_attend(st):
    B, Hq, Hkv, S, W, N = (st[n] for n in ("B", "Hq", "Hkv", "S", "window", "sinks"))
    new, lengths = _new_tokens(st).long(), st["lengths"].long()
    if W:   # the sinks, then the span that the new tokens' windows cover
        span = torch.arange(min(W + S - 1, st["longest"]), device="cuda")
        start = (lengths - new - W + 1).clamp(min=N)[:, None]
        pos = torch.cat([torch.arange(N, device="cuda").expand(B, -1), start + span], 1)
    else:
        pos = torch.arange(st["longest"], device="cuda").expand(B, -1)
    there = pos < lengths[:, None]
    k, v = (x.transpose(1, 2)[:, :, None] for x in _plain_rows(st, torch.where(there, pos, 0)))   # (B, Hkv, 1, n, D)
    q = st["q"].float().unflatten(1, (Hkv, Hq // Hkv)) * st["scale"]
    s = q @ k.mT                                                                                  # (B, Hkv, group, S, n)
    at = ((lengths - new)[:, None] + torch.arange(S, device="cuda"))[:, None, None, :, None]
    key = pos[:, None, None, None]
    seen = there[:, None, None, None] & (key <= at)
    if W:
        seen = seen & ((key > at - W) | (key < N))
    s = s.masked_fill_(~seen, -torch.inf)
    top = s.amax(-1, keepdim=True).clamp_(min=-3e38)
    p = s.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = (p @ v / total).flatten(1, 2).to(st["q"].dtype)
    lse = (top + total.log()).flatten(1, 2)[..., 0]
    row = (torch.arange(S, device="cuda") < new[:, None])[:, None]
    st["out"].copy_(torch.where(row[..., None], out, st["out"]))
    st["lse"].copy_(torch.where(row, lse, st["lse"]))
    return {"out": st["out"], "lse": st["lse"]}


# --------------------------------------------------------------------------- one pass
def _own(st):
    from torch_mojo_backend_b200 import _lib, raw

    if st["kind"] in ("train", "prefill"):
        how = {"window": st["window"], "sinks": st["sinks"], "causal": _lib.CAUSAL_BOTTOM_RIGHT, "scale": st["scale"]}
        q, k, v = st["q"], st["k"], st["v"]
        out, lse = raw.window_fwd(q, k, v, **how)
        res = {"out": out, "lse": lse}
        if st["kind"] == "train":
            res["dq"], res["dk"], res["dv"] = raw.window_bwd(st["grad"], q, k, v, out, lse, **how)
        return res
    cache = raw.PagedKV(*st["pages"])
    if st["kind"] == "attend":
        out, lse = raw.paged_attention(st["q"], cache, st["table"], st["lengths"], new_lengths=st["new"], window=st["window"],
                                       sinks=st["sinks"], scale=st["scale"], out=st["out"], lse=st["lse"])
        return {"out": out, "lse": lse}
    if st["kind"] == "append":
        raw.paged_append(st["k"], st["v"], cache, st["table"], st["lengths"], new_lengths=st["new"], rotary=(st["cos"], st["sin"]),
                         interleaved=st["interleaved"], q=st["q"], q_out=st["q_out"])
        if st["bits"] == 16:
            return {"q": st["q_out"], "k_pages": cache.k, "v_pages": cache.v}
    k, v = raw.paged_gather(cache, st["table"], st["lengths"], st["longest"])
    return {"k": k, "v": v} if st["kind"] == "gather" else {"q": st["q_out"], "k": k, "v": v}


def run(state):
    if own:
        return _own(state)
    kind = state["kind"]
    if kind in ("train", "prefill"):
        return _plain_window(state)
    return {"append": _plain_append, "attend": _plain_attend, "gather": _plain_gather}[kind](state)


# --------------------------------------------------------------------------- the same in 64 bits
def _exact_window(case, seed):
    st = prepare(case, seed)
    q, k, v, W, N = st["q"], st["k"], st["v"], case["window"], case["sinks"]
    (B, Hq, Sq, D), (Hkv, Sk) = q.shape, k.shape[1:3]
    group, scale, grad = Hq // Hkv, D ** -0.5, st.get("grad")
    f64 = {"dtype": torch.float64, "device": "cuda"}
    res = {"out": torch.empty(q.shape, **f64), "lse": torch.empty(q.shape[:3], **f64)}
    if grad is not None:
        res.update(dq=torch.empty(q.shape, **f64), dk=torch.zeros(k.shape, **f64), dv=torch.zeros(v.shape, **f64))
    for b in range(B):
        for h in range(Hq):
            k64, v64 = k[b, h // group].double(), v[b, h // group].double()
            for r0 in range(0, Sq, 2048):
                r = slice(r0, min(Sq, r0 + 2048))
                p0, p1 = r.start + Sk - Sq, r.stop + Sk - Sq      # positions of these rows
                w = slice(max(0, p0 - W + 1), p1)                 # the keys of their windows; the sinks ahead of it apart
                n = min(N, w.start)
                k2, v2 = torch.cat([k64[:n], k64[w]]), torch.cat([v64[:n], v64[w]])
                key = torch.cat([torch.arange(n), torch.arange(w.start, w.stop)]).cuda()
                pos = torch.arange(p0, p1).cuda()[:, None]
                s = q[b, h, r].double() @ k2.T * scale
                s[(key > pos) | ((pos - key >= W) & (key >= N))] = -torch.inf
                res["lse"][b, h, r] = torch.logsumexp(s, -1)
                p = torch.softmax(s, -1)
                res["out"][b, h, r] = o = p @ v2
                if grad is not None:
                    g = grad[b, h, r].double()
                    ds = p * (g @ v2.T - (g * o).sum(1, keepdim=True))
                    res["dq"][b, h, r] = ds @ k2 * scale
                    dk, dv = ds.T @ q[b, h, r].double() * scale, p.T @ g
                    for name, x in (("dk", dk), ("dv", dv)):
                        res[name][b, h // group, :n] += x[:n]
                        res[name][b, h // group, w] += x[n:]
    return res


def _exact_sequence(st, b, n):
    """k and v of the first n tokens of sequence b, (H, n, D) in 64 bits."""
    at = st["table"][b, :-(-n // st["page"])].long()
    rows = [p[at].transpose(0, 1).flatten(1, 2)[:, :n] for p in st["pages"]]
    if st["bits"] == 16:
        return rows[0].double(), rows[1].double()
    D, res = st["D"], []
    for codes, scales, order in ((rows[0], rows[2], _k_order(D)), (rows[1], rows[3], _v_order(D))):
        x = torch.empty((*codes.shape[:2], D), dtype=torch.float64, device="cuda")
        for half in (0, 1):
            element = torch.from_numpy(np.ascontiguousarray(order[half::2])).cuda()
            of = element // _GROUP
            x[..., element] = (codes.int() // 16 ** half % 16).double() * scales[..., of, 0].double() + scales[..., of, 1].double()
        res.append(x)
    return res


def _exact_attend(case, seed):
    st = prepare(case, seed)
    B, Hq, Hkv, S, D, W, N = (case[n] for n in ("B", "Hq", "Hkv", "S", "D", "window", "sinks"))
    res = {"out": st["out"].double(), "lse": st["lse"].double()}
    lengths = st["lengths"].tolist()
    new = st["new"].tolist() if st["new"] is not None else [S] * B
    for b in range(B):
        n, t = lengths[b], new[b]
        k, v = _exact_sequence(st, b, n)
        key = torch.arange(n, device="cuda")
        pos = torch.arange(n - t, n, device="cuda")[:, None]
        hidden = key > pos
        if W:
            hidden |= (pos - key >= W) & (key >= N)
        for h in range(Hq):
            s = st["q"][b, h, :t].double() @ k[h * Hkv // Hq].T * D ** -0.5
            s[hidden] = -torch.inf
            res["lse"][b, h, :t] = torch.logsumexp(s, -1)
            res["out"][b, h, :t] = torch.softmax(s, -1) @ v[h * Hkv // Hq]
    return res


def _exact_rotated(x, pos, rotary, interleaved, cos, sin):
    """x (H, n, D) at positions `pos` (n), as complex numbers times cos + i sin."""
    y, R = x.double().clone(), rotary
    turn = torch.complex(cos[pos].double(), sin[pos].double())
    if interleaved:
        z = torch.complex(y[..., 0:R:2], y[..., 1:R:2]) * turn
        y[..., 0:R:2], y[..., 1:R:2] = z.real, z.imag
    else:
        z = torch.complex(y[..., :R // 2], y[..., R // 2:R]) * turn
        y[..., :R // 2], y[..., R // 2:R] = z.real, z.imag
    return y


def _exact_append(case, seed):
    """Rotated queries and, in a 16-bit cache, the pages.  What a 4-bit cache then holds depends on where roundings fall: none of it
    has a value of its own in 64 bits but for the new tokens' absence."""
    st = prepare(case, seed)
    q = st["q_out"].double()
    k_pages, v_pages = (p.double() for p in st["pages"][:2]) if case["bits"] == 16 else (None, None)
    lengths = st["lengths"].tolist()
    new = st["new"].tolist() if st["new"] is not None else [case["S"]] * case["B"]
    for b in range(case["B"]):
        t = new[b]
        pos = torch.arange(lengths[b] - t, lengths[b], device="cuda")
        how = (pos, case["rotary"], case["interleaved"], st["cos"], st["sin"])
        q[b, :, :t] = _exact_rotated(st["q"][b, :, :t], *how)
        if case["bits"] == 16:
            page, slot = st["table"][b, pos // case["page"]].long(), pos % case["page"]
            k_pages[page, :, slot] = _exact_rotated(st["k"][b, :, :t], *how).transpose(0, 1)
            v_pages[page, :, slot] = st["v"][b, :, :t].double().transpose(0, 1)
    if case["bits"] == 16:
        return {"q": q, "k_pages": k_pages, "v_pages": v_pages}
    return {"q": q, "k": None, "v": None}


def _exact_gather(case, seed):
    st = prepare(case, seed)
    k, v = (torch.zeros((case["B"], case["Hkv"], case["longest"], case["D"]), dtype=torch.float64, device="cuda") for _ in range(2))
    for b, n in enumerate(st["lengths"].tolist()):
        k[b, :, :n], v[b, :, :n] = _exact_sequence(st, b, n)
    return {"k": k, "v": v}


def exact(case, seed):
    if case["kind"] in ("train", "prefill"):
        # 64-bit products of the pairs that the chunks hold
        cost = 4 * case["B"] * case["Hq"] * case["Sq"] * min(case["Sk"], case["window"] + case["sinks"] + 2048) * case["D"]
        return _exact_window(case, seed) if cost * (3.5 if case["kind"] == "train" else 1) < 4e13 else None
    return {"append": _exact_append, "attend": _exact_attend, "gather": _exact_gather}[case["kind"]](case, seed)
