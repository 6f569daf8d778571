"""Attention over a window of keys and the first ones, forward and backward (``-m gpu``), against the formula in 64 bits.

The bounds are element by element, from the roundings that the kernels make.  With u half a step of the type (relative), s the
relative error of a probability (that of its score: an fp32 sum of D products, and of the exponential), A = P |V|:
  out: P is rounded before it multiplies V, out after                           u A + u |out| + 3 s A
  lse: the error of a score, and of an fp32 sum of n terms
  dV:  the same with |dO| for |V|                                                u P^T|dO| + u |dV| + ...
  dS = P (dP - rowsum(dO out)): rounded before it is multiplied on; the row sum is taken of the rounded out, off by
       u R with R = |dO| |out|                                                   E = u |dS| + u P R + s (|dS| + P R + P |dP|)
  dQ, dK: scale E |K| + u |dQ|, scale E^T |Q| + u |dK|
A 16-bit float of the fp16 kind has no smaller step than 2^-24, so a rounding there is off by u times the value or by t = 2^-25,
whichever is more: t is added wherever u is, once per rounded term.
"""

import pytest
import torch

from torch_mojo_backend_b200 import _lib, raw

pytestmark = pytest.mark.gpu

TL, BR = _lib.CAUSAL_TOP_LEFT, _lib.CAUSAL_BOTTOM_RIGHT


def inputs(seed, B, Hq, Hkv, Sq, Sk, D, dtype, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    draw = lambda *shape: (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)
    return draw(B, Hq, Sq, D), draw(B, Hkv, Sk, D), draw(B, Hkv, Sk, D), draw(B, Hq, Sq, D)


def visible(Sq, Sk, causal, window, sinks):
    """(Sq, Sk) of truth values."""
    p = torch.arange(Sq, device="cuda")[:, None] + (Sk - Sq if causal == BR else 0)
    j = torch.arange(Sk, device="cuda")[None]
    return (j <= p) & ((j > p - window) | (j < sinks))


def reference(q, k, v, grad, causal, window, sinks):
    """name -> (value in 64 bits, bound of the error)"""
    (B, Hq, Sq, D), (Hkv, Sk) = q.shape, k.shape[1:3]
    scale, group = D ** -0.5, Hq // Hkv
    u = torch.finfo(q.dtype).eps / 2
    t = 2.0 ** -25 if q.dtype == torch.float16 else 0.0
    seen = visible(Sq, Sk, causal, window, sinks)
    q, grad = (t.double().unflatten(1, (Hkv, group)) for t in (q, grad))
    k, v = (t.double()[:, :, None] for t in (k, v))
    s = (q @ k.mT * scale).masked_fill(~seen, -torch.inf)
    lse = torch.logsumexp(s, -1)
    p = torch.exp(s - lse.clamp(min=-1e300)[..., None])
    # an fp32 sum of D products, each at most 2^-23 off (tensor cores truncate), the exponential 2^-21, a row sum of n terms
    n = int(seen.sum(1).max())
    e = float((q.abs() @ k.abs().mT).max()) * scale * D * 2 ** -23 + 2.0 ** -21 + n * 2.0 ** -24
    out = p @ v
    a = p @ v.abs()
    least = t * seen.double()
    res = {"out": (out, u * (a + out.abs()) + t + least @ v.abs() + 3 * e * a), "lse": (lse, e + 2.0 ** -23 * lse.abs())}
    dp = grad @ v.mT
    row = (grad * out).sum(-1, keepdim=True)
    ds = p * (dp - row)
    r = (grad.abs() * (out.abs() + a)).sum(-1, keepdim=True)
    r = r + t * grad.abs().sum(-1, keepdim=True) / u
    es = u * (ds.abs() + p * r) + least + 3 * e * (ds.abs() + p * r + p * (grad.abs() @ v.abs().mT))
    dv, dva = ((x.mT @ y).sum(2) for x, y in ((p, grad), (p, grad.abs())))
    dq, dk = ds @ k * scale, (ds.mT @ q).sum(2) * scale
    rows = 1 + group * Sq * 2.0 ** -24 / max(e, 1e-30)   # sums over query rows are longer
    res["dv"] = dv, u * (dva + dv.abs()) + t + (least.mT @ grad.abs()).sum(2) + 3 * e * rows * dva
    res["dq"] = dq, es @ k.abs() * scale + u * dq.abs() + t
    res["dk"] = dk, (es.mT @ q.abs()).sum(2) * scale * (1 + (rows - 1) * e / u) + u * dk.abs() + t
    return {n: (x.flatten(1, 2) if n in ("out", "lse", "dq") else x, b.flatten(1, 2) if n in ("out", "lse", "dq") else b)
            for n, (x, b) in res.items()}


def check(name, got, want, bound):
    got = got.double()
    if name == "lse":
        assert torch.equal(torch.isneginf(got), torch.isneginf(want)), "rows that see no key"
        got, want, bound = (torch.where(torch.isneginf(want), 0.0, t) for t in (got, want, bound))
    assert torch.isfinite(got).all(), name
    over = ((got - want).abs() - bound - 1e-30).max().item()
    assert over <= 0, f"{name}: {over:.3e} over its bound; largest error {(got - want).abs().max().item():.3e}"


def run_both(q, k, v, grad, causal, window, sinks):
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out, lse = raw.window_fwd(q, k, v, window=window, sinks=sinks, causal=causal, status=status)
    dq, dk, dv = raw.window_bwd(grad, q, k, v, out, lse, window=window, sinks=sinks, causal=causal, status=status)
    torch.cuda.synchronize()
    assert int(status) == 0
    return {"out": out, "lse": lse, "dq": dq, "dk": dk, "dv": dv}


CASES = [
    # B, Hq, Hkv, Sq, Sk, D, causal, window, sinks
    (1, 2, 2, 1, 1, 64, TL, 1, 0),            # one token
    (2, 4, 2, 7, 7, 128, TL, 3, 1),
    (1, 4, 1, 300, 300, 64, TL, 1, 0),        # every row sees itself alone
    (1, 4, 1, 300, 300, 128, TL, 1, 2),
    (2, 4, 2, 513, 513, 128, TL, 128, 0),     # the window ends on tile borders, one row behind the last
    (2, 4, 2, 640, 640, 64, TL, 129, 4),
    (1, 6, 3, 1000, 1000, 128, TL, 200, 130),   # sinks that end inside the second block
    (1, 2, 2, 900, 900, 64, TL, 64, 900),     # sinks of everything: the causal mask
    (1, 2, 1, 700, 700, 128, TL, 5000, 0),    # a window of everything
    (1, 2, 1, 700, 700, 64, TL, 1 << 40, 1 << 40),
    (1, 2, 2, 130, 1500, 128, BR, 300, 4),    # new queries behind a longer sequence
    (3, 4, 4, 33, 2050, 64, BR, 1024, 1),
    (1, 4, 2, 600, 200, 128, BR, 50, 2),      # 400 rows without a key
    (1, 4, 2, 900, 200, 64, TL, 64, 0),       # rows whose window lies behind the last key
    (1, 4, 2, 900, 200, 128, TL, 64, 3),      # ... and who see the sinks alone
    (2, 4, 2, 900, 100, 64, TL, 64, 129),     # ... more sinks than keys
    (2, 4, 2, 900, 230, 128, TL, 5, 300),
    (1, 1, 1, 2900, 2900, 128, TL, 64, 4),    # few heads: the sinks' tile is shared by several blocks
    (1, 8, 2, 2100, 2100, 64, TL, 256, 200),
    (1, 4, 2, 200, 3000, 128, BR, 1500, 4),   # few heads, which share K/V: their keys are shared by several blocks
    (1, 8, 1, 70, 2500, 128, BR, 1024, 130),
    (2, 6, 2, 1100, 1100, 128, TL, 150, 64),  # three heads to a K/V head; sinks of half a block
    (1, 4, 2, 1100, 1100, 128, TL, 150, 65),
    (1, 4, 2, 1100, 1100, 64, TL, 100, 192),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,Hq,Hkv,Sq,Sk,D,causal,window,sinks", CASES)
def test_against_the_formula(B, Hq, Hkv, Sq, Sk, D, causal, window, sinks, dtype):
    q, k, v, grad = inputs(3, B, Hq, Hkv, Sq, Sk, D, dtype)
    got = run_both(q, k, v, grad, causal, window, sinks)
    for name, (want, bound) in reference(q, k, v, grad, causal, window, sinks).items():
        check(name, got[name], want, bound)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_scores_far_below_zero_behind_a_block_that_a_row_does_not_see(dtype):
    """The first block a row's tile visits may hold no key of the row: its maximum must not start at zero there."""
    q, k, v, grad = inputs(5, 1, 2, 2, 520, 520, 128, dtype, std=0.5)
    k = (-q.float() * 4 + k.float() * 0.1 - 2).to(dtype)     # every score is some -100
    got = run_both(q, k, v, grad, TL, 130, 0)
    for name, (want, bound) in reference(q, k, v, grad, TL, 130, 0).items():
        check(name, got[name], want, bound)


def test_keys_that_are_not_finite_behind_the_mask():
    """Scores behind the mask are replaced, whatever they are."""
    q, k, v, grad = inputs(6, 1, 2, 1, 400, 400, 64, torch.bfloat16)
    clean = run_both(q, k, v, grad, TL, 100, 2)
    bad = k.clone()
    bad[:, :, 20] = float("nan")   # seen by rows 20 .. 119 alone
    bad[:, :, 30] = float("inf")
    out, lse = raw.window_fwd(q, bad, v, window=100, sinks=2)
    apart = [0, 10, 19, 131, 200, 399]
    assert torch.equal(out[:, :, apart], clean["out"][:, :, apart]) and torch.equal(lse[:, :, apart], clean["lse"][:, :, apart])
    assert torch.isnan(out[:, :, 60]).all()


def test_strided_views_and_given_outputs():
    """Views of one fused projection, a sequence-major output, statistics and workspace of the caller's."""
    B, Hq, Hkv, S, D = 2, 6, 2, 345, 64
    g = torch.Generator(device="cuda").manual_seed(8)
    fused = torch.randn(B, S, (Hq + 2 * Hkv) * D, generator=g, device="cuda").bfloat16()
    q, k, v = (t.unflatten(2, (-1, D)).transpose(1, 2) for t in fused.split([Hq * D, Hkv * D, Hkv * D], 2))
    grad = torch.randn(B, S, Hq, D, generator=g, device="cuda").bfloat16().transpose(1, 2)
    out = torch.empty(B, S, Hq, D, dtype=torch.bfloat16, device="cuda").transpose(1, 2)
    lse = torch.empty(B, Hq, S, device="cuda")
    raw.window_fwd(q, k, v, window=77, sinks=5, out=out, lse=lse)
    need = _lib.window_bwd_workspace_bytes(B, Hq, Hkv, S, S, D, _lib.BF16, 77, 5)
    workspace = torch.full((need,), 255, dtype=torch.uint8, device="cuda")   # NaN everywhere
    dq, dk, dv = raw.window_bwd(grad, q, k, v, out, lse, window=77, sinks=5, workspace=workspace)
    got = {"out": out, "lse": lse, "dq": dq, "dk": dk, "dv": dv}
    for name, (want, bound) in reference(q, k, v, grad, TL, 77, 5).items():
        check(name, got[name], want, bound)


def test_gradients_against_differences():
    """fp32: (L(x + h d) - L(x - h d)) / 2h against <gradient, d>, L = <out, grad>.  L's terms are off by some 2^-20 of their
    size (sums of 60 keys), 2^-20 |L|_1 / h in the quotient; the third derivative's part is h^2 of the quotient's size."""
    q, k, v, grad = inputs(9, 1, 2, 1, 150, 150, 64, torch.float32, std=0.5)
    got = run_both(q, k, v, grad, TL, 50, 3)
    h = 2.0 ** -6
    for i, name in enumerate(("dq", "dk", "dv")):
        d = torch.randn(got[name].shape, generator=torch.Generator(device="cuda").manual_seed(i), device="cuda")
        values = []
        for sign in (1, -1):
            x = [q, k, v]
            x[i] = x[i] + sign * h * d
            out, _ = raw.window_fwd(*x, window=50, sinks=3)
            values.append(out.double() * grad.double())
        quotient = (values[0].sum() - values[1].sum()).item() / (2 * h)
        want = (got[name].double() * d.double()).sum().item()
        size = (got[name].double() * d.double()).norm().item()
        noise = 2.0 ** -20 * values[0].norm().item() / h      # (independent errors add up in 2-norm)
        assert abs(quotient - want) <= 10 * noise + 50 * h * h * size, (name, quotient, want)


def test_a_call_is_ordered_on_its_stream_and_can_be_captured():
    q, k, v, grad = inputs(10, 1, 2, 1, 2048, 2048, 128, torch.bfloat16)
    want = run_both(q, k, v, grad, TL, 200, 4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = run_both(q, k, v, grad, TL, 200, 4)
    torch.cuda.current_stream().wait_stream(side)
    for n in want:
        assert torch.equal(want[n], again[n]), n
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = raw.window_fwd(q, k, v, window=200, sinks=4)
        dq, dk, dv = raw.window_bwd(grad, q, k, v, out, lse, window=200, sinks=4)
    q2, k2, v2, grad2 = inputs(11, 1, 2, 1, 2048, 2048, 128, torch.bfloat16)
    for dst, src in ((q, q2), (k, k2), (v, v2), (grad, grad2)):
        dst.copy_(src)
    graph.replay()
    want = run_both(q2, k2, v2, grad2, TL, 200, 4)
    for n, t in (("out", out), ("lse", lse), ("dq", dq), ("dk", dk), ("dv", dv)):
        assert torch.equal(want[n], t), n


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Sq,Sk,window,sinks", [(1, 1, 1, 0), (1, 129, 128, 0), (1, 1000, 100, 3), (1, 5000, 5001, 0), (2, 777, 1, 1), (5, 640, 130, 200)])
def test_few_rows_against_a_longer_key_sequence(Sq, Sk, window, sinks, D, dtype):
    q, k, v, grad = inputs(12, 2, 4, 2, Sq, Sk, D, dtype)
    got = run_both(q, k, v, grad, BR, window, sinks)
    for name, (want, bound) in reference(q, k, v, grad, BR, window, sinks).items():
        check(name, got[name], want, bound)
