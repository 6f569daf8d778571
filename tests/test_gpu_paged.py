"""The paged key/value cache: append, attention over the pages, reading back (``-m gpu``), against the formulas in 64 bits.

Bounds of the attention, element by element (u half a step of the type, s the relative error of a probability, A = P |V|):
  16 bits: P is rounded to the type before it multiplies V, out after        u A + u |out| + 3 s A
  4 bits:  P vs is rounded to the type before it multiplies c - 8, and P is before it multiplies vs and vm, whose sums make that
           of P (vm + 8 vs).  With F = sum(P vs |c - 8|), G = sum(P |vm + 8 vs|):    u (F + G) + u |out| + 3 s (F + G)
           scores: sums of q ks c and of q km
           The sums of P vm and of 8 P vs are taken in 32 bits and then added, so a step of theirs counts by what each of them is
           and not by their sum: 2^-23 (keys + 4) sum(P (|vm| + 8 vs))
All but u |out| times 1 + u, since it is the sum with these errors that is rounded to the type.
A float16 has no step below 2^-24: t = 2^-25 more for each rounding to it.  Appending and reading back round once, in a given
order: their results are equal to the formula in fp32, bit for bit.
"""

import random

import pytest
import torch

from torch_mojo_backend_b200 import _lib, raw

pytestmark = pytest.mark.gpu


def k_element(D):
    """Element that code i of a key's row stands for."""
    return [32 * G + 8 * t + j for t in range(4) for G in range(D // 32) for j in range(8)]


def v_element(D):
    return [32 * G + 4 * g + j for g in range(8) for G in range(D // 32) for j in range(4)]


def quantised(x):
    """(codes, scale, minimum) of x (..., D), codes by element."""
    g = x.float().unflatten(-1, (-1, 32))
    low = g.amin(-1)
    scale = ((g.amax(-1) - low) / 15).to(x.dtype)
    codes = ((g - low[..., None]) / scale.float()[..., None]).round().clamp(0, 15)
    return torch.where(scale[..., None] == 0, 0, codes).flatten(-2), scale, low.to(x.dtype)


def packed(codes, element):
    c = codes[..., element].to(torch.uint8)
    return c[..., 0::2] | c[..., 1::2] << 4


def unpacked(codes, element):
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).float()
    out = torch.empty_like(c)
    out[..., element] = c
    return out


class Pool:
    """A pool of pages whose unused places are NaN (codes of NaN scales), and sequences in it."""

    def __init__(self, seed, lengths, Hkv, D, page, dtype, bits, std=1.0, extra_width=1):
        self.g = torch.Generator(device="cuda").manual_seed(seed)
        self.D, self.dtype, self.bits, self.page, self.Hkv = D, dtype, bits, page, Hkv
        counts = [-(-n // page) for n in lengths]
        order = list(range(sum(counts) + 2))
        random.Random(seed).shuffle(order)
        table = torch.full((len(lengths), max(counts + [1]) + extra_width), -7, dtype=torch.int32)
        at = 0
        for b, n in enumerate(counts):
            table[b, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
            at += n
        self.table, self.lengths = table.cuda(), torch.tensor(lengths, dtype=torch.int32, device="cuda")
        self.cache = raw.PagedKV.empty(len(order), Hkv, page, D, dtype=dtype, bits=bits)
        for t in self.cache:
            if t is not None:
                t.fill_(float("nan")) if t.is_floating_point() else t.fill_(0xA5)
        # what a sequence holds, (Hkv, n, D) of the type; the values behind it in 64 bits
        self.k = [self.draw(Hkv, n, D, std=std) for n in lengths]
        self.v = [self.draw(Hkv, n, D, std=std) for n in lengths]
        for b, n in enumerate(lengths):
            self.put(b, 0, self.k[b], self.v[b])

    def draw(self, *shape, std=1.0):
        return (torch.randn(shape, generator=self.g, device="cuda") * std).to(self.dtype)

    def place(self, b, start, n):
        pos = torch.arange(start, start + n, device="cuda")
        return self.table[b, pos // self.page].long(), pos % self.page

    def put(self, b, start, k, v):
        page, slot = self.place(b, start, k.shape[1])
        rows = [x.transpose(0, 1) for x in (k, v)]
        if self.bits == 16:
            for pages, r in zip(self.cache, rows):
                pages[page, :, slot] = r
            return
        for pages, scales, r, element in ((self.cache.k, self.cache.k_scales, rows[0], k_element(self.D)),
                                          (self.cache.v, self.cache.v_scales, rows[1], v_element(self.D))):
            codes, scale, low = quantised(r)
            pages[page, :, slot] = packed(codes, element)
            scales[page, :, slot] = torch.stack([scale, low], -1)

    def held(self, b, n=None):
        """k, v of sequence b as the cache holds them, (Hkv, n, D) in 32 bits, and with 4 bits the sizes of the two parts that the
        kernel takes them in: scale * code and minimum (of a value: code - 8 and the minimum + 8 scales, then |minimum| + 8 scales)."""
        n = self.k[b].shape[1] if n is None else n
        page, slot = self.place(b, 0, n)
        got = []
        for pages, scales, element in ((self.cache.k, self.cache.k_scales, k_element(self.D)),
                                       (self.cache.v, self.cache.v_scales, v_element(self.D))):
            rows = pages[page, :, slot].transpose(0, 1)
            if self.bits == 16:
                got.append((rows.float(), rows.float().abs(), None, None))
                continue
            s = scales[page, :, slot].transpose(0, 1).float()
            codes = unpacked(rows, element).unflatten(-1, (-1, 32))
            middle = 0 if pages is self.cache.k else 8
            parts = (codes * s[..., :1] + s[..., 1:], (codes - middle).abs() * s[..., :1], (s[..., 1:] + middle * s[..., :1]).abs().expand_as(codes),
                     (s[..., 1:].abs() + middle * s[..., :1]).expand_as(codes))
            got.append(tuple(x.flatten(-2) for x in parts))
        return got


def expected(pool, q, b, n, window, sinks):
    """(out, its bound), (lse, its bound) of the n new tokens of sequence b; q (Hq, S, D)."""
    (k, _, _, _), (v, scaled, low, apart) = pool.held(b)
    Hq, length, D = q.shape[0], k.shape[1], q.shape[2]
    u = torch.finfo(q.dtype).eps / 2
    t = 2.0 ** -25 if q.dtype == torch.float16 else 0.0
    group = Hq // pool.Hkv
    k, v, scaled = (x.double().repeat_interleave(group, 0) for x in (k, v, scaled))
    q = q[:, :n].double()
    pos = torch.arange(length - n, length, device="cuda")[:, None]
    key = torch.arange(length, device="cuda")[None]
    seen = key <= pos
    if window:
        seen &= (key > pos - window) | (key < sinks)
    s = (q @ k.mT * D ** -0.5).masked_fill(~seen, -torch.inf)
    lse = torch.logsumexp(s, -1)
    p = torch.exp(s - lse.clamp(min=-1e300)[..., None])
    out = p @ v
    a = p @ v.abs()
    # an fp32 sum of D products, each at most 2^-23 off
    size = float((q.abs() @ k.abs().mT).max()) * D ** -0.5
    if pool.bits == 4:
        (_, ks, km, _), _ = pool.held(b)
        size = float((q.abs() @ (ks + km).double().repeat_interleave(group, 0).mT).max()) * D ** -0.5
    e = size * D * 2 ** -23 + 2.0 ** -20 + int(seen.sum(1).max()) * 2.0 ** -24
    if pool.bits == 16:
        bound = (1 + u) * ((u + 3 * e) * a + t * (seen.double() @ v.abs())) + u * out.abs() + t
    else:
        low = low.double().repeat_interleave(group, 0)
        bound = (u + 3 * e) * (p @ scaled + p @ low) + t * 8 * seen.sum(1, keepdim=True) + t * (seen.double() @ low)
        bound += 2.0 ** -23 * (seen.sum(1, keepdim=True) + 4) * (p @ apart.double().repeat_interleave(group, 0))
        bound = (1 + u) * bound + u * out.abs() + t
    return (out, bound), (lse, e + 2.0 ** -22 * lse.abs())


def check(name, got, want, bound):
    got = got.double()
    assert torch.isfinite(got).all(), name
    over = ((got - want).abs() - bound - 1e-30).max().item()
    assert over <= 0, f"{name}: {over:.3e} over its bound; largest error {(got - want).abs().max().item():.3e}"


ATTEND = [
    # lengths, new tokens (None: all of S), S, Hq, Hkv, D, page, window, sinks
    ([1], None, 1, 1, 1, 64, 16, 0, 0),
    ([1, 2, 15, 16, 17], None, 1, 8, 2, 128, 16, 0, 0),
    ([300, 0, 33, 1000], None, 1, 8, 8, 64, 16, 0, 0),            # an idle place in the batch
    ([5000, 700], None, 1, 32, 8, 128, 64, 0, 0),
    ([2000], None, 1, 4, 1, 128, 4096, 0, 0),                     # one page, far from full
    ([900, 901, 64], None, 1, 12, 1, 64, 32, 0, 0),               # two tiles of rows
    ([900, 70], None, 3, 40, 2, 128, 16, 0, 0),                   # four tiles of rows
    ([513, 100, 7], [4, 1, 2], 4, 8, 2, 128, 16, 0, 0),           # padded rows
    ([40, 3, 0], [37, 3, 0], 37, 4, 2, 64, 16, 0, 0),             # a prompt; nothing at all
    ([1500], None, 1300, 8, 2, 64, 64, 0, 0),                     # a long prompt: 325 tiles of rows
    ([1000, 30, 1], None, 1, 8, 2, 128, 16, 100, 4),              # window and sinks
    ([1000, 130, 129, 128], None, 1, 4, 4, 64, 32, 128, 0),
    ([700, 20, 40], [3, 2, 3], 3, 8, 2, 128, 16, 17, 5),          # a gap between sinks and window inside a step
    ([700, 300], None, 2, 4, 4, 64, 16, 1, 1),
    ([700, 300], None, 1, 4, 2, 128, 16, 250, 60),
    ([3000], None, 5, 2, 2, 128, 64, 40, 900),                    # more sinks than window
    ([2, 5], None, 4, 4, 4, 64, 16, 3, 1),                        # fewer keys than new tokens: the first ones see nothing
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("lengths,new,S,Hq,Hkv,D,page,window,sinks", ATTEND)
def test_attention_against_the_formula(lengths, new, S, Hq, Hkv, D, page, window, sinks, bits, dtype):
    pool = Pool(1, lengths, Hkv, D, page, dtype, bits)
    q = pool.draw(len(lengths), Hq, S, D)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    n = torch.tensor(new, dtype=torch.int32, device="cuda") if new else None
    out, lse = torch.full_like(q, 3.0), torch.full(q.shape[:3], 5.0, device="cuda")
    raw.paged_attention(q, pool.cache, pool.table, pool.lengths, new_lengths=n, window=window, sinks=sinks, out=out, lse=lse,
                        status=status)
    torch.cuda.synchronize()
    assert int(status) == 0
    for b, length in enumerate(lengths):
        t = new[b] if new else S
        assert (out[b, :, t:] == 3.0).all() and (lse[b, :, t:] == 5.0).all(), "rows behind the new tokens are left as they are"
        none = max(0, t - length)   # new tokens that are not there
        assert (out[b, :, :none] == 0).all() and torch.isneginf(lse[b, :, :none]).all()
        if t > none:
            (o, ob), (l, lb) = expected(pool, q[b, :, none:], b, t - none, window, sinks)
            check("out", out[b, :, none:t], o, ob)
            check("lse", lse[b, :, none:t], l, lb)


@pytest.mark.parametrize("bits", [16, 4])
def test_places_that_no_row_sees_are_not_read(bits):
    """Pages ahead of a window belong to others, and what a page holds behind the last key is not set: NaN in both."""
    pool = Pool(2, [700, 530], 2, 128, 32, torch.bfloat16, bits)
    q = pool.draw(2, 8, 2, 128)
    want = raw.paged_attention(q, pool.cache, pool.table, pool.lengths, window=90, sinks=3)
    for b, n in enumerate((700, 530)):
        page, slot = pool.place(b, 3, n - 2 - 90 + 1 - 3)   # keys 3 .. behind the first new token's window
        for t in (pool.cache[:2] if bits == 16 else pool.cache[2:]):
            t[page, :, slot] = float("nan")
    table = pool.table.clone()
    table[0, 1:(700 - 91) // 32] = -1     # and the pages themselves may be gone
    got = raw.paged_attention(q, pool.cache, table, pool.lengths, window=90, sinks=3)
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])


@pytest.mark.parametrize("bits", [16, 4])
def test_large_scores_that_keep_rising_move_the_maximum(bits):
    """Scores from -90 to 90, later keys higher: the running maximum has to move many times."""
    pool = Pool(3, [1500], 1, 64, 16, torch.float16, bits)
    ramp = torch.linspace(-11, 11, 1500, device="cuda").half()
    pool.k[0] = (pool.k[0] * 0.05 + ramp[None, :, None]).half()
    pool.put(0, 0, pool.k[0], pool.v[0])
    q = (pool.draw(1, 4, 1, 64) * 0.05 + 1.0).half()
    out, lse = raw.paged_attention(q, pool.cache, pool.table, pool.lengths)
    (o, ob), (l, lb) = expected(pool, q[0], 0, 1, 0, 0)
    check("out", out[0], o, ob)
    check("lse", lse[0], l, lb)


def rotated(x, cos, sin, interleaved):
    """x (..., D) in fp32, every operation rounded, then to x's type."""
    R, y = 2 * cos.shape[-1], x.float()
    a, b = (y[..., 0:R:2], y[..., 1:R:2]) if interleaved else (y[..., :R // 2], y[..., R // 2:R])
    a, b = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
    return torch.cat([turned, y[..., R:]], -1).to(x.dtype)


APPEND = [
    # lengths with the new tokens, new tokens, S, Hq, Hkv, D, page, R, interleaved
    ([1], None, 1, 2, 1, 64, 16, 64, False),
    ([17, 1, 0, 40], [1, 1, 0, 1], 1, 4, 4, 128, 16, 128, False),
    ([50, 16, 33], [50, 3, 1], 50, 6, 2, 128, 16, 64, True),
    ([50, 16, 33], [50, 3, 1], 50, 6, 2, 64, 32, 32, False),
    ([100, 90], None, 77, 3, 3, 64, 64, 16, True),
    ([5, 9], None, 7, 0, 2, 128, 16, 0, False),     # nothing turns, no queries; two tokens that are not there
    ([300], None, 200, 1, 1, 128, 128, 128, True),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("lengths,new,S,Hq,Hkv,D,page,R,interleaved", APPEND)
def test_append_and_gather_against_the_formula(lengths, new, S, Hq, Hkv, D, page, R, interleaved, bits, dtype):
    pool = Pool(4, lengths, Hkv, D, page, dtype, bits)
    B = len(lengths)
    fused = pool.draw(B, S, (Hq + 2 * Hkv) * D)
    q, k, v = (t.unflatten(2, (-1, D)).transpose(1, 2) for t in fused.split([Hq * D, Hkv * D, Hkv * D], 2))
    v[:, :, 0, :32] = 1.5        # a group of equal elements: its scale is zero
    angle = torch.arange(max(lengths), device="cuda", dtype=torch.float64)[:, None] * 100.0 ** -torch.arange(R // 2, device="cuda")
    cos, sin = angle.cos().float(), angle.sin().float()
    before = [t.clone() if t is not None else None for t in pool.cache]
    q_out = torch.full((B, Hq, S, D), 3.0, dtype=dtype, device="cuda") if Hq else None
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    n = torch.tensor(new, dtype=torch.int32, device="cuda") if new else None
    raw.paged_append(k, v, pool.cache, pool.table, pool.lengths, new_lengths=n, rotary=(cos, sin) if R else None,
                     interleaved=interleaved, q=q if Hq else None, q_out=q_out, status=status)
    after = [t.clone() if t is not None else None for t in pool.cache]
    for t, b in zip(pool.cache, before):
        if t is not None:
            t.copy_(b)
    for b, length in enumerate(lengths):
        t = new[b] if new else S
        none = max(0, t - length)
        if t > none:
            pos = torch.arange(length - t + none, length, device="cuda")
            turn = (lambda x: rotated(x, cos[pos], sin[pos], interleaved)) if R else (lambda x: x)
            pool.put(b, length - t + none, turn(k[b, :, none:t]), v[b, :, none:t])
            if Hq:
                assert torch.equal(q_out[b, :, none:t], turn(q[b, :, none:t]))
        if Hq:
            assert (q_out[b, :, t:] == 3.0).all() and (q_out[b, :, :none] == 3.0).all()
    for got, want in zip(after, pool.cache):   # everywhere, the places that nothing is appended to among them
        if got is not None:
            same = got.view(torch.uint8) == want.view(torch.uint8) if got.dtype != torch.uint8 else got == want
            both = same if got.dtype == torch.uint8 else same.unflatten(-1, (-1, 2)).all(-1) | (got == want)   # (-0 is 0)
            assert both.all()
    longest = max(lengths) + 5
    gk, gv = raw.paged_gather(pool.cache, pool.table, pool.lengths, longest, status=status)
    torch.cuda.synchronize()
    assert int(status) == 0
    for b, length in enumerate(lengths):
        assert (gk[b, :, length:] == 0).all() and (gv[b, :, length:] == 0).all()
        (wk, *_), (wv, *_) = pool.held(b, length)
        assert torch.equal(gk[b, :, :length], wk.to(dtype)) and torch.equal(gv[b, :, :length], wv.to(dtype))


def test_groups_that_are_not_finite_read_nan():
    pool = Pool(5, [20], 1, 64, 16, torch.bfloat16, 4)
    k, v = pool.draw(1, 1, 2, 64), pool.draw(1, 1, 2, 64)
    k[0, 0, 0, 3], k[0, 0, 1, 40], v[0, 0, 1, 5] = float("nan"), float("inf"), -float("inf")
    raw.paged_append(k, v, pool.cache, pool.table, pool.lengths)
    gk, gv = raw.paged_gather(pool.cache, pool.table, pool.lengths, 20)
    assert torch.isnan(gk[0, 0, 18, :32]).all() and torch.isfinite(gk[0, 0, 18, 32:]).all()
    assert torch.isnan(gk[0, 0, 19, 32:]).all() and torch.isfinite(gk[0, 0, 19, :32]).all()
    assert torch.isnan(gv[0, 0, 19, :32]).all() and torch.isfinite(gv[0, 0, 18]).all()


def test_queries_in_place():
    pool = Pool(6, [30, 8], 2, 128, 16, torch.float16, 16)
    q, k, v = pool.draw(2, 4, 3, 128), pool.draw(2, 2, 3, 128), pool.draw(2, 2, 3, 128)
    angle = torch.rand(40, 64, device="cuda")
    rotary = (angle.cos(), angle.sin())
    want = raw.paged_append(k, v, pool.cache, pool.table, pool.lengths, rotary=rotary, q=q)
    got = raw.paged_append(k, v, pool.cache, pool.table, pool.lengths, rotary=rotary, q=q, q_out=q)
    assert got is q and torch.equal(q, want)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("what", ["page", "negative page", "length", "negative length", "new", "position"])
def test_indexes_out_of_range_are_reported_and_never_used(what, bits):
    """The kernels check what comes from device memory before they use it: the sequence's results are NaN, its neighbour's are not."""
    pool = Pool(7, [100, 90], 2, 64, 16, torch.bfloat16, bits)
    q, k, v = pool.draw(2, 4, 2, 64), pool.draw(2, 2, 2, 64), pool.draw(2, 2, 2, 64)
    want, _ = raw.paged_attention(q, pool.cache, pool.table, pool.lengths)
    table, lengths, new = pool.table.clone(), pool.lengths.clone(), torch.full_like(pool.lengths, 2)
    angle = torch.rand(95 if what == "position" else 200, 32, device="cuda")
    if what == "page":
        table[0, 6] = pool.cache.k.shape[0]
    elif what == "negative page":
        table[0, 6] = -1
    elif what == "length":
        lengths[0] = table.shape[1] * 16 + 1
    elif what == "negative length":
        lengths[0] = -3
    elif what == "new":
        new[0] = 3
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    report = lambda: _lib.status_to_error(int(status)) == _lib.ERR_BAD_INDEX and not status.zero_().any()
    if what != "position":
        out, lse = raw.paged_attention(q, pool.cache, table, lengths, new_lengths=new, status=status)
        assert report() and torch.isnan(out[0]).all() and torch.isnan(lse[0]).all() and torch.equal(out[1], want[1])
    if what not in ("position", "new"):
        gk, gv = raw.paged_gather(pool.cache, table, lengths, 100, status=status)
        bad = slice(96, 100) if "page" in what else slice(0, 100)
        assert report() and torch.isnan(gk[0, :, bad]).all() and torch.isnan(gv[0, :, bad]).all() and torch.isfinite(gk[1]).all()
    before = [t.clone() if t is not None else None for t in pool.cache]
    raw.paged_append(k, v, pool.cache, table, lengths, new_lengths=new, rotary=(angle.cos(), angle.sin()), status=status)
    assert report()
    pages = {int(p) for p in pool.table[0, :7]}
    for t, b in zip(pool.cache, before):
        if t is not None:
            for p in pages:   # nothing of the sequence was written
                assert torch.equal(t[p].view(torch.uint8), b[p].view(torch.uint8))
    assert not torch.equal(pool.cache.k, before[0])


TEAMS = [
    # lengths, S, Hq, Hkv, D, page, window, sinks
    ([9000], 1, 8, 1, 128, 16, 0, 0),
    ([1], 1, 8, 1, 128, 64, 0, 0),                        # far fewer keys than the table has room for: teams without any
    ([20000, 0, 33], 1, 8, 1, 64, 64, 0, 0),
    ([12345, 17], 3, 12, 2, 64, 32, 0, 0),                # 18 rows: two tiles
    ([9000, 12], 1, 32, 4, 128, 64, 0, 0),
    ([70000], 2, 4, 1, 64, 128, 65536, 5),                # a window of as many keys
    ([9000, 8500], 4, 16, 2, 128, 16, 9000, 4),           # (sixteen units of 9000 keys: one cluster each)
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("lengths,S,Hq,Hkv,D,page,window,sinks", TEAMS)
def test_several_clusters_share_the_keys_of_a_head(lengths, S, Hq, Hkv, D, page, window, sinks, bits, dtype):
    pool = Pool(11, lengths, Hkv, D, page, dtype, bits, extra_width=131072 // page)
    q = pool.draw(len(lengths), Hq, S, D)
    new = torch.tensor([min(S, n) for n in lengths], dtype=torch.int32, device="cuda")
    before = _lib.launch_count()
    call = lambda **how: raw.paged_attention(q, pool.cache, pool.table, pool.lengths, new_lengths=new, window=window,   # noqa: E731
                                             sinks=sinks, **how)
    out, lse = call()
    launches = 1 if window == 9000 else 2
    assert _lib.launch_count() == before + launches
    one, _ = call(workspace=torch.empty(0, dtype=torch.uint8, device="cuda"))
    assert _lib.launch_count() == before + launches + 1
    need = _lib.paged_attention_workspace_bytes(len(lengths), Hq, Hkv, S, D, 131072)
    dirty = torch.full((need + 64,), 255, dtype=torch.uint8, device="cuda")   # NaN
    again, again_lse = call(workspace=dirty[:need])
    assert torch.equal(again, out) and torch.equal(again_lse, lse) and (dirty[need:] == 255).all()
    call(workspace=dirty[:need // 3])                                         # room for fewer
    assert (dirty[need:] == 255).all()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        later, _ = call()
    graph.replay()
    assert torch.equal(later, out)
    for b, length in enumerate(lengths):
        t = int(new[b])
        assert (out[b, :, t:] == 0).all() and torch.isneginf(lse[b, :, t:]).all()
        if t:
            (o, ob), (l, lb) = expected(pool, q[b], b, t, window, sinks)
            check("out", out[b, :, :t], o, ob)
            check("one cluster", one[b, :, :t], o, ob)
            check("lse", lse[b, :, :t], l, lb)
    table, status = pool.table.clone(), torch.zeros(1, dtype=torch.int32, device="cuda")
    if lengths[0]:
        table[0, 0 if not window or sinks else (lengths[0] - 1) // page] = -1   # a page that some team reads
        bad, bad_lse = raw.paged_attention(q, pool.cache, table, pool.lengths, new_lengths=new, window=window, sinks=sinks, status=status)
        t = int(new[0])
        assert _lib.status_to_error(int(status)) == _lib.ERR_BAD_INDEX
        assert torch.isnan(bad[0, :, :t]).all() and torch.isnan(bad_lse[0, :, :t]).all()
        assert torch.equal(bad[1:], out[1:])


@pytest.mark.parametrize("bits", [16, 4])
def test_a_serving_run(bits):
    """Prompts appended, decoded with sinks and a window token by token in one captured graph whose device tensors change, and
    read back: every step's result is that of the formula over what the cache holds."""
    Hq, Hkv, D, page, dtype = 8, 2, 128, 16, torch.bfloat16
    pool = Pool(8, [0, 0, 0], Hkv, D, page, dtype, bits, extra_width=8)
    pool.table.copy_(torch.arange(27, device="cuda").reshape(3, 9).flip(1))
    pool.cache = raw.PagedKV.empty(27, Hkv, page, D, dtype=dtype, bits=bits)
    prompt = torch.tensor([60, 33, 0], dtype=torch.int32, device="cuda")
    angle = torch.arange(160, device="cuda", dtype=torch.float64)[:, None] * 1000.0 ** -(torch.arange(64, device="cuda") / 64)
    rotary = (angle.cos().float(), angle.sin().float())
    q, k, v = pool.draw(3, Hq, 60, D), pool.draw(3, Hkv, 60, D), pool.draw(3, Hkv, 60, D)
    turned = raw.paged_append(k, v, pool.cache, pool.table, prompt, new_lengths=prompt, rotary=rotary, q=q)
    # the prompt's own attention: dense operators over what was read back
    gk, gv = raw.paged_gather(pool.cache, pool.table, prompt, 60)
    dense, _ = raw.window_fwd(turned, gk, gv, window=40, sinks=2)
    paged, _ = raw.paged_attention(turned, pool.cache, pool.table, prompt, new_lengths=prompt, window=40, sinks=2)
    u = torch.finfo(dtype).eps / 2
    for b, n in ((0, 60), (1, 33)):   # (the read-back rounds a 4-bit value once more; values are below 5, their sum of weights is 1)
        assert (dense[b, :, :n].float() - paged[b, :, :n].float()).abs().max() < 8 * u * 5
    # decoding: sequence 2 joins late
    lengths, new = prompt.clone(), torch.zeros_like(prompt)
    q1, k1, v1 = (torch.empty(3, h, 1, D, dtype=dtype, device="cuda") for h in (Hq, Hkv, Hkv))
    out, lse = torch.zeros(3, Hq, 1, D, dtype=dtype, device="cuda"), torch.zeros(3, Hq, 1, device="cuda")
    turned = torch.zeros_like(q1)

    def step():
        raw.paged_append(k1, v1, pool.cache, pool.table, lengths, new_lengths=new, rotary=rotary, q=q1, q_out=turned)
        raw.paged_attention(turned, pool.cache, pool.table, lengths, new_lengths=new, window=40, sinks=2, out=out, lse=lse)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(20):
        new.copy_(torch.tensor([1, 1, 1 if i >= 3 else 0], dtype=torch.int32))
        lengths.add_(new)
        for t in (q1, k1, v1):
            t.copy_(pool.draw(*t.shape))
        graph.replay()
        for b in range(3 if i >= 3 else 2):
            pool.k[b] = torch.empty(Hkv, int(lengths[b]), D)   # (its length is what counts)
            (o, ob), (l, lb) = expected(pool, turned[b], b, 1, 40, 2)
            check("out", out[b], o, ob)
            check("lse", lse[b], l, lb)


def test_an_ordered_side_stream():
    pool = Pool(9, [600, 300], 2, 128, 16, torch.bfloat16, 4)
    q = pool.draw(2, 8, 1, 128)
    want, _ = raw.paged_attention(q, pool.cache, pool.table, pool.lengths)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, _ = raw.paged_attention(q, pool.cache, pool.table, pool.lengths)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(want, got)


def test_pages_beyond_32_bits():
    """A pool of more than 2^32 elements: the last pages are reached."""
    pages, D, page = 17000, 128, 256
    k = torch.zeros(pages, 8, page, D, dtype=torch.bfloat16, device="cuda")   # 4.46e9 elements, 8.9 GB
    cache = raw.PagedKV(k, k)
    table = torch.tensor([[pages - 1, 0, pages - 2]], dtype=torch.int32, device="cuda")
    lengths = torch.tensor([700], dtype=torch.int32, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(1, 8, 700, D, generator=g, device="cuda").bfloat16()
    raw.paged_append(x, x, cache, table, lengths)
    gk, _ = raw.paged_gather(cache, table, lengths, 700)
    assert torch.equal(gk, x)
    q = torch.randn(1, 8, 1, D, generator=g, device="cuda").bfloat16()
    out, _ = raw.paged_attention(q, cache, table, lengths)
    s = torch.softmax(q.double() @ x.double().mT * D ** -0.5, -1)
    a = s @ x.double().abs()
    assert ((out.double() - s @ x.double()).abs() <= 2 ** -8 * (a + 2 * out.double().abs()) + 2 ** -12 * a).all()


@pytest.mark.parametrize("bits", [16, 4])
def test_clusters_of_every_size_without_a_workspace(bits):
    """A KV head has up to 16 blocks, by the calls' model, with a workspace or without; each size that it takes is right."""
    calls = {}
    for keys in [*range(64, 8192, 64), 16384, 32768, 65536]:
        peers, teams, warps = _lib.paged_attention_shares(1, 4, 1, 1, 128, _lib.BF16, bits, keys)
        assert teams == 1
        calls.setdefault((peers, warps), keys)
    assert {8, 16} <= {peers for peers, _ in calls} and max(calls)[0] == 16
    need = _lib.paged_attention_workspace_bytes(1, 4, 1, 1, 128, 131072)
    assert _lib.paged_attention_shares(1, 4, 1, 1, 128, _lib.BF16, bits, 131072, need)[1] > 1
    none = torch.empty(0, dtype=torch.uint8, device="cuda")
    for keys in calls.values():
        pool = Pool(12, [keys], 1, 128, 64, torch.bfloat16, bits)
        q = pool.draw(1, 4, 1, 128)
        out, lse = raw.paged_attention(q, pool.cache, pool.table, pool.lengths, longest=keys, workspace=none)
        (o, ob), (l, lb) = expected(pool, q[0], 0, 1, 0, 0)
        check("out", out[0], o, ob)
        check("lse", lse[0], l, lb)


@pytest.mark.parametrize("D,Hq", [(64, 3), (128, 8)])
@pytest.mark.parametrize("padded", [True, False])
def test_a_new_tensor_of_queries_is_whole(padded, D, Hq):
    """Rows that no new token has are zero in the tensor that the call makes, and NaN where an index is out of range."""
    lengths = [2, 0, 30, 40, 999, 20]        # fewer tokens than S; an idle place; all there; behind the angles; no such length
    S, new = 5, [4, 0, 5, 5, 5, 2]
    pool = Pool(13, [2, 0, 30, 40, 45, 20], 2, D, 16, torch.bfloat16, 16)
    pool.lengths.copy_(torch.tensor(lengths))
    q, k, v = pool.draw(6, Hq, S, D), pool.draw(6, 2, S, D), pool.draw(6, 2, S, D)
    angle = torch.rand(38, D // 2, device="cuda")
    rotary = angle.cos(), angle.sin()
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    n = torch.tensor(new, dtype=torch.int32, device="cuda") if padded else None
    held = torch.full_like(q, 3.0)
    raw.paged_append(k, v, pool.cache, pool.table, pool.lengths, new_lengths=n, rotary=rotary, q=q, q_out=held)
    torch.full_like(q, 7.0)                  # (what its memory held)
    out = raw.paged_append(k, v, pool.cache, pool.table, pool.lengths, new_lengths=n, rotary=rotary, q=q, status=status)
    assert _lib.status_to_error(int(status)) == _lib.ERR_BAD_INDEX
    for b in range(6):
        t = new[b] if padded else S
        for s in range(S):
            pos = lengths[b] - t + s
            row, given = out[b, :, s], held[b, :, s]
            if b == 4 or (s < t and pos >= 38):
                assert torch.isnan(row).all() and (given == 3.0).all()
            elif s >= t or pos < 0:
                assert (row == 0).all() and (given == 3.0).all()
            else:
                want = rotated(q[b, :, s], rotary[0][pos], rotary[1][pos], False)
                assert torch.equal(row, want) and torch.equal(given, want)
