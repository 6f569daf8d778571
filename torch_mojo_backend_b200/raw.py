"""Calls into the C ABI for plain ``torch.cuda`` tensors.

The `mojo` device layer (``flash_ops.py``) sits beside this; tests and the benchmark also use
it directly, the way the reference's GPU tests call the bridge with hand-built buffers
(tests/test_eager_kernels.py:9754-9765).  Nothing here computes attention: every function
validates metadata, allocates outputs with torch's CUDA allocator and enqueues library
kernels on torch's current stream.
"""

from __future__ import annotations

import math
from typing import NamedTuple

import torch

from . import _lib

_DTYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}


def dtype_code(dtype: torch.dtype) -> int:
    try:
        return _DTYPES[dtype]
    except KeyError:
        raise NotImplementedError(f"b200fa supports float32, bfloat16 and float16, got {dtype}") from None


def t4(t: torch.Tensor) -> _lib.Tensor4:
    return _lib.Tensor4.make(t.data_ptr(), tuple(t.shape), tuple(t.stride()))


def _t4b(t: torch.Tensor) -> bytes:
    """`t4` as the packed bytes that the newer entry points take (a third of the time)."""
    if t.dim() != 4:
        raise ValueError("b200fa tensors are 4-D (batch, heads, seq, head_dim)")
    return _lib.pack_tensor4(t.data_ptr(), *t.shape, *t.stride())


def _stream_and_device(t: torch.Tensor) -> tuple[int, int]:
    dev = t.device.index if t.device.index is not None else torch.cuda.current_device()
    return torch._C._cuda_getCurrentRawStream(dev), dev


def default_scale(head_dim: int) -> float:
    return 1.0 / math.sqrt(head_dim)


def flash_fwd(q, k, v, *, causal, scale: float | None = None, out=None, lse=None, status=None,
              simt: bool = False, dropout=None, whole_heads: int = 0):
    """out, lse = attention forward on CUDA tensors shaped (B, H, S, D).

    ``out`` defaults to a new contiguous (B, Hq, Sq, D) tensor; pass a pre-allocated (possibly
    strided) tensor to choose the storage layout.  ``lse`` is fp32 (B, Hq, Sq).  ``causal`` is a
    bool (True: diagonal from the top-left corner) or one of ``_lib.CAUSAL_*``; ``dropout`` is
    None or ``(p, philox_seed, philox_offset)``; ``simt`` takes the exact-fp32 FMA kernels, which an fp32
    forward at head dimension 128 should whose results go into ``flash_bwd`` (that one is FMA arithmetic there, and
    its gradients lean on both having the same errors in the scores).  A call that computes a piece of a larger problem
    (some batch entries or whole groups of heads, one rank's shard) has the bits of one call over the
    whole if it is told the whole's batch * query heads in ``whole_heads``.
    """
    if q.device.type != "cuda":
        raise RuntimeError("b200fa kernels need CUDA memory; there is no CPU implementation")
    B, Hq, Sq, D = q.shape
    if scale is None:
        scale = default_scale(D)
    if out is None:
        out = torch.empty((B, Hq, Sq, D), dtype=q.dtype, device=q.device)
    if lse is None:
        lse = torch.empty((B, Hq, Sq), dtype=torch.float32, device=q.device)
    stream, dev = _stream_and_device(q)
    rc = _lib.fwd(t4(q), t4(k), t4(v), t4(out), lse.data_ptr(), dtype_code(q.dtype), causal, float(scale),
                  stream, dev, status.data_ptr() if status is not None else 0, simt=simt, dropout=dropout,
                  whole_heads=whole_heads)
    if rc != _lib.OK:
        raise _lib.B200FAError(rc, "b200fa_fwd")
    return out, lse


def flash_fwd_splitkv(q, k, v, *, causal, scale: float | None = None, out=None, lse=None, workspace=None,
                      whole_heads: int = 0):
    """out, lse = the split-KV (decode) forward on CUDA tensors shaped (B, H, S, D); needs
    ``(Hq / Hkv) * Sq <= 16``.  ``whole_heads`` as for ``flash_fwd``."""
    if q.device.type != "cuda":
        raise RuntimeError("b200fa kernels need CUDA memory; there is no CPU implementation")
    B, Hq, Sq, D = q.shape
    Hkv, Sk = k.shape[1], k.shape[2]
    if scale is None:
        scale = default_scale(D)
    if out is None:
        out = torch.empty((B, Hq, Sq, D), dtype=q.dtype, device=q.device)
    if lse is None:
        lse = torch.empty((B, Hq, Sq), dtype=torch.float32, device=q.device)
    need = _lib.fwd_splitkv_workspace_bytes(B, Hq, Hkv, Sq, Sk, D, whole_heads)
    if workspace is None:
        workspace = torch.empty((need,), dtype=torch.uint8, device=q.device)
    stream, dev = _stream_and_device(q)
    rc = _lib.fwd_splitkv(t4(q), t4(k), t4(v), t4(out), lse.data_ptr(), workspace.data_ptr(),
                          workspace.numel() * workspace.element_size(), dtype_code(q.dtype), causal, float(scale),
                          stream, dev, whole_heads=whole_heads)
    if rc != _lib.OK:
        raise _lib.B200FAError(rc, "b200fa_fwd_splitkv")
    return out, lse


def flash_bwd(dout, q, k, v, out, lse, *, causal, scale: float | None = None, dq=None, dk=None,
              dv=None, workspace=None, status=None, simt: bool = False, parts: int = 7, dropout=None):
    """dq, dk, dv = attention backward on CUDA tensors shaped (B, H, S, D)."""
    if q.device.type != "cuda":
        raise RuntimeError("b200fa kernels need CUDA memory; there is no CPU implementation")
    B, Hq, S, D = q.shape
    Hkv = k.shape[1]
    if scale is None:
        scale = default_scale(D)
    if dq is None:
        dq = torch.empty((B, Hq, S, D), dtype=q.dtype, device=q.device)
    if dk is None:
        dk = torch.empty(tuple(k.shape), dtype=q.dtype, device=q.device)
    if dv is None:
        dv = torch.empty(tuple(v.shape), dtype=q.dtype, device=q.device)
    code = dtype_code(q.dtype)
    need = _lib.bwd_workspace_bytes(B, Hq, Hkv, S, D, code)
    if workspace is None:
        workspace = torch.empty((need,), dtype=torch.uint8, device=q.device)
    stream, dev = _stream_and_device(q)
    rc = _lib.bwd(t4(q), t4(k), t4(v), t4(out), t4(dout), lse.data_ptr(), t4(dq), t4(dk), t4(dv),
                  workspace.data_ptr(), workspace.numel() * workspace.element_size(), code, causal, float(scale),
                  stream, dev, status.data_ptr() if status is not None else 0, simt=simt, parts=parts,
                  dropout=dropout)
    if rc != _lib.OK:
        raise _lib.B200FAError(rc, "b200fa_bwd")
    return dq, dk, dv


def _need_cuda(q) -> None:
    if q.device.type != "cuda":
        raise RuntimeError("b200fa kernels need CUDA memory; there is no CPU implementation")


def _same_kind(q, others) -> None:
    """Pointers are all that the library sees of a tensor: its type and device are checked here."""
    dtype, device = q.dtype, q.device
    for t in others:
        if t is not None and (t.dtype is not dtype or t.device != device):
            raise ValueError(f"expected {dtype} tensors on {device}, got {t.dtype} on {t.device}")


def _fp32_statistic(lse, shape, device) -> None:
    if lse.dtype != torch.float32 or tuple(lse.shape) != tuple(shape) or not lse.is_contiguous() or lse.device != device:
        raise ValueError(f"lse has to be a contiguous float32 tensor of shape {tuple(shape)} on {device}")


def window_fwd(q, k, v, *, window: int, sinks: int = 0, causal=True, scale: float | None = None, out=None, lse=None,
               status=None):
    """out, lse = causal attention over the last ``window`` keys and the first ``sinks`` ones.

    ``causal``: True (diagonal from the top-left corner) or ``_lib.CAUSAL_BOTTOM_RIGHT`` (new queries against a longer
    key sequence).  With p the last key that the diagonal lets a row see, the row sees key j iff ``j <= p`` and
    (``j > p - window`` or ``j < sinks``).  Shapes, types and results as for ``flash_fwd``; a row that sees no key is 0
    with lse -inf.  Values behind the mask have to be finite where a visible key shares their block of 128.
    """
    _need_cuda(q)
    B, Hq, Sq, D = q.shape
    if scale is None:
        scale = default_scale(D)
    if out is None:
        out = torch.empty((B, Hq, Sq, D), dtype=q.dtype, device=q.device)
    if lse is None:
        lse = torch.empty((B, Hq, Sq), dtype=torch.float32, device=q.device)
    else:
        _fp32_statistic(lse, (B, Hq, Sq), q.device)
    _same_kind(q, (k, v, out))
    stream, dev = _stream_and_device(q)
    rc = _lib.window_fwd(_t4b(q), _t4b(k), _t4b(v), _t4b(out), lse.data_ptr(), dtype_code(q.dtype), causal, window, sinks,
                         float(scale), stream, dev, status.data_ptr() if status is not None else 0)
    if rc != _lib.OK:
        raise _lib.B200FAError(rc, "b200fa_window_fwd")
    return out, lse


def window_bwd(dout, q, k, v, out, lse, *, window: int, sinks: int = 0, causal=True, scale: float | None = None, dq=None,
               dk=None, dv=None, workspace=None, status=None):
    """dq, dk, dv of ``window_fwd``, whose ``out`` and ``lse`` are given."""
    _need_cuda(q)
    B, Hq, S, D = q.shape
    Hkv, Sk = k.shape[1], k.shape[2]
    if scale is None:
        scale = default_scale(D)
    if dq is None:
        dq = torch.empty((B, Hq, S, D), dtype=q.dtype, device=q.device)
    if dk is None:
        dk = torch.empty(tuple(k.shape), dtype=q.dtype, device=q.device)
    if dv is None:
        dv = torch.empty(tuple(v.shape), dtype=q.dtype, device=q.device)
    _fp32_statistic(lse, (B, Hq, S), q.device)
    _same_kind(q, (dout, k, v, out, dq, dk, dv))
    code = dtype_code(q.dtype)
    need = _lib.window_bwd_workspace_bytes(B, Hq, Hkv, S, Sk, D, code, window, sinks)
    if workspace is None:
        workspace = torch.empty((need,), dtype=torch.uint8, device=q.device)
    stream, dev = _stream_and_device(q)
    rc = _lib.window_bwd(_t4b(q), _t4b(k), _t4b(v), _t4b(out), _t4b(dout), lse.data_ptr(), _t4b(dq), _t4b(dk), _t4b(dv),
                         workspace.data_ptr(), workspace.numel() * workspace.element_size(), code, causal, window, sinks,
                         float(scale), stream, dev, status.data_ptr() if status is not None else 0)
    if rc != _lib.OK:
        raise _lib.B200FAError(rc, "b200fa_window_bwd")
    return dq, dk, dv


class PagedKV(NamedTuple):
    """The pages of a key/value cache: a pool that the sequences' block tables name pages of.

    16 bits: ``k`` and ``v`` are (pages, Hkv, page_size, D) bfloat16 or float16.  4 bits: they are uint8 codes, two to a byte,
    (pages, Hkv, page_size, D / 2), and ``k_scales`` and ``v_scales`` hold a scale and a minimum of the 16-bit type for every 32
    elements, (pages, Hkv, page_size, D / 32, 2); an element is code * scale + minimum (the order of the codes: see
    ``b200fa_paged_kv`` in include/b200fa.h).  ``page_size`` is a power of two from 16 to 4096.
    """

    k: torch.Tensor
    v: torch.Tensor
    k_scales: torch.Tensor | None = None
    v_scales: torch.Tensor | None = None

    @classmethod
    def empty(cls, pages: int, heads: int, page_size: int, head_dim: int, *, dtype=torch.bfloat16, bits: int = 16,
              device="cuda") -> "PagedKV":
        """A pool whose contents are not set."""
        dtype_code(dtype)
        if bits == 16:
            return cls(*(torch.empty((pages, heads, page_size, head_dim), dtype=dtype, device=device) for _ in range(2)))
        if bits != 4 or head_dim % 64:
            raise NotImplementedError(f"a paged cache has 16 or 4 bits and a head dimension of 64 or 128, got {bits} and {head_dim}")
        codes = [torch.empty((pages, heads, page_size, head_dim // 2), dtype=torch.uint8, device=device) for _ in range(2)]
        return cls(*codes, *(torch.empty((pages, heads, page_size, head_dim // 32, 2), dtype=dtype, device=device)
                             for _ in range(2)))

    @property
    def dtype(self) -> torch.dtype:
        """The 16-bit type of the elements, or of the scales."""
        return (self.k if self.k_scales is None else self.k_scales).dtype


def _int32(name, t, batch: int, device) -> int:
    if t.dtype is not torch.int32 or t.dim() != 1 or t.shape[0] != batch or t.device != device or not t.is_contiguous():
        raise ValueError(f"{name} has to be a contiguous int32 tensor of shape {(batch,)} on {device}")
    return t.data_ptr()


def _paged(cache: PagedKV, block_table, lengths, new_lengths, batch: int):
    """(the cache as the library takes it, its 16-bit type, KV heads, head dimension, device, tokens that a row of the table has room
    for); pointers are all that the library sees, so types, shapes and devices are checked here."""
    k, v, ks, vs = cache
    device, shape = k.device, k.shape
    if device.type != "cuda":
        raise RuntimeError("b200fa kernels need CUDA memory; there is no CPU implementation")
    if len(shape) != 4 or v.shape != shape or v.dtype is not k.dtype or v.device != device or not (k.is_contiguous() and v.is_contiguous()):
        raise ValueError("the pages of k and v have to be contiguous and alike, (pages, heads, page_size, head_dim)")
    pages, heads, page_size, width = shape
    if ks is None:
        dtype, bits, ks_ptr, vs_ptr = k.dtype, 16, 0, 0
        if vs is not None:
            raise ValueError("16-bit pages have no scales")
    else:
        if k.dtype is not torch.uint8:
            raise ValueError("4-bit pages are uint8 codes")
        width *= 2
        want = (pages, heads, page_size, width // 32, 2)
        if vs is None or vs.dtype is not ks.dtype or any(
                tuple(s.shape) != want or s.device != device or not s.is_contiguous() for s in (ks, vs)):
            raise ValueError(f"the scales of a 4-bit cache have to be contiguous and alike, {want}")
        dtype, bits, ks_ptr, vs_ptr = ks.dtype, 4, ks.data_ptr(), vs.data_ptr()
    table_shape = block_table.shape
    if (len(table_shape) != 2 or table_shape[0] != batch or block_table.dtype is not torch.int32 or block_table.device != device
            or (table_shape[1] > 1 and block_table.stride(1) != 1)):
        raise ValueError(f"the block table has to be int32, (batch = {batch}, pages of a sequence), on {device}")
    packed = _lib.pack_paged_kv(
        k.data_ptr(), v.data_ptr(), ks_ptr, vs_ptr, block_table.data_ptr(), _int32("lengths", lengths, batch, device),
        _int32("new_lengths", new_lengths, batch, device) if new_lengths is not None else 0,
        pages, heads, page_size, width, batch, table_shape[1], block_table.stride(0), dtype_code(dtype), bits)
    return packed, dtype, heads, width, device, table_shape[1] * page_size


def paged_append(k, v, cache: PagedKV, block_table, lengths, *, new_lengths=None, rotary=None, interleaved: bool = False, q=None,
                 q_out=None, status=None):
    """Writes the new tokens' ``k`` and ``v`` (B, Hkv, S, D) to the pages, k rotated by position, and returns the rotated ``q``.

    ``block_table``: (B, pages of a sequence) int32; ``lengths``: (B,) int32, tokens in the cache with the new ones;
    ``new_lengths``: (B,) int32, how many of the S tokens are new ones (the first of each row; None: all).  Token s is written at
    position ``length - new + s``.  ``rotary``: (cos, sin), float32 (positions, R / 2): the first R elements turn, in pairs
    (i, i + R / 2) or, ``interleaved``, (2 i, 2 i + 1).  ``q``: (B, Hq, S, D), rotated the same way to ``q_out`` (a new tensor by
    default; q itself will do), whose rows behind a sequence's new tokens, or of tokens before position 0, are left as they are (in a new
    tensor zero, and NaN where a length or position is out of range).  ``status``: an int32 tensor of one element, zero, that reports a
    page, length or position out of range (include/b200fa.h).
    """
    B, Hkv, S, D = k.shape
    c, dtype, heads, head_dim, device, _ = _paged(cache, block_table, lengths, new_lengths, B)
    if D != head_dim or Hkv != heads or k.dtype is not dtype or k.device != device:
        raise ValueError(f"k and v have to be {dtype} of {heads} heads of {head_dim} on {device}")
    _same_kind(k, (v, q, q_out))
    cos_ptr = sin_ptr = rotary_dim = positions = 0
    if rotary is not None:
        cos, sin = rotary
        if (cos.dim() != 2 or sin.shape != cos.shape or cos.dtype is not torch.float32 or sin.dtype is not torch.float32
                or cos.device != device or sin.device != device or not (cos.is_contiguous() and sin.is_contiguous())):
            raise ValueError(f"rotary is (cos, sin), contiguous float32 (positions, R / 2) on {k.device}")
        cos_ptr, sin_ptr, positions, rotary_dim = cos.data_ptr(), sin.data_ptr(), cos.shape[0], 2 * cos.shape[1]
    if q is None and q_out is not None:
        raise ValueError("q_out without q")
    clear = q is not None and q_out is None
    if clear:
        q_out = torch.empty(tuple(q.shape), dtype=q.dtype, device=q.device)
    stream, dev = _stream_and_device(k)
    rc = _lib.paged_append(c, _t4b(k), _t4b(v), _t4b(q) if q is not None else None, _t4b(q_out) if q is not None else None, cos_ptr, sin_ptr,
                           rotary_dim, positions, interleaved, stream, dev, status.data_ptr() if status is not None else 0, clear)
    if rc != _lib.OK:
        raise _lib.B200FAError(rc, "b200fa_paged_append")
    return q_out


def paged_attention(q, cache: PagedKV, block_table, lengths, *, new_lengths=None, window: int = 0, sinks: int = 0,
                    scale: float | None = None, out=None, lse=None, longest: int = 0, workspace=None, status=None):
    """out, lse = causal attention of the newest tokens' ``q`` (B, Hq, S, D) over the pages of their sequences.

    ``block_table``, ``lengths`` and ``new_lengths`` as for ``paged_append``, which comes first: the new tokens see each other and
    themselves.  ``window`` > 0: the last ``window`` keys and the first ``sinks`` ones alone.  Rows behind a sequence's new tokens
    are left as they are (out zero and lse -inf in new tensors).  ``longest``: a hint, the longest of the lengths, where the block
    table is much wider.  ``workspace``: scratch on q's device, for calls of few KV heads (a new tensor by default; one without
    elements keeps a KV head to one cluster).
    """
    B, Hq, S, D = q.shape
    c, dtype, heads, head_dim, device, keys = _paged(cache, block_table, lengths, new_lengths, B)
    if D != head_dim or q.dtype is not dtype or q.device != device:
        raise ValueError(f"q has to be {dtype} of head dimension {head_dim} on {device}")
    if scale is None:
        scale = default_scale(D)
    if out is None:
        out = (torch.empty if new_lengths is None else torch.zeros)((B, Hq, S, D), dtype=q.dtype, device=q.device)
    if lse is None:
        lse = torch.empty((B, Hq, S), dtype=torch.float32, device=q.device)
        if new_lengths is not None:
            lse.fill_(-math.inf)
    else:
        _fp32_statistic(lse, (B, Hq, S), q.device)
    _same_kind(q, (out,))
    scratch = scratch_bytes = 0
    if workspace is None and keys >= _lib.PAGED_TEAM_KEYS:
        keys = min(keys, longest or keys, window + sinks + S if window else keys)
        need = _lib.paged_attention_workspace_bytes(B, Hq, heads, S, D, keys)
        if need:
            workspace = torch.empty((need,), dtype=torch.uint8, device=device)
    if workspace is not None:
        if workspace.device != device or not workspace.is_contiguous():
            raise ValueError(f"workspace has to be contiguous, on {device}")
        scratch, scratch_bytes = workspace.data_ptr(), workspace.numel() * workspace.element_size()
    stream, dev = _stream_and_device(q)
    rc = _lib.paged_attention(c, _t4b(q), _t4b(out), lse.data_ptr(), window, sinks, float(scale), longest, stream, dev,
                              status.data_ptr() if status is not None else 0, scratch, scratch_bytes)
    if rc != _lib.OK:
        raise _lib.B200FAError(rc, "b200fa_paged_attention")
    return out, lse


def paged_gather(cache: PagedKV, block_table, lengths, length: int, *, k=None, v=None, status=None):
    """k, v = the first ``length`` tokens of every sequence, (B, Hkv, length, D) of the cache's 16-bit type; rows behind a
    sequence's own length are zero.  ``k`` and ``v``: tensors to write to."""
    B = lengths.shape[0]
    c, dtype, heads, head_dim, device, _ = _paged(cache, block_table, lengths, None, B)
    shape = (B, heads, length, head_dim)
    if k is None:
        k = torch.empty(shape, dtype=dtype, device=device)
    if v is None:
        v = torch.empty(shape, dtype=dtype, device=device)
    for t in (k, v):
        if tuple(t.shape) != shape or t.dtype is not dtype or t.device != device:
            raise ValueError(f"k and v have to be {dtype} of shape {shape} on {device}")
    stream, dev = _stream_and_device(k)
    rc = _lib.paged_gather(c, _t4b(k), _t4b(v), stream, dev, status.data_ptr() if status is not None else 0)
    if rc != _lib.OK:
        raise _lib.B200FAError(rc, "b200fa_paged_gather")
    return k, v
