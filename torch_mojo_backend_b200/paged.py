"""A paged key/value cache on the `mojo` device: the calls of ``raw.PagedKV`` on mojo tensors.

The pool of pages, block tables and lengths are those of ``b200fa_paged_kv`` (include/b200fa.h); a mojo tensor is the memory of
its CUDA device, so the methods hand the same addresses to the same calls, on the current CUDA stream, and pass the device's
status word along: ``torch.mojo.synchronize()`` raises when a page, a length or a position was out of range.  No counterpart in
the reference, whose decode path takes dense caches of at most 4096 keys
(torch_mojo_backend/eager_kernels/aten_fast.py:9171-9203).
"""

from __future__ import annotations

import torch

from . import flash_ops, raw
from .tensor import TorchMojoTensor, payload


def _cuda(name: str, t):
    """The CUDA tensor behind a mojo tensor."""
    if t is None:
        return None
    held = payload(t)
    if held is None:
        raise RuntimeError(f"PagedKVCache: {name} has to be a mojo tensor, got {type(t).__name__}")
    return held._cuda_view()


def _refuse_gradients(names, tensors) -> None:
    """Asked only where gradients are recorded: 0.3 us a tensor on the host."""
    for i, t in enumerate(tensors):
        if getattr(t, "requires_grad", False):
            name = names[min(i, len(names) - 1)]
            raise NotImplementedError(f"PagedKVCache: {name} requires a gradient, and nothing goes back through a cache; call it under torch.no_grad()")


class _Status:
    """The device's status word in the form the calls in ``raw`` take one."""

    __slots__ = ("index",)

    def __init__(self, index: int) -> None:
        self.index = index

    def data_ptr(self) -> int:
        return flash_ops._status_ptr(self.index)


class PagedKVCache:
    """A pool of ``pages`` pages of ``page_size`` tokens (a power of two, 16 to 4096) of every KV head.

    ``bits`` 16: pages hold ``dtype`` (bfloat16 or float16); 4: codes with a scale and a minimum of ``dtype`` for every 32
    elements.  Which pages a sequence has is the caller's: every call takes the ``block_table`` (B, pages of a sequence) and the
    ``lengths`` (B,), int32 mojo tensors that are read on the device (``raw.paged_append`` says how, and what ``new_lengths``
    are).  A call is safe beside others on other streams as long as no two write, or one writes and another reads, the same
    places; it keeps no workspace (a call's own scratch is allocated on the stream it runs on).  Nothing is differentiated: where gradients
    are recorded, a tensor that requires one is refused (``NotImplementedError``).
    """

    def __init__(self, pages: int, kv_heads: int, page_size: int, head_dim: int, *, dtype=torch.bfloat16, bits: int = 16,
                 device="mojo") -> None:
        if dtype not in (torch.bfloat16, torch.float16):
            raise NotImplementedError(f"a paged cache holds bfloat16 or float16, got {dtype}")
        if head_dim not in (64, 128) or page_size not in (16, 32, 64, 128, 256, 512, 1024, 2048, 4096):
            raise NotImplementedError("a paged cache needs head_dim 64 or 128 and a page_size that is a power of two from 16 to 4096")
        from .device_module import _index_of

        index = _index_of(device)
        self.kv = raw.PagedKV.empty(pages, kv_heads, page_size, head_dim, dtype=dtype, bits=bits, device=torch.device("cuda", index))
        self._status = _Status(index)

    @property
    def dtype(self) -> torch.dtype:
        return self.kv.dtype

    def append(self, key, value, block_table, lengths, *, new_lengths=None, rotary=None, interleaved: bool = False, query=None):
        """Writes the new tokens' ``key`` and ``value`` (B, Hkv, S, D); returns ``query`` rotated as the keys are, if given.
        ``rotary``: (cos, sin), float32 (positions, R / 2) mojo tensors."""
        if torch.is_grad_enabled():
            _refuse_gradients(("key", "value", "query", "rotary"), (key, value, query, *(rotary or ())))
        if rotary is not None:
            rotary = tuple(_cuda("rotary", t) for t in rotary)
        out = raw.paged_append(_cuda("key", key), _cuda("value", value), self.kv, _cuda("block_table", block_table),
                               _cuda("lengths", lengths), new_lengths=_cuda("new_lengths", new_lengths), rotary=rotary,
                               interleaved=interleaved, q=_cuda("query", query), status=self._status)
        return None if out is None else TorchMojoTensor._from_cuda(out)

    def attention(self, query, block_table, lengths, *, new_lengths=None, window: int = 0, sinks: int = 0, scale: float | None = None,
                  longest: int = 0, return_lse: bool = False):
        """Causal attention of the newest tokens' ``query`` (B, Hq, S, D) over the pages."""
        if torch.is_grad_enabled():
            _refuse_gradients(("query",), (query,))
        out, lse = raw.paged_attention(_cuda("query", query), self.kv, _cuda("block_table", block_table), _cuda("lengths", lengths),
                                       new_lengths=_cuda("new_lengths", new_lengths), window=window, sinks=sinks, scale=scale,
                                       longest=longest, status=self._status)
        out = TorchMojoTensor._from_cuda(out)
        return (out, TorchMojoTensor._from_cuda(lse)) if return_lse else out

    def gather(self, block_table, lengths, length: int):
        """The first ``length`` tokens of every sequence as dense (B, Hkv, length, D) keys and values, zero behind a sequence's own."""
        k, v = raw.paged_gather(self.kv, _cuda("block_table", block_table), _cuda("lengths", lengths), length, status=self._status)
        return TorchMojoTensor._from_cuda(k), TorchMojoTensor._from_cuda(v)
