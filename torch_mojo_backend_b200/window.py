"""Window attention on the `mojo` device: causal attention over the last keys and the first ones, with its gradients.

``window_attention`` is to ``b200fa_window_fwd`` / ``b200fa_window_bwd`` what ``F.scaled_dot_product_attention`` is to
``b200fa_fwd`` / ``b200fa_bwd`` (``flash_ops.py``): eligibility from metadata alone, zero-copy layouts, outputs and gradients
in the layout of the tensors they belong to, ``NotImplementedError`` from the forward for what the kernels do not serve.  There
is no aten operator for it, so the gradient is an autograd function of this module.  No counterpart in the reference, whose
window argument no entry point reaches (torch_mojo_backend/eager_flash_attention/fa4_fwd_common.mojo:26-29).
"""

from __future__ import annotations

import contextlib
import math

import torch

from . import _lib, autocast, flash_ops, tensor
from .tensor import TorchMojoTensor, payload


def _packed(t: TorchMojoTensor) -> bytes:
    return _lib.pack_tensor4(t._ptr, *t._shape, *t._strides)


def _inputs(query, key, value, window, sinks, scale, enable_gqa):
    inputs = flash_ops.flash_inputs(query, key, value, None, 0.0, True, scale, enable_gqa)
    sizes_fit = all(isinstance(n, int) and not isinstance(n, bool) for n in (window, sinks)) and window >= 1 and sinks >= 0
    if inputs is None or not sizes_fit:
        raise NotImplementedError(
            "window_attention on the mojo device needs fp32/bf16/fp16 (B,H,S,D) tensors, head_dim 64 or 128, a positive scale, "
            "enable_gqa=True when the key/value head count differs, window >= 1 and sinks >= 0"
        )
    return inputs


def _forward(q, k, v, window, sinks, causal, scale):
    batch, heads_q, seq, _ = q._shape
    index = q._device_index
    q_used, k_used, v_used = (flash_ops.prepare(t) for t in (q, k, v))
    out = flash_ops._alloc_like_layout(q._shape, q._dtype, index, flash_ops.bthd_stored(q_used))
    lse = TorchMojoTensor._alloc((batch, heads_q, seq), torch.float32, index)
    flash_ops._log("window_fwd q=%s k=%s window=%d sinks=%d", q._shape, k._shape, window, sinks)
    rc = _lib.window_fwd(_packed(q_used), _packed(k_used), _packed(v_used), _packed(out), lse._ptr, flash_ops._DTYPE_CODES[q._dtype],
                         causal, window, sinks, scale, flash_ops._stream_for(index), index, flash_ops._status_ptr(index))
    flash_ops._check(rc, "b200fa_window_fwd")
    return out, lse


def _backward(dout, q, k, v, out, lse, window, sinks, causal, scale):
    batch, heads_q, seq, head_dim = q._shape
    index = q._device_index
    code = flash_ops._DTYPE_CODES[q._dtype]
    q_used, k_used, v_used, out_used, dout_used = (flash_ops.prepare(t) for t in (q, k, v, out, dout))
    dq, dk, dv = (flash_ops._alloc_like_layout(t._shape, q._dtype, index, flash_ops.bthd_stored(t)) for t in (q_used, k_used, v_used))
    nbytes = _lib.window_bwd_workspace_bytes(batch, heads_q, k._shape[1], seq, k._shape[2], head_dim, code, window, sinks)
    workspace = tensor._alloc_holder(nbytes, index)
    flash_ops._log("window_bwd q=%s k=%s window=%d sinks=%d", q._shape, k._shape, window, sinks)
    rc = _lib.window_bwd(_packed(q_used), _packed(k_used), _packed(v_used), _packed(out_used), _packed(dout_used), lse._ptr, _packed(dq),
                         _packed(dk), _packed(dv), workspace.data_ptr(), nbytes, code, causal, window, sinks, scale,
                         flash_ops._stream_for(index), index, flash_ops._status_ptr(index))
    flash_ops._check(rc, "b200fa_window_bwd")
    return dq, dk, dv


@contextlib.contextmanager
def _on_stream(stream):
    """A backward on the forward's stream (None: no CUDA memory, no stream).  What else the engine has to do for it (sums of a tensor's
    gradients, gradients of views) goes to the current stream of the engine's thread: the two wait for one another, and in the end the
    forward's, where the caller goes on, for the other.  A stream that is being captured cannot wait for one that is not: it becomes the
    thread's current one until the pass is over."""
    if stream is None:
        yield
        return
    tensor.take_back_stream()
    current = torch.cuda.current_stream(stream.device)
    if current == stream:
        yield
        return
    with torch.cuda.stream(stream):
        lend = torch.cuda.is_current_stream_capturing()
        if lend:
            with torch.cuda.stream(current):
                lend = not torch.cuda.is_current_stream_capturing()
        if not lend:
            stream.wait_stream(current)
        yield
    if lend:
        tensor.lend_stream(stream)
    else:
        current.wait_stream(stream)
        torch.autograd.Variable._execution_engine.queue_callback(lambda: stream.wait_stream(current))


class _WindowAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, query, key, value, window, sinks, causal, scale):
        q, k, v = payload(query), payload(key), payload(value)
        out, lse = _forward(q, k, v, window, sinks, causal, scale)
        ctx.save_for_backward(query, key, value, out, lse)
        ctx.how = window, sinks, causal, scale
        # The engine calls the backward from a thread of its own, whose current stream is not the caller's (`_on_stream`)
        ctx.stream = torch.cuda.current_stream(q._device_index) if q._holder.is_cuda else None
        ctx.mark_non_differentiable(lse)
        ctx.set_materialize_grads(False)
        return out, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, _):
        if dout is None:
            return (None,) * 7
        query, key, value, out, lse = (payload(t) for t in ctx.saved_tensors)
        with _on_stream(ctx.stream):
            return (*_backward(payload(dout), query, key, value, out, lse, *ctx.how), None, None, None, None)


def window_attention(query, key, value, window: int, *, sinks: int = 0, bottom_right: bool = False, scale: float | None = None,
                     enable_gqa: bool = False, return_lse: bool = False):
    """Causal attention in which a query sees the last ``window`` keys of its causal range and the first ``sinks`` ones.

    Tensors, types, ``scale`` and ``enable_gqa`` as for ``F.scaled_dot_product_attention`` on the device.  The last key a query
    i may see is i, or, ``bottom_right``, i + Sk - Sq (new queries against a longer key sequence).  Differentiable once, on the
    stream that the call was made on (which a graph that also holds other operators of the device needs for all of them: on a stream that
    is not the default one, call its backward under ``torch.autograd.set_multithreading_enabled(False)``); ``return_lse``: the logsumexp of the scaled, visible scores too, (B, H, Sq) float32,
    which has no gradient.  Under ``torch.autocast("mojo")`` the tensors are cast to its type, as for the attention operators.
    """
    if torch.is_autocast_enabled("mojo"):
        query, key, value = (autocast._to_autocast_dtype(t) for t in (query, key, value))
    q, _, _ = _inputs(query, key, value, window, sinks, scale, enable_gqa)
    scale = 1.0 / math.sqrt(q._shape[3]) if scale is None else float(scale)
    causal = _lib.CAUSAL_BOTTOM_RIGHT if bottom_right else _lib.CAUSAL_TOP_LEFT
    out, lse = _WindowAttention.apply(query, key, value, window, sinks, causal, scale)
    return (out, lse) if return_lse else out
