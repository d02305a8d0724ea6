"""``torch.ops.fusedmm_b200.csr``: the C ABI as a PyTorch custom operator (CUDA tensors, zero copy, enqueued on
torch's current stream).  This is the binding a GNN framework built on PyTorch would call (the reference ships a
CMake file "for DGL integration", ``CMakeLists.txt:1``); autograd is not defined for it.

    import fusedmm_b200.torch_op            # registers the operator
    z = torch.ops.fusedmm_b200.csr(rowptr, colidx, val, x, y, imessage, sop_kind, beta, z_in)

The attention form of that call, with its gradients (CUDA tensors, on torch's current stream):

    q, k = qk_norm_rotary(q, k, pos, freq, q_weight=wq, k_weight=wk, eps=1e-6)   # norm of each head, rotation by positions
    transposed = csr_transpose(rowptr, colidx, n)                                # once for a pattern that stays
    out = diff_attention(rowptr, colidx, q, k, v, lam, transposed=transposed)    # difference of two softmax maps
"""
from __future__ import annotations

from typing import Optional

import torch

from . import api


@torch.library.custom_op("fusedmm_b200::csr", mutates_args=(), device_types="cuda")
def csr(rowptr: torch.Tensor, colidx: torch.Tensor, val: Optional[torch.Tensor], x: torch.Tensor, y: torch.Tensor,
        imessage: int, sop_kind: int, beta: float, z_in: Optional[torch.Tensor]) -> torch.Tensor:
    """Z = fusedMM_csr(imessage; CSR(rowptr, colidx, val); X, Y), rows of Z = rows of X.  ``z_in`` is the Z the
    message accumulates into (messages the reference has no optimised kernel for always accumulate; the four
    optimised ones only when beta != 0); ``None`` means zeros."""
    m, k = x.shape
    n = y.shape[0]
    z = torch.zeros((m, k), dtype=x.dtype, device=x.device) if z_in is None else z_in.clone()
    stream = torch.cuda.current_stream(x.device)
    handle = stream.cuda_stream
    if handle == 0:  # the legacy default stream is the C ABI's "synchronous" value: run synchronously
        handle = None
    # nnz = colidx.numel() bounds the edges of the rows, so the library sizes its split-row scratch before it
    # enqueues anything and the call needs no later status check
    with torch.cuda.device(x.device):
        st = api.fusedMM_csr(imessage, m, n, k, 1.0, int(colidx.numel()), m, n, val, colidx, rowptr[:-1], rowptr[1:],
                             x.contiguous(), k, y.contiguous(), k, float(beta), z, k, sop=int(sop_kind), stream=handle)
    if st != 0:
        raise api.FusedMMError(f"fusedMM_csr failed: {api.status_string(st)} ({st})")
    return z


@csr.register_fake
def _(rowptr, colidx, val, x, y, imessage, sop_kind, beta, z_in):
    return torch.empty_like(x)


# ---- attention over the edges of a CSR -----------------------------------------------------------------------------
_lib = torch.library.Library("fusedmm_b200", "FRAGMENT")
_lib.define("qk_norm_rotary(Tensor q, Tensor? k, Tensor? pos, Tensor? freq, Tensor? q_weight, Tensor? k_weight, float? eps, "
            "bool interleaved) -> (Tensor, Tensor)")
_lib.define("qk_norm_rotary_backward(Tensor q, Tensor? k, Tensor? pos, Tensor? freq, Tensor? q_weight, Tensor? k_weight, "
            "float? eps, bool interleaved, Tensor dq_out, Tensor? dk_out) -> (Tensor, Tensor, Tensor, Tensor)")
_lib.define("diff_attention(Tensor rowptr, Tensor colidx, Tensor? bias, Tensor q, Tensor k, Tensor v, Tensor lam, float scale, "
            "Tensor? t_rowptr, Tensor? t_row, Tensor? t_edge) -> (Tensor, Tensor)")
_lib.define("diff_attention_backward(Tensor rowptr, Tensor colidx, Tensor? bias, Tensor q, Tensor k, Tensor v, Tensor lam, "
            "float scale, Tensor lse, Tensor dout, Tensor t_rowptr, Tensor t_row, Tensor? t_edge) -> (Tensor, Tensor, Tensor, Tensor)")
_lib.define("csr_transpose(Tensor rowptr, Tensor colidx, int n) -> (Tensor, Tensor, Tensor)")


def _stream(device):
    return torch.cuda.current_stream(device).cuda_stream or api.LEGACY_STREAM


def _check(status, name):
    if status != 0:
        raise api.FusedMMError(f"{name} failed: {api.status_string(status)} ({status})")


def _scratch(size, name, device):
    if size < 0:
        _check(size, name)
    return torch.empty(max(size, 1), dtype=torch.uint8, device=device)


def _rotary_cuda(q, k, pos, freq, q_weight, k_weight, eps, interleaved):
    with torch.cuda.device(q.device):
        q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        k_out = torch.empty(k.shape if k is not None else (0,), dtype=q.dtype, device=q.device)
        _check(api.qk_norm_rotary(q, k, q_weight, k_weight, pos, freq, eps, interleaved, q_out, k_out if k is not None else None,
                                  _stream(q.device)), "qk_norm_rotary")
    return q_out, k_out


def _rotary_backward_cuda(q, k, pos, freq, q_weight, k_weight, eps, interleaved, dq_out, dk_out):
    dev = q.device
    with torch.cuda.device(dev):
        dq = torch.empty(q.shape, dtype=q.dtype, device=dev)
        dk = torch.empty(k.shape if k is not None else (0,), dtype=q.dtype, device=dev)
        dw = [torch.empty(q.shape[2] if w is not None else 0, dtype=torch.float32, device=dev) for w in (q_weight, k_weight)]
        weights = q_weight is not None or k_weight is not None
        ws = _scratch(api.qk_norm_rotary_backward_workspace(q.shape[0], q.shape[2]), "qk_norm_rotary_backward", dev) if weights else None
        _check(api.qk_norm_rotary_backward(q, k, q_weight, k_weight, pos, freq, eps, interleaved, dq_out, dk_out, dq,
                                           dk if k is not None else None, dw[0] if q_weight is not None else None,
                                           dw[1] if k_weight is not None else None, ws, _stream(dev)), "qk_norm_rotary_backward")
    return dq, dk, dw[0], dw[1]


def _attention_cuda(rowptr, colidx, bias, q, k, v, lam, scale, t_rowptr=None, t_row=None, t_edge=None):
    api._attention_args(rowptr, colidx, bias, q, k, v, lam, scale)  # before anything is sized by its shapes
    dev = q.device
    with torch.cuda.device(dev):
        m, heads = q.shape[:2]
        out = torch.empty((m, heads, v.shape[2]), dtype=q.dtype, device=dev)
        lse = torch.empty((m, heads, 2), dtype=torch.float32, device=dev)
        ws = _scratch(api.diff_attention_workspace(False, q, k, v, colidx.numel()), "diff_attention", dev)
        _check(api.diff_attention(rowptr, colidx, bias, q, k, v, lam, scale, out, lse, ws, _stream(dev)), "diff_attention")
    return out, lse


def _attention_backward_cuda(rowptr, colidx, bias, q, k, v, lam, scale, lse, dout, t_rowptr, t_row, t_edge):
    dev = q.device
    with torch.cuda.device(dev):
        dq = torch.empty(q.shape, dtype=q.dtype, device=dev)
        dk = torch.empty(k.shape, dtype=k.dtype, device=dev)
        dv = torch.empty(v.shape, dtype=v.dtype, device=dev)
        dlam = torch.empty(lam.shape, dtype=torch.float32, device=dev)
        ws = _scratch(api.diff_attention_workspace(True, q, k, v, colidx.numel()), "diff_attention_backward", dev)
        _check(api.diff_attention_backward(rowptr, colidx, bias, q, k, v, lam, scale, lse, dout, t_rowptr, t_row, t_edge, dq, dk,
                                           dv, dlam, ws, _stream(dev)), "diff_attention_backward")
    return dq, dk, dv, dlam


def _transpose_cuda(rowptr, colidx, n):
    api._pattern_args(rowptr, colidx)
    dev, nnz = rowptr.device, colidx.numel()
    with torch.cuda.device(dev):
        ws = _scratch(api.csr_transpose_workspace(rowptr.numel() - 1, n, nnz), "csr_transpose", dev)
        t_rowptr = torch.empty(n + 1, dtype=rowptr.dtype, device=dev)
        t_row, t_edge = torch.empty(nnz, dtype=torch.int32, device=dev), torch.empty(nnz, dtype=torch.int32, device=dev)
        _check(api.csr_transpose(rowptr, colidx, n, t_rowptr, t_row, t_edge, ws, _stream(dev)), "csr_transpose")
    return t_rowptr, t_row, t_edge


def _dense_rows(t):
    """A gradient whose last axes are not dense (an expanded one, say) is laid out anew."""
    return t if t.stride(-1) == 1 and t.stride(0) != 0 and t.stride(1) != 0 else t.contiguous()


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, pos, freq, q_weight, k_weight, eps, interleaved):
        with torch._C._AutoDispatchBelowAutograd():
            out = torch.ops.fusedmm_b200.qk_norm_rotary(q, k, pos, freq, q_weight, k_weight, eps, interleaved)
        ctx.save_for_backward(q, k, pos, freq, q_weight, k_weight)
        ctx.args = eps, interleaved
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dq_out, dk_out):
        q, k, pos, freq, q_weight, k_weight = ctx.saved_tensors
        if ctx.needs_input_grad[2] or ctx.needs_input_grad[3]:
            raise api.FusedMMError("qk_norm_rotary has no gradient for pos and freq")
        eps, interleaved = ctx.args
        dq, dk, dwq, dwk = torch.ops.fusedmm_b200.qk_norm_rotary_backward(
            q, k, pos, freq, q_weight, k_weight, eps, interleaved, _dense_rows(dq_out), None if k is None else _dense_rows(dk_out))
        need = ctx.needs_input_grad
        return (dq if need[0] else None, dk if k is not None and need[1] else None, None, None,
                dwq.to(q_weight.dtype) if need[4] else None, dwk.to(k_weight.dtype) if need[5] else None, None, None)


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rowptr, colidx, bias, q, k, v, lam, scale, t_rowptr, t_row, t_edge):
        with torch._C._AutoDispatchBelowAutograd():
            out, lse = torch.ops.fusedmm_b200.diff_attention(rowptr, colidx, bias, q, k, v, lam, scale, t_rowptr, t_row, t_edge)
        ctx.save_for_backward(rowptr, colidx, bias, q, k, v, lam, lse, t_rowptr, t_row, t_edge)
        ctx.scale = scale
        ctx.mark_non_differentiable(lse)
        return out, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, _):
        rowptr, colidx, bias, q, k, v, lam, lse, t_rowptr, t_row, t_edge = ctx.saved_tensors
        if ctx.needs_input_grad[2]:
            raise api.FusedMMError("diff_attention has no gradient for bias")
        if t_rowptr is None:
            t_rowptr, t_row, t_edge = torch.ops.fusedmm_b200.csr_transpose(rowptr, colidx, k.shape[0])
        grads = torch.ops.fusedmm_b200.diff_attention_backward(rowptr, colidx, bias, q, k, v, lam, ctx.scale, lse,
                                                               _dense_rows(dout), t_rowptr, t_row, t_edge)
        return (None, None, None, *[g if need else None for g, need in zip(grads, ctx.needs_input_grad[3:7])], None, None, None, None)


_lib.impl("qk_norm_rotary", _rotary_cuda, "CUDA")
_lib.impl("qk_norm_rotary_backward", _rotary_backward_cuda, "CUDA")
_lib.impl("diff_attention", _attention_cuda, "CUDA")
_lib.impl("diff_attention_backward", _attention_backward_cuda, "CUDA")
_lib.impl("csr_transpose", _transpose_cuda, "CUDA")
_lib.impl("qk_norm_rotary", lambda *args: _Rotary.apply(*args), "AutogradCUDA")
_lib.impl("diff_attention", lambda *args: _Attention.apply(*args), "AutogradCUDA")


@torch.library.register_fake("fusedmm_b200::qk_norm_rotary", lib=_lib)
def _(q, k, pos, freq, q_weight, k_weight, eps, interleaved):
    return q.new_empty(q.shape), q.new_empty(k.shape if k is not None else (0,))


@torch.library.register_fake("fusedmm_b200::qk_norm_rotary_backward", lib=_lib)
def _(q, k, pos, freq, q_weight, k_weight, eps, interleaved, dq_out, dk_out):
    def weight(w):
        return q.new_empty(q.shape[2] if w is not None else 0, dtype=torch.float32)
    return q.new_empty(q.shape), q.new_empty(k.shape if k is not None else (0,)), weight(q_weight), weight(k_weight)


@torch.library.register_fake("fusedmm_b200::diff_attention", lib=_lib)
def _(rowptr, colidx, bias, q, k, v, lam, scale, t_rowptr, t_row, t_edge):
    m, heads = q.shape[:2]
    return q.new_empty((m, heads, v.shape[2])), q.new_empty((m, heads, 2), dtype=torch.float32)


@torch.library.register_fake("fusedmm_b200::diff_attention_backward", lib=_lib)
def _(rowptr, colidx, bias, q, k, v, lam, scale, lse, dout, t_rowptr, t_row, t_edge):
    return q.new_empty(q.shape), k.new_empty(k.shape), v.new_empty(v.shape), lam.new_empty(lam.shape)


@torch.library.register_fake("fusedmm_b200::csr_transpose", lib=_lib)
def _(rowptr, colidx, n):
    return rowptr.new_empty(n + 1), rowptr.new_empty(colidx.numel(), dtype=torch.int32), rowptr.new_empty(colidx.numel(), dtype=torch.int32)


def qk_norm_rotary(q, k=None, pos=None, freq=None, *, q_weight=None, k_weight=None, eps=None, interleaved=False):
    """Norm of each head and rotation by the position of its row, in one pass; differentiable in q, k and the weights.

    ``q`` and ``k`` are [rows, heads, d] (views are fine as long as the last axis is dense; ``k`` may be left out, and
    alone the result of ``q`` is returned).  With ``eps`` every head is divided by its root mean square and multiplied by
    ``q_weight`` / ``k_weight`` [d] (ones if left out).  With ``pos`` [rows] or [rows, axes] (up to four axes; integers or
    coordinates) and ``freq`` [axes, pairs] (float64) the pairs (i, i + pairs), or (2i, 2i + 1) with ``interleaved``, turn
    by ``pos @ freq``; a pair that belongs to one axis has zeros on the others; elements behind the pairs pass."""
    q_out, k_out = torch.ops.fusedmm_b200.qk_norm_rotary(q, k, pos, freq, q_weight, k_weight, eps, interleaved)
    return q_out if k is None else (q_out, k_out)


def diff_attention(rowptr, colidx, q, k, v, lam, *, bias=None, scale=None, transposed=None, return_lse=False):
    """Differential attention over the edges of a CSR; differentiable in q, k, v and lam.

    ``q`` [m, heads, 2, d], ``k`` [n, kv_heads, 2, d], ``v`` [n, kv_heads, dv], ``lam`` [heads] or [m, heads] (float32):
    for each row the softmax maps of the two parts over its edges are formed, the second times ``lam`` is taken from the
    first, and the rows of ``v`` are summed with the differences: [m, heads, dv].  ``colidx`` lists rows of k and v (nodes,
    or the slots of a cache); an id outside [0, n) or a ``bias`` of -inf drops the edge; rows without edges give zeros.
    ``scale`` is 1/sqrt(d) if left out.  ``transposed``: what :func:`csr_transpose` made of this pattern; without it a
    backward pass makes it again.  With ``return_lse`` also the logarithms of the maps' sums, [m, heads, 2]."""
    t = (None, None, None) if transposed is None else transposed
    out, lse = torch.ops.fusedmm_b200.diff_attention(rowptr, colidx, bias, q, k, v, lam, q.shape[-1] ** -0.5 if scale is None else scale, *t)
    return (out, lse) if return_lse else out


def csr_transpose(rowptr, colidx, n):
    """The transposed pattern of a CSR with ``n`` columns: row pointers of the columns, the rows of their edges and the
    edges' positions in ``colidx`` (edges outside [0, n) left out).  What ``diff_attention(transposed=...)`` takes."""
    return torch.ops.fusedmm_b200.csr_transpose(rowptr, colidx, n)
