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
from torch.autograd import forward_ad

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


def _check(status, name):
    if status != 0:
        raise api.FusedMMError(f"{name} failed: {api.status_string(status)} ({status})")


class _On:
    """Makes a tensor's device the current one for a call (nothing to do as a rule) and gives torch's stream on it."""
    __slots__ = ("device", "index", "guard", "stream")

    def __init__(self, device):
        self.device, self.index, self.guard = device, device.index, None

    def __enter__(self):
        if self.index != torch.cuda.current_device():
            self.guard = torch.cuda.device(self.index)
            self.guard.__enter__()
        self.stream = torch._C._cuda_getCurrentRawStream(self.index) or api.LEGACY_STREAM
        return self

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)

    def empty(self, shape, dtype):
        return torch.empty(shape, dtype=dtype, device=self.device)

    def scratch(self, size, name):
        if size < 0:
            _check(size, name)
        return torch.empty(size or 1, dtype=torch.uint8, device=self.device)


def _rotary_cuda(q, k, pos, freq, q_weight, k_weight, eps, interleaved):
    args = api.rotary_args(q, k, q_weight, k_weight, pos, freq, eps, interleaved)
    with _On(q.device) as on:
        q_out = on.empty(q.shape, q.dtype)
        k_out = on.empty(k.shape if k is not None else 0, q.dtype)
        _check(api.qk_norm_rotary(args, q_out, k_out if k is not None else None, on.stream), "qk_norm_rotary")
    return q_out, k_out


def _rotary_backward_cuda(q, k, pos, freq, q_weight, k_weight, eps, interleaved, dq_out, dk_out):
    args = api.rotary_args(q, k, q_weight, k_weight, pos, freq, eps, interleaved)
    with _On(q.device) as on:
        dq = on.empty(q.shape, q.dtype)
        dk = on.empty(k.shape if k is not None else 0, q.dtype)
        dwq = on.empty(q.shape[2], torch.float32) if q_weight is not None else None
        dwk = on.empty(q.shape[2], torch.float32) if k_weight is not None else None
        ws = None
        if dwq is not None or dwk is not None:
            ws = on.scratch(api.qk_norm_rotary_backward_workspace(q.shape[0], q.shape[2]), "qk_norm_rotary_backward")
        _check(api.qk_norm_rotary_backward(args, q, k, dq_out, dk_out, dq, dk if k is not None else None, dwq, dwk, ws, on.stream),
               "qk_norm_rotary_backward")
        none = None if dwq is not None and dwk is not None else on.empty(0, torch.float32)
    return dq, dk, none if dwq is None else dwq, none if dwk is None else dwk


def _attention_forward(rowptr, colidx, bias, q, k, v, lam, scale, want_lse):
    args = api.attention_args(rowptr, colidx, bias, q, k, v, lam, scale)
    with _On(q.device) as on:
        m, heads = q.shape[0], q.shape[1]
        out = on.empty((m, heads, v.shape[2]), q.dtype)
        lse = on.empty((m, heads, 2), torch.float32) if want_lse else None
        ws = on.scratch(api.diff_attention_workspace(False, args), "diff_attention")
        _check(api.diff_attention(args, out, lse, ws, on.stream), "diff_attention")
    return out, lse


def _attention_cuda(rowptr, colidx, bias, q, k, v, lam, scale, t_rowptr=None, t_row=None, t_edge=None):
    return _attention_forward(rowptr, colidx, bias, q, k, v, lam, scale, True)


def _attention_backward_cuda(rowptr, colidx, bias, q, k, v, lam, scale, lse, dout, t_rowptr, t_row, t_edge):
    args = api.attention_args(rowptr, colidx, bias, q, k, v, lam, scale)
    with _On(q.device) as on:
        dq, dk, dv = on.empty(q.shape, q.dtype), on.empty(k.shape, k.dtype), on.empty(v.shape, v.dtype)
        dlam = on.empty(lam.shape, torch.float32)
        ws = on.scratch(api.diff_attention_workspace(True, args, dout.data_ptr(), *api._rows(dout, "dout")), "diff_attention_backward")
        _check(api.diff_attention_backward(args, q, k, v, lse, dout, (t_rowptr, t_row, t_edge), dq, dk, dv, dlam, ws, on.stream),
               "diff_attention_backward")
    return dq, dk, dv, dlam


def _transpose_cuda(rowptr, colidx, n):
    api._pattern_bits(rowptr, colidx)
    nnz = colidx.shape[0]
    with _On(rowptr.device) as on:
        ws = on.scratch(api.csr_transpose_workspace(rowptr.shape[0] - 1, n, nnz), "csr_transpose")
        t_rowptr, t_row, t_edge = on.empty(n + 1, rowptr.dtype), on.empty(nnz, torch.int32), on.empty(nnz, torch.int32)
        _check(api.csr_transpose(rowptr, colidx, n, t_rowptr, t_row, t_edge, ws, on.stream), "csr_transpose")
    return t_rowptr, t_row, t_edge


def _dense_rows(t):
    """A gradient whose last axis is not dense, or whose rows coincide (an expanded one), is laid out anew."""
    stride = t.stride()
    return t if stride[-1] == 1 and stride[0] != 0 and stride[1] != 0 else t.contiguous()


# (names of this module: looking them up in torch's takes as long as the calls)
_is_compiling, _is_tracing = torch.compiler.is_compiling, torch._C._is_tracing
_dispatch_modes, _function_modes = torch._C._len_torch_dispatch_stack, torch._C._len_torch_function_stack
_transforms, _Tensor, _Parameter = torch._C._functorch.peek_interpreter_stack, torch.Tensor, torch.nn.Parameter


def _plain(*tensors):
    """True if these are ordinary CUDA tensors (none that stores its numbers negated) and nothing watches torch's operators:
    the call may then go straight to the library, without a round through the dispatcher (some 30 us)."""
    if _is_compiling() or _dispatch_modes() or _function_modes():
        return False
    # under an open level of forward mode tensors may have a tangent, which the dispatcher refuses; a trace records operators
    if forward_ad._current_level >= 0 or _is_tracing() or _transforms() is not None:
        return False
    for t in tensors:
        if t is not None and ((type(t) is not _Tensor and type(t) is not _Parameter) or not t.is_cuda or t.is_neg()):
            return False
    return True


def _below(op, *args):
    """A call of an operator from its own autograd layer."""
    with torch._C._AutoDispatchBelowAutograd():
        return op(*args)


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, pos, freq, q_weight, k_weight, eps, interleaved):
        ctx.save_for_backward(q, k, pos, freq, q_weight, k_weight)
        ctx.args = eps, interleaved
        args = (q, k, pos, freq, q_weight, k_weight, eps, interleaved)
        return _rotary_cuda(*args) if _plain(*args[:6]) else _below(torch.ops.fusedmm_b200.qk_norm_rotary, *args)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dq_out, dk_out):
        q, k, pos, freq, q_weight, k_weight = ctx.saved_tensors
        need = ctx.needs_input_grad
        if need[2] or need[3]:
            raise api.FusedMMError("qk_norm_rotary has no gradient for pos and freq")
        eps, interleaved = ctx.args
        plain = _plain(q, k, pos, freq, q_weight, k_weight, dq_out, dk_out)
        run = _rotary_backward_cuda if plain else torch.ops.fusedmm_b200.qk_norm_rotary_backward
        dq, dk, dwq, dwk = run(q, k, pos, freq, q_weight, k_weight, eps, interleaved, _dense_rows(dq_out),
                               None if k is None else _dense_rows(dk_out))
        return (dq if need[0] else None, dk if need[1] else None, None, None, dwq.to(q_weight.dtype) if need[4] else None,
                dwk.to(k_weight.dtype) if need[5] else None, None, None)


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rowptr, colidx, bias, q, k, v, lam, scale, t_rowptr, t_row, t_edge):
        if _plain(rowptr, colidx, bias, q, k, v, lam):
            out, lse = _attention_forward(rowptr, colidx, bias, q, k, v, lam, scale, True)
        else:
            out, lse = _below(torch.ops.fusedmm_b200.diff_attention, rowptr, colidx, bias, q, k, v, lam, scale, t_rowptr, t_row, t_edge)
        ctx.save_for_backward(rowptr, colidx, bias, q, k, v, lam, lse, t_rowptr, t_row, t_edge)
        ctx.scale = scale
        ctx.mark_non_differentiable(lse)
        return out, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, _):
        rowptr, colidx, bias, q, k, v, lam, lse, t_rowptr, t_row, t_edge = ctx.saved_tensors
        need = ctx.needs_input_grad
        if need[2]:
            raise api.FusedMMError("diff_attention has no gradient for bias")
        plain = _plain(rowptr, colidx, bias, q, k, v, lam, lse, dout, t_rowptr, t_row, t_edge)
        if t_rowptr is None:
            t_rowptr, t_row, t_edge = (_transpose_cuda if plain else torch.ops.fusedmm_b200.csr_transpose)(rowptr, colidx, k.shape[0])
        run = _attention_backward_cuda if plain else torch.ops.fusedmm_b200.diff_attention_backward
        grads = run(rowptr, colidx, bias, q, k, v, lam, ctx.scale, lse, _dense_rows(dout), t_rowptr, t_row, t_edge)
        return (None, None, None, *[g if n else None for g, n in zip(grads, need[3:7])], None, None, None, None)


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
    args = (q, k, pos, freq, q_weight, k_weight, eps, interleaved)
    if not _plain(q, k, pos, freq, q_weight, k_weight):
        q_out, k_out = torch.ops.fusedmm_b200.qk_norm_rotary(*args)
    elif torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, pos, freq, q_weight, k_weight)):
        q_out, k_out = _Rotary.apply(*args)
    else:
        q_out, k_out = _rotary_cuda(*args)
    return q_out if k is None else (q_out, k_out)


def diff_attention(rowptr, colidx, q, k, v, lam, *, bias=None, scale=None, transposed=None, return_lse=False):
    """Differential attention over the edges of a CSR; differentiable in q, k, v and lam.

    ``q`` [m, heads, 2, d], ``k`` [n, kv_heads, 2, d], ``v`` [n, kv_heads, dv], ``lam`` [heads] or [m, heads] (float32):
    for each row the softmax maps of the two parts over its edges are formed, the second times ``lam`` is taken from the
    first, and the rows of ``v`` are summed with the differences: [m, heads, dv].  ``colidx`` lists rows of k and v (nodes,
    or the slots of a cache); an id outside [0, n) or a ``bias`` of -inf drops the edge; rows without edges give zeros.
    ``scale`` is 1/sqrt(d) if left out.  ``transposed``: what :func:`csr_transpose` made of this pattern; without it a
    backward pass makes it again.  With ``return_lse`` also the logarithms of the maps' sums, [m, heads, 2] (no gradient)."""
    t = (None, None, None) if transposed is None else transposed
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    if not _plain(rowptr, colidx, bias, q, k, v, lam, *t):
        out, lse = torch.ops.fusedmm_b200.diff_attention(rowptr, colidx, bias, q, k, v, lam, scale, *t)
    elif torch.is_grad_enabled() and any(x is not None and x.requires_grad for x in (q, k, v, lam, bias)):
        out, lse = _Attention.apply(rowptr, colidx, bias, q, k, v, lam, scale, *t)
    else:
        out, lse = _attention_forward(rowptr, colidx, bias, q, k, v, lam, scale, return_lse)
    return (out, lse) if return_lse else out


def csr_transpose(rowptr, colidx, n):
    """The transposed pattern of a CSR with ``n`` columns: row pointers of the columns, the rows of their edges and the
    edges' positions in ``colidx`` (edges outside [0, n) left out).  What ``diff_attention(transposed=...)`` takes."""
    return _transpose_cuda(rowptr, colidx, n) if _plain(rowptr, colidx) else torch.ops.fusedmm_b200.csr_transpose(rowptr, colidx, n)
