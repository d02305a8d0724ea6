"""Calls of the attention operators that torch records, transforms or compiles, run on the GPU."""
import pytest
import torch
from torch.autograd import forward_ad

from attention_cases import random_pattern
from fusedmm_b200 import torch_op

pytestmark = pytest.mark.gpu


def layer_inputs(dtype=torch.bfloat16):
    gen = torch.Generator().manual_seed(4)
    rowptr, colidx = (x.cuda() for x in random_pattern(gen, 30, 30, 6))
    x, k = (torch.randn(s, generator=gen).to(dtype).cuda() for s in ((30, 8, 16), (30, 4, 16)))
    v, lam, w = torch.randn(30, 2, 32, generator=gen).to(dtype).cuda(), torch.rand(4, generator=gen).cuda(), torch.rand(16, generator=gen).cuda()
    pos, freq = torch.arange(30).cuda(), torch.rand(1, 8, generator=gen, dtype=torch.float64).cuda()

    def layer(x, k, v, lam, w):
        q, k = torch_op.qk_norm_rotary(x, k, pos, freq, q_weight=w, k_weight=w, eps=1e-6)
        return torch_op.diff_attention(rowptr, colidx, q.view(30, 4, 2, 16), k.view(30, 2, 2, 16), v, lam)

    return layer, (x, k, v, lam, w)


def test_a_traced_layer_computes(cuda_device):
    layer, args = layer_inputs()
    traced = torch.jit.trace(layer, args, check_trace=False)
    other = [a.flip(0).contiguous() for a in args]
    assert torch.equal(traced(*args), layer(*args)) and torch.equal(traced(*other), layer(*other))


def test_a_compiled_layer_computes_and_trains(cuda_device):
    layer, args = layer_inputs()
    compiled = torch.compile(layer, backend="aot_eager", fullgraph=True)
    grads = []
    for fn in (layer, compiled):
        leaves = [a.detach().requires_grad_() for a in args]
        out = fn(*leaves)
        grads.append((out, *torch.autograd.grad(out, leaves, torch.ones_like(out))))
    for a, b in zip(*grads):
        assert torch.equal(a, b)
    with torch.no_grad():
        assert torch.equal(compiled(*args), layer(*args))


def test_tangents_are_refused(cuda_device):
    layer, args = layer_inputs()
    for i in range(len(args)):
        with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="jvp"):
            layer(*(forward_ad.make_dual(a, torch.ones_like(a)) if i == j else a for j, a in enumerate(args)))


def test_positions_of_mirrored_points(cuda_device):
    """The coordinates of conjugate points: views that store their numbers negated."""
    z = torch.randn(50, dtype=torch.complex64, device="cuda")
    x, freq = torch.randn(50, 2, 16, device="cuda", requires_grad=True), torch.rand(1, 8, dtype=torch.float64, device="cuda")
    results = []
    for pos in (z.conj().imag, (-z.imag).contiguous()):
        y = torch_op.qk_norm_rotary(x, None, pos, freq)
        results.append((y, *torch.autograd.grad(y, x, torch.ones_like(y)), torch_op.qk_norm_rotary(x.detach(), None, pos, freq)))
    for a, b in zip(*results):
        assert torch.equal(a, b)
