"""Differential attention with the largest head counts and strides."""
import pytest
import torch

from attention_cases import attention_reference, check
from fusedmm_b200 import api, torch_op

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def test_workspace_at_the_largest_head_counts(cuda_device):
    """One piece of the work has parts above the soft limit of the scratch: the size is what it must be."""
    fn = api._attn_fn("diff_attention_workspace", api._l, api._i, api._i, api._i, api._l, api._l, api._l, api._i, api._i, api._i, api._i)
    for dtype in (0, 2, 3):
        for heads, kvh in ((4097, 4097), (29128, 29128), (65536, 65536), (65536, 1), (65535, 1)):
            for d, dv in ((128, 256), (64, 128), (1, 1), (33, 200)):
                for m, n, nnz in ((1, 1, 1), (4, 6, 20), (3000, 50, 100000), (1 << 31, 7, 1 << 33)):
                    forward = fn(0, 1, dtype, m, n, nnz, heads, kvh, d, dv)
                    backward = fn(1, 0, dtype, m, n, nnz, heads, kvh, d, dv)
                    assert 0 < forward < 1 << 40 and backward >= m * heads * 36, (dtype, heads, kvh, d, dv, m, n, nnz)


@pytest.mark.parametrize("dtype,heads,kvh,d,dv", [(BF16, 4097, 4097, 128, 256), (F32, 29128, 29128, 128, 130), (BF16, 65536, 1, 64, 128), (F16, 7711, 7711, 128, 256)])
def test_many_heads(cuda_device, dtype, heads, kvh, d, dv):
    gen = torch.Generator().manual_seed(heads)
    m, n = 2, 3
    rowptr, colidx = torch.tensor([0, 1, 4]), torch.tensor([2, 0, 2, 1], dtype=torch.int32)
    q, k, v, dout = (torch.randn(s, generator=gen).to(dtype) for s in ((m, heads, 2, d), (n, kvh, 2, d), (n, kvh, dv), (m, heads, dv)))
    lam = torch.rand(heads, generator=gen)
    leaves = [x.cuda().requires_grad_() for x in (q, k, v, lam)]
    out = torch_op.diff_attention(rowptr.cuda(), colidx.cuda(), *leaves)
    grads = torch.autograd.grad(out, leaves, dout.cuda())
    want = attention_reference(rowptr, colidx, None, q, k, v, lam, d ** -0.5, dout)
    for name, got in zip(("out", "dq", "dk", "dv", "dlam"), (out, *grads)):
        check(got, want[name], name)


def spread(gen, dtype, shape, strides, base):
    """A tensor of ``shape`` on the GPU with these strides, over ``base``."""
    x = torch.as_strided(base, shape, strides)
    x.copy_(torch.randn(shape, generator=gen).to(dtype))
    return x


@pytest.mark.parametrize("rows,heads,far", [(2, 3, "rows"), (3, 2, "heads")])
def test_rotation_of_rows_and_heads_far_apart(cuda_device, rows, heads, far):
    """Strides of 2^31 bytes and more; the results are those of dense copies, bit for bit."""
    gen = torch.Generator().manual_seed(1)
    d, wide = 64, (1 << 30) + 8
    strides = (wide, 2 * d, 1) if far == "rows" else (2 * d, wide, 1)
    base = [torch.empty(2 * wide + 1024, dtype=BF16, device="cuda") for _ in range(2)]
    q = spread(gen, BF16, (rows, heads, d), strides, base[0])
    k = spread(gen, BF16, (rows, heads, d), strides, base[0][d:])
    dy = spread(gen, BF16, (rows, heads, d), strides, base[1])
    pos, freq = torch.arange(rows, device="cuda") * 1000, torch.rand(1, 32, generator=gen, dtype=torch.float64).cuda()
    w = torch.rand(d, generator=gen).cuda()
    results = []
    for dense in (False, True):
        leaves = [x.contiguous() if dense else x for x in (q, k)]
        leaves = [x.detach().requires_grad_() for x in leaves] + [w.detach().requires_grad_()]
        y = torch_op.qk_norm_rotary(leaves[0], leaves[1], pos, freq, q_weight=leaves[2], k_weight=leaves[2], eps=1e-6)
        g = dy.contiguous() if dense else dy
        results.append((*y, *torch.autograd.grad(y, leaves, (g, g))))
    for a, b in zip(*results):
        assert torch.equal(a, b)
