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


@pytest.mark.parametrize("dtype", [BF16, F32, F16])
def test_heads_of_a_cache_far_apart(cuda_device, dtype):
    """A [kv heads, slots, ...] cache seen through a transposed view, its heads 2^31 bytes apart; queries, weights and the result's
    gradient likewise.  The results are those of dense copies, bit for bit."""
    gen = torch.Generator().manual_seed(2)
    m, n, heads, kvh, d, dv = 4, 30, 4, 2, 16, 32
    wide = (1 << 31) // dtype.itemsize + 64
    base = torch.empty(3 * wide + 65536, dtype=dtype, device="cuda")
    rowptr, colidx = torch.tensor([0, 20, 20, 25, 700]).cuda(), torch.randint(0, n, (700,), generator=gen, dtype=torch.int32).cuda()
    q = spread(gen, dtype, (m, heads, 2, d), (2 * d, wide, d, 1), base)
    k = spread(gen, dtype, (n, kvh, 2, d), (2 * d, wide, d, 1), base[8192:])
    v = spread(gen, dtype, (n, kvh, dv), (dv, wide, 1), base[16384:])
    dout = spread(gen, dtype, (m, heads, dv), (dv, wide, 1), base[32768:])
    lam = spread(gen, F32, (m, heads), (heads, 1), torch.empty(64, device="cuda"))
    assert k.stride(1) * dtype.itemsize > 1 << 31
    results = []
    for dense in (False, True):
        leaves = [(x.contiguous() if dense else x).detach().requires_grad_() for x in (q, k, v, lam)]
        out = torch_op.diff_attention(rowptr, colidx, *leaves)
        results.append((out, *torch.autograd.grad(out, leaves, dout.contiguous() if dense else dout)))
    for a, b in zip(*results):
        assert torch.equal(a, b)


def test_rows_far_apart(cuda_device):
    """Rows of queries and weights may be 2^31 bytes apart in the forward pass, and so may gathered rows that are packed first."""
    gen = torch.Generator().manual_seed(3)
    heads, kvh, d, dv = 4, 2, 16, 32
    wide = (1 << 31) // 2 + 64
    base = torch.empty(2 * wide + 65536, dtype=BF16, device="cuda")
    rowptr, colidx = torch.tensor([0, 5, 9]).cuda(), torch.randint(0, 3, (9,), generator=gen, dtype=torch.int32).cuda()
    q = spread(gen, BF16, (2, heads, 2, d), (wide, 2 * d, d, 1), base)
    k = spread(gen, BF16, (3, kvh, 2, d), (2 * d * kvh, 2 * d, d, 1), base[8192:])
    v = spread(gen, BF16, (3, kvh, dv), (kvh * dv, dv, 1), base[16384:])
    lam = spread(gen, F32, (2, heads), (wide, 1), torch.empty(wide + 64, device="cuda"))
    assert torch.equal(torch_op.diff_attention(rowptr, colidx, q, k, v, lam), torch_op.diff_attention(rowptr, colidx, q.contiguous(), k, v, lam.contiguous()))
    far = spread(gen, BF16, (3, kvh, 2, d), (wide, 2 * d, d, 1), base[32768:])
    with pytest.raises(api.FusedMMError, match="limit|-4"):
        torch_op.diff_attention(rowptr, colidx, q, far, v, lam)
    odd, q = spread(gen, BF16, (3, kvh, 2, 7), (wide, 14, 7, 1), base[32768:]), spread(gen, BF16, (2, heads, 2, 7), (wide, 14, 7, 1), base)
    assert torch.equal(torch_op.diff_attention(rowptr, colidx, q, odd, v, lam), torch_op.diff_attention(rowptr, colidx, q.contiguous(), odd.contiguous(), v, lam))


@pytest.mark.parametrize("dtype,kvh,d,dv,n", [(BF16, 2, 64, 128, 9_000_000), (F32, 1, 32, 64, 18_000_000), (BF16, 1, 60, 120, 19_000_000)])
def test_offsets_beyond_32_bits_in_a_long_cache(cuda_device, dtype, kvh, d, dv, n):
    """Slots behind 2^32 bytes (and elements' counts behind 2^31) of a cache give what dense copies of them give."""
    gen = torch.Generator().manual_seed(5)
    heads, length = 2 * kvh, 600
    ids = torch.cat((torch.tensor([0, n - 1]), torch.randint(n // 2, n, (length,), generator=gen))).unique().int()[torch.randperm(400, generator=gen)]
    rowptr = torch.tensor([0, 150, 400]).cuda()
    small = [torch.randn(400, kvh, 2, d, generator=gen).to(dtype).cuda(), torch.randn(400, kvh, dv, generator=gen).to(dtype).cuda()]
    large = [torch.empty(n, *x.shape[1:], dtype=dtype, device="cuda") for x in small]
    assert large[0].nbytes > 1 << 32 and large[1].nbytes > 1 << 32
    for x, y in zip(large, small):
        x[ids.long().cuda()] = y
    q, dout, lam = torch.randn(2, heads, 2, d, generator=gen).to(dtype).cuda(), torch.randn(2, heads, dv, generator=gen).to(dtype).cuda(), torch.rand(heads, generator=gen).cuda()
    results = []
    for kv, colidx in ((small, torch.arange(400, dtype=torch.int32)), (large, ids)):
        leaves = [x.detach().requires_grad_() for x in (q, *kv, lam)]
        out = torch_op.diff_attention(rowptr, colidx.cuda(), *leaves)
        dq, dk, dvv, dlam = torch.autograd.grad(out, leaves, dout)
        at = colidx.long().cuda()
        assert bool(dk[at].any()) and int(torch.count_nonzero(dk[-1])) == int(torch.count_nonzero(dk[at[colidx == len(dk) - 1]]))
        results.append((out, dq, dk[at], dvv[at], dlam))
        del leaves, dk, dvv
    for a, b in zip(*results):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype,rows,heads,d", [(BF16, 2_200_000, 8, 128), (F32, 1_100_000, 9, 130)])
def test_rotation_beyond_32_bits(cuda_device, dtype, rows, heads, d):
    """The last rows of more than 2^31 elements and 2^32 bytes."""
    gen = torch.Generator().manual_seed(6)
    x = torch.empty(rows, heads, d, dtype=dtype, device="cuda")
    assert x.numel() * dtype.itemsize > 1 << 32
    x.zero_()
    last = torch.randn(3, heads, d, generator=gen).to(dtype).cuda()
    x[-3:] = last
    pos, freq, w = torch.arange(rows, device="cuda"), torch.rand(1, 32, generator=gen, dtype=torch.float64).cuda(), torch.rand(d, generator=gen).cuda()
    results = []
    for a, p in ((x, pos), (last, pos[-3:])):
        a, ww = a.detach().requires_grad_(), w.detach().requires_grad_()
        y = torch_op.qk_norm_rotary(a, None, p, freq, q_weight=ww, eps=1e-6)
        (dx,) = torch.autograd.grad(y, a, torch.ones_like(y))
        results.append((y[-3:].clone(), dx[-3:].clone()))
        del y, dx
    for a, b in zip(*results):
        assert torch.equal(a, b)
