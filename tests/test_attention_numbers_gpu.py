"""Differential attention where 32 bits are few: scores of a mask's size, values with a mean, one edge far above the others.
Against plain evaluations in 64 bits."""
import math

import pytest
import torch

from attention_cases import HALF_STEP, HALF_SUBNORMAL, attention_reference, check
from fusedmm_b200 import torch_op

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def rows_of(lengths, n, gen):
    rowptr = torch.zeros(len(lengths) + 1, dtype=torch.int64)
    rowptr[1:] = torch.cumsum(torch.tensor(lengths), 0)
    return rowptr, torch.randint(0, n, (int(rowptr[-1]),), generator=gen, dtype=torch.int32)


def gradients(rowptr, colidx, bias, q, k, v, lam, scale, dout):
    leaves = [x.cuda().requires_grad_() for x in (q, k, v, lam)]
    out = torch_op.diff_attention(rowptr.cuda(), colidx.cuda(), *leaves, bias=None if bias is None else bias.cuda(), scale=scale)
    return dict(zip(("out", "dq", "dk", "dv", "dlam"), (out, *torch.autograd.grad(out, leaves, dout.cuda()))))


SHAPES = [(F32, 4, 2, 32, 64), (F32, 4, 1, 8, 16), (F32, 3, 3, 5, 7), (BF16, 8, 2, 64, 128), (BF16, 4, 4, 16, 32), (BF16, 3, 1, 33, 20),
          (BF16, 2, 2, 128, 256), (F16, 6, 3, 20, 36), (F16, 2, 1, 64, 128)]
LENGTHS = {"few long rows": [1, 3, 700, 0, 5000], "many short rows": [1, 2, 30, 0, 9, 17] * 400}


@pytest.mark.parametrize("lengths", LENGTHS)
@pytest.mark.parametrize("mask", [-1e9, torch.finfo(F32).min])
@pytest.mark.parametrize("dtype,heads,kvh,d,dv", SHAPES)
def test_rows_whose_edges_all_carry_a_finite_mask(cuda_device, dtype, heads, kvh, d, dv, mask, lengths):
    """A finite mask on all of a row's edges leaves equal weights, in the gradients too: next to it the products (below 32) and
    the logarithm of the sum vanish (32-bit numbers near 1e9 are 64 apart).  Zero queries, or zero keys, without a mask give the
    same weights, so the gradients are the 64-bit evaluation's of those: dk's with zero keys, the others' with zero queries."""
    gen = torch.Generator().manual_seed(d)
    n = 90
    rowptr, colidx = rows_of(LENGTHS[lengths], n, gen)
    m = len(rowptr) - 1
    q, k, v, dout = (torch.randn(s, generator=gen).to(dtype) for s in ((m, heads, 2, d), (n, kvh, 2, d), (n, kvh, dv), (m, heads, dv)))
    lam, bias, scale = torch.rand(m, heads, generator=gen), torch.full((colidx.numel(),), mask), d ** -0.5
    got = gradients(rowptr, colidx, bias, q, k, v, lam, scale, dout)
    want = attention_reference(rowptr, colidx, None, torch.zeros_like(q), k, v, lam, scale, dout)
    want["dk"] = attention_reference(rowptr, colidx, None, q, torch.zeros_like(k), v, lam, scale, dout)["dk"]
    for name in got:
        check(got[name], want[name], name)


@pytest.mark.parametrize("mask", [-3e4, -1e6])
@pytest.mark.parametrize("dtype,heads,kvh,d,dv", [(F32, 2, 1, 16, 32), (BF16, 2, 1, 16, 32), (F16, 2, 1, 16, 32)])
def test_weights_of_masked_rows_add_up(cuda_device, dtype, heads, kvh, d, dv, mask):
    """With scores of some thousands the log-sum keeps few digits; each map's weights still add up to 1: with dout and v of ones
    dP is dv on every edge, so dlam is -dv, dq is 0 and the sum of dv over the columns (1 - lam) for every row."""
    gen = torch.Generator().manual_seed(1)
    m, n = 300, 50
    rowptr, colidx = rows_of([7, 100, 33] * (m // 3), n, gen)
    q, k = (torch.randn(s, generator=gen).to(dtype) for s in ((m, heads, 2, d), (n, kvh, 2, d)))
    v, dout, lam = torch.ones(n, kvh, dv, dtype=dtype), torch.ones(m, heads, dv, dtype=dtype), torch.full((m, heads), 0.25)
    got = gradients(rowptr, colidx, torch.full((colidx.numel(),), mask), q, k, v, lam, 0.25, dout)
    # sums of up to 100 positive terms and a division by another: 2 (100 + 8) steps of 2^-23; dq: weights split to 16 bits
    assert float((got["dlam"] + dv).abs().max()) <= dv * 216 * 2.0 ** -23
    assert float(got["dq"].abs().max()) <= 0.25 * dv * 4 * (216 * 2.0 ** -23 + 2.0 ** -16)
    # dv: a column's sum of p is rounded to the type
    total = got["dv"].double().sum((0, 1))
    assert float((total - m * heads * 0.75).abs().max()) <= m * heads * 0.75 * (2 * HALF_STEP[dtype] + 216 * 2.0 ** -23 + 2.0 ** -16)


@pytest.mark.parametrize("lengths", ["one row", "rows", "long row"])
@pytest.mark.parametrize("gap", [5, 10, 14, 17, 18, 24])
@pytest.mark.parametrize("dtype,heads,kvh,d,dv", [(F16, 8, 2, 64, 128), (F16, 4, 4, 16, 32), (F16, 3, 1, 20, 36), (F16, 2, 1, 128, 256), (BF16, 8, 2, 64, 128),
                                                  (F32, 4, 2, 32, 64)])
def test_a_first_edge_far_above_the_others(cuda_device, dtype, heads, kvh, d, dv, gap, lengths):
    """The edge with the largest score has a value of zero, so the result is what the small weights bring."""
    gen = torch.Generator().manual_seed(gap)
    n = 3000
    rowptr, colidx = rows_of({"one row": [1000], "rows": [250] * 700, "long row": [100000]}[lengths], n, gen)
    m = len(rowptr) - 1
    colidx[colidx == 0] = 1
    colidx[rowptr[:-1]] = 0
    bias = torch.zeros(colidx.numel())
    bias[rowptr[:-1]] = gap
    q, k = ((0.3 * torch.randn(s, generator=gen)).to(dtype) for s in ((m, heads, 2, d), (n, kvh, 2, d)))
    v = (1 + 0.1 * torch.randn(n, kvh, dv, generator=gen)).to(dtype)
    v[0] = 0
    lam = torch.full((heads,), 0.25)
    out = torch_op.diff_attention(*(x.cuda() for x in (rowptr, colidx, q, k, v, lam)), bias=bias.cuda(), scale=0.1)
    value, bound = attention_reference(rowptr, colidx, bias, q, k, v, lam, 0.1)["out"]
    # beside the bound of large weights: half's weights lie on a grid of 2^-44 of the row's largest at worst
    grid = 2.0 ** -45 * 1.25 * 1.5 * (rowptr[1:] - rowptr[:-1])[:, None, None] if dtype == F16 else 0
    check(out, (value, bound + grid))


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("base,gap", [(1e8, 8), (-1e8, 8), (3e7, 6), (3e7, 4), (1e6, 5.5), (0, 5)])
def test_a_later_edge_a_little_above_the_others(cuda_device, dtype, base, gap):
    """Scores whose 32-bit neighbours are 8, 2 and 1/16 apart: the edge above the others comes late in its row, after sums were
    taken against a smaller maximum.  Zero queries: the scores are the biases, exactly."""
    gen = torch.Generator().manual_seed(3)
    rowptr, colidx = rows_of([200, 1, 777, 90], 60, gen)
    q, k, v = torch.zeros(4, 4, 2, 16, dtype=dtype), torch.randn(60, 2, 2, 16, generator=gen).to(dtype), torch.randn(60, 2, 32, generator=gen).to(dtype)
    bias, lam = torch.full((colidx.numel(),), float(base)), torch.full((4,), 0.25)
    bias[rowptr[1:] - 1] += gap
    assert bool((bias[rowptr[1:] - 1] - base == gap).all())
    out = torch_op.diff_attention(*(x.cuda() for x in (rowptr, colidx, q, k, v, lam)), bias=bias.cuda())
    check(out, attention_reference(rowptr, colidx, bias - base, q, k, v, lam, 0.25)["out"])


@pytest.mark.parametrize("dtype,low,high,degree,heads,kvh,d,dv", [
    (F32, 1e5, 1e5 + 1, 60, 4, 2, 32, 64), (F32, 1e5, 1e5 + 1, 2500, 2, 1, 8, 16), (F32, 1e5, 1e5 + 1, 13, 3, 3, 5, 7),
    (BF16, 256, 258, 53, 8, 2, 64, 128), (BF16, 256, 258, 53, 4, 4, 16, 32), (BF16, 256, 258, 53, 4, 1, 128, 256), (BF16, 256, 258, 1700, 2, 1, 32, 64),
    (F16, 2000, 2001, 60, 4, 2, 32, 64), (F16, 2000, 2001, 60, 3, 1, 33, 20),
])
def test_gradient_of_queries_where_values_have_a_mean(cuda_device, dtype, low, high, degree, heads, kvh, d, dv):
    """dq is a sum of p (dP - D) k: what it loses must go by the differences of dP and not by dP.  All scores are equal (zero
    queries), dout has a single one, so p and dP are known and the bound can be close."""
    gen = torch.Generator().manual_seed(degree)
    m, n = (40, 70) if degree < 1000 else (3, 500)
    rowptr, colidx = rows_of([degree] * m, n, gen)
    q, k = torch.zeros(m, heads, 2, d, dtype=dtype), (1 + torch.rand(n, kvh, 2, d, generator=gen)).to(dtype)
    v = torch.where(torch.rand(n, kvh, dv, generator=gen) < 0.5, low, high).to(dtype)
    dout = torch.zeros(m, heads, dv, dtype=dtype)
    dout[..., dv // 2] = 1
    lam, scale = torch.full((m, heads), 0.5), 0.5
    got = gradients(rowptr, colidx, None, q, k, v, lam, scale, dout)["dq"]
    want = attention_reference(rowptr, colidx, None, q, k, v, lam, scale, dout)["dq"][0]
    half = HALF_STEP[dtype]
    # p = 1/degree up to a factor that all edges share; p (dP - c), with c one of the dP, and p are split (bf16) and summed with
    # k up to 2; then (D - c) times the sum of p k: four terms of at most (high - low) 2
    step, split = (2.0 ** -23, 2.0 ** -16) if dtype == BF16 else (2.0 ** -24, 0)
    slack = scale * 4 * (high - low) * 2 * (split + (degree + 16) * step)
    check(got, (want, half * want.abs() + (1 + half) * slack))


@pytest.mark.parametrize("lengths", ["one row", "rows", "long row"])
@pytest.mark.parametrize("gap", [6, 10, 14])
@pytest.mark.parametrize("dtype,heads,kvh,d,dv", [(F32, 4, 2, 32, 64), (F32, 3, 3, 5, 7), (BF16, 8, 2, 64, 128), (BF16, 4, 4, 16, 32), (BF16, 2, 1, 32, 64),
                                                  (BF16, 2, 2, 128, 256), (F16, 4, 2, 32, 64)])
def test_gradient_of_queries_where_one_edge_has_nearly_all_the_weight(cuda_device, dtype, heads, kvh, d, dv, gap, lengths):
    """dq = sum of p (dP - D) k is small there, since D is nearly the dP of the heavy edge, and must keep its digits.

    dq is the covariance of dP and k under p.  To first order an error e_p of p (relative) brings p e_p (dP - D) (k - K), K the sum
    of p k, and one of dP brings p e_dP (k - K).  The sums of p (dP - c) k and p k are rounded (split in bf16) relative to their
    terms; c is some dP (R from D at most) until the heavy edge comes, and then within 2 W of D, W = sum p |dP - D|."""
    gen = torch.Generator().manual_seed(gap + d)
    n = 400
    rowptr, colidx = rows_of({"one row": [1000], "rows": [250] * 300, "long row": [20000]}[lengths], n, gen)
    m = len(rowptr) - 1
    at = rowptr[:-1] + (torch.rand(m, generator=gen) * (rowptr[1:] - rowptr[:-1])).long()
    bias = torch.zeros(colidx.numel())
    bias[at] = gap + math.log(int(rowptr[1]) / 250)
    q, k = ((0.3 * torch.randn(s, generator=gen)).to(dtype) for s in ((m, heads, 2, d), (n, kvh, 2, d)))
    v = torch.randn(n, kvh, dv, generator=gen).to(dtype)
    dout = (torch.randn(m, heads, dv, generator=gen) * (64 if dtype == F16 else 1)).to(dtype)
    lam, scale = torch.full((m, heads), 0.5), d ** -0.5
    got = gradients(rowptr, colidx, bias, q, k, v, lam, scale, dout)["dq"].detach().cpu().double()
    step, split, half = (2.0 ** -24, 0, HALF_STEP[dtype]) if dtype != BF16 else (2.0 ** -23, 2.0 ** -16, HALF_STEP[dtype])
    tiny = HALF_SUBNORMAL[dtype] + 1e-30
    kv = torch.arange(heads) // (heads // kvh)
    for u in range(0, m, max(1, m // 7)):
        e = torch.arange(int(rowptr[u]), int(rowptr[u + 1]))
        ke, ve, qu, du = k.double()[colidx[e].long()][:, kv], v.double()[colidx[e].long()][:, kv], q[u].double(), dout[u].double()
        score = scale * (ke * qu).sum(-1) + bias[e].double()[:, None, None]
        p = torch.softmax(score, 0)
        dp, dpabs = (ve * du).sum(-1)[..., None], (ve.abs() * du.abs()).sum(-1)[..., None]
        off = dp - (p * dp).sum(0)
        factor = scale * torch.tensor([1.0, -0.5], dtype=torch.float64)[:, None]
        want = factor * (p[..., None] * off[..., None] * ke).sum(0)
        away, wide = (ke - (p[..., None] * ke).sum(0)).abs(), off.abs().amax(0)
        mean_off = (p * off.abs()).sum(0)
        of_p = 2 * step * (16 + (d + 2) * scale * (ke.abs() * qu.abs()).sum(-1) + 2 * score.abs())
        heavy = (e == at[u])[:, None, None]
        sums = (p[..., None] * torch.where(heavy, 2 * mean_off, 2 * wide)[..., None] * ke.abs()).sum(0) + 2 * mean_off[..., None] * (p[..., None] * ke.abs()).sum(0)
        slack = factor.abs() * ((p * of_p)[..., None] * off.abs()[..., None] * away + (p * step * (dv + 2) * dpabs)[..., None] * away).sum(0)
        slack = slack + factor.abs() * (2 * split + step * (len(e) + 32)) * sums
        check(got[u], (want, half * want.abs() + (1 + half) * slack + tiny), "dq")
