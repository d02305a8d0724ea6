"""Differential attention over CSR edges, the norm and rotation before it, and the transposed pattern, on the GPU against
plain evaluations in 64 bits."""
import math

import pytest
import torch

from attention_cases import HALF_STEP, attention_reference, check, random_pattern, rotary_reference
from fusedmm_b200 import api, torch_op

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def gen_of(seed):
    return torch.Generator().manual_seed(seed)


def randn(gen, dtype, *shape):
    return torch.randn(shape, generator=gen).to(dtype)


def make(gen, dtype, rowptr, colidx, m, n, heads, kvh, d, dv, bias=False, row_lam=False):
    t = dict(rowptr=rowptr, colidx=colidx, q=randn(gen, dtype, m, heads, 2, d), k=randn(gen, dtype, n, kvh, 2, d),
             v=randn(gen, dtype, n, kvh, dv), lam=torch.rand((m, heads) if row_lam else (heads,), generator=gen) - 0.2,
             bias=None)
    if bias:
        t["bias"] = randn(gen, F32, colidx.numel())
        t["bias"][torch.rand(colidx.numel(), generator=gen) < 0.15] = -math.inf
    return {a: None if x is None else x.cuda() for a, x in t.items()}


def run_all(t, scale, dout, transposed=None):
    leaves = [t[a].detach().requires_grad_() for a in ("q", "k", "v", "lam")]
    out, lse = torch_op.diff_attention(t["rowptr"], t["colidx"], *leaves, bias=t["bias"], scale=scale, transposed=transposed,
                                       return_lse=True)
    grads = torch.autograd.grad(out, leaves, dout)
    return dict(out=out, lse=lse, dq=grads[0], dk=grads[1], dv=grads[2], dlam=grads[3])


def compare(t, scale, dout, transposed=None):
    got = run_all(t, scale, dout, transposed)
    want = attention_reference(t["rowptr"], t["colidx"], t["bias"], t["q"], t["k"], t["v"], t["lam"], scale, dout)
    for name in want:
        check(got[name], want[name], name)
    return got


# dtype, m, n, mean degree, hub, heads, kv heads, d, dv, bias, a weight for each row
SHAPES = [
    (F32, 40, 50, 6, 0, 2, 2, 8, 16, False, False),
    (F32, 33, 70, 9, 700, 4, 2, 32, 64, True, False),
    (F32, 21, 30, 5, 0, 4, 1, 128, 256, False, True),
    (F32, 50, 40, 4, 1500, 1, 1, 64, 64, True, True),
    (F32, 30, 31, 7, 0, 3, 3, 5, 7, True, False),
    (F32, 30, 31, 7, 600, 6, 2, 18, 30, False, False),
    (BF16, 64, 90, 8, 900, 8, 2, 64, 128, False, False),
    (BF16, 37, 90, 8, 0, 4, 4, 16, 32, True, True),
    (BF16, 37, 90, 8, 650, 4, 1, 128, 256, True, False),
    (BF16, 37, 90, 8, 600, 2, 2, 32, 64, False, False),
    (BF16, 37, 90, 8, 0, 5, 1, 33, 21, True, False),
    (F16, 64, 90, 8, 600, 6, 3, 64, 128, False, True),
    (F16, 29, 60, 5, 0, 3, 1, 20, 36, True, False),
    (F16, 29, 60, 5, 555, 8, 8, 4, 4, False, False),
    (F16, 29, 60, 5, 0, 2, 1, 128, 1, True, False),
    (F16, 29, 60, 5, 0, 2, 1, 1, 200, True, False),
    (BF16, 41, 60, 6, 600, 8, 1, 64, 64, True, False),     # more query heads of a kv head than a product holds
    (BF16, 41, 60, 6, 600, 6, 2, 32, 64, True, True),      # three query heads: columns left over, three rounds of the columns
    (BF16, 41, 60, 6, 0, 14, 2, 16, 32, False, False),
    (BF16, 41, 60, 6, 600, 4, 2, 128, 256, True, False),
    (BF16, 41, 60, 6, 600, 5, 5, 128, 100, False, False),
    (BF16, 41, 60, 6, 600, 4, 4, 9, 18, True, False),      # packed rows, four kv heads at once
    (F16, 41, 60, 6, 600, 8, 8, 12, 20, True, True),
    (F32, 41, 60, 6, 600, 8, 2, 16, 32, True, False),
    (F32, 41, 60, 6, 600, 2, 2, 4, 4, True, False),
]


@pytest.mark.parametrize("case", range(len(SHAPES)))
def test_attention_and_gradients(cuda_device, case):
    dtype, m, n, mean, hub, heads, kvh, d, dv, bias, row_lam = SHAPES[case]
    gen = gen_of(case)
    ptr, idx = ((torch.int32, torch.int32), (torch.int64, torch.int32), (torch.int64, torch.int64), (torch.int32, torch.int64))[case % 4]
    rowptr, colidx = random_pattern(gen, m, n, mean, ptr, idx, hub)
    t = make(gen, dtype, rowptr, colidx, m, n, heads, kvh, d, dv, bias, row_lam)
    dout = randn(gen, dtype, m, heads, dv).cuda()
    plan = torch_op.csr_transpose(t["rowptr"], t["colidx"], n) if case % 2 else None
    compare(t, d ** -0.5, dout, plan)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("length", [1, 2, 31, 32, 33, 255, 256, 257, 1000, 5003])
def test_single_row(cuda_device, dtype, length):
    """One token over a list of slots: from one slot to lists that are cut over many blocks."""
    gen = gen_of(length)
    n = length + 40
    rowptr = torch.tensor([0, length], dtype=torch.int32)
    colidx = torch.randperm(n, generator=gen)[:length].to(torch.int32)
    t = make(gen, dtype, rowptr, colidx, 1, n, 8, 2, 64, 128)
    compare(t, 0.125, randn(gen, dtype, 1, 8, 128).cuda())


@pytest.mark.parametrize("dtype,d,dv", [(BF16, 33, 47), (F16, 20, 36), (F32, 7, 9)])
@pytest.mark.parametrize("n", [300, 40000])
def test_rows_that_are_no_vectors_of_small_and_large_caches(cuda_device, dtype, d, dv, n):
    """They are packed first: all rows of a small cache, the listed ones of a large one."""
    gen = gen_of(n + d)
    rowptr = torch.tensor([0, 700, 700, 1500], dtype=torch.int32)
    colidx = torch.randint(-1, n + 1, (1500,), generator=gen).to(torch.int64)
    t = make(gen, dtype, rowptr, colidx, 3, n, 4, 2, d, dv, bias=True)
    want = attention_reference(t["rowptr"], t["colidx"], t["bias"], t["q"], t["k"], t["v"], t["lam"], 0.2)
    out, lse = torch_op.diff_attention(t["rowptr"], t["colidx"], t["q"], t["k"], t["v"], t["lam"], bias=t["bias"], scale=0.2, return_lse=True)
    check(out, want["out"], "out")
    check(lse, want["lse"], "lse")


@pytest.mark.parametrize("dtype,heads,kvh,d,dv", [(BF16, 8, 2, 64, 128), (BF16, 4, 4, 128, 256), (F32, 2, 1, 32, 64), (F16, 3, 3, 16, 32)])
def test_one_long_row(cuda_device, dtype, heads, kvh, d, dv):
    """Hundreds of parts joined; the gradients too."""
    gen = gen_of(77)
    n, length = 3000, 60000
    rowptr = torch.tensor([0, 0, length, length + 2], dtype=torch.int64)
    colidx = torch.randint(0, n, (length + 2,), generator=gen, dtype=torch.int32)
    t = make(gen, dtype, rowptr, colidx, 3, n, heads, kvh, d, dv)
    compare(t, d ** -0.5, randn(gen, dtype, 3, heads, dv).cuda())


def test_two_streams_at_once(cuda_device):
    """Calls that run side by side have scratch of their own."""
    gen = gen_of(21)
    rowptr, colidx = random_pattern(gen, 2000, 1500, 20, torch.int64, torch.int32, hub=30000)
    t = make(gen, BF16, rowptr, colidx, 2000, 1500, 8, 2, 64, 128)
    u = make(gen, BF16, rowptr, colidx, 2000, 1500, 8, 2, 64, 128)
    dout = randn(gen, BF16, 2000, 8, 128).cuda()
    want = [run_all(x, 0.125, dout) for x in (t, u)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        got = []
        for s, x in zip(streams, (t, u)):
            with torch.cuda.stream(s):
                got.append(run_all(x, 0.125, dout))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            for name in b:
                assert torch.equal(a[name], b[name]), name


def test_rows_of_very_different_lengths(cuda_device):
    gen = gen_of(5)
    lengths = torch.tensor([0, 1, 3000, 0, 17, 511, 512, 513, 2, 700, 0])
    rowptr = torch.zeros(12, dtype=torch.int64)
    rowptr[1:] = torch.cumsum(lengths, 0)
    colidx = torch.randint(0, 333, (int(rowptr[-1]),), generator=gen, dtype=torch.int32)
    for heads, kvh, d, dv in ((4, 4, 32, 64), (8, 2, 64, 128), (12, 3, 16, 16)):
        t = make(gen, BF16, rowptr, colidx, 11, 333, heads, kvh, d, dv, bias=True, row_lam=True)
        compare(t, 0.2, randn(gen, BF16, 11, heads, dv).cuda())


@pytest.mark.parametrize("dtype,heads,kvh,d,dv", [(BF16, 4, 4, 16, 32), (F32, 2, 2, 8, 16), (F16, 2, 1, 20, 36)])
def test_many_long_rows(cuda_device, dtype, heads, kvh, d, dv):
    """More long rows than there are warps: each warp has rows of its own, cut at its pieces."""
    gen = gen_of(15)
    m, n = 2600, 400
    lengths = torch.randint(60, 700, (m,), generator=gen)
    rowptr = torch.zeros(m + 1, dtype=torch.int64)
    rowptr[1:] = torch.cumsum(lengths, 0)
    colidx = torch.randint(0, n, (int(rowptr[-1]),), generator=gen, dtype=torch.int32)
    t = make(gen, dtype, rowptr, colidx, m, n, heads, kvh, d, dv)
    compare(t, 0.2, randn(gen, dtype, m, heads, dv).cuda())


def test_many_short_rows_and_columns_nobody_asks_for(cuda_device):
    gen = gen_of(6)
    rowptr, colidx = random_pattern(gen, 20000, 100, 2, torch.int64, torch.int32)
    t = make(gen, F32, rowptr, colidx, 20000, 20500, 2, 1, 8, 8)
    got = compare(t, 0.3, randn(gen, F32, 20000, 2, 8).cuda())
    assert not got["dk"][100:].any() and not got["dv"][100:].any()


def test_masked_edges_are_not_read(cuda_device):
    """NaN and infinities in slots that only dropped edges name; ids outside the range; a row whose edges are all dropped."""
    gen = gen_of(7)
    m, n = 9, 40
    rowptr, colidx = random_pattern(gen, m, n, 12, torch.int32, torch.int32, empty=0.0)
    t = make(gen, F32, rowptr, colidx, m, n, 4, 2, 16, 32, bias=True)
    ids = t["colidx"]
    ids[::5] = -1
    ids[3::7] = n
    t["bias"][ids == 11] = -math.inf
    a, b = int(rowptr[4]), int(rowptr[5])
    t["bias"][a:b] = -math.inf
    dout = randn(gen, F32, m, 4, 32).cuda()
    got = compare(t, 0.25, dout)
    assert not got["out"][4].any() and bool((got["lse"][4] == -math.inf).all()) and not got["dq"][4].any()
    for bad in (math.nan, math.inf):
        t["k"][11], t["v"][11] = bad, bad
        again = run_all(t, 0.25, dout)
        for name in got:
            assert torch.equal(again[name], got[name]), name


def test_bias_of_the_lowest_value(cuda_device):
    """A finite mask is no mask: where all of a row's edges have it, the row's weights are equal."""
    low = torch.finfo(F32).min
    rowptr = torch.tensor([0, 4, 7], dtype=torch.int32).cuda()
    colidx = torch.tensor([0, 1, 2, 3, 0, 1, 2], dtype=torch.int32).cuda()
    gen = gen_of(8)
    q, k, v = (randn(gen, F32, *s).cuda() for s in ((2, 1, 2, 8), (4, 1, 2, 8), (4, 1, 8)))
    lam = torch.tensor([0.25]).cuda()
    bias = torch.tensor([low, low, low, low, low, 0.5, 0.0]).cuda()
    out, lse = torch_op.diff_attention(rowptr, colidx, q, k, v, lam, bias=bias, return_lse=True)
    # four equal weights in each map: 0.75 of the mean of v (4 terms, two products: 8 roundings)
    want = 0.75 * v[:, 0].double().mean(0)
    assert bool(((out[0, 0].double() - want).abs() <= 8 * 2.0 ** -24 * v.abs().double().max()).all())
    rest = attention_reference(torch.tensor([0, 2]), torch.tensor([1, 2]), torch.tensor([0.5, 0.0]), q[1:], k, v, lam, 8 ** -0.5)
    check(out[1:], rest["out"], "out")
    assert bool(lse[0].isfinite().all())


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("heads,kvh", [(2, 2), (4, 4), (4, 1), (6, 3)])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("where", ["k", "v"])
def test_a_bad_number_shows_where_it_counts_and_nowhere_else(cuda_device, dtype, heads, kvh, bad, where):
    """One NaN or infinity in k or v of one kv head: rows that have the edge, at heads of that kv head, and no others differ."""
    gen = gen_of(9)
    m, n, d = 60, 40, 8
    rowptr, colidx = random_pattern(gen, m, n, 4, torch.int32, torch.int32, empty=0.1)
    t = make(gen, dtype, rowptr, colidx, m, n, heads, kvh, d, 16)
    hit = int(colidx[int(rowptr[20])])
    dout = randn(gen, dtype, m, heads, 16).cuda()
    # Rows that share a block with the bad number are summed once more by themselves, in another order: they need not keep their
    # bits.  The bounds of the 64-bit evaluation hold for every order of a row's sums.
    want = attention_reference(t["rowptr"], t["colidx"], None, t["q"], t["k"], t["v"], t["lam"], 0.3, dout)
    t[where][hit, 0].reshape(-1)[3] = bad
    got = run_all(t, 0.3, dout)
    rows = torch.repeat_interleave(torch.arange(m), (rowptr[1:] - rowptr[:-1]).long())
    touched = torch.zeros(m, dtype=torch.bool)
    touched[rows[colidx == hit]] = True
    near = torch.zeros(n, dtype=torch.bool)  # columns with an edge of a touched row
    near[colidx[touched[rows]].long()] = True
    mine = torch.arange(heads) < heads // kvh
    for name, first, own in (("out", touched, mine), ("dq", touched, mine), ("dk", near, torch.arange(kvh) < 1), ("dv", near, torch.arange(kvh) < 1)):
        value, bound = want[name]
        for part in ((~first, slice(None)), (slice(None), ~own)):
            check(got[name].cpu()[part[0]][:, part[1]], (value[part[0]][:, part[1]], bound[part[0]][:, part[1]]), name)
    shown = got["out"][touched][:, mine]
    if where == "k" and bad == math.nan:
        assert bool(shown.isnan().all())
    elif where == "v":
        assert bool((~shown[..., 3].isfinite()).all()) and bool(shown[..., :3].isfinite().all())


def test_views_of_a_packed_projection_and_a_gradient_that_is_expanded(cuda_device):
    gen = gen_of(10)
    m = 50
    for dtype, d, off in ((BF16, 32, 0), (F32, 32, 0), (F16, 32, 3), (F32, 16, 1)):
        rowptr, colidx = random_pattern(gen, m, m, 6, torch.int64, torch.int32)
        width = 4 * 2 * d + 2 * 2 * d + 2 * 2 * d + off + 5
        packed = randn(gen, dtype, m, width).cuda()
        at = [off, off + 8 * d, off + 12 * d, off + 16 * d]
        t = dict(rowptr=rowptr.cuda(), colidx=colidx.cuda(), bias=None, lam=torch.rand(4, generator=gen).cuda(),
                 q=packed[:, at[0]:at[1]].view(m, 4, 2, d), k=packed[:, at[1]:at[2]].view(m, 2, 2, d),
                 v=packed[:, at[2]:at[3]].view(m, 2, 2 * d))
        assert not t["q"].is_contiguous()
        compare(t, 0.2, torch.full((1, 1, 1), 0.5, dtype=dtype).cuda().expand(m, 4, 2 * d))


def test_heads_in_another_order_of_axes(cuda_device):
    """k and v as [heads, slots, ...] caches, seen through transposed views."""
    gen = gen_of(11)
    rowptr, colidx = random_pattern(gen, 20, 30, 9, torch.int32, torch.int32)
    t = make(gen, BF16, rowptr, colidx, 20, 30, 4, 2, 64, 128)
    t["k"] = t["k"].transpose(0, 1).contiguous().transpose(0, 1)
    t["v"] = t["v"].transpose(0, 1).contiguous().transpose(0, 1)
    compare(t, 0.125, randn(gen, BF16, 20, 4, 128).cuda())


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("m,n,nnz", [(0, 5, 0), (5, 0, 0), (4, 3, 0), (3, 0, 6)])
def test_nothing_to_attend_to(cuda_device, m, n, nnz, dtype):
    """No rows, no columns, no edges, or edges that all point outside: zeros, and no gradient."""
    rowptr = torch.zeros(m + 1, dtype=torch.int64)
    if nnz:
        rowptr[1:] = torch.arange(1, m + 1) * (nnz // m)
    t = make(gen_of(1), dtype, rowptr, torch.zeros(nnz, dtype=torch.int32), m, n, 2, 1, 8, 8)
    got = run_all(t, 1.0, torch.ones(m, 2, 8, dtype=dtype).cuda())
    assert got["out"].shape == (m, 2, 8) and not got["out"].any()
    for name in ("dq", "dk", "dv", "dlam"):
        assert not got[name].any(), name


def test_gradient_against_differences(cuda_device):
    """The kernels' gradients along random directions against central differences of the 64-bit evaluation."""
    gen = gen_of(12)
    rowptr, colidx = random_pattern(gen, 15, 18, 6, torch.int32, torch.int32)
    t = make(gen, F32, rowptr, colidx, 15, 18, 4, 2, 12, 10, bias=True, row_lam=True)
    dout = randn(gen, F32, 15, 4, 10).cuda()
    got = run_all(t, 0.3, dout)

    def value(**moved):
        a = {**{x: t[x].cpu().double() for x in ("q", "k", "v", "lam")}, **moved}
        out = attention_reference(t["rowptr"], t["colidx"], t["bias"], a["q"], a["k"], a["v"], a["lam"], 0.3)["out"][0]
        return float((out * dout.cpu().double()).sum())

    for name, grad in (("q", "dq"), ("k", "dk"), ("v", "dv"), ("lam", "dlam")):
        x = t[name].cpu().double()
        way = torch.randn(x.shape, generator=gen, dtype=torch.float64)
        h = 1e-5
        diff = (value(**{name: x + h * way}) - value(**{name: x - h * way})) / (2 * h)
        mine = float((got[grad].cpu().double() * way).sum())
        # the difference's own error is h^2 times third derivatives (1e-10 times sums of hundreds) and 1e-16/h times the value
        scale = float((got[grad].cpu().double().abs() * way.abs()).sum())
        assert abs(diff - mine) <= 2e-5 * scale + 1e-6, (name, diff, mine)


def test_same_bits_on_every_run_and_on_another_stream(cuda_device):
    gen = gen_of(13)
    rowptr, colidx = random_pattern(gen, 400, 300, 20, torch.int64, torch.int32, hub=4000)
    t = make(gen, BF16, rowptr, colidx, 400, 300, 4, 2, 32, 64, bias=True)
    dout = randn(gen, BF16, 400, 4, 64).cuda()
    first = run_all(t, 0.2, dout)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = run_all(t, 0.2, dout)
    torch.cuda.current_stream().wait_stream(side)
    for name in first:
        assert torch.equal(first[name], second[name]), name


def test_captured_and_replayed(cuda_device):
    """Norm and rotation, then attention, in a graph that is replayed on new inputs; two graphs hold scratch of their own."""
    gen = gen_of(14)
    m, length = 3, 700
    rowptr = torch.tensor([0, 0, length, 2 * length], dtype=torch.int32).cuda()
    colidx = torch.randint(0, 900, (2 * length,), generator=gen, dtype=torch.int32).cuda()
    t = make(gen, BF16, rowptr.cpu(), colidx.cpu(), m, 900, 8, 2, 64, 128)
    pos = torch.tensor([5, 70000, 1], dtype=torch.int64).cuda()
    freq = 10000.0 ** (-torch.arange(32, dtype=torch.float64) / 32).cuda()
    w = torch.rand(64, generator=gen).cuda()

    def step():
        q = torch_op.qk_norm_rotary(t["q"].view(m, 16, 64), None, pos, freq, q_weight=w, eps=1e-6)
        return torch_op.diff_attention(rowptr, colidx, q.view(m, 8, 2, 64), t["k"], t["v"], t["lam"])

    warm = torch.cuda.Stream()
    warm.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(warm):
        step()
    torch.cuda.current_stream().wait_stream(warm)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            result = step()
        graphs.append((g, result))
    for seed in (1, 2):
        t["q"].copy_(randn(gen_of(seed), BF16, m, 8, 2, 64))
        pos.add_(1)
        want = step()
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for _, result in graphs:
            assert torch.equal(result, want)


def test_synchronous_call_of_the_c_entry(cuda_device):
    """stream NULL: the result is there when the call returns."""
    gen = gen_of(15)
    rowptr, colidx = random_pattern(gen, 30, 40, 6, torch.int64, torch.int32)
    t = make(gen, F32, rowptr, colidx, 30, 40, 2, 2, 8, 16)
    want = torch_op.diff_attention(t["rowptr"], t["colidx"], t["q"], t["k"], t["v"], t["lam"], scale=0.5)
    out = torch.empty_like(want)
    args = api.attention_args(t["rowptr"], t["colidx"], None, t["q"], t["k"], t["v"], t["lam"], 0.5)
    ws = torch.empty(api.diff_attention_workspace(False, args), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    assert api.diff_attention(args, out, None, ws, None) == 0
    assert torch.equal(out, want)
    assert api.diff_attention(args, out, None, ws[: ws.numel() - 1], None) == -3


@pytest.mark.parametrize("m,n,mean,ptr,idx", [(1, 1, 3, torch.int32, torch.int32), (300, 250, 9, torch.int64, torch.int32),
                                             (5000, 70000, 7, torch.int32, torch.int64), (40, 3, 2000, torch.int64, torch.int64)])
def test_transposed_pattern(cuda_device, m, n, mean, ptr, idx):
    gen = gen_of(m)
    rowptr, colidx = random_pattern(gen, m, n, mean, ptr, idx, hub=3 * mean)
    if colidx.numel() > 10:
        colidx[3::11] = -1
        colidx[5::13] = n
    t_rowptr, t_row, t_edge = (x.cpu() for x in torch_op.csr_transpose(rowptr.cuda(), colidx.cuda(), n))
    row = torch.repeat_interleave(torch.arange(m), (rowptr[1:] - rowptr[:-1]).long())
    keep = torch.nonzero((colidx >= 0) & (colidx < n)).flatten()
    order = keep[torch.sort(colidx[keep].long(), stable=True).indices]
    assert t_rowptr.dtype == ptr and int(t_rowptr[-1]) == len(keep)
    assert torch.equal(t_rowptr.long(), torch.cat((torch.zeros(1, dtype=torch.long), torch.cumsum(torch.bincount(colidx[keep].long(), minlength=n), 0))))
    assert torch.equal(t_edge[:len(keep)].long(), order) and torch.equal(t_row[:len(keep)].long(), row[order])


def test_transposed_pattern_of_many_edges(cuda_device):
    """The sort's long tiles, three digits of columns."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    m, n, nnz = 40000, 100000, (4 << 20) + 77
    rowptr = torch.zeros(m + 1, dtype=torch.int64, device="cuda")
    rowptr[1:-1] = torch.sort(torch.randint(0, nnz, (m - 1,), generator=gen, device="cuda")).values
    rowptr[-1] = nnz
    colidx = torch.randint(0, n, (nnz,), generator=gen, device="cuda", dtype=torch.int32)
    t_rowptr, t_row, t_edge = torch_op.csr_transpose(rowptr, colidx, n)
    order = torch.sort(colidx, stable=True).indices
    row = torch.repeat_interleave(torch.arange(m, device="cuda"), rowptr[1:] - rowptr[:-1])
    assert torch.equal(t_edge.long(), order) and torch.equal(t_row.long(), row[order])
    assert torch.equal(t_rowptr[1:], torch.cumsum(torch.bincount(colidx.long(), minlength=n), 0)) and int(t_rowptr[0]) == 0


def test_patterns_that_break_their_contract_stay_in_bounds(cuda_device):
    """Row pointers that decrease or leave the list, and wild column ids: wrong rows, no access outside, later calls are right."""
    gen = gen_of(19)
    rowptr, colidx = random_pattern(gen, 300, 200, 8, torch.int64, torch.int64, hub=700)
    for dtype in (F32, BF16, F16):
        t = make(gen, dtype, rowptr, colidx, 300, 200, 4, 2, 16, 32)
        dout = randn(gen, dtype, 300, 4, 32).cuda()
        bad = dict(t)
        bad["rowptr"] = t["rowptr"][torch.randperm(301, generator=gen).cuda()].contiguous()
        bad["rowptr"][::7] += 10 ** 12
        bad["rowptr"][::11] -= 10 ** 12
        bad["colidx"] = t["colidx"].clone()
        bad["colidx"][::3] += 10 ** 15
        bad["colidx"][::5] -= 2 ** 33
        run_all(bad, 0.25, dout)
        torch.cuda.synchronize()
        compare(t, 0.25, dout)


def test_row_pointers_that_start_behind_the_first_edge(cuda_device):
    """A run of rows of a larger pattern: edges before the first and behind the last row pointer belong to nobody."""
    gen = gen_of(16)
    rowptr, colidx = random_pattern(gen, 60, 50, 6, torch.int64, torch.int32, hub=600)
    t = make(gen, F32, rowptr, colidx, 60, 50, 2, 1, 16, 16, bias=True)
    part = slice(7, 40)
    s = dict(t, rowptr=t["rowptr"][7:41], q=t["q"][part])
    compare(s, 0.25, randn(gen, F32, 33, 2, 16).cuda())


# ---- norm and rotation ---------------------------------------------------------------------------------------------------
# dtype, rows, q heads, k heads, d, pairs, axes, position type, interleaved, norm, weights, weight type
ROTARY = [
    (F32, 7, 2, 1, 32, 16, 1, torch.int64, False, True, True, F32),
    (F32, 300, 4, 4, 40, 16, 2, F32, True, True, True, F32),
    (F32, 33, 3, 0, 256, 128, 4, torch.float64, False, True, True, F32),
    (F32, 20, 2, 2, 7, 3, 1, torch.int32, True, True, True, F32),
    (F32, 20, 2, 3, 1, 0, 0, None, False, True, True, F32),
    (BF16, 70, 8, 2, 128, 64, 1, torch.int64, False, True, True, BF16),
    (BF16, 70, 8, 2, 64, 32, 3, torch.int32, True, True, False, F32),
    (BF16, 1, 16, 4, 256, 100, 1, torch.int64, False, True, True, F32),
    (BF16, 513, 1, 1, 16, 8, 2, torch.int32, False, False, False, F32),
    (F16, 64, 5, 3, 80, 40, 2, torch.int32, False, True, True, F16),
    (F16, 64, 5, 3, 90, 21, 2, torch.int32, True, True, True, F16),
    (F16, 2000, 2, 1, 96, 16, 1, torch.int64, True, True, True, F32),
    (BF16, 90, 3, 2, 40, 20, 1, F32, True, True, True, F32),      # interleaved pairs that end inside a unit
    (BF16, 90, 3, 2, 40, 20, 2, F32, False, True, True, F32),     # halves of whole 8-byte vectors
    (F16, 90, 1, 2, 44, 8, 1, torch.int32, True, True, False, F32),
    (F32, 90, 1, 2, 24, 6, 1, torch.int32, True, True, True, F32),
    (F16, 50, 2, 0, 252, 126, 1, torch.int64, False, True, True, F16),
    (F32, 50, 2, 0, 252, 126, 1, torch.int64, True, True, True, F32),
    (F16, 90, 3, 2, 234, 36, 1, torch.int64, False, True, True, F16),     # rows in twos, more of them than two a lane
    (BF16, 90, 3, 2, 254, 127, 2, torch.int32, True, True, True, F32),
    (F32, 90, 3, 2, 254, 2, 1, torch.int64, False, True, True, F32),
    (BF16, 90, 3, 2, 46, 16, 2, F32, False, True, True, F32),             # in twos, one unit a lane
    (F32, 90, 3, 2, 10, 3, 1, torch.int32, True, True, True, F32),
    (F16, 90, 1, 2, 2, 1, 1, torch.int32, True, True, True, F32),
    (BF16, 90, 3, 2, 40, 15, 2, F32, False, True, True, F32),             # single elements, fewer than the lanes
    (F32, 90, 3, 2, 255, 127, 1, torch.int64, True, True, True, F32),     # and more
]


@pytest.mark.parametrize("case", range(len(ROTARY)))
def test_norm_and_rotation_with_gradients(cuda_device, case):
    dtype, rows, hq, hk, d, pairs, axes, pt, interleaved, norm, weights, wt = ROTARY[case]
    gen = gen_of(100 + case)
    q, k = randn(gen, dtype, rows, hq, d).cuda(), randn(gen, dtype, rows, hk, d).cuda() if hk else None
    pos = freq = None
    if pairs:
        pos = (torch.randint(0, 1 << 20, (rows, axes), generator=gen).to(pt) if not pt.is_floating_point else
               (torch.randn(rows, axes, generator=gen) * 100).to(pt)).cuda()
        freq = torch.rand(axes, pairs, generator=gen, dtype=torch.float64).cuda()
    eps = 1e-6 if norm else None
    wq, wk = (randn(gen, wt, d).cuda(), randn(gen, wt, d).cuda() if hk else None) if weights else (None, None)
    leaves = [x.detach().requires_grad_() if x is not None else None for x in (q, k, wq, wk)]
    got = torch_op.qk_norm_rotary(leaves[0], leaves[1], pos, freq, q_weight=leaves[2], k_weight=leaves[3], eps=eps, interleaved=interleaved)
    got = (got, None) if k is None else got
    dy = [randn(gen, dtype, rows, hq, d).cuda(), randn(gen, dtype, rows, hk, d).cuda() if hk else None]
    live = [x for x in leaves if x is not None]
    grads = dict(zip([id(x) for x in live], torch.autograd.grad([g for g in got if g is not None], live, [g for g in dy if g is not None])))
    for i, (x, w) in enumerate(((q, wq), (k, wk))):
        if x is None:
            continue
        want = rotary_reference(x, w, pos, freq, eps, interleaved, dy[i])
        check(got[i], want["y"], "y")
        check(grads[id(leaves[i])], want["dx"], "dx")
        if w is not None:
            value, bound = want["dw"]
            check(grads[id(leaves[2 + i])], (value, bound + HALF_STEP[wt] * value.abs()), "dw")


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_norm_and_rotation_of_views(cuda_device, dtype):
    """Packed projections at aligned and odd offsets, heads before rows, positions of one row for all."""
    gen = gen_of(200)
    rows, d = 37, 32
    freq = torch.rand(1, 16, generator=gen, dtype=torch.float64).cuda()
    pos = torch.tensor([9]).cuda().expand(rows)
    for off in (0, 1, 4):
        packed = randn(gen, dtype, rows, 6 * d + off).cuda()
        q, k = packed[:, off:off + 4 * d].view(rows, 4, d), packed[:, off + 4 * d:].view(rows, 2, d)
        for a, b in ((q, k), (q.transpose(0, 1).contiguous().transpose(0, 1), k.transpose(0, 1).contiguous().transpose(0, 1))):
            y = torch_op.qk_norm_rotary(a, b, pos, freq, eps=1e-5)
            for x, z in ((a, y[0]), (b, y[1])):
                check(z, rotary_reference(x, None, pos, freq, 1e-5, False)["y"], "y")


def test_norm_of_zeros_and_no_rows(cuda_device):
    y = torch_op.qk_norm_rotary(torch.zeros(3, 2, 8, device="cuda"), eps=1e-6)
    assert not y.any()
    x = torch.zeros(0, 2, 8, device="cuda", requires_grad=True)
    w = torch.ones(8, device="cuda", requires_grad=True)
    y = torch_op.qk_norm_rotary(x, q_weight=w, eps=1e-6)
    dx, dw = torch.autograd.grad(y, (x, w), torch.zeros_like(y))
    assert y.shape == (0, 2, 8) and dx.shape == (0, 2, 8) and not dw.any()


def test_a_layer_of_both(cuda_device):
    """Projection -> norm and rotation by 2-D positions -> attention over a graph -> loss; gradients of every weight against
    the same layer in elementary operations and 64 bits."""
    gen = gen_of(300)
    m, heads, kvh, d = 60, 4, 2, 16
    rowptr, colidx = random_pattern(gen, m, m, 7, torch.int64, torch.int32, hub=640)
    rowptr, colidx = rowptr.cuda(), colidx.cuda()
    x = randn(gen, F32, m, 24).cuda()
    wide = heads * 2 * d + kvh * 2 * d + kvh * 2 * d
    weights = [(randn(gen, F32, 24, wide) * 0.2).cuda(), (1 + 0.1 * randn(gen, F32, d)).cuda(), (1 + 0.1 * randn(gen, F32, d)).cuda(),
               torch.rand(heads, generator=gen).cuda()]
    pos = (torch.randn(m, 2, generator=gen) * 10).cuda()
    freq = torch.zeros(2, 8, dtype=torch.float64)
    freq[0, :4], freq[1, 4:] = torch.rand(4, generator=gen), torch.rand(4, generator=gen)
    freq = freq.cuda()
    goal = randn(gen, F32, m, heads, 2 * d).cuda()

    def split(w):
        y = x.to(w.dtype) @ w
        a, b = heads * 2 * d, heads * 2 * d + kvh * 2 * d
        return y[:, :a].view(m, heads * 2, d), y[:, a:b].view(m, kvh * 2, d), y[:, b:].view(m, kvh, 2 * d)

    def ours(w, wq, wk, lam):
        q, k, v = split(w)
        q, k = torch_op.qk_norm_rotary(q, k, pos, freq, q_weight=wq, k_weight=wk, eps=1e-6)
        return torch_op.diff_attention(rowptr, colidx, q.view(m, heads, 2, d), k.view(m, kvh, 2, d), v, lam,
                                       transposed=torch_op.csr_transpose(rowptr, colidx, m))

    def plain(w, wq, wk, lam):
        q, k, v = split(w)
        ang = (pos.double() @ freq)[:, None]

        def turn(t, u):
            t = t / torch.sqrt((t * t).mean(-1, keepdim=True) + 1e-6) * u
            a, b = t[..., :8], t[..., 8:]
            return torch.cat((a * ang.cos() - b * ang.sin(), b * ang.cos() + a * ang.sin()), -1)

        q, k = turn(q, wq).view(m, heads, 2, d), turn(k, wk).view(m, kvh, 2, d)
        count = torch.zeros(m, m, dtype=torch.float64, device="cuda")
        row = torch.repeat_interleave(torch.arange(m, device="cuda"), rowptr[1:] - rowptr[:-1])
        count.index_put_((row, colidx.long()), torch.ones(len(row), dtype=torch.float64, device="cuda"), accumulate=True)
        k, v = k.repeat_interleave(heads // kvh, 1), v.repeat_interleave(heads // kvh, 1)
        s = torch.einsum("uhcd,vhcd->hcuv", q, k) * d ** -0.5
        e = torch.exp(s - s.amax(-1, keepdim=True)) * count
        p = e / e.sum(-1, keepdim=True).clamp_min(1e-300)
        return torch.einsum("huv,vhe->uhe", p[:, 0] - lam[:, None, None] * p[:, 1], v)

    grads = []
    for fn, t in ((ours, F32), (plain, torch.float64)):
        leaves = [w.to(t).requires_grad_() for w in weights]
        loss = ((fn(*leaves) - goal.to(t)) ** 2).sum()
        grads.append(torch.autograd.grad(loss, leaves))
    for a, b in zip(*grads):
        # sums of up to 60 x 700 x 32 terms in 32 bits with cancellation: 2^-24 times a few thousand of the largest entry
        assert float((a.double() - b).abs().max()) <= 4096 * 2.0 ** -24 * float(b.abs().max())


def test_no_gradient_for_masks_and_positions(cuda_device):
    gen = gen_of(17)
    rowptr, colidx = random_pattern(gen, 5, 5, 3, torch.int32, torch.int32, empty=0.0)
    t = make(gen, F32, rowptr, colidx, 5, 5, 1, 1, 8, 8)
    bias = torch.zeros(colidx.numel(), device="cuda", requires_grad=True)
    out = torch_op.diff_attention(t["rowptr"], t["colidx"], t["q"], t["k"], t["v"], t["lam"], bias=bias)
    with pytest.raises(api.FusedMMError, match="bias"):
        out.sum().backward()
    pos = torch.zeros(5, device="cuda", requires_grad=True)
    y = torch_op.qk_norm_rotary(t["k"][:, :, 0], None, pos, torch.ones(1, 2, dtype=torch.float64, device="cuda"))
    with pytest.raises(api.FusedMMError, match="pos"):
        y.sum().backward()


def test_shapes_of_gradients_for_a_compiler(cuda_device):
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        q = torch.empty(6, 4, 2, 8, dtype=BF16, device="cuda", requires_grad=True)
        k, v = torch.empty(9, 2, 2, 8, dtype=BF16, device="cuda"), torch.empty(9, 2, 12, dtype=BF16, device="cuda")
        rowptr, colidx = torch.empty(7, dtype=torch.int64, device="cuda"), torch.empty(30, dtype=torch.int32, device="cuda")
        out = torch_op.diff_attention(rowptr, colidx, q, k, v, torch.empty(4, device="cuda"))
        assert torch.autograd.grad(out, q, torch.empty_like(out))[0].shape == q.shape
        x = torch.empty(6, 4, 8, device="cuda", requires_grad=True)
        y = torch_op.qk_norm_rotary(x, eps=1e-6)
        assert torch.autograd.grad(y, x, torch.empty_like(y))[0].shape == x.shape


def test_operators_of_torch_and_functions_agree(cuda_device):
    """torch.ops.fusedmm_b200.* (the way of a compiled program) and the module's functions make the same calls."""
    gen = gen_of(18)
    rowptr, colidx = random_pattern(gen, 20, 30, 6, torch.int64, torch.int32)
    t = make(gen, BF16, rowptr, colidx, 20, 30, 4, 2, 16, 32)
    dout = randn(gen, BF16, 20, 4, 32).cuda()
    want = run_all(t, 0.25, dout)
    leaves = [t[a].detach().requires_grad_() for a in ("q", "k", "v", "lam")]
    out, lse = torch.ops.fusedmm_b200.diff_attention(t["rowptr"], t["colidx"], None, *leaves, 0.25, None, None, None)
    grads = torch.autograd.grad(out, leaves, dout)
    for a, b in zip((out, lse, *grads), (want[n] for n in ("out", "lse", "dq", "dk", "dv", "dlam"))):
        assert torch.equal(a, b)
    x, w = t["k"][:, :, 0].contiguous(), torch.rand(16, generator=gen).cuda()
    assert torch.equal(torch_op.qk_norm_rotary(x, q_weight=w, eps=1e-6),
                       torch.ops.fusedmm_b200.qk_norm_rotary(x, None, None, None, w, None, 1e-6, False)[0])
