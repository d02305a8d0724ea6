"""Refusals of the attention operators, checked before anything reaches a GPU, and the shapes they announce to a compiler."""
import ctypes as C

import pytest
import torch

from fusedmm_b200 import api, torch_op

I, L, P, D = C.c_int32, C.c_int64, C.c_void_p, C.c_double


def good_attention(m=4, n=5, nnz=7, heads=4, kvh=2, d=8, dv=16, dtype=torch.float32):
    return dict(rowptr=torch.tensor([0, nnz] + [nnz] * (m - 1), dtype=torch.int32), colidx=torch.zeros(nnz, dtype=torch.int32),
                bias=None, q=torch.zeros(m, heads, 2, d, dtype=dtype), k=torch.zeros(n, kvh, 2, d, dtype=dtype),
                v=torch.zeros(n, kvh, dv, dtype=dtype), lam=torch.zeros(heads), scale=1.0)


@pytest.mark.parametrize("change,text", [
    (dict(q=torch.zeros(4, 4, 2, 8, dtype=torch.float64)), "float32, bfloat16 or float16"),
    (dict(k=torch.zeros(5, 2, 2, 8, dtype=torch.bfloat16)), "share one type"),
    (dict(q=torch.zeros(4, 4, 3, 8)), "heads, 2, d"),
    (dict(q=torch.zeros(3, 4, 2, 8)), "rowptr"),
    (dict(k=torch.zeros(5, 2, 2, 9)), "d of q"),
    (dict(k=torch.zeros(5, 3, 2, 8), v=torch.zeros(5, 3, 16)), "multiple"),
    (dict(v=torch.zeros(6, 2, 16)), "v must be"),
    (dict(v=torch.zeros(5, 2, 300)), "dv between"),
    (dict(q=torch.zeros(4, 4, 2, 129), k=torch.zeros(5, 2, 2, 129)), "d must be between"),
    (dict(lam=torch.zeros(3)), "lam must be"),
    (dict(lam=torch.zeros(4, dtype=torch.float64)), "lam must be float32"),
    (dict(lam=torch.zeros(1, 4).expand(4, 4)), "lam must be"),
    (dict(lam=torch.zeros(5, 4)), "lam must be"),
    (dict(bias=torch.zeros(6)), "bias"),
    (dict(bias=torch.zeros(7, dtype=torch.float64)), "bias"),
    (dict(rowptr=torch.zeros(5)), "rowptr must be int32"),
    (dict(colidx=torch.zeros(14, dtype=torch.int32)[::2]), "dense vector"),
    (dict(q=torch.zeros(4, 4, 8, 2).transpose(2, 3)), "must be dense"),
    (dict(), "CUDA tensor"),
])
def test_attention_refuses(change, text):
    with pytest.raises(ValueError, match=text):
        api.attention_args(**{**good_attention(), **change})


def good_rotary(**change):
    return {**dict(q=torch.zeros(6, 3, 16), k=torch.zeros(6, 1, 16), q_weight=None, k_weight=None, pos=torch.zeros(6, 2),
                   freq=torch.zeros(2, 8, dtype=torch.float64), eps=1e-6, interleaved=False), **change}


@pytest.mark.parametrize("change,text", [
    (dict(q=torch.zeros(6, 3, 16, dtype=torch.float64)), "float32, bfloat16 or float16"),
    (dict(q=torch.zeros(6, 48)), "rows, heads, d"),
    (dict(k=torch.zeros(5, 1, 16)), "k must be"),
    (dict(k=torch.zeros(6, 1, 16, dtype=torch.float16)), "share one type"),
    (dict(q=torch.zeros(6, 3, 300), k=None), "between 1 and 256"),
    (dict(pos=None), "come together"),
    (dict(freq=None), "come together"),
    (dict(freq=torch.zeros(2, 8)), "float64"),
    (dict(freq=torch.zeros(3, 8, dtype=torch.float64)), "axes, pairs"),
    (dict(freq=torch.zeros(2, 9, dtype=torch.float64)), "half of d"),
    (dict(pos=torch.zeros(5, 2)), "pos must be"),
    (dict(pos=torch.zeros(6, 5), freq=torch.zeros(5, 8, dtype=torch.float64)), "one to four"),
    (dict(pos=torch.zeros(6, 2, dtype=torch.int16)), "pos must be"),
    (dict(q_weight=torch.zeros(15)), "d entries"),
    (dict(q_weight=torch.zeros(16), eps=None), "without eps"),
    (dict(q_weight=torch.zeros(16, dtype=torch.bfloat16)), "type of q"),
    (dict(k_weight=torch.zeros(16), k=None), "without k"),
    (dict(eps=-1.0), "negative"),
    (dict(q=torch.zeros(6, 16, 3).transpose(1, 2)), "must be dense"),
    (dict(), "CUDA tensor"),
])
def test_rotary_refuses(change, text):
    with pytest.raises(ValueError, match=text):
        api.rotary_args(**good_rotary(**change))


def test_c_entries_check_their_arguments_first():
    """Statuses of calls that are wrong whatever the machine: -3 invalid argument, -4 beyond a limit."""
    lib = api.lib()
    ws = lib.fusedmm_b200_diff_attention_workspace
    ws.restype, ws.argtypes = L, [I, I, I, L, L, L, I, I, I, I]
    assert ws(0, 1, 1, 4, 4, 8, 2, 1, 8, 8) == -3           # double
    assert ws(0, 1, 0, -1, 4, 8, 2, 1, 8, 8) == -3
    assert ws(0, 1, 0, 4, 4, 8, 3, 2, 8, 8) == -3           # heads no multiple of kv heads
    assert ws(0, 1, 0, 4, 4, 8, 2, 1, 129, 8) == -4
    assert ws(0, 1, 0, 4, 4, 8, 2, 1, 8, 257) == -4
    fwd = lib.fusedmm_b200_diff_attention
    fwd.restype, fwd.argtypes = I, list(api._ATTN_IN) + [P, P, P, L, P]
    good = dict(dtype=0, pb=32, ib=32, m=4, n=4, nnz=8, rp=256, ci=256, bias=None, h=2, kvh=1, d=8, dv=8, q=256, ldq=32, hsq=16, k=256,
                ldk=16, hsk=16, v=256, ldv=8, hsv=8, lam=256, ldlam=0, scale=1.0, out=256, lse=None, ws=256, wb=1 << 40, stream=None)
    for change, status in ((dict(pb=16), -3), (dict(ib=8), -3), (dict(m=-1), -3), (dict(dtype=7), -3), (dict(h=0), -3),
                           (dict(q=None), -3), (dict(k=None), -3), (dict(ci=None), -3), (dict(lam=None), -3), (dict(out=None), -3),
                           (dict(d=200), -4), (dict(m=1 << 60), -4), (dict(m=0), 0)):
        assert fwd(*{**good, **change}.values()) == status, change
    back = lib.fusedmm_b200_diff_attention_backward
    back.restype, back.argtypes = I, list(api._ATTN_IN) + [P, P, L, L, P, P, P, P, P, P, P, P, L, P]
    good = dict(list(good.items())[:25], lse=256, do=256, ldo=16, hso=8, tp=256, tr=256, te=None, dq=256, dk=256, dvo=256, dlam=256, ws=256,
                wb=1 << 40, stream=None)
    for change, status in ((dict(m=(1 << 31) - 1), -4), (dict(lse=None), -3), (dict(do=None), -3), (dict(tp=None), -3), (dict(tr=None), -3),
                           (dict(bias=256), -3), (dict(dlam=None), -3), (dict(dk=None), -3)):
        assert back(*{**good, **change}.values()) == status, change
    tr = lib.fusedmm_b200_csr_transpose
    tr.restype, tr.argtypes = I, [I, I, L, L, L, P, P, P, P, P, P, L, P]
    assert tr(32, 32, 4, 4, 1 << 31, 256, 256, 256, 256, 256, 256, 1 << 40, None) == -4
    assert tr(32, 16, 4, 4, 8, 256, 256, 256, 256, 256, 256, 1 << 40, None) == -3
    assert tr(32, 32, 4, 4, 8, 256, None, 256, 256, 256, 256, 1 << 40, None) == -3
    assert tr(32, 32, 4, 4, 8, 256, 256, 256, 256, 256, 256, 8, None) == -3      # too little scratch
    assert tr(32, 32, 4, 4, 8, 256, 256, 256, 256, 256, 260, 1 << 40, None) == -3  # not aligned
    rot = lib.fusedmm_b200_qk_norm_rotary
    rot.restype, rot.argtypes = I, list(api._ROTARY_IN) + [P, P, P]
    good = dict(dtype=0, rows=4, hq=2, hk=1, d=8, q=256, ldq=16, hsq=8, k=256, ldk=8, hsk=8, wt=0, wq=None, wk=None, norm=1, eps=1e-6, pt=0,
                pos=256, ldp=1, asp=1, axes=1, freq=256, pairs=4, il=0, qo=256, ko=256, stream=None)
    for change, status in ((dict(dtype=1), -3), (dict(pairs=5), -3), (dict(axes=5), -3), (dict(axes=0), -3), (dict(pt=4), -3), (dict(d=257), -4),
                           (dict(eps=float("nan")), -3), (dict(norm=0, wq=256), -3), (dict(wt=2), -3), (dict(q=None), -3), (dict(freq=None), -3),
                           (dict(rows=0, q=None, k=None, pos=None, freq=None), 0)):
        assert rot(*{**good, **change}.values()) == status, change


def test_host_tensors_have_no_kernel():
    a = good_attention()
    with pytest.raises(NotImplementedError):
        torch_op.diff_attention(a["rowptr"], a["colidx"], a["q"], a["k"], a["v"], a["lam"])
    with pytest.raises(NotImplementedError):
        torch_op.qk_norm_rotary(torch.zeros(2, 2, 8), eps=1e-6)


def test_shapes_for_a_compiler():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        dev = "cuda"
        q = torch.empty(6, 4, 2, 8, dtype=torch.bfloat16, device=dev)
        k, v = torch.empty(9, 2, 2, 8, dtype=torch.bfloat16, device=dev), torch.empty(9, 2, 12, dtype=torch.bfloat16, device=dev)
        rowptr, colidx = torch.empty(7, dtype=torch.int64, device=dev), torch.empty(30, dtype=torch.int32, device=dev)
        lam = torch.empty(4, device=dev)
        t = torch_op.csr_transpose(rowptr, colidx, 9)
        assert [x.shape[0] for x in t] == [10, 30, 30] and t[0].dtype == torch.int64
        out, lse = torch_op.diff_attention(rowptr, colidx, q, k, v, lam, transposed=t, return_lse=True)
        assert out.shape == (6, 4, 12) and out.dtype == torch.bfloat16 and lse.shape == (6, 4, 2)
        a, b = torch_op.qk_norm_rotary(torch.empty(6, 4, 8, device=dev), torch.empty(6, 2, 8, device=dev), eps=1e-6)
        assert a.shape == (6, 4, 8) and b.shape == (6, 2, 8)


@pytest.fixture
def stand_in(monkeypatch):
    """Host tensors in the place of CUDA ones: the library calls of the forward pass are stood in for and log their inputs."""
    calls = []

    def rotary(q, k, pos, freq, q_weight, k_weight, eps, interleaved):
        calls.append((q, k, pos, freq, q_weight, k_weight))
        return torch.zeros_like(q), torch.zeros_like(q if k is None else k)

    def attention(rowptr, colidx, bias, q, k, v, lam, scale, *_):
        calls.append((rowptr, colidx, bias, q, k, v, lam))
        return q.new_zeros(q.shape[0], q.shape[1], v.shape[2]), torch.zeros(q.shape[:3])

    monkeypatch.setattr(torch.Tensor, "is_cuda", property(lambda t: True), raising=False)
    monkeypatch.setattr(torch_op, "_rotary_cuda", rotary)
    monkeypatch.setattr(torch_op, "_attention_forward", attention)
    kernels = torch.library.Library("fusedmm_b200", "IMPL")
    kernels.impl("qk_norm_rotary", rotary, "CPU")
    kernels.impl("diff_attention", attention, "CPU")
    kernels.impl("qk_norm_rotary", lambda *args: torch_op._Rotary.apply(*args), "AutogradCPU")
    kernels.impl("diff_attention", lambda *args: torch_op._Attention.apply(*args), "AutogradCPU")
    yield calls
    kernels._destroy()


def attention_call(**change):
    a = {**good_attention(), **change}
    return torch_op.diff_attention(a["rowptr"], a["colidx"], a["q"], a["k"], a["v"], a["lam"], scale=a["scale"])


def test_forward_mode_is_refused(stand_in):
    """There is no forward-mode derivative: a tangent is refused and not dropped, also without a gradient mode."""
    from torch.autograd import forward_ad
    for grad in (True, False):
        with torch.set_grad_enabled(grad), forward_ad.dual_level():
            dual = lambda *shape: forward_ad.make_dual(torch.ones(shape), torch.ones(shape))
            with pytest.raises(NotImplementedError, match="jvp"):
                torch_op.qk_norm_rotary(dual(3, 2, 8), eps=1e-6)
            with pytest.raises(NotImplementedError, match="jvp"):
                torch_op.qk_norm_rotary(torch.ones(3, 2, 8), q_weight=dual(8), eps=1e-6)
            with pytest.raises(NotImplementedError, match="jvp"):
                attention_call(lam=dual(4))
    assert not torch_op.qk_norm_rotary(torch.ones(3, 2, 8), eps=1e-6).requires_grad


@pytest.mark.parametrize("trains", [False, True])
def test_a_trace_holds_the_operators(stand_in, trains):
    """torch.jit.trace records the operators, not the allocation of their results alone."""
    a = good_attention()
    for call, name, x in ((lambda q: torch_op.qk_norm_rotary(q, eps=1e-6), "fusedmm_b200::qk_norm_rotary", torch.ones(3, 2, 8)),
                          (lambda q: torch_op.diff_attention(a["rowptr"], a["colidx"], q, a["k"], a["v"], a["lam"], scale=1.0),
                           "fusedmm_b200::diff_attention", torch.ones(4, 4, 2, 8))):
        nodes = [n.kind() for n in torch.jit.trace(call, (x.requires_grad_(trains),), check_trace=False).graph.nodes()]
        assert name in nodes and not any(n.startswith(("aten::", "^")) for n in nodes), nodes


@pytest.mark.parametrize("trains", [False, True])
def test_numbers_that_are_stored_negated(stand_in, trains):
    """The imaginary part of a conjugate is a view that stores its numbers negated: the library gets the numbers themselves."""
    z = torch.complex(torch.rand(3), 1 + torch.rand(3))
    pos = z.conj().imag
    assert pos.is_neg()
    torch_op.qk_norm_rotary(torch.ones(3, 2, 8, requires_grad=trains), None, pos, torch.ones(1, 4, dtype=torch.float64))
    got = stand_in[-1][2]
    assert not got.is_neg() and torch.equal(got, -z.imag)
    q = torch._neg_view(torch.ones(4, 4, 2, 8)).requires_grad_(trains)
    attention_call(q=q)
    assert not stand_in[-1][3].is_neg()


def test_sizes_whose_products_leave_64_bits():
    ws = api.lib().fusedmm_b200_diff_attention_workspace
    ws.restype, ws.argtypes = L, [I, I, I, L, L, L, I, I, I, I]
    assert ws(0, 1, 0, 1 << 48, 4, 8, 65536, 1, 8, 8) == -4
    assert ws(1, 1, 2, 4, 4, 1 << 48, 4096, 1, 8, 8) == -4


def test_strides_of_the_rotation_have_no_limit():
    """-3: the made-up addresses are no device memory, which is looked at behind the limits (-4)."""
    rot = api.lib().fusedmm_b200_qk_norm_rotary
    rot.restype, rot.argtypes = I, list(api._ROTARY_IN) + [P, P, P]
    good = dict(dtype=2, rows=4, hq=2, hk=1, d=8, q=256, ldq=16, hsq=8, k=256, ldk=8, hsk=8, wt=0, wq=None, wk=None, norm=1, eps=1e-6, pt=0,
                pos=256, ldp=1, asp=1, axes=1, freq=256, pairs=4, il=0, qo=256, ko=256, stream=None)
    for name in ("ldq", "hsq", "ldk", "hsk"):
        assert rot(*{**good, name: 1 << 31}.values()) == -3, name
        assert rot(*{**good, name: -1}.values()) == -4, name


def test_strides_of_the_attention():
    """-4 for row strides of gathered rows alone; what else is far apart gets on to the looks at the device."""
    fwd, back = api.lib().fusedmm_b200_diff_attention, api.lib().fusedmm_b200_diff_attention_backward
    fwd.restype, fwd.argtypes = I, list(api._ATTN_IN) + [P, P, P, L, P]
    back.restype, back.argtypes = I, list(api._ATTN_IN) + [P, P, L, L, P, P, P, P, P, P, P, P, L, P]
    good = dict(dtype=0, pb=32, ib=32, m=4, n=4, nnz=8, rp=256, ci=256, bias=None, h=2, kvh=1, d=8, dv=8, q=256, ldq=32, hsq=16, k=256,
                ldk=16, hsk=16, v=256, ldv=8, hsv=8, lam=256, ldlam=0, scale=1.0, out=256, lse=None, ws=256, wb=1 << 40, stream=None)
    more = dict(list(good.items())[:25], lse=256, do=256, ldo=16, hso=8, tp=256, tr=256, te=None, dq=256, dk=256, dvo=256, dlam=256, ws=256,
                wb=1 << 40, stream=None)
    for name in ("ldq", "hsq", "ldk", "hsk", "ldv", "hsv", "ldlam", "ldo", "hso"):
        far = {name: 1 << 30}
        if name in good:
            assert (fwd(*{**good, **far}.values()) == -4) == (name in ("ldk", "ldv")), name
            assert fwd(*{**good, name: -4}.values()) == -4, name
        assert (back(*{**more, **far}.values()) == -4) == (name in ("ldk", "ldv", "ldq", "ldo")), name
        assert back(*{**more, name: -4}.values()) == -4, name
        assert back(*{**more, **far, "d": 7}.values()) != -4, name  # packed first
