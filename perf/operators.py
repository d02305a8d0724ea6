"""Cases of the attention operators: differential attention over the edges of a CSR pattern, and the per-head norm and
position rotation that make its queries and keys.  ``listed()`` names the cases, ``draw`` gives more of the same ranges,
``run`` makes one pass: the plain form (elementary torch operations, 32 bits) or, with ``own``, the framework's operators."""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-6


# ---- the cases ---------------------------------------------------------------------------------------------------------
def _rotary(rows, hq, hk, d, dtype, axes, pairs, positions, **more):
    case = dict(op="rotary", rows=rows, hq=hq, hk=hk, d=d, dtype=dtype, axes=axes, pairs=pairs,
                positions=positions, train=False, norm=True, interleaved=False, packed=False)
    case.update(more)
    return case


def _attention(graph, rows, edges, h, hk, d, dv, dtype, **more):
    case = dict(op="attention", graph=graph, rows=rows, edges=edges, h=h, hk=hk, d=d, dv=dv, dtype=dtype,
                train=False, bias=False, row_lam=False, plan=False)
    case.update(more)
    return case


def listed():
    return [
        # one decoding step of a few sequences far into their texts: latency
        _rotary(4, 16, 4, 128, "bf16", 1, 64, "far", name="rotary_step"),
        # training rows whose positions are time, height and width; queries and keys are views of one packed projection
        _rotary(16384, 16, 4, 64, "bf16", 3, 32, "grid", train=True, packed=True, name="rotary_video_train"),
        # nodes with the coordinates of a 2-D graph layout, part of the head rotated, pairs side by side, an odd row count
        _rotary(100003, 4, 4, 40, "f32", 2, 16, "layout", interleaved=True, name="rotary_layout_f32"),
        # the queries and keys of a long text at once
        _rotary(65536, 32, 8, 128, "bf16", 1, 64, "far", name="rotary_text"),
        # one token of one sequence over a short cache: latency
        _attention("cache", 1, 1000, 8, 2, 64, 128, "bf16", name="attention_step_one"),
        # one token of each of many sequences of very different lengths, the cache in scattered pages of 16 slots
        _attention("cache", 48, 262144, 16, 4, 64, 128, "bf16", name="attention_step_batch"),
        # training over a causal window, the pattern new in each step (no transposed pattern kept)
        _attention("window", 4096, 4096 * 128, 8, 2, 64, 128, "bf16", train=True, name="attention_window_train"),
        # a graph transformer's layer on a skewed graph of fixed edges, edge biases, some of them -inf (dropped edges)
        _attention("rmat", 16384, 425984, 4, 4, 32, 64, "f32", train=True, bias=True, plan=True, name="attention_rmat_train_f32"),
        # inference on a uniform graph, sizes that are no multiples of a vector, a weight of its own for each row
        _attention("uniform", 50021, 800000, 3, 1, 20, 36, "f16", row_lam=True, name="attention_uniform_odd"),
        # a large skewed graph, training
        _attention("rmat", 1 << 19, 1 << 23, 4, 4, 32, 64, "bf16", train=True, plan=True, name="attention_rmat_train_large"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    dtype = rng.choice(["f32", "bf16", "f16"])
    if rng.random() < 0.4:
        d = rng.choice([16, 32, 40, 64, 80, 96, 128, 200, 256, rng.randrange(10, 129) * 2])
        hk = rng.choice([1, 2, 3, 4, 8])
        hq = hk * rng.choice([1, 2, 4, 5])
        axes = rng.choice([1, 1, 2, 3])
        pairs = d // 2 if rng.random() < 0.6 else rng.randrange(max(1, axes), d // 2 + 1)
        rows = max(1, _log(rng, 1, min(100000, 300000000 // ((hq + hk) * d))))
        return _rotary(rows, hq, hk, d, dtype, axes, pairs, rng.choice(["far", "grid", "layout"]),
                       train=rng.random() < 0.5, norm=rng.random() < 0.85, interleaved=rng.random() < 0.3,
                       packed=rng.random() < 0.4)
    graph = rng.choice(["cache", "window", "rmat", "uniform"])
    hk = rng.choice([1, 2, 3, 4])
    h = hk * rng.choice([1, 1, 2, 3, 4])
    d = rng.choice([8, 16, 32, 40, 64, 128, rng.randrange(5, 120)])
    dv = rng.choice([d, 2 * d, 2 * d, rng.randrange(4, 200)])
    edges = _log(rng, 500, min(4000000, 1000000000 // (h * (2 * d + dv))))
    if graph == "cache":
        rows = min(_log(rng, 1, 96), max(1, edges // 8))
    elif graph == "window":
        rows = max(1, edges // min(_log(rng, 8, 512), edges))
    else:
        rows = max(1, edges // _log(rng, 3, 40))
    return _attention(graph, rows, edges, h, hk, d, dv, dtype, train=graph != "cache" and rng.random() < 0.6,
                      bias=rng.random() < 0.4, row_lam=rng.random() < 0.4, plan=rng.random() < 0.5)


# ---- inputs ------------------------------------------------------------------------------------------------------------
def _pattern(case, gen, dev):
    """-> rowptr, colidx, number of columns.  The edges are ``case["edges"]`` or, for a window, what fits before row 0."""
    m, e, graph = case["rows"], case["edges"], case["graph"]
    if graph == "cache":  # lengths spread over a factor of 16 around the mean, slots in shuffled pages of 16
        share = torch.exp(torch.rand(m, generator=gen, device=dev, dtype=torch.float64) * math.log(16.0))
        length = torch.floor(share / share.sum() * e).to(torch.int64)
        length[0] += e - length.sum()
        pages = (length + 15) // 16
        first_page = torch.cumsum(pages, 0) - pages
        rowptr = torch.zeros(m + 1, dtype=torch.int64, device=dev)
        rowptr[1:] = torch.cumsum(length, 0)
        total = int(pages.sum())
        table = torch.randperm(total, generator=gen, device=dev)
        row = torch.repeat_interleave(torch.arange(m, device=dev), length)
        t = torch.arange(e, device=dev) - rowptr[row]
        return rowptr.to(torch.int32), (table[first_page[row] + t // 16] * 16 + t % 16).to(torch.int32), total * 16
    if graph == "window":  # row i sees itself and the rows before it, as many as the mean says
        w = max(1, e // m)
        length = torch.clamp(torch.arange(1, m + 1, device=dev), max=w)
        rowptr = torch.zeros(m + 1, dtype=torch.int64, device=dev)
        rowptr[1:] = torch.cumsum(length, 0)
        row = torch.repeat_interleave(torch.arange(m, device=dev), length)
        col = row - length[row] + 1 + torch.arange(row.numel(), device=dev) - rowptr[row]
        return rowptr.to(torch.int32), col.to(torch.int32), m
    if graph == "rmat":  # recursive quadrants 0.57, 0.19, 0.19, 0.05: hub rows and rows without an edge
        bits = max(1, (m - 1).bit_length())
        row = torch.zeros(e, dtype=torch.int64, device=dev)
        col = torch.zeros(e, dtype=torch.int64, device=dev)
        for _ in range(bits):
            u = torch.rand(e, generator=gen, device=dev)
            row = row * 2 + (u >= 0.76)
            col = col * 2 + (((u >= 0.57) & (u < 0.76)) | (u >= 0.95))
        row, col = row % m, col % m
    else:
        row = torch.randint(0, m, (e,), generator=gen, device=dev)
        col = torch.randint(0, m, (e,), generator=gen, device=dev)
    key = torch.sort(row * m + col).values
    row, col = key // m, key % m
    rowptr = torch.zeros(m + 1, dtype=torch.int64, device=dev)
    rowptr[1:] = torch.cumsum(torch.bincount(row, minlength=m), 0)
    return rowptr, col.to(torch.int32), m  # 64-bit row pointers with 32-bit column ids


def _randn(gen, dev, dtype, *shape):
    return torch.randn(shape, generator=gen, device=dev, dtype=torch.float32).to(dtype)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    if case["op"] == "rotary":
        rows, hq, hk, d = case["rows"], case["hq"], case["hk"], case["d"]
        if case["packed"]:  # views of one projection of queries, keys and values
            proj = _randn(gen, dev, dtype, rows, hq + 2 * hk, d)
            q, k = proj[:, :hq], proj[:, hq:hq + hk]
        else:
            q, k = _randn(gen, dev, dtype, rows, hq, d), _randn(gen, dev, dtype, rows, hk, d)
        a, p = case["axes"], case["pairs"]
        if case["positions"] == "far":
            pos = torch.randint(0, 1 << 20, (rows, a), generator=gen, device=dev)
        elif case["positions"] == "grid":
            pos = torch.randint(0, 512, (rows, a), generator=gen, device=dev, dtype=torch.int32)
        else:
            pos = _randn(gen, dev, torch.float32, rows, a) * 30
        # the pairs are shared out among the axes in runs, each with its own ladder of frequencies
        freq = torch.zeros((a, p), dtype=torch.float64, device=dev)
        bound = [p * i // a for i in range(a + 1)]
        for i in range(a):
            n = bound[i + 1] - bound[i]
            freq[i, bound[i]:bound[i + 1]] = 10000.0 ** (-torch.arange(n, dtype=torch.float64, device=dev) / n)
        s = dict(case=case, q=q, k=k, pos=pos, freq=freq, wq=None, wk=None, eps=None)
        if case["norm"]:
            s.update(wq=1 + 0.1 * _randn(gen, dev, torch.float32, d), wk=1 + 0.1 * _randn(gen, dev, torch.float32, d), eps=EPS)
        if case["train"]:
            s.update(dq=_randn(gen, dev, dtype, rows, hq, d), dk=_randn(gen, dev, dtype, rows, hk, d))
            if own:
                for name in ("q", "k", "wq", "wk"):
                    if s[name] is not None:
                        s[name] = s[name].detach().requires_grad_()
        return s
    rowptr, colidx, n = _pattern(case, gen, dev)
    m, h, hk, d, dv, e = case["rows"], case["h"], case["hk"], case["d"], case["dv"], colidx.numel()
    s = dict(case=case, rowptr=rowptr, colidx=colidx, n=n, bias=None, plan=None,
             q=_randn(gen, dev, dtype, m, h, 2, d), k=_randn(gen, dev, dtype, n, hk, 2, d), v=_randn(gen, dev, dtype, n, hk, dv),
             scale=d ** -0.5)
    s["lam"] = 0.2 + 0.6 * torch.rand((m, h) if case["row_lam"] else (h,), generator=gen, device=dev)
    if case["bias"]:  # one edge in ten is dropped
        s["bias"] = _randn(gen, dev, torch.float32, e)
        s["bias"][torch.rand(e, generator=gen, device=dev) < 0.1] = -math.inf
    if case["train"]:
        s["do"] = _randn(gen, dev, dtype, m, h, dv)
        if own:
            from fusedmm_b200 import torch_op
            for name in ("q", "k", "v", "lam"):
                s[name] = s[name].detach().requires_grad_()
            if case["plan"]:  # a program with fixed edges keeps the transposed pattern beside the pattern
                s["plan"] = torch_op.csr_transpose(rowptr, colidx, n)
    return s


# ---- one pass ----------------------------------------------------------------------------------------------------------
def run(s):
    case = s["case"]
    if own:
        return _own_rotary(s) if case["op"] == "rotary" else _own_attention(s)
    return _plain_rotary(s) if case["op"] == "rotary" else _plain_attention(s)


def _own_rotary(s):
    from fusedmm_b200 import torch_op
    case = s["case"]
    q, k = torch_op.qk_norm_rotary(s["q"], s["k"], s["pos"], s["freq"], q_weight=s["wq"], k_weight=s["wk"], eps=s["eps"],
                                   interleaved=case["interleaved"])
    if not case["train"]:
        return q, k
    leaves = [s["q"], s["k"]] + ([s["wq"], s["wk"]] if case["norm"] else [])
    return (q.detach(), k.detach(), *torch.autograd.grad((q, k), leaves, (s["dq"], s["dk"])))


def _own_attention(s):
    from fusedmm_b200 import torch_op
    out = torch_op.diff_attention(s["rowptr"], s["colidx"], s["q"], s["k"], s["v"], s["lam"], bias=s["bias"],
                                  scale=s["scale"], transposed=s["plan"])
    if not s["case"]["train"]:
        return out
    return (out.detach(), *torch.autograd.grad(out, [s["q"], s["k"], s["v"], s["lam"]], s["do"]))


def _turn(x, cos, sin, p, interleaved):
    """Turns the pairs of the last axis by the angles; what lies behind the 2p rotated elements passes."""
    if interleaved:
        a, b = x[..., 0:2 * p:2], x[..., 1:2 * p:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    else:
        a, b = x[..., :p], x[..., p:2 * p]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    return torch.cat((turned, x[..., 2 * p:]), dim=-1)


def _plain_rotary(s):
    case, p = s["case"], s["case"]["pairs"]
    angle = s["pos"].double() @ s["freq"]  # 64 bits: positions go far
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    outs, grads, wgrads = [], [], []
    for name in ("q", "k"):
        x, w = s[name], s["w" + name]
        xf = x.float()
        if case["norm"]:
            r = torch.rsqrt((xf * xf).mean(-1, keepdim=True) + s["eps"])
            xn = xf * r
            y = xn * w
        else:
            y = xf
        outs.append(_turn(y, cos, sin, p, case["interleaved"]).to(x.dtype))
        if case["train"]:
            g = _turn(s["d" + name].float(), cos, -sin, p, case["interleaved"])
            if case["norm"]:
                wgrads.append((g * xn).sum((0, 1)))
                g = g * w
                g = r * (g - xn * (g * xn).mean(-1, keepdim=True))
            grads.append(g.to(x.dtype))
    return (*outs, *grads, *wgrads)


def _plain_attention(s):
    case = s["case"]
    m, n, h, e, dv = case["rows"], s["n"], case["h"], s["colidx"].numel(), case["dv"]
    group, dtype, train = h // case["hk"], s["q"].dtype, case["train"]
    dev = s["q"].device
    row = torch.repeat_interleave(torch.arange(m, device=dev), (s["rowptr"][1:] - s["rowptr"][:-1]).long(), output_size=e)
    col = s["colidx"].long()
    out = torch.empty((m, h, dv), dtype=dtype, device=dev)
    if train:
        dq = torch.empty_like(s["q"])
        dk = torch.zeros(s["k"].shape, device=dev)
        dvv = torch.zeros(s["v"].shape, device=dev)
        dlam = torch.zeros_like(s["lam"])
    for i in range(h):
        g = i // group
        qe, ke, ve = s["q"][row, i].float(), s["k"][col, g].float(), s["v"][col, g].float()
        lam = s["lam"][:, i] if case["row_lam"] else s["lam"][i].expand(m)
        score = (qe * ke).sum(-1) * s["scale"]
        if s["bias"] is not None:
            score = score + s["bias"][:, None]
        top = torch.full((m, 2), -math.inf, device=dev).scatter_reduce(0, row[:, None].expand(e, 2), score, "amax")
        top = torch.where(top == -math.inf, torch.zeros_like(top), top)
        pr = torch.exp(score - top[row])
        total = torch.zeros((m, 2), device=dev).index_add(0, row, pr)
        pr = pr / torch.where(total == 0, torch.ones_like(total), total)[row]
        weight = pr[:, 0] - lam[row] * pr[:, 1]
        out[:, i] = torch.zeros((m, dv), device=dev).index_add(0, row, weight[:, None] * ve).to(dtype)
        if not train:
            continue
        doe = s["do"][row, i].float()
        dvv[:, g].index_add_(0, col, weight[:, None] * doe)
        dp = (doe * ve).sum(-1, keepdim=True)
        delta = torch.zeros((m, 2), device=dev).index_add(0, row, pr * dp)
        sign = torch.stack((torch.ones_like(lam), -lam), dim=-1)
        ds = sign[row] * pr * (dp - delta[row]) * s["scale"]
        dq[:, i] = torch.zeros((m, 2, qe.shape[-1]), device=dev).index_add(0, row, ds[..., None] * ke).to(dtype)
        dk[:, g].index_add_(0, col, ds[..., None] * qe)
        if case["row_lam"]:
            dlam[:, i] = -delta[:, 1]
        else:
            dlam[i] = -delta[:, 1].sum()
    return (out, dq, dk.to(dtype), dvv.to(dtype), dlam) if train else out


# ---- the definition in 64 bits -------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotary":
        return _exact_rotary(s)
    if s["colidx"].numel() * case["h"] * (2 * case["d"] + case["dv"]) > 5_000_000_000:
        return None
    return _exact_attention(s)


def _exact_rotary(s):
    """Pairs as complex numbers times exp(i angle); the gradients by differentiation."""
    case, p = s["case"], s["case"]["pairs"]
    turn = torch.exp(1j * (s["pos"].double()[:, :, None] * s["freq"]).sum(1))[:, None]
    leaves, outs = [], []
    for name in ("q", "k"):
        x = s[name].detach().double().requires_grad_(case["train"])
        y = x
        if case["norm"]:
            w = s["w" + name].detach().double().requires_grad_(case["train"])
            y = x / torch.sqrt(x.square().sum(-1, keepdim=True) / case["d"] + s["eps"]) * w
            leaves.append((x, w))
        else:
            leaves.append((x, None))
        z = torch.complex(y[..., 0:2 * p:2], y[..., 1:2 * p:2]) if case["interleaved"] else torch.complex(y[..., :p], y[..., p:2 * p])
        z = z * turn
        parts = torch.view_as_real(z).reshape(*y.shape[:-1], 2 * p) if case["interleaved"] else torch.cat((z.real, z.imag), -1)
        outs.append(torch.cat((parts, y[..., 2 * p:]), -1))
    if not case["train"]:
        return tuple(outs)
    wanted = [x for x, _ in leaves] + [w for _, w in leaves if w is not None]
    grads = torch.autograd.grad(outs, wanted, (s["dq"].double(), s["dk"].double()))
    return (*[o.detach() for o in outs], *grads)


def _exact_attention(s):
    """Edges summed through differences of a running total would lose digits, so each row's sums go through a product with
    its indicator (a sparse matrix); the gradients by differentiation, one query head at a time."""
    case = s["case"]
    m, n, h, e = case["rows"], s["n"], case["h"], s["colidx"].numel()
    dev, group = s["q"].device, case["h"] // case["hk"]
    row = torch.searchsorted(s["rowptr"].long(), torch.arange(e, device=dev), right=True) - 1
    col = s["colidx"].long()
    keep = None if s["bias"] is None else s["bias"] > -math.inf
    if keep is not None:
        row, col = row[keep], col[keep]
    rows_of = torch.sparse_coo_tensor(torch.stack((row, torch.arange(row.numel(), device=dev))),
                                      torch.ones(row.numel(), dtype=torch.float64, device=dev), (m, row.numel()),
                                      check_invariants=False)
    outs = []
    total = dict(q=torch.zeros(s["q"].shape, dtype=torch.float64, device=dev), k=torch.zeros(s["k"].shape, dtype=torch.float64, device=dev),
                 v=torch.zeros(s["v"].shape, dtype=torch.float64, device=dev), lam=torch.zeros(s["lam"].shape, dtype=torch.float64, device=dev))
    for i in range(h):
        g, train = i // group, case["train"]
        q = s["q"][:, i].detach().double().requires_grad_(train)
        k, v = (s[t][:, g].detach().double().requires_grad_(train) for t in ("k", "v"))
        lam = s["lam"][..., i].detach().double().requires_grad_(train)
        weight = 0
        for c in range(2):
            score = s["scale"] * torch.einsum("ed,ed->e", q[row, c], k[col, c])
            if keep is not None:
                score = score + s["bias"][keep].double()
            weights = torch.exp(score)[:, None]  # scores stay far below 700
            share = weights / torch.sparse.mm(rows_of, weights)[row]
            weight = share if c == 0 else weight - (lam[row, None] if case["row_lam"] else lam) * share
        o = torch.sparse.mm(rows_of, weight * v[col])
        outs.append(o.detach())
        if train:
            for t, grad in zip(("q", "k", "v", "lam"), torch.autograd.grad(o, (q, k, v, lam), s["do"][:, i].double())):
                if t == "lam":
                    total[t][..., i] += grad
                else:
                    total[t][:, i if t == "q" else g] += grad
    out = torch.stack(outs, 1)
    return (out, total["q"], total["k"], total["v"], total["lam"]) if case["train"] else out


# ---- what a pass cannot do without -----------------------------------------------------------------------------------------
def work(case):
    b = SIZE[case["dtype"]]
    if case["op"] == "rotary":
        elements = case["rows"] * (case["hq"] + case["hk"]) * case["d"]
        positions = case["rows"] * case["axes"] * (8 if case["positions"] == "far" else 4)
        if case["train"]:  # forward reads x and writes y; backward reads x and dy and writes dx
            return {"bytes": 5 * elements * b + 2 * positions, "flops": 22 * elements}
        return {"bytes": 2 * elements * b + positions, "flops": 7 * elements}
    m, e, h, hk, d, dv = (case[t] for t in ("rows", "edges", "h", "hk", "d", "dv"))
    n = m if case["graph"] != "cache" else e
    if case["graph"] == "window":
        w = max(1, e // m)
        e = w * m - w * (w - 1) // 2 if m >= w else m * (m + 1) // 2
    q, kv, out = m * h * 2 * d * b, n * hk * (2 * d + dv) * b, m * h * dv * b
    ids = e * (4 + (4 if case["bias"] else 0)) + (m + 1) * 4 + (m if case["row_lam"] else 1) * h * 4
    forward = e * h * (4 * d + 4 * dv)
    if not case["train"]:
        return {"bytes": q + kv + out + ids, "flops": forward}
    # backward: both scores and dP once more, then dq, dk and dv
    return {"bytes": 3 * (q + kv) + 2 * out + 2 * ids, "flops": forward + e * h * (12 * d + 4 * dv)}
