"""GPU: the state-space layer's serving operators (norm with 8-bit output, block-scaled 8-bit product, causal
convolution, scan, single-token step) against their formulas in 64 bits, in both builds.

Tolerances, element by element: a 16-bit output is off by half a step, EPS / 2 of its value; fp32 arithmetic adds a
count of roundings of 2^-24, each relative to the sum of the magnitudes that enter (the bounds below count them
generously, as n additions in any order cost at most n roundings)."""
import math

import pytest
import torch

from actalker_amd import _lib, ops

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.fixture(autouse=True)
def _seed():
    torch.manual_seed(99)


@pytest.fixture(autouse=True, params=["bf16", "fp16"])
def act(request):
    with ops.compute_dtype(torch.float16 if request.param == "fp16" else torch.bfloat16):
        yield request.param


def half():
    return torch.finfo(ops.act_dtype()).eps / 2


def low(*shape, scale=1.0):
    return (torch.randn(*shape) * scale).to(ops.act_dtype())


def near(got, want, tol, what=""):
    """|got - want| <= tol everywhere (64 bits)."""
    d = (got.double().cpu() - want).abs()
    bad = ~(d <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {d[bad].max()} where {tol[bad].max()} is allowed"


# ------------------------------------------------------------------------------------------ norm
def norm_ref(x, gamma, eps, res):
    s = x.double() if res is None else x.double() + res.double()
    y = s / (s.square().mean(1, keepdim=True) + eps).sqrt()
    return (y if gamma is None else y * gamma.double()), s


# a row's squares are summed in at most C / 64 + 8 additions a lane and two joins; the root halves the error, the
# quotient, root and two products add a few more: C / 64 + 32 roundings cover every kernel
def norm_tol(C):
    return (C / 64 + 32) * U


def least_normal():
    return torch.finfo(ops.act_dtype()).tiny * torch.finfo(ops.act_dtype()).eps      # one subnormal step


@pytest.mark.parametrize("M,C", [(1, 1), (1, 64), (3, 127), (5, 320), (2, 1018), (7, 1280), (129, 640), (3, 1600), (4, 2560),
                                 (2, 5120), (3, 8000), (1, 16384), (2, 16392), (2, 20001)])
@pytest.mark.parametrize("res", ["none", "same", "float"])
def test_rmsnorm(dev, M, C, res):
    x, gamma = low(M, C), 1 + 0.2 * torch.randn(C)
    r = None if res == "none" else (3 * torch.randn(M, C)).to(ops.act_dtype() if res == "same" else torch.float32)
    got = ops.rmsnorm(x.to(dev), gamma.to(dev), 1e-5, residual=None if r is None else r.to(dev))
    y, s = norm_ref(x, gamma, 1e-5, r)
    if r is not None:
        got, kept = got
        assert kept.dtype == r.dtype
        step = half() if res == "same" else U
        near(kept, s, s.abs() * (step + U) + least_normal(), "sum")
    near(got, y, y.abs() * (half() + norm_tol(C)) + least_normal(), "y")


@pytest.mark.parametrize("M,C", [(1, 5), (2, 128), (3, 200), (5, 320), (3, 1306), (130, 640), (4, 2560), (2, 5120), (1, 16640)])
@pytest.mark.parametrize("res", ["none", "float"])
def test_rmsnorm_fp8(dev, M, C, res):
    x, gamma = low(M, C), 1 + 0.2 * torch.randn(C)
    x[0, : min(C, 128)] = 0                       # a block of zeros
    r = None if res == "none" else torch.randn(M, C)
    if r is not None:
        r[0, : min(C, 128)] = 0
    out = ops.rmsnorm_fp8(x.to(dev), gamma.to(dev), 1e-5, residual=None if r is None else r.to(dev))
    y, s = norm_ref(x, gamma, 1e-5, r)
    check_fp8(out[0], out[1], y, norm_tol(C))
    if r is not None:
        near(out[2], s, s.abs() * 2 * U, "sum")


def check_fp8(q, scale, y, rel):
    """Codes times scales against y: e4m3 is off by 2^-4 of the value, or half a subnormal step, 2^-10, of the scale."""
    M, C = y.shape
    kb = -(-C // 128)
    assert q.dtype == ops.FP8 and q.shape == (M, C) and scale.shape == (M, kb)
    pad = torch.nn.functional.pad(y, (0, kb * 128 - C)).view(M, kb, 128)
    want = pad.abs().amax(2).clamp_min(2.0 ** -100) / 448
    near(scale, want, want * (rel + 4 * U), "scale")
    big = want.repeat_interleave(128, 1)[:, :C]
    near(q.float().cpu().double() * scale.double().cpu().repeat_interleave(128, 1)[:, :C], y,
         torch.maximum(y.abs() * 2.0 ** -4, big * 2.0 ** -10) * (1 + 2.0 ** -10) + y.abs() * (rel + 4 * U), "codes")


def test_quant_fp8_strided_and_special(dev):
    x = low(9, 700, scale=5.0)
    x[2, 130] = float("nan")
    x[3, 3] = float("inf")
    d = x.to(dev)
    q, s = ops.quant_fp8(d)
    q2, s2 = ops.quant_fp8(torch.cat([d, d], 1)[:, 700:])        # rows at another stride
    assert torch.equal(q.view(torch.uint8), q2.view(torch.uint8)) and torch.equal(s.nan_to_num(7), s2.nan_to_num(7))
    rows = [0, 1, 4, 5, 6, 7, 8]
    check_fp8(q[rows], s[rows], x[rows].double(), 4 * U)
    assert torch.isnan(s[2, 1]) and torch.isnan(q.float()[2, 128:256]).all()
    assert not torch.isnan(q.float()[2, :128]).any() and not torch.isnan(s[2, 2:]).any()
    assert torch.isinf(s[3, 0]) and torch.isnan(q.float()[3, 3]) and (q.float()[3, :3] == 0).all()


def test_rmsnorm_in_place_and_empty(dev):
    x, r, gamma = low(33, 640), torch.randn(33, 640), torch.ones(640)
    y, s = norm_ref(x, gamma, 1e-5, r)
    xd, rd = x.to(dev), r.to(dev)
    got, kept = ops.rmsnorm(xd, gamma.to(dev), 1e-5, residual=rd, sum_out=rd, out=xd)
    assert got.data_ptr() == xd.data_ptr() and kept.data_ptr() == rd.data_ptr()
    near(xd, y, y.abs() * (half() + norm_tol(640)) + least_normal())
    near(rd, s, s.abs() * 2 * U)
    e = torch.empty(0, 640, device=dev, dtype=ops.act_dtype())
    assert ops.rmsnorm(e, gamma.to(dev)).shape == (0, 640)
    q, sc = ops.rmsnorm_fp8(e, None)
    assert q.shape == (0, 640) and sc.shape == (0, 5)


# ------------------------------------------------------------------------------------------ product
def wide_of(q, s, rows):
    big = s.double().repeat_interleave(rows, 0)[: q.shape[0]].repeat_interleave(128, 1)[:, : q.shape[1]]
    return q.float().double() * big


@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 16, 128), (1, 2560, 2560), (2, 130, 144), (7, 640, 320), (16, 1000, 1024), (17, 257, 96),
                                   (33, 2090, 1360), (64, 5120, 640), (65, 96, 2000), (130, 384, 4096), (256, 256, 128),
                                   (300, 320, 320), (513, 1030, 1306), (1000, 512, 2560), (2049, 768, 640)])
@pytest.mark.parametrize("case", ["plain", "f32_bias", "res"])
def test_gemm_fp8(dev, M, N, K, case):
    a, w = low(M, K), torch.randn(N, K) / math.sqrt(K)
    q, s = ops.quant_fp8(a.to(dev))
    wq, wsc = ops.pack_fp8(w.to(dev))
    bias = torch.randn(N) if case == "f32_bias" else None
    res = low(M, N) if case == "res" else None
    out = ops.gemm_fp8(q, s, wq, wsc, bias=None if bias is None else bias.to(dev),
                       residual=None if res is None else res.to(dev), out_f32=case == "f32_bias")
    A, W = wide_of(q.cpu(), s.cpu(), 1), wide_of(wq.cpu(), wsc.cpu(), 128)
    want, size = A @ W.t(), A.abs() @ W.abs().t()
    for more in (bias, res):
        if more is not None:
            want, size = want + more.double(), size + more.double().abs()
    assert out.shape == (M, N) and out.dtype == (torch.float32 if case == "f32_bias" else ops.act_dtype())
    # at most K additions and four products and sums a term
    tol = size * (K + 8) * U
    if case != "f32_bias":
        tol = tol + want.abs() * half() + least_normal() + unit_loss(A, W, dev)
    near(out, want, tol)


def unit_loss(A, W, dev):
    """What the 8-bit matrix unit may drop. It adds products in groups of 8 consecutive k, aligned to the group's largest,
    and cuts each below 2^-13 of the power of two at or under that one; products of two 4-bit significands have 8 bits, so
    the largest loses nothing and each of the other 7 less than 2^-13 of it: 7 * 2^-13 of every group's largest product.
    (fp32 outputs do not use this unit.)"""
    K = A.shape[1]
    A, W = (torch.nn.functional.pad(t.abs(), (0, -K % 8)).float().to(dev) for t in (A, W))
    loss = torch.zeros(A.shape[0], W.shape[0], device=dev)
    for k in range(0, A.shape[1], 8):
        top = A[:, k, None] * W[:, k]
        for j in range(k + 1, k + 8):
            top = torch.maximum(top, A[:, j, None] * W[:, j])
        loss += top
    return loss.double().cpu() * 7 * 2.0 ** -13 * (1 + 2.0 ** -10)


def test_gemm_fp8_scales_of_any_stride_and_range(dev):
    """Scales far apart, in rows or in columns, and a NaN scale that reaches its rows alone."""
    M, N, K = 70, 200, 520
    q = torch.randn(M, K).to(ops.FP8)
    w = torch.randn(N, K).to(ops.FP8)
    s, ws = torch.exp(6 * torch.randn(M, 5)), torch.exp(6 * torch.randn(2, 5)) * 1e-3
    one = ops.gemm_fp8(q.to(dev), s.to(dev), w.to(dev), ws.to(dev), out_f32=True)
    two = ops.gemm_fp8(q.to(dev), s.t().contiguous().to(dev).t(), w.to(dev), ws.t().contiguous().to(dev).t(), out_f32=True)
    assert torch.equal(one, two)
    A, W = wide_of(q, s, 1), wide_of(w, ws, 128)
    near(one, A @ W.t(), (A.abs() @ W.abs().t()) * (K + 8) * U)
    s[3, 2] = float("nan")
    bad = ops.gemm_fp8(q.to(dev), s.to(dev), w.to(dev), ws.to(dev), out_f32=True)
    assert torch.isnan(bad[3]).all() and torch.equal(bad[[0, 1, 2, 4, 69]], one[[0, 1, 2, 4, 69]])


@pytest.mark.parametrize("M", [1, 40, 300])
def test_gemm_fp8_writes_only_its_output(dev, M):
    """Output columns inside a wider buffer, the residual updated in place, the same bits on every call."""
    N, K = 328, 640
    q, s = ops.quant_fp8(low(M, K).to(dev))
    wq, wsc = ops.pack_fp8(torch.randn(N, K).to(dev))
    buf = torch.full((M + 1, 512), 5.0, device=dev, dtype=ops.act_dtype())
    out = ops.gemm_fp8(q, s, wq, wsc, out=buf[:M, 64:64 + N])
    want = ops.gemm_fp8(q, s, wq, wsc)
    assert torch.equal(out, want)
    rest = buf.clone()
    rest[:M, 64:64 + N] = 5.0
    assert (rest == 5.0).all()
    r = low(M, N).to(dev)
    sum_ = ops.gemm_fp8(q, s, wq, wsc, residual=r)
    assert torch.equal(ops.gemm_fp8(q, s, wq, wsc, residual=r, out=r), sum_)


# ------------------------------------------------------------------------------------------ sequences
def cuts_of(lens):
    c = [0]
    for n in lens:
        c.append(c[-1] + n)
    return c


def conv_ref(x, w, bias, cuts, state, fresh, silu):
    """(y, its tolerance, new state); y NaN where no sequence holds the row."""
    T, D = x.shape
    W = w.shape[1]
    y, tol = torch.full((T, D), math.nan, dtype=torch.float64), torch.zeros(T, D, dtype=torch.float64)
    new = state.double().clone()
    for i, (a, b) in enumerate(zip(cuts, cuts[1:])):
        if a == b:
            continue
        head = torch.zeros(W - 1, D, dtype=torch.float64) if fresh[i] else state[i].double()
        xs = torch.cat([head, x[a:b].double()])
        v = bias.double() + sum(xs[j:j + b - a] * w[:, j].double() for j in range(W))
        size = bias.double().abs() + sum((xs[j:j + b - a] * w[:, j].double()).abs() for j in range(W))
        y[a:b] = v * torch.sigmoid(v) if silu else v
        # silu's slope is below 1.1; its own exponential, sum and quotient cost 8 roundings and the argument's scaling |v| more
        t = 1.1 * size * (W + 1) * U
        if silu:
            t = t + y[a:b].abs() * (8 + v.abs() * 2) * U
        tol[a:b] = t + y[a:b].abs() * half() + least_normal()
        new[i] = xs[-(W - 1):]
    return y, tol, new


LENS = [[1], [2], [3, 0, 1, 2], [17], [16, 16, 1], [15, 2, 40, 1, 1, 30], [100, 0, 0, 29], [33] * 9]


@pytest.mark.parametrize("lens", LENS, ids=str)
@pytest.mark.parametrize("D,W,silu", [(8, 4, True), (64, 2, True), (130, 3, False), (520, 4, True)])
def test_causal_conv(dev, lens, D, W, silu):
    cuts = cuts_of(lens)
    T, n = cuts[-1] + 3, len(lens)                # three rows behind the last sequence
    x, w, bias = low(T, D), torch.randn(D, W), torch.randn(D)
    state, fresh = low(n, W - 1, D), torch.rand(n) < 0.3
    y, tol, new = conv_ref(x, w, bias, cuts, state, fresh, silu)
    perm = torch.randperm(n + 2)[:n]              # places in a larger pool
    pool = low(n + 2, W - 1, D)
    pool[perm] = state
    rows = torch.cat([low(T, D), x, low(T, D)], 1).to(dev)            # the middle columns of wider rows
    out = torch.full((T, D), 3.0, device=dev, dtype=ops.act_dtype())
    kept = pool.to(dev)
    ops.causal_conv(rows[:, D:2 * D], w.to(dev), bias.to(dev), silu=silu, starts=torch.tensor(cuts, dtype=torch.int32, device=dev),
                    state=kept, slots=perm.to(torch.int32).to(dev), fresh=fresh.to(dev), out=out)
    near(out[:cuts[-1]], y[:cuts[-1]], tol[:cuts[-1]])
    assert (out[cuts[-1]:] == 3.0).all()
    want = pool.clone()
    want[perm] = new.to(ops.act_dtype())
    assert torch.equal(kept.cpu(), want)


def scan_ref(u, dl, A, B, C, D, z, bias, softplus, cuts, state, fresh):
    """(y, tolerance, new state, its tolerance). Every row costs a state at most 4 roundings and the time step's 12, all
    relative to the sum of magnitudes `big`, which runs through the same recurrence; a decay's exponent is off by 14
    roundings of |dt A|, and x exp(-x) < 0.4 keeps that below 6 more a row."""
    T, dim = u.shape
    N = A.shape[1]
    G = B.shape[1] // N
    grp = torch.arange(dim) // (dim // G)
    u, dl, A, B, C = (t.double() for t in (u, dl, A, B, C))
    y, tol = torch.full((T, dim), math.nan, dtype=torch.float64), torch.zeros(T, dim, dtype=torch.float64)
    new, ntol = state.double().clone(), torch.zeros_like(state, dtype=torch.float64)
    for i, (a, b) in enumerate(zip(cuts, cuts[1:])):
        if a == b:
            continue
        h = torch.zeros(dim, N, dtype=torch.float64) if fresh[i] else state[i].double().clone()
        big = h.abs()
        for t in range(a, b):
            x = dl[t] + (0 if bias is None else bias.double())
            dt = torch.nn.functional.softplus(x, threshold=60) if softplus else x
            e = torch.exp(dt[:, None] * A)
            add = (dt * u[t])[:, None] * B[t].view(G, N)[grp]
            h, big = e * h + add, e * big + add.abs()
            c = C[t].view(G, N)[grp]
            v, size = (h * c).sum(1), (big * c.abs()).sum(1)
            if D is not None:
                v, size = v + D.double() * u[t], size + (D.double() * u[t]).abs()
            err = size * (24 * (t - a + 1) + N + 16) * U
            if z is not None:
                g = z[t].double() * torch.sigmoid(z[t].double())
                v, err = v * g, err * g.abs() + (v * g).abs() * (10 + 2 * z[t].double().abs()) * U
            y[t], tol[t] = v, err + v.abs() * half() + least_normal()
        new[i], ntol[i] = h, big * (24 * (b - a) + 16) * U
    return y, tol, new, ntol


def scan_case(lens, dim, N, G, kind, extra=0):
    T = sum(lens) + extra
    kt = ops.act_dtype() if kind == "low" else torch.float32
    bc = torch.randn(T, 2 * G * N).to(kt)
    return dict(u=low(T, dim), delta=(0.7 * torch.randn(T, dim)).to(kt), A=-torch.exp(0.5 * torch.randn(dim, N)),
                B=bc[:, :G * N], C=bc[:, G * N:], D=torch.randn(dim), z=low(T, dim), delta_bias=torch.randn(dim) - 2,
                state=torch.randn(len(lens), dim, N))


def to(dev, s, *names):
    return {k: s[k].to(dev) for k in names}


IN = ("u", "delta", "A", "B", "C", "D", "z", "delta_bias")


@pytest.mark.parametrize("lens", LENS + [[300], [257, 0, 500], [64, 64, 64], [63, 1, 129, 200, 7]], ids=str)
@pytest.mark.parametrize("dim,N,G,kind", [(8, 16, 1, "low"), (70, 16, 1, "float"), (128, 16, 2, "low"), (40, 5, 2, "float"),
                                          (64, 8, 1, "low"), (36, 24, 1, "low"), (20, 64, 1, "float")])
def test_ssm_scan(dev, lens, dim, N, G, kind):
    cuts = cuts_of(lens)
    s = scan_case(lens, dim, N, G, kind, extra=2)
    fresh = torch.rand(len(lens)) < 0.3
    y, tol, new, ntol = scan_ref(*(s[k] for k in IN), True, cuts, s["state"], fresh)
    kept = s["state"].to(dev)
    out = torch.full(s["u"].shape, 3.0, device=dev, dtype=ops.act_dtype())
    ops.ssm_scan(**to(dev, s, *IN), starts=torch.tensor(cuts, dtype=torch.int32, device=dev), state=kept,
                 fresh=fresh.to(dev), out=out)
    near(out[:cuts[-1]], y[:cuts[-1]], tol[:cuts[-1]], "y")
    assert (out[cuts[-1]:] == 3.0).all()
    near(kept, new, ntol, "state")


@pytest.mark.parametrize("nb,L", [(1, 40), (1, 700), (5, 33), (3, 200), (40, 1)])
@pytest.mark.parametrize("plain", [False, True])
def test_ssm_scan_equal_sequences(dev, nb, L, plain):
    """``nb`` equal sequences; without gate, skip, bias, softplus and state as well."""
    s = scan_case([L] * nb, 48, 16, 2, "float")
    cuts = cuts_of([L] * nb)
    args = to(dev, s, "u", "delta", "A", "B", "C")
    if plain:
        s["delta"] = s["delta"].abs()
        args["delta"] = s["delta"].to(dev)
        zero = torch.zeros_like(s["state"])
        y, tol, _, _ = scan_ref(*(s[k] for k in IN[:5]), None, None, None, False, cuts, zero, [False] * nb)
        near(ops.ssm_scan(**args, softplus=False, nb=nb), y, tol)
    else:
        y, tol, new, ntol = scan_ref(*(s[k] for k in IN), True, cuts, s["state"], [False] * nb)
        kept = s["state"].to(dev)
        near(ops.ssm_scan(**to(dev, s, *IN), nb=nb, state=kept), y, tol)
        near(kept, new, ntol)


def test_ssm_scan_strong_decay_and_growth(dev):
    """Time steps that forget everything in one row, none at all, A = 0 and A > 0, and a NaN that stays in its channel."""
    lens = [90, 30]
    s = scan_case(lens, 16, 16, 1, "float")
    s["delta"][5] = 80.0
    s["delta"][6] = -200.0
    s["A"][3] = 0.0
    s["A"][4] = 0.01
    cuts = cuts_of(lens)
    y, tol, new, ntol = scan_ref(*(s[k] for k in IN), True, cuts, s["state"], [False, True])
    kept = s["state"].to(dev)
    run = lambda k: ops.ssm_scan(**to(dev, s, *IN), starts=torch.tensor(cuts, dtype=torch.int32, device=dev), state=k,   # noqa: E731
                                 fresh=torch.tensor([False, True], device=dev))
    out = run(kept)
    near(out, y, tol)
    near(kept, new, ntol)
    s["u"][7, 2] = float("nan")
    out2 = run(s["state"].to(dev))
    assert torch.isnan(out2[7:90, 2]).all() and not torch.isnan(out2[:7]).any() and not torch.isnan(out2[90:]).any()
    keep = [c for c in range(16) if c != 2]
    assert torch.equal(out2[:, keep], out[:, keep])


@pytest.mark.parametrize("n,dim,N,G,W", [(1, 8, 16, 1, 4), (3, 70, 16, 2, 3), (300, 24, 16, 1, 2), (5, 64, 5, 1, 4), (9, 33, 64, 1, 4),
                                         (4, 2560, 16, 1, 4)])
def test_steps(dev, n, dim, N, G, W):
    """One token of each sequence through convolution and scan, with a padded batch: two sequences without a place."""
    s = scan_case([1] * n, dim, N, G, "low")
    w, bias, cst = torch.randn(dim, W), torch.randn(dim), low(n, W - 1, dim)
    cuts = list(range(n + 1))
    slots = torch.arange(n, dtype=torch.int32)
    if n > 2:
        slots[1], slots[2] = -1, n
    live = [i for i in range(n) if 0 <= slots[i] < n]
    dead = [i for i in range(n) if i not in live]
    y, tol, new = conv_ref(s["u"], w, bias, cuts, cst, [False] * n, True)
    kept = cst.to(dev)
    out = torch.full((n, dim), 3.0, device=dev, dtype=ops.act_dtype())
    ops.causal_conv_step(s["u"].to(dev), w.to(dev), bias.to(dev), state=kept, slots=slots.to(dev), out=out)
    near(out[live], y[live], tol[live])
    assert (out[dead] == 3.0).all() and torch.equal(kept.cpu()[dead], cst[dead])
    assert torch.equal(kept.cpu()[live], new[live].to(ops.act_dtype()))
    y, tol, new, ntol = scan_ref(*(s[k] for k in IN), True, cuts, s["state"], [False] * n)
    kept = s["state"].to(dev)
    out.fill_(3.0)
    ops.ssm_step(**to(dev, s, *IN), state=kept, slots=slots.to(dev), out=out)
    near(out[live], y[live], tol[live])
    near(kept[live], new[live], ntol[live])
    assert (out[dead] == 3.0).all() and torch.equal(kept.cpu()[dead], s["state"][dead])


def test_padding_sequences_in_prompts(dev):
    lens = [50, 90, 20, 130]
    cuts = cuts_of(lens)
    s = scan_case(lens, 64, 16, 1, "low")
    slots = torch.tensor([2, 7, 0, 1], dtype=torch.int32, device=dev)       # the second one has no place
    st = torch.tensor(cuts, dtype=torch.int32, device=dev)
    order = s["state"][[2, 0, 0, 1]]
    y, tol, new, ntol = scan_ref(*(s[k] for k in IN), True, cuts, order, [False] * 4)
    kept = s["state"][:3].to(dev)
    out = torch.full(s["u"].shape, 3.0, device=dev, dtype=ops.act_dtype())
    ops.ssm_scan(**to(dev, s, *IN), starts=st, state=kept, slots=slots, out=out)
    live = [t for t in range(cuts[-1]) if not 50 <= t < 140]
    near(out[live], y[live], tol[live])
    assert (out[50:140] == 3.0).all()
    near(kept, new[[2, 3, 0]], ntol[[2, 3, 0]])
    w, bias, cst = torch.randn(64, 4), torch.randn(64), low(3, 3, 64)
    yc, tolc, newc = conv_ref(s["u"], w, bias, cuts, cst[[2, 0, 0, 1]], [False] * 4, True)
    kept = cst.to(dev)
    out.fill_(3.0)
    ops.causal_conv(s["u"].to(dev), w.to(dev), bias.to(dev), starts=st, state=kept, slots=slots, out=out)
    near(out[live], yc[live], tolc[live])
    assert (out[50:140] == 3.0).all()
    assert torch.equal(kept.cpu(), newc[[2, 3, 0]].to(ops.act_dtype()))


def test_offsets_that_lie(dev):
    """Offsets out of order or out of range, and slots out of range, touch nothing outside the tensors."""
    T, dim = 200, 64
    s = scan_case([T], dim, 16, 1, "low")
    guard = torch.full((3 * T, dim), 3.0, device=dev, dtype=ops.act_dtype())
    pool = torch.full((6, dim, 16), 3.0, device=dev)
    cpool = torch.full((6, 3, dim), 3.0, device=dev, dtype=ops.act_dtype())
    w = torch.randn(dim, 4, device=dev)
    for offs in ([-5, 50, 1 << 30], [150, 20, 90], [7, 7, 7], [300, 400, 500], [90, 10, 0]):
        st = torch.tensor(offs, dtype=torch.int32, device=dev)
        sl = torch.tensor([1, 1 << 30], dtype=torch.int32, device=dev)
        ops.ssm_scan(**to(dev, s, *IN), starts=st, state=pool[2:4], slots=sl, out=guard[T:2 * T])
        ops.causal_conv(s["u"].to(dev), w, starts=st, state=cpool[2:4], slots=sl, out=guard[T:2 * T])
    assert (guard[:T] == 3.0).all() and (guard[2 * T:] == 3.0).all()
    for p in (pool, cpool):
        assert (p[:3] == 3.0).all() and (p[4:] == 3.0).all()


# ------------------------------------------------------------------------------------------ together
class Layer:
    """One gated state-space layer in 8-bit products, as a server runs it."""

    def __init__(self, dev, width=256, inner=384, N=16, R=16, W=4):
        self.w, self.d, self.N, self.R = width, inner, N, R
        pk = lambda n, k: ops.pack_fp8(torch.randn(n, k, device=dev) / math.sqrt(k))                 # noqa: E731
        self.gamma = 1 + 0.1 * torch.randn(width, device=dev)
        self.win, self.wx, self.wout = pk(2 * inner, width), pk(R + 2 * N, inner), pk(width, inner)
        self.wdt = (torch.randn(inner, R, device=dev) / 4).to(ops.act_dtype())
        self.cw, self.cb = torch.randn(inner, W, device=dev) / 2, 0.1 * torch.randn(inner, device=dev)
        self.A, self.D = -torch.exp(0.3 * torch.randn(inner, N, device=dev)), torch.ones(inner, device=dev)
        self.dtb = torch.randn(inner, device=dev) - 3

    def states(self, n, dev):
        return (torch.zeros(n, 3, self.d, device=dev, dtype=ops.act_dtype()), torch.zeros(n, self.d, self.N, device=dev))

    def __call__(self, x, stream, states, starts=None):
        q, s, stream = ops.rmsnorm_fp8(x, self.gamma, residual=stream)
        xz = ops.gemm_fp8(q, s, *self.win)
        xi, z = xz[:, :self.d], xz[:, self.d:]
        step = starts is None
        u = ops.causal_conv_step(xi, self.cw, self.cb, state=states[0]) if step else \
            ops.causal_conv(xi, self.cw, self.cb, state=states[0], starts=starts)
        p = ops.gemm_fp8(*ops.quant_fp8(u), *self.wx)
        delta = ops.gemm(p, self.wdt, out_f32=True)
        kw = dict(D=self.D, z=z, delta_bias=self.dtb, state=states[1])
        b, c = p[:, self.R:self.R + self.N], p[:, self.R + self.N:]
        y = ops.ssm_step(u, delta, self.A, b, c, **kw) if step else ops.ssm_scan(u, delta, self.A, b, c, starts=starts, **kw)
        return ops.gemm_fp8(*ops.quant_fp8(y), *self.wout), stream


def test_layer_prompt_then_tokens(dev):
    """A prompt in one piece, in two pieces, and its last tokens one by one: the same sequences, so the same outputs up
    to roundings that the 8-bit codes pass on (a code that falls to the other side moves by 2^-3 of its value; the
    outputs of the two runs are compared in the mean, at one 8-bit rounding, 2^-4)."""
    lay = Layer(dev)
    lens, n = [70, 131], 2
    T = sum(lens)
    x, r = low(T, 256).to(dev), low(T, 256).to(dev)
    st = torch.tensor(cuts_of(lens), dtype=torch.int32, device=dev)
    whole = lay.states(n, dev)
    y, stream = lay(x, r, whole, st)
    at = lambda k: torch.cat([torch.arange(a + k[0], a + k[1]) if k[1] is not None else torch.arange(a + k[0], b)   # noqa: E731
                              for a, b in zip(cuts_of(lens), cuts_of(lens)[1:])])
    parts = lay.states(n, dev)
    first = [n_ - 40 for n_ in lens]
    idx = torch.cat([torch.arange(c, c + f) for c, f in zip(cuts_of(lens), first)]).to(dev)
    ya, _ = lay(x[idx], r[idx], parts, torch.tensor(cuts_of(first), dtype=torch.int32, device=dev))
    idx2 = torch.cat([torch.arange(c + f, c + f + 37) for c, f in zip(cuts_of(lens), first)]).to(dev)
    yb, _ = lay(x[idx2], r[idx2], parts, torch.tensor([0, 37, 74], dtype=torch.int32, device=dev))
    rel = lambda a, b: float((a.double() - b.double()).norm() / b.double().norm())                 # noqa: E731
    assert torch.equal(stream, (x.float() + r.float()).to(ops.act_dtype()))
    assert rel(ya, y[idx]) < 2.0 ** -4 and rel(yb, y[idx2]) < 2.0 ** -4
    for k in range(3):
        idx3 = torch.tensor([c + f + 37 + k for c, f in zip(cuts_of(lens), first)], device=dev)
        yc, _ = lay(x[idx3], r[idx3], parts)
        assert rel(yc, y[idx3]) < 2.0 ** -4
    assert rel(parts[1], whole[1]) < 2.0 ** -4 and rel(parts[0], whole[0]) < 2.0 ** -4


def test_layer_step_in_a_graph_and_on_a_stream(dev):
    """A captured token step, replayed with eager work between, gives the eager run's bits; so does a side stream."""
    lay = Layer(dev)
    n = 5
    xs, rs = [low(n, 256).to(dev) for _ in range(6)], [low(n, 256).to(dev) for _ in range(6)]
    eager, es = [], lay.states(n, dev)
    for x, r in zip(xs, rs):
        eager.append([t.clone() for t in lay(x, r, es)])
    x, r, gs = xs[0].clone(), rs[0].clone(), lay.states(n, dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        lay(x, r, lay.states(n, dev))
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = lay(x, r, gs)
    for k in range(6):
        x.copy_(xs[k])
        r.copy_(rs[k])
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], eager[k][0]) and torch.equal(out[1], eager[k][1])
        lay(xs[0], rs[0], lay.states(n, dev))
    assert torch.equal(gs[1], es[1]) and torch.equal(gs[0], es[0])
    st = torch.tensor([0, 100, 230], dtype=torch.int32, device=dev)
    xp, rp = low(230, 256).to(dev), low(230, 256).to(dev)
    a, b = lay.states(2, dev), lay.states(2, dev)
    want = lay(xp, rp, a, st)[0]
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = lay(xp, rp, b, st)[0]
    side.synchronize()
    assert torch.equal(got, want) and torch.equal(a[1], b[1])


# ------------------------------------------------------------------------------------------ refusals
def test_refusals(dev):
    dt = ops.act_dtype()
    x, g = low(4, 64).to(dev), torch.ones(64, device=dev)
    q, s = ops.quant_fp8(x)
    wq, ws = ops.pack_fp8(torch.randn(32, 64, device=dev))
    w, st = torch.randn(64, 4, device=dev), torch.zeros(4, 3, 64, device=dev, dtype=dt)
    A, B, h = -torch.rand(64, 16, device=dev), low(4, 16).to(dev), torch.zeros(4, 64, 16, device=dev)
    bad = [
        lambda: ops.rmsnorm(x.float(), g), lambda: ops.rmsnorm(x, g.to(dt)), lambda: ops.rmsnorm(x, g[:32]),
        lambda: ops.rmsnorm(x.t(), None), lambda: ops.rmsnorm(x, g, residual=x[:2]), lambda: ops.rmsnorm(x, g, sum_out=x),
        lambda: ops.rmsnorm(x, g.clone().requires_grad_()), lambda: ops.rmsnorm(x, g, residual=x.double()),
        lambda: ops.rmsnorm(x, g, residual=x.clone(), sum_out=x[1:]), lambda: ops.rmsnorm(x.cpu(), g), lambda: ops.rmsnorm(x[0], g),
        lambda: ops.gemm_fp8(q, s, wq[:, :32], ws), lambda: ops.gemm_fp8(q, s[:2], wq, ws), lambda: ops.gemm_fp8(x, s, wq, ws),
        lambda: ops.gemm_fp8(q, s, wq, ws.to(dt)), lambda: ops.gemm_fp8(q, s, wq, ws, bias=g), lambda: ops.gemm_fp8(q, s, wq, ws, residual=x),
        lambda: ops.pack_fp8(g),
        lambda: ops.causal_conv(x, w[:, :1]), lambda: ops.causal_conv(x, w, nb=3), lambda: ops.causal_conv(x, w, out=x),
        lambda: ops.causal_conv(x, w, nb=4, state=st[:, :2]), lambda: ops.causal_conv(x, w, nb=4, state=st[:3]),
        lambda: ops.causal_conv(x, w, nb=4, slots=torch.zeros(4, dtype=torch.int32, device=dev)),
        lambda: ops.causal_conv(x, w, starts=torch.zeros(3, device=dev)), lambda: ops.causal_conv(x, w, nb=4, state=st, fresh=g[:4]),
        lambda: ops.causal_conv(x, w, nb=4, state=st, slots=torch.zeros(3, dtype=torch.int32, device=dev)),
        lambda: ops.ssm_scan(x, x, A[:, :7], B, B), lambda: ops.ssm_scan(x, x.double(), A, B, B), lambda: ops.ssm_scan(x, x, A, B, B.float()),
        lambda: ops.ssm_scan(x, x, torch.zeros(64, 65, device=dev), low(4, 65).to(dev), low(4, 65).to(dev)),
        lambda: ops.ssm_scan(x, x, A, B, B, out=x), lambda: ops.ssm_scan(x, x, A, B, B, z=x[:2]), lambda: ops.ssm_scan(x, x, A, B, B, state=h.to(dt)),
        lambda: ops.ssm_step(x, x, A, B, B, state=h[:2]), lambda: ops.ssm_step(x, x, A, B, B, state=h.transpose(1, 2)),
    ]
    for k, f in enumerate(bad):
        with pytest.raises(_lib.ActhError):
            f()
            pytest.fail(f"call {k} was not refused")
    for y in (x, g, st, h):
        assert torch.isfinite(y).all()


@pytest.mark.parametrize("M,N,K", [(3, 40, 50), (40, 200, 333), (70, 1500, 1001), (700, 1030, 517)])
@pytest.mark.parametrize("f32", [False, True])
def test_gemm_fp8_rows_at_any_address(dev, M, N, K, f32):
    """Operands inside wider rows, at odd offsets and pitches, with values beside them that must not enter."""
    big = torch.full((M, K + 11), 448.0).to(ops.FP8)
    wide = torch.full((N, K + 7), 448.0).to(ops.FP8)
    big[:, 5:5 + K] = torch.randn(M, K).to(ops.FP8)
    wide[:, 3:3 + K] = torch.randn(N, K).to(ops.FP8)
    s, ws = 0.5 + torch.rand(M, -(-K // 128)), 0.5 + torch.rand(-(-N // 128), -(-K // 128))
    a, w = big.to(dev)[:, 5:5 + K], wide.to(dev)[:, 3:3 + K]
    out = ops.gemm_fp8(a, s.to(dev), w, ws.to(dev), out_f32=f32)
    A, W = wide_of(big[:, 5:5 + K], s, 1), wide_of(wide[:, 3:3 + K], ws, 128)
    want = A @ W.t()
    tol = (A.abs() @ W.abs().t()) * (K + 8) * U
    near(out, want, tol if f32 else tol + want.abs() * half() + least_normal() + unit_loss(A, W, dev))


@pytest.mark.parametrize("N,G,z,last,L", [(16, 2, True, True, 75), (16, 1, False, True, 300), (8, 2, False, False, 33), (40, 1, True, True, 1)])
def test_selective_scan_fn_gate_and_last_state(dev, N, G, z, last, L):
    """The drop-in's gate, last state and other state counts: (batch, dim, L) operands, fp32 delta, B and C."""
    from actalker_amd.selective_scan_interface import selective_scan_fn
    b, dim = 3, 32
    s = scan_case([L] * b, dim, N, G, "float")
    y, tol, new, ntol = scan_ref(*(s[k] for k in IN[:6]), s["z"] if z else None, s["delta_bias"], True, cuts_of([L] * b),
                                 torch.zeros(b, dim, N), [False] * b)
    seq = lambda t: t.view(b, L, -1).transpose(1, 2).contiguous().to(dev)                            # noqa: E731
    grp = lambda t: t.reshape(b, L, G, N).permute(0, 2, 3, 1).contiguous().to(dev)                   # noqa: E731
    out = selective_scan_fn(seq(s["u"]), seq(s["delta"]), s["A"].to(dev), grp(s["B"]), grp(s["C"]), s["D"].to(dev),
                            z=seq(s["z"]) if z else None, delta_bias=s["delta_bias"].to(dev), delta_softplus=True,
                            return_last_state=last)
    if last:
        out, state = out
        near(state, new, ntol)
    assert out.shape == (b, dim, L) and out.dtype == ops.act_dtype()
    near(out.transpose(1, 2).reshape(b * L, dim), y, tol)
    with pytest.raises(NotImplementedError):
        selective_scan_fn(seq(s["u"]), seq(s["delta"]), torch.zeros(dim, 65, device=dev), grp(s["B"]), grp(s["C"]))


def test_gemm_fp8_more_row_blocks_than_a_group(dev):
    """Several rounds of large tiles, a last group of fewer row blocks, ragged in every size."""
    M, N, K = 256 * 33 + 17, 256 * 9 + 40, 144
    q, s = ops.quant_fp8(low(M, K).to(dev))
    wq, wsc = ops.pack_fp8(torch.randn(N, K).to(dev) / 12)
    out = ops.gemm_fp8(q, s, wq, wsc)
    big = lambda t, c, r: t.float() * c.repeat_interleave(r, 0)[:t.shape[0]].repeat_interleave(128, 1)[:, :K]     # noqa: E731
    A, W = big(q, s, 1), big(wq, wsc, 128)
    want, size = (A @ W.t()).cpu().double(), (A.abs() @ W.abs().t()).cpu().double()
    # 7 * 2^-13 of each group's largest product is at most 2^-10 of its sum of magnitudes
    near(out, want, want.abs() * half() + size * (2.0 ** -10 + 2 * (K + 8) * U) + least_normal())


def test_prompts_in_a_graph_with_changing_offsets(dev):
    """A captured prompt batch: rows, offsets, slots and states change between the replays; eager work runs between."""
    lay = Layer(dev)
    T, n = 400, 4
    x, r = low(T, 256).to(dev), low(T, 256).to(dev)
    st = torch.tensor([0, 50, 60, 300, 400], dtype=torch.int32, device=dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        lay(x, r, lay.states(n, dev), st)
    torch.cuda.current_stream().wait_stream(side)
    gs = lay.states(n, dev)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = lay(x, r, gs, st)
    es = lay.states(n, dev)
    for offs in ([0, 50, 60, 300, 400], [0, 0, 399, 400, 400], [0, 400, 400, 400, 400], [0, 100, 200, 300, 400]):
        x.copy_(low(T, 256))
        r.copy_(low(T, 256))
        st.copy_(torch.tensor(offs, dtype=torch.int32))
        want = [t.clone() for t in lay(x.clone(), r.clone(), es, st.clone())]
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
        assert torch.equal(gs[0], es[0]) and torch.equal(gs[1], es[1])


def test_calls_without_rows(dev):
    dt = ops.act_dtype()
    e, w, A = torch.empty(0, 64, device=dev, dtype=dt), torch.randn(64, 4, device=dev), -torch.rand(64, 16, device=dev)
    bc = torch.empty(0, 16, device=dev, dtype=dt)
    kept, h = low(2, 3, 64).to(dev), torch.randn(2, 64, 16, device=dev)
    c0, h0 = kept.clone(), h.clone()
    st = torch.zeros(3, dtype=torch.int32, device=dev)
    assert ops.causal_conv(e, w, starts=st, state=kept).shape == (0, 64)
    assert ops.ssm_scan(e, e, A, bc, bc, starts=st, state=h).shape == (0, 64)
    assert ops.causal_conv_step(e, w, state=kept).shape == (0, 64) and ops.ssm_step(e, e, A, bc, bc, state=h).shape == (0, 64)
    x, b = low(5, 64).to(dev), low(5, 16).to(dev)
    out = torch.full((5, 64), 3.0, device=dev, dtype=dt)                 # rows, but only empty sequences
    ops.causal_conv(x, w, starts=st, state=kept, out=out)
    ops.ssm_scan(x, x, A, b, b, starts=st, state=h, out=out)
    assert (out == 3.0).all() and torch.equal(kept, c0) and torch.equal(h, h0)


def test_output_beside_its_operand(dev):
    """An output in other columns of an operand's rows is taken, one that shares any is not."""
    rows = low(40, 192).to(dev)
    w, st = torch.randn(64, 3, device=dev), torch.tensor([0, 11, 40], dtype=torch.int32, device=dev)
    want = ops.causal_conv(rows[:, :64].contiguous(), w, starts=st)
    ops.causal_conv(rows[:, :64], w, starts=st, out=rows[:, 64:128])
    assert torch.equal(rows[:, 64:128], want)
    for cols in (slice(32, 96), slice(0, 64)):
        with pytest.raises(_lib.ActhError):
            ops.causal_conv(rows[:, :64], w, starts=st, out=rows[:, cols])


def test_many_sequences_of_one_row(dev):
    """More sequences than a launch's second dimension could hold."""
    n, dim = 70001, 8
    s = scan_case([1], dim, 16, 1, "low")
    u = low(n, dim).to(dev)
    args = dict(A=s["A"].to(dev), D=s["D"].to(dev), delta_bias=s["delta_bias"].to(dev))
    bc, delta = low(n, 32).to(dev), low(n, dim).to(dev)
    h = torch.randn(n, dim, 16, device=dev)
    kept = h.clone()
    y = ops.ssm_step(u, delta, B=bc[:, :16], C=bc[:, 16:], state=kept, **args)
    w, cst = torch.randn(dim, 4), low(n, 3, dim).to(dev)
    ckept = cst.clone()
    c = ops.causal_conv_step(u, w.to(dev), state=ckept)
    at = torch.tensor([0, 1, 65534, 65535, 65536, n - 1], device=dev)
    sub, csub = h[at].clone(), cst[at].clone()
    want = ops.ssm_step(u[at], delta[at], B=bc[at, :16], C=bc[at, 16:], state=sub, **args)
    # the two kernels add a row's 16 products and the skip in other orders, and each rounds its sum once
    size = (sub.abs() * bc[at, None, 16:].float().abs()).sum(2) + (args["D"] * u[at].float()).abs()
    near(y[at], want.double().cpu(), (2 * half() * want.float().abs() + 40 * U * size).double().cpu() + least_normal())
    near(kept[at], sub.double().cpu(), sub.double().cpu().abs() * 4 * U)
    assert torch.equal(c[at], ops.causal_conv_step(u[at], w.to(dev), state=csub)) and torch.equal(ckept[at], csub)


def test_offsets_past_32_bits(dev, act):
    """Rows, slots and tiles whose element offsets do not fit 32 bits (one build; the address code is the same)."""
    if act == "fp16":
        pytest.skip("the address code does not depend on the activation type")
    dt = ops.act_dtype()
    x = torch.zeros(140000, 16384, device=dev, dtype=dt)                  # 2.3e9 elements
    x[-1] = low(16384).to(dev)
    q, s = ops.rmsnorm_fp8(x, None)
    q1, s1 = ops.rmsnorm_fp8(x[-1:].clone(), None)
    assert torch.equal(q[-1].view(torch.uint8), q1[0].view(torch.uint8)) and torch.equal(s[-1], s1[0])
    wq, wsc = ops.pack_fp8(torch.randn(64, 16384, device=dev))
    far, by_itself = ops.gemm_fp8(q, s, wq, wsc)[-1000:].double(), ops.gemm_fp8(q[-1000:].clone(), s[-1000:].contiguous(), wq, wsc).double()
    assert (far[:-1] == 0).all() and far[-1].abs().max() > 0              # another kernel: other sums, each rounded once
    assert float((far - by_itself).norm() / by_itself.norm()) < 2 * half()
    del q, s
    w = torch.randn(16384, 4, device=dev)
    st = torch.tensor([0, 7, 139990, 140000], dtype=torch.int32, device=dev)
    y = ops.causal_conv(x, w, starts=st)
    assert torch.equal(y[-10:], ops.causal_conv(x[-10:].clone(), w))
    del x, y
    dim, N = 2048, 64                                                     # slots of 2^17 floats, 2.6e9 in all
    pool = torch.empty(20000, dim, N, device=dev)
    u, b = low(6, dim).to(dev), low(6, N).to(dev)
    A, start = -torch.rand(dim, N, device=dev), torch.randn(1, dim, N, device=dev)
    pool[19999] = start[0]
    one = start.clone()
    sl = torch.tensor([19999], dtype=torch.int32, device=dev)
    assert torch.equal(ops.ssm_scan(u, u, A, b, b, state=pool, slots=sl), ops.ssm_scan(u, u, A, b, b, state=one))
    assert torch.equal(ops.ssm_step(u[:1], u[:1], A, b[:1], b[:1], state=pool, slots=sl), ops.ssm_step(u[:1], u[:1], A, b[:1], b[:1], state=one))
    assert torch.equal(pool[19999], one[0])


def test_chunks_whose_decay_leaves_fp32(dev):
    """A long row of time steps over which exp(A sum dt) overflows or underflows while every state stays in range."""
    s = scan_case([400], 16, 16, 1, "float")
    s["delta"] = torch.zeros(400, 16)
    s["delta"][32:48] = 1.0
    s["delta"][300:] = 0.1
    s["A"][:] = -1.0
    s["A"][2], s["A"][3], s["A"][4], s["A"][5] = 6.0, 6.0, -6.0, 9.0
    s["u"][:, 2:6] = 0
    s["state"][0, 2], s["state"][0, 3], s["state"][0, 4], s["state"][0, 5] = 1e-30, 0.0, 1e30, 0.0
    s["delta"][300:, 2:4] = 0.0
    s["u"][395:, 5] = 1.0                                    # nothing, growth past every number, then something
    s["delta"][300:395, 5] = 2.0
    s["z"] = torch.ones_like(s["z"])
    s["C"] = s["C"] * 1e-20                                  # outputs inside 16 bits' range
    s["D"] = torch.zeros(16)
    for starts in (None, torch.tensor([0, 400], dtype=torch.int32, device=dev)):
        args = (s["u"], s["delta"], s["A"], s["B"], s["C"], s["D"], s["z"], None, False)
        y, tol, new, ntol = scan_ref(*args, [0, 400], s["state"], [False])
        kept = s["state"].to(dev)
        out = ops.ssm_scan(**to(dev, s, "u", "delta", "A", "B", "C", "D", "z"), softplus=False, starts=starts, state=kept)
        keep = [c for c in range(16) if c != 4] if ops.act_dtype() is torch.float16 else list(range(16))      # 1e30 * 1e-20
        near(out[:, keep], y[:, keep], tol[:, keep], "y")
        near(kept, new, ntol, "state")


def test_padded_batch_inside_a_tile(dev):
    """Many empty sequences in one place, in the middle of the rows, with sequences behind them."""
    lens = [5] + [0] * 700 + [9, 0, 0, 20] + [0] * 300
    n, D = len(lens), 64
    cuts = cuts_of(lens)
    x, w, bias, st = low(cuts[-1] + 3, D), torch.randn(D, 4), torch.randn(D), low(n, 3, D)
    y, tol, new = conv_ref(x, w, bias, cuts, st, [False] * n, True)
    kept, out = st.to(dev), torch.full(x.shape, 3.0, device=dev, dtype=ops.act_dtype())
    ops.causal_conv(x.to(dev), w.to(dev), bias.to(dev), starts=torch.tensor(cuts, dtype=torch.int32, device=dev), state=kept, out=out)
    near(out[:cuts[-1]], y[:cuts[-1]], tol[:cuts[-1]])
    assert (out[cuts[-1]:] == 3.0).all() and torch.equal(kept.cpu(), new.to(ops.act_dtype()))


def test_more_rows_than_a_launch(dev, act):
    """Norms and steps of so many rows that one launch could not hold a block each (the split does not depend on the type)."""
    if act == "fp16":
        pytest.skip("the launches do not depend on the activation type")
    n = (1 << 24) + 37
    dt = ops.act_dtype()
    at = torch.tensor([0, 1, (1 << 24) - 9, (1 << 24) - 8, (1 << 24) - 7, (1 << 24) - 1, 1 << 24, n - 1], device=dev)
    x, r = torch.randn(n, 3, device=dev).to(dt), torch.randn(n, 3, device=dev)
    (y, s), (y1, s1) = ops.rmsnorm(x, None, residual=r), ops.rmsnorm(x[at], None, residual=r[at])
    assert torch.equal(y[at], y1) and torch.equal(s, x.float() + r)
    q, sc = ops.quant_fp8(x)
    q1, sc1 = ops.quant_fp8(x[at])
    assert torch.equal(q[at].view(torch.uint8), q1.view(torch.uint8)) and torch.equal(sc[at], sc1)
    del y, s, q, sc, r
    u, w = x[:, :1].contiguous(), torch.tensor([[0.5, 2.0]], device=dev)
    st = torch.randn(n, 1, 1, device=dev).to(dt)
    kept = st.clone()
    y = ops.causal_conv_step(u, w, state=kept, silu=False)                # 16-bit sums of two exact products
    assert torch.equal(kept[:, 0], u) and torch.equal(y, (0.5 * st[:, 0].float() + 2.0 * u.float()).to(dt))
    perm = (n - 1 - torch.arange(n, device=dev)).int()
    fresh = torch.zeros(n, dtype=torch.bool, device=dev)
    fresh[-1] = True
    kept = st.clone()
    y = ops.causal_conv_step(u, w, state=kept, slots=perm, fresh=fresh, silu=False)
    old = st.flip(0)[:, 0].float()
    old[-1] = 0
    assert torch.equal(kept.flip(0)[:, 0], u) and torch.equal(y, (0.5 * old + 2.0 * u.float()).to(dt))
    A = torch.zeros(1, 1, device=dev)                                     # no decay: h + delta u B, powers of two apart
    b = torch.ones(n, 1, device=dev)
    delta = torch.full((n, 1), 0.5, device=dev)
    h = torch.randint(-8, 9, (n, 1, 1), device=dev).float()
    ui = torch.randint(-8, 9, (n, 1), device=dev).to(dt)
    for slots in (None, perm):
        kept = h.clone()
        y = ops.ssm_step(ui, delta, A, b, b, state=kept, slots=slots, softplus=False)
        want = (h if slots is None else h.flip(0))[:, 0] + 0.5 * ui.float()
        assert torch.equal(kept[:, 0] if slots is None else kept.flip(0)[:, 0], want) and torch.equal(y.float(), want)


@pytest.mark.parametrize("W", [2, 3, 4])
@pytest.mark.parametrize("T,D", [(600, 8192), (2300, 8195)])
def test_causal_conv_of_every_tile(dev, T, D, W):
    """Rows and channels enough for tiles of 8 and of 16 rows: each channel as in a call of a few channels, bit for bit."""
    cuts = [0, 1, 1, 3, 7, 100, 115, 116, 118, 333, 333, T - 5]
    n = len(cuts) - 1
    x, w, bias, st = low(T, D).to(dev), torch.randn(D, W).to(dev), torch.randn(D).to(dev), low(n, W - 1, D).to(dev)
    args = dict(starts=torch.tensor(cuts, dtype=torch.int32, device=dev), fresh=(torch.rand(n) < 0.3).to(dev))
    kept, out = st.clone(), torch.full_like(x, 3.0)
    ops.causal_conv(x, w, bias, state=kept, out=out, **args)
    for at in (slice(0, 40), slice(4000, 4040), slice(D - 40, D)):
        k, o = st[:, :, at].contiguous(), torch.full_like(x[:, at], 3.0)
        ops.causal_conv(x[:, at].contiguous(), w[at].contiguous(), bias[at].contiguous(), state=k, out=o, **args)
        assert torch.equal(out[:, at], o) and torch.equal(kept[:, :, at], k)
