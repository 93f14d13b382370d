"""GPU: the serving operators' kernels at the sizes where each of their forms is chosen, against 64 bits or exact values,
and what a call owes the framework around it. Tolerances as in test_serving_ops_gpu.py."""
import math

import pytest
import torch

from actalker_amd import _lib, ops
from tests.test_serving_ops_gpu import (IN, _seed, act, cuts_of, half, least_normal, low, near, scan_case, scan_ref,      # noqa: F401
                                        to)

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


# ------------------------------------------------------------------------------------------ product
@pytest.mark.parametrize("M,N,K", [(1, 8200, 528), (1, 16, 128), (16, 70, 640), (5, 8200, 517), (17, 300, 640), (32, 1030, 333),
                                   (300, 320, 272), (130, 1030, 144), (700, 640, 512), (700, 640, 509)])
def test_gemm_fp8_few_rows_keep_small_products(dev, M, N, K):
    """Large products that cancel beside one small one: every partial sum has at most 23 bits between its first and last
    (2^15 .. 2^-7), so fp32 sums are exact in any order, and what is left is a power of two times 1 or 1.5, exact in 16 bits."""
    a, w = torch.zeros(M, K), (2.0 ** (torch.arange(N) % 3))[:, None].repeat(1, K)
    n16 = K // 16
    a[:, 0:16 * n16:16], a[:, 8:16 * n16:16] = 256.0, -256.0
    m = torch.arange(M)
    a[m, 16 * (m % n16) + 1 + m % 7] = (1 + 0.5 * (m % 2)) * 2.0 ** -6
    want = ((1 + 0.5 * (m % 2)) * 2.0 ** -6)[:, None] * w[:, 0]
    s, ws = torch.ones(M, -(-K // 128)), torch.ones(-(-N // 128), -(-K // 128))
    for f32 in (False, True):
        out = ops.gemm_fp8(a.to(ops.FP8).to(dev), s.to(dev), w.to(ops.FP8).to(dev), ws.to(dev), out_f32=f32)
        assert torch.equal(out.float().cpu(), want)


def product_and_size(a, s, w, ws, bias=None, res=None):
    """The product in 64 bits on the device, and the sum of the magnitudes that enter it."""
    big = lambda t, c, r: t.double() * c.double().repeat_interleave(r, 0)[:t.shape[0]].repeat_interleave(128, 1)[:, :t.shape[1]]   # noqa: E731
    A, W = big(a.float(), s, 1), big(w.float(), ws, 128).t().contiguous()
    want, size = A @ W, A.abs() @ W.abs()
    for more in (bias, res):
        if more is not None:
            want, size = want + more.double(), size + more.double().abs()
    return want, size


# a product of K > 0 in one call of each form: (M, N, K, operands inside wider rows)
FORMS = [(1, 10250, 2560, False), (16, 8203, 517, True), (16, 8200, 520, False), (33, 640, 1306, False), (1000, 512, 517, True),
         (1000, 512, 512, False), (1100, 1030, 1306, True), (1100, 1030, 1296, False),
         (4096 - 13, 2560 - 24, 656, False),       # 160 large tiles, none of them halved
         (9216 - 37, 2560 - 21, 1296, False)]      # 360 large tiles, the last 104 in halves


@pytest.mark.parametrize("M,N,K,inside", FORMS)
@pytest.mark.parametrize("more", ["none", "bias_res", "f32"])
def test_gemm_fp8_forms(dev, M, N, K, inside, more):
    """Element by element: 7 * 2^-13 of each group's largest product, the most that the 8-bit unit may drop, is at most
    2^-10 of the sum of magnitudes. In the norm: what it drops of a product has the product's sign and is at most 2^-13 of
    its group's largest, uniformly spread, so over random signs at most sqrt(7 / 3) 2^-13 of the product's norm, which
    adds to the outputs' own rounding as squares do."""
    a, w = low(M, K).to(dev), (torch.randn(N, K) / math.sqrt(K)).to(dev)
    (q, s), (wq, wsc) = ops.quant_fp8(a), ops.pack_fp8(w)
    if inside:
        pad = lambda t, l, r: torch.nn.functional.pad(t.view(torch.uint8), (l, r), value=0x7e).view(ops.FP8)[:, l:l + K]   # noqa: E731
        q, wq = pad(q, 3, 8), pad(wq, 5, 2)
    bias = torch.randn(N, device=dev) if more == "bias_res" else None
    res = low(M, N).to(dev) if more == "bias_res" else None
    out = ops.gemm_fp8(q, s, wq, wsc, bias=bias, residual=res, out_f32=more == "f32")
    want, size = product_and_size(q, s, wq, wsc, bias, res)
    err = (out.double() - want).abs()
    if more == "f32":
        assert (err <= size * (K + 8) * U).all()
        return
    assert (err <= size * (2.0 ** -10 + (K + 8) * U) + want.abs() * half() + least_normal()).all()
    product = want if res is None else product_and_size(q, s, wq, wsc)[0]
    own = want.to(out.dtype).double() - want
    assert float(err.square().sum()) <= 1.002 * float(own.square().sum()) + 7 / 3 * 2.0 ** -26 * float(product.square().sum())


@pytest.mark.parametrize("M,N,K", [(2, 40, 256), (300, 640, 256), (1100, 1030, 256), (4096, 2560, 256)])
@pytest.mark.parametrize("f32", [False, True])
def test_gemm_fp8_a_code_that_is_no_number(dev, M, N, K, f32):
    """A NaN code reaches its row, or its column, and nothing else."""
    q, s = ops.quant_fp8(low(M, K).to(dev))
    w, ws = ops.pack_fp8(torch.randn(N, K, device=dev))
    good = ops.gemm_fp8(q, s, w, ws, out_f32=f32)
    q.view(torch.uint8)[M // 2, 200] = 0x7f
    w.view(torch.uint8)[N - 3, 5] = 0xff
    bad = ops.gemm_fp8(q, s, w, ws, out_f32=f32)
    hit = torch.zeros(M, N, dtype=torch.bool, device=dev)
    hit[M // 2], hit[:, N - 3] = True, True
    assert torch.equal(torch.isnan(bad), hit) and torch.equal(bad[~hit], good[~hit])


# ------------------------------------------------------------------------------------------ scan and steps
def channels(s, at, G):
    """The call's operands for the channels `at` of one group alone, on the CPU."""
    dim, N = s["A"].shape
    g = at.start // (dim // G)
    assert (at.stop - 1) // (dim // G) == g
    cut = {k: s[k][..., at].contiguous() for k in ("u", "delta", "z", "D", "delta_bias")}
    return dict(cut, A=s["A"][at], B=s["B"][:, g * N:(g + 1) * N], C=s["C"][:, g * N:(g + 1) * N], state=s["state"][:, at])


@pytest.mark.parametrize("dim,N,G,kind", [(2048, 16, 1, "low"), (2051, 16, 1, "float"), (2051, 12, 1, "low"), (4104, 16, 2, "float"),
                                          (2048, 12, 512, "low")])
@pytest.mark.parametrize("lens", [[2900, 0, 1, 1299], [4200], [1400] * 3], ids=str)
def test_ssm_scan_of_wide_layers(dev, dim, N, G, kind, lens):
    """Rows and channels enough for one lane a channel: chunks with and without a carry, a last piece of channels that is
    whole, cut or shorter than 8 (groups of 4), the first, middle and last channels of the first and last group."""
    s = scan_case(lens, dim, N, G, kind, extra=3 if len(set(lens)) > 1 else 0)
    T, cuts, n = s["u"].shape[0], cuts_of(lens), len(lens)
    assert T // 64 * (-(-dim // 64)) >= 2048
    fresh = torch.rand(n) < 0.3
    kept, out = s["state"].to(dev), torch.full((T, dim), 3.0, device=dev, dtype=ops.act_dtype())
    how = dict(nb=n) if T == cuts[-1] and len(set(lens)) == 1 else dict(starts=torch.tensor(cuts, dtype=torch.int32, device=dev))
    ops.ssm_scan(**to(dev, s, *IN), state=kept, fresh=fresh.to(dev), out=out, **how)
    dg = dim // G
    first = [slice(0, 4)] if dg < 12 else [slice(0, 9), slice(59, 70), slice(dg - 12, dg)]
    for at in first + [slice(dim - dg + a.start, dim - dg + a.stop) for a in first] * (G > 1):
        c = channels(s, at, G)
        y, tol, new, ntol = scan_ref(*(c[k] for k in IN), True, cuts, c["state"], fresh)
        near(out[:cuts[-1], at], y[:cuts[-1]], tol[:cuts[-1]], f"y {at}")
        near(kept[:, at], new, ntol, f"state {at}")
    assert (out[cuts[-1]:] == 3.0).all()


@pytest.mark.parametrize("n,dim,N,G", [(257, 2560, 16, 1), (257, 2560, 5, 1), (129, 1284, 24, 2), (131, 640, 64, 1), (257, 1024, 8, 1), (12001, 12, 16, 1)])
@pytest.mark.parametrize("beside", [False, True])
def test_ssm_step_of_many_sequences(dev, n, dim, N, G, beside):
    """Sequences enough that a lane takes two, an odd number of them, some without a place and some that start from zeros;
    B and C at whole or odd addresses."""
    s = scan_case([1] * n, dim, N, G, "low")
    slots, fresh = torch.randperm(n + 3)[:n].to(torch.int32), torch.rand(n) < 0.2
    slots[5], slots[n - 1] = -1, n + 3                 # the first and the second of a pair
    live = [i for i in range(n) if 0 <= slots[i] < n + 3]
    at = slots[live].long()
    pool = torch.randn(n + 3, dim, N)
    state = torch.zeros(n, dim, N)
    state[live] = pool[at]
    y, tol, new, ntol = scan_ref(*(s[k] for k in IN), True, list(range(n + 1)), state, fresh)
    kept, out = pool.to(dev), torch.full((n, dim), 3.0, device=dev, dtype=ops.act_dtype())
    args = to(dev, s, *IN)
    if beside:
        rows = torch.cat([s["B"][:, :1], s["B"], s["C"], s["C"][:, :1]], 1).to(dev)
        args["B"], args["C"] = rows[:, 1:1 + G * N], rows[:, 1 + G * N:1 + 2 * G * N]
    ops.ssm_step(**args, state=kept, slots=slots.to(dev), fresh=fresh.to(dev), out=out)
    near(out[live], y[live], tol[live], "y")
    near(kept[at], new[live], ntol[live], "state")
    dead = [i for i in range(n) if i not in live]
    rest = [i for i in range(n + 3) if i not in set(at.tolist())]
    assert (out[dead] == 3.0).all() and torch.equal(kept.cpu()[rest], pool[rest])


# ------------------------------------------------------------------------------------------ around a call
def calls(dev, n=4, d=64):
    """Every entry point as (name, operands by name, call of them); the states and outputs are among the operands."""
    dt = ops.act_dtype()
    q, s = ops.quant_fp8(low(n, d).to(dev))
    w, ws = ops.pack_fp8(torch.randn(48, d, device=dev))
    x = lambda: low(n, d).to(dev)                                                                     # noqa: E731
    scan = lambda **k: dict(u=x(), delta=x(), A=-torch.rand(d, 16, device=dev), B=low(n, 16).to(dev), C=low(n, 16).to(dev),   # noqa: E731
                            z=x(), state=torch.zeros(n, d, 16, device=dev), out=x(), **k)
    conv = lambda: dict(x=x(), w=torch.randn(d, 4, device=dev), bias=torch.randn(d, device=dev),      # noqa: E731
                        state=torch.zeros(n, 3, d, device=dev, dtype=dt), out=x())
    st = torch.tensor([0, 1, n], dtype=torch.int32, device=dev)
    return [
        ("rmsnorm", dict(x=x(), gamma=torch.ones(d, device=dev), residual=x(), sum_out=x(), out=x()), ops.rmsnorm),
        ("rmsnorm_fp8", dict(x=x(), gamma=torch.ones(d, device=dev), residual=torch.randn(n, d, device=dev),
                             sum_out=torch.zeros(n, d, device=dev)), ops.rmsnorm_fp8),
        ("quant_fp8", dict(x=x()), ops.quant_fp8),
        ("gemm_fp8", dict(a=q, a_scale=s, w=w, w_scale=ws, bias=torch.ones(48, device=dev), residual=low(n, 48).to(dev),
                          out=torch.empty(n, 48, device=dev, dtype=dt)), ops.gemm_fp8),
        ("causal_conv", dict(conv(), starts=st), ops.causal_conv), ("causal_conv_step", conv(), ops.causal_conv_step),
        ("ssm_scan", scan(starts=st), ops.ssm_scan), ("ssm_step", scan(), ops.ssm_step),
    ]


def test_operands_with_a_tangent_are_refused(dev):
    from torch.autograd import forward_ad
    for name, args, f in calls(dev):
        f(**args)
        with forward_ad.dual_level():
            f(**args)
            for k, t in args.items():
                if t.dtype in (torch.float32, ops.act_dtype()):
                    with torch.no_grad(), pytest.raises(_lib.ActhError, match="forward-mode"):
                        f(**dict(args, **{k: forward_ad.make_dual(t, torch.ones_like(t))}))


def test_written_tensors_count_up_their_version(dev):
    """States and given outputs, and nothing else; so a backward that needs a state's old values refuses to run."""
    for name, args, f in calls(dev):
        before = {k: t._version for k, t in args.items()}
        f(**args)
        for k, t in args.items():
            assert (t._version > before[k]) == (k in ("sum_out", "out", "state")), (name, k)
    _, args, f = calls(dev)[-1]
    scale = torch.ones(1, device=dev, requires_grad=True)
    y = (scale * args["state"]).sum()
    with torch.no_grad():
        f(**args)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with torch.inference_mode():
        f(**dict(args, state=torch.zeros_like(args["state"])))
    empty = dict(args, **{k: args[k][:0] for k in ("u", "delta", "B", "C", "z", "out")})
    version = args["state"]._version
    f(**empty)
    assert args["state"]._version == version


def test_steps_of_a_batch_that_has_run_empty(dev):
    for name, args, f in calls(dev):
        if name.endswith("_step"):
            kept = args["state"].fill_(2.0)
            rows = {k: t if k in ("w", "bias", "A", "state") else t[:0] for k, t in args.items()}
            none = torch.empty(0, dtype=torch.int32, device=dev)
            assert f(**rows, slots=none, fresh=none.bool()).shape == (0, 64)
            assert f(**dict(rows, state=kept[:0]), slots=none).shape == (0, 64)
            assert (kept == 2.0).all()
