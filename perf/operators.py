"""The operators of a gated state-space layer as it is served, timed at the sizes it is served at.

One layer is: root-mean-square norm of the residual stream (with the addition that updates it, and an output in 8
bits), the projections as 8-bit products with a scale for each block of 128, the short causal convolution and the
selective scan, for prompts and for single new tokens. Each case names one of these operators and its sizes;
``prepare`` makes what a program has in hand before the call, ``run`` makes the call: with ``own`` through
``actalker_amd.ops``, otherwise in elementary torch operations.
"""
import contextlib
import math
import random

import torch

own = False

EIGHT = torch.float8_e4m3fn
TOP = 448.0                 # the largest e4m3 value
LEAST = 2.0 ** -100         # least block maximum: a block of zeros keeps a scale that can be divided by
BLOCK = 128
EPS = 1e-5


# ------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # the norm in front of a layer, for one new token of one sequence: latency
        dict(name="norm, one token, 8 bits", op="norm", dtype="bf16", rows=1, width=2560, residual="same", eight=True),
        # the norm over one 96 x 96 latent frame's tokens with a float residual stream, 16-bit output
        dict(name="norm, one frame, float residual", op="norm", dtype="fp16", rows=9216, width=1280, residual="float",
             eight=False),
        # a long batch of prompts
        dict(name="norm, prompts, 8 bits", op="norm", dtype="bf16", rows=32768, width=5120, residual="same", eight=True),
        # a projection of one new token: the weights' bytes
        dict(name="product, one token", op="product", dtype="bf16", rows=1, width=2560, out=10240, bias=False,
             residual=False, wide=False),
        # a short ragged batch through a projection whose sizes fill no tile and no block
        dict(name="product, odd sizes", op="product", dtype="fp16", rows=77, width=1360, out=2090, bias=True,
             residual=False, wide=True),
        # a projection of a long batch of prompts, added to the residual stream: matrix rate
        dict(name="product, prompts", op="product", dtype="bf16", rows=16384, width=5120, out=2560, bias=False,
             residual=True, wide=False),
        # the convolution over a few short prompts, odd width
        dict(name="convolution, short prompts", op="conv", dtype="fp16", tokens=1000, width=1306, taps=3, seqs=7),
        # the convolution over a long batch of prompts
        dict(name="convolution, prompts", op="conv", dtype="bf16", tokens=32768, width=5120, taps=4, seqs=24),
        # the scan of one long prompt: few rows, a long axis
        dict(name="scan, one long prompt", op="scan", dtype="bf16", tokens=8192, width=2560, states=16, groups=1,
             seqs=1, gated=True, wide=False),
        # the scan of a ragged batch of prompts that go on from kept states
        dict(name="scan, ragged prompts", op="scan", dtype="fp16", tokens=16384, width=5120, states=16, groups=2,
             seqs=19, gated=True, wide=True),
        # one new token of one sequence through convolution and scan: latency
        dict(name="step, one sequence", op="step", dtype="bf16", width=2560, states=16, taps=4, seqs=1),
        # one new token of many sequences: the states' bytes
        dict(name="step, many sequences", op="step", dtype="bf16", width=5120, states=16, taps=4, seqs=512),
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["norm", "product", "conv", "scan", "step"])
    dtype = rng.choice(["bf16", "fp16"])
    if op == "norm":
        width = _log(rng, 64, 8192)
        if rng.random() < 0.6:
            width = max(64, width // 64 * 64)
        rows = _log(rng, 1, max(1, 100_000_000 // width))
        return dict(op=op, dtype=dtype, rows=rows, width=width, residual=rng.choice(["none", "same", "float"]),
                    eight=rng.random() < 0.6)
    if op == "product":
        width, out = _log(rng, 64, 10240), _log(rng, 8, 10240)
        if rng.random() < 0.8:
            width = max(64, width // 16 * 16)
        rows = _log(rng, 1, max(1, min(32768, 200_000_000_000 // (width * out))))
        return dict(op=op, dtype=dtype, rows=rows, width=width, out=out, bias=rng.random() < 0.5,
                    residual=rng.random() < 0.5, wide=rng.random() < 0.3)
    if op == "conv":
        width = _log(rng, 32, 8192)
        tokens = _log(rng, 1, max(1, 160_000_000 // width))
        return dict(op=op, dtype=dtype, tokens=tokens, width=width, taps=rng.choice([2, 3, 4]),
                    seqs=min(tokens, _log(rng, 1, 64)))
    if op == "scan":
        states = rng.choice([16, 16, 16, 8, 24, 32, 64])
        groups = rng.choice([1, 1, 2])
        width = _log(rng, 32, 8192) // groups * groups
        tokens = _log(rng, 1, max(1, min(16384, 1_200_000_000 // (width * states))))
        return dict(op=op, dtype=dtype, tokens=tokens, width=width, states=states, groups=groups,
                    seqs=min(tokens, _log(rng, 1, 64)), gated=rng.random() < 0.7, wide=rng.random() < 0.5)
    width = _log(rng, 32, 8192)
    return dict(op=op, dtype=dtype, width=width, states=rng.choice([16, 16, 8, 32]), taps=rng.choice([2, 3, 4]),
                seqs=_log(rng, 1, max(1, 2_400_000 // width)))


# ------------------------------------------------------------------------------------------ inputs
def _dtype(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float16


def _starts(tokens, seqs, seed):
    """Row offsets of ``seqs`` ragged sequences that fill ``tokens`` rows."""
    rng = random.Random(seed * 7919 + tokens * 31 + seqs)
    cuts = sorted(rng.randrange(0, tokens + 1) for _ in range(seqs - 1))
    return [0] + cuts + [tokens]


def _to_eight(x, rows_of_block):
    """e4m3 values and float scales of x (r, c) with a scale for each block of rows_of_block x 128."""
    r, c = x.shape
    kb, rb = -(-c // BLOCK), -(-r // rows_of_block)
    y = torch.nn.functional.pad(x, (0, kb * BLOCK - c, 0, rb * rows_of_block - r))
    y = y.view(rb, rows_of_block, kb, BLOCK)
    scale = y.abs().amax(dim=(1, 3)).clamp_min(LEAST) / TOP
    q = (y / scale[:, None, :, None]).clamp(-TOP, TOP).reshape(rb * rows_of_block, kb * BLOCK)[:r, :c]
    return q.to(EIGHT).contiguous(), scale


def _scan_inputs(case, tokens, g, dev, dt):
    w, n = case["width"], case["states"]
    gn = case.get("groups", 1) * n
    rnd = lambda *s: torch.randn(*s, generator=g, device=dev)                                     # noqa: E731
    uni = lambda *s: torch.rand(*s, generator=g, device=dev)                                      # noqa: E731
    kind = torch.float32 if case.get("wide") else dt
    proj = rnd(tokens, 2 * gn).to(kind)                                # one projection's rows: [B | C]
    s = dict(u=rnd(tokens, w).to(dt), delta=(0.5 * rnd(tokens, w)).to(kind), B=proj[:, :gn], C=proj[:, gn:],
             A=-torch.exp(torch.log(torch.arange(1, n + 1, device=dev).float()) + 0.2 * rnd(w, n)), D=1 + 0.1 * rnd(w))
    rate = torch.exp(uni(w) * math.log(100.0) + math.log(1e-3))        # time steps from 1e-3 to 1e-1 ...
    s["delta_bias"] = rate + torch.log(-torch.expm1(-rate))            # ... behind the softplus
    s["z"] = rnd(tokens, w).to(dt) if case.get("gated", True) else None
    return s


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(int(seed) * 1000003 + 17)
    dt = _dtype(case)
    rnd = lambda *s: torch.randn(*s, generator=g, device=dev)                                     # noqa: E731
    s = dict(case=dict(case), dt=dt)
    op = case["op"]
    if op == "norm":
        r, w = case["rows"], case["width"]
        s["x"] = rnd(r, w).to(dt)
        s["gamma"] = 1 + 0.1 * rnd(w)
        s["residual"] = None
        if case["residual"] != "none":       # a residual stream has a few channels far larger than the others
            s["residual"] = (2 * rnd(r, w) * torch.exp(rnd(w))).to(dt if case["residual"] == "same" else torch.float32)
    elif op == "product":
        r, k, n = case["rows"], case["width"], case["out"]
        s["a"], a_scale = _to_eight(rnd(r, k) * torch.exp(0.5 * rnd(k)), 1)
        s["a_scale"] = a_scale.t().contiguous().t()      # as the norm gives it: a block's scales next to each other
        s["w"], s["w_scale"] = _to_eight(rnd(n, k) / math.sqrt(k), BLOCK)
        s["bias"] = rnd(n) if case["bias"] else None
        s["residual"] = rnd(r, n).to(dt) if case["residual"] else None
    elif op == "conv":
        t, w, taps, n = case["tokens"], case["width"], case["taps"], case["seqs"]
        s["x"] = rnd(t, w).to(dt)
        s["w"], s["bias"] = rnd(w, taps) / math.sqrt(taps), 0.1 * rnd(w)
        s["cuts"] = _starts(t, n, int(seed))
        s["starts"] = torch.tensor(s["cuts"], dtype=torch.int32, device=dev)
        s["state"] = rnd(n, taps - 1, w).to(dt)
    elif op == "scan":
        n = case["seqs"]
        s.update(_scan_inputs(case, case["tokens"], g, dev, dt))
        s["cuts"] = _starts(case["tokens"], n, int(seed))
        s["starts"] = torch.tensor(s["cuts"], dtype=torch.int32, device=dev)
        s["state"] = rnd(n, case["width"], case["states"])
    else:
        n, w, taps = case["seqs"], case["width"], case["taps"]
        s.update(_scan_inputs(case, n, g, dev, dt))
        s["x"] = s.pop("u")                                            # the scan's input is the convolution's output
        s["w"], s["bias"] = rnd(w, taps) / math.sqrt(taps), 0.1 * rnd(w)
        s["conv_state"] = rnd(n, taps - 1, w).to(dt)
        s["state"] = rnd(n, w, case["states"])
    if op in ("conv", "scan"):
        lens = torch.tensor([b - a for a, b in zip(s["cuts"], s["cuts"][1:])], device=dev)
        s["full"] = lens.nonzero()[:, 0]                               # the sequences that have tokens, and ...
        s["first"] = s["starts"][:-1][s["full"]].long()                # ... their first and ...
        s["last"] = s["starts"][1:][s["full"]].long() - 1              # ... last rows
        s["longest"] = int(lens.max())
        s["of_row"] = torch.repeat_interleave(torch.arange(n, device=dev), lens)
    return s


# ------------------------------------------------------------------------------------------ one pass
def run(s):
    if own:
        return _run_own(s)
    return _PLAIN[s["case"]["op"]](s)


def _run_own(s):
    from actalker_amd import ops
    op = s["case"]["op"]
    with ops.compute_dtype(s["dt"]) if s["dt"] == torch.float16 else contextlib.nullcontext():
        if op == "norm":
            if s["case"]["eight"]:
                return ops.rmsnorm_fp8(s["x"], s["gamma"], EPS, residual=s["residual"])
            return ops.rmsnorm(s["x"], s["gamma"], EPS, residual=s["residual"])
        if op == "product":
            return ops.gemm_fp8(s["a"], s["a_scale"], s["w"], s["w_scale"], bias=s["bias"], residual=s["residual"],
                                out_f32=s["case"]["wide"])
        if op == "conv":
            y = ops.causal_conv(s["x"], s["w"], s["bias"], starts=s["starts"], state=s["state"])
            return y, s["state"]
        if op == "scan":
            y = ops.ssm_scan(s["u"], s["delta"], s["A"], s["B"], s["C"], D=s["D"], z=s["z"],
                             delta_bias=s["delta_bias"], starts=s["starts"], state=s["state"])
            return y, s["state"]
        u = ops.causal_conv_step(s["x"], s["w"], s["bias"], state=s["conv_state"])
        y = ops.ssm_step(u, s["delta"], s["A"], s["B"], s["C"], D=s["D"], z=s["z"], delta_bias=s["delta_bias"],
                         state=s["state"])
        return y, s["conv_state"], s["state"]


def _plain_norm(s):
    x = s["x"].float()
    if s["residual"] is not None:
        x = x + s["residual"].float()
    y = x * torch.rsqrt(x.square().mean(dim=1, keepdim=True) + EPS) * s["gamma"]
    out = _to_eight(y, 1) if s["case"]["eight"] else (y.to(s["dt"]),)
    return out + (x.to(s["residual"].dtype),) if s["residual"] is not None else out


def _from_eight(q, scale, rows_of_block):
    r, c = q.shape
    big = scale.repeat_interleave(rows_of_block, dim=0)[:r].repeat_interleave(BLOCK, dim=1)[:, :c]
    return q.float() * big


def _plain_product(s):
    y = _from_eight(s["a"], s["a_scale"], 1) @ _from_eight(s["w"], s["w_scale"], BLOCK).t()
    if s["bias"] is not None:
        y = y + s["bias"]
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y if s["case"]["wide"] else y.to(s["dt"])


def _silu(x):
    return x / (1 + torch.exp(-x))


def _plain_conv(s):
    """Every row's inputs are taken tap by tap, from the rows before it or from its sequence's kept inputs."""
    x, state, taps = s["x"].float(), s["state"].float(), s["case"]["taps"]
    row = torch.arange(x.shape[0], device=x.device)
    place = row - s["starts"].long()[s["of_row"]]                      # the row's place in its sequence
    back = torch.arange(taps - 1, -1, -1, device=x.device)             # how far back each tap looks
    from_row = (row[:, None] - back).clamp_min(0)
    from_kept = (place[:, None] - back + taps - 1).clamp(0, taps - 2)
    seen = [torch.where((place >= taps - 1 - j)[:, None], x[from_row[:, j]], state[s["of_row"], from_kept[:, j]])
            for j in range(taps)]
    y = _silu(sum(v * s["w"][:, j] for j, v in enumerate(seen)) + s["bias"])
    for j in range(1, taps):                                           # the last taps - 1 inputs are kept
        s["state"][s["full"], j - 1] = seen[j][s["last"]].to(s["dt"])
    return y.to(s["dt"]), s["state"]


def _softplus(x):
    return torch.where(x > 20, x, torch.log1p(torch.exp(x.clamp_max(20))))


def _steps(s, u):
    """Decay and input of every step and state: (rows, width, states)."""
    w, n = s["A"].shape
    dt = _softplus(s["delta"].float() + s["delta_bias"])
    groups = s["B"].shape[1] // n
    B = s["B"].float().view(-1, groups, n).repeat_interleave(w // groups, dim=1)
    return torch.exp(dt[:, :, None] * s["A"]), (dt * u)[:, :, None] * B


def _read(s, h, u):
    """y from the states h (rows, width, states)."""
    w, n = s["A"].shape
    groups = s["C"].shape[1] // n
    y = (h.view(-1, groups, w // groups, n) * s["C"].float().view(-1, groups, 1, n)).sum(dim=3).view(-1, w)
    y = y + s["D"] * u
    if s["z"] is not None:
        y = y * _silu(s["z"].float())
    return y.to(s["dt"])


def _plain_scan(s):
    """h_t = a_t h_(t-1) + b_t by doubling: after k rounds each row holds the sum over its last 2^k rows."""
    u = s["u"].float()
    a, h = _steps(s, u)
    h[s["first"]] += a[s["first"]] * s["state"][s["full"]]
    a[s["first"]] = 0
    step = 1
    while step < s["longest"]:
        more = a[step:] * h[:-step]
        a = torch.cat([a[:step], a[step:] * a[:-step]])
        h[step:] += more
        step *= 2
    s["state"][s["full"]] = h[s["last"]]
    return _read(s, h, u), s["state"]


def _plain_step(s):
    x = torch.cat([s["conv_state"].float(), s["x"].float()[:, None]], dim=1)
    u = _silu((x * s["w"].t()).sum(dim=1) + s["bias"]).to(s["dt"]).float()
    s["conv_state"].copy_(x[:, 1:])
    a, b = _steps(s, u)
    s["state"].copy_(a * s["state"] + b)
    return _read(s, s["state"], u), s["conv_state"], s["state"]


_PLAIN = dict(norm=_plain_norm, product=_plain_product, conv=_plain_conv, scan=_plain_scan, step=_plain_step)


# ------------------------------------------------------------------------------------------ bytes and operations
def work(case):
    op = case["op"]
    if op == "norm":
        n = case["rows"] * case["width"]
        stream = {"none": 0, "same": 4, "float": 8}[case["residual"]]
        return dict(bytes=n * (2 + stream + (1 + 4 / BLOCK if case["eight"] else 2)) + 4 * case["width"], flops=6 * n)
    if op == "product":
        r, k, n = case["rows"], case["width"], case["out"]
        kb = -(-k // BLOCK)
        out = r * n * ((4 if case["wide"] else 2) + (2 if case["residual"] else 0)) + (4 * n if case["bias"] else 0)
        return dict(bytes=r * k + 4 * r * kb + n * k + 4 * kb * -(-n // BLOCK) + out, flops=2 * r * k * n)
    if op == "conv":
        n, taps = case["tokens"] * case["width"], case["taps"]
        return dict(bytes=4 * n + case["width"] * (4 * taps + 4 + 4 * (taps - 1) * case["seqs"]),
                    flops=n * (2 * taps + 5))
    w, n, q = case["width"], case["states"], case["seqs"]
    rows = case.get("tokens", q)
    kind = 4 if case.get("wide") else 2
    each = rows * (w * (4 + kind + (2 if case.get("gated", True) else 0)) + 2 * case.get("groups", 1) * n * kind)
    total = each + 8 * q * w * n + 4 * w * (n + 2)
    flops = rows * w * (7 * n + 10)
    if op == "step":
        total += 4 * q * w * (case["taps"] - 1) + w * (4 * case["taps"] + 4)
        flops += q * w * (2 * case["taps"] + 5)
    return dict(bytes=total, flops=flops)


# ------------------------------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    s = {k: v.double() if torch.is_tensor(v) and v.is_floating_point() and v.dtype != EIGHT else v for k, v in s.items()}
    return _EXACT[case["op"]](case, s)


def _exact_norm(case, s):
    x = s["x"] if s["residual"] is None else s["x"] + s["residual"]
    y = x / (x.pow(2).sum(1, keepdim=True) / x.shape[1] + EPS).sqrt() * s["gamma"]
    kept = [] if s["residual"] is None else [x]
    if not case["eight"]:
        return [y] + kept
    scale = torch.stack([part.abs().max(dim=1).values for part in y.split(BLOCK, dim=1)], dim=1).clamp(min=LEAST) / TOP
    column = torch.arange(x.shape[1], device=x.device) // BLOCK
    return [y / scale[:, column]] + [scale] + kept


def _exact_product(case, s):
    y = torch.zeros(case["rows"], case["out"], dtype=torch.float64, device=s["a"].device)
    row = torch.arange(case["out"], device=y.device) // BLOCK
    for b, (a, w) in enumerate(zip(s["a"].split(BLOCK, dim=1), s["w"].split(BLOCK, dim=1))):
        y += (a.double() @ w.double().t()) * s["a_scale"][:, b, None] * s["w_scale"][row, b]
    for more in ("bias", "residual"):
        if s[more] is not None:
            y = y + s[more]
    return y


def _exact_conv_rows(x, w, bias, taps):
    """x holds taps - 1 kept inputs and then the rows."""
    y = bias + torch.zeros_like(x[taps - 1:])
    for j in range(taps):
        y = y + x[j:x.shape[0] - (taps - 1 - j)] * w[:, j]
    return y * torch.sigmoid(y)


def _exact_conv(case, s):
    taps, y, state = case["taps"], [], []
    for i, (a, b) in enumerate(zip(s["cuts"], s["cuts"][1:])):
        x = torch.cat([s["state"][i], s["x"][a:b]])
        y.append(_exact_conv_rows(x, s["w"], s["bias"], taps))
        state.append(x[x.shape[0] - (taps - 1):])
    return [torch.cat(y), torch.stack(state)]


def _exact_recur(s, u, rows, h):
    """One token of several sequences: rows are their rows, h their states (sequences, width, states)."""
    w, n = s["A"].shape
    group = torch.arange(w, device=u.device) // (w // (s["B"].shape[1] // n))
    dt = torch.logaddexp(s["delta"][rows] + s["delta_bias"], torch.zeros((), dtype=torch.float64, device=u.device))
    B, C = (s[k][rows].view(rows.numel(), -1, n)[:, group] for k in ("B", "C"))
    h = torch.exp(dt.unsqueeze(-1) * s["A"]) * h + (dt * u).unsqueeze(-1) * B
    y = torch.einsum("bwn,bwn->bw", h, C) + s["D"] * u
    if s["z"] is not None:
        y = y * s["z"][rows] * torch.sigmoid(s["z"][rows])
    return y, h


def _exact_scan(case, s):
    lens = [b - a for a, b in zip(s["cuts"], s["cuts"][1:])]
    order = sorted(range(len(lens)), key=lambda i: -lens[i])           # so that the first ones are those still going
    h = s["state"][order]
    first = torch.tensor([s["cuts"][i] for i in order], device=h.device)
    y = torch.empty_like(s["u"])
    going = len(order)
    for t in range(max(lens)):
        while lens[order[going - 1]] <= t:
            going -= 1
        rows = first[:going] + t
        y[rows], h[:going] = _exact_recur(s, s["u"][rows], rows, h[:going])
    state = torch.empty_like(h)
    state[order] = h
    return [y, state]


def _exact_step(case, s):
    taps, n = case["taps"], case["seqs"]
    x = torch.cat([s["conv_state"], s["x"][:, None]], dim=1)
    u = _exact_conv_rows(x.transpose(0, 1).reshape(taps, -1), s["w"].repeat(n, 1), s["bias"].repeat(n), taps).view(n, -1)
    u = u.to(_dtype(case)).double()                                    # the convolution's output is held in 16 bits
    y, h = _exact_recur(s, u, torch.arange(n, device=u.device), s["state"])
    return [y, x[:, 1:], h]


_EXACT = dict(norm=_exact_norm, product=_exact_product, conv=_exact_conv, scan=_exact_scan, step=_exact_step)
