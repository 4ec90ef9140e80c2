"""Workloads of the expert-product and block-norm operators.

Four operators stand around the MoE block's router: matrix products grouped by
expert (forward and both gradients), MXFP4 quantisation (blocks of 32 values
in 4-bit E2M1 sharing one power-of-two E8M0 scale), the grouped product of
MXFP4 operands, and the norms before and after a block fused with its gate
and residual scale (forward and backward).

With `own` false `run` computes them in elementary torch operations, with it
true through this repository's `MoeLayerEngine`.
"""
import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "f32": torch.float32}


# --------------------------------------------------------------------------
# cases
# --------------------------------------------------------------------------
def listed():
    return [
        # One decoded token of the Qwen3-shaped layer: gate and up rows of its eight experts.
        {"name": "mm_token", "op": "mm", "tokens": 1, "top_k": 8, "experts": 128, "zipf": 0.0,
         "n": 1536, "k": 2048, "dtype": "bf16", "out": "bf16"},
        # A serving batch of the OLMoE-shaped layer: down rows, fp32 sums for the combine.
        {"name": "mm_batch", "op": "mm", "tokens": 64, "top_k": 8, "experts": 64, "zipf": 1.1,
         "n": 2048, "k": 1024, "dtype": "fp16", "out": "f32"},
        # Prefill of 4096 tokens with skewed expert popularity: gate and up rows.
        {"name": "mm_prefill", "op": "mm", "tokens": 4096, "top_k": 8, "experts": 128,
         "zipf": 1.1, "n": 1536, "k": 2048, "dtype": "bf16", "out": "bf16"},
        # Fine-tuning step on a small ragged batch of a many-expert layer, odd widths in padded rows.
        {"name": "mm_grad_odd", "op": "mm_grad", "tokens": 333, "top_k": 4, "experts": 72,
         "zipf": 0.6, "n": 517, "k": 1001, "dtype": "fp16", "out": "f32"},
        # Training step over 4096 tokens: both gradients of the down product.
        {"name": "mm_grad_train", "op": "mm_grad", "tokens": 4096, "top_k": 8, "experts": 128,
         "zipf": 1.1, "n": 2048, "k": 768, "dtype": "bf16", "out": "bf16"},
        # Activations of a decode batch gathered to their routes and quantised.
        {"name": "mx_rows", "op": "mx", "tokens": 32, "top_k": 8, "experts": 64, "zipf": 0.0,
         "k": 2048, "dtype": "bf16", "gather": True},
        # All gate and up rows of a layer quantised when a checkpoint is loaded.
        {"name": "mx_weights", "op": "mx", "tokens": 196608, "top_k": 1, "experts": 1,
         "zipf": 0.0, "k": 2048, "dtype": "bf16", "gather": False},
        # A small decode batch through the 4-bit experts.
        {"name": "mxmm_decode", "op": "mxmm", "tokens": 8, "top_k": 8, "experts": 128,
         "zipf": 0.0, "n": 1536, "k": 2048, "dtype": "bf16", "out": "bf16"},
        # Prefill of 4096 tokens through the 4-bit experts.
        {"name": "mxmm_prefill", "op": "mxmm", "tokens": 4096, "top_k": 8, "experts": 128,
         "zipf": 1.1, "n": 1536, "k": 2048, "dtype": "bf16", "out": "bf16"},
        # The residual stream of one decoded token.
        {"name": "norm_token", "op": "norm", "tokens": 1, "hidden": 2048, "res": "f32",
         "dtype": "f32", "post": True, "gate": False},
        # The residual stream of a prefill: fp32 residual, bf16 branch, a gate for each token.
        {"name": "norm_prefill", "op": "norm", "tokens": 4096, "hidden": 2048, "res": "f32",
         "dtype": "bf16", "post": True, "gate": True},
        # Its backward pass in a training step.
        {"name": "norm_grad", "op": "norm_grad", "tokens": 8192, "hidden": 2048, "res": "bf16",
         "dtype": "bf16", "post": True, "gate": True},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi):
    """A width: half of the draws any number, half a multiple of 64."""
    w = _log_int(rng, lo, hi)
    return w if rng.random() < 0.5 else max(64, w // 64 * 64)


def draw(rng):
    op = rng.choice(["mm", "mm", "mm_grad", "mm_grad", "mx", "mxmm", "mxmm", "norm", "norm_grad"])
    if op in ("norm", "norm_grad"):
        res, dtype = rng.choice([("f32", "f32"), ("bf16", "bf16"), ("fp16", "fp16"),
                                 ("f32", "bf16"), ("f32", "fp16")])
        return {"op": op, "tokens": _log_int(rng, 1, 8192), "hidden": _width(rng, 64, 2048),
                "res": res, "dtype": dtype, "post": rng.random() < 0.7,
                "gate": rng.random() < 0.5}
    c = {"op": op, "tokens": _log_int(rng, 1, 4096), "experts": rng.choice([8, 16, 64, 72, 128]),
         "zipf": rng.choice([0.0, 0.6, 1.1]), "dtype": rng.choice(["bf16", "fp16"])}
    c["top_k"] = rng.choice([1, 2, 4, 8])
    c["k"] = _width(rng, 64, 2048)
    if op == "mx":
        c["gather"] = rng.random() < 0.5
        c["dtype"] = rng.choice(["bf16", "fp16", "f32"])
        return c
    c["n"] = _width(rng, 64, 1536)
    c["out"] = rng.choice([c["dtype"], "f32"])
    return c


def counts(case):
    """Rows of each popularity rank: tokens * top_k routes over the experts by
    a Zipf law, at most `tokens` to one expert."""
    T, E = case["tokens"], case["experts"]
    R = T * case["top_k"]
    w = [(r + 1.0) ** -case["zipf"] for r in range(E)]
    c, left, free = [0.0] * E, float(R), set(range(E))
    while left > 1e-6 and free:
        s = sum(w[e] for e in free)
        for e in sorted(free):
            c[e] += left * w[e] / s
        left = sum(max(0.0, x - T) for x in c)
        c = [min(x, float(T)) for x in c]
        free = {e for e in free if c[e] < T}
    n = [int(x) for x in c]
    rest, e = R - sum(n), 0
    while rest > 0:
        if n[e % E] < T:
            n[e % E] += 1
            rest -= 1
        e += 1
    return n


# --------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------
def _rows(shape, std, dtype, g):
    """Normal values in rows whose stride is padded to 16 bytes, as a program
    with odd widths keeps them."""
    ld = -(-shape[-1] // 8) * 8
    full = torch.empty(*shape[:-1], ld, device="cuda", dtype=dtype)
    for part in (full if full.dim() == 3 else [full]):  # by expert, so that no fp32 copy of all is held
        part.copy_(torch.randn(part.shape, device="cuda", generator=g) * std)
    return full[..., :shape[-1]]


def _engine():
    import doantotnghiepmoe_b200 as M
    if not hasattr(_engine, "e"):
        _engine.e = M.MoeLayerEngine(M.MoeConfig(2048, 1024, 64, 8, True, 1, 1))
    return _engine.e


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = {"case": case}
    dt = _DT[case["dtype"]]
    if case["op"] in ("norm", "norm_grad"):
        T, H, rd = case["tokens"], case["hidden"], _DT[case["res"]]
        norm = lambda *sh: torch.randn(*sh, device="cuda", generator=g)
        s["x"] = (2.0 * norm(T, H)).to(rd)
        s["y"] = norm(T, H).to(dt)
        s["w_pre"] = 1.0 + 0.2 * norm(H)
        s["w_post"] = 1.0 + 0.2 * norm(H) if case["post"] else None
        s["gate"] = torch.sigmoid(norm(T)) if case["gate"] else None
        s["scale"], s["eps"] = 0.875, 1e-5
        if case["op"] == "norm_grad":
            s["dx_out"] = (0.01 * norm(T, H)).to(rd)
            s["dh"] = (0.01 * norm(T, H)).to(dt)
    else:
        E, T, k = case["experts"], case["tokens"], case["k"]
        c = counts(case)
        perm = torch.randperm(E, device="cuda", generator=g).tolist()
        sizes = [0] * E
        for r, e in enumerate(perm):
            sizes[e] = c[r]
        R = sum(sizes)
        off = [0]
        for x in sizes:
            off.append(off[-1] + x)
        s["off"] = off
        s["seg_off"] = torch.tensor(off, dtype=torch.int32, device="cuda")
        # tokens of each expert's rows, ascending: a run of a shuffled cycle
        order = torch.randperm(T, device="cuda", generator=g)
        tok = order[torch.arange(R, device="cuda") % T]
        key = torch.repeat_interleave(torch.arange(E, device="cuda"),
                                      torch.tensor(sizes, device="cuda")) * T + tok
        s["token"] = (torch.sort(key).values % T).to(torch.int32)
        if case["op"] in ("mm", "mm_grad"):
            s["x"] = _rows((R, k), 1.0, dt, g)
            s["w"] = _rows((E, case["n"], k), 0.02, dt, g)
            if case["op"] == "mm_grad":
                s["dout"] = _rows((R, case["n"]), 0.01, dt, g)
        else:
            # a few channels with large values, as hidden states have them
            x = torch.randn(T, k, device="cuda", generator=g)
            x[:, :: max(1, k // 5)] *= 20.0
            s["x"] = x.to(dt)
            if case["op"] == "mxmm":
                n = case["n"]
                wc = torch.empty(E * n, -(-k // 32) * 16, dtype=torch.uint8, device="cuda")
                ws = torch.zeros(E * n, -(-k // 128) * 4, dtype=torch.uint8, device="cuda")
                for e in range(E):
                    q, sc = _mx_encode(0.02 * torch.randn(n, k, device="cuda", generator=g))
                    wc[e * n:(e + 1) * n] = q
                    ws[e * n:(e + 1) * n, :sc.shape[1]] = sc
                s["wc"], s["ws"] = wc, ws
    if own:
        s["engine"] = _engine()
    return s


# --------------------------------------------------------------------------
# plain forms
# --------------------------------------------------------------------------
_LEVELS = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _pow2(e):
    """2^e in fp32 from its bits, for whole numbers -127 <= e <= 127."""
    e = e.to(torch.int32)
    return torch.where(e > -127, (e + 127) << 23, torch.full_like(e, 1 << 22)).view(torch.float32)


def _mx_split(x):
    """fp32 [rows, k] -> (magnitude codes, sign bits, scale bytes) by blocks
    of 32: scale 2^(floor(log2 max|x|) - 2), elements rounded to the nearest
    E2M1 value (ties to the even code), values past 6 held at 6; a block with
    an infinity or a NaN has the scale byte 255, which stands for NaN."""
    rows, k = x.shape
    nb = -(-k // 32)
    x = torch.nn.functional.pad(x, (0, nb * 32 - k)).view(rows, nb, 32)
    amax = x.abs().amax(-1)
    e = torch.frexp(amax)[1] - 3  # amax = m * 2^(e + 3), m in [0.5, 1)
    e = torch.where(amax > 0, e, torch.full_like(e, -127)).clamp(-127, 127)
    v = (x * _pow2(-e)[..., None]).abs()
    mids = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0]
    code = torch.zeros_like(v, dtype=torch.uint8)
    for i, m in enumerate(mids):  # a tie goes up where that code is even
        code += ((v >= m) if i % 2 else (v > m)).to(torch.uint8)
    bad = ~torch.isfinite(x).all(-1)
    sb = torch.where(bad, torch.full_like(e, 255), e + 127).to(torch.uint8)
    return torch.where(bad[..., None], torch.zeros_like(code), code), torch.signbit(x), sb


def _mx_encode(x):
    code, sign, sb = _mx_split(x)
    nib = (code | (sign.to(torch.uint8) << 3)).flatten(1)
    return nib[:, 0::2] | (nib[:, 1::2] << 4), sb


def _mx_decode(codes, scales, k):
    nb = -(-k // 32)
    lut = torch.tensor(_LEVELS + [-v for v in _LEVELS], device=codes.device)
    nib = torch.stack((codes & 15, codes >> 4), -1).flatten(1)
    sb = scales[:, :nb].to(torch.int32)
    sc = _pow2((sb - 127).clamp(max=127))
    sc = torch.where(sb == 255, torch.full_like(sc, math.nan), sc)
    v = lut[nib.long()].view(codes.shape[0], nb, 32) * sc[..., None]
    return v.flatten(1)[:, :k]


def _mx_values(x):
    """The values that the codes of fp32 x stand for."""
    code, sign, sb = _mx_split(x)
    lut = torch.tensor(_LEVELS, device=x.device)
    v = lut[code.long()]
    v = torch.where(sign, -v, v)
    e = sb.to(torch.int32) - 127
    v = v * _pow2(e.clamp(max=127))[..., None]
    v = torch.where((sb == 255)[..., None], torch.full_like(v, math.nan), v)
    return v.flatten(1)[:, :x.shape[1]]


def _segments(s):
    off = s["off"]
    return [(e, off[e], off[e + 1]) for e in range(len(off) - 1) if off[e + 1] > off[e]]


def _plain_norm(s):
    x, y = s["x"].float(), s["y"].float()
    if s["w_post"] is not None:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + s["eps"]) * s["w_post"]
    if s["gate"] is not None:
        y = y * s["gate"][:, None]
    xo = x * s["scale"] + y
    h = xo * torch.rsqrt((xo * xo).mean(-1, keepdim=True) + s["eps"]) * s["w_pre"]
    return xo.to(s["x"].dtype), h.to(s["y"].dtype)


def _plain_norm_grad(s):
    x, y, dh = s["x"].float(), s["y"].float(), s["dh"].float()
    rq = torch.rsqrt((x * x).mean(-1, keepdim=True) + s["eps"])
    t = dh * s["w_pre"]
    dx_out = s["dx_out"].float() + rq * t - x * rq ** 3 * (t * x).mean(-1, keepdim=True)
    dw_pre = (dh * x * rq).sum(0)
    gate = s["gate"][:, None] if s["gate"] is not None else 1.0
    if s["w_post"] is not None:
        rp = torch.rsqrt((y * y).mean(-1, keepdim=True) + s["eps"])
        z = y * rp * s["w_post"]
        t = dx_out * gate * s["w_post"]
        dy = rp * t - y * rp ** 3 * (t * y).mean(-1, keepdim=True)
        dw_post = (dx_out * gate * y * rp).sum(0)
    else:
        z, dy, dw_post = y, dx_out * gate, None
    dgate = (dx_out * z).sum(-1) if s["gate"] is not None else None
    return ((dx_out * s["scale"]).to(s["x"].dtype), dy.to(s["y"].dtype), dgate, dw_post, dw_pre)


def _plain(s):
    case, op = s["case"], s["case"]["op"]
    if op == "norm":
        return _plain_norm(s)
    if op == "norm_grad":
        return _plain_norm_grad(s)
    if op == "mx":
        x = s["x"].float()
        if case["gather"]:
            x = x[s["token"].long()]
        return _mx_values(x).to(s["x"].dtype)
    out_dt = _DT[case["out"]]
    if op == "mm":
        x, w = s["x"], s["w"]
        out = torch.empty(x.shape[0], w.shape[1], device="cuda", dtype=out_dt)
        for e, a, b in _segments(s):
            out[a:b] = torch.mm(x[a:b].float(), w[e].float().t())
        return out
    if op == "mm_grad":
        x, w, dout = s["x"], s["w"], s["dout"]
        dx = torch.empty(x.shape, device="cuda", dtype=out_dt)
        dw = torch.zeros(w.shape, device="cuda", dtype=out_dt)
        for e, a, b in _segments(s):
            d = dout[a:b].float()
            dx[a:b] = torch.mm(d, w[e].float())
            dw[e] = torch.mm(d.t(), x[a:b].float())
        return dx, dw
    n, k = case["n"], case["k"]
    x = _mx_values(s["x"].float()[s["token"].long()])
    out = torch.empty(x.shape[0], n, device="cuda", dtype=out_dt)
    for e, a, b in _segments(s):
        w = _mx_decode(s["wc"][e * n:(e + 1) * n], s["ws"][e * n:(e + 1) * n], k)
        out[a:b] = torch.mm(x[a:b], w.t())
    return out


# --------------------------------------------------------------------------
# the framework's calls
# --------------------------------------------------------------------------
def _own(s):
    case, op, eng = s["case"], s["case"]["op"], s["engine"]
    st = torch.cuda.current_stream()
    if op == "norm":
        xo, h = torch.empty_like(s["x"]), torch.empty_like(s["y"])
        eng.block_norm(s["x"], xo, h, s["w_pre"], y=s["y"], w_post=s["w_post"], gate=s["gate"],
                       post_norm=s["w_post"] is not None, residual_scale=s["scale"], eps=s["eps"],
                       stream=st)
        return xo, h
    if op == "norm_grad":
        H = case["hidden"]
        f32 = dict(device="cuda", dtype=torch.float32)
        dx, dy = torch.empty_like(s["x"]), torch.empty_like(s["y"])
        dgate = torch.empty(case["tokens"], **f32) if s["gate"] is not None else None
        dw_post = torch.empty(H, **f32) if s["w_post"] is not None else None
        dw_pre = torch.empty(H, **f32)
        eng.block_norm_backward(s["dx_out"], s["dh"], s["x"], s["w_pre"], dx, dw_pre, y=s["y"],
                                w_post=s["w_post"], gate=s["gate"], dy=dy, dw_post=dw_post,
                                dgate=dgate, post_norm=s["w_post"] is not None,
                                residual_scale=s["scale"], eps=s["eps"], stream=st)
        return dx, dy, dgate, dw_post, dw_pre
    if op == "mx":
        rows = s["token"] if case["gather"] else None
        R = s["off"][-1] if case["gather"] else case["tokens"]
        codes, scales = eng.mxfp4_empty(R, case["k"])
        eng.mxfp4_quantize(s["x"], codes, scales, rows=rows, stream=st)
        out = torch.empty(R, case["k"], device="cuda", dtype=s["x"].dtype)
        eng.mxfp4_dequantize(codes, scales, out, stream=st)
        return out
    out_dt = _DT[case["out"]]
    if op == "mm":
        out = torch.empty(s["x"].shape[0], case["n"], device="cuda", dtype=out_dt)
        eng.grouped_mm(s["x"], s["w"], s["seg_off"], out, stream=st)
        return out
    if op == "mm_grad":
        dx = torch.empty(s["x"].shape, device="cuda", dtype=out_dt)
        dw = torch.empty(s["w"].shape, device="cuda", dtype=out_dt)
        eng.grouped_mm_dgrad(s["dout"], s["w"], s["seg_off"], dx, stream=st)
        eng.grouped_mm_wgrad(s["dout"], s["x"], s["seg_off"], dw, stream=st)
        return dx, dw
    R = s["off"][-1]
    codes, scales = eng.mxfp4_empty(R, case["k"])
    eng.mxfp4_quantize(s["x"], codes, scales, rows=s["token"], stream=st)
    out = torch.empty(R, case["n"], device="cuda", dtype=out_dt)
    eng.grouped_mm_mxfp4(codes, scales, s["wc"], s["ws"], s["seg_off"], case["k"], out, stream=st)
    return out


def run(state):
    return _own(state) if own else _plain(state)


# --------------------------------------------------------------------------
# work and exact values
# --------------------------------------------------------------------------
_SZ = {"bf16": 2, "fp16": 2, "f32": 4}


def work(case):
    T, sz, op = case["tokens"], _SZ[case["dtype"]], case["op"]
    if op in ("norm", "norm_grad"):
        H, rz = case["hidden"], _SZ[case["res"]]
        vec = 4 * H * (2 if case["post"] else 1) + (4 * T if case["gate"] else 0)
        if op == "norm":
            return {"bytes": 2 * T * H * (rz + sz) + vec, "flops": 10 * T * H}
        return {"bytes": 3 * T * H * (rz + sz) + 2 * vec, "flops": 24 * T * H}
    k = case["k"]
    c = counts(case)
    R, active = sum(c), sum(1 for x in c if x)
    if op == "mx":
        rows = R if case["gather"] else T
        nb = -(-k // 32)
        return {"bytes": T * k * sz + rows * k * sz + 2 * rows * nb * 17, "flops": 4 * rows * k}
    n, oz, E = case["n"], _SZ[case["out"]], case["experts"]
    if op == "mm":
        return {"bytes": R * k * sz + active * n * k * sz + R * n * oz + 4 * (E + 1),
                "flops": 2 * R * n * k}
    if op == "mm_grad":
        return {"bytes": R * (n + k) * sz + active * n * k * sz + R * k * oz + E * n * k * oz,
                "flops": 4 * R * n * k}
    row = -(-k // 32) * 17
    return {"bytes": T * k * sz + 2 * R * row + active * n * row + R * n * oz + 4 * R,
            "flops": 2 * R * n * k}


def _grid64(x):
    """The nearest values of each block's 4-bit grid in 64 bits, by distance
    to the sixteen values of the grid; NaN over a block that has a value
    without a finite one."""
    rows, k = x.shape
    pad = torch.zeros(rows, -k % 32, dtype=torch.float64, device=x.device)
    b = torch.cat((x, pad), 1).view(rows, -1, 32)
    top = b.abs().max(-1, keepdim=True).values
    # the exponent field of a 64-bit number is the floor of its binary logarithm
    exp = (top.view(torch.int64) >> 52) - 1023
    step = ((torch.clamp(exp - 2, -127, 127) + 1023) << 52).view(torch.float64)
    u = b.abs() / step
    near = torch.full_like(u, 0.0)
    best = u.clone()
    for i, lv in enumerate(_LEVELS[1:], 1):
        d = (u - lv).abs()
        take = (d < best) | ((d == best) & (i % 2 == 0))
        near = torch.where(take, torch.full_like(u, lv), near)
        best = torch.where(take, d, best)
    v = torch.copysign(near, b) * step
    v = torch.where(torch.isfinite(b).all(-1, keepdim=True), v, torch.full_like(v, math.nan))
    return v.view(rows, -1)[:, :k]


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "norm":
        x, y = s["x"].double(), s["y"].double()
        gate = 1.0 if s["gate"] is None else s["gate"].double().view(-1, 1)
        if s["w_post"] is not None:
            rms = torch.sqrt(torch.einsum("th,th->t", y, y) / y.shape[1] + s["eps"])
            y = y / rms.view(-1, 1) * s["w_post"].double()
        xo = s["scale"] * x + gate * y
        rms = torch.sqrt(torch.einsum("th,th->t", xo, xo) / xo.shape[1] + s["eps"])
        return xo, xo / rms.view(-1, 1) * s["w_pre"].double()
    if op == "norm_grad":
        # the Jacobian of n = v / rms(v) applied to c is (c - n <c, n> / H) / rms
        def unit(v):
            rms = torch.sqrt(torch.einsum("th,th->t", v, v) / v.shape[1] + s["eps"]).view(-1, 1)
            return v / rms, rms

        def back(c, n, rms):
            return (c - n * (torch.einsum("th,th->t", c, n) / n.shape[1]).view(-1, 1)) / rms

        x, y, dh = s["x"].double(), s["y"].double(), s["dh"].double()
        gate = torch.ones(1, 1, dtype=torch.float64, device="cuda")
        if s["gate"] is not None:
            gate = s["gate"].double().view(-1, 1)
        n, rms = unit(x)
        dxo = s["dx_out"].double() + back(dh * s["w_pre"].double(), n, rms)
        dw_pre = torch.einsum("th,th->h", dh, n)
        if s["w_post"] is not None:
            w = s["w_post"].double()
            n, rms = unit(y)
            dy = back(dxo * gate * w, n, rms)
            dw_post = torch.einsum("th,th->h", dxo * gate, n)
            z = n * w
        else:
            dy, dw_post, z = dxo * gate, None, y
        dgate = torch.einsum("th,th->t", dxo, z) if s["gate"] is not None else None
        return s["scale"] * dxo, dy, dgate, dw_post, dw_pre
    if op == "mx":
        v = s["x"].double()
        if case["gather"]:
            return _grid64(v).index_select(0, s["token"].long())
        return torch.cat([_grid64(p) for p in v.split(16384)])
    off = s["off"]
    if op == "mm":
        return torch.cat([s["x"][off[e]:off[e + 1]].double() @ s["w"][e].double().mT
                          for e in range(case["experts"])])
    if op == "mm_grad":
        dx, dw = [], []
        for e in range(case["experts"]):
            d, x = s["dout"][off[e]:off[e + 1]].double(), s["x"][off[e]:off[e + 1]].double()
            dx.append(torch.einsum("rn,nk->rk", d, s["w"][e].double()))
            dw.append(torch.einsum("rn,rk->nk", d, x))
        return torch.cat(dx), torch.stack(dw)
    x = _grid64(s["x"].double()).index_select(0, s["token"].long())
    n, k, out = case["n"], case["k"], []
    grid = torch.tensor([sg * v for sg in (1.0, -1.0) for v in _LEVELS], dtype=torch.float64,
                        device="cuda")
    for e in range(case["experts"]):
        if off[e] == off[e + 1]:
            continue
        c = s["wc"][e * n:(e + 1) * n]
        w = torch.empty(n, 2 * c.shape[1], dtype=torch.float64, device="cuda")
        w[:, 0::2], w[:, 1::2] = grid[(c % 16).int()], grid[(c // 16).int()]
        sb = s["ws"][e * n:(e + 1) * n, :c.shape[1] // 16].long()
        w *= ((sb - 127 + 1023) << 52).view(torch.float64).repeat_interleave(32, 1)
        out.append(x[off[e]:off[e + 1]] @ w[:, :k].mT)
    return torch.cat(out)
