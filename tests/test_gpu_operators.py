"""Grouped products, MXFP4 and block norms on the GPU against plain 64-bit
forms.  Whole-number inputs whose sums fit fp32 make the products exact, so
most of them are compared bit for bit; the rest is held to bounds counted in
roundings (half a step of the result's type, u = 2^-24 for an fp32 one)."""
import threading

import numpy as np
import pytest

torch = pytest.importorskip("torch")
import doantotnghiepmoe_b200 as M  # noqa: E402
from doantotnghiepmoe_b200 import _lib  # noqa: E402

pytestmark = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
U = 2.0 ** -24


@pytest.fixture(scope="module")
def eng():
    e = M.MoeLayerEngine(M.MoeConfig(64, 32, 8, 2, True, 16, 1))
    s = torch.cuda.Stream()
    e.set_stream(s)
    with torch.cuda.stream(s):  # the tests' own tensors are made on the handle's stream
        yield e
    torch.cuda.synchronize()
    e.close()


def half_step(t):
    return torch.finfo(t).eps / 2


def offsets(sizes, gap=0):
    off = np.concatenate(([0], np.cumsum(sizes)))
    return torch.tensor(off, dtype=torch.int32, device="cuda"), int(off[-1]) + gap


def whole(shape, dtype, seed, top=3, pad=8):
    """Whole numbers in rows padded to a multiple of `pad` elements."""
    g = torch.Generator().manual_seed(seed)
    ld = -(-shape[-1] // pad) * pad
    full = torch.randint(-top, top + 1, (*shape[:-1], ld), generator=g).to("cuda", dtype)
    return full[..., :shape[-1]]


def rounded(ref, dtype):
    return ref.to(F32).to(dtype)


SIZES = {
    "one": [1],
    "tokens": [0, 1, 0, 0, 2, 1, 0, 0],
    "ragged": [5, 0, 130, 257, 1, 64, 0, 300],
    "tiles": [256, 512, 128, 16],
    "many": [(7 * e) % 23 for e in range(72)],
    "most": [e % 3 for e in range(256)],
    "none": [0, 0, 0],
}
SHAPES = [("one", 1, 1), ("one", 16, 8), ("tokens", 129, 64), ("tokens", 768, 520),
          ("ragged", 136, 200), ("ragged", 257, 65), ("tiles", 256, 128), ("many", 40, 33),
          ("most", 72, 16), ("none", 32, 32)]


def check_grouped(eng, sizes, n, k, dtype, out_dtype, pad, gap=3, stream=None):
    E = len(sizes)
    off, R = offsets(sizes, gap)
    x, dout = whole((R, k), dtype, 1, pad=pad), whole((R, n), dtype, 2, pad=pad)
    w = whole((E, n, k), dtype, 3, pad=pad)
    keep = 77.0
    out = torch.full((R, n + 3), keep, device="cuda", dtype=out_dtype)[:, :n]
    dx = torch.full((R, k + 1), keep, device="cuda", dtype=out_dtype)[:, :k]
    dw = torch.full((E, n, k), keep, device="cuda", dtype=out_dtype)
    eng.grouped_mm(x, w, off, out)
    eng.grouped_mm_dgrad(dout, w, off, dx)
    eng.grouped_mm_wgrad(dout, x, off, dw)
    eng.sync_status()
    o = off.tolist()
    for e in range(E):
        a, b = o[e], o[e + 1]
        xe, de, we = x[a:b].double(), dout[a:b].double(), w[e].double()
        assert torch.equal(out[a:b], rounded(xe @ we.T, out_dtype)), e
        assert torch.equal(dx[a:b], rounded(de @ we, out_dtype)), e
        assert torch.equal(dw[e], rounded(de.T @ xe, out_dtype)), e
    assert (out[o[-1]:] == keep).all() and (dx[o[-1]:] == keep).all()
    assert (out.as_strided((R, 3), (n + 3, 1), n) == keep).all()


@pytest.mark.parametrize("sizes,n,k", SHAPES)
@pytest.mark.parametrize("dtype,out_dtype", [(BF, F32), (HF, HF), (BF, BF)])
def test_grouped_products_exact(eng, sizes, n, k, dtype, out_dtype):
    check_grouped(eng, SIZES[sizes], n, k, dtype, out_dtype, pad=8)


@pytest.mark.parametrize("sizes,n,k", [("ragged", 65, 33), ("tokens", 8, 7), ("one", 3, 1)])
def test_grouped_products_without_alignment(eng, sizes, n, k):
    check_grouped(eng, SIZES[sizes], n, k, HF, F32, pad=1)


@pytest.mark.parametrize("n,k,out_dtype", [(48, 2056, F32), (641, 640, F32), (1300, 1281, F32),
                                           (72, 4104, F32), (1300, 1281, BF)])
def test_grouped_long_sums(eng, n, k, out_dtype):
    """Sums longer than the ring and than one part, an expert with thousands of rows."""
    check_grouped(eng, [3, 2500, 0, 17, 641], n, k, BF, out_dtype, pad=8)


def test_grouped_normal_values(eng):
    """Normal inputs: each of the k fp32 additions is off by at most a step
    (2 u, the tensor cores may truncate) of the sum of the magnitudes."""
    sizes, n, k = [40, 0, 300, 7], 264, 1000
    off, R = offsets(sizes)
    g = torch.Generator("cuda").manual_seed(0)
    x = torch.randn(R, k, device="cuda", generator=g).to(BF)
    w = (0.02 * torch.randn(4, n, k, device="cuda", generator=g)).to(BF)
    for dt in (F32, BF):
        out = torch.empty(R, n, device="cuda", dtype=dt)
        eng.grouped_mm(x, w, off, out)
        o = off.tolist()
        for e in range(4):
            xe, we = x[o[e]:o[e + 1]].double(), w[e].double()
            ref, mag = xe @ we.T, xe.abs() @ we.abs().T
            tol = 2 * U * k * mag + half_step(dt) * ref.abs()
            assert ((out[o[e]:o[e + 1]].double() - ref).abs() <= tol).all()


# Each addition to a sum in tensor memory is cut off: it loses half a step on average,
# 0.36 * 2^-23 of the sum (the mean of 1 / mantissa is 0.72), always towards zero.  Over
# the n additions of one sum of normal products (16 of K each) that adds up to
# 0.36 * 2^-23 n / sqrt(3) of the result's norm, as partial sums i < j have the
# correlation sqrt(i / j).  With at most 256 of K a sum, n = 16: 4.0e-7, and adding K /
# 256 <= 16 such sums with rounding makes it 4.1e-7 at most.  Sums of 512 of K would
# give 8.0e-7 by that count (4.7e-7 were measured), one sum of 1024 1.6e-6 (1.0e-6).
@pytest.mark.parametrize("K", [640, 1024, 2000, 4096])
def test_grouped_fp32_sums_in_parts(eng, K):
    """fp32 results of normal values, forward and both gradients, the norm of the
    error against 64 bits."""
    g = torch.Generator("cuda").manual_seed(K)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g).to(BF)
    x, w, wt, d = r(200, K), r(2, 144, K), r(2, K, 144), r(200, K)
    off, _ = offsets([130, 70])
    out, dx, dw = (torch.empty(s, device="cuda") for s in ((200, 144), (200, 144), (1, 136, 144)))
    eng.grouped_mm(x, w, off, out)
    eng.grouped_mm_dgrad(d, wt, off, dx)
    xr, dr = r(K, 144), r(K, 136)
    eng.grouped_mm_wgrad(dr, xr, offsets([K])[0], dw)
    eng.sync_status()
    seg = [slice(0, 130), slice(130, 200)]
    ref = [torch.cat([x[s].double() @ w[e].double().T for e, s in enumerate(seg)]),
           torch.cat([d[s].double() @ wt[e].double() for e, s in enumerate(seg)]),
           dr.double().T @ xr.double()]
    for got, want in zip((out, dx, dw[0]), ref):
        assert float((got.double() - want).norm() / want.norm()) <= 4.5e-7


# A part of a 16-bit result's sum takes at most 512 additions (8192 of K, fp16) or 4096
# (65536, bf16).  Each loses less than a step, 2^-23 of the partial sum, whose mean over
# a same-signed sum is half of the result: 2^-15 and 2^-12 at most, a sixteenth of the
# result type's half step.  The parts' rounded additions (at most 64) and the result's
# own rounding to fp32 are below another sixteenth.
@pytest.mark.parametrize("dtype,K", [(HF, 2 ** 18), (BF, 2 ** 20), (HF, 20000), (HF, 8192),
                                     (BF, 100001)])
def test_grouped_16_bit_sums_of_one_sign(eng, dtype, K):
    """16-bit results over many values of one sign: forward, dgrad and the weight
    gradient of an expert with that many rows (and of one with few)."""
    g = torch.Generator("cuda").manual_seed(K)
    r = lambda *s: (1 + torch.rand(*s, device="cuda", generator=g))
    pad = -(-K // 8) * 8
    x = r(5, pad).to(dtype)[:, :K]
    w = (r(1, 16, pad) / 32).to(dtype)[:, :, :K]
    out = torch.empty(5, 16, device="cuda", dtype=dtype)
    eng.grouped_mm(x, w, offsets([5])[0], out)
    wt = (r(1, K, 16) / 32).to(dtype)
    dx = torch.empty(5, 16, device="cuda", dtype=dtype)
    eng.grouped_mm_dgrad(x, wt, offsets([5])[0], dx)
    xr, dr = r(K + 9, 16).to(dtype), (r(K + 9, 8) / 32).to(dtype)
    dw = torch.empty(3, 8, 16, device="cuda", dtype=dtype)
    eng.grouped_mm_wgrad(dr, xr, offsets([9, 0, K])[0], dw)
    eng.sync_status()
    for got, ref in ((out, x.double() @ w[0].double().T), (dx, x.double() @ wt[0].double()),
                     (dw[0], dr[:9].double().T @ xr[:9].double()),
                     (dw[2], dr[9:].double().T @ xr[9:].double())):
        assert ((got.double() - ref).abs() <= 1.125 * half_step(dtype) * ref.abs()).all()
    assert (dw[1] == 0).all()


def test_grouped_nan_rows_stay_with_their_expert(eng):
    """Experts next to one with NaN and infinite rows keep exact results."""
    sizes, n, k = [21, 37, 70, 5], 72, 136
    off, R = offsets(sizes, gap=9)
    x, dout, w = whole((R, k), BF, 4), whole((R, n), BF, 5), whole((4, n, k), BF, 6)
    o = off.tolist()
    for t in (x, dout):
        t[o[1]:o[2]] = float("nan")
        t[o[3]:o[4]] = float("inf")
        t[o[4]:] = float("nan")
    w[1] = float("nan")
    out, dx = (torch.empty(R, m, device="cuda") for m in (n, k))
    dw = torch.empty(4, n, k, device="cuda")
    eng.grouped_mm(x, w, off, out)
    eng.grouped_mm_dgrad(dout, w, off, dx)
    eng.grouped_mm_wgrad(dout, x, off, dw)
    for e in (0, 2):
        xe, de, we = x[o[e]:o[e + 1]].double(), dout[o[e]:o[e + 1]].double(), w[e].double()
        assert torch.equal(out[o[e]:o[e + 1]], (xe @ we.T).float())
        assert torch.equal(dx[o[e]:o[e + 1]], (de @ we).float())
        assert torch.equal(dw[e], (de.T @ xe).float())
    assert out[o[1]:o[2]].isnan().all() and dx[o[1]:o[2]].isnan().all() and dw[1].isnan().all()


def test_grouped_experts_inside_merged_weights(eng):
    """w as a view of merged experts: gate and up rows of [gate | up | down]."""
    E, I, H = 3, 40, 64
    merged = whole((E, 3 * I * H), HF, 7)
    w = merged.as_strided((E, 2 * I, H), (3 * I * H, H, 1))
    off, R = offsets([9, 0, 30])
    x = whole((R, H), HF, 8)
    out = torch.empty(R, 2 * I, device="cuda", dtype=HF)
    eng.grouped_mm(x, w, off, out)
    o = off.tolist()
    for e in range(E):
        assert torch.equal(out[o[e]:o[e + 1]],
                           rounded(x[o[e]:o[e + 1]].double() @ w[e].double().T, HF))


def test_grouped_offsets_past_32_bits(eng):
    """Row strides that put the last rows more than 2^31 elements away."""
    R, n, k, ld = 40000, 24, 40, 65536
    x = torch.empty(R, ld, device="cuda", dtype=BF)[:, :k]
    out = torch.empty(R, ld, device="cuda", dtype=BF)[:, :n]
    x.copy_(whole((R, k), BF, 9))
    w = whole((2, n, k), BF, 10)
    off, _ = offsets([100, R - 100])
    eng.grouped_mm(x, w, off, out)
    assert torch.equal(out[:100], rounded(x[:100].double() @ w[0].double().T, BF))
    assert torch.equal(out[100:], rounded(x[100:].double() @ w[1].double().T, BF))


def test_grouped_bad_offsets_are_reported(eng):
    """Decreasing and outlying offsets: clamped, nothing outside [0, R) is
    touched, and sync_status reports it."""
    x, w = whole((20, 16), BF, 11), whole((3, 8, 16), BF, 12)
    buf = torch.full((60, 8), 5.0, device="cuda")
    for bad in ([0, 12, 4, 20], [-3, 5, 9, 20], [0, 5, 9, 1000]):
        off = torch.tensor(bad, dtype=torch.int32, device="cuda")
        eng.grouped_mm(x, w, off, buf[20:40])
        with pytest.raises(M.MoeError):
            eng.sync_status()
        assert (buf[:20] == 5).all() and (buf[40:] == 5).all()
    eng.sync_status()


def test_grouped_product_rows_bilinear(eng):
    """Both gradients against differences: the product is linear in x and in w,
    so with whole numbers a difference of the sum <c, out> is exact."""
    sizes, n, k = [13, 0, 50], 24, 40
    off, R = offsets(sizes)
    x, w, c = whole((R, k), BF, 13), whole((3, n, k), BF, 14), whole((R, n), BF, 15)
    dxi, dwi = whole((R, k), BF, 16, top=1), whole((3, n, k), BF, 17, top=1)
    out = [torch.empty(R, n, device="cuda") for _ in range(3)]
    eng.grouped_mm(x, w, off, out[0])
    eng.grouped_mm((x + dxi).contiguous(), w, off, out[1])
    eng.grouped_mm(x, (w + dwi).contiguous(), off, out[2])
    dx, dw = torch.empty(R, k, device="cuda"), torch.empty(3, n, k, device="cuda")
    eng.grouped_mm_dgrad(c, w, off, dx)
    eng.grouped_mm_wgrad(c, x, off, dw)
    f = [(c.double() * o.double()).sum() for o in out]
    assert f[1] - f[0] == (dx.double() * dxi.double()).sum()
    assert f[2] - f[0] == (dw.double() * dwi.double()).sum()


# --------------------------------------------------------------------------
# MXFP4
# --------------------------------------------------------------------------
LEVELS = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def mx_ref(x):
    """(nibbles [R, 32 nb], scale bytes [R, nb], values [R, k]) of x in 64 bits."""
    x = x.double().cpu()
    R, k = x.shape
    nb = -(-k // 32)
    b = torch.cat((x, torch.zeros(R, nb * 32 - k, dtype=torch.float64)), 1).view(R, nb, 32)
    top = b.abs().amax(-1)
    e = ((top.view(torch.int64) >> 52) - 1023 - 2).clamp(-127, 127)
    bad = ~torch.isfinite(b).all(-1)
    step = ((e + 1023) << 52).view(torch.float64)[..., None]
    d = ((b / step).abs()[..., None] - LEVELS).abs()
    near = d.min(-1, keepdim=True).values
    tie = d == near  # at most two neighbours: the even code
    first = tie.int().argmax(-1)
    code = torch.where((tie.sum(-1) == 2) & (first % 2 == 1), first + 1, first)
    code = torch.where(torch.isfinite(b), code, torch.zeros_like(code))
    code = torch.where(bad[..., None], torch.zeros_like(code), code)
    val = torch.copysign(LEVELS[code], b) * step
    val = torch.where(bad[..., None], torch.full_like(val, float("nan")), val)
    sign = torch.signbit(b) & ~bad[..., None]
    nib = code + 8 * sign.long()
    sb = torch.where(bad, torch.full_like(e, 255), e + 127)
    return nib.view(R, -1), sb, val.view(R, -1)[:, :k]


def mx_bytes(nib):
    return (nib[:, 0::2] + 16 * nib[:, 1::2]).to(torch.uint8)


@pytest.mark.parametrize("R,k", [(1, 1), (3, 31), (2, 32), (5, 33), (7, 100), (1, 256), (4, 1000),
                                 (33, 2048), (2, 4104), (5, 20000), (700, 9000)])
@pytest.mark.parametrize("dtype", [F32, BF, HF])
def test_mxfp4_quantize_and_back(eng, R, k, dtype):
    g = torch.Generator().manual_seed(R * 1000 + k)
    x = torch.randn(R, k, generator=g) * torch.exp2(torch.randint(-8, 8, (R, k), generator=g))
    x = x.to(dtype).cuda()
    codes, scales = eng.mxfp4_empty(R, k)
    codes.fill_(0x55), scales.fill_(0x55)
    eng.mxfp4_quantize(x, codes, scales)
    nib, sb, val = mx_ref(x)
    assert torch.equal(codes.cpu(), mx_bytes(nib))
    want = torch.zeros(scales.shape, dtype=torch.uint8)
    want[:, :sb.shape[1]] = sb.to(torch.uint8)
    assert torch.equal(scales.cpu(), want)
    for dt in (F32, dtype):
        out = torch.empty(R, k, device="cuda", dtype=dt)
        eng.mxfp4_dequantize(codes, scales, out)
        assert torch.equal(out.cpu(), val.float().to(dt))


def test_mxfp4_borders(eng):
    """Ties between levels, values past the top, powers of two and their
    neighbours, the smallest and largest scales, zeros, infinities and NaN."""
    rows = []
    mids = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0]
    base = torch.tensor(LEVELS.tolist() + mids + [7.0, 7.99], dtype=F32)
    for e in (-60, -1, 0, 3, 100):
        r = torch.zeros(32)
        r[:17], r[17:31] = base, -base[:14]
        rows.append(r * 2.0 ** e)
    for v in (2.0 ** -126, 2.0 ** -127, 2.0 ** -149, 2.0 ** -120, 3.4e38, 2.0 ** 127):
        r = torch.zeros(32)
        r[0], r[5], r[6] = v, -v / 2, v / 4
        rows.append(r)
    one = torch.ones(32)
    nxt = torch.nextafter(one, 2 * one) * 4
    rows += [one, nxt, torch.nextafter(one, 0 * one), torch.zeros(32), -torch.zeros(32)]
    for v in (float("inf"), -float("inf"), float("nan")):
        r = torch.ones(32)
        r[31] = v
        rows.append(r)
    x = torch.stack(rows + [torch.ones(32)]).cuda()
    codes, scales = eng.mxfp4_empty(*x.shape)
    eng.mxfp4_quantize(x, codes, scales)
    nib, sb, val = mx_ref(x)
    assert torch.equal(codes.cpu(), mx_bytes(nib))
    assert torch.equal(scales.cpu()[:, :1], sb.to(torch.uint8))
    out = torch.empty_like(x)
    eng.mxfp4_dequantize(codes, scales, out)
    assert torch.equal(out.cpu().nan_to_num(nan=123.0), val.float().nan_to_num(nan=123.0))


def test_mxfp4_index_and_strides(eng):
    """Rows by index (the same one twice among them), strided and unaligned
    sources; an index outside the source gives zeros and is reported."""
    x = torch.randn(9, 70, device="cuda")[:, 3:67]
    idx = torch.tensor([8, 0, 0, 5, 8, 2], dtype=torch.int32, device="cuda")
    codes, scales = eng.mxfp4_empty(6, 64)
    eng.mxfp4_quantize(x, codes, scales, rows=idx)
    eng.sync_status()
    nib, sb, _ = mx_ref(x[idx.long()])
    assert torch.equal(codes.cpu(), mx_bytes(nib))
    assert torch.equal(scales.cpu()[:, :2], sb.to(torch.uint8))
    idx[1], idx[3] = -1, 9
    eng.mxfp4_quantize(x, codes, scales, rows=idx)
    with pytest.raises(M.MoeError):
        eng.sync_status()
    assert (codes[[1, 3]] == 0).all() and torch.equal(codes.cpu()[4:], mx_bytes(nib)[4:])
    out = torch.full((6, 69), 9.0, device="cuda", dtype=BF)
    eng.mxfp4_dequantize(codes, scales, out[:, 1:65])
    assert (out[:, 0] == 9).all() and (out[:, 65:] == 9).all()


def mx_random(rows, k, seed, lo=126, hi=128):
    """Random codes with scales 2^(lo - 127) .. 2^(hi - 127), and their values."""
    g = torch.Generator().manual_seed(seed)
    nb = -(-k // 32)
    nib = torch.randint(0, 16, (rows, nb * 32), generator=g)
    nib[:, k:] = 0
    sb = torch.randint(lo, hi + 1, (rows, nb), generator=g)
    scales = torch.zeros(rows, -(-nb // 4) * 4, dtype=torch.uint8)
    scales[:, :nb] = sb.to(torch.uint8)
    val = torch.where(nib >= 8, -LEVELS[nib % 8], LEVELS[nib % 8]).view(rows, nb, 32)
    val = (val * torch.exp2(sb.double() - 127)[..., None]).view(rows, -1)[:, :k]
    return mx_bytes(nib).cuda(), scales.cuda(), val.cuda()


@pytest.mark.parametrize("sizes,n,k", SHAPES + [("ragged", 300, 512), ("tiles", 128, 1000),
                                                ("tokens", 1536, 2048), ("many", 130, 160)])
@pytest.mark.parametrize("out_dtype", [F32, BF, HF])
def test_mxfp4_product_exact(eng, sizes, n, k, out_dtype):
    """Values are multiples of 1/4 up to 12 and 2048 products of them stay
    below 2^24 sixteenths: the sums are exact in fp32."""
    sizes = SIZES[sizes]
    E = len(sizes)
    off, R = offsets(sizes, gap=2)
    xc, xs, xv = mx_random(R, k, 1)
    wc, ws, wv = mx_random(E * n, k, 2, lo=127, hi=127)
    out = torch.full((R, n), 77.0, device="cuda", dtype=out_dtype)
    eng.grouped_mm_mxfp4(xc, xs, wc, ws, off, k, out)
    eng.sync_status()
    o = off.tolist()
    for e in range(E):
        ref = xv[o[e]:o[e + 1]] @ wv[e * n:(e + 1) * n].T
        assert torch.equal(out[o[e]:o[e + 1]], rounded(ref, out_dtype)), e
    assert (out[o[-1]:] == 77).all()


def test_mxfp4_product_scales(eng):
    """Scales over a wide range: each block's product is exact, the sum over
    blocks is off by at most 2 u of the magnitudes a block of additions."""
    sizes, n, k = [70, 3], 140, 700
    off, R = offsets(sizes)
    xc, xs, xv = mx_random(R, k, 3, lo=100, hi=150)
    wc, ws, wv = mx_random(2 * n, k, 4, lo=110, hi=140)
    out = torch.empty(R, n, device="cuda")
    eng.grouped_mm_mxfp4(xc, xs, wc, ws, off, k, out)
    o = off.tolist()
    for e in range(2):
        xe, we = xv[o[e]:o[e + 1]], wv[e * n:(e + 1) * n]
        tol = 2 * U * k * (xe.abs() @ we.abs().T)
        assert ((out[o[e]:o[e + 1]].double() - xe @ we.T).abs() <= tol).all()


# One addition to a sum in tensor memory takes 64 of K here: with at most 2048 of K in a
# sum, 0.36 * 2^-23 * 32 / sqrt(3) = 7.9e-7 of the result's norm by the count for the
# 16-bit products above, and the rounded additions of the parts add 1e-8.  One sum of
# all 8192 would give 3.2e-6 by that count, of 16384 6.3e-6 (2.5e-6 measured).
@pytest.mark.parametrize("K", [2048, 8192, 16384, 16000])
def test_mxfp4_fp32_sums_in_parts(eng, K):
    """fp32 results of normal values whose blocks' scales differ, the norm of the
    error against 64 bits."""
    g = torch.Generator("cuda").manual_seed(K)
    r = lambda n: (torch.randn(n, K // 32, 32, device="cuda", generator=g) * torch.exp2(
        torch.randint(-6, 7, (n, K // 32, 1), device="cuda", generator=g).float())).view(n, K)
    off, _ = offsets([140, 60])
    x, w = eng.mxfp4_empty(200, K), eng.mxfp4_empty(2 * 144, K)
    xv, wv = r(200), r(2 * 144)
    eng.mxfp4_quantize(xv, *x)
    eng.mxfp4_quantize(wv, *w)
    eng.mxfp4_dequantize(*x, xv)
    eng.mxfp4_dequantize(*w, wv)
    out = torch.empty(200, 144, device="cuda")
    eng.grouped_mm_mxfp4(*x, *w, off, K, out)
    eng.sync_status()
    xv, wv = xv.double(), wv.double().view(2, 144, K)
    ref = torch.cat((xv[:140] @ wv[0].T, xv[140:] @ wv[1].T))
    assert float((out.double() - ref).norm() / ref.norm()) <= 9e-7


@pytest.mark.parametrize("sizes,n,k,out_dtype", [
    ("ragged", 136, 4352, F32), ("tiles", 300, 2080, F32), ("tokens", 129, 10000, F32),
    ("many", 40, 2049, F32), ("none", 32, 8192, F32), ("tokens", 8, 140000, HF)])
def test_mxfp4_long_sums_exact(eng, sizes, n, k, out_dtype):
    """Sums of several parts over every kind of tile.  Values are multiples of 1/4 up
    to 12, scaled down so that 16-bit results stay finite; with signs at random the
    sums of up to 140000 products stay below 2^24 of their grid."""
    sizes = SIZES[sizes]
    E = len(sizes)
    off, R = offsets(sizes, gap=2)
    xc, xs, xv = mx_random(R, k, 1)
    wc, ws, wv = mx_random(E * n, k, 2, lo=123, hi=123)
    out = torch.full((R, n), 77.0, device="cuda", dtype=out_dtype)
    eng.grouped_mm_mxfp4(xc, xs, wc, ws, off, k, out)
    eng.sync_status()
    o = off.tolist()
    for e in range(E):
        ref = xv[o[e]:o[e + 1]] @ wv[e * n:(e + 1) * n].T
        assert torch.equal(out[o[e]:o[e + 1]], rounded(ref, out_dtype)), e
    assert (out[o[-1]:] == 77).all()


# 2^20 of K in parts of 2^17: 2048 additions of one sign lose at most 2^-23 each of a
# sum whose mean is half of the result, 2^-13, a quarter of fp16's half step.  (One sum of
# all was 3.1e-4 short, two thirds of half a step, beside the rounding.)
def test_mxfp4_fp16_sums_of_one_sign(eng):
    K, n, R = 2 ** 20, 64, 40
    g = torch.Generator("cuda").manual_seed(1)
    c, v = [], []
    for rows, shift in ((R, 0), (n, -24)):
        r = 1 + torch.rand(rows, K // 32, 32, device="cuda", generator=g)
        r *= torch.exp2(torch.randint(-6, 7, (rows, K // 32, 1), device="cuda", generator=g) +
                        float(shift))
        c += eng.mxfp4_empty(rows, K)
        eng.mxfp4_quantize(r.view(rows, K), *c[-2:])
        v.append(torch.empty(rows, K, device="cuda"))
        eng.mxfp4_dequantize(*c[-2:], v[-1])
    out = torch.empty(R, n, device="cuda", dtype=HF)
    eng.grouped_mm_mxfp4(*c, offsets([R])[0], K, out)
    eng.sync_status()
    ref = v[0].double() @ v[1].double().T
    assert 1 < float(ref.min()) and float(ref.max()) < 60000
    assert ((out.double() - ref).abs() <= 1.25 * half_step(HF) * ref).all()


def test_mxfp4_product_nan_blocks(eng):
    """A NaN block makes the outputs that use it NaN and no others."""
    sizes, n, k = [5, 6], 40, 96
    off, R = offsets(sizes)
    xc, xs, xv = mx_random(R, k, 5)
    wc, ws, wv = mx_random(2 * n, k, 6, lo=127, hi=127)
    xs[4, 1] = 255
    ws[n + 7, 2] = 255
    out = torch.empty(R, n, device="cuda")
    eng.grouped_mm_mxfp4(xc, xs, wc, ws, off, k, out)
    ref = torch.cat((xv[:5] @ wv[:n].T, xv[5:] @ wv[n:].T)).float()
    ref[4] = float("nan")
    ref[5:, 7] = float("nan")
    assert torch.equal(out.isnan(), ref.isnan())
    assert torch.equal(out.nan_to_num(nan=0.0), ref.nan_to_num(nan=0.0))


# --------------------------------------------------------------------------
# Norms of a block
# --------------------------------------------------------------------------
PAIRS = [(F32, F32), (BF, BF), (HF, HF), (F32, BF), (F32, HF)]
# (rows, width): one row, odd widths, a warp's and a block's edges, wide rows
NORM_SHAPES = [(1, 1), (1, 2048), (3, 7), (5, 32), (2, 257), (700, 64), (9, 1000), (4, 2056),
               (2, 5000), (2, 16384), (2, 16383), (1300, 136), (2500, 250), (1300, 505), (601, 2048), (602, 1001), (500, 4096), (450, 8192)]


def norm_inputs(T, H, rd, bd, seed, gate=True):
    g = torch.Generator("cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)
    return dict(x=(2 * r(T, H)).to(rd), y=r(T, H).to(bd), w_pre=1 + 0.3 * r(H),
                w_post=1 + 0.3 * r(H), gate=torch.sigmoid(r(T)) if gate else None)


def norm_ref(i, post, scale, eps):
    d = {k: None if v is None else v.double() for k, v in i.items()}
    g = 1.0 if d["gate"] is None else d["gate"][:, None]
    z = d["y"]
    if post:
        z = z / (z.pow(2).mean(-1, keepdim=True) + eps).sqrt() * d["w_post"]
    xo = scale * d["x"] + g * z
    mag = (scale * d["x"]).abs() + (g * z).abs()
    rms = (xo.pow(2).mean(-1, keepdim=True) + eps).sqrt()
    return xo, xo / rms * d["w_pre"], mag, mag / rms * d["w_pre"].abs()


# A thread adds at most 64 squares in a row and joins them over 5 + 8 steps;
# 1 / rms halves that error, and the products around it add fewer than 10:
# 64 u of the magnitudes is above all of it.  The second norm carries the
# first one's error through x_out and through its own rms: 192 u.
@pytest.mark.parametrize("T,H", NORM_SHAPES)
@pytest.mark.parametrize("rd,bd", PAIRS)
@pytest.mark.parametrize("post,gate", [(True, True), (True, False), (False, True)])
def test_block_norm(eng, T, H, rd, bd, post, gate):
    i = norm_inputs(T, H, rd, bd, T + H, gate)
    xo, h = torch.empty_like(i["x"]), torch.empty_like(i["y"])
    eng.block_norm(i["x"], xo, h, i["w_pre"], y=i["y"], w_post=i["w_post"], gate=i["gate"],
                   post_norm=post, residual_scale=0.75, eps=1e-5)
    rx, rh, mx, mh = norm_ref(i, post, 0.75, 1e-5)
    row = mx.pow(2).mean(-1, keepdim=True).sqrt() / (rx.pow(2).mean(-1, keepdim=True) + 1e-5).sqrt()
    tiny = torch.finfo(rd).tiny, torch.finfo(bd).tiny
    assert ((xo.double() - rx).abs() <= 64 * U * mx + half_step(rd) * rx.abs() + tiny[0]).all()
    assert ((h.double() - rh).abs() <= 192 * U * mh * (1 + row) +
            half_step(bd) * rh.abs() + tiny[1]).all()


@pytest.mark.parametrize("T,H", [(5, 264), (700, 1024), (2, 4096)])
@pytest.mark.parametrize("rd,bd", [(BF, BF), (F32, HF)])
def test_norms_off_a_16_byte_border(eng, T, H, rd, bd):
    """Widths that 16-byte accesses would take, from addresses that they would not."""
    i = norm_inputs(T, H, rd, bd, T + H)
    place = lambda t: torch.cat((t.new_zeros(1), t.flatten()))[1:].view(t.shape)
    off = {k: None if v is None else place(v) for k, v in i.items()}
    assert off["x"].data_ptr() % 16 and off["w_pre"].data_ptr() % 16
    xo, h = place(i["x"]), place(i["y"])
    eng.block_norm(off["x"], xo, h, off["w_pre"], y=off["y"], w_post=off["w_post"],
                   gate=off["gate"], residual_scale=0.75, eps=1e-5)
    rx, rh, mx, mh = norm_ref(i, True, 0.75, 1e-5)
    row = mx.pow(2).mean(-1, keepdim=True).sqrt() / (rx.pow(2).mean(-1, keepdim=True) + 1e-5).sqrt()
    tiny = torch.finfo(rd).tiny, torch.finfo(bd).tiny
    assert ((xo.double() - rx).abs() <= 64 * U * mx + half_step(rd) * rx.abs() + tiny[0]).all()
    assert ((h.double() - rh).abs() <= 192 * U * mh * (1 + row) +
            half_step(bd) * rh.abs() + tiny[1]).all()
    dxo, dh = (torch.randn(T, H, device="cuda").to(t) for t in (rd, bd))
    got = dict(dx=place(dxo), dy=place(dh), dw_pre=place(i["w_pre"]), dw_post=place(i["w_pre"]),
               dgate=torch.empty(T, device="cuda"))
    eng.block_norm_backward(place(dxo), place(dh), off["x"], off["w_pre"], got["dx"],
                            got["dw_pre"], y=off["y"], w_post=off["w_post"], gate=off["gate"],
                            dy=got["dy"], dw_post=got["dw_post"], dgate=got["dgate"],
                            residual_scale=0.75, eps=1e-5)
    ref, mag = backward_ref(i, dxo, dh, True, 0.75, 1e-5)
    for k, v in got.items():
        steps = 256 + (T if k.startswith("dw") else 0)
        tol = steps * U * mag[k] + half_step(v.dtype) * ref[k].abs() + torch.finfo(v.dtype).tiny
        assert ((v.double() - ref[k]).abs() <= tol).all(), k


def test_block_norm_parts(eng):
    """Without y (the first norm alone), without h (behind the last block),
    without gains, in place, and rows in wider buffers."""
    T, H = 6, 72
    i = norm_inputs(T, H, F32, BF, 3)
    h = torch.empty_like(i["y"])
    eng.block_norm(i["x"], None, h, i["w_pre"])
    x = i["x"].double()
    ref = x / (x.pow(2).mean(-1, keepdim=True) + 1e-5).sqrt() * i["w_pre"].double()
    assert ((h.double() - ref).abs() <= (64 * U + half_step(BF)) * ref.abs()).all()
    full = [torch.empty_like(i["x"]), torch.empty_like(i["y"])]
    eng.block_norm(i["x"], *full, i["w_pre"], y=i["y"], w_post=i["w_post"], gate=i["gate"])
    only = torch.empty_like(i["x"])
    eng.block_norm(i["x"], only, None, y=i["y"], w_post=i["w_post"], gate=i["gate"])
    assert torch.equal(only, full[0])
    wide_x = torch.full((T, H + 8), 5.0, device="cuda")
    wide_y = torch.full((T, H + 16), 5.0, device="cuda", dtype=BF)
    xv, yv = wide_x[:, :H], wide_y[:, :H]
    xv.copy_(i["x"]), yv.copy_(i["y"])
    eng.block_norm(xv, xv, yv, i["w_pre"], y=yv, w_post=i["w_post"], gate=i["gate"])
    assert torch.equal(xv, full[0]) and torch.equal(yv, full[1])
    assert (wide_x[:, H:] == 5).all() and (wide_y[:, H:] == 5).all()
    ones = torch.ones(H, device="cuda")
    a, b = ([torch.empty_like(i["x"]), torch.empty_like(i["y"])] for _ in range(2))
    eng.block_norm(i["x"], *a, None, y=i["y"])
    eng.block_norm(i["x"], *b, ones, y=i["y"], w_post=ones, gate=torch.ones(T, device="cuda"))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def backward_ref(i, dxo, dh, post, scale, eps):
    """Gradients by autograd of the 64-bit formula at x_out, and bounds of the
    terms that are added into each (their magnitudes)."""
    d = {k: None if v is None else v.double().clone().requires_grad_() for k, v in i.items()}
    x = d["x"]  # x_out of the pass
    rms = (x.pow(2).mean(-1, keepdim=True) + eps).sqrt()
    dh_, dxo_ = dh.double(), dxo.double()
    (dX,) = torch.autograd.grad(x / rms * d["w_pre"], x, dh_, retain_graph=True)
    (dwp,) = torch.autograd.grad(x / rms * d["w_pre"], d["w_pre"], dh_)
    D = (dX + dxo_).detach()
    g = torch.ones_like(D[:, :1]) if d["gate"] is None else d["gate"][:, None]
    z = d["y"]
    if post:
        z = z / (z.pow(2).mean(-1, keepdim=True) + eps).sqrt() * d["w_post"]
    out = g * z
    want = [d["y"]] + ([d["w_post"]] if post else []) + ([d["gate"]] if d["gate"] is not None else [])
    gr = dict(zip([id(w) for w in want], torch.autograd.grad(out, want, D)))
    with torch.no_grad():
        x, rms, c = x.detach(), rms.detach(), (dh_ * d["w_pre"]).detach()
        mD = dxo_.abs() + c.abs() / rms + x.abs() / rms ** 3 * (c * x).abs().mean(-1, keepdim=True)
        y, w = d["y"].detach(), d["w_post"].detach() if post else torch.ones_like(x[0])
        rp = 1 / (y.pow(2).mean(-1, keepdim=True) + eps).sqrt() if post else torch.ones_like(rms)
        mS = (mD * w.abs() * y.abs()).sum(-1, keepdim=True)
        my = g.detach() * rp * (mD * w.abs())
        if post:
            my = my + g.detach() * rp ** 3 * y.abs() * mS / y.shape[1]
        mag = dict(dx=scale * mD, dy=my, dgate=(rp * mS)[:, 0],
                   dw_pre=(dh_ * x / rms).abs().sum(0),
                   dw_post=(g.detach() * mD * y.abs() * rp).sum(0))
    ref = dict(dx=scale * D, dy=gr[id(d["y"])], dw_pre=dwp,
               dw_post=gr[id(d["w_post"])] if post else None,
               dgate=gr[id(d["gate"])] if d["gate"] is not None else None)
    return {k: None if v is None else v.detach() for k, v in ref.items()}, mag


# Row sums as above (at most 64 + 13 additions), three of them in a chain with
# fewer than 20 products: 256 u of the magnitudes; over the rows a CTA and
# the joining kernel add at most T more steps.
@pytest.mark.parametrize("T,H", NORM_SHAPES)
@pytest.mark.parametrize("rd,bd", PAIRS)
@pytest.mark.parametrize("post,gate", [(True, True), (False, True), (True, False)])
def test_block_norm_backward(eng, T, H, rd, bd, post, gate):
    i = norm_inputs(T, H, rd, bd, 7 * T + H, gate)
    g = torch.Generator("cuda").manual_seed(1)
    dxo = torch.randn(T, H, device="cuda", generator=g).to(rd)
    dh = torch.randn(T, H, device="cuda", generator=g).to(bd)
    f = dict(device="cuda", dtype=F32)
    got = dict(dx=torch.empty_like(i["x"]), dy=torch.empty_like(i["y"]),
               dw_pre=torch.empty(H, **f), dw_post=torch.empty(H, **f) if post else None,
               dgate=torch.empty(T, **f) if gate else None)
    eng.block_norm_backward(dxo, dh, i["x"], i["w_pre"], got["dx"], got["dw_pre"], y=i["y"],
                            w_post=i["w_post"], gate=i["gate"], dy=got["dy"],
                            dw_post=got["dw_post"], dgate=got["dgate"], post_norm=post,
                            residual_scale=0.75, eps=1e-5)
    ref, mag = backward_ref(i, dxo, dh, post, 0.75, 1e-5)
    for k, v in got.items():
        if v is None:
            continue
        steps = 256 + (T if k.startswith("dw") else 0)
        tol = steps * U * mag[k] + half_step(v.dtype) * ref[k].abs() + torch.finfo(v.dtype).tiny
        bad = (v.double() - ref[k]).abs() > tol
        assert not bad.any(), (k, int(bad.sum()))


def test_block_norm_backward_parts(eng):
    """Absent gradients are zeros, absent outputs are not needed, gradients in
    place, no rows; the gains' gradients are the same bits each time."""
    T, H = 900, 264
    i = norm_inputs(T, H, F32, F32, 5)
    dxo, dh = torch.randn(T, H, device="cuda"), torch.randn(T, H, device="cuda")
    zero = torch.zeros_like(dxo)

    def call(dxo, dh, **kw):
        o = [torch.empty_like(dxo if dxo is not None else dh) for _ in range(2)]
        w = [torch.empty(H, device="cuda") for _ in range(2)]
        eng.block_norm_backward(dxo, dh, i["x"], i["w_pre"], o[0], w[0], y=i["y"],
                                w_post=i["w_post"], gate=i["gate"], dy=o[1], dw_post=w[1], **kw)
        return o + w

    for a, b in ((call(None, dh), call(zero, dh)), (call(dxo, None), call(dxo, zero)),
                 (call(dxo, dh), call(dxo, dh))):
        assert all(torch.equal(p, q) for p, q in zip(a, b))
    ref = call(dxo, dh)
    a, b = dxo.clone(), dh.clone()
    eng.block_norm_backward(a, b, i["x"], i["w_pre"], a, y=i["y"], w_post=i["w_post"],
                            gate=i["gate"], dy=b)
    assert torch.equal(a, ref[0]) and torch.equal(b, ref[1])
    eng.block_norm_backward(dxo, dh, i["x"], i["w_pre"], a)  # the first norm alone
    assert torch.equal(a, ref[0])
    w = torch.full((H,), 3.0, device="cuda")
    e = torch.empty(0, H, device="cuda")
    eng.block_norm_backward(e, e, e, i["w_pre"], torch.empty_like(e), w)
    assert (w == 0).all()


# The bounds of test_block_norm_backward count the roundings of the formula, whose
# terms stay in fp32's range here: the squares reach 2^100 and 2^-100, and the
# results differ from rows of size one by the powers of two alone.
@pytest.mark.parametrize("T,H", [(3, 264), (3, 257), (1, 2048), (700, 1032), (2500, 64)])
@pytest.mark.parametrize("rd,bd", [(F32, F32), (F32, BF), (BF, BF)])
@pytest.mark.parametrize("exponent,eps", [(50, 1e-5), (-50, 0.0)])
@pytest.mark.parametrize("post", [True, False])
def test_block_norm_backward_of_far_rows(eng, T, H, rd, bd, exponent, eps, post):
    """Rows of 2^50 and, without eps, of 2^-50: the terms along the row itself
    neither vanish nor overflow."""
    i = norm_inputs(T, H, rd, bd, 9 * T + H)
    i["x"], i["y"] = i["x"] * 2.0 ** exponent, i["y"] * 2.0 ** exponent
    g = torch.Generator("cuda").manual_seed(2)
    dxo = torch.randn(T, H, device="cuda", generator=g) * 2.0 ** -exponent
    dxo, dh = dxo.to(rd), torch.randn(T, H, device="cuda", generator=g).to(bd)
    f = dict(device="cuda", dtype=F32)
    got = dict(dx=torch.empty_like(i["x"]), dy=torch.empty_like(i["y"]),
               dw_pre=torch.empty(H, **f), dw_post=torch.empty(H, **f) if post else None,
               dgate=torch.empty(T, **f))
    eng.block_norm_backward(dxo, dh, i["x"], i["w_pre"], got["dx"], got["dw_pre"], y=i["y"],
                            w_post=i["w_post"], gate=i["gate"], dy=got["dy"],
                            dw_post=got["dw_post"], dgate=got["dgate"], post_norm=post,
                            residual_scale=0.75, eps=eps)
    ref, mag = backward_ref(i, dxo, dh, post, 0.75, eps)
    for k, v in got.items():
        if v is None:
            continue
        steps = 256 + (T if k.startswith("dw") else 0)
        tol = steps * U * mag[k] + half_step(v.dtype) * ref[k].abs() + torch.finfo(v.dtype).tiny
        bad = ~((v.double() - ref[k]).abs() <= tol)
        assert not bad.any(), (k, int(bad.sum()))


def test_block_norm_of_far_rows(eng):
    """The forward pass of the same rows."""
    for exponent, eps in ((50, 1e-5), (-50, 0.0)):
        for T, H in ((3, 264), (3, 257)):
            i = norm_inputs(T, H, F32, F32, T + H)
            i["x"], i["y"] = i["x"] * 2.0 ** exponent, i["y"] * 2.0 ** exponent
            xo, h = torch.empty_like(i["x"]), torch.empty_like(i["y"])
            eng.block_norm(i["x"], xo, h, i["w_pre"], y=i["y"], w_post=i["w_post"],
                           gate=i["gate"], residual_scale=0.75, eps=eps)
            rx, rh, mx, mh = norm_ref(i, True, 0.75, eps)
            row = mx.pow(2).mean(-1, keepdim=True).sqrt() / rx.pow(2).mean(-1, keepdim=True).sqrt()
            assert ((xo.double() - rx).abs() <= 64 * U * mx + U * rx.abs()).all()
            assert ((h.double() - rh).abs() <= 192 * U * mh * (1 + row) + U * rh.abs()).all()


def test_block_norm_gradient_by_differences(eng):
    """<c, x_out> + <d, h> along a direction: the central difference of the fp32
    forward pass.  With steps of 2^-8 the difference is off by its third
    derivative (2^-16) and by the roundings of the values, 2^8 u sqrt(TH) of
    them: 1e-3 of the gradient's size is above both."""
    T, H = 4, 96
    i = norm_inputs(T, H, F32, F32, 11)
    c, d = torch.randn(T, H, device="cuda"), torch.randn(T, H, device="cuda")
    dirs = {k: torch.randn_like(i[k]) for k in ("x", "y", "w_pre", "w_post", "gate")}

    def fwd(t):
        j = {k: v + t * dirs[k] for k, v in i.items()}
        xo, h = torch.empty_like(i["x"]), torch.empty_like(i["y"])
        eng.block_norm(j["x"], xo, h, j["w_pre"], y=j["y"], w_post=j["w_post"], gate=j["gate"],
                       residual_scale=0.5)
        return xo, h

    val = lambda o: (o[0].double() * c).sum() + (o[1].double() * d).sum()
    diff = (val(fwd(2.0 ** -8)) - val(fwd(-2.0 ** -8))) * 2.0 ** 7
    xo, _ = fwd(0.0)
    dx, dy = torch.empty_like(xo), torch.empty_like(xo)
    dwq, dwp, dg = (torch.empty_like(i[k]) for k in ("w_pre", "w_post", "gate"))
    eng.block_norm_backward(c, d, xo, i["w_pre"], dx, dwq, y=i["y"], w_post=i["w_post"],
                            gate=i["gate"], dy=dy, dw_post=dwp, dgate=dg, residual_scale=0.5)
    terms = [(a.double() * dirs[k]).sum() for a, k in
             ((dx, "x"), (dy, "y"), (dwq, "w_pre"), (dwp, "w_post"), (dg, "gate"))]
    assert abs(float(sum(terms) - diff)) <= 1e-3 * float(sum(t.abs() for t in terms))


@pytest.mark.parametrize("dt,widths", [(F32, (1152, 1536)), (BF, (2048, 1032))])
def test_block_norm_backward_from_two_threads(eng, dt, widths):
    """Two engines on two host threads, each with its own width and stream: the
    widths run the same kernel with rings of different sizes, and no call is
    refused.  The calls go straight to the C ABI, which two threads are inside of
    at the same time then (the interpreter's lock is free only there)."""
    T, L, jobs = 600, M.lib(), []
    for j, H in enumerate(widths):
        i = norm_inputs(T, H, dt, dt, 100 + H)
        g = torch.Generator("cuda").manual_seed(H)
        dxo, dh = (torch.randn(T, H, device="cuda", generator=g).to(dt) for _ in range(2))
        e, stream = M.MoeLayerEngine(M.MoeConfig(64, 32, 8, 2, True, 16, 1)), torch.cuda.Stream()
        got, ref = ([torch.empty_like(dxo), torch.empty_like(dh)] for _ in range(2))
        eng.block_norm_backward(dxo, dh, i["x"], i["w_pre"], ref[0], y=i["y"],
                                w_post=i["w_post"], gate=i["gate"], dy=ref[1])
        need = L.moe_block_norm_backward_workspace(e._h, T, H)
        ws = torch.empty(need, dtype=torch.uint8, device="cuda")
        code = {F32: _lib.MOE_DT_F32, BF: _lib.MOE_DT_BF16}[dt]
        d = _lib.MoeBlockNormDesc(T, H, code, code, H, H, 1, 1.0, 1e-5)
        args = (e._h, d, *(t.data_ptr() for t in (dxo, dh, i["x"], i["y"], i["w_post"], i["gate"],
                                                  i["w_pre"], *got)),
                None, None, None, ws.data_ptr(), need, stream.cuda_stream)
        jobs.append(dict(args=args, e=e, got=got, ref=ref, stream=stream, keep=(i, dxo, dh, ws),
                         refused=0))
    torch.cuda.synchronize()
    start = threading.Barrier(2)

    def work(job):
        f, args = L.moe_block_norm_backward, job["args"]
        start.wait(60)
        for n in range(10000):
            job["refused"] += f(*args) != _lib.MOE_OK
            if n % 500 == 499:
                job["stream"].synchronize()

    threads = [threading.Thread(target=work, args=(j,)) for j in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    errors = [(j["refused"], L.moe_last_error(j["e"]._h)) for j in jobs]
    for j in jobs:
        j["e"].close()
    assert [n for n, _ in errors] == [0, 0], errors
    for j in jobs:
        assert all(map(torch.equal, j["got"], j["ref"]))


@pytest.mark.parametrize("dt,widths", [(F32, (1152, 1536)), (BF, (2048, 1032))])
def test_block_norm_backward_widths_in_one_graph(eng, dt, widths):
    """One graph with both widths, the larger ring captured first."""
    jobs = []
    for H in widths:
        i = norm_inputs(600, H, dt, dt, 200 + H)
        dx, ref = torch.empty_like(i["x"]), torch.empty_like(i["x"])
        eng.block_norm_backward(i["x"], i["y"], i["x"], i["w_pre"], ref)
        jobs.append((i, dx, ref))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for i, dx, _ in jobs:
            eng.block_norm_backward(i["x"], i["y"], i["x"], i["w_pre"], dx,
                                    stream=torch.cuda.current_stream())
    graph.replay()
    torch.cuda.synchronize()
    for _, dx, ref in jobs:
        assert torch.equal(dx, ref)


def one_row(width, dtype, seed, stride=None):
    """[1, width] with a row stride that addresses nothing."""
    ld = stride or 3 * width + 1
    t = torch.zeros(2, ld, device="cuda", dtype=dtype)[:1, :width]
    t.copy_(whole((1, width), dtype, seed))
    assert t.stride() == (ld, 1)
    return t


def test_one_row_has_no_stride(eng):
    """A single row out of a wider buffer beside contiguous tensors, in every
    call: its stride means nothing, so the results are those of a copy."""
    H, n = 264, 136
    x, y = one_row(H, F32, 1), one_row(H, BF, 2)
    pre, post = torch.rand(H, device="cuda"), torch.rand(H, device="cuda")
    res = []
    for a, b in ((x, y), (x.contiguous().view(1, H), y.clone().view(1, H))):
        xo, h = torch.empty(1, H, device="cuda"), torch.empty(1, H, device="cuda", dtype=BF)
        eng.block_norm(a, xo, h, pre, y=b, w_post=post)
        dx, dy = torch.empty(1, H, device="cuda"), one_row(H, BF, 3, stride=1001)
        dw = torch.empty(H, device="cuda")
        eng.block_norm_backward(a, h, xo, pre, dx, dw, y=b, w_post=post, dy=dy)
        c = eng.mxfp4_empty(1, H)
        eng.mxfp4_quantize(a, *c)
        back = one_row(H, F32, 4, stride=777)
        eng.mxfp4_dequantize(*c, back)
        res.append([xo, h, dx, dy.clone(), dw, *c, back.clone()])
    assert all(map(torch.equal, *res))
    off, _ = offsets([0, 1, 0])
    w = whole((3, n, H), BF, 5)
    d = one_row(n, BF, 6)
    out, dx = one_row(n, F32, 7, stride=555), one_row(H, F32, 8, stride=555)
    dw = torch.empty(3, n, H, device="cuda")
    eng.grouped_mm(y, w, off, out)
    eng.grouped_mm_dgrad(d, w, off, dx)
    eng.grouped_mm_wgrad(d, y, off, dw)
    eng.sync_status()
    assert torch.equal(out, (y.double() @ w[1].double().T).float())
    assert torch.equal(dx, (d.double() @ w[1].double()).float())
    assert torch.equal(dw[1], (d.double().T @ y.double()).float())
    assert (dw[0] == 0).all() and (dw[2] == 0).all()


def test_one_row_with_any_stride_at_the_c_abi(eng):
    """The stride of a single row is not looked at, 0 and huge numbers included."""
    L, k, n = M.lib(), 72, 40
    st = torch.cuda.current_stream().cuda_stream
    x, w = whole((1, k), BF, 1), whole((1, n, k), BF, 2)
    off, _ = offsets([1])
    for ld in (0, -5, 3, 2 ** 50):
        out, h = torch.full((n,), 7.0, device="cuda"), torch.full((k,), 7.0, device="cuda")
        back = torch.full((k,), 7.0, device="cuda")
        d = _lib.MoeGroupedDesc(1, 1, n, k, _lib.MOE_DT_BF16, _lib.MOE_DT_F32, ld, k, 0, ld)
        assert L.moe_grouped_mm(eng._h, d, x.data_ptr(), w.data_ptr(), off.data_ptr(),
                                out.data_ptr(), st) == _lib.MOE_OK
        b = _lib.MoeBlockNormDesc(1, k, _lib.MOE_DT_F32, _lib.MOE_DT_F32, ld, ld, 1, 1.0, 1e-5)
        xf = x.float()
        assert L.moe_block_norm(eng._h, b, xf.data_ptr(), None, None, None, None, None,
                                h.data_ptr(), st) == _lib.MOE_OK
        c = eng.mxfp4_empty(1, k)
        assert L.moe_mxfp4_quantize(eng._h, x.data_ptr(), _lib.MOE_DT_BF16, ld, 1, None, 1, k,
                                    *(t.data_ptr() for t in c), st) == _lib.MOE_OK
        assert L.moe_mxfp4_dequantize(eng._h, *(t.data_ptr() for t in c), 1, k, back.data_ptr(),
                                      _lib.MOE_DT_F32, ld, st) == _lib.MOE_OK
        eng.sync_status()
        torch.cuda.synchronize()
        assert torch.equal(out, (x.double() @ w[0].double().T).float()[0])
        ref = xf[0].double() / (xf.double().pow(2).mean() + 1e-5).sqrt()
        assert ((h.double() - ref).abs() <= 65 * U * ref.abs()).all()
        assert torch.equal(back.cpu(), mx_ref(x)[2][0].float())


# --------------------------------------------------------------------------
# together, streams, graphs, refusals
# --------------------------------------------------------------------------
def moe_block(eng, s, stream=None):
    """Norm, permutation, both products of a SwiGLU expert (16-bit or 4-bit),
    combine, and the next norm: what a caller builds from the operators."""
    T, H, K, I = s["T"], s["H"], s["K"], s["I"]
    R, dev = T * K, "cuda"
    h = torch.empty(T, H, device=dev, dtype=BF)
    eng.block_norm(s["x"], None, h, s["g0"], stream=stream)
    ids = torch.empty(T, K, dtype=torch.int32, device=dev)
    gates = torch.empty(T, K, device=dev)
    off = torch.empty(s["E"] + 1, dtype=torch.int32, device=dev)
    tok, slot = (torch.empty(R, dtype=torch.int32, device=dev) for _ in range(2))
    hf = h.float()
    eng.route_permute(0, hf, ids, gates, off, tok, slot, stream=stream)
    gu = torch.empty(R, 2 * I, device=dev)
    y = torch.empty(R, H, device=dev)
    if s["mx"]:
        c = eng.mxfp4_empty(R, H)
        eng.mxfp4_quantize(h, *c, rows=tok, stream=stream)
        eng.grouped_mm_mxfp4(*c, *s["wgu4"], off, H, gu, stream=stream)
    else:
        eng.grouped_mm(h[tok.long()], s["wgu"], off, gu, stream=stream)
    act = (torch.nn.functional.silu(gu[:, :I]) * gu[:, I:]).to(BF)
    if s["mx"]:
        c = eng.mxfp4_empty(R, I)
        eng.mxfp4_quantize(act, *c, stream=stream)
        eng.grouped_mm_mxfp4(*c, *s["wd4"], off, I, y, stream=stream)
    else:
        eng.grouped_mm(act, s["wd"], off, y, stream=stream)
    flat = torch.zeros(R, H, device=dev)
    flat[tok.long() * K + slot.long()] = y
    out = (flat.view(T, K, H) * gates[..., None]).sum(1).to(BF)
    x1, h1 = torch.empty_like(s["x"]), torch.empty_like(out)
    eng.block_norm(s["x"], x1, h1, s["g1"], y=out, w_post=s["g2"], stream=stream)
    return dict(h=h, gu=gu, act=act, y=y, out=out, x1=x1, h1=h1, ids=ids, gates=gates, off=off,
                tok=tok)


def block_state(eng, mx, T=16, H=64, I=32, E=8, K=2):
    g = torch.Generator("cuda").manual_seed(21)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)
    s = dict(T=T, H=H, I=I, E=E, K=K, mx=mx, x=r(T, H), g0=1 + 0.1 * r(H), g1=1 + 0.1 * r(H),
             g2=1 + 0.1 * r(H), wgu=(0.1 * r(E, 2 * I, H)).to(BF), wd=(0.1 * r(E, H, I)).to(BF))
    for name, w in (("wgu4", s["wgu"]), ("wd4", s["wd"])):
        flat = w.reshape(-1, w.shape[-1])
        s[name] = eng.mxfp4_empty(*flat.shape)
        eng.mxfp4_quantize(flat, *s[name])
    from oracle import oracle as O
    lw = O.synth_layer(5, 0, H, I, E, K, True)
    s["layer"] = [torch.from_numpy(np.ascontiguousarray(a)).cuda()
                  for a in (lw.experts, lw.scales, lw.router)]
    eng.set_layer_packed(0, *s["layer"])
    return s


@pytest.mark.parametrize("mx", [False, True])
def test_block_of_operators(eng, mx):
    """Each step against the 64-bit form of the same step's inputs."""
    s = block_state(eng, mx)
    r = moe_block(eng, s)
    eng.sync_status()
    o, tok = r["off"].tolist(), r["tok"].long()
    assert o[-1] == s["T"] * s["K"]
    wgu, wd = s["wgu"].double(), s["wd"].double()
    xin, act = r["h"][tok].double(), r["act"].double()
    if mx:
        wgu = mx_ref(s["wgu"].reshape(-1, s["H"]))[2].view(wgu.shape).cuda()
        wd = mx_ref(s["wd"].reshape(-1, s["I"]))[2].view(wd.shape).cuda()
        xin, act = mx_ref(xin)[2].cuda(), mx_ref(act)[2].cuda()
    for e in range(s["E"]):
        a, b = o[e], o[e + 1]
        for got, p, q in ((r["gu"], xin, wgu), (r["y"], act, wd)):
            ref, mag = p[a:b] @ q[e].T, p[a:b].abs() @ q[e].abs().T
            assert ((got[a:b].double() - ref).abs() <= 2 * U * p.shape[1] * mag).all()
    i = dict(x=s["x"], y=r["out"], w_pre=s["g1"], w_post=s["g2"], gate=None)
    rx, rh, mxx, mh = norm_ref(i, True, 1.0, 1e-5)
    assert ((r["x1"].double() - rx).abs() <= 65 * U * mxx).all()
    assert ((r["h1"].double() - rh).abs() <= 600 * U * mh + half_step(BF) * rh.abs()).all()


def test_training_step_in_a_graph(eng):
    """Forward and backward of a product and a norm captured together, and
    replayed on new inputs in the same buffers; another eager run of the same
    calls lives meanwhile."""
    sizes, n, k = [30, 0, 77, 1], 72, 64
    off, R = offsets(sizes)
    buf = dict(x=whole((R, k), BF, 1), w=whole((4, n, k), BF, 2), d=whole((R, n), BF, 3))
    res = dict(out=torch.empty(R, n, device="cuda"), dx=torch.empty(R, k, device="cuda"),
               dw=torch.empty(4, n, k, device="cuda"), dn=torch.empty(R, n, device="cuda"),
               dg=torch.empty(n, device="cuda"))
    gain = torch.rand(n, device="cuda")

    def step(stream):
        eng.grouped_mm(buf["x"], buf["w"], off, res["out"], stream=stream)
        eng.block_norm_backward(None, res["out"], res["out"], gain, res["dn"], res["dg"],
                                stream=stream)
        eng.grouped_mm_dgrad(buf["d"], buf["w"], off, res["dx"], stream=stream)
        eng.grouped_mm_wgrad(buf["d"], buf["x"], off, res["dw"], stream=stream)

    step(torch.cuda.current_stream())
    eager = {a: v.clone() for a, v in res.items()}
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(torch.cuda.current_stream())
    for v in res.values():
        v.zero_()
    graph.replay()
    assert all(torch.equal(res[a], eager[a]) for a in res)
    for a, seed in (("x", 4), ("w", 5), ("d", 6)):
        buf[a].copy_(whole(tuple(buf[a].shape), BF, seed))
    graph.replay()
    got = {a: v.clone() for a, v in res.items()}
    step(torch.cuda.current_stream())
    assert all(torch.equal(res[a], got[a]) for a in res)


def test_two_graphs_at_once(eng):
    """Two captured backward passes and products replayed side by side on two
    streams: each has its own workspace, so both keep their bits."""
    T, H, n = 700, 512, 136
    off, _ = offsets([300, 0, 395, 5])
    jobs = []
    for j in range(2):
        i = norm_inputs(T, H, F32, F32, 70 + j)
        d = dict(i=i, x=whole((T, H), BF, 80 + j), w=whole((4, n, H), BF, 90 + j),
                 dx=torch.empty(T, H, device="cuda"), dg=torch.empty(H, device="cuda"),
                 out=torch.empty(T, n, device="cuda"))

        def step(d=d):
            s = torch.cuda.current_stream()
            eng.block_norm_backward(d["i"]["x"], d["i"]["y"], d["i"]["x"], d["i"]["w_pre"],
                                    d["dx"], d["dg"], stream=s)
            eng.grouped_mm(d["x"], d["w"], off, d["out"], stream=s)

        step()
        d["ref"] = [d[k].clone() for k in ("dx", "dg", "out")]
        d["graph"], d["stream"] = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(d["graph"]):
            step()
        jobs.append(d)
    torch.cuda.synchronize()
    for _ in range(5):
        for d in jobs:
            for k in ("dx", "dg", "out"):
                d[k].zero_()
        torch.cuda.synchronize()
        for d in jobs:
            with torch.cuda.stream(d["stream"]):
                for _ in range(3):
                    d["graph"].replay()
        torch.cuda.synchronize()
        for d in jobs:
            assert all(torch.equal(d[k], r) for k, r in zip(("dx", "dg", "out"), d["ref"]))


def test_two_streams_at_once(eng):
    """The same calls on two streams at the same time, without shared state."""
    streams = [torch.cuda.Stream(), torch.cuda.default_stream()]
    T, H, n = 600, 256, 264
    off, _ = offsets([200, 0, 395, 5])
    ins = [dict(x=whole((T, H), BF, 30 + j), w=whole((4, n, H), BF, 40 + j)) for j in range(2)]
    nrm = [norm_inputs(T, H, F32, F32, 50 + j) for j in range(2)]
    outs = [[dict(o=torch.empty(T, n, device="cuda"), dw=torch.empty(H, device="cuda"),
                  dx=torch.empty(T, H, device="cuda")) for _ in range(2)] for _ in range(2)]
    torch.cuda.synchronize()
    for rep in range(2):  # 0: side by side, 1: one after the other
        for _ in range(5):
            for j, st in enumerate(streams):
                eng.grouped_mm(ins[j]["x"], ins[j]["w"], off, outs[rep][j]["o"], stream=st)
                eng.block_norm_backward(nrm[j]["x"], nrm[j]["y"], nrm[j]["x"], nrm[j]["w_pre"],
                                        outs[rep][j]["dx"], outs[rep][j]["dw"], stream=st)
                if rep:
                    torch.cuda.synchronize()
    torch.cuda.synchronize()
    for j in range(2):
        for key in ("o", "dw", "dx"):
            assert torch.equal(outs[0][j][key], outs[1][j][key])


def test_default_stream_is_torchs(eng):
    """torch's default stream, whose handle is 0, orders a call behind the work
    that makes its inputs and before the work that reads its result."""
    off, _ = offsets([100, 156])
    w = whole((2, 64, 512), BF, 1)
    with torch.cuda.stream(torch.cuda.default_stream()):
        torch.cuda.synchronize()
        a = torch.ones(4096, 4096, device="cuda")
        for _ in range(4):  # some milliseconds of work in front
            a = a @ a / 4096
        x = (a[:256, :512] * 2).to(BF)
        out = torch.zeros(256, 64, device="cuda")
        eng.grouped_mm(x, w, off, out, stream=torch.cuda.current_stream())
        got = out + 0
        x.zero_()
        torch.cuda.synchronize()
    two = torch.full((256, 512), 2.0, dtype=torch.float64, device="cuda")
    ref = torch.cat((two[:100] @ w[0].double().T, two[100:] @ w[1].double().T))
    assert torch.equal(got, ref.float())


def test_handle_stream_and_profile(eng):
    """stream=None runs on the handle's stream; the calls appear in its profile."""
    e = M.MoeLayerEngine(M.MoeConfig(64, 32, 8, 2, True, 4, 1))
    x, w = whole((10, 32), HF, 1), whole((2, 8, 32), HF, 2)
    off, _ = offsets([4, 6])
    out = torch.empty(10, 8, device="cuda")
    dg = torch.empty(32, device="cuda")
    torch.cuda.synchronize()
    e.profile(True)
    e.grouped_mm(x, w, off, out)
    assert e.last_launch_count() == 1
    e.block_norm_backward(None, x, x, None, torch.empty_like(x), dg)
    e.sync_status()
    assert set(e.profile_read()) >= {"grouped_mm", "block_norm_backward"}
    assert torch.equal(out[:4], (x[:4].double() @ w[0].double().T).float())
    e.close()


def test_refusals(eng):
    """Each refused call launches nothing, names its reason and leaves the
    engine usable."""
    x, w, out = whole((10, 32), BF, 1), whole((2, 8, 32), BF, 2), torch.zeros(10, 8, device="cuda")
    off, _ = offsets([4, 6])
    bad = [
        lambda: eng.grouped_mm(x.cpu(), w, off, out),
        lambda: eng.grouped_mm(x.half(), w, off, out),
        lambda: eng.grouped_mm(x.float(), w.float(), off, out),
        lambda: eng.grouped_mm(x, w, off, out.half()),
        lambda: eng.grouped_mm(x, w, off.long(), out),
        lambda: eng.grouped_mm(x, w, off[:2], out),
        lambda: eng.grouped_mm(x[:, :24], w, off, out),
        lambda: eng.grouped_mm(x[:9], w, off, out),
        lambda: eng.grouped_mm(x, w[0], off, out),
        lambda: eng.grouped_mm(x, w, off.repeat_interleave(2)[::2], out),
        lambda: eng.grouped_mm(x, w.transpose(1, 2), off, out),
        lambda: eng.grouped_mm(x.t().contiguous().t(), w, off, out),
        lambda: eng.grouped_mm(x[:1].expand(10, 32), w, off, out),
        lambda: eng.grouped_mm(x, w[:1].expand(2, 8, 32), off, out),
        lambda: eng.grouped_mm(x, torch.zeros(257, 8, 32, device="cuda", dtype=BF),
                               torch.zeros(258, dtype=torch.int32, device="cuda"), out),
        lambda: eng.grouped_mm_wgrad(out, x, off, torch.zeros(2, 8, 32, device="cuda")),
        lambda: eng.mxfp4_quantize(x.int(), *eng.mxfp4_empty(10, 32)),
        lambda: eng.mxfp4_quantize(x, *eng.mxfp4_empty(9, 32)),
        lambda: eng.mxfp4_quantize(x, *eng.mxfp4_empty(10, 64)),
        lambda: eng.mxfp4_quantize(x, *eng.mxfp4_empty(10, 32), rows=off),
        lambda: eng.mxfp4_dequantize(*eng.mxfp4_empty(10, 32), out[:9]),
        lambda: eng.grouped_mm_mxfp4(*eng.mxfp4_empty(10, 32), *eng.mxfp4_empty(15, 32), off, 32,
                                     out),
        lambda: eng.block_norm(x, x, x.half(), None),
        lambda: eng.block_norm(x, x, x, w),
        lambda: eng.block_norm(x, None, None),
        lambda: eng.block_norm(x, x, x, None, eps=-1.0),
        lambda: eng.block_norm(x, x, x, None, y=x, gate=torch.ones(9, device="cuda")),
        lambda: eng.block_norm(torch.zeros(1, 16400, device="cuda"), None,
                               torch.zeros(1, 16400, device="cuda")),
        lambda: eng.block_norm_backward(None, None, x, None, x),
        lambda: eng.block_norm_backward(x, x, x, None, x, y=x),
        lambda: eng.block_norm_backward(x, x, x, None, x, dgate=torch.ones(10, device="cuda")),
        lambda: eng.block_norm_backward(x, x, x, None, x, y=x, dy=x, post_norm=False,
                                        dw_post=torch.zeros(32, device="cuda")),
    ]
    for j, call in enumerate(bad):
        with pytest.raises(M.MoeError) as err:
            call()
        assert err.value.status == _lib.MOE_ERR_INVALID, j
    assert (out == 0).all()
    eng.grouped_mm(x, w, off, out)
    eng.sync_status()
