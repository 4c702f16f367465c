"""4-bit floating-point operators (ops/fp4.py) against 64-bit forms written from their definition."""
import math

import pytest
import torch

from glm53.ops import fp4
from glm53.ops import kernels as K

pytestmark = pytest.mark.gpu
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32
FMTS = list(fp4.FORMATS)
MAGS = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


# ---------------------------------------------------------------------------------------------- 64-bit definition
def ceil_pow2(t):
    f, e = torch.frexp(t)                      # t = f 2^e, f in [0.5, 1)
    return torch.where(t > 0, torch.ldexp(torch.ones_like(t), torch.where(f == 0.5, e - 1, e)), torch.zeros_like(t))


def e4m3(t):
    """t >= 0 to the nearest e4m3 value (ties to even), in 64 bits."""
    _, e = torch.frexp(t.clamp_min(2.0 ** -6))
    step = torch.ldexp(torch.ones_like(t), e - 4)
    return torch.round(t / step) * step


def scales(x, fmt, bound=None):
    """[R, K / block, 1] element scales of x (64 bits)."""
    b = x.view(x.shape[0], -1, 16 if fmt == "nvfp4" else 32)
    amax = b.abs().amax(-1, keepdim=True)
    if fmt == "mxfp4":
        return ceil_pow2(amax / 6)
    top = amax.amax(1, keepdim=True) if bound is None else x.new_full((x.shape[0], 1, 1), bound)
    row = ceil_pow2(top / (448 * 6)).clamp_min(2.0 ** -100)
    return e4m3(torch.where(row > 0, amax / torch.where(row > 0, row, 1.0) / 6, 0.0)) * row


def quant(x, fmt, bound=None):
    """Q(x) in 64 bits: the nearest of the eight magnitudes, ties to the even code."""
    x = x.double()
    s = scales(x, fmt, bound)
    b = x.view(x.shape[0], -1, 16 if fmt == "nvfp4" else 32)
    q = torch.where(s > 0, b.abs() / torch.where(s > 0, s, 1.0), 0.0)
    mags = torch.tensor(MAGS, dtype=torch.float64, device=x.device)
    mid = (mags[1:] + mags[:-1]) / 2
    lo = torch.bucketize(q, mid)               # codes with q above the middle below them; a tie stays at the lower code
    lo = lo + ((lo < 7) & (q == mid[lo.clamp_max(6)]) & (lo % 2 == 1)).long()
    return (torch.sign(b) * mags[lo] * s).view(x.shape)


def acts(rows, k, seed=0, dtype=BF):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, k, generator=g, device="cuda")
    x *= 1 + 7 * (torch.rand(k, generator=g, device="cuda") < 0.05)
    return x.to(dtype)


def weight(n, k, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    w = torch.randn(n, k, generator=g, device="cuda") * k ** -0.5
    return (w * (0.5 + torch.rand(n, 1, generator=g, device="cuda"))).to(BF)


def sums_tol(a, w):
    """Bound of the fp32 sums: every addition of a K-term sum off by at most 2^-23 of the sum of magnitudes (a tensor core
    may truncate), twice K additions (products of a block, blocks)."""
    return 2 * a.shape[1] * 2.0 ** -23 * (a.abs() @ w.abs().t())


def act_tol(x, w, fmt):
    """Bound of what the expansion of 16-bit activations leaves out (x, w in 64 bits): a block's elements are rounded to
    multiples of 2^(e-21), 2^e the binade of its largest, so by at most 2^-22 of that; in nvfp4 a block more than 2^17
    below the row's largest is rounded as one at 2^-17 (2^-39 of the row's largest)."""
    blk = 16 if fmt == "nvfp4" else 32
    amax = x.abs().view(x.shape[0], -1, blk).amax(-1)
    wsum = w.abs().view(w.shape[0], -1, blk).sum(-1)
    if fmt == "nvfp4":
        amax = torch.maximum(amax, 2.0 ** -17 * amax.amax(1, keepdim=True))
    return 2.0 ** -22 * amax @ wsum.t()


def half(dtype):
    return torch.finfo(dtype).eps / 2


# ------------------------------------------------------------------------------------------------------ quantise
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("rows,k", [(1, 32), (3, 96), (128, 256), (129, 288), (5, 1536), (300, 4096), (7, 12288),
                                    (2, 16384), (3, 17408)])
@pytest.mark.parametrize("dtype", [BF, F16])
def test_quantize_reads_back_the_definition(fmt, rows, k, dtype):
    x = acts(rows, k, rows + k, dtype)
    m = fp4.quantize4(x, fmt)
    assert (m.rows, m.k, m.fmt) == (rows, k, fmt)
    ref = quant(x, fmt)
    for out in (F32, BF):
        assert torch.equal(fp4.dequantize4(m, out).double(), ref)


def test_quantize_nv_takes_any_multiple_of_16():
    for k in (16, 48, 272, 1040):
        x = acts(9, k, k)
        assert torch.equal(fp4.dequantize4(fp4.quantize4(x, "nvfp4"), F32).double(), quant(x, "nvfp4"))


@pytest.mark.parametrize("fmt", FMTS)
def test_quantize_ties_zeros_and_far_magnitudes(fmt):
    # every multiple of 1/8 up to 8 times powers of two: all the ties between codes and between scales
    base = torch.arange(-64, 64, device="cuda").float() / 8
    x = torch.stack([base * s for s in (1.0, 0.75, 1.25, 3.0, 7.0, 2.0 ** -20, 2.0 ** 30, 2.0 ** -90, 2.0 ** 110)])
    x = torch.cat([x, torch.zeros(1, 128, device="cuda")]).to(BF)
    x[3, :64] = 0
    x[4, 5:] *= 2.0 ** -14
    assert torch.equal(fp4.dequantize4(fp4.quantize4(x, fmt), F32).double(), quant(x, fmt))
    h = (x[:5].float()).to(F16)
    assert torch.equal(fp4.dequantize4(fp4.quantize4(h, fmt), F32).double(), quant(h, fmt))


@pytest.mark.parametrize("fmt", FMTS)
def test_quantize_infinity_and_nan(fmt):
    x = acts(6, 128, 3)
    x[1, 40] = math.inf
    x[2, 100] = math.nan
    x[4, 0] = -math.inf
    y = fp4.dequantize4(fp4.quantize4(x, fmt), F32)
    ref = quant(x.where(torch.isfinite(x), 0), fmt)
    bad = torch.zeros(6, 128, dtype=torch.bool, device="cuda")
    for r, c in ((1, 40), (2, 100), (4, 0)):
        if fmt == "nvfp4":
            bad[r] = True
        else:
            bad[r, c // 32 * 32:c // 32 * 32 + 32] = True
    assert torch.equal(torch.isnan(y), bad)
    assert torch.equal(y[~bad].double(), ref[~bad])


@pytest.mark.parametrize("fmt", FMTS)
def test_quantize_strided_rows_and_outputs(fmt):
    big = acts(20, 1000, 5)
    for off in (0, 8, 1, 3):                   # 16-byte aligned rows or not
        x = big[::2, off:off + 320]
        m = fp4.quantize4(x, fmt)
        ref = quant(x, fmt)
        for dt in (BF, F32, F16):
            out = torch.full((12, 337), 7.0, dtype=dt, device="cuda")
            fp4.dequantize4(m, out=out[1:11, off:off + 320])
            assert torch.equal(out[1:11, off:off + 320].double(), ref.to(dt).double())
            out[1:11, off:off + 320] = 7.0
            assert (out == 7.0).all()


# ------------------------------------------------------------------------------------------- linear, few rows
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("n,k", [(1, 32), (64, 96), (127, 256), (129, 544), (1000, 1536), (4096, 2048), (640, 12288),
                                 (24576, 512), (384, 17408)])
@pytest.mark.parametrize("m", [1, 7, 8, 9, 16])
def test_linear_few_rows(fmt, n, k, m):
    x, w = acts(m, k, m), weight(n, k, n)
    w4 = fp4.quantize4(w, fmt)
    wq = quant(w, fmt)
    ref = x.double() @ wq.t()
    tol = sums_tol(x.double(), wq) + act_tol(x.double(), wq, fmt)
    y = fp4.linear4(x, w4, torch.empty(m, n, dtype=F32, device="cuda"), K.GEMV_F32)
    assert ((y.double() - ref).abs() <= tol).all()
    yb = fp4.linear4(x, w4, torch.empty(m, n, dtype=BF, device="cuda"))
    assert torch.equal(yb, y.to(BF))
    acc = torch.randn(m, n, device="cuda")
    ya = fp4.linear4(x, w4, acc.clone(), K.GEMV_F32_ACC)
    assert torch.equal(ya, acc + y)
    assert torch.equal(fp4.linear4(x, w4, torch.empty_like(y), K.GEMV_F32, act4=True), y)     # 16 rows: exact


@pytest.mark.parametrize("k", [16, 48, 80, 272])
def test_linear_nv_takes_any_multiple_of_16(k):
    w = weight(70, k, k)
    w4, wq = fp4.quantize4(w, "nvfp4"), quant(w, "nvfp4")
    for m, act4 in ((1, False), (20, False), (300, False), (20, True), (300, True)):
        x = acts(m, k, m)
        a = quant(x, "nvfp4") if act4 else x.double()
        y = fp4.linear4(x, w4, torch.empty(m, 70, dtype=F32, device="cuda"), K.GEMV_F32, act4=act4)
        assert ((y.double() - a @ wq.t()).abs() <= sums_tol(a, wq) + act_tol(a, wq, "nvfp4")).all(), (m, act4)


@pytest.mark.parametrize("fmt", FMTS)
def test_linear_few_rows_magnitudes_and_views(fmt):
    n, k = 200, 576
    wq_src = weight(n, k, 2)
    wq_src[3] = 0
    wq_src[5] *= 2.0 ** 40
    wq_src[6] *= 2.0 ** -40
    w4, wq = fp4.quantize4(wq_src, fmt), quant(wq_src, fmt)
    big = acts(30, 700, 4)
    big[2] *= 2.0 ** 90
    big[4] *= 2.0 ** -60
    big[6] = 0
    for off in (0, 1, 8):
        x = big[0:22:2, off:off + k]
        ref = x.double() @ wq.t()
        tol = sums_tol(x.double(), wq) + act_tol(x.double(), wq, fmt)
        out = torch.full((13, 301), 5.0, dtype=F32, device="cuda")
        fp4.linear4(x, w4, out[1:12, 3:203], K.GEMV_F32)
        y = out[1:12, 3:203].double()
        # row 1 times weight row 5 is of the order 2^90 * 8 * 2^40: where the sum of magnitudes passes fp32's largest
        # (2^128), a partial sum can, and the result is then an infinity or, with both signs, NaN
        over = x.double().abs() @ wq.abs().t() >= 2.0 ** 128
        assert over.sum() == 1
        assert ((y - ref).abs() <= tol)[~over].all()
        out[1:12, 3:203] = 5.0
        assert (out == 5.0).all()
    x = acts(4, k, 9)
    x[1, 7], x[2, 9] = math.inf, math.nan
    y = fp4.linear4(x, w4, torch.empty(4, n, dtype=F32, device="cuda"), K.GEMV_F32)
    assert torch.isfinite(y[0]).all() and torch.isfinite(y[3]).all()
    assert not torch.isfinite(y[1]).any() and torch.isnan(y[2]).all()


@pytest.mark.parametrize("fmt", FMTS)
def test_linear_reads_nan_weights_as_nan(fmt):
    w = weight(256, 512, 3)
    w[10, 20] = math.nan
    w4 = fp4.quantize4(w, fmt)
    for m, act4 in ((3, False), (40, True), (70, False), (150, True), (270, False)):
        y = fp4.linear4(acts(m, 512, m), w4, torch.empty(m, 256, dtype=F32, device="cuda"), K.GEMV_F32, act4=act4)
        bad = torch.zeros(256, dtype=torch.bool, device="cuda")
        bad[10] = True
        assert torch.equal(torch.isnan(y).any(0), bad) and torch.isnan(y[:, 10]).all()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("m", [17, 40, 63, 64, 200, 256, 257, 300])
def test_linear_exact_activations_above_16_rows(fmt, m):
    n, k = 300, 800
    x, w = acts(m, k, m), weight(n, k, 5)
    w4, wq = fp4.quantize4(w, fmt), quant(w, fmt)
    ref = x.double() @ wq.t()
    tol = sums_tol(x.double(), wq) + act_tol(x.double(), wq, fmt)
    y = fp4.linear4(x, w4, torch.zeros(m, n, dtype=F32, device="cuda"), K.GEMV_F32)
    assert ((y.double() - ref).abs() <= tol).all()
    y2 = fp4.linear4(x, w4, y.clone(), K.GEMV_F32_ACC)
    assert ((y2.double() - 2 * ref).abs() <= 2 * tol + half(F32) * 2 * ref.abs()).all()
    odd = acts(m, k + 1, m)[:, 1:]
    ref = odd.double() @ wq.t()
    y = fp4.linear4(odd, w4, torch.zeros(m, n, dtype=BF, device="cuda"))
    tol = sums_tol(odd.double(), wq) + act_tol(odd.double(), wq, fmt)
    assert ((y.double() - ref).abs() <= tol + half(BF) * (ref.abs() + tol)).all()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("m,n,k", [(96, 70, 544), (97, 1, 32), (97, 129, 4128), (112, 257, 96), (256, 128, 2080), (257, 385, 544),
                                   (300, 640, 12288), (512, 200, 1024), (513, 130, 1056), (1025, 300, 320), (1100, 20000, 96),
                                   (2500, 1000, 160)])
def test_linear_exact_activations_many_rows(fmt, m, n, k):
    """Both sides of the row counts and widths where the product changes its shape: groups of rows, one or two mma, a split
    of K over a cluster, an odd number of 128-row blocks."""
    x, w = acts(m, k, m), weight(n, k, n)
    w4, wq = fp4.quantize4(w, fmt), quant(w, fmt)
    ref = x.double() @ wq.t()
    tol = sums_tol(x.double(), wq) + act_tol(x.double(), wq, fmt)
    out = torch.full((m + 2, n + 5), 5.0, dtype=F32, device="cuda")
    y = fp4.linear4(x, w4, out[1:m + 1, 2:n + 2], K.GEMV_F32)
    assert ((y.double() - ref).abs() <= tol).all()
    got = y.clone()
    out[1:m + 1, 2:n + 2] = 5.0
    assert (out == 5.0).all()
    assert torch.equal(fp4.linear4(x, w4, torch.empty(m, n, dtype=BF, device="cuda")), got.to(BF))
    acc = torch.randn(m, n, device="cuda")
    assert torch.equal(fp4.linear4(x, w4, acc.clone(), K.GEMV_F32_ACC), acc + got)
    fp4.check_errors()


@pytest.mark.parametrize("fmt", FMTS)
def test_linear_many_rows_magnitudes_and_views(fmt):
    n, k, m = 200, 576, 140
    src = weight(n, k, 2)
    src[3] = 0
    src[5] *= 2.0 ** 40
    src[6] *= 2.0 ** -40
    src[7] *= 2.0 ** -100
    src[8] *= 2.0 ** 120
    w4, wq = fp4.quantize4(src, fmt), quant(src, fmt)
    big = acts(2 * m, 700, 4)
    big[4] *= 2.0 ** -60
    big[6] = 0
    for off in (0, 1, 8):
        x = big[::2, off:off + k]
        ref = x.double() @ wq.t()
        tol = sums_tol(x.double(), wq) + act_tol(x.double(), wq, fmt)
        # products are summed 2^-8 lower in nvfp4: one below 2^-126 may lose what lies under 2^-149
        tol += k * 2.0 ** -141
        y = fp4.linear4(x, w4, torch.empty(m, n, dtype=F32, device="cuda"), K.GEMV_F32)
        assert ((y.double() - ref).abs() <= tol).all()
    one = acts(1, k, 6).expand(m, k)                    # the same row again and again
    y = fp4.linear4(one, w4, torch.empty(m, n, dtype=F32, device="cuda"), K.GEMV_F32)
    assert torch.equal(y, y[:1].expand(m, n))
    assert torch.equal(y, fp4.linear4(one.contiguous(), w4, torch.empty_like(y), K.GEMV_F32))
    x = acts(m, k, 9)
    x[1, 7], x[130, 9] = math.inf, math.nan
    y = fp4.linear4(x, w4, torch.empty(m, n, dtype=F32, device="cuda"), K.GEMV_F32)
    fine = torch.ones(m, dtype=torch.bool, device="cuda")
    fine[1] = fine[130] = False
    assert torch.isfinite(y[fine]).all()
    assert not torch.isfinite(y[1]).any() and torch.isnan(y[130]).all()


def test_linear_takes_every_scale():
    """Imported images: every code under every finite scale, through each product that keeps activations exact."""
    for fmt in FMTS:
        nv = fmt == "nvfp4"
        n, k = 256, 256
        src = fp4.quantize4(weight(n, k, 1), fmt)
        codes = torch.arange(256, device="cuda", dtype=torch.uint8).repeat(src.codes.numel() // 256)
        sc = torch.arange(src.scales.numel(), device="cuda") % 256
        # finite, and with a sum of products inside fp32
        sc = torch.where((sc & 127) == 127, 1, sc & 127) if nv else sc.clamp(0, 240)
        m4 = fp4.Matrix4.from_parts(codes, sc.to(torch.uint8), torch.ones_like(src.row_scale) if nv else None, n, k, fmt)
        w = fp4.dequantize4(m4, F32).double()
        for m in (1, 40, 100, 300):
            x = torch.ones(m, k, dtype=BF, device="cuda")
            x[:, ::3] = -0.5
            y = fp4.linear4(x, m4, torch.empty(m, n, dtype=F32, device="cuda"), K.GEMV_F32)
            ref, tol = x.double() @ w.t(), sums_tol(x.double(), w) + k * 2.0 ** -126
            assert ((y.double() - ref).abs() <= tol).all(), (fmt, m)


# ------------------------------------------------------------------------------------- linear, 4-bit activations
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("m,n,k", [(17, 8, 32), (64, 128, 64), (100, 100, 96), (65, 20000, 96), (128, 200, 4128), (127, 4096, 96), (128, 256, 256), (129, 257, 288),
                                   (300, 1000, 1536), (70, 130, 4128), (1000, 520, 320), (2500, 4100, 544),
                                   (4096, 2048, 1024), (2433, 2817, 96), (129, 19100, 288)])
def test_linear_4bit_activations(fmt, m, n, k):
    x, w = acts(m, k, m), weight(n, k, n)
    w4 = fp4.quantize4(w, fmt)
    xq, wq = quant(x, fmt), quant(w, fmt)
    ref, tol = xq @ wq.t(), sums_tol(xq, wq)
    y = fp4.linear4(x, w4, torch.empty(m, n, dtype=F32, device="cuda"), K.GEMV_F32, act4=True)
    assert ((y.double() - ref).abs() <= tol).all()
    yb = fp4.linear4(x, w4, torch.empty(m, n, dtype=BF, device="cuda"), act4=True)
    assert torch.equal(yb, y.to(BF))
    ya = fp4.linear4(x, w4, y.clone(), K.GEMV_F32_ACC, act4=True)
    assert torch.equal(ya, y + y)
    fp4.check_errors()


@pytest.mark.parametrize("fmt", FMTS)
def test_linear_4bit_activations_views_and_odd_values(fmt):
    n, k, m = 333, 416, 150
    w = weight(n, k, 8)
    w4, wq = fp4.quantize4(w, fmt), quant(w, fmt)
    big = acts(2 * m, 600, 6)
    big[4] *= 2.0 ** 60
    big[6] = 0
    x = big[::2, 5:5 + k]
    out = torch.full((m + 2, 401), 5.0, dtype=BF, device="cuda")
    fp4.linear4(x, w4, out[1:m + 1, 3:3 + n], act4=True)
    xq = quant(x, fmt)
    ref, tol = xq @ wq.t(), sums_tol(xq, wq)
    assert ((out[1:m + 1, 3:3 + n].double() - ref).abs() <= tol + half(BF) * (ref.abs() + tol)).all()
    out[1:m + 1, 3:3 + n] = 5.0
    assert (out == 5.0).all()
    x = x.clone()
    x[3, 100] = math.inf
    y = fp4.linear4(x, w4, torch.empty(m, n, dtype=F32, device="cuda"), K.GEMV_F32, act4=True)
    assert torch.isnan(y[3]).all() and torch.isfinite(torch.cat([y[:3], y[4:]])).all()


# --------------------------------------------------------------------------------------------------- gated block
def gated(x, gate, up, limit):
    g, u = (x @ gate.t()).clamp(max=limit), (x @ up.t()).clamp(-limit, limit)
    return g * torch.sigmoid(g) * u


def h_slack(h, err, fmt, bound):
    """How far each quantised activation may be off when the activation is off by `err`: one code step where h lies
    within err of a border between codes, and the change of scale where the block's maximum lies so near a border
    between scales."""
    blk = 16 if fmt == "nvfp4" else 32
    s = scales(h, fmt, bound)
    b, e = h.view(h.shape[0], -1, blk), err.view(h.shape[0], -1, blk)
    q = torch.where(s > 0, b.abs() / torch.where(s > 0, s, 1.0), 0.0)
    mid = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=torch.float64, device=h.device)
    near = torch.zeros_like(q, dtype=torch.bool)
    for m in mid:
        near |= (q - m).abs() * s <= 2 * e
    step = torch.where(near, 2.0 * s, 0.0)
    amax, eb = b.abs().amax(-1, keepdim=True), e.amax(-1, keepdim=True)

    def scale_of(a):
        if fmt == "mxfp4":
            return ceil_pow2(a / 6)
        row = ceil_pow2(torch.full((), bound / (448 * 6), dtype=torch.float64, device=h.device))
        return e4m3(a / row / 6) * row
    moved = scale_of((amax - 2 * eb).clamp_min(0)) != scale_of(amax + 2 * eb)
    return torch.where(moved, 2 * b.abs() + 2 * s, step).view(h.shape)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("m,k,width,n", [(1, 4096, 2048, 512), (8, 512, 96, 40), (16, 288, 1536, 200), (5, 64, 32, 1),
                                         (33, 256, 160, 128), (64, 512, 96, 40), (150, 256, 1536, 200), (257, 512, 96, 40),
                                         (300, 256, 1536, 200), (97, 2080, 96, 40), (520, 1024, 160, 300),
                                         (1040, 256, 2048, 130)])
def test_mlp_exact_activations(fmt, m, k, width, n):
    limit = 2.0
    x, gate, up, down = acts(m, k, m), weight(width, k, 1), weight(width, k, 2), weight(n, width, 3)
    mlp = fp4.pack_mlp4(gate, up, down, fmt)
    gq, uq, dq = quant(gate, fmt), quant(up, fmt), quant(down, fmt)
    xd = x.double()
    h = gated(xd, gq, uq, limit)
    # gate and up sums, then the activation (derivative at most 1.1 limit in either), exp and the division: 2^-20
    eg = sums_tol(xd, gq) + act_tol(xd, gq, fmt)
    eu = sums_tol(xd, uq) + act_tol(xd, uq, fmt)
    eh = 1.1 * limit * (eg + eu) + 2.0 ** -20 * h.abs()
    eh = eh + half(BF) * (h.abs() + eh)
    ref = h @ dq.t()
    tol = eh @ dq.abs().t() + sums_tol(h.abs() + eh, dq) + act_tol(h.abs() + eh, dq, fmt)
    y = fp4.mlp4(x, mlp, torch.empty(m, n, dtype=F32, device="cuda"), limit)
    assert ((y.double() - ref).abs() <= tol).all()
    yb = fp4.mlp4(x, mlp, torch.empty(m, n, dtype=BF, device="cuda"), limit, K.GEMV_BF16)
    assert torch.equal(yb, y.to(BF))
    acc = torch.randn(m, n, device="cuda")
    assert torch.equal(fp4.mlp4(x, mlp, acc.clone(), limit, K.GEMV_F32_ACC), acc + y)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("m,k,width,n", [(17, 256, 32, 8), (40, 512, 96, 40), (130, 288, 160, 200), (257, 1024, 1536, 300),
                                         (2500, 320, 4128, 264), (2433, 96, 1376, 64)])
def test_mlp_4bit_activations(fmt, m, k, width, n):
    limit = 2.0
    x, gate, up, down = acts(m, k, m), weight(width, k, 1), weight(width, k, 2), weight(n, width, 3)
    mlp = fp4.pack_mlp4(gate, up, down, fmt)
    xq, gq, uq, dq = quant(x, fmt), quant(gate, fmt), quant(up, fmt), quant(down, fmt)
    h = gated(xq, gq, uq, limit)
    eh = 1.1 * limit * (sums_tol(xq, gq) + sums_tol(xq, uq)) + 2.0 ** -20 * h.abs()
    hq = quant(h, fmt, limit * limit)
    slack = h_slack(h, eh, fmt, limit * limit)
    ref = hq @ dq.t()
    tol = slack @ dq.abs().t() + sums_tol(hq.abs() + slack, dq)
    y = fp4.mlp4(x, mlp, torch.empty(m, n, dtype=F32, device="cuda"), limit, act4=True)
    assert ((y.double() - ref).abs() <= tol).all()
    # and close in the mean: the sums are off by about 2^-22, so one activation in 2^18 or fewer changes its code, each
    # by at most its own size
    assert (y.double() - ref).norm() <= 0.01 * ref.norm()
    yb = fp4.mlp4(x, mlp, torch.empty(m, n, dtype=BF, device="cuda"), limit, K.GEMV_BF16, act4=True)
    assert torch.equal(yb, y.to(BF))
    fp4.check_errors()


@pytest.mark.parametrize("fmt", FMTS)
def test_mlp_keeps_a_nan_row(fmt):
    mlp = fp4.pack_mlp4(weight(96, 256, 1), weight(96, 256, 2), weight(64, 96, 3), fmt)
    for m, act4 in ((4, False), (40, True), (140, True), (40, False), (80, False), (270, False)):
        x = acts(m, 256, m)
        x[2, 17] = math.nan
        y = fp4.mlp4(x, mlp, torch.empty(m, 64, dtype=F32, device="cuda"), 10.0, act4=act4)
        assert torch.isnan(y[2]).all() and torch.isfinite(torch.cat([y[:2], y[3:]])).all(), (m, act4)


def test_mlp_without_a_clamp():
    mlp = fp4.pack_mlp4(weight(64, 256, 1), weight(64, 256, 2), weight(64, 64, 3), "mxfp4")
    x = acts(20, 256, 3)
    wide = fp4.mlp4(x, mlp, torch.empty(20, 64, dtype=F32, device="cuda"), 1e4, act4=True)
    assert torch.equal(fp4.mlp4(x, mlp, torch.empty_like(wide), math.inf, act4=True), wide)
    assert torch.equal(fp4.mlp4(x[:9], mlp, torch.empty_like(wide[:9]), math.inf),
                       fp4.mlp4(x[:9], mlp, torch.empty_like(wide[:9]), 1e4))


# ---------------------------------------------------------------------------------------- graphs, streams, reuse
@pytest.mark.parametrize("m,act4", [(3, False), (12, False), (30, False), (90, False), (90, True),
                                    (200, True), (270, False), (600, False)])
def test_graph_replay_and_streams(m, act4):
    """Quantise, project and run the block as one captured graph, replayed on new inputs, beside eager calls on another
    stream: all the same bits."""
    k, width, n = 512, 320, 264
    w4 = fp4.quantize4(weight(k, k, 4), "nvfp4")
    mlp = fp4.pack_mlp4(weight(width, k, 1), weight(width, k, 2), weight(n, width, 3), "mxfp4")
    x = acts(m, k, 1)

    def step(x):
        t = fp4.linear4(x, w4, torch.empty(m, k, dtype=BF, device="cuda"), act4=act4)
        t = fp4.dequantize4(fp4.quantize4(t, "mxfp4"))
        return fp4.mlp4(t, mlp, torch.empty(m, n, dtype=F32, device="cuda"), 10.0, act4=act4)

    inputs = [acts(m, k, s) for s in (2, 3)]
    want = [step(i) for i in inputs]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(x)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(x)
    side = []
    for i, w in zip(inputs, want):
        x.copy_(i)
        s.wait_stream(torch.cuda.current_stream())
        g.replay()
        with torch.cuda.stream(s):
            side += [step(i) for _ in range(3)]
        torch.cuda.synchronize()
        assert torch.equal(out, w)
        assert all(torch.equal(t, w) for t in side[-3:])
    fp4.check_errors()


def test_weights_written_just_before_their_product():
    """The product may be launched right behind the quantisation of its weights (programmatic launches included)."""
    x = acts(4, 2048, 1)
    for i in range(20):
        w = weight(2048, 2048, i)
        fp4.linear4(x, fp4.quantize4(weight(512, 2048, 99)), torch.empty(4, 512, dtype=F32, device="cuda"), K.GEMV_F32)
        w4 = fp4.quantize4(w, "nvfp4")
        y = fp4.linear4(x, w4, torch.empty(4, 2048, dtype=F32, device="cuda"), K.GEMV_F32)
        torch.cuda.synchronize()
        assert torch.equal(y, fp4.linear4(x, w4, torch.empty_like(y), K.GEMV_F32))


@pytest.mark.parametrize("m,act4", [(3, False), (60, False), (60, True), (150, False), (150, True), (700, False)])
def test_sums_added_call_after_call(m, act4):
    """Products that add into y right behind one another (rows of odd length: two CTAs share sectors of y) see each other's
    sums."""
    n, k = 389, 512
    w4 = fp4.quantize4(weight(n, k, 4), "nvfp4")
    xs = [acts(m, k, s) for s in range(4)]

    def chain(wait):
        y = torch.zeros(m, n, device="cuda")
        for i in range(40):
            fp4.linear4(xs[i % 4], w4, y, K.GEMV_F32_ACC, act4=act4)
            if wait:
                torch.cuda.synchronize()
        return y
    want = chain(True)
    assert all(torch.equal(chain(False), want) for _ in range(5))


def test_first_calls_inside_a_capture():
    """In a fresh process, each product's first launch may be a captured one."""
    import os
    import subprocess
    import sys
    code = """
import torch, sys
sys.path.insert(0, sys.argv[1])
from glm53.ops import fp4, kernels as K
w = fp4.quantize4(torch.randn(256, 512, device='cuda').to(torch.bfloat16))
m = fp4.pack_mlp4(*(torch.randn(64, 512, device='cuda').to(torch.bfloat16) for _ in range(2)),
                  torch.randn(96, 64, device='cuda').to(torch.bfloat16))
xs = [torch.randn(r, 512, device='cuda').to(torch.bfloat16) for r in (1, 12, 30, 300)]
def calls():
    out = []
    for x in xs:
        for act4 in (False, True):
            y = torch.empty(x.shape[0], 256, device='cuda', dtype=torch.float32)
            z = torch.empty(x.shape[0], 96, device='cuda', dtype=torch.float32)
            out += [fp4.linear4(x, w, y, K.GEMV_F32, act4=act4), fp4.mlp4(x, m, z, 10.0, act4=act4),
                    fp4.dequantize4(fp4.quantize4(x, 'mxfp4'))]
    return out
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    got = calls()
g.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(got, calls()))
fp4.check_errors()
print('captured', len(got))
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code, root], capture_output=True, text=True, timeout=300, cwd=root)
    assert r.returncode == 0 and "captured 24" in r.stdout, r.stderr[-2000:]


def test_empty_batch():
    w4 = fp4.quantize4(weight(64, 64, 1))
    mlp = fp4.pack_mlp4(weight(64, 64, 1), weight(64, 64, 2), weight(64, 64, 3))
    x, y = torch.empty(0, 64, dtype=BF, device="cuda"), torch.empty(0, 64, dtype=F32, device="cuda")
    assert fp4.linear4(x, w4, y, K.GEMV_F32).shape == (0, 64) and fp4.mlp4(x, mlp, y, 10.0).shape == (0, 64)


# ------------------------------------------------------------------------------------------------------ refusals
def test_refusals():
    dev = "cuda"
    w4 = fp4.quantize4(weight(64, 96, 1))
    x, y = acts(3, 96, 1), torch.empty(3, 64, dtype=BF, device=dev)
    bad = [
        lambda: fp4.quantize4(torch.zeros(4, 24, dtype=BF, device=dev)),                    # K % 16
        lambda: fp4.quantize4(torch.zeros(4, 48, dtype=BF, device=dev), "mxfp4"),           # K % 32
        lambda: fp4.quantize4(torch.zeros(4, 64, device=dev)),                              # fp32 input
        lambda: fp4.quantize4(torch.zeros(4, 64, dtype=BF)),                                # host
        lambda: fp4.quantize4(torch.zeros(64, 4, dtype=BF, device=dev).t()),                # inner stride
        lambda: fp4.quantize4(torch.zeros(0, 64, dtype=BF, device=dev)),
        lambda: fp4.quantize4(torch.zeros(2, 4, 64, dtype=BF, device=dev)),
        lambda: fp4.dequantize4(w4, out=torch.empty(64, 95, dtype=BF, device=dev)),
        lambda: fp4.dequantize4(w4, out=torch.empty(1, 96, dtype=BF, device=dev).expand(64, 96)),
        lambda: fp4.dequantize4(w4, torch.float64),
        lambda: fp4.linear4(x[:, :64], w4, y),
        lambda: fp4.linear4(x.float(), w4, y),
        lambda: fp4.linear4(x, w4, y, K.GEMV_F32),                                          # bf16 y
        lambda: fp4.linear4(x, w4, y[:, :63]),
        lambda: fp4.linear4(x, w4, y[:2]),
        lambda: fp4.linear4(x, w4, y, K.GEMV_SWIGLU),
        lambda: fp4.linear4(x.cpu(), w4, y),
        lambda: fp4.linear4(x, w4, y.cpu()),
        lambda: fp4.linear4(x, w4, y[:1].expand(3, 64)),
        lambda: fp4.Matrix4.from_parts(w4.codes[:-1], w4.scales, w4.row_scale, 64, 96, "nvfp4"),
        lambda: fp4.Matrix4.from_parts(w4.codes, w4.scales, None, 64, 96, "nvfp4"),
        lambda: fp4.Matrix4.from_parts(w4.codes, w4.scales, w4.row_scale, 129, 96, "nvfp4"),
    ]
    mlp = fp4.pack_mlp4(weight(64, 96, 1), weight(64, 96, 2), weight(64, 64, 3))
    y32 = torch.empty(40, 64, dtype=F32, device=dev)
    x40 = acts(40, 96, 1)
    bad += [
        lambda: fp4.mlp4(x40, mlp, y32, 0.0),
        lambda: fp4.mlp4(x40, mlp, y32, math.nan),
        lambda: fp4.mlp4(x40, mlp, y32, math.inf, act4=True),                               # nvfp4 needs a finite limit
        lambda: fp4.mlp4(x40, mlp, y32[:39], 10.0),
        lambda: fp4.mlp4(x40, fp4.MLP4(mlp.down, mlp.down, 64), y32, 10.0),
    ]
    for i, f in enumerate(bad):
        with pytest.raises((RuntimeError, ValueError)):
            f()
            pytest.fail(f"call {i} was accepted")
    with pytest.raises(ValueError):
        fp4.quantize4(x, "fp4")
    with pytest.raises(ValueError):
        fp4.pack_mlp4(weight(48, 96, 1), weight(48, 96, 2), weight(64, 48, 3))
    with pytest.raises(ValueError):
        fp4.pack_mlp4(weight(64, 96, 1), weight(64, 64, 2), weight(64, 64, 3))
    torch.cuda.synchronize()
