"""4-bit operators at the edges of their arguments."""

import pytest
import torch

from glm53.ops import fp4
from glm53.ops import kernels as K
from test_gpu_fp4 import BF, F32, FMTS, act_tol, acts, gated, h_slack, quant, sums_tol, weight

pytestmark = pytest.mark.gpu


def fill_free_memory(byte=255, sizes=(512, 4096, 1 << 15, 1 << 17, 1 << 19, 4 << 20)):
    """Leaves the allocator's free blocks full of one byte (255: NaN in every type)."""
    torch.cuda.empty_cache()
    keep = [torch.full((n,), byte, dtype=torch.uint8, device="cuda") for n in sizes for _ in range(64)]
    torch.cuda.synchronize()
    del keep


def check_mlp_act4(fmt, m, k, width, n, limit):
    """mlp4 with 4-bit activations against 64 bits.  |silu(min(g, L))| <= max(L, 0.2785) and |u| <= L: the bound that the
    nvfp4 row scale of h has to fit."""
    x, gate, up, down = acts(m, k, m), weight(width, k, 1), weight(width, k, 2), weight(n, width, 3)
    mlp = fp4.pack_mlp4(gate, up, down, fmt)
    xq, gq, uq, dq = quant(x, fmt), quant(gate, fmt), quant(up, fmt), quant(down, fmt)
    h = gated(xq, gq, uq, limit)
    bound = max(limit, 0.2785) * limit
    # |silu'| <= 1.1 times |u| <= L, and |silu| <= max(L, 0.2785) times the error of u; exp and the division: 2^-20
    eh = 1.1 * max(limit, 0.2785) * (sums_tol(xq, gq) + sums_tol(xq, uq)) + 2.0 ** -20 * h.abs()
    hq = quant(h, fmt, bound)
    slack = h_slack(h, eh, fmt, bound)
    ref = hq @ dq.t()
    tol = slack @ dq.abs().t() + sums_tol(hq.abs() + slack, dq)
    fill_free_memory()
    y = fp4.mlp4(x, mlp, torch.zeros(m, n, dtype=F32, device="cuda"), limit, act4=True)
    assert ((y.double() - ref).abs() <= tol).all()
    # few codes change (those within the sums' error of a border), each by at most its own size
    assert (y.double() - ref).norm() <= 0.01 * ref.norm()


# limits whose square lies on both sides of the powers of two of the row scale: 1 for 36.7 < limit <= 51.8
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("m", [17, 64, 128, 129])
@pytest.mark.parametrize("limit", [36.0, 40.0, 50.0, 51.84, 60.0])
def test_mlp_4bit_activations_wide_limits(fmt, m, limit):
    check_mlp_act4(fmt, m, 256, 160, 72, limit)


# below 0.2785 the gate's lowest value, -0.2785, is further out than the limit
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("m", [17, 100, 200])
@pytest.mark.parametrize("limit", [0.01, 0.1, 0.25, 0.28])
def test_mlp_4bit_activations_small_limits(fmt, m, limit):
    check_mlp_act4(fmt, m, 256, 160, 72, limit)


@pytest.mark.parametrize("m,n,k", [(1, 38400, 6144), (4, 38400, 6144), (16, 38400, 6144), (96, 6400, 12288)])
def test_linear_repeats_itself_over_many_row_blocks(m, n, k):
    """Clusters that share blocks of weight rows and go through three or more: the exchange of a block must not reach a rank
    that still reads the one two before it."""
    fmt = "mxfp4"
    x, w4 = acts(m, k, m), fp4.quantize4(weight(n, k, 3), fmt)
    y = fp4.linear4(x, w4, torch.empty(m, n, dtype=F32, device="cuda"), K.GEMV_F32)
    for _ in range(50):
        assert torch.equal(fp4.linear4(x, w4, torch.empty_like(y), K.GEMV_F32), y)
    some = torch.arange(0, n, 97, device="cuda")
    wq = fp4.dequantize4(w4, F32)[some].double()
    tol = sums_tol(x.double(), wq) + act_tol(x.double(), wq, fmt)
    assert ((y[:, some].double() - x.double() @ wq.t()).abs() <= tol).all()
    fp4.check_errors()


PATHS = [(3, 200, False), (12, 200, False), (40, 200, False), (90, 200, False), (150, 200, False), (700, 200, False),
         (20, 200, True), (128, 200, True), (150, 200, True), (2600, 1800, True)]


def far(m, n, k=256):
    x, w = acts(m, k, m), weight(n, k, 5)
    x[0] = 2.0 ** -64
    x[1] = 2.0 ** 80
    x[1, ::2] *= -1
    x[2] = 2.0 ** 118
    w[0] = 2.0 ** -65
    w[1] = 2.0 ** 80
    w[2] = 2.0 ** -4
    w[3] *= 2.0 ** -60
    return x, w


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("m,n,act4", PATHS)
def test_linear_scales_far_apart(fmt, m, n, act4):
    """Results inside fp32's range come out whatever the scales of the two rows are."""
    x, w = far(m, n)
    w4, wq = fp4.quantize4(w, fmt), quant(w, fmt)
    a = quant(x, fmt) if act4 else x.double()
    y = fp4.linear4(x, w4, torch.empty(m, n, dtype=F32, device="cuda"), K.GEMV_F32, act4=act4).double()
    mag = a.abs() @ wq.abs().t()
    # where the sum of magnitudes nears fp32's largest a partial sum may be an infinity; a last rounding below 2^-126 is off by
    # at most 2^-149
    tol = sums_tol(a, wq) + (0 if act4 else act_tol(a, wq, fmt)) + 2.0 ** -149
    fine = mag < 2.0 ** 127
    assert fine[0].all() and fine[2, 0] and fine[2, 2] and fine[2, 4:].all()
    assert ((y - a @ wq.t()).abs() <= tol)[fine].all()


@pytest.mark.parametrize("m,n,act4", PATHS)
def test_linear_zero_sums_of_large_rows(m, n, act4):
    """nvfp4: codes and block scales of +-2^80 and 2^80 sum to 0 exactly, and 0 times any row scales is 0."""
    x, w = far(m, n)
    y = fp4.linear4(x, fp4.quantize4(w, "nvfp4"), torch.empty(m, n, dtype=F32, device="cuda"), K.GEMV_F32, act4=act4)
    assert y[1, 0] == 0 and y[1, 1] == 0 and y[1, 2] == 0


@pytest.mark.parametrize("m,width", [(150, 160), (2600, 928)])
def test_mlp_zero_gates_of_large_rows(m, width):
    """A gate whose sum is 0 gives 0, with 4-bit activations, too, whatever its row scales."""
    k = 256
    x = acts(m, k, m)
    x[1::2] = 2.0 ** 80
    x[1::2, ::2] *= -1
    mlp = fp4.pack_mlp4(torch.full((width, k), 2.0 ** 80, dtype=BF, device="cuda"), weight(width, k, 2), weight(64, width, 3))
    y = fp4.mlp4(x, mlp, torch.empty(m, 64, dtype=F32, device="cuda"), 10.0, act4=True)
    assert (y[1::2] == 0).all() and torch.isfinite(y).all()


def test_check_errors_waits_for_every_stream():
    s, ev = torch.cuda.Stream(), torch.cuda.Event()
    with torch.cuda.stream(s):
        torch.cuda._sleep(100_000_000)                  # about 50 ms
        ev.record()
    fp4.check_errors()
    assert ev.query()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("m,act4", [(1, False), (8, False), (12, False), (30, False), (90, False), (90, True), (150, False),
                                    (150, True)])
def test_products_chained_through_one_pair_of_buffers(fmt, m, act4):
    """Each product reads what the launch before it wrote, and writes what that one read: the bits of a run with a wait after
    every call."""
    k = 1024
    w4 = fp4.quantize4(weight(k, k, 4), fmt)
    x = acts(m, k, 1)

    def chain(wait):
        bufs = [x.clone(), torch.empty_like(x)]
        for i in range(40):
            fp4.linear4(bufs[i % 2], w4, bufs[1 - i % 2], act4=act4)
            if wait:
                torch.cuda.synchronize()
        return bufs[0]
    want = chain(True)
    assert torch.isfinite(want).all() and want.any()
    assert all(torch.equal(chain(False), want) for _ in range(5))
    fp4.check_errors()


@pytest.mark.parametrize("fmt", FMTS)
def test_longest_rows(fmt):
    """A row of more than 65535 times 1024 columns, there and back."""
    k = 65535 * 1024 + 4096 + 32
    x = acts(1, k, 1)
    y = fp4.dequantize4(fp4.quantize4(x, fmt))
    torch.cuda.synchronize()
    ref = quant(x, fmt)
    assert torch.equal(y.double(), ref)


def tiny(rows, k):
    """Rows around 2^-70, 2^-95, 2^-105, 2^-120 and among bf16's subnormals."""
    x = acts(rows, k, 3)
    for i, e in enumerate((-70, -95, -105, -120, -128)):
        x[i] = (x[i].double() * 2.0 ** e).to(BF)
    return x


def test_quantize_smallest_magnitudes():
    x = tiny(6, 256)
    assert torch.equal(fp4.dequantize4(fp4.quantize4(x, "nvfp4"), F32).double(), quant(x, "nvfp4"))
    # mxfp4: scales from 2^-126; from there on codes are multiples of 2^-127
    b = x.double().view(6, -1, 32)
    s = torch.exp2(torch.ceil(torch.log2(b.abs().amax(-1, keepdim=True) / 6))).clamp_min(2.0 ** -126)
    low = s == 2.0 ** -126
    assert low[4].all() and not low[0].any()
    y = fp4.dequantize4(fp4.quantize4(x, "mxfp4"), F32).double().view(b.shape)
    q = b.abs() / s
    # half the distance of the two codes around q: 1/4 below 2, 1/2 below 4, 1 below 6
    assert ((y - b).abs() <= s * torch.where(q <= 2, 0.25, torch.where(q <= 4, 0.5, 1.0))).all()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("m", [6, 12, 40, 150])
def test_linear_smallest_magnitudes(fmt, m):
    n, k = 136, 512
    x, w = tiny(m, k), weight(n, k, 5)
    w4, wq = fp4.quantize4(w, fmt), quant(w, fmt)
    y = fp4.linear4(x, w4, torch.empty(m, n, dtype=F32, device="cuda"), K.GEMV_F32)
    # what the expansion (and, widened, fp32's own range) leaves out of an element of such rows: 2^-124
    tol = sums_tol(x.double(), wq) + act_tol(x.double(), wq, fmt) + 2.0 ** -124 * wq.abs().sum(1)
    assert ((y.double() - x.double() @ wq.t()).abs() <= tol).all()
