"""4-bit operators at the edges of their arguments."""

import pytest
import torch

from glm53.ops import fp4
from glm53.ops import kernels as K
from test_gpu_fp4 import F32, FMTS, act_tol, acts, gated, h_slack, quant, sums_tol, weight

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
