"""4-bit products under extreme scales: tensor scales whose product passes the ends of
fp32 where the outputs do not, and mxfp4 scales that cancel."""
import pytest
import torch

import moe_b200
from test_gpu_fp4 import check_product, one, rows, values

pytestmark = pytest.mark.gpu
# one launch, split kernel, pair kernel
SHAPES = [(3, 130, 96), (40, 257, 1056), (700, 4000, 288)]


def products(x, w, ga, gb, dtype):
    a, b = moe_b200.quantize_fp4(x, global_scale=ga), moe_b200.quantize_fp4(w, global_scale=gb)
    got = moe_b200.matmul_fp4(*a, *b, a_global_scale=ga, b_global_scale=gb, dtype=dtype)
    lin = moe_b200.linear_fp4(x, *b, x_global_scale=ga, w_global_scale=gb, dtype=dtype)
    assert torch.equal(got, lin)
    return got, values(*a, "nvfp4", ga), values(*b, "nvfp4", gb)


@pytest.mark.parametrize("t,n,k", SHAPES)
@pytest.mark.parametrize("ea,eb", [(-70, -70), (-100, -40), (-20, -110), (-120, -30)])
def test_tensor_scales_with_a_subnormal_product(cuda_device, t, n, k, ea, eb):
    """Scales of about 2^-140 to 2^-150 together, outputs of about 2^-115."""
    ga, gb = one(1.37 * 2.0 ** ea), one(1.71 * 2.0 ** eb)
    x = rows(t, k, torch.float32, t + k, 400.0) * ga
    w = rows(n, k, torch.float32, n + k, 400.0) * gb
    got, a, b = products(x, w, ga, gb, torch.float32)
    check_product(got, a, b, k, torch.float32)
    assert (got != 0).float().mean() > 0.99
    got, a, b = products(x, w, ga, gb, torch.bfloat16)
    check_product(got, a, b, k, torch.bfloat16)


@pytest.mark.parametrize("t,n,k", SHAPES)
@pytest.mark.parametrize("ea,eb", [(70, 70), (100, 40), (15, 125), (126, 14)])
def test_tensor_scales_with_an_infinite_product(cuda_device, t, n, k, ea, eb):
    """Scales of 2^140 together; sums of a few products of the smallest values, and none."""
    ga, gb = one(1.37 * 2.0 ** ea), one(1.71 * 2.0 ** eb)
    gen = torch.Generator(device="cuda").manual_seed(t)
    x = torch.zeros(t, k, device="cuda")
    w = torch.zeros(n, k, device="cuda")
    x[:, ::16] = torch.randint(-3, 4, (t, (k + 15) // 16), generator=gen, device="cuda") * 2.0 ** -10 * ga
    w[:, ::32] = torch.randint(-3, 4, (n, (k + 31) // 32), generator=gen, device="cuda") * 2.0 ** -10 * gb
    x[0] = 0
    w[n - 1] = 0
    got, a, b = products(x, w, ga, gb, torch.float32)
    exact = a @ b.t()
    fine = exact.abs() < 2.0 ** 127
    assert fine.float().mean() > 0.5 and (exact != 0).any()
    assert got[fine].isfinite().all()
    # sums of a few small multiples of 2^-20, exact in fp32; two factors round once each
    assert ((got.double() - exact).abs() <= exact.abs() * 2.0 ** -23)[fine].all()
    assert (got[0] == 0).all() and (got[:, n - 1] == 0).all()


@pytest.mark.parametrize("t,n,k", SHAPES)
@pytest.mark.parametrize("e", [-100, -60, 60, 100])
def test_mxfp4_scales_that_cancel(cuda_device, t, n, k, e):
    """Powers of two in one operand and their inverse in the other change no bit."""
    x, w = rows(t, k, torch.float32, t + k), rows(n, k, torch.float32, n + k, 0.02)
    for dtype in (torch.float32, torch.bfloat16):
        want = moe_b200.linear_fp4(x, *moe_b200.quantize_fp4(w, "mxfp4"), "mxfp4", dtype=dtype)
        got = moe_b200.linear_fp4(x * 2.0 ** e, *moe_b200.quantize_fp4(w * 2.0 ** -e, "mxfp4"), "mxfp4", dtype=dtype)
        assert torch.equal(got, want)
