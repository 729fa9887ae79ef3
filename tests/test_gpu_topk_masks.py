"""Masked experts in route_topk: logits of -inf or NaN, with a bias and in groups."""
import math

import pytest
import torch

from test_gpu_topk import run_and_check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("masked", [-math.inf, math.nan])
def test_masked_experts_with_a_bias(cuda_device, score, masked):
    """A -inf or NaN logit is a score of 0: chosen by its bias, with weight 0; a -inf or
    NaN bias is chosen last."""
    x = torch.randn(40, 64, generator=torch.Generator(device="cuda").manual_seed(4), device="cuda")
    x[::2, [3, 40]] = masked
    bias = torch.zeros(64, device="cuda")
    bias[3], bias[40] = 2.0, -2.0
    bias[7] = masked
    for renormalize in (True, False):
        idx, w = run_and_check(x, 5, bias=bias, score=score, renormalize=renormalize)
        assert (idx[:, 0] == 3).all() and (w[::2, 0] == 0).all() and (w[1::2, 0] > 0).all()
        assert not ((idx == 40) | (idx == 7)).any()
        idx, w = run_and_check(x, 6, bias=bias, score=score, renormalize=renormalize, n_group=4, topk_group=2)
        assert (idx[:, 0] == 3).all()
    without, _ = run_and_check(x[::2], 32, score=score)
    assert not ((without == 3) | (without == 40)).any()


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("masked", [-math.inf, math.nan])
@pytest.mark.parametrize("e", [16, 64, 512, 1024])
def test_masked_experts_in_groups(cuda_device, e, masked, score):
    """Groups of which the mask leaves one expert or none are ranked by what is left."""
    x = torch.randn(60, e, generator=torch.Generator(device="cuda").manual_seed(e), device="cuda")
    per = x.view(60, 4, -1)
    per[::3, 0, 1:] = masked          # one expert left in the first group
    per[::3, 0, 0] = 6.0
    per[1::3, 1] = masked             # none in the second
    per[::2, 2, ::2] = masked
    bias = 0.1 * torch.randn(e, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    for b in (None, bias, bias.bfloat16()):
        for group_score in ("top2", "max"):
            for kept in (1, 2, 3):
                run_and_check(x, 4, bias=b, score=score, n_group=4, topk_group=kept, group_score=group_score)
