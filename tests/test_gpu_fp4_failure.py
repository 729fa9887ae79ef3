"""Bounded waits of the 4-bit products, without a GPU fault: MOE_FP4_TEST_STALL makes the
MMA warps wait on a barrier that nothing completes.  Every kernel then gives up, lets
its copies land, fills its tiles with NaN, frees its TMEM and returns; the error
word tells of the wait, and the next product is right."""
import json
import os
import subprocess
import sys

import pytest
import torch

import moe_b200
from fp4_stall_worker import stalled
from moe_b200 import _lib

pytestmark = pytest.mark.gpu

SPLIT_SITES, PAIR_SITES = {40, 41, 42, 43}, {50, 51, 52, 53, 54}
WORKER = os.path.join(os.path.dirname(os.path.abspath(__file__)), "fp4_stall_worker.py")


@pytest.mark.parametrize("cases,sites", [
    # one CTA and clusters, tokens quantised inside (more and fewer K blocks than stages), before, and beforehand
    ([(3, 200, 96, False), (1, 4096, 7168, False), (4, 300, 7168, False), (40, 500, 2080, False), (200, 300, 7168, True)],
     SPLIT_SITES),
    # CTA pairs; their bound of 2 s for copies in flight is part of it
    ([(700, 4000, 512, True), (1000, 2100, 2080, False)], PAIR_SITES)])
def test_waits_that_run_out(cuda_device, cases, sites):
    check(cases, sites)


def test_tiles_after_the_one_whose_wait_ran_out(cuda_device):
    """A pair's later tiles are NaN too: their barrier phases never come."""
    check([(2500, 2100, 2080, False), (6001, 5003, 352, True)], PAIR_SITES)


@pytest.mark.parametrize("t,n,k,quantised", [(2, 300, 512, False), (60, 300, 1024, True), (90, 300, 1024, True)])
def test_an_error_is_read_once(cuda_device, t, n, k, quantised):
    assert moe_b200.fp4_device_error() == (0, 0)
    x = torch.ones(t, k, device="cuda", dtype=torch.bfloat16)
    w = moe_b200.quantize_fp4(torch.ones(n, k, device="cuda"))
    want = moe_b200.linear_fp4(x, *w)
    st, out = stalled(x, w, "nvfp4", quantised)
    assert st == 0 and out.isnan().all()
    code, info = moe_b200.fp4_device_error()
    assert code == _lib.MOE_ERR_TIMEOUT and info in (SPLIT_SITES if t < 65 else PAIR_SITES)
    assert moe_b200.fp4_device_error() == (0, 0)
    # the next product leaves none, and the next time-out is told of again
    assert torch.equal(moe_b200.linear_fp4(x, *w), want) and moe_b200.fp4_device_error() == (0, 0)
    stalled(x, w, "nvfp4", quantised)
    assert moe_b200.fp4_device_error()[0] == _lib.MOE_ERR_TIMEOUT
    assert moe_b200.fp4_device_error() == (0, 0)


def check(cases, sites):
    # a process of its own: the error word is the device's
    p = subprocess.run([sys.executable, WORKER, json.dumps(cases)], capture_output=True, text=True, timeout=300)
    assert p.returncode == 0, p.stderr[-2000:]
    got = json.loads(p.stdout.splitlines()[-1])
    assert len(got["results"]) == 2 * len(cases)
    for r in got["results"]:
        assert r["status"] == 0 and r["nan"] and r["after"], r
        # 10 ms of the first try, the limit, and for a pair 2 s; far from a limit for each stage
        assert r["seconds"] < (3.0 if sites is PAIR_SITES else 1.0), r
    code, info = got["error"]
    assert code == _lib.MOE_ERR_TIMEOUT and info in sites
