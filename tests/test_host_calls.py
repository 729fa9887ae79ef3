"""What the entry points ask of the CUDA runtime, on the CPU: ``host_calls.c`` takes the
runtime's place and writes down whose attributes are set and which kernels start."""
import os
import subprocess

import pytest

from moe_b200 import _lib

TESTS = os.path.dirname(os.path.abspath(__file__))
INCLUDE = os.path.join(os.path.dirname(TESTS), "include")


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    exe = str(tmp_path_factory.mktemp("host") / "host_calls")
    subprocess.run(["gcc", "-std=gnu11", "-Wall", "-rdynamic", "-I", INCLUDE, os.path.join(TESTS, "host_calls.c"), "-o", exe,
                    "-ldl"], check=True)
    return exe


def calls(program, *names, fail=""):
    """{call: (status, kernels set up, kernels launched)} of the entry points called in this order."""
    _lib.load()
    # the library still asks for the runtime's file, whose functions the program's precede
    with open("/proc/self/maps") as f:
        runtime = {os.path.dirname(line.split()[-1]) for line in f if "libcudart.so" in line}
    env = dict(os.environ, LD_LIBRARY_PATH=":".join([*sorted(runtime), os.environ.get("LD_LIBRARY_PATH", "")]))
    p = subprocess.run([program, _lib.LIB_PATH, fail, *names], capture_output=True, text=True, timeout=60, env=env)
    assert p.returncode == 0, p.stderr
    got, setup, launched = {}, [], []
    for line in p.stdout.splitlines():
        what, name, *status = line.split()
        if what == "call":
            got[name] = int(status[0]), setup, launched
            setup, launched = [], []
        else:
            (launched if what == "launch" else setup).append(name)
    assert list(got) == list(names)
    return got


def test_operators_set_up_their_own_kernels(program):
    """A norm, a routing or a quantisation needs no product's kernels loaded, the layer
    none of the 4-bit products', and they none of the layer's."""
    got = calls(program, "norm", "route", "quantize", "forward", "linear", "matmul")
    for name in ("norm", "route", "quantize"):
        st, setup, launched = got[name]
        assert st == 0 and setup == [] and len(launched) == 1, name
    st, setup, launched = got["forward"]
    assert st == 0 and setup and not any("fp4" in k for k in setup + launched)
    st, setup, launched = got["linear"]
    assert st == 0 and setup and all("fp4" in k for k in setup) and len(launched) == 1
    st, setup, launched = got["matmul"]
    assert st == 0 and setup == [] and len(launched) == 1      # set up once


@pytest.mark.parametrize("fail,fine,refused", [("fp4", ("norm", "route", "quantize", "forward"), ("linear", "matmul")),
                                               ("moe_gemm", ("norm", "route", "quantize", "linear", "matmul"), ("forward",))])
def test_a_kernel_that_cannot_be_set_up_stops_its_own_operators(program, fail, fine, refused):
    got = calls(program, *refused, *fine, fail=fail)
    for name in fine:
        assert got[name][0] == 0, name
    for name in refused:
        assert got[name][0] == _lib.MOE_ERR_CUDA and got[name][2] == [], name
