"""Microscaled 4-bit matrices: codes and scales equal the definition bit for bit
(both round exact quotients), products against the sum of the values in 64 bits.

Bound of a product: values times values are exact; the tensor core adds the
products of a K = 64 step aligned to the largest of them and the steps to an fp32
accumulator, each addition losing at most 2^-23 of the sums' magnitude, so the sum
is within (64 + K / 64) * 2^-23 * sum |a||b|.  The tensor scales multiply with two
roundings and the output rounds once.
"""
import pytest
import torch

import moe_b200

pytestmark = pytest.mark.gpu

RUN = {"mxfp4": 32, "nvfp4": 16}
LEVELS = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)


def e4m3_values():
    return torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()


def nearest_even(v, values):
    """Index of the value nearest to v >= 0, ties to the even index."""
    i = torch.searchsorted(values, v).clamp(max=len(values) - 1)
    lo = (i - 1).clamp(min=0)
    dl, dh = v - values[lo], values[i] - v
    up = (dh < dl) | ((dh == dl) & (i % 2 == 0))
    return torch.where(up, i, lo)


def reference_quantize(x, fmt, g=None):
    """(codes one per element, scale codes [R, runs], values) on the CPU."""
    x = x.double().cpu()
    r, k = x.shape
    b = x.view(r, -1, RUN[fmt])
    amax = b.abs().amax(-1)
    bad = ~torch.isfinite(b).all(-1)
    amax = torch.where(bad, torch.zeros_like(amax), amax)
    if fmt == "mxfp4":
        e = (torch.frexp(amax)[1] - 3).clamp(min=-127)
        e = torch.where(amax == 0, torch.full_like(e, -127), e)
        scale, d = (e + 127), torch.exp2(e.double())
        nan = 255
    else:
        g = torch.ones((), dtype=torch.float64) if g is None else g.double().cpu().reshape(())
        # amax / (6 g) against the borders: both sides times 6 g are exact in 64 bits
        vals = e4m3_values()
        scale = nearest_even(amax, vals * (6 * g))
        scale = torch.where(amax > 0, scale.clamp(min=1), torch.zeros_like(scale))
        d = vals[scale] * g
        nan = 127
    # |x| / d against the levels, times d (exact: 2 + 4 + 24 bits)
    lv = LEVELS[None, None, :] * d[..., None]
    a = b.abs()
    mids = (lv[..., 1:] + lv[..., :-1]) / 2
    code = torch.zeros(b.shape, dtype=torch.int64)
    for i in range(7):
        m = mids[..., i:i + 1]
        code += (a >= m if i % 2 == 1 else a > m).long()
    code = torch.where(d[..., None] > 0, code, torch.zeros_like(code))
    values = LEVELS[code] * d[..., None] * torch.where(torch.signbit(b), -1.0, 1.0)
    code = code + 8 * torch.signbit(b).long()
    code = torch.where(bad[..., None], torch.zeros_like(code), code)
    scale = torch.where(bad, torch.full_like(scale, nan), scale)
    values = torch.where(bad[..., None], torch.full_like(values, float("nan")), values)
    return code.view(r, k), scale, values.view(r, k)


def unpack(codes):
    c = codes.cpu().long()
    return torch.stack((c & 15, c >> 4), -1).view(c.shape[0], -1)


def unblock(scales, r, runs):
    """Row-major scales and the bytes that fill up the last blocks."""
    s = scales.cpu().long()
    rb, cb = s.shape[:2]
    full = s.permute(0, 3, 2, 1, 4).reshape(rb * 128, cb * 4)
    pad = full.clone()
    pad[:r, :runs] = 0
    return full[:r, :runs], pad


def check_quantize(x, fmt, g=None):
    codes, scales = moe_b200.quantize_fp4(x, fmt, global_scale=g)
    r, k = x.shape
    assert tuple(scales.shape) == moe_b200.fp4_scales_shape(r, k, fmt)
    ref_c, ref_s, ref_v = reference_quantize(x, fmt, g)
    got_s, pad = unblock(scales, r, k // RUN[fmt])
    assert torch.equal(got_s, ref_s), (got_s != ref_s).nonzero()[:4]
    assert (pad == 0).all()
    got_c = unpack(codes)
    assert torch.equal(got_c, ref_c), (got_c != ref_c).nonzero()[:4]
    v = moe_b200.dequantize_fp4(codes, scales, fmt, global_scale=g, dtype=torch.float32).cpu().double()
    assert torch.equal(v.isnan(), ref_v.isnan())
    fine = ~ref_v.isnan()
    assert ((v - ref_v).abs() <= ref_v.abs() * 2.0 ** -24 + 2.0 ** -150)[fine].all()
    for dt in (torch.bfloat16, torch.float16):
        h = moe_b200.dequantize_fp4(codes, scales, fmt, global_scale=g, dtype=dt)
        assert torch.equal(h.cpu().view(torch.int16)[fine], v.float().to(dt).view(torch.int16)[fine])
    return codes, scales


def rows(r, k, dtype, seed, scale=1.0):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return (scale * torch.randn(r, k, generator=gen, device="cuda")).to(dtype)


def one(v):
    return torch.full((1,), v, dtype=torch.float32, device="cuda")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("r,k", [(1, 32), (1, 7168), (3, 96), (127, 160), (128, 256), (129, 288), (300, 1024)])
def test_quantise_is_exact(cuda_device, r, k, dtype):
    x = rows(r, k, dtype, r + k)
    check_quantize(x, "mxfp4")
    check_quantize(x, "nvfp4")
    check_quantize(x, "nvfp4", one(7.3 / 2688))      # many quotients on or beside borders
    check_quantize(x, "nvfp4", one(8.0 / 2688))
    check_quantize(x, "nvfp4", x.abs().max().float().reshape(1) / 2688)


def test_quantise_extremes(cuda_device):
    x = rows(16, 128, torch.float32, 5)
    x[0] = 0
    x[1] *= 1e-40          # subnormals
    x[2] *= 1e38
    x[3, :32] = torch.finfo(torch.float32).max
    x[4, 3], x[5, 40], x[6, 100] = float("nan"), float("inf"), -float("inf")
    x[7] = -0.0
    x[8, 1:] = 1e-30       # one large value beside tiny ones
    x[9] = torch.exp2(torch.arange(128, device="cuda").float() - 140)
    check_quantize(x, "mxfp4")
    for g in (None, one(1e-3), one(1e30), one(1e-30), one(2.0 ** -140)):
        check_quantize(x, "nvfp4", g)
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0] * 4, device="cuda")[None].repeat(4, 1)
    ties[1] *= -1
    ties[2] *= 0.5
    check_quantize(ties, "mxfp4")
    check_quantize(ties, "nvfp4")
    for g in (one(0.0), one(-1.0), one(float("nan")), one(float("inf"))):
        _, s = moe_b200.quantize_fp4(x, "nvfp4", global_scale=g)
        assert (unblock(s, 16, 8)[0] == 127).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_quantise_16_bit_extremes(cuda_device, dtype):
    """Every finite value of the type, as the largest of its run and beside larger
    ones; subnormals, zeros, infinities and NaN."""
    bits = torch.arange(1 << 16, dtype=torch.int32, device="cuda").to(torch.int16)
    every = bits.view(dtype).view(-1, 256)
    keep = torch.isfinite(every)
    x = torch.where(keep, every, torch.zeros_like(every))
    perm = torch.randperm(x.numel(), generator=torch.Generator().manual_seed(7)).to("cuda")
    mixed = x.flatten()[perm].view(-1, 256)
    for m in (x, mixed, mixed[:, :96].contiguous()):
        check_quantize(m, "mxfp4")
        for g in (None, one(1.0 / 2688), one(3.0 / 7), one(2.0 ** -20)):
            check_quantize(m, "nvfp4", g)
    check_quantize(every, "mxfp4")
    check_quantize(every, "nvfp4")


@pytest.mark.parametrize("exponent", [-140, -127, -120, -116, -100, 100, 119, 121, 122, 124, 126, 127])
def test_quantise_under_a_tensor_scale_near_the_ends_of_fp32(cuda_device, exponent):
    """Values on and next to the borders of two codes, as bf16 has them, in runs of every
    scale below 2^-5: the odd multiples of a large tensor scale that tell the side pass
    the end of fp32, the values themselves do not."""
    codes = torch.arange(1, 16)
    s = e4m3_values()[codes]
    borders = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0], dtype=torch.float64)
    for m in list(range(1, 64, 2)) + [127, 255, 2 ** 23 + 1, 2 ** 24 - 1]:
        g = m * 2.0 ** (exponent - m.bit_length() + 1)      # in [2^exponent, 2^(exponent + 1))
        on = (borders[None] * (s * g)[:, None]).float().bfloat16()
        ulp = on.view(torch.int16)
        row = torch.cat((on, (ulp[:, :7] + 1).view(torch.bfloat16), -on,
                         (ulp[:, :7] - 1).clamp(min=0).view(torch.bfloat16)), 1)
        x = torch.cat((row, torch.zeros(15, 2, dtype=torch.bfloat16)), 1).to("cuda")
        assert x.isfinite().all()
        # runs of 16: the first holds its largest value, the second the negative ones
        check_quantize(x, "nvfp4", one(g))


def test_quantise_strided_input_and_views(cuda_device):
    wide = rows(40, 640, torch.bfloat16, 6)
    for x in (wide[:, 64:384], wide[::2, :128], wide[:, 3:35], wide.t()[:, :32]):
        c, s = check_quantize(x, "nvfp4")
        c2, s2 = moe_b200.quantize_fp4(x.contiguous(), "nvfp4")
        assert torch.equal(c, c2) and torch.equal(s, s2)
    big = torch.zeros(40, 320, dtype=torch.uint8, device="cuda")
    c, s = moe_b200.quantize_fp4(wide, "mxfp4")
    big[:, :].copy_(c)
    v = moe_b200.dequantize_fp4(big[5:], moe_b200.quantize_fp4(wide[5:], "mxfp4")[1], "mxfp4")
    assert torch.equal(v, moe_b200.dequantize_fp4(c, s, "mxfp4")[5:])
    c, s = moe_b200.quantize_fp4(wide[:0], "mxfp4")
    assert c.shape == (0, 320) and moe_b200.dequantize_fp4(c, s, "mxfp4").shape == (0, 640)


def values(codes, scales, fmt, g=None):
    """The matrix in 64 bits, without the tensor scale's rounding."""
    v = moe_b200.dequantize_fp4(codes, scales, fmt, dtype=torch.float32).double()
    return v if g is None else v * g.double()


def check_product(got, a, b, k, dtype):
    exact = a @ b.t()
    size = a.abs() @ b.abs().t()
    step = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[dtype]
    tiny = {torch.float32: 1e-40, torch.bfloat16: 1e-38, torch.float16: 2.0 ** -25}[dtype]
    bound = size * ((64 + k / 64 + 2) * 2.0 ** -23) * (1 + step) + exact.abs() * step + tiny
    err = (got.double() - exact).abs()
    assert got.dtype == dtype and (err <= bound).all(), ((err / bound).max(), (err > bound).nonzero()[:4])


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("t,n,k", [
    (1, 1, 32), (1, 128, 7168), (2, 130, 64), (3, 20000, 512), (4, 257, 2080), (4, 1000, 7168), (3, 129, 96),
    (5, 300, 1056), (15, 300, 320), (16, 128, 256), (17, 129, 1056), (31, 4096, 512),
    (33, 100, 2048), (64, 512, 96), (65, 1000, 480), (127, 127, 128), (128, 256, 1024), (129, 384, 288),
    (300, 200, 7168), (257, 1025, 2080), (600, 2048, 256), (1000, 1000, 512),
])
def test_product(cuda_device, t, n, k, fmt):
    x, w = rows(t, k, torch.bfloat16, t + k), rows(n, k, torch.bfloat16, n + k, 0.02)
    ga = gb = None
    if fmt == "nvfp4":
        ga, gb = x.abs().max().float().reshape(1) / 2688, w.abs().max().float().reshape(1) / 2688
    a, b = moe_b200.quantize_fp4(x, fmt, global_scale=ga), moe_b200.quantize_fp4(w, fmt, global_scale=gb)
    va, vb = values(*a, fmt, ga), values(*b, fmt, gb)
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        got = moe_b200.matmul_fp4(*a, *b, fmt, a_global_scale=ga, b_global_scale=gb, dtype=dtype)
        check_product(got, va, vb, k, dtype)
        again = moe_b200.matmul_fp4(*a, *b, fmt, a_global_scale=ga, b_global_scale=gb, dtype=dtype)
        assert torch.equal(got, again)
        # quantised on the way: the same product
        lin = moe_b200.linear_fp4(x, *b, fmt, x_global_scale=ga, w_global_scale=gb, dtype=dtype)
        assert torch.equal(lin, got)
    assert moe_b200.fp4_device_error() == (0, 0)


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("t,n,k", [(2500, 2100, 2080), (2100, 4000, 7168), (4200, 4100, 1440), (6001, 5003, 352)])
def test_product_of_many_tiles_a_pair(cuda_device, t, n, k, fmt):
    """Two to seven tiles for each CTA pair, fewer and more K blocks than the ring has
    stages, ragged ends: the ring's phases, both accumulators and the scale slots are
    used again and again."""
    x, w = rows(t, k, torch.bfloat16, t + k), rows(n, k, torch.bfloat16, n + k, 0.02)
    # every tile has rows of its own magnitude: one tile's sums or scales in another's place would show
    x *= torch.exp2(torch.arange(t, device="cuda") // 256 % 5 - 2.0)[:, None].bfloat16()
    w *= torch.exp2(torch.arange(n, device="cuda") // 256 % 3 - 1.0)[:, None].bfloat16()
    ga = gb = None
    if fmt == "nvfp4":
        ga, gb = x.abs().max().float().reshape(1) / 2688, w.abs().max().float().reshape(1) / 2688
    a, b = moe_b200.quantize_fp4(x, fmt, global_scale=ga), moe_b200.quantize_fp4(w, fmt, global_scale=gb)
    va, vb = values(*a, fmt, ga), values(*b, fmt, gb)
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        got = moe_b200.matmul_fp4(*a, *b, fmt, a_global_scale=ga, b_global_scale=gb, dtype=dtype)
        check_product(got, va, vb, k, dtype)
        assert torch.equal(got, moe_b200.matmul_fp4(*a, *b, fmt, a_global_scale=ga, b_global_scale=gb, dtype=dtype))
        lin = moe_b200.linear_fp4(x, *b, fmt, x_global_scale=ga, w_global_scale=gb, dtype=dtype)
        assert torch.equal(lin, got)
    assert moe_b200.fp4_device_error() == (0, 0)


def test_every_scale_and_column_lands_in_its_place(cuda_device):
    """Each row and run of both operands has a scale of its own, each column a
    code of its own: one wrong byte of scales moves a run's share of an output (1/32 of
    the columns, halved or doubled), far outside the bound."""
    for fmt in ("mxfp4", "nvfp4"):
        run, k, t, n = RUN[fmt], 512, 256, 256
        gen = torch.Generator(device="cuda").manual_seed(8)

        def matrix(r):
            e = torch.randint(-3, 4, (r, k // run, 1), generator=gen, device="cuda").float()
            m = torch.tensor([0.0, 0.5, 1, 1.5, 2, 3, 4, 6], device="cuda")
            v = m[torch.randint(0, 8, (r, k // run, run), generator=gen, device="cuda")]
            v[..., 0] = 6.0
            return (v * torch.exp2(e)).view(r, k)

        x, w = matrix(t), matrix(n)     # representable
        a, b = moe_b200.quantize_fp4(x, fmt), moe_b200.quantize_fp4(w, fmt)
        assert torch.equal(moe_b200.dequantize_fp4(*a, fmt, dtype=torch.float32), x)
        got = moe_b200.matmul_fp4(*a, *b, fmt, dtype=torch.float32)
        check_product(got, x.double(), w.double(), k, torch.float32)


def test_product_strided_operands_and_output(cuda_device):
    x, w = rows(50, 256, torch.bfloat16, 11), rows(200, 512, torch.bfloat16, 12)
    a, b = moe_b200.quantize_fp4(x), moe_b200.quantize_fp4(w[:, 256:].contiguous())
    wide, scales = moe_b200.quantize_fp4(w)
    right = wide[:, 128:]               # the codes of columns 256.. as a slice of the wide matrix
    assert torch.equal(right, b[0])
    want = moe_b200.matmul_fp4(*a, *b)
    assert torch.equal(moe_b200.matmul_fp4(*a, right, b[1]), want)
    for off in (0, 1, 3, 8):
        buf = torch.full((50, 300), 9.0, device="cuda", dtype=torch.bfloat16)
        out = buf[:, off:off + 200]
        assert moe_b200.matmul_fp4(*a, *b, out=out) is out
        assert torch.equal(out, want)
        assert (buf[:, :off] == 9).all() and (buf[:, off + 200:] == 9).all()
    assert moe_b200.matmul_fp4(a[0][:0], a[1][:0], *b).shape == (0, 200)
    assert moe_b200.linear_fp4(x[:0], *b).shape == (0, 200)
    xs = rows(50, 300, torch.float32, 13)[:, 20:276]
    assert torch.equal(moe_b200.linear_fp4(xs, *b), moe_b200.linear_fp4(xs.contiguous(), *b))


@pytest.mark.parametrize("t", [1, 4, 40])
def test_product_beside_its_input(cuda_device, t):
    """x and out as columns of one buffer, either first; out in x itself is refused."""
    x, b = rows(t, 256, torch.bfloat16, 31), moe_b200.quantize_fp4(rows(248, 256, torch.bfloat16, 32))
    want = moe_b200.linear_fp4(x, *b)
    for at, to in ((0, 256), (256, 8), (248, 0)):
        buf = torch.full((t, 512), 9.0, device="cuda", dtype=torch.bfloat16)
        buf[:, at:at + 256] = x
        moe_b200.linear_fp4(buf[:, at:at + 256], *b, out=buf[:, to:to + 248])
        assert torch.equal(buf[:, to:to + 248], want) and torch.equal(buf[:, at:at + 256], x)
        with pytest.raises(AssertionError):
            moe_b200.linear_fp4(buf[:, at:at + 256], *b, out=buf[:, at + 8:at + 256])
        assert torch.equal(buf[:, at:at + 256], x)


@pytest.mark.parametrize("t,n,k", [(3, 200, 96), (40, 200, 96), (200, 300, 7168), (700, 300, 96), (700, 4000, 512)])
def test_product_writes_its_output_alone(cuda_device, t, n, k):
    """Rows and columns around a strided, oddly aligned output stay as they were, on
    every kernel's tiles that end inside."""
    x, b = rows(t, k, torch.bfloat16, 21), moe_b200.quantize_fp4(rows(n, k, torch.bfloat16, 22))
    for dtype in (torch.float32, torch.bfloat16):
        want = moe_b200.linear_fp4(x, *b, dtype=dtype)
        for off, pad in ((1, 3), (4, 8)):
            buf = torch.full((t + 2, n + off + pad), 9.0, device="cuda", dtype=dtype)
            out = buf[1:t + 1, off:off + n]
            moe_b200.linear_fp4(x, *b, dtype=dtype, out=out)
            assert torch.equal(out, want)
            buf[1:t + 1, off:off + n] = 9.0
            assert (buf == 9.0).all()


def test_offsets_past_32_bits(cuda_device):
    k, r = 7168, 2 ** 31 // 7168 + 200
    x = torch.zeros(r, k, dtype=torch.bfloat16, device="cuda")
    x[-300:] = rows(300, k, torch.bfloat16, 23)
    for fmt in ("mxfp4", "nvfp4"):
        c, s = moe_b200.quantize_fp4(x, fmt)
        assert (c[:-300] == 0).all()
        first = r // 128 * 128 - 128           # whole blocks of rows at the end
        c2, s2 = moe_b200.quantize_fp4(x[first:], fmt)
        assert torch.equal(c[first:], c2) and torch.equal(s[first // 128:], s2)
        v = moe_b200.dequantize_fp4(c, s, fmt)
        assert torch.equal(v[first:], moe_b200.dequantize_fp4(c2, s2, fmt))
        del c, s, v
    del x
    t, n = 2 ** 20, 2100
    x, b = rows(t, 32, torch.bfloat16, 24), moe_b200.quantize_fp4(rows(n, 32, torch.bfloat16, 25))
    out = moe_b200.linear_fp4(x, *b)
    for part in (slice(0, 700), slice(t // 2, t // 2 + 700), slice(t - 700, t)):
        assert torch.equal(out[part], moe_b200.linear_fp4(x[part], *b))


def test_non_finite_values_stay_in_their_row(cuda_device):
    x, w = rows(40, 256, torch.bfloat16, 14), rows(140, 256, torch.bfloat16, 15)
    clean = moe_b200.linear_fp4(x, *moe_b200.quantize_fp4(w))
    x[7, 100], w[33, 5] = float("inf"), float("nan")
    for fmt in ("nvfp4", "mxfp4"):
        got = moe_b200.linear_fp4(x, *moe_b200.quantize_fp4(w, fmt), fmt)
        nan = got.isnan()
        assert nan[7].all() and nan[:, 33].all() and nan.sum() == 140 + 40 - 1
        if fmt == "nvfp4":
            assert torch.equal(got[~nan], clean[~nan])


def test_two_calls_at_once_and_graphs(cuda_device):
    """Calls on two streams, and two captured graphs replayed together, keep
    their own buffers."""
    w = moe_b200.quantize_fp4(rows(512, 1024, torch.bfloat16, 16))
    xs = [rows(t, 1024, torch.bfloat16, t) for t in (5, 40, 200)]
    want = [moe_b200.linear_fp4(x, *w) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for s, x in zip(streams, xs):
            with torch.cuda.stream(s):
                got.append(moe_b200.linear_fp4(x, *w))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs, outs = [], []
    for s, x in zip(streams, xs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs.append(moe_b200.linear_fp4(x, *w))
        graphs.append(g)
    for _ in range(3):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_dequantise_into_half_aligned_output(cuda_device, fmt, dtype):
    """An output that starts 16 bytes past a 32-byte boundary takes other stores."""
    c, s = moe_b200.quantize_fp4(rows(131, 352, torch.bfloat16, 41), fmt)
    want = moe_b200.dequantize_fp4(c, s, fmt, dtype=dtype)
    n = 16 // want.element_size()
    buf = torch.full((131 * 352 + 2 * n,), 9.0, device="cuda", dtype=dtype)
    out = buf[n:-n].view(131, 352)
    assert out.data_ptr() % 32 == 16
    moe_b200.dequantize_fp4(c, s, fmt, dtype=dtype, out=out)
    assert torch.equal(out, want) and (buf[:n] == 9).all() and (buf[-n:] == 9).all()
