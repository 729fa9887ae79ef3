"""Cases and plain forms of the operators around the MoE layer.

Four operators, all of them steps a serving program makes next to ``moe_b200.run``:

* ``norm``    residual addition + RMS norm + e4m3 output with 1x128 scales (the
  layer's ``hidden_states`` / ``hidden_states_scale``) and the normed rows;
* ``route``   routing to experts: softmax or sigmoid scores, selection bias,
  groups, top-k, renormalised weights;
* ``quant4``  microscaled 4-bit quantisation, returned as the values it stands for;
* ``linear4`` product of 16-bit activations, quantised on the way, with a weight
  held in microscaled 4 bits.

``run`` computes them in elementary torch operations, or with ``own = True``
through the package's entry points.
"""
import math
import os
import sys

import torch

own = False

_LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)     # magnitudes of e2m1
_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BLOCK = {"mxfp4": 32, "nvfp4": 16}


def _package():
    if "moe_b200" not in sys.modules:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                        "mlsys26-flashinfer-moe_b200"))
    import moe_b200
    return moe_b200


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # one decode token entering the layer: launch latency
        dict(name="norm_t1_h7168", op="norm", t=1, h=7168, x="bf16", residual="same", weight="bf16"),
        # an odd batch with the residual stream kept in fp32
        dict(name="norm_t901_h2048", op="norm", t=901, h=2048, x="fp16", residual="fp32", weight="fp32"),
        # a prefill chunk of the benchmark's layer
        dict(name="norm_t8192_h7168", op="norm", t=8192, h=7168, x="bf16", residual="same", weight="bf16"),
        # decode batch with the benchmark's grouped sigmoid routing
        dict(name="route_sigmoid_t64_e256", op="route", t=64, e=256, k=8, score="sigmoid", bias=True, n_group=8,
             topk_group=4, group_score="top2", renorm=True, x="fp32"),
        # odd batch and expert count, groups by their best expert, weights not renormalised
        dict(name="route_softmax_t901_e72", op="route", t=901, e=72, k=6, score="softmax", bias=False, n_group=8,
             topk_group=3, group_score="max", renorm=False, x="bf16"),
        # prefill over many experts, no groups, a bias that balances the load
        dict(name="route_softmax_t16384_e512", op="route", t=16384, e=512, k=8, score="softmax", bias=True, n_group=1,
             topk_group=1, group_score="max", renorm=True, x="fp32"),
        # a few decode rows
        dict(name="quant4_mx_t33_k2048", op="quant4", t=33, k=2048, fmt="mxfp4", x="fp16"),
        # prefill activations, or a weight being laid out
        dict(name="quant4_nv_t4096_k7168", op="quant4", t=4096, k=7168, fmt="nvfp4", x="bf16"),
        # one decode token through an expert-sized gate/up projection: weight bandwidth and latency
        dict(name="linear4_nv_t1_k7168_n4096", op="linear4", t=1, k=7168, n=4096, fmt="nvfp4", x="bf16"),
        # a decode batch through the down projection
        dict(name="linear4_mx_t64_k2048_n7168", op="linear4", t=64, k=2048, n=7168, fmt="mxfp4", x="bf16"),
        # ragged in every direction
        dict(name="linear4_nv_t901_k480_n1000", op="linear4", t=901, k=480, n=1000, fmt="nvfp4", x="fp16"),
        # a prefill chunk through the gate/up projection
        dict(name="linear4_nv_t8192_k7168_n4096", op="linear4", t=8192, k=7168, n=4096, fmt="nvfp4", x="bf16"),
    ]


def _spread(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "route", "quant4", "linear4"])
    x = rng.choice(["bf16", "fp16"])
    if op == "norm":
        return dict(op=op, t=_spread(rng, 1, 8192), h=128 * _spread(rng, 1, 56), x=x,
                    residual=rng.choice(["none", "same", "fp32"]), weight=rng.choice([x, "fp32"]))
    if op == "route":
        e = _spread(rng, 8, 512)
        groups = [g for g in range(1, 17) if e % g == 0 and e // g >= 2]
        n_group = rng.choice(groups)
        topk_group = rng.randint(1, n_group)
        return dict(op=op, t=_spread(rng, 1, 16384), e=e, k=rng.randint(1, min(16, topk_group * (e // n_group))),
                    score=rng.choice(["softmax", "sigmoid"]), bias=rng.random() < 0.5, n_group=n_group,
                    topk_group=topk_group, group_score=rng.choice(["top2", "max"]), renorm=rng.random() < 0.5,
                    x=rng.choice(["bf16", "fp16", "fp32"]))
    fmt = rng.choice(["mxfp4", "nvfp4"])
    k = 32 * _spread(rng, 1, 224)
    if op == "quant4":
        return dict(op=op, t=_spread(rng, 1, 4096), k=k, fmt=fmt, x=rng.choice(["bf16", "fp16", "fp32"]))
    return dict(op=op, t=_spread(rng, 1, 8192), k=k, n=_spread(rng, 1, 4096), fmt=fmt, x=x)


def work(case):
    """Bytes every operand crosses the memory bus once, and multiply-adds counted as two."""
    c = case
    if c["op"] == "norm":
        n, xb = c["t"] * c["h"], _DTYPES[c["x"]].itemsize
        rb = {"none": 0, "same": xb, "fp32": 4}[c["residual"]]
        return dict(bytes=n * (xb + 2 * rb + xb + 1) + 4 * n // 128 + c["h"] * _DTYPES[c["weight"]].itemsize,
                    flops=8 * n)
    if c["op"] == "route":
        n = c["t"] * c["e"]
        return dict(bytes=n * _DTYPES[c["x"]].itemsize + 8 * c["t"] * c["k"] + (4 * c["e"] if c["bias"] else 0),
                    flops=4 * n)
    blk = _BLOCK[c["fmt"]]
    if c["op"] == "quant4":
        n = c["t"] * c["k"]
        return dict(bytes=n * (_DTYPES[c["x"]].itemsize + 2), flops=4 * n)
    t, k, n = c["t"], c["k"], c["n"]
    return dict(bytes=t * k * 2 + n * k // 2 + n * (k // blk) + t * n * 2, flops=2 * t * k * n)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _e2m1(v):
    """Index of the nearest e2m1 magnitude, ties to the even index."""
    return ((v > 0.25).to(torch.uint8) + (v >= 0.75) + (v > 1.25) + (v >= 1.75) + (v > 2.5) + (v >= 3.5) + (v > 5.0))


def _plain_quant4(x, fmt, g):
    """Rows -> (4-bit codes one per byte, scale codes, values without the tensor scale).

    Quotients are taken in 64 bits: a tensor scale that is a ratio of small numbers puts
    many of them on or next to the border of two codes."""
    t, k = x.shape
    b = x.double().reshape(t, -1, _BLOCK[fmt])
    amax = b.abs().amax(dim=-1)
    if fmt == "mxfp4":       # power-of-two scale that puts amax into [4, 8)
        e = ((amax.float().view(torch.int32) >> 23) - 129).clamp(-127, 127)
        s, codes = torch.ldexp(torch.ones_like(amax), e), (e + 127).to(torch.uint8)
        d = s
    else:                    # e4m3 scale of amax / 6, at least its smallest value for a non-zero block
        s = (amax / (6.0 * g.double())).clamp(max=448.0)
        i = torch.bucketize(s, _e4m3_borders(x.device))
        codes = torch.where(amax > 0, i.clamp(min=1), torch.zeros_like(i)).to(torch.uint8)
        s = codes.view(torch.float8_e4m3fn).double()
        d = s * g.double()
    q = torch.where(d[..., None] > 0, b.abs() / d[..., None], torch.zeros_like(b))
    i = _e2m1(q)
    levels = torch.tensor(_LEVELS, device=x.device, dtype=torch.float64)
    v = torch.where(b < 0, -levels[i.long()], levels[i.long()]) * s[..., None]
    return (i + 8 * torch.signbit(b)).reshape(t, k), codes, v.float().reshape(t, k)


def _e4m3_borders(device):
    """Borders of neighbouring non-negative e4m3 values; the border itself goes to the even code."""
    v = torch.arange(127, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn).double()
    mid = (v[1:] + v[:-1]) / 2
    even_above = torch.arange(1, 127, device=device) % 2 == 0
    return torch.where(even_above, torch.nextafter(mid, torch.zeros_like(mid)), mid)


def _blocked(scales):
    """Row-major scales [R, B] -> [R/128, B/4, 32, 4, 4], rows and columns filled up with 0."""
    r, b = scales.shape
    rb, cb = (r + 127) // 128, (b + 3) // 4
    full = torch.zeros(rb * 128, cb * 4, dtype=torch.uint8, device=scales.device)
    full[:r, :b] = scales
    return full.view(rb, 4, 32, cb, 4).permute(0, 3, 2, 1, 4).contiguous()


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    c = dict(case)
    dt = _DTYPES[c["x"]]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    if c["op"] == "norm":
        c["in"] = normal(c["t"], c["h"]).to(dt)
        c["w"] = (1.0 + 0.1 * normal(c["h"])).to(_DTYPES[c["weight"]])
        c["res"] = None if c["residual"] == "none" else \
            (2.0 * normal(c["t"], c["h"])).to(dt if c["residual"] == "same" else torch.float32)
    elif c["op"] == "route":
        c["in"] = normal(c["t"], c["e"]).to(dt)
        c["b"] = 0.1 * normal(c["e"]) if c["bias"] else None
    else:
        c["in"] = normal(c["t"], c["k"]).to(dt)
        # a calibrated tensor scale: the largest activation seen was 7.3
        c["gx"] = torch.full((1,), 7.3 / (6.0 * 448.0), device="cuda") if c["fmt"] == "nvfp4" else None
        if c["op"] == "linear4":
            w = (0.02 * normal(c["n"], c["k"])).to(torch.bfloat16)
            c["gw"] = (w.abs().amax().float() / (6.0 * 448.0)).reshape(1) if c["fmt"] == "nvfp4" else None
            i, c["w_scale_rows"], _ = _plain_quant4(w, c["fmt"], c["gw"])
            c["w_codes"] = (i[:, 0::2] + 16 * i[:, 1::2]).to(torch.uint8)   # even columns in the low half of a byte
            c["w_scales"] = _blocked(c["w_scale_rows"])
    return c


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(state):
    s = state
    if own:
        m = _package()
        if s["op"] == "norm":
            q, scale, normed, res = m.rms_norm_quantize_1x128(s["in"], s["w"], 1e-6, residual=s["res"], normed=True)
            return [q, scale, normed] + ([] if res is None else [res])
        if s["op"] == "route":
            return list(m.route_topk(s["in"], s["k"], bias=s["b"], score=s["score"], n_group=s["n_group"],
                                     topk_group=s["topk_group"], group_score=s["group_score"],
                                     renormalize=s["renorm"], routed_scaling_factor=2.5))
        if s["op"] == "quant4":
            codes, scales = m.quantize_fp4(s["in"], s["fmt"], global_scale=s["gx"])
            return m.dequantize_fp4(codes, scales, s["fmt"], global_scale=s["gx"], dtype=torch.bfloat16)
        return m.linear_fp4(s["in"], s["w_codes"], s["w_scales"], s["fmt"], x_global_scale=s["gx"],
                            w_global_scale=s["gw"])
    return {"norm": _norm, "route": _route, "quant4": _quant4, "linear4": _linear4}[s["op"]](s)


def _norm(s):
    h = s["in"].float()
    if s["res"] is not None:
        h = h + s["res"].float()
    y = h * torch.rsqrt(h.square().mean(dim=-1, keepdim=True) + 1e-6) * s["w"].float()
    b = y.view(y.shape[0], -1, 128)
    scale = (b.abs().amax(dim=-1) * (1.0 / 448.0)).clamp(min=1e-12)
    q = (b / scale[..., None]).view(y.shape).to(torch.float8_e4m3fn)
    out = [q, scale.t().contiguous(), y.to(s["in"].dtype)]
    return out if s["res"] is None else out + [h.to(s["res"].dtype)]


def _route(s):
    x = s["in"].double()     # 64 bits: scores of neighbouring experts are compared
    t, e, g, k = s["t"], s["e"], s["n_group"], s["k"]
    p = torch.softmax(x, dim=-1) if s["score"] == "softmax" else torch.sigmoid(x)
    choice = p if s["b"] is None else p + s["b"].double()
    if g > 1:
        per = choice.view(t, g, e // g)
        rank = per.amax(dim=-1) if s["group_score"] == "max" else per.sort(dim=-1, descending=True)[0][..., :2].sum(-1)
        best = rank.sort(dim=-1, descending=True, stable=True)[1][:, :s["topk_group"]]
        keep = torch.zeros(t, g, dtype=torch.bool, device=x.device).scatter_(1, best, True)
        choice = torch.where(keep[..., None], per, torch.full_like(per, -math.inf)).view(t, e)
    idx = choice.sort(dim=-1, descending=True, stable=True)[1][:, :k]
    w = p.gather(1, idx)
    if s["renorm"]:
        w = w / (w.sum(dim=-1, keepdim=True) + 1e-20)
    return [idx.to(torch.int32), (w * 2.5).float()]


def _quant4(s):
    v = _plain_quant4(s["in"], s["fmt"], s["gx"])[2]
    return (v if s["gx"] is None else v * s["gx"]).to(torch.bfloat16)


def _linear4(s):
    levels = torch.tensor(_LEVELS + tuple(-v for v in _LEVELS), device=s["in"].device)
    c = s["w_codes"]
    w = levels[torch.stack((c & 15, c >> 4), dim=-1).long()].view(s["n"], -1, _BLOCK[s["fmt"]])
    if s["fmt"] == "mxfp4":
        ws = torch.ldexp(torch.ones_like(s["w_scale_rows"], dtype=torch.float32), s["w_scale_rows"].int() - 127)
    else:
        ws = s["w_scale_rows"].view(torch.float8_e4m3fn).float()
    w = (w * ws[..., None]).view(s["n"], s["k"])
    y = _plain_quant4(s["in"], s["fmt"], s["gx"])[2] @ w.t()
    if s["fmt"] == "nvfp4":
        y = y * (s["gx"] * s["gw"])
    return y.to(s["in"].dtype)


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------

def _grid(v, mantissa, emin, top):
    """Nearest value (ties to even) of a float with `mantissa` fraction bits, smallest normal exponent `emin`."""
    e = torch.frexp(v)[1].double() - 1
    step = torch.exp2(e.clamp(min=emin) - mantissa)
    return (torch.round(v / step) * step).clamp(-top, top)


def _exact_quant4(x, fmt, g):
    b = x.double().view(x.shape[0], -1, _BLOCK[fmt])
    top = b.abs().max(dim=-1, keepdim=True)[0]
    if fmt == "mxfp4":
        s = torch.exp2((torch.frexp(top)[1].double() - 3).clamp(-127, 127))
    else:
        s = _grid(top / (6 * g.double()), 3, -6, 448.0)
        s = torch.where((top > 0) & (s == 0), s + 2.0 ** -9, s) * g.double()
    q = _grid(torch.where(s > 0, b / s, torch.zeros_like(b)), 1, 0, 6.0)
    return (q * s).view(x.shape)


def exact(case, seed):
    s = prepare(case, seed)
    x = s["in"].double()
    if s["op"] == "norm":
        if s["res"] is not None:
            x = x + s["res"].double()
        y = x / torch.sqrt((x * x).sum(dim=-1, keepdim=True) / s["h"] + 1e-6) * s["w"].double()
        top = torch.linalg.vector_norm(y.view(s["t"], -1, 128), ord=math.inf, dim=-1) / 448.0
        q = _grid(y.view(s["t"], -1, 128) / top[..., None], 3, -6, 448.0).view(s["t"], s["h"])
        return [q, top.t(), y] + ([] if s["res"] is None else [x])
    if s["op"] == "route":
        z = x - x.max(dim=-1, keepdim=True)[0]
        p = torch.exp(z) / torch.exp(z).sum(-1, keepdim=True) if s["score"] == "softmax" else 1 / (1 + torch.exp(-x))
        c = p if s["b"] is None else p + s["b"].double()
        if s["n_group"] > 1:
            per = c.view(s["t"], s["n_group"], -1)
            rank = per.topk(2 if s["group_score"] == "top2" else 1, dim=-1)[0].sum(-1)
            order = torch.arange(s["n_group"], device=x.device)
            ahead = (rank[:, None, :] > rank[:, :, None]) | \
                ((rank[:, None, :] == rank[:, :, None]) & (order[None, None, :] < order[None, :, None]))
            c = per.masked_fill((ahead.sum(-1) >= s["topk_group"])[..., None], -math.inf).view(s["t"], -1)
        picked = []
        for _ in range(s["k"]):
            at = (c == c.max(dim=-1, keepdim=True)[0]).double().argmax(dim=-1, keepdim=True)   # the lowest of equals
            picked.append(p.gather(1, at))
            c = c.scatter(1, at, -math.inf)
        w = torch.cat(picked, dim=1)
        return [None, 2.5 * (w / (w.sum(-1, keepdim=True) + 1e-20) if s["renorm"] else w)]
    if s["op"] == "quant4":
        return _exact_quant4(s["in"], s["fmt"], s["gx"])
    c = torch.stack((s["w_codes"] % 16, s["w_codes"] // 16), dim=-1).view(s["n"], -1).double()
    m = c % 8
    w = torch.where(m < 2, m / 2, (1 + (m % 2) / 2) * torch.exp2(torch.div(m, 2, rounding_mode="floor") - 1))
    w = torch.where(c >= 8, -w, w).view(s["n"], -1, _BLOCK[s["fmt"]])
    r = s["w_scale_rows"].double()
    if s["fmt"] == "mxfp4":
        r = torch.exp2(r - 127)
    else:
        f = torch.div(r, 8, rounding_mode="floor")
        r = torch.where(f == 0, (r % 8) * 2.0 ** -9, (1 + (r % 8) / 8) * torch.exp2(f - 7)) * s["gw"].double()
    return _exact_quant4(s["in"], s["fmt"], s["gx"]) @ (w * r[..., None]).view(s["n"], -1).t()
