"""Workloads of the block-scaled 8-bit floating-point operators: what each call reads, writes and computes.

Three operators of a linear layer whose activations and weights are held as e4m3 codes with one fp32 scale for each
block of 128 channels (activations: per row and block; weights: per 128 x 128 block):

    rms    residual addition + root-mean-square norm of a row, written as codes and block scales
    quant  a row (or value * silu(gate) of a gated MLP's first product) as codes and block scales
    gemm   the product of such codes with such weights, bias, rounded to bf16 / f16 / f32

A case is a dict of sizes and types. `run` computes it with elementary torch operations, or, where `own` is set,
through the package's public calls.
"""

import math

import torch

own = False

GROUP = 128      # channels that share one scale
TOP = 448.0      # largest finite e4m3 value
TINY = 2.0 ** -126  # smallest scale: below it 1 / scale would not be finite
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}

_gpu = None


def _context():
    """The one context a program opens."""
    global _gpu
    if _gpu is None:
        from h3metal_b200.gpu import Gpu
        _gpu = Gpu()
    return _gpu


# ---- cases ----------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one token of a decoding step: its norm is all latency
        {"name": "rms 1x3840", "op": "rms", "m": 1, "d": 3840, "x": "bf16", "y": "bf16"},
        # a 1024 x 1024 image's tokens in the 6B block
        {"name": "rms 4608x3840", "op": "rms", "m": 4608, "d": 3840, "x": "bf16", "y": "bf16"},
        # a 2048 x 2048 image in the 33B block, fp32 residual stream with a bf16 product added
        {"name": "rms 17408x6144 f32", "op": "rms", "m": 17408, "d": 6144, "x": "f32", "y": "bf16"},
        # the gated MLP's activation for a handful of tokens
        {"name": "quant 7x10240 gated", "op": "quant", "m": 7, "d": 10240, "x": "bf16", "gated": True},
        # a padded batch of a width that is no multiple of the block, plain rows
        {"name": "quant 1031x1000", "op": "quant", "m": 1031, "d": 1000, "x": "f16", "gated": False},
        # the gated MLP's activation of the 33B block
        {"name": "quant 17408x16384 gated", "op": "quant", "m": 17408, "d": 16384, "x": "bf16", "gated": True},
        # decoding: one token against the 6B block's first product
        {"name": "gemm 1x11520x3840", "op": "gemm", "m": 1, "n": 11520, "k": 3840, "out": "bf16", "bias": False},
        # sixteen sequences decoded together, the 6B block's last product
        {"name": "gemm 16x3840x10240", "op": "gemm", "m": 16, "n": 3840, "k": 10240, "out": "bf16", "bias": True},
        # odd in every size, fp32 results
        {"name": "gemm 129x771x1000 f32", "op": "gemm", "m": 129, "n": 771, "k": 1000, "out": "f32", "bias": True},
        # a short prompt
        {"name": "gemm 512x20480x3840", "op": "gemm", "m": 512, "n": 20480, "k": 3840, "out": "bf16", "bias": False},
        # the 6B block at 1024 x 1024
        {"name": "gemm 4608x11520x3840", "op": "gemm", "m": 4608, "n": 11520, "k": 3840, "out": "bf16", "bias": True},
        # the 33B block at 2048 x 2048
        {"name": "gemm 17408x18432x6144", "op": "gemm", "m": 17408, "n": 18432, "k": 6144, "out": "bf16", "bias": False},
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A channel count: mostly whole blocks or whole 16s, now and then any number."""
    step = rng.choice([128, 128, 64, 16, 1])
    return max(lo, min(hi, _spread(rng, lo, hi) // step * step))


def draw(rng):
    op = rng.choice(["rms", "quant", "gemm", "gemm"])
    if op == "rms":
        d = _width(rng, 64, 16384)
        m = _spread(rng, 1, min(66560, 17408 * 6144 // d))
        x = rng.choice(["bf16", "bf16", "f16", "f32"])
        return {"op": op, "m": m, "d": d, "x": x, "y": rng.choice(["none", x, "bf16"])}
    if op == "quant":
        d = _width(rng, 64, 32768)
        m = _spread(rng, 1, min(66560, 17408 * 8192 // d))
        return {"op": op, "m": m, "d": d, "x": rng.choice(["bf16", "bf16", "f16", "f32"]), "gated": rng.random() < 0.5}
    k = _width(rng, 64, 16384)
    n = _width(rng, 16, min(32768, 32768 * 6144 // k))
    m = _spread(rng, 1, min(17408, 17408 * 18432 * 6144 // (n * k)))
    return {"op": op, "m": m, "n": n, "k": k, "out": rng.choice(["bf16", "bf16", "f16", "f32"]), "bias": rng.random() < 0.5}


# ---- what a program holds before the call ---------------------------------------------------------------------------
def _groups(k):
    return -(-k // GROUP)


def _stride(k):
    """Row stride of codes: whole 16-byte pieces."""
    return -(-k // 16) * 16


def _draw_rows(gen, m, d, dtype):
    """Rows as they come out of a product: N(0, 1) with a few channels twenty times as large."""
    x = torch.randn(m, d, generator=gen, device="cuda")
    loud = torch.randperm(d, generator=gen, device="cuda")[:max(1, d // 500)]
    x[:, loud] *= 20.0
    return x.to(dtype)


def _coded(x, rows):
    """e4m3 codes and scales of blocks of `rows` x 128 values: codes [n][stride(k)], scales [ceil(n / rows)][ceil(k / 128)]."""
    n, k = x.shape
    codes = torch.zeros(n, _stride(k), device="cuda", dtype=torch.float8_e4m3fn)
    scales = torch.empty(-(-n // rows), _groups(k), device="cuda")
    for g in range(scales.shape[1]):
        part = x[:, g * GROUP:(g + 1) * GROUP]
        top = part.abs().amax(1)
        if rows > 1:
            top = torch.nn.functional.pad(top, (0, -n % rows)).reshape(-1, rows).amax(1)
        s = torch.where(top > 0, top / TOP, torch.ones_like(top))
        scales[:, g] = s
        codes[:, g * GROUP:g * GROUP + part.shape[1]] = \
            (part / s.repeat_interleave(rows)[:n, None]).clamp(-TOP, TOP).to(torch.float8_e4m3fn)
    return codes, scales


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    m = case["m"]
    st = dict(case)
    if case["op"] == "gemm":
        n, k = case["n"], case["k"]
        st["a"], sa = _coded(_draw_rows(gen, m, k, torch.float32), 1)
        st["sa"] = sa.T.contiguous()  # a block's scales of all rows side by side
        st["w"], st["sw"] = _coded(torch.randn(n, k, generator=gen, device="cuda") * 0.02, GROUP)
        st["b"] = torch.randn(n, generator=gen, device="cuda") * 0.1 if case["bias"] else None
        st["c"] = torch.empty(m, n, device="cuda", dtype=TYPES[case["out"]])
    else:
        d = case["d"]
        wide = 2 * d if case.get("gated") else d
        size = {"f32": 4}.get(case["x"], 2)
        pad = -wide % (16 // size)  # rows start on 16-byte boundaries
        st["rows"] = _draw_rows(gen, m, wide + pad, TYPES[case["x"]])
        st["codes"] = torch.zeros(m, _stride(d), device="cuda", dtype=torch.float8_e4m3fn)
        st["scales"] = torch.empty(_groups(d), m, device="cuda")
        if case["op"] == "rms":
            st["gain"] = 1 + 0.1 * torch.randn(d, generator=gen, device="cuda")
            st["sum"] = torch.empty_like(st["rows"])
            if case["y"] != "none":
                st["add"] = _draw_rows(gen, m, d + -d % (4 if case["y"] == "f32" else 8), TYPES[case["y"]])
    if own:  # the views of these buffers that a program makes once, where it allocates them
        g = _context()
        st["g"] = g
        for key in ("a", "sa", "w", "sw", "b", "c", "rows", "codes", "scales", "gain", "sum", "add"):
            if st.get(key) is not None:
                st["v_" + key] = g.wrap(st[key])
        if case["op"] == "gemm":
            from h3metal_b200.ops import QWeight
            st["v_weight"] = QWeight("f8", st["v_w"], st["v_sw"], case["n"], case["k"], bias=st.get("v_b"))
    return st


# ---- one pass -------------------------------------------------------------------------------------------------------
def _encode(v, st):
    """The rows v (fp32) as codes and scales in st's buffers."""
    m, d = v.shape
    full = torch.nn.functional.pad(v, (0, -d % GROUP)).reshape(m, -1, GROUP)
    top = full.abs().amax(2)
    s = torch.where(top > 0, (top / TOP).clamp_min(TINY), torch.ones_like(top))
    st["scales"].copy_(s.T)
    st["codes"][:, :d] = (full / s[:, :, None]).clamp(-TOP, TOP).reshape(m, -1)[:, :d].to(torch.float8_e4m3fn)
    return st["codes"][:, :d], st["scales"]


EPS = 1e-6  # added to the mean square before its root


def run(st):
    op = st["op"]
    if own:
        from h3metal_b200 import ops
        g, m = st["g"], st["m"]
        if op == "gemm":
            ops.gemm_f8(g, st["v_a"], st["v_weight"], st["v_c"], m, sa=st["v_sa"])
            return st["c"]
        d, wide = st["d"], st["rows"].shape[1]
        if op == "quant":
            ops.quant_f8(g, st["v_rows"], st["v_codes"], st["v_scales"], m, d, swiglu=st["gated"], x_stride=wide)
            return {"codes": st["codes"][:, :d], "scales": st["scales"]}
        if "add" in st:
            ops.rms_f8(g, st["v_rows"], st["v_gain"], st["v_codes"], st["v_scales"], m, d, eps=EPS, x_stride=wide,
                       y=st["v_add"], y_stride=st["add"].shape[1], res=st["v_sum"], res_stride=wide)
            return {"codes": st["codes"][:, :d], "scales": st["scales"], "sum": st["sum"][:, :d]}
        ops.rms_f8(g, st["v_rows"], st["v_gain"], st["v_codes"], st["v_scales"], m, d, eps=EPS, x_stride=wide)
        return {"codes": st["codes"][:, :d], "scales": st["scales"]}

    if op == "gemm":
        n, k = st["n"], st["k"]
        spread = lambda s: s.repeat_interleave(GROUP, dim=1)[:, :k]  # noqa: E731
        a = st["a"][:, :k].float() * spread(st["sa"].T)
        w = st["w"][:, :k].float() * spread(st["sw"]).repeat_interleave(GROUP, dim=0)[:n]
        v = a @ w.T
        if st["b"] is not None:
            v = v + st["b"]
        st["c"].copy_(v)
        return st["c"]
    d = st["d"]
    if op == "quant":
        v = st["rows"][:, :d].float()
        if st["gated"]:
            gate = st["rows"][:, d:2 * d].float()
            v = v * (gate / (1 + torch.exp(-gate)))
        codes, scales = _encode(v, st)
        return {"codes": codes, "scales": scales}
    v = st["rows"][:, :d].float()
    if "add" in st:
        st["sum"][:, :d] = v + st["add"][:, :d].float()  # the stream is what is kept, and what is normed
        v = st["sum"][:, :d].float()
    v = v * torch.rsqrt((v * v).mean(1, keepdim=True) + EPS) * st["gain"]
    codes, scales = _encode(v, st)
    if "add" in st:
        return {"codes": codes, "scales": scales, "sum": st["sum"][:, :d]}
    return {"codes": codes, "scales": scales}


# ---- what a pass cannot do without ----------------------------------------------------------------------------------
def _size(name):
    return {"none": 0, "f32": 4}.get(name, 2)


def work(case):
    m = case["m"]
    if case["op"] == "gemm":
        n, k = case["n"], case["k"]
        scales = 4 * (m * _groups(k) + _groups(n) * _groups(k)) + (4 * n if case["bias"] else 0)
        return {"bytes": m * k + n * k + scales + m * n * _size(case["out"]), "flops": 2 * m * n * k}
    d = case["d"]
    out = m * d + 4 * m * _groups(d)
    if case["op"] == "quant":
        wide = 2 if case["gated"] else 1
        return {"bytes": m * d * wide * _size(case["x"]) + out, "flops": (8 if case["gated"] else 3) * m * d}
    stream = m * d * _size(case["x"])
    added = m * d * _size(case["y"]) + (stream if case["y"] != "none" else 0)
    return {"bytes": stream + added + 4 * d + out, "flops": 8 * m * d}


# ---- the definition in 64 bits --------------------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "gemm":
        total = torch.zeros(case["m"], case["n"], dtype=torch.float64, device="cuda")
        for g in range(_groups(case["k"])):
            cols = slice(g * GROUP, min(case["k"], (g + 1) * GROUP))
            per_out = st["sw"][:, g].double()[torch.arange(case["n"], device="cuda") // GROUP]
            left = st["a"][:, cols].double() * st["sa"][g].double()[:, None]
            total.addmm_(left, (st["w"][:, cols].double() * per_out[:, None]).T)
        return total if st["b"] is None else total + st["b"].double()
    d = case["d"]
    codes = torch.empty(case["m"], d, dtype=torch.float64, device="cuda")
    scales = torch.empty(_groups(d), case["m"], dtype=torch.float64, device="cuda")
    kept = torch.empty(case["m"], d, dtype=torch.float64, device="cuda") if "add" in st else None
    for r in range(0, case["m"], 1024):
        rows = slice(r, min(case["m"], r + 1024))
        v = st["rows"][rows, :d].double()
        if case["op"] == "quant" and case["gated"]:
            v = v * torch.nn.functional.silu(st["rows"][rows, d:2 * d].double())
        if case["op"] == "rms":
            if kept is not None:
                kept[rows] = v + st["add"][rows, :d].double()
                v = kept[rows].to(TYPES[case["x"]]).double()  # the stream's own rounding is part of the definition
            v = v / (v.square().sum(1, keepdim=True) / d + EPS).sqrt() * st["gain"].double()
        for g in range(_groups(d)):
            part = v[:, g * GROUP:(g + 1) * GROUP]
            s = part.abs().max(1).values / TOP
            s = torch.where(s > 0, s.clamp(min=TINY), torch.ones_like(s))
            scales[g, rows] = s
            codes[rows, g * GROUP:(g + 1) * GROUP] = part / s[:, None]  # before its rounding to eight bits
    out = {"codes": codes, "scales": scales}
    if kept is not None:
        out["sum"] = kept
    return out
