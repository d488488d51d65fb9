"""Measured cases of the 4-bit floating point operators and the rotary embedding.

Operators
  quantize   a bf16 matrix to 4-bit floating point in groups (``mxfp4``: 32
             values share an E8M0 scale; ``nvfp4``: 16 values share an E4M3
             scale, times one scale for the whole tensor) and back to values
  linear     bf16 activations times an exactly dequantized 4-bit weight
  linear4    activations quantized to the weight's 4-bit form in the call,
             then the product of the two quantized operands
  rotary     rotary positions on the heads of a projection: half or
             interleaved pairs, the leading part of each head or all of it,
             one or several position axes, frequencies shared by the heads or
             one row for each

``own`` selects the framework's calls; otherwise ``run`` computes the plain
forms from elementary torch operations in 32 bits (angles in 64).
"""

from __future__ import annotations

import math
import os
import sys

import torch

own = False

E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)  # values of the 3-bit magnitudes
GROUP = {"mxfp4": 32, "nvfp4": 16}


def _ltxq():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ltx-2-mlx_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import ltxq

    return ltxq


# ---------------------------------------------------------------- cases


def listed():
    return [
        # activations of one audio clip's attention, an odd row count and a ragged width
        {"name": "quantize_nvfp4_201x2080", "op": "quantize", "fmt": "nvfp4", "rows": 201, "k": 2080, "std": 1.0, "g": 1.0},
        # the rows of a long video and of its unconditional copy in front of a projection
        {"name": "quantize_mxfp4_16384x4096", "op": "quantize", "fmt": "mxfp4", "rows": 16384, "k": 4096, "std": 1.0, "g": 1.0},
        # one token through the widest projection: weight bandwidth and latency
        {"name": "linear_nvfp4_1x4096x16384", "op": "linear", "fmt": "nvfp4", "m": 1, "k": 4096, "n": 16384},
        # the audio stream's tokens through its feed-forward input
        {"name": "linear_mxfp4_201x2048x8192", "op": "linear", "fmt": "mxfp4", "m": 201, "k": 2048, "n": 8192},
        # a short video's attention projection
        {"name": "linear_mxfp4_3456x4096x4096", "op": "linear", "fmt": "mxfp4", "m": 3456, "k": 4096, "n": 4096},
        # a few tokens, odd counts on every axis
        {"name": "linear4_nvfp4_9x2080x1048", "op": "linear4", "fmt": "nvfp4", "m": 9, "k": 2080, "n": 1048},
        # the audio stream's cross attention projection
        {"name": "linear4_mxfp4_751x2048x2048", "op": "linear4", "fmt": "mxfp4", "m": 751, "k": 2048, "n": 2048},
        # a long video's feed-forward output: the largest product
        {"name": "linear4_nvfp4_9216x16384x4096", "op": "linear4", "fmt": "nvfp4", "m": 9216, "k": 16384, "n": 4096},
        # the next token of two sequences, far into a long context
        {"name": "rotary_half_2x1x32x128", "op": "rotary", "b": 2, "t": 1, "heads": 32, "d": 128, "rot": 128, "layout": "half",
         "dtype": "bfloat16", "axes": 1, "per_head": False, "far": 100000, "factor": 8.0, "inverse": False},
        # the latent tokens of a long video: three position axes, a row of frequencies for each head
        {"name": "rotary_half_1x9216x32x128_axes", "op": "rotary", "b": 1, "t": 9216, "heads": 32, "d": 128, "rot": 128,
         "layout": "half", "dtype": "bfloat16", "axes": 3, "per_head": True, "far": 2048, "factor": 1.0, "inverse": False},
        # text rows, adjacent pairs, rotated whole
        {"name": "rotary_pairs_2x1024x32x64", "op": "rotary", "b": 2, "t": 1024, "heads": 32, "d": 64, "rot": 64,
         "layout": "interleaved", "dtype": "bfloat16", "axes": 1, "per_head": False, "far": 4096, "factor": 1.0, "inverse": False},
        # the gradient's rotation in fp32, part of an odd-sized head, positions of a very long context
        {"name": "rotary_part_back_3x1601x7x80_fp32", "op": "rotary", "b": 3, "t": 1601, "heads": 7, "d": 80, "rot": 36,
         "layout": "half", "dtype": "float32", "axes": 1, "per_head": False, "far": 2000000, "factor": 32.0, "inverse": True},
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("quantize", "linear", "linear4", "rotary"))
    fmt = rng.choice(("mxfp4", "nvfp4"))
    if op == "quantize":
        rows, k = _spread(rng, 1, 16384), 32 * _spread(rng, 2, 512)
        rows = max(1, min(rows, 16384 * 4096 // k))
        return {"op": op, "fmt": fmt, "rows": rows, "k": k, "std": rng.choice((1.0, 0.02)),
                "g": rng.choice((1.0, 0.015625)) if fmt == "nvfp4" else 1.0}
    if op in ("linear", "linear4"):
        m, k, n = _spread(rng, 1, 9216), 32 * _spread(rng, 2, 512), 8 * _spread(rng, 8, 2048)
        m = max(1, min(m, 9216 * 16384 * 4096 // (k * n)))
        return {"op": op, "fmt": fmt, "m": m, "k": k, "n": n}
    heads, d = rng.randint(1, 32), 2 * _spread(rng, 8, 128)
    b = rng.choice((1, 1, 2, 3))
    t = max(1, min(_spread(rng, 1, 9216), 9216 * 4096 // (b * heads * d)))
    return {"op": op, "b": b, "t": t, "heads": heads, "d": d, "rot": rng.choice((d, d, 2 * rng.randint(1, d // 2))),
            "layout": rng.choice(("half", "interleaved")), "dtype": rng.choice(("bfloat16", "bfloat16", "float32")),
            "axes": rng.choice((1, 1, 3)), "per_head": rng.random() < 0.3, "far": _spread(rng, 64, 2000000),
            "factor": rng.choice((1.0, 8.0, 32.0)), "inverse": rng.random() < 0.4}


# ---------------------------------------------------------------- inputs


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _pack(codes):
    """4-bit codes [R, L] -> uint32 words [R, L / 8], element 0 in the low bits."""
    c = codes.to(torch.uint8).view(codes.shape[0], -1, 2)
    return (c[..., 0] | (c[..., 1] << 4)).contiguous().view(torch.uint32)


def _frequencies(case):
    """Rotation per unit of position, float64: 10000^(-2i/rot), the slow ones stretched by ``factor`` with a
    linear ramp between 32 and 1 turns over an original length of 4096; [rot/2], or [heads, rot/2] where each
    head has its own part of one geometric series.  With them the position axis of each."""
    half = case["rot"] // 2
    count = half * (case["heads"] if case["per_head"] else 1)
    i = torch.arange(count, dtype=torch.float64)
    f = 10000.0 ** (-i / count)
    if case["factor"] != 1.0:
        turns = 4096 * f / (2 * math.pi)
        keep = ((turns - 1) / 31).clamp(0, 1)
        f = f * keep + f / case["factor"] * (1 - keep)
    shape = (case["heads"], half) if case["per_head"] else (half,)
    axes = (torch.arange(count) % case["axes"]).to(torch.int32).view(shape)
    return f.view(shape).cuda(), axes.cuda()


def prepare(case, seed):
    gen = _gen(seed)

    def normal(*shape, std=1.0, dtype=torch.bfloat16):
        return (torch.randn(*shape, generator=gen, device="cuda") * std).to(dtype)

    if case["op"] == "quantize":
        s = {"case": case, "x": normal(case["rows"], case["k"], std=case["std"])}
        if own:
            s["ltxq"] = _ltxq()
        return s
    if case["op"] in ("linear", "linear4"):
        fmt = case["fmt"]
        g = 0.015625 if fmt == "nvfp4" else 1.0
        codes, scales = _quantize(normal(case["n"], case["k"], std=0.02).float(), fmt, g)
        s = {"case": case, "x": normal(case["m"], case["k"]), "weight": _pack(codes), "scales": scales, "g": g}
        del codes
        if own:
            lin = _ltxq().QuantizedLinear(s["weight"], s["scales"], group_size=GROUP[fmt], bits=4, mode=fmt, global_scale=g)
            s["linear"] = lin.set_compute("fp4") if case["op"] == "linear4" else lin
        return s
    b, t, heads, d = case["b"], case["t"], case["heads"], case["d"]
    dtype = getattr(torch, case["dtype"])
    # the queries' columns of a fused projection's output: rows three times as long as the slice
    x = normal(b, t, 3 * heads * d, dtype=dtype)[..., :heads * d]
    f, axes = _frequencies(case)
    if case["axes"] == 1:  # consecutive positions up to `far`, another start for each sequence
        start = torch.randint(max(0, case["far"] - t) + 1, (b, 1), generator=gen, device="cuda")
        pos = start + torch.arange(t, device="cuda")
    else:  # coordinates within each axis, halves among them
        pos = torch.randint(0, 2 * case["far"], (b, case["axes"], t), generator=gen, device="cuda").float() / 2
    scale = 1.0 if case["factor"] == 1.0 else 0.1 * math.log(case["factor"]) + 1.0
    s = {"case": case, "x": x, "pos": pos, "freqs": f, "axes": axes, "scale": scale}
    if own:
        s["ltxq"] = _ltxq()
    return s


# ---------------------------------------------------------------- plain forms


def _exponent(v):
    """floor(log2 v) of positive values (0 gives a small number)."""
    return torch.frexp(v).exponent - 1


def _quantize(x, fmt, g):
    """x [R, L] fp32 -> codes [R, L] (sign in bit 3) and scale bytes [R, L / group]."""
    r, n = x.shape
    y = (x / g).view(r, -1, GROUP[fmt])
    amax = y.abs().amax(-1, keepdim=True)
    if fmt == "mxfp4":
        e = torch.where(amax > 0, _exponent(amax) - 2, -127).clamp(-127, 127)
        byte = e + 127
        q = torch.ldexp(y, -e)
    else:
        v = amax / 6
        e = _exponent(v).clamp(min=-6)
        s = (torch.round(torch.ldexp(v, 3 - e)) * torch.ldexp(torch.ones_like(v), e - 3)).clamp(max=448.0)
        e = torch.where(s > 0, _exponent(s), -6).clamp(min=-6)  # the rounding may have reached the next power
        units = torch.ldexp(s, 3 - e).int()  # 8..15, or below 8 in the smallest binade
        byte = torch.where(units < 8, units, (e + 7) * 8 + units - 8)
        q = torch.where(s > 0, y / s, 0.0)
    a = q.abs().clamp(max=6.0)
    # steps of 0.5 below 2, of 1 up to 4, of 2 up to 6
    code = torch.where(a < 2, torch.round(a * 2), torch.where(a < 4, 2 + torch.round(a), 4 + torch.round(a / 2)))
    code = code.int() + torch.where(y.signbit(), 8, 0)
    return code.view(r, n).to(torch.uint8), byte.view(r, -1).to(torch.uint8)


def _values(codes, scales, fmt, g):
    """The fp32 values of codes and scale bytes."""
    r, n = codes.shape
    c = codes.int()
    v = torch.tensor(E2M1, device=codes.device)[c & 7] * (1 - 2 * (c >> 3))
    b = scales.int()
    if fmt == "mxfp4":
        s = torch.ldexp(torch.ones_like(b, dtype=torch.float32), b - 127)
    else:
        s = torch.where(b < 8, b * 2.0 ** -9, torch.ldexp(1 + (b & 7) / 8.0, (b >> 3) - 7))
    return (v.view(r, -1, GROUP[fmt]) * s[..., None] * g).view(r, n)


def _unpack(words):
    b = words.view(torch.uint8)
    return torch.stack([b & 15, b >> 4], dim=-1).view(b.shape[0], -1)


def _rotary(x, pos, freqs, axes, heads, layout, scale, inverse):
    b, t, w = x.shape
    d = w // heads
    half = freqs.shape[-1]
    f = freqs.view(-1, half)  # [1 or heads, half]
    p = pos.double().view(b, -1, t).transpose(1, 2)  # [b, t, axes]
    a = p[:, :, axes.long().view(-1)].view(b, t, -1, half) * f
    cos, sin = (torch.cos(a) * scale).float(), (torch.sin(a) * scale).float()
    if inverse:
        sin = -sin
    y = x.float().reshape(b, t, heads, d).clone()
    if layout == "half":
        lo, hi = slice(0, half), slice(half, 2 * half)
    else:
        lo, hi = slice(0, 2 * half, 2), slice(1, 2 * half, 2)
    u, v = y[..., lo].clone(), y[..., hi].clone()
    y[..., lo] = u * cos - v * sin
    y[..., hi] = v * cos + u * sin
    return y.view(b, t, w).to(x.dtype)


# ---------------------------------------------------------------- one pass


def run(state):
    case = state["case"]
    op = case["op"]
    if own:
        if op == "quantize":
            q = state["ltxq"].FP4Tensor.quantize(state["x"], case["fmt"], global_scale=case["g"])
            return q.dequantize()
        if op in ("linear", "linear4"):
            return state["linear"](state["x"])
        return state["ltxq"].rotary(state["x"], state["pos"], state["freqs"], case["heads"], layout=case["layout"],
                                    axes=state["axes"] if case["axes"] > 1 else None, scale=state["scale"],
                                    inverse=case["inverse"])
    if op == "quantize":
        codes, scales = _quantize(state["x"].float(), case["fmt"], case["g"])
        return _values(codes, scales, case["fmt"], case["g"]).to(torch.bfloat16)
    if op == "rotary":
        return _rotary(state["x"], state["pos"], state["freqs"], state["axes"], case["heads"], case["layout"],
                       state["scale"], case["inverse"])
    x = state["x"].float()
    if op == "linear4":
        x = _values(*_quantize(x, case["fmt"], 1.0), case["fmt"], 1.0)
    w = _values(_unpack(state["weight"]), state["scales"], case["fmt"], state["g"])
    return (x @ w.t()).to(torch.bfloat16)


# ---------------------------------------------------------------- what a pass needs


def work(case):
    if case["op"] == "quantize":  # values in, codes and scales out; those in, values out
        n = case["rows"] * case["k"]
        packed = n / 2 + n / GROUP[case["fmt"]]
        return {"bytes": 2 * n + packed + packed + 2 * n, "flops": 4 * n}
    if case["op"] in ("linear", "linear4"):
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": 2 * m * k + n * k / 2 + n * k / GROUP[case["fmt"]] + 2 * m * n, "flops": 2 * m * n * k}
    rows = case["b"] * case["t"]
    size = 2 if case["dtype"] == "bfloat16" else 4
    pos = 8 if case["axes"] == 1 else 4 * case["axes"]
    freqs = case["rot"] // 2 * (case["heads"] if case["per_head"] else 1)
    return {"bytes": 2 * rows * case["heads"] * case["d"] * size + rows * pos + 8 * freqs, "flops": 3 * rows * case["heads"] * case["rot"]}


# ---------------------------------------------------------------- the definition in 64 bits


def _round_to_table(v, table):
    """Index of the entry of the ascending table that is nearest to v, a tie going to the even index."""
    mid = (table[1:] + table[:-1]) / 2
    below, upto = torch.searchsorted(mid, v, right=False), torch.searchsorted(mid, v, right=True)
    return torch.where(below == upto, below, below + below % 2)


def _exact_values(x, fmt, g):
    """Quantized and read back, in 64 bits: nearest entries of the tables of all E2M1 and scale values."""
    r, n = x.shape
    y = (x.double() / g).view(-1, GROUP[fmt])
    top = y.abs().amax(-1)
    if fmt == "mxfp4":  # the largest power of two with 4 * scale <= the largest magnitude
        powers = 2.0 ** torch.arange(-127, 128, dtype=torch.float64, device=x.device)
        s = powers[(torch.searchsorted(4 * powers, top, right=True) - 1).clamp(min=0)]
    else:
        i = torch.arange(127, dtype=torch.float64, device=x.device)
        table = torch.where(i < 8, i / 512, (1 + (i % 8) / 8) * 2.0 ** ((i // 8) - 7))
        s = table[_round_to_table(top / 6, table)]
    levels = torch.tensor(E2M1, dtype=torch.float64, device=x.device)
    step = torch.where(s > 0, s, 1.0)[:, None]
    v = levels[_round_to_table(y.abs() / step, levels)] * y.sign() * s[:, None] * g
    return v.view(r, n)


def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op == "quantize":
        return _exact_values(state["x"], case["fmt"], case["g"])
    if op == "rotary":
        b, t, heads, d = case["b"], case["t"], case["heads"], case["d"]
        half = case["rot"] // 2
        x = state["x"].double().reshape(b, t, heads, d)
        pos = state["pos"].double().view(b, case["axes"], t)
        angle = torch.zeros(b, t, heads, half, dtype=torch.float64, device=x.device)
        f, axes = state["freqs"].expand(heads, half), state["axes"].expand(heads, half)
        for k in range(case["axes"]):
            angle += pos[:, k, :, None, None] * torch.where(axes == k, f, 0.0)
        turn = torch.polar(torch.full_like(angle, state["scale"]), -angle if case["inverse"] else angle)
        head, rest = x[..., :2 * half], x[..., 2 * half:]
        if case["layout"] == "interleaved":
            z = torch.view_as_complex(head.reshape(b, t, heads, half, 2).contiguous()) * turn
            head = torch.view_as_real(z).reshape(b, t, heads, 2 * half)
        else:
            z = torch.complex(head[..., :half], head[..., half:]) * turn
            head = torch.cat([z.real, z.imag], dim=-1)
        return torch.cat([head, rest], dim=-1).view(b, t, heads * d)
    codes = _unpack(state["weight"]).long()
    levels = torch.tensor(E2M1 + tuple(-v for v in E2M1), dtype=torch.float64, device=codes.device)
    byte = torch.arange(256, dtype=torch.float64, device=codes.device)
    if case["fmt"] == "mxfp4":
        table = 2.0 ** (byte - 127)
    else:
        table = torch.where(byte < 8, byte / 512, (1 + (byte % 8) / 8) * 2.0 ** ((byte // 8) - 7))
    group = GROUP[case["fmt"]]
    w = levels[codes] * table[state["scales"].long()].repeat_interleave(group, dim=1) * state["g"]
    x = state["x"].double()
    if op == "linear4":
        x = _exact_values(x, case["fmt"], 1.0)
    return x @ w.t()
