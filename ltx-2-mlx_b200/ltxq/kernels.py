"""Drop-in replacements for ``LTX_2_MLX.kernels`` (fused_ops.py).

``adaln_norm_fused(x, scale, shift, eps)`` and ``gated_add_fused(residual,
branch, gate)`` keep the reference's names, argument order and return dtype
(fused_ops.py:237, 398).  Unlike the reference they never fall back to a
second implementation: every supported input (bf16/fp32 ``x``, fp32/bf16
vectors, broadcast, per-batch or per-token vectors, any eps, any C that is a
multiple of 8) runs the CUDA kernel, and anything else raises ``ValueError``.
"""

from __future__ import annotations

import ctypes
import math
import struct

import torch

from . import _lib

_DT = {torch.bfloat16: _lib.BF16, torch.float32: _lib.F32}


def _public_raw_stream(device: int) -> int:
    return torch.cuda.current_stream(device).cuda_stream


# The current device and a device's current stream: torch's own functions where it has them (built with CUDA; a
# microsecond or two less per call), else the public ones.
_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", _public_raw_stream)


def _stream() -> int:
    return _raw_stream(_device())


def _require_cuda(t: torch.Tensor, name: str) -> None:
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (there is no CPU path)")


def vec_arg(v: torch.Tensor, rows_shape: tuple[int, ...], C: int, name: str, keep: list) -> _lib.Vec:
    """Describe a per-channel vector broadcast against activations of shape
    ``rows_shape + (C,)``: all-singleton leading dims -> one vector for all
    rows; (B, 1, C) -> one vector per batch entry; (B, T, C) -> per token."""
    _require_cuda(v, name)
    if v.dtype not in _DT:
        raise ValueError(f"{name} dtype must be bfloat16 or float32, got {v.dtype}")
    if v.shape[-1] != C:
        raise ValueError(f"{name} last dim {v.shape[-1]} != {C}")
    if v.stride(-1) != 1:
        v = v.contiguous()
    keep.append(v)
    lead = tuple(v.shape[:-1])
    numel_lead = 1
    for d in lead:
        numel_lead *= d
    if numel_lead == 1:  # one vector for all rows (a strided view is used in place)
        return _lib.Vec(v.data_ptr(), _DT[v.dtype], 0, 0, 0)
    rows = 1
    for d in rows_shape:
        rows *= d
    if numel_lead == rows:  # (B, T, C): one vector per row
        if not v.is_contiguous():
            v = v.contiguous()
            keep.append(v)
        return _lib.Vec(v.data_ptr(), _DT[v.dtype], 0, 1, C)
    if len(rows_shape) >= 2 and len(lead) >= 1 and lead[0] == rows_shape[0] and numel_lead == rows_shape[0]:
        # (B, 1, C): one vector per batch entry, B vectors at the view's batch stride
        return _lib.Vec(v.data_ptr(), _DT[v.dtype], 0, rows // rows_shape[0], v.stride(0))
    raise ValueError(f"{name} shape {tuple(v.shape)} does not broadcast against {rows_shape + (C,)}")


class MXActivation:
    """Activations in the input form of the block-scaled GEMMs
    (``ltxq_mx_act``: per term [M, K] E4M3 codes and E8M0 scales in the MMA's
    atom layout; ``terms`` 2 or 1).  Written by ``adaln_modulate`` /
    ``head_gate`` with ``mx_terms`` and by ``QuantizedLinear`` with
    ``mx_out``, read by ``QuantizedLinear``; the bits are those
    ``ltxq_mx_split`` gives for the bf16 values.  One device buffer holds
    every part."""

    def __init__(self, rows_shape: tuple[int, ...], K: int, terms: int, device):
        if terms not in (1, 2):
            raise ValueError("terms must be 1 or 2")
        self.rows_shape = tuple(rows_shape)
        self.K = int(K)
        self.terms = int(terms)
        self.M = math.prod(self.rows_shape)
        codes, sf = ctypes.c_size_t(0), ctypes.c_size_t(0)
        if not _lib.load().ltxq_mx_split_sizes(self.M, self.K, ctypes.byref(codes), ctypes.byref(sf)):
            raise ValueError(f"no MX form for {self.M} x {self.K} (K % 128 == 0 and M > 0 needed)")
        cb, sb = _align(codes.value), _align(sf.value)
        self.buffer = torch.empty(terms * (cb + sb), dtype=torch.uint8, device=device)
        base = self.buffer.data_ptr()
        self._parts = (base, base + cb if terms == 2 else None, base + terms * cb,
                       base + terms * cb + sb if terms == 2 else None)

    @property
    def shape(self) -> tuple[int, ...]:
        return self.rows_shape + (self.K,)

    @property
    def device(self):
        return self.buffer.device

    def tensors(self) -> tuple:
        """(hi, lo, sf_hi, sf_lo) as uint8 views of the buffer: codes [M, K],
        scale atoms flat (ltxq_mx_split_sizes bytes); lo / sf_lo None for one
        term."""
        codes, sf = ctypes.c_size_t(0), ctypes.c_size_t(0)
        _lib.load().ltxq_mx_split_sizes(self.M, self.K, ctypes.byref(codes), ctypes.byref(sf))
        base = self.buffer.data_ptr()
        out = []
        for ptr, n, shape in zip(self._parts, (codes.value, codes.value, sf.value, sf.value),
                                 ((self.M, self.K), (self.M, self.K), (-1,), (-1,))):
            out.append(None if ptr is None else self.buffer[ptr - base:ptr - base + n].view(shape))
        return tuple(out)

    def struct(self) -> _lib.MxAct:
        hi, lo, sf_hi, sf_lo = self._parts
        return _lib.MxAct(hi, lo, sf_hi, sf_lo, self.terms, 0)

    @classmethod
    def split(cls, x: torch.Tensor, terms: int) -> "MXActivation":
        """The MX form of bf16 ``x`` (``ltxq_mx_split``)."""
        _require_cuda(x, "x")
        if x.dtype != torch.bfloat16:
            raise ValueError("x must be bfloat16")
        x = x.contiguous()
        act = cls(tuple(x.shape[:-1]), x.shape[-1], terms, x.device)
        hi, lo, sf_hi, sf_lo = act._parts
        _lib.check(_lib.load().ltxq_mx_split(x.data_ptr(), act.M, act.K, terms, hi, lo, sf_hi, sf_lo, _stream()),
                   "mx_split")
        return act


def _align(n: int) -> int:
    return (n + 255) & ~255


def mx_output_ok(C: int) -> bool:
    """Whether the row kernels (AdaLN, head gate) can write C channels in the
    MX form (32-channel groups held by lane quads, at most 4096 channels for
    the AdaLN pass)."""
    return C % 128 == 0 and C <= 4096


FP4_MODES = {"mxfp4": _lib.MXFP4, "nvfp4": _lib.NVFP4}


def _on(t: torch.Tensor):
    """Context in which ``t``'s device is the current one (its stream and
    launches are the ones used)."""
    return torch.cuda.device(t.device)


class FP4Tensor:
    """A matrix in 4-bit floating point, the input form of products of two
    quantized operands (``ltxq_fp4_act``): E2M1 codes [M, K / 2] bytes and
    group scales in the block-scaled MMA's atom layout.

    ``mode`` "mxfp4": 32 values along K share an E8M0 scale; "nvfp4": 16 share
    an E4M3 scale, times ``global_scale`` (one number for the tensor).  A group
    that holds an infinity or a NaN reads back as NaN.  K must be a multiple of
    32.  Written by ``quantize``, read by ``dequantize`` and by a
    ``QuantizedLinear`` of the same mode whose compute is "fp4"; one quantized
    tensor serves every projection that reads it."""

    def __init__(self, rows_shape: tuple[int, ...], K: int, mode: str, device, global_scale: float = 1.0):
        if mode not in FP4_MODES:
            raise ValueError(f"mode must be one of {sorted(FP4_MODES)}, got {mode!r}")
        if K <= 0 or K % 32 != 0:
            raise ValueError(f"K must be a positive multiple of 32, got {K}")
        if global_scale != 1.0:
            if mode != "nvfp4":
                raise ValueError("global_scale is nvfp4 only")
            if not 2.0 ** -64 <= global_scale <= 2.0 ** 64:
                raise ValueError("global_scale must be within [2^-64, 2^64]")
        self.rows_shape = tuple(rows_shape)
        self.K = int(K)
        self.mode = mode
        self.global_scale = float(global_scale)
        self.M = M = math.prod(self.rows_shape)
        self._st = None
        self._code_bytes = M * (K // 2)
        self._scale_bytes = (K + 255) // 256 * ((M + 127) // 128) * (2048 if mode == "nvfp4" else 1024)
        self._scale_off = _align(self._code_bytes)
        self.buffer = torch.empty(self._scale_off + self._scale_bytes, dtype=torch.uint8, device=device)

    @property
    def shape(self) -> tuple[int, ...]:
        return self.rows_shape + (self.K,)

    @property
    def device(self):
        return self.buffer.device

    def tensors(self) -> tuple[torch.Tensor, torch.Tensor]:
        """(codes [M, K / 2], scale atoms flat) as uint8 views of the buffer."""
        return (self.buffer[:self._code_bytes].view(self.M, self.K // 2),
                self.buffer[self._scale_off:self._scale_off + self._scale_bytes])

    def struct(self) -> _lib.Fp4Act:
        base = self.buffer.data_ptr()
        kept = self._st
        if kept is None or kept[0] is not self.buffer or kept[1] != (base, self.mode, self.global_scale):
            buf = self.buffer
            if (buf.dtype != torch.uint8 or not buf.is_contiguous() or buf.numel() < self._scale_off + self._scale_bytes
                    or base % 16):
                raise ValueError("the buffer of an FP4Tensor holds its codes and scales: uint8, contiguous, 16-byte "
                                 f"aligned, {self._scale_off + self._scale_bytes} bytes")
            st = _lib.Fp4Act(base, base + self._scale_off, FP4_MODES[self.mode], self.global_scale)
            kept = self._st = (buf, (base, self.mode, self.global_scale), st)
        return kept[2]

    def __getstate__(self):
        """Copies make a descriptor of their own: it holds addresses."""
        return self.__dict__ | {"_st": None}

    @classmethod
    def quantize(cls, x: torch.Tensor, mode: str = "nvfp4", global_scale: float = 1.0) -> "FP4Tensor":
        """bf16 ``x`` (..., K) quantized along K."""
        _require_cuda(x, "x")
        if x.dtype != torch.bfloat16:
            raise ValueError(f"x must be bfloat16, got {x.dtype}")
        if x.dim() < 1:
            raise ValueError("x must have at least one dimension")
        dev = x.get_device()
        if dev != _device():
            with torch.cuda.device(dev):
                return cls.quantize(x, mode, global_scale)
        t = cls(x.shape[:-1], x.shape[-1], mode, x.device, global_scale)
        if t.M == 0:
            return t
        stride = t.K
        if not x.is_contiguous() or x.data_ptr() % 16:
            x = x.reshape(t.M, t.K)  # rows at one stride; copied where they are not
            if x.stride(1) != 1 or x.stride(0) % 8 != 0 or x.stride(0) < t.K or x.data_ptr() % 16:
                x = x.clone(memory_format=torch.contiguous_format)
            stride = x.stride(0) if t.M > 1 else t.K
        _lib.check(_lib.load().ltxq_fp4_quantize(x.data_ptr(), t.M, t.K, stride, t.struct(), _raw_stream(dev)),
                   "fp4_quantize")
        return t

    def dequantize(self) -> torch.Tensor:
        """The values, as bf16 of the quantized tensor's shape."""
        dev = self.buffer.get_device()
        if dev != _device():
            with torch.cuda.device(dev):
                return self.dequantize()
        out = self.buffer.new_empty(self.rows_shape + (self.K,), dtype=torch.bfloat16)
        if self.M:
            _lib.check(_lib.load().ltxq_fp4_dequantize(self.struct(), self.M, self.K, out.data_ptr(), _raw_stream(dev)),
                       "fp4_dequantize")
        return out


def fp4_global_scale(x: torch.Tensor) -> float:
    """A ``global_scale`` for quantizing ``x`` to nvfp4: the power of two that
    puts the scale of the group with the largest magnitude just inside E4M3's
    range (448), so that small weights do not fall into its subnormals.  Reads
    one number back from the device."""
    amax = float(x.detach().abs().amax()) if x.numel() else 0.0
    if not math.isfinite(amax) or amax == 0.0:
        return 1.0
    return 2.0 ** max(-64, min(64, math.ceil(math.log2(amax / (6.0 * 448.0)))))


def prologue(norm: int, eps: float, scale, shift, rows_shape, C, keep) -> _lib.Prologue:
    return _lib.Prologue(norm, float(eps), vec_arg(scale, rows_shape, C, "scale", keep),
                         vec_arg(shift, rows_shape, C, "shift", keep))


def adaln_modulate(x: torch.Tensor, scale: torch.Tensor, shift: torch.Tensor, eps: float = 1e-6,
                   norm: str = "rms", mx_terms: int = 0):
    """``bf16(norm(x) * (1 + scale) + shift)`` with norm in {"rms", "layer",
    "none"}; "none" is the text cross-attention context modulation
    (transformer.py:379).  ``mx_terms`` 1 or 2 returns the result as an
    ``MXActivation`` instead (the next block-scaled GEMM's input; bf16 x,
    ``mx_output_ok(C)``)."""
    _require_cuda(x, "x")
    if x.dtype not in _DT:
        raise ValueError(f"x dtype must be bfloat16 or float32, got {x.dtype}")
    x = x.contiguous()
    C = x.shape[-1]
    rows_shape = tuple(x.shape[:-1])
    keep: list = []
    nk = {"rms": _lib.NORM_RMS, "layer": _lib.NORM_LAYER, "none": _lib.NORM_NONE}[norm]
    pro = prologue(nk, eps, scale, shift, rows_shape, C, keep)
    lib = _lib.load()
    if mx_terms:
        act = MXActivation(rows_shape, C, mx_terms, x.device)
        st = act.struct()
        _lib.check(lib.ltxq_adaln_modulate_mx(x.data_ptr(), act.M, C, ctypes.byref(pro), None, ctypes.byref(st),
                                              _stream()), "adaln_modulate_mx")
        return act
    out = torch.empty_like(x)
    _lib.check(lib.ltxq_adaln_modulate(x.data_ptr(), _DT[x.dtype], x.numel() // C, C, ctypes.byref(pro),
                                       out.data_ptr(), _stream()), "adaln_modulate")
    return out


def adaln_norm_fused(x: torch.Tensor, scale: torch.Tensor, shift: torch.Tensor, eps: float) -> torch.Tensor:
    """``(rms_norm(x) * (1 + scale) + shift).astype(x.dtype)``
    (fused_ops.py:237 / transformer.py:21-37)."""
    return adaln_modulate(x, scale, shift, eps, "rms")


def gated_add_fused(residual: torch.Tensor, branch: torch.Tensor, gate: torch.Tensor,
                    gate_then_add: bool = False) -> torch.Tensor:
    """``(residual + branch * gate).astype(residual.dtype)``
    (fused_ops.py:398 / transformer.py:40-50).  ``gate_then_add=True`` gives
    the text cross-attention form ``residual + bf16(branch * gate)``
    (transformer.py:387, 484)."""
    _require_cuda(residual, "residual")
    _require_cuda(branch, "branch")
    if residual.dtype != torch.bfloat16 or branch.dtype != torch.bfloat16:
        raise ValueError("residual and branch must be bfloat16")
    if residual.shape != branch.shape:
        raise ValueError(f"shape mismatch {tuple(residual.shape)} vs {tuple(branch.shape)}")
    residual = residual.contiguous()
    branch = branch.contiguous()
    C = residual.shape[-1]
    keep: list = []
    g = vec_arg(gate, tuple(residual.shape[:-1]), C, "gate", keep)
    out = torch.empty_like(residual)
    mode = _lib.GATE_THEN_ADD if gate_then_add else _lib.GATED_ADD
    _lib.check(_lib.load().ltxq_gated_add(residual.data_ptr(), branch.data_ptr(), ctypes.byref(g),
                                          residual.numel() // C, C, mode, out.data_ptr(), _stream()),
               "gated_add")
    return out


def head_gate(out: torch.Tensor, gate_logits: torch.Tensor, heads: int, mx_terms: int = 0):
    """``out * (2 * sigmoid(gate_logits))[..., None]`` per head
    (attention.py:559-601).  ``mx_terms`` as in ``adaln_modulate``.
    ``gate_logits`` may be a column slice of a wider tensor (rows at a
    uniform stride, heads contiguous): it is read in place."""
    _require_cuda(out, "out")
    _require_cuda(gate_logits, "gate_logits")
    if out.dtype != torch.bfloat16 or gate_logits.dtype != torch.bfloat16:
        raise ValueError("head_gate expects bfloat16 tensors")
    out = out.contiguous()
    width = out.shape[-1]
    rows = out.numel() // width
    if gate_logits.numel() != rows * heads or gate_logits.shape[-1] != heads:
        raise ValueError("gate_logits must have one value per (row, head)")
    try:
        gl = gate_logits.view(rows, heads)
    except RuntimeError:  # rows not at one uniform stride
        gl = gate_logits.contiguous().view(rows, heads)
    if gl.stride(1) != 1 or (rows > 1 and gl.stride(0) < heads):
        gl = gl.contiguous()
    lstride = gl.stride(0) if rows > 1 else heads
    if mx_terms:
        act = MXActivation(tuple(out.shape[:-1]), width, mx_terms, out.device)
        st = act.struct()
        _lib.check(_lib.load().ltxq_head_gate_ex(out.data_ptr(), gl.data_ptr(), lstride, rows, heads, width // heads,
                                                 None, ctypes.byref(st), _stream()), "head_gate_ex")
        return act
    res = torch.empty_like(out)
    _lib.check(_lib.load().ltxq_head_gate_ex(out.data_ptr(), gl.data_ptr(), lstride, rows, heads, width // heads,
                                             res.data_ptr(), None, _stream()), "head_gate_ex")
    return res


def qk_norm_rope_pair(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor, heads: int,
                      eps: float = 1e-6, pe: tuple | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """``qk_norm_rope`` of Q and K over the same rows and RoPE tables in one
    pass (the tables are read once): the self-attention's Q/K norm and
    rotation (attention.py:580-587)."""
    for t, name in ((q, "q"), (k, "k")):
        _require_cuda(t, name)
        if t.dtype != torch.bfloat16 or t.stride(-1) != 1 or t.dim() != 3:
            raise ValueError(f"{name} must be a (B, T, W) bfloat16 tensor with unit column stride")
    if q.shape != k.shape:
        raise ValueError("q and k must have the same shape")
    b, t, width = q.shape
    q = q if q.stride(0) == t * q.stride(1) else q.contiguous()
    k = k if k.stride(0) == t * k.stride(1) else k.contiguous()
    d = width // heads
    wq, wk = q_weight.float().contiguous(), k_weight.float().contiguous()
    oq = torch.empty((b, t, width), dtype=torch.bfloat16, device=q.device)
    ok = torch.empty_like(oq)
    cos = sin = None
    if pe is not None:
        cos, sin = pe[0].float().contiguous(), pe[1].float().contiguous()
        if cos.shape != (b, heads, t, d // 2) and cos.shape != (1, heads, t, d // 2):
            raise ValueError(f"RoPE table shape {tuple(cos.shape)} does not match {(b, heads, t, d // 2)}")
        if cos.shape[0] != b:
            cos, sin = cos.expand(b, -1, -1, -1).contiguous(), sin.expand(b, -1, -1, -1).contiguous()
    _lib.check(_lib.load().ltxq_qk_norm_rope_pair(
        q.data_ptr(), k.data_ptr(), b * t, q.stride(1), k.stride(1), heads, d, wq.data_ptr(), wk.data_ptr(),
        float(eps), cos.data_ptr() if cos is not None else None, sin.data_ptr() if sin is not None else None, t,
        oq.data_ptr(), ok.data_ptr(), _stream()), "qk_norm_rope_pair")
    return oq, ok


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, heads: int, scale: float | None = None) -> torch.Tensor:
    """``softmax(q k^T * scale) v`` per head (the block's
    ``mx.fast.scaled_dot_product_attention``, attention.py:170-302) on
    (B, T, heads*D) rows: q (B, Tq, W), k / v (B, Tk, W), any row stride with
    unit column stride (column slices of a fused projection are read in
    place).  D = W / heads must be 64 or 128; scale defaults to 1/sqrt(D).
    Returns contiguous (B, Tq, heads*D) bf16."""
    for t, name in ((q, "q"), (k, "k"), (v, "v")):
        _require_cuda(t, name)
        if t.dtype != torch.bfloat16 or t.dim() != 3 or t.stride(-1) != 1:
            raise ValueError(f"{name} must be a (B, T, W) bfloat16 tensor with unit column stride")
    b, tq, width = q.shape
    if k.shape != v.shape or k.shape[0] != b or k.shape[2] != width:
        raise ValueError("k and v must be (B, Tk, W) with q's B and W")
    tk = k.shape[1]
    if width % heads != 0:
        raise ValueError("W must be a multiple of heads")
    d = width // heads
    if scale is None:
        scale = 1.0 / math.sqrt(d)

    def rows(t):  # (B, T, W) with one row stride across batch and tokens
        if t.stride(0) != t.shape[1] * t.stride(1):
            t = t.contiguous()
        return t

    q, k, v = rows(q), rows(k), rows(v)
    out = torch.empty((b, tq, width), dtype=torch.bfloat16, device=q.device)
    _lib.check(_lib.load().ltxq_attention(q.data_ptr(), k.data_ptr(), v.data_ptr(), b, tq, tk, heads, d, q.stride(1),
                                          k.stride(1), v.stride(1), float(scale), out.data_ptr(), _stream()),
               "attention")
    return out


def qk_norm_rope(x: torch.Tensor, weight: torch.Tensor, heads: int, eps: float = 1e-6,
                 pe: tuple | None = None) -> torch.Tensor:
    """QK RMSNorm (attention.py:320-329) then split RoPE (rope.py:53-90) in one
    pass.  x: (B, T, heads*D) bf16, any row stride with unit column stride;
    pe: (cos, sin) fp32 (B, heads, T, D/2) or None.  Returns contiguous
    (B, T, heads*D) bf16."""
    _require_cuda(x, "x")
    if x.dtype != torch.bfloat16 or x.stride(-1) != 1 or x.dim() != 3:
        raise ValueError("x must be a (B, T, W) bfloat16 tensor with unit column stride")
    b, t, width = x.shape
    if x.stride(0) != t * x.stride(1):
        x = x.contiguous()
    d = width // heads
    w = weight.float().contiguous()
    out = torch.empty((b, t, width), dtype=torch.bfloat16, device=x.device)
    cos = sin = None
    if pe is not None:
        cos, sin = pe[0].float().contiguous(), pe[1].float().contiguous()
        if cos.shape != (b, heads, t, d // 2) and cos.shape != (1, heads, t, d // 2):
            raise ValueError(f"RoPE table shape {tuple(cos.shape)} does not match {(b, heads, t, d // 2)}")
        if cos.shape[0] != b:
            cos, sin = cos.expand(b, -1, -1, -1).contiguous(), sin.expand(b, -1, -1, -1).contiguous()
    _lib.check(_lib.load().ltxq_qk_norm_rope(x.data_ptr(), b * t, x.stride(1), heads, d, w.data_ptr(), float(eps),
                                             cos.data_ptr() if cos is not None else None,
                                             sin.data_ptr() if sin is not None else None, t, out.data_ptr(),
                                             _stream()), "qk_norm_rope")
    return out


_POS = {torch.int32: _lib.POS_I32, torch.int64: _lib.POS_I64, torch.float32: _lib.POS_F32, torch.float64: _lib.POS_F64}
_ROTARY_ARGS = struct.Struct("@PPii5q3q3qP3qiiPPiifi")  # _lib.RotaryArgs
_ROTARY_LAYOUT = {"half": _lib.ROTARY_HALF, "interleaved": _lib.ROTARY_INTERLEAVED}


def rotary(x: torch.Tensor, positions: torch.Tensor, freqs: torch.Tensor, heads: int, *, layout: str = "half",
           axes: torch.Tensor | None = None, scale: float = 1.0, inverse: bool = False,
           out: torch.Tensor | None = None) -> torch.Tensor:
    """Rotary positions on one operand of attention, the angles formed in the
    kernel (no cos / sin tables): pair i of a head turns by ``positions *
    freqs[i]`` and is multiplied by ``scale``.

    ``x``: bf16 or fp32, (B, T, heads*D) or (B, T, heads, D), any strides with
    a unit last one (a column slice of a fused projection, a transposed
    (B, heads, T, D)).  ``layout`` "half" pairs elements i and i + R/2 of a
    head (the split form of rope.py:53-90), "interleaved" 2i and 2i + 1, with
    R = 2 * freqs.shape[-1] <= D; elements past R pass through.  ``freqs``:
    float64, radians per unit of position, (R/2,) or (heads, R/2)
    (``rope.rotary_frequencies``, ``rope.grid_rotary``).  ``positions``:
    int32, int64, float32 or float64, (T,) or (B, T); with ``axes`` (int32,
    freqs' shape: the position axis of each frequency) (A, T) or (B, A, T).
    An axis outside [0, A) gives NaN.

    ``inverse`` turns back by the same angles with the same scale: the
    gradient of the forward call.  ``out`` (x's shape and type, memory of its
    own for every element) may be ``x``, or share no element with it, which
    has to show from the strides: two overlapping ranges of memory are taken
    where both have the same ones.
    Returns ``out``, contiguous where it is made here."""
    _require_cuda(x, "x")
    _require_cuda(positions, "positions")
    _require_cuda(freqs, "freqs")
    dt, shape, fshape, pshape = _DT.get(x.dtype), x.shape, freqs.shape, positions.shape
    if dt is None:
        raise ValueError(f"x dtype must be bfloat16 or float32, got {x.dtype}")
    if layout not in _ROTARY_LAYOUT:
        raise ValueError(f"layout must be 'half' or 'interleaved', got {layout!r}")
    four = len(shape) == 4
    if heads <= 0 or not (four or len(shape) == 3) or (four and shape[2] != heads):
        raise ValueError(f"x must be (B, T, {heads} * D) or (B, T, {heads}, D), got {tuple(shape)}")
    if not four and shape[2] % heads != 0:
        raise ValueError("x's last dimension must be a multiple of heads")
    b, t = shape[0], shape[1]
    d = shape[3] if four else shape[2] // heads
    per_head = len(fshape) == 2
    if freqs.dtype != torch.float64 or not (per_head or len(fshape) == 1) or (per_head and fshape[0] != heads):
        raise ValueError(f"freqs must be float64 (R/2,) or ({heads}, R/2), got {freqs.dtype} {tuple(fshape)}")
    r = 2 * fshape[-1]
    if r > d:
        raise ValueError(f"freqs rotate {r} elements but a head has {d}")
    pos_type = _POS.get(positions.dtype)
    if pos_type is None:
        raise ValueError(f"positions must be int32, int64, float32 or float64, got {positions.dtype}")
    lead = len(pshape) - (1 if axes is None else 2)
    if lead not in (0, 1) or pshape[-1] != t or (lead and pshape[0] != b):
        raise ValueError(f"positions shape {tuple(pshape)} does not match {b} x {t} tokens")
    n_axes = 1
    if axes is not None:
        _require_cuda(axes, "axes")
        if axes.dtype != torch.int32 or axes.shape != fshape:
            raise ValueError("axes must be int32 with the shape of freqs")
        n_axes = pshape[-2]
        axes = axes.contiguous()
        if n_axes < 1:
            raise ValueError("positions have no axis")
    dev = x.get_device()
    if positions.get_device() != dev or freqs.get_device() != dev or (axes is not None and axes.get_device() != dev) or (
            out is not None and out.get_device() != dev):
        raise ValueError(f"positions, freqs, axes and out must be on x's device ({x.device})")
    if d == 0:
        raise ValueError("heads have no elements")
    if dev != _device():
        with torch.cuda.device(dev):
            return rotary(x, positions, freqs, heads, layout=layout, axes=axes, scale=scale, inverse=inverse, out=out)
    if x.stride(-1) != 1 and x.shape[-1] > 1:
        if out is x:
            raise ValueError("an in-place rotation needs x with a unit last stride")
        x = x.contiguous()
    if not -3e38 <= scale <= 3e38:
        raise ValueError(f"scale must be finite, got {scale}")
    if out is None:
        out = torch.empty_like(x, memory_format=torch.contiguous_format)
    elif out.shape != x.shape or out.dtype != x.dtype or (out.stride(-1) != 1 and out.shape[-1] > 1):
        raise ValueError("out must have x's shape and type and a unit last stride")
    if x.numel() == 0:
        return out
    freqs = freqs.contiguous()
    xs, os, ps = x.stride(), out.stride(), positions.stride()
    args = _ROTARY_ARGS.pack(
        x.data_ptr(), out.data_ptr(), dt, _ROTARY_LAYOUT[layout], b, t, heads, d, r, xs[0], xs[1], xs[2] if four else d,
        os[0], os[1], os[2] if four else d, positions.data_ptr(), ps[0] if lead else 0, ps[-2] if axes is not None else 0,
        ps[-1], pos_type, n_axes, freqs.data_ptr(), axes.data_ptr() if axes is not None else 0, per_head, bool(inverse),
        scale, 0)
    _lib.check(_lib.load().ltxq_rotary(args, _raw_stream(dev)), "rotary")
    return out
