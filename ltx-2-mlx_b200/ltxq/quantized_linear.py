"""Quantized linear layers over the reference's MLX cache layout.

``QuantizedLinear`` mirrors MLX ``nn.QuantizedLinear`` as the reference uses
it (LTX_2_MLX/loader/transformer_cache.py:1436-1462 builds the empty module,
:1238-1267 fills ``weight``/``scales``/``biases`` from ``mx.quantize``,
``bias`` stays bf16): the same attribute names and dtypes, the same
``mode``/``group_size``/``bits`` semantics and defaults (:797-811), and
``__call__(x) -> y``.  ``pretransposed=True`` gives the reference's
``_PretransposedQuantizedLinear`` (:177-193) whose packed arrays were built
from ``W.T``.  The 4-bit floating point modes "mxfp4" and "nvfp4" (the
reference's defaults 32/4 and 16/4) compute either from the dequantized weight
or, with ``set_compute("fp4")``, as a product of two quantized operands.

The forward pass is one launch of the sm_100a quantized GEMM with the
block's epilogue fused (bias, GELU, gated residual); there is no CPU path.
"""

from __future__ import annotations

import ctypes
import math

import torch

from . import _lib
from .kernels import (FP4_MODES, FP4Tensor, MXActivation, _device, _on, _raw_stream, _require_cuda, _stream, prologue,
                      vec_arg)

QUANT_DEFAULTS = {"affine": (64, 4), "mxfp8": (32, 8), "mxfp4": (32, 4), "nvfp4": (16, 4)}
_MODE = {"affine": _lib.AFFINE, "mxfp8": _lib.MXFP8, **FP4_MODES}
# the types that an fp4 weight's scales come in: their bytes, or the format itself
_SCALES = {"mxfp4": (torch.uint8, torch.int8, torch.float8_e8m0fnu),
           "nvfp4": (torch.uint8, torch.int8, torch.float8_e4m3fn)}
# how the GEMM computes (include/ltxq.h LTXQ_COMPUTE_*): "dequant" (bf16
# tensor cores over the exactly dequantized weight), "mx2" / "mx1" (native
# block-scaled fp8 MMAs on mxfp8 weights, activations in two / one MXFP8 terms),
# "fp4" (block-scaled fp4 MMAs on mxfp4 / nvfp4 weights, activations quantized
# to the weight's format)
COMPUTE = {"dequant": _lib.COMPUTE_DEQUANT, "mx2": _lib.COMPUTE_MX2, "mx1": _lib.COMPUTE_MX1,
           "fp4": _lib.COMPUTE_FP4}


def _capturing() -> bool:
    """Whether the current stream records a graph."""
    return torch.cuda.is_current_stream_capturing()


def _wait_device(device) -> None:
    torch.cuda.synchronize(device)


def _wait_stream() -> None:
    torch.cuda.current_stream().synchronize()


def _version(t: torch.Tensor) -> int:
    """torch's in-place version counter (tensors made in inference mode have none)."""
    return 0 if t.is_inference() else t._version


def quant_defaults(mode: str, group_size: int | None, bits: int | None) -> tuple[int, int]:
    """``_quant_defaults`` (transformer_cache.py:797-811) for the modes this
    path implements."""
    if mode not in QUANT_DEFAULTS:
        raise ValueError(f"Unsupported quantization mode: {mode}")
    gs, b = QUANT_DEFAULTS[mode]
    return group_size or gs, bits or b


class QuantizedLinear:
    _q4 = None  # the descriptor of an fp4 weight's products (_qweight4)
    _fp4_packed = (None, None, None)  # scale tensor, its state, the memory its scales are packed in (_fp4_scales)

    def __init__(self, weight: torch.Tensor, scales: torch.Tensor, biases: torch.Tensor | None = None,
                 bias: torch.Tensor | None = None, *, group_size: int, bits: int, mode: str = "affine",
                 pretransposed: bool = False, in_features: int | None = None, out_features: int | None = None,
                 global_scale: float = 1.0):
        if mode not in _MODE:
            raise ValueError(f"Unsupported quantization mode: {mode}")
        if mode != "nvfp4" and global_scale != 1.0:
            raise ValueError("global_scale is nvfp4 only")
        if not 2.0 ** -64 <= global_scale <= 2.0 ** 64:
            raise ValueError("global_scale must be within [2^-64, 2^64]")
        self.global_scale = float(global_scale)
        for t, name in ((weight, "weight"), (scales, "scales")):
            _require_cuda(t, name)
        self.weight = weight.contiguous()
        self.scales = scales.contiguous()
        self.biases = biases.contiguous() if biases is not None else None
        self.bias = bias.contiguous() if bias is not None else None
        self.group_size = int(group_size)
        self.bits = int(bits)
        self.mode = mode
        self.pretransposed = bool(pretransposed)
        packed_rows = self.weight.shape[0]
        packed_len = self.weight.shape[1] * 32 // self.bits
        if pretransposed:
            self.in_features = in_features or packed_rows
            self.out_features = out_features or packed_len
        else:
            self.out_features = out_features or packed_rows
            self.in_features = in_features or packed_len
        if mode == "affine" and self.biases is None:
            raise ValueError("affine quantization needs biases")
        if mode in FP4_MODES:
            self._check_fp4()
        self.compute = "dequant"

    def _check_fp4(self) -> None:
        """The fp4 arrays fit the layer: what the kernels read lies inside them."""
        rows, length = ((self.in_features, self.out_features) if self.pretransposed
                        else (self.out_features, self.in_features))
        if (self.bits, self.group_size) != (4, QUANT_DEFAULTS[self.mode][0]):
            raise ValueError(f"{self.mode} has 4 bits and group_size {QUANT_DEFAULTS[self.mode][0]}")
        for t, name, shape, types in ((self.weight, "weight", (rows, length // 8), (torch.uint32, torch.int32)),
                                      (self.scales, "scales", (rows, length // self.group_size), _SCALES[self.mode]),
                                      (self.bias, "bias", (self.out_features,), (torch.bfloat16,))):
            if t is None:
                continue
            if tuple(t.shape) != shape or t.dtype not in types or not t.is_contiguous():
                raise ValueError(f"{self.mode} {name} must be a contiguous {shape} of one of {types}, got "
                                 f"{tuple(t.shape)} {t.dtype}")
            if t.device != self.weight.device:
                raise ValueError(f"{name} is on {t.device}, the weight on {self.weight.device}")
        if length % self.group_size:
            raise ValueError(f"{length} values do not divide into groups of {self.group_size}")

    def set_compute(self, compute: str) -> "QuantizedLinear":
        """Select how GEMMs over this weight compute (``COMPUTE``); the MX
        modes apply to mxfp8 weights and "fp4" to mxfp4 / nvfp4 weights, both
        in the standard layout; other weights keep the dequantizing kernels."""
        if compute not in COMPUTE:
            raise ValueError(f"unknown compute mode {compute!r}")
        self.compute = compute
        self._mx_scales = None
        self._q4 = None
        self._fp4_packed = (None, None, self._fp4_packed[2])  # packed again, in place
        if compute != "dequant":
            self.mx_scales()  # packed now, not in every replay of a later stream capture
        return self

    def mx_scales(self) -> torch.Tensor | None:
        """The weight scales repacked for the block-scaled MMA of the MX modes
        (``ltxq_mx_pack_weight_scales``) or of "fp4"
        (``ltxq_fp4_pack_weight_scales``), made once and again only when the
        scale tensor changes; None where those modes do not apply."""
        if self.computes_fp4():
            return self._fp4_scales()
        if getattr(self, "compute", "dequant") in ("dequant", "fp4") or self.mode != "mxfp8" or self.pretransposed:
            return None
        if self.in_features % 512 != 0:
            return None
        key = (self.scales.data_ptr(), self.scales._version)
        cached = getattr(self, "_mx_scales", None)
        if cached is None or cached[0] != key:
            lib = _lib.load()
            q = self._qweight_base(0, None)
            nbytes = lib.ltxq_mx_weight_scales_size(ctypes.byref(q))
            buf = torch.empty(nbytes, dtype=torch.uint8, device=self.scales.device)
            _lib.check(lib.ltxq_mx_pack_weight_scales(ctypes.byref(q), buf.data_ptr(), _stream()), "mx_pack_weight_scales")
            cached = (key, buf)
            self._mx_scales = cached
        return cached[1]

    def _fp4_scales(self) -> torch.Tensor:
        """The packed scales of "fp4".  They belong to one scale tensor (the
        object, kept here) in one state: another tensor, or one changed in
        place, is packed again by the next call or ``set_compute``, into the
        same memory, which captured graphs read.  A graph replayed after such
        a change therefore needs one of the two first.  Tensors made in
        inference mode do not count their changes, and writes through ``.data``,
        by a replayed graph or from outside torch count for none: after those
        call ``set_compute``, which always packs.

        Calls on other streams cannot be told of a packing that they did not
        ask for, so the host waits: for the device before memory is packed
        again, which they may still read, and for the packing itself.

        Inside a stream capture packing would only be recorded: memory of the
        graph's own takes it there, packed by every replay, and nothing is
        noted as packed."""
        scales, state, buf = self._fp4_packed
        now = (self.scales.data_ptr(), _version(self.scales))
        if scales is not self.scales or state != now:
            self._check_fp4()
            with _on(self.scales):
                lib = _lib.load()
                q = self._qweight_base(0, None)
                nbytes = lib.ltxq_fp4_weight_scales_size(ctypes.byref(q))
                recorded = _capturing()
                if recorded or buf is None or buf.numel() != nbytes or buf.device != self.scales.device:
                    buf = torch.empty(nbytes, dtype=torch.uint8, device=self.scales.device)
                else:
                    _wait_device(buf.device)
                _lib.check(lib.ltxq_fp4_pack_weight_scales(ctypes.byref(q), buf.data_ptr(), _stream()),
                           "fp4_pack_weight_scales")
                if not recorded:
                    _wait_stream()
            if not recorded:
                self._fp4_packed = (self.scales, now, buf)
        return buf

    def computes_fp4(self) -> bool:
        """Whether products over this weight are of two fp4 operands."""
        return (getattr(self, "compute", "dequant") == "fp4" and self.mode in FP4_MODES and not self.pretransposed
                and self.in_features % 32 == 0)

    # ------------------------------------------------------------------ build
    @classmethod
    def from_linear(cls, weight: torch.Tensor, bias: torch.Tensor | None = None, group_size: int | None = None,
                    bits: int | None = None, mode: str = "affine", pretransposed: bool = False,
                    global_scale: float = 1.0) -> "QuantizedLinear":
        """Quantize a bf16 ``nn.Linear`` weight [out, in] on the GPU
        (``nn.QuantizedLinear.from_linear`` / ``mx.quantize``).
        ``global_scale`` (nvfp4): the tensor's scale, as
        ``kernels.fp4_global_scale(weight)`` picks one; 1 is the reference's
        cache layout, which has none."""
        _require_cuda(weight, "weight")
        if mode in FP4_MODES:
            with _on(weight):
                return cls._from_linear(weight, bias, group_size, bits, mode, pretransposed, global_scale)
        if global_scale != 1.0:
            raise ValueError("global_scale is nvfp4 only")
        return cls._from_linear(weight, bias, group_size, bits, mode, pretransposed, 1.0)

    @classmethod
    def _from_linear(cls, weight, bias, group_size, bits, mode, pretransposed, global_scale):
        gs, b = quant_defaults(mode, group_size, bits)
        w = weight.to(torch.bfloat16)
        n_out, k_in = w.shape
        src = w.t().contiguous() if pretransposed else w.contiguous()
        rows, length = src.shape
        packed = torch.empty((rows, length * b // 32), dtype=torch.uint32, device=w.device)
        if mode == "affine":
            scales = torch.empty((rows, length // gs), dtype=torch.bfloat16, device=w.device)
            biases = torch.empty_like(scales)
        else:
            scales = torch.empty((rows, length // gs), dtype=torch.uint8, device=w.device)
            biases = None
        q = _lib.QWeight(packed.data_ptr(), scales.data_ptr(), biases.data_ptr() if biases is not None else None,
                         None, n_out, k_in, _MODE[mode], b, gs,
                         _lib.LAYOUT_PRETRANSPOSED if pretransposed else _lib.LAYOUT_STD, global_scale=global_scale)
        _lib.check(_lib.load().ltxq_quantize(src.data_ptr(), ctypes.byref(q), _stream()), "quantize")
        bias_bf16 = bias.to(torch.bfloat16).contiguous() if bias is not None else None
        return cls(packed, scales, biases, bias_bf16, group_size=gs, bits=b, mode=mode,
                   pretransposed=pretransposed, in_features=k_in, out_features=n_out, global_scale=global_scale)

    # ------------------------------------------------------------------ views
    def _qweight_base(self, flags: int, mx_scales) -> _lib.QWeight:
        return _lib.QWeight(
            self.weight.data_ptr(), self.scales.data_ptr(),
            self.biases.data_ptr() if self.biases is not None else None,
            self.bias.data_ptr() if self.bias is not None else None,
            self.out_features, self.in_features, _MODE[self.mode], self.bits, self.group_size,
            _lib.LAYOUT_PRETRANSPOSED if self.pretransposed else _lib.LAYOUT_STD, flags,
            COMPUTE[getattr(self, "compute", "dequant")], mx_scales, getattr(self, "global_scale", 1.0))

    def qweight(self) -> _lib.QWeight:
        if self.mode in FP4_MODES:
            kept = self._qweight4()
            q = type(kept).from_buffer_copy(kept)
            q.packed = kept.packed
            return q
        mx = self.mx_scales()
        return self._qweight_base(self.data_flags(), mx.data_ptr() if mx is not None else None)

    def data_flags(self) -> int:
        """LTXQ_QW_* flags of the packed data (``ltxq_qweight_scan``), cached
        until the weight or scale tensors change (torch's in-place version
        counters).  ``fast_path = False`` asserts none (the general
        conversion everywhere)."""
        if self.mode != "mxfp8" or not getattr(self, "fast_path", True):
            return 0
        key = (self.weight.data_ptr(), self.weight._version, self.scales.data_ptr(), self.scales._version)
        cached = getattr(self, "_flags_cache", None)
        if cached is None or cached[0] != key:
            q = _lib.QWeight(self.weight.data_ptr(), self.scales.data_ptr(), None, None, self.out_features,
                             self.in_features, _MODE[self.mode], self.bits, self.group_size,
                             _lib.LAYOUT_PRETRANSPOSED if self.pretransposed else _lib.LAYOUT_STD, 0)
            flags = ctypes.c_uint32(0)
            _lib.check(_lib.load().ltxq_qweight_scan(ctypes.byref(q), ctypes.byref(flags), _stream()), "qweight_scan")
            cached = (key, int(flags.value))
            self._flags_cache = cached
        return cached[1]

    def dequantize(self) -> torch.Tensor:
        """bf16 weight: [out, in] (standard) or [in, out] (pretransposed)."""
        shape = (self.in_features, self.out_features) if self.pretransposed else (self.out_features, self.in_features)
        out = torch.empty(shape, dtype=torch.bfloat16, device=self.weight.device)
        if self.mode in FP4_MODES:
            self._check_fp4()
            q = self._qweight_base(0, None)  # reads the scales as they lie, not the packed ones
            with _on(self.weight):
                _lib.check(_lib.load().ltxq_dequantize(ctypes.byref(q), out.data_ptr(), _stream()), "dequantize")
            return out
        q = self.qweight()
        _lib.check(_lib.load().ltxq_dequantize(ctypes.byref(q), out.data_ptr(), _stream()), "dequantize")
        return out

    def mx_terms(self, M: int) -> int:
        """Terms of the MX input a GEMM of M rows over this weight takes (2 for
        "mx2", 1 for "mx1"), or 0 where it runs the dequantizing kernels (or
        the fp4 ones)."""
        if self.compute in ("dequant", "fp4") or M <= 0:
            return 0
        q = self.qweight()
        if not _lib.load().ltxq_qlinear_mx_supported(M, ctypes.byref(q)):
            return 0
        return 2 if self.compute == "mx2" else 1

    # ---------------------------------------------------------------- forward
    def _epilogue(self, x_rows_shape, keep, gelu=False, residual=None, gate=None, gate_then_add=False):
        epi = _lib.Epilogue()
        if residual is not None:
            if gate is None:
                raise ValueError("gated epilogue needs a gate")
            _require_cuda(residual, "residual")
            if residual.dtype != torch.bfloat16:
                raise ValueError("residual must be bfloat16")
            residual = residual.contiguous()
            keep.append(residual)
            if residual.numel() != math.prod(x_rows_shape) * self.out_features:
                raise ValueError("residual shape does not match the output")
            epi.kind = _lib.EPI_GATE_THEN_ADD if gate_then_add else _lib.EPI_GATED_RESIDUAL
            epi.gate = vec_arg(gate, x_rows_shape, self.out_features, "gate", keep)
            epi.residual = residual.data_ptr()
        else:
            epi.kind = _lib.EPI_GELU if gelu else _lib.EPI_NONE
        return epi

    def __call__(self, x: torch.Tensor, *, gelu: bool = False, residual: torch.Tensor | None = None,
                 gate: torch.Tensor | None = None, gate_then_add: bool = False,
                 adaln: tuple | None = None, split_k: bool = True, mx_out: int = 0):
        """``y = x @ dequant(W).T + bias`` with optional fused consumers:
        ``gelu=True`` (project_in), ``residual``/``gate`` (gated residual add),
        and ``adaln=(scale, shift, eps[, norm])`` (the AdaLN prologue).

        ``split_k=False`` gives the library no workspace for split-K partials,
        so a GEMM with few tokens runs unsplit (one pass over K per tile).

        ``x`` may be an ``MXActivation`` (``mx_terms(M)`` terms): the
        block-scaled GEMM reads it directly (``ltxq_qlinear_mx``).  With such
        an input, ``mx_out`` 1 or 2 returns the result (bias, GELU applied) as
        an ``MXActivation`` of that many terms for the next GEMM.

        With compute "fp4" on an mxfp4 / nvfp4 weight, ``x`` is quantized to
        the weight's format in the call (nvfp4: with global_scale 1, which
        saturates past 6 * 448), or comes as an ``FP4Tensor`` of it.  Many rows
        over such a weight otherwise (from 768 rows and 48 tiles of 256 x 256
        outputs on) take a workspace of the dequantized weight, 2 bytes per
        value (134 MB at 4096 x 16384), besides that of split-K partials."""
        if self.mode in FP4_MODES or isinstance(x, FP4Tensor):
            if mx_out:
                raise ValueError("mx_out needs an MXActivation input (the block-scaled fp8 kernels)")
            return self._call_fp4(x, gelu, residual, gate, gate_then_add, adaln, split_k)
        if isinstance(x, MXActivation):
            return self._call_mx(x, gelu, residual, gate, gate_then_add, mx_out)
        if mx_out:
            raise ValueError("mx_out needs an MXActivation input (the block-scaled kernels)")
        _require_cuda(x, "x")
        if x.dtype != torch.bfloat16:
            raise ValueError(f"x must be bfloat16, got {x.dtype}")
        if x.shape[-1] != self.in_features:
            raise ValueError(f"x last dim {x.shape[-1]} != in_features {self.in_features}")
        x = x.contiguous()
        rows_shape = tuple(x.shape[:-1])
        M = x.numel() // self.in_features
        keep: list = []
        epi = self._epilogue(rows_shape, keep, gelu, residual, gate, gate_then_add)
        out = torch.empty(rows_shape + (self.out_features,), dtype=torch.bfloat16, device=x.device)
        q = self.qweight()
        lib = _lib.load()
        if adaln is not None:
            scale, shift, eps = adaln[:3]
            norm = adaln[3] if len(adaln) > 3 else "rms"
            nk = {"rms": _lib.NORM_RMS, "layer": _lib.NORM_LAYER, "none": _lib.NORM_NONE}[norm]
            pro = prologue(nk, eps, scale, shift, rows_shape, self.in_features, keep)
            ws_bytes = lib.ltxq_adaln_qlinear_workspace_size(M, ctypes.byref(q))
            ws = torch.empty(max(ws_bytes, 1), dtype=torch.uint8, device=x.device)
            _lib.check(lib.ltxq_adaln_qlinear(x.data_ptr(), M, ctypes.byref(pro), ctypes.byref(q), ctypes.byref(epi),
                                              out.data_ptr(), ws.data_ptr(), ws_bytes, _stream()), "adaln_qlinear")
        else:
            ws_bytes = lib.ltxq_qlinear_workspace_size(M, ctypes.byref(q)) if split_k else 0
            ws = torch.empty(ws_bytes, dtype=torch.uint8, device=x.device) if ws_bytes else None
            _lib.check(lib.ltxq_qlinear(x.data_ptr(), M, ctypes.byref(q), ctypes.byref(epi), out.data_ptr(),
                                        ws.data_ptr() if ws is not None else None, ws_bytes, _stream()), "qlinear")
        return out

    def _qweight4(self) -> _lib.QWeight:
        """``qweight()`` of an fp4 weight, kept for its arrays and settings (the
        objects, where they lie and their shapes: an address alone may be
        another array's by now) and made and checked again for others.  The
        packed scales are brought up to date first: their memory may have been
        packed for other scales since (by another reader of this weight),
        which no pointer shows."""
        w, s, b = self.weight, self.scales, self.bias
        key = (w.data_ptr(), w.shape, s.data_ptr(), s.shape, (b.data_ptr(), b.shape) if b is not None else None,
               self.out_features, self.in_features, self.mode, self.bits, self.group_size, self.pretransposed,
               self.compute, self.global_scale)
        kept = self._q4
        if kept is not None and kept[0] is w and kept[1] is s and kept[2] is b and kept[3] == key:
            q = kept[4]
            if q.packed is None:
                return q
            scales, state, buf = self._fp4_packed
            if scales is s and buf is q.packed and state == (key[2], _version(s)):
                return q
        self._check_fp4()
        packed = self._fp4_scales() if self.computes_fp4() else None
        q = self._qweight_base(0, packed.data_ptr() if packed is not None else None)
        q.packed = packed  # memory of a recorded packing belongs to this descriptor alone
        if packed is None or packed is self._fp4_packed[2]:
            self._q4 = (w, s, b, key, q)
        return q

    def __getstate__(self):
        """Copies make their own: the descriptor holds addresses, and memory for
        packed scales belongs to one weight."""
        return {k: v for k, v in self.__dict__.items() if k not in ("_q4", "_fp4_packed")}

    def _call_fp4(self, x, gelu, residual, gate, gate_then_add, adaln, split_k):
        """Products over an mxfp4 / nvfp4 weight, from bf16 rows or an ``FP4Tensor``."""
        packed = isinstance(x, FP4Tensor)
        if packed:
            if not self.computes_fp4() or x.mode != self.mode:
                raise ValueError(f"an {x.mode} input needs an {x.mode} weight whose compute is 'fp4' (weight: "
                                 f"{self.mode}, compute: {self.compute})")
            if adaln is not None:
                raise ValueError("adaln takes bf16 activations")
            device = x.buffer.device
        else:
            if isinstance(x, MXActivation):
                raise ValueError("an MXActivation input needs an mxfp8 weight")
            _require_cuda(x, "x")
            if x.dtype != torch.bfloat16:
                raise ValueError(f"x must be bfloat16, got {x.dtype}")
            device = x.device
        dev = self.weight.get_device()
        if device.index != dev:
            raise ValueError(f"x is on {device}, the weight on {self.weight.device}")
        if x.shape[-1] != self.in_features:
            raise ValueError(f"x last dim {x.shape[-1]} != in_features {self.in_features}")
        if residual is not None or adaln is not None:
            for t in (residual, gate, *(adaln[:2] if adaln is not None else ())):
                if hasattr(t, "get_device") and t.get_device() != dev:  # what is no tensor is refused below
                    raise ValueError(f"residual, gate, scale and shift must be on the weight's device "
                                     f"({self.weight.device}), got {t.device}")
        if dev != _device():
            with torch.cuda.device(dev):
                return self._call_fp4(x, gelu, residual, gate, gate_then_add, adaln, split_k)
        rows_shape = x.shape[:-1]
        out = (x.buffer if packed else x).new_empty((*rows_shape, self.out_features), dtype=torch.bfloat16)
        M = x.M if packed else x.numel() // self.in_features
        if M == 0:
            return out
        keep: list = []
        epi = None  # no epilogue
        if gelu or residual is not None:
            epi = self._epilogue(tuple(rows_shape), keep, gelu, residual, gate, gate_then_add)
        q, lib, stream = self._qweight4(), _lib.load(), _raw_stream(dev)
        if packed:
            _lib.check(lib.ltxq_qlinear_fp4(x.struct(), M, q, epi, out.data_ptr(), stream), "qlinear_fp4")
            return out
        if not x.is_contiguous() or x.data_ptr() % 16:
            x = x.clone(memory_format=torch.contiguous_format)
        pro = None
        if adaln is not None:
            norm = {"rms": _lib.NORM_RMS, "layer": _lib.NORM_LAYER, "none": _lib.NORM_NONE}[
                adaln[3] if len(adaln) > 3 else "rms"]
            pro = prologue(norm, adaln[2], adaln[0], adaln[1], tuple(rows_shape), self.in_features, keep)
            ws_bytes = lib.ltxq_adaln_qlinear_workspace_size(M, q)
        else:
            ws_bytes = (lib.ltxq_qlinear_workspace_size if split_k else lib.ltxq_qlinear_unsplit_workspace_size)(M, q)
        ws = out.new_empty((ws_bytes,), dtype=torch.uint8) if ws_bytes else None
        ws_ptr = ws.data_ptr() if ws is not None else None
        if pro is not None:
            _lib.check(lib.ltxq_adaln_qlinear(x.data_ptr(), M, pro, q, epi, out.data_ptr(), ws_ptr, ws_bytes, stream),
                       "adaln_qlinear")
        else:
            _lib.check(lib.ltxq_qlinear(x.data_ptr(), M, q, epi, out.data_ptr(), ws_ptr, ws_bytes, stream), "qlinear")
        return out

    def _call_mx(self, x: MXActivation, gelu, residual, gate, gate_then_add, mx_out):
        if x.K != self.in_features:
            raise ValueError(f"x last dim {x.K} != in_features {self.in_features}")
        if mx_out and residual is not None:
            raise ValueError("mx_out takes the none / GELU epilogues only")
        keep: list = []
        epi = self._epilogue(x.rows_shape, keep, gelu, residual, gate, gate_then_add)
        q = self.qweight()
        xs = x.struct()
        out = None
        out_struct = None
        if mx_out:
            out = MXActivation(x.rows_shape, self.out_features, mx_out, x.device)
            out_struct = out.struct()
            out_ptr = None
        else:
            out = torch.empty(x.rows_shape + (self.out_features,), dtype=torch.bfloat16, device=x.device)
            out_ptr = out.data_ptr()
        _lib.check(_lib.load().ltxq_qlinear_mx(ctypes.byref(xs), x.M, ctypes.byref(q), ctypes.byref(epi), out_ptr,
                                               ctypes.byref(out_struct) if out_struct is not None else None,
                                               _stream()), "qlinear_mx")
        return out

    def __repr__(self) -> str:
        return (f"QuantizedLinear(in={self.in_features}, out={self.out_features}, mode={self.mode}, "
                f"bits={self.bits}, group_size={self.group_size}, pretransposed={self.pretransposed})")
