"""MXFP4 (microscaled 4-bit floating point): quantisation and expert weights.

No counterpart in the reference, whose experts are BF16.  A block of 32 values
along the last axis shares one E8M0 scale byte ``b`` (``2**(b - 127)``); each
value is an E2M1 code (0, .5, 1, 1.5, 2, 3, 4, 6 with a sign bit), two per
byte, the even element in the low nibble: 4.25 bits per value.  ``quantize_mxfp4``
sets ``b = max(floor(log2 max|x|) - 2 + 127, 0)`` and rounds to nearest even,
saturating at 6.  An expert of an ``Mxfp4ExpertSlab`` takes 0.27 of its BF16
bytes, which is what a decode step streams.
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass

import torch

from . import _lib
from ._lib import Mxfp4Weights, lib
from .runtime import PROJECTIONS, Packed, _call, _require_cuda_bf16, check_slab, ffn_workspace_bytes

BLOCK = 32
_DTYPES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_FP16, torch.float32: _lib.DTYPE_FP32}


@dataclass
class Mxfp4:
    """Quantised tensor: ``codes`` uint8 [..., K/2], ``scales`` uint8 [..., K/32]."""
    codes: torch.Tensor
    scales: torch.Tensor

    @property
    def shape(self):
        return torch.Size((*self.codes.shape[:-1], self.codes.shape[-1] * 2))


def _matrix(x):
    """(rows, columns, row stride) of a tensor read as a matrix of its last axis."""
    cols = x.shape[-1]
    rows = x.numel() // cols if cols else 0
    if x.is_contiguous():
        return rows, cols, cols
    if x.ndim == 2 and x.stride(1) == 1 and x.stride(0) >= cols:
        return rows, cols, x.stride(0)
    raise ValueError("x must be contiguous, or a matrix with contiguous rows")


def quantize_mxfp4(x):
    """MXFP4 of a BF16, FP16 or FP32 CUDA tensor along its last axis (a multiple
    of 32).  A matrix may have a row stride; a block holding an infinity or NaN
    reads back as NaN."""
    if not isinstance(x, torch.Tensor) or not x.is_cuda or x.dtype not in _DTYPES:
        raise ValueError("x must be a BF16, FP16 or FP32 CUDA tensor")
    shape = x.shape
    if len(shape) < 1 or shape[-1] < 1 or shape[-1] % BLOCK:
        raise ValueError("the last axis must be a positive multiple of 32")
    rows, cols, ld = _matrix(x)
    codes = x.new_empty((*shape[:-1], cols // 2), dtype=torch.uint8)
    scales = x.new_empty((*shape[:-1], cols // BLOCK), dtype=torch.uint8)
    _call(x.device, lib.pdx_mxfp4_quantize, x.data_ptr(), _DTYPES[x.dtype], rows, cols, ld, codes.data_ptr(),
          scales.data_ptr())
    return Mxfp4(codes, scales)


def _require_mxfp4(name, q, ndim=None):
    if not isinstance(q, Mxfp4):
        raise ValueError(f"{name} must be an Mxfp4")
    for t in (q.codes, q.scales):
        if not t.is_cuda or t.dtype != torch.uint8 or not t.is_contiguous():
            raise ValueError(f"{name} must hold contiguous uint8 CUDA tensors")
    shape = q.codes.shape
    if (q.codes.device != q.scales.device or len(shape) < 1 or shape[-1] < 1 or shape[-1] % (BLOCK // 2)
            or q.scales.shape != (*shape[:-1], shape[-1] * 2 // BLOCK) or (ndim is not None and len(shape) != ndim)):
        raise ValueError(f"{name}: codes must be [..., K/2] and scales [..., K/32], K a positive multiple of 32")


def dequantize_mxfp4(q, dtype=torch.bfloat16):
    """The values an ``Mxfp4`` stands for, rounded to ``dtype`` (BF16 and FP32
    hold them exactly, but for FP32's and BF16's own range)."""
    _require_mxfp4("q", q)
    if dtype not in _DTYPES:
        raise ValueError("dtype must be BF16, FP16 or FP32")
    shape = q.shape
    out = q.codes.new_empty(shape, dtype=dtype)
    cols = shape[-1]
    _call(out.device, lib.pdx_mxfp4_dequantize, q.codes.data_ptr(), q.scales.data_ptr(), out.numel() // cols, cols, cols,
          _DTYPES[dtype], out.data_ptr())
    return out


def _round128(n):
    return (n + 127) // 128 * 128


class Mxfp4ExpertSlab:
    """MXFP4 experts of one layer in equal slots (``pdx_mxfp4_weights``): the
    4-bit counterpart of ``ExpertSlab``, accepted wherever the layer, the stack
    and the PDScope runtime take a slab.

    ``hidden`` and ``inter`` are multiples of 32; a slot's rows and columns are
    padded with zeros to multiples of 128, and codes and scales are stored as
    the 128 x 128 tiles that a product streams (each tile one run of memory).  ``slot_of_expert`` (int32 CUDA [E],
    optional) maps expert ids to slots."""

    def __init__(self, num_slots, hidden, inter, device, slot_of_expert=None):
        if num_slots < 1 or hidden < BLOCK or inter < BLOCK or hidden % BLOCK or inter % BLOCK:
            raise ValueError("hidden and inter must be positive multiples of 32")
        self.num_slots, self.hidden, self.inter = num_slots, hidden, inter
        self.slot_of_expert = slot_of_expert
        self._hp, self._ip = _round128(hidden), _round128(inter)
        per = self._hp * self._ip
        self.codes = torch.zeros((num_slots, 3 * per // 2), dtype=torch.uint8, device=device)
        self.scales = torch.zeros((num_slots, 3 * per // BLOCK), dtype=torch.uint8, device=device)
        if slot_of_expert is not None and (slot_of_expert.dtype != torch.int32 or slot_of_expert.ndim != 1
                                           or slot_of_expert.device != self.codes.device
                                           or not slot_of_expert.is_contiguous()):
            raise ValueError("slot_of_expert must be a contiguous int32 vector on the slab's device")
        self.struct = Mxfp4Weights(codes=self.codes.data_ptr(), scales=self.scales.data_ptr(),
                                   code_stride=3 * per // 2, scale_stride=3 * per // BLOCK, num_slots=num_slots,
                                   slot_of_expert=slot_of_expert.data_ptr() if slot_of_expert is not None else None)

    def _tiles(self, slots, j):
        """Code tiles [n, row tile, column tile, r, byte] and scale tiles
        [n, row tile, column tile, r % 32, r / 32, c / 32] of projection j."""
        rows, cols = (self._ip, self._hp) if j < 2 else (self._hp, self._ip)
        grid, per = (-1, rows // 128, cols // 128), self._hp * self._ip
        return (self.codes[slots, j * per // 2:(j + 1) * per // 2].view(*grid, 128, 64),
                self.scales[slots, j * per // BLOCK:(j + 1) * per // BLOCK].view(*grid, 32, 4, 4))

    def _shape(self, j):
        return (self.inter, self.hidden) if j < 2 else (self.hidden, self.inter)

    def store(self, first, gate, up, down):
        """Write the experts ``gate``, ``up`` [n, I, H] and ``down`` [n, H, I] (Mxfp4) into slots first .. first+n-1."""
        for j, (name, q) in enumerate(zip(PROJECTIONS, (gate, up, down))):
            _require_mxfp4(name, q, 3)
            n = q.codes.shape[0]
            if q.shape[1:] != self._shape(j) or n != gate.codes.shape[0] or first < 0 or first + n > self.num_slots:
                raise ValueError(f"{name} does not fit the slab's slots")
            rows, cols = self._shape(j)
            codes, scales = self._tiles(slice(first, first + n), j)
            nr, nc = codes.shape[1:3]
            c = torch.zeros((n, nr * 128, nc * 64), dtype=torch.uint8, device=q.codes.device)
            c[:, :rows, :cols // 2] = q.codes
            codes.copy_(c.view(n, nr, 128, nc, 64).transpose(2, 3))
            s = torch.zeros((n, nr * 128, nc * 4), dtype=torch.uint8, device=q.scales.device)
            s[:, :rows, :cols // BLOCK] = q.scales
            scales.copy_(s.view(n, nr, 4, 32, nc, 4).permute(0, 1, 4, 3, 2, 5))

    def load(self, slot):
        """The slot's experts as {gate_proj, up_proj, down_proj} Mxfp4 matrices."""
        out = {}
        for j, name in enumerate(PROJECTIONS):
            rows, cols = self._shape(j)
            codes, scales = self._tiles(slice(slot, slot + 1), j)
            nr, nc = codes.shape[1:3]
            c = codes[0].transpose(1, 2).reshape(nr * 128, nc * 64)
            s = scales[0].permute(0, 3, 2, 1, 4).reshape(nr * 128, nc * 4)
            out[name] = Mxfp4(c[:rows, :cols // 2].contiguous(), s[:rows, :cols // BLOCK].contiguous())
        return out

    def expert_tensors(self, slot):
        """One slot's weights as BF16 tensors, as ``ExpertSlab.expert_tensors`` returns them."""
        return {name: dequantize_mxfp4(q) for name, q in self.load(slot).items()}

    @classmethod
    def from_quantized(cls, gate, up, down, slot_of_expert=None):
        """Lay out the quantised projections ``gate``, ``up`` [E, I, H] and ``down`` [E, H, I]."""
        _require_mxfp4("gate", gate, 3)
        experts, inter, hidden = gate.shape
        slab = cls(experts, hidden, inter, gate.codes.device, slot_of_expert)
        slab.store(0, gate, up, down)
        return slab

    @classmethod
    def from_tensors(cls, experts, slot_of_expert=None):
        """Quantise a list of {gate_proj, up_proj, down_proj} dicts (BF16, FP16 or FP32 CUDA matrices)."""
        g0 = experts[0]["gate_proj"]
        inter, hidden = g0.shape
        slab = cls(len(experts), hidden, inter, g0.device, slot_of_expert)
        for s, ex in enumerate(experts):
            qs = [quantize_mxfp4(ex[name]) for name in PROJECTIONS]
            slab.store(s, *(Mxfp4(q.codes.unsqueeze(0), q.scales.unsqueeze(0)) for q in qs))
        return slab

    @classmethod
    def from_slab(cls, slab):
        """Quantise a BF16 ``ExpertSlab``, slot by slot."""
        out = cls(slab.num_slots, slab.hidden, slab.inter, slab.storage.device, slab.slot_of_expert)
        for s in range(slab.num_slots):
            qs = [quantize_mxfp4(t) for t in (slab.expert_tensors(s)[name] for name in PROJECTIONS)]
            out.store(s, *(Mxfp4(q.codes.unsqueeze(0), q.scales.unsqueeze(0)) for q in qs))
        return out


def moe_ffn_mxfp4(x, packed, slab, out=None):
    """Unweighted expert rows [T*k, H] of a packed batch on MXFP4 experts:
    ``out[p] = down(silu(gate(x[t])) * up(x[t]))`` for packed row p of token t,
    with exact weights and FP32 sums.  Rounded are the result, once to BF16; the
    input of ``down``, to within 2**-9 of each value or 2**-21 of the largest of its
    32; and values of x below 2**-13 of the largest of their 32, by 2**-21 of that
    one at most.  A row of x with an infinity or NaN gives rows of NaN.  ``packed``
    is ``pack``'s result for the batch ``x`` [T, H]."""
    _require_cuda_bf16("x", x, 2)
    t_count, hidden = x.shape
    if not isinstance(slab, Mxfp4ExpertSlab) or not isinstance(packed, Packed):
        raise ValueError("moe_ffn_mxfp4 needs pack()'s result and an Mxfp4ExpertSlab")
    experts = packed.counts.shape[0]
    check_slab(slab, experts, hidden, x.device)
    if packed.tokens.device != x.device:
        raise ValueError("x, the packing and the slab must be on one device")
    rows = packed.tokens.shape[0]
    if t_count < 1 or rows % t_count:
        raise ValueError("the packing does not belong to this batch")
    if out is None:
        out = x.new_empty((rows, hidden))
    else:
        _require_cuda_bf16("out", out, 2)
        if out.shape != (rows, hidden) or out.device != x.device:
            raise ValueError("out must be [T*k, H] on the device of x")
    # from the stream-ordered allocator: calls on two streams or in two graphs share no scratch
    nbytes = ffn_workspace_bytes(slab, rows, experts)
    ws = x.new_empty((nbytes,), dtype=torch.uint8)
    _call(x.device, lib.pdx_mxfp4_ffn_grouped, x.data_ptr(), t_count, packed.tokens.data_ptr(),
          packed.offsets.data_ptr(), packed.active.data_ptr(), experts, rows, ctypes.byref(slab.struct), hidden,
          slab.inter, out.data_ptr(), ws.data_ptr(), nbytes)
    return out
