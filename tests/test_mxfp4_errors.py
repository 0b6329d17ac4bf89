"""Refusals of the MXFP4 and block-norm entry points, on the CPU: the Python
checks raise ValueError, the C ABI returns its status, before any device work."""
import ctypes

import numpy as np
import pytest
import torch

import pdscope_b200 as pdx
from pdscope_b200 import _lib
from pdscope_b200.stack import ResidentMoEStack
from tests import mxfp4_ref as ref

PTR, NULL = ctypes.c_void_p(256), ctypes.c_void_p(0)


def test_definition_round_trip():
    """The 64-bit definition: halves round to even, the largest value fills [4, 8)."""
    x = np.array([4.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.9] + [0.0] * 23)
    codes, scales = ref.quantize(x)
    assert scales.tolist() == [127]
    assert ref.dequantize(codes, scales)[:9].tolist() == [4.0, 0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, 6.0]


@pytest.mark.parametrize("x", (torch.zeros(4, 64), torch.zeros(4, 64, dtype=torch.int32), None))
def test_quantize_refuses(x):
    with pytest.raises(ValueError):
        pdx.quantize_mxfp4(x)


def test_dequantize_refuses():
    with pytest.raises(ValueError):
        pdx.dequantize_mxfp4(torch.zeros(4, 32, dtype=torch.uint8))
    with pytest.raises(ValueError):
        pdx.dequantize_mxfp4(pdx.Mxfp4(torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.uint8)))


@pytest.mark.parametrize("cols,rows,ld,dtype", ((31, 4, 31, 0), (0, 4, 0, 0), (64, -1, 64, 0), (64, 4, 63, 0),
                                                (64, 4, 64, 3), (64, 4, 64, -1)))
def test_matrix_status(cols, rows, ld, dtype):
    assert _lib.lib.pdx_mxfp4_quantize(PTR, dtype, rows, cols, ld, PTR, PTR, NULL) == _lib.PDX_ERR_INVALID
    assert _lib.lib.pdx_mxfp4_dequantize(PTR, PTR, rows, cols, ld, dtype, PTR, NULL) == _lib.PDX_ERR_INVALID


def test_null_and_unaligned_status():
    assert _lib.lib.pdx_mxfp4_quantize(NULL, 0, 1, 32, 32, PTR, PTR, NULL) == _lib.PDX_ERR_INVALID
    assert _lib.lib.pdx_mxfp4_quantize(PTR, 0, 1, 32, 32, ctypes.c_void_p(258), PTR, NULL) == _lib.PDX_ERR_INVALID
    assert _lib.lib.pdx_mxfp4_quantize(NULL, 0, 0, 32, 32, NULL, NULL, NULL) == _lib.PDX_OK


def _weights(**kw):
    d = dict(codes=256, scales=256, code_stride=3 * 128 * 128 // 2, scale_stride=3 * 128 * 4, num_slots=2)
    d.update(kw)
    return _lib.Mxfp4Weights(**d)


def _ffn(w, hidden=128, inter=128, tokens=2, rows=4, experts=2, gathered=True, ws=PTR, nbytes=1 << 40):
    return _lib.lib.pdx_mxfp4_ffn_grouped(PTR, tokens, PTR if gathered else NULL, PTR, PTR, experts, rows,
                                          ctypes.byref(w), hidden, inter, PTR, ws, nbytes, NULL)


def test_ffn_status():
    assert _ffn(_weights(), tokens=0) == _lib.PDX_ERR_INVALID
    assert _ffn(_weights(), rows=0) == _lib.PDX_ERR_INVALID
    assert _ffn(_weights(), hidden=48) == _lib.PDX_ERR_UNSUPPORTED
    assert _ffn(_weights(), inter=16) == _lib.PDX_ERR_UNSUPPORTED
    assert _ffn(_weights(), gathered=False) == _lib.PDX_ERR_INVALID
    assert _ffn(_weights(codes=None)) == _lib.PDX_ERR_INVALID
    assert _ffn(_weights(codes=264)) == _lib.PDX_ERR_INVALID
    assert _ffn(_weights(num_slots=0)) == _lib.PDX_ERR_INVALID
    assert _ffn(_weights(), experts=1025) == _lib.PDX_ERR_UNSUPPORTED
    assert _ffn(_weights(scale_stride=3 * 128 * 4 + 16)) == _lib.PDX_ERR_INVALID
    assert _ffn(_weights(num_slots=1 << 23)) == _lib.PDX_ERR_UNSUPPORTED
    assert _lib.lib.pdx_mxfp4_ffn_grouped(ctypes.c_void_p(264), 2, PTR, PTR, PTR, 2, 4, ctypes.byref(_weights()), 128,
                                          128, PTR, PTR, 1 << 40, NULL) == _lib.PDX_ERR_INVALID
    assert _ffn(_weights(code_stride=128)) == _lib.PDX_ERR_INVALID
    assert _ffn(_weights(), ws=NULL) == _lib.PDX_ERR_WORKSPACE
    assert _ffn(_weights(), ws=ctypes.c_void_p(128)) == _lib.PDX_ERR_WORKSPACE
    assert _ffn(_weights(), nbytes=64) == _lib.PDX_ERR_WORKSPACE


def test_workspace_queries():
    lib = _lib.lib
    for shape in ((1, 128, 32, 32), (512, 128, 2048, 768), (99600, 128, 2048, 768)):
        assert lib.pdx_mxfp4_ffn_workspace_bytes(*shape) > 0
    assert (lib.pdx_mxfp4_layer_workspace_bytes(64, 2048, 128, 8, 768)
            >= lib.pdx_mxfp4_ffn_workspace_bytes(512, 128, 2048, 768) + 512 * 2048 * 2)


def _norm(args, tokens=2, hidden=64, y=PTR, residual=PTR, stream=PTR, normed=PTR):
    return _lib.lib.pdx_block_norm(y, residual, tokens, hidden, ctypes.byref(args), stream, normed, NULL)


def test_block_norm_status():
    def a(**kw):
        return _lib.BlockNormArgs(**dict(dict(eps=1e-6, pre=1, residual_scale=1, block_scale=1), **kw))
    assert _norm(a(), tokens=0) == _lib.PDX_ERR_INVALID
    assert _norm(a(), residual=NULL) == _lib.PDX_ERR_INVALID
    assert _norm(a(), stream=NULL, normed=NULL) == _lib.PDX_ERR_INVALID
    assert _norm(a(), hidden=0) == _lib.PDX_ERR_UNSUPPORTED
    assert _norm(a(), hidden=8193) == _lib.PDX_ERR_UNSUPPORTED
    assert _norm(a(post=3)) == _lib.PDX_ERR_INVALID
    assert _norm(a(pre=-1)) == _lib.PDX_ERR_INVALID
    assert _norm(a(eps=0)) == _lib.PDX_ERR_INVALID
    assert _norm(a(eps=float("nan"))) == _lib.PDX_ERR_INVALID
    assert _norm(a(gate=256, gate_row=-1)) == _lib.PDX_ERR_INVALID
    combine = _lib.lib.pdx_combine_block_norm
    args = a()
    assert combine(PTR, 4, PTR, NULL, 2, 2, 64, PTR, ctypes.byref(args), PTR, PTR, NULL) == _lib.PDX_ERR_INVALID
    assert combine(PTR, 4, PTR, PTR, 2, 0, 64, PTR, ctypes.byref(args), PTR, PTR, NULL) == _lib.PDX_ERR_INVALID
    assert combine(PTR, 4, PTR, PTR, 2, 33, 64, PTR, ctypes.byref(args), PTR, PTR, NULL) == _lib.PDX_ERR_UNSUPPORTED


def test_block_status():
    args = _lib.BlockNormArgs(eps=1e-6, pre=1)
    w, w4 = _lib.ExpertWeights(), _weights()

    def block(bf16, mx, mode=0):
        return _lib.lib.pdx_moe_block(PTR, PTR, 2, 128, 4, 2, 1, ctypes.byref(w) if bf16 else None,
                                      ctypes.byref(w4) if mx else None, 128, PTR, ctypes.byref(args), PTR, PTR, NULL,
                                      NULL, NULL, NULL, mode, PTR, 1 << 40, NULL)
    assert block(False, False) == _lib.PDX_ERR_INVALID
    assert block(True, True) == _lib.PDX_ERR_INVALID
    assert block(False, True, mode=2) == _lib.PDX_ERR_INVALID


def test_block_norm_refuses():
    x = torch.zeros(2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="residual"):
        pdx.block_norm(x, x)
    with pytest.raises(ValueError, match="either norm"):
        pdx.block_norm(x, x, norm=pdx.BlockNorm(), post="rms")
    for bad, match in ((dict(post="batch"), "post and pre"), (dict(gate_act="tanh"), "gate_act"),
                       (dict(post_weight=x[0]), "post_weight"), (dict(gate=torch.zeros(3, 64)), "gate")):
        with pytest.raises(ValueError, match=match):
            pdx.BlockNorm(**bad).args(2, 64, torch.bfloat16, x.device)
    for shape in ((3, 64), (2, 32), (1, 2, 64)):
        with pytest.raises(ValueError, match="broadcast"):
            pdx.BlockNorm(gate=torch.zeros(shape, dtype=torch.bfloat16)).args(2, 64, torch.bfloat16, x.device)
    a = pdx.BlockNorm(gate=torch.zeros(2, 1, dtype=torch.bfloat16)).args(2, 64, torch.bfloat16, x.device)
    assert (a.gate_row, a.gate_col) == (1, 0)


def test_slab_refuses():
    for hidden, inter in ((48, 64), (64, 0), (0, 64)):
        with pytest.raises(ValueError):
            pdx.Mxfp4ExpertSlab(1, hidden, inter, "cpu")
    with pytest.raises(ValueError):
        pdx.Mxfp4ExpertSlab(2, 64, 64, "cpu", slot_of_expert=torch.zeros(2))
    slab = pdx.Mxfp4ExpertSlab(2, 64, 64, "cpu")
    with pytest.raises(ValueError):
        pdx.moe_ffn_mxfp4(torch.zeros(2, 64, dtype=torch.bfloat16), None, slab)


def test_stack_refuses_norms():
    gate = torch.zeros(4, 64, dtype=torch.bfloat16)
    slab = pdx.Mxfp4ExpertSlab(4, 64, 64, "cpu")
    with pytest.raises(ValueError, match="norms"):
        ResidentMoEStack([gate], [slab], norms=[pdx.BlockNorm()])
    with pytest.raises(ValueError, match="residual_dtype"):
        ResidentMoEStack([gate], [slab], residual_dtype=torch.float32)
    with pytest.raises(ValueError, match="residual stream"):
        ResidentMoEStack([gate], [slab]).residual(1)


def test_expert_parallel_refuses_mxfp4():
    from pdscope_b200.expert_parallel import ExpertParallelMoE
    gate = torch.zeros(4, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="BF16 experts"):
        ExpertParallelMoE(gate, pdx.Mxfp4ExpertSlab(4, 64, 64, "cpu"), rank=0, world=1)


def _bf16_slab(slots, hidden, inter, slot_of_expert=None):
    """What a BF16 slab shows of itself, on the CPU (an ExpertSlab needs a CUDA tensor)."""
    from types import SimpleNamespace
    return SimpleNamespace(hidden=hidden, inter=inter, num_slots=slots, slot_of_expert=slot_of_expert,
                           storage=torch.zeros(1, dtype=torch.bfloat16), struct=_lib.ExpertWeights())


def test_stack_refuses_slabs_that_do_not_fit():
    gate = torch.zeros(4, 64, dtype=torch.bfloat16)
    slab, short = pdx.Mxfp4ExpertSlab(4, 64, 64, "cpu"), torch.zeros(3, dtype=torch.int32)
    ResidentMoEStack([gate, gate], [slab, pdx.Mxfp4ExpertSlab(4, 64, 96, "cpu")])      # sizes of I may differ
    ResidentMoEStack([gate, gate], [slab, _bf16_slab(4, 64, 96)])
    for bad, match in ((pdx.Mxfp4ExpertSlab(4, 32, 64, "cpu"), "hidden"), (pdx.Mxfp4ExpertSlab(3, 64, 64, "cpu"), "fewer"),
                       (pdx.Mxfp4ExpertSlab(4, 64, 64, "cpu", slot_of_expert=short), "fewer"),
                       (pdx.Mxfp4ExpertSlab(4, 64, 64, "meta"), "device"),
                       (_bf16_slab(4, 32, 64), "hidden"), (_bf16_slab(4, 64, 64, short), "fewer"),
                       (_bf16_slab(4, 64, 64, torch.zeros(4, dtype=torch.int32, device="meta")), "device")):
        with pytest.raises(ValueError, match=match):
            ResidentMoEStack([gate, gate], [slab, bad])
    with pytest.raises(ValueError, match="alike"):
        ResidentMoEStack([gate, torch.zeros(5, 64, dtype=torch.bfloat16)], [slab, slab])
    # fewer slots than experts is an error of the routing, not of a BF16 slab, which may be any object of the sizes
    ResidentMoEStack([gate], [_bf16_slab(3, 64, 64)])
    bare = _bf16_slab(4, 64, 64)
    del bare.storage, bare.slot_of_expert
    ResidentMoEStack([gate], [bare])


@pytest.mark.parametrize("dtype,at", ((0, 257), (1, 257), (2, 258), (2, 257)))
def test_matrix_refuses_split_elements(dtype, at):
    """A pointer between two elements would fault on the device."""
    odd = ctypes.c_void_p(at)
    assert _lib.lib.pdx_mxfp4_quantize(odd, dtype, 1, 32, 32, PTR, PTR, NULL) == _lib.PDX_ERR_INVALID
    assert _lib.lib.pdx_mxfp4_dequantize(PTR, PTR, 1, 32, 32, dtype, odd, NULL) == _lib.PDX_ERR_INVALID


def test_block_norm_refuses_split_elements():
    def a(**kw):
        return _lib.BlockNormArgs(**dict(dict(eps=1e-6, pre=1, residual_scale=1, block_scale=1), **kw))
    odd, half = ctypes.c_void_p(257), ctypes.c_void_p(258)
    assert _norm(a(), y=odd) == _lib.PDX_ERR_INVALID
    assert _norm(a(), residual=odd) == _lib.PDX_ERR_INVALID
    assert _norm(a(residual_fp32=1), residual=half) == _lib.PDX_ERR_INVALID
    assert _norm(a(residual_fp32=1), stream=half) == _lib.PDX_ERR_INVALID
    assert _norm(a(), normed=odd) == _lib.PDX_ERR_INVALID
    for name in ("post_weight", "pre_weight", "gate"):
        assert _norm(a(**{name: 257})) == _lib.PDX_ERR_INVALID
    args = a()
    for rows, weights, inverse in ((odd, PTR, PTR), (PTR, odd, PTR), (PTR, PTR, half)):
        assert _lib.lib.pdx_combine_block_norm(rows, 4, weights, inverse, 2, 2, 64, PTR, ctypes.byref(args), PTR, PTR,
                                               NULL) == _lib.PDX_ERR_INVALID


def test_ffn_refuses_split_elements_and_huge_slabs():
    half, w = ctypes.c_void_p(258), _weights()
    for tokens, offsets, active in ((half, PTR, PTR), (PTR, half, PTR), (PTR, PTR, half)):
        assert _lib.lib.pdx_mxfp4_ffn_grouped(PTR, 2, tokens, offsets, active, 2, 4, ctypes.byref(w), 128, 128, PTR, PTR,
                                              1 << 40, NULL) == _lib.PDX_ERR_INVALID
    assert _ffn(_weights(slot_of_expert=258)) == _lib.PDX_ERR_INVALID
    # slots x tiles past 64 bits: 384 rows of codes a slot x 2^57 slots = 3 2^64
    assert _ffn(_weights(num_slots=1 << 57)) == _lib.PDX_ERR_UNSUPPORTED
    assert _ffn(_weights(num_slots=(1 << 63) - 1)) == _lib.PDX_ERR_UNSUPPORTED
