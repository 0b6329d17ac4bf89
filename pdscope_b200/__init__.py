"""B200-native (sm_100a) MoE expert execution path for PDScope.

The compute lives in ``libpdx_moe.so`` (C ABI: include/pdx_moe.h); ``_lib``
binds it and ``runtime`` mirrors the reference's Python interface.  Importing
the package itself does not load the library (so ``pdscope_b200.build`` can
rebuild it); the first use of any runtime name loads it and raises if it is
missing -- there is no fallback.
"""
_RUNTIME_NAMES = ("PDScopeCudaRuntime", "PdxGpuBackend", "ExpertSlab", "ResidentMoELayer", "Routing", "combine",
                  "compact_expert_groups", "expert_forward", "expert_groups", "pack", "route", "topk_from_logits",
                  "BlockNorm", "block_norm", "combine_block_norm")
_MXFP4_NAMES = ("Mxfp4", "Mxfp4ExpertSlab", "dequantize_mxfp4", "moe_ffn_mxfp4", "quantize_mxfp4")


def __getattr__(name):
    if name in _RUNTIME_NAMES:
        from . import runtime as module
    elif name in _MXFP4_NAMES:
        from . import mxfp4 as module
    else:
        raise AttributeError(name)
    value = globals()[name] = getattr(module, name)   # later uses find it without this function
    return value
