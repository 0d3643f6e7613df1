"""modelc_b200 -- B200-native (sm_100a) speculative-decoding step for modelc.

The compute path is ``libmodelc_cuda.so`` (hand-written CUDA, C ABI in
``include/modelc_cuda.h``); this package is a thin host binding of it.
"""
from ._lib import McError, lib, last_error  # noqa: F401
from .generate import (KV_FP32, KV_INT8, KV_MIXED, CacheLookup, GenerationConfig,  # noqa: F401
                       KvSnapshot, LlamaDraftModel, MlpDraftModel, NgramDraftModel,
                       PrefixCache, Session, forward_llama_cached, sample_rows,
                       speculative_generate, tp_unique_id)
from .model import (LLAMA2_70B, LLAMA3_8B, PRESETS, TINY, TINYLLAMA,  # noqa: F401
                    LlamaConfig, Linear, QTensor, Weights, quantize_int8_rows,
                    quantize_int8_tensor, synth_weights, synth_weights_torch)

# The paged serving operators work on torch tensors: torch is imported with
# the first of them that is used.
_PAGED = ("PagedStep", "RopeScaling", "kv4_append", "kv4_attention", "kv4_pool", "kv4_read",
          "paged_slots", "prompt_attention", "rope", "rope_frequencies", "rope_table")


def __getattr__(name):
    if name == "paged" or name in _PAGED:
        from importlib import import_module
        paged = import_module(".paged", __name__)
        globals().update({n: getattr(paged, n) for n in _PAGED})
        return globals()[name]
    raise AttributeError(f"module {__name__!r} has no attribute {name!r}")


__version__ = "0.1.0"
