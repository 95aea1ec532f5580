"""gateddeltanet_amd -- MI355X-native GatedDeltaNet-1.3B decode engine
(batch-1, plus multi-stream decode).

The compute path is libgdn_amd.so (hand-written gfx950 HIP kernels behind the
C ABI of include/gdn_amd.h); this package is its Python host mirror.
"""
from .engine import (  # noqa: F401
    ACTIVATION_LAYOUT,
    CONTRACT_BF16W_FP32S,
    BatchState,
    CONTRACT_FP32,
    CONTRACT_REF,
    EXCHANGE_REGIONS,
    EXCHANGE_WORDS,
    GDNError,
    PREFILL_CHUNKED,
    PREFILL_SCAN,
    Model,
    RunState,
    batch_gemm,
    bf16_round,
    default_config,
    gemv,
    prefill_gemm,
    recurrence,
    synth_normal,
    synth_tokens,
    synth_uniform,
)

_DEVICE_OPS = ("delta_prefill", "delta_step", "logits_process", "sample_tokens")


def __getattr__(name: str):
    """The operators on torch tensors, imported (with torch) at first use."""
    if name in _DEVICE_OPS:
        from . import device_ops
        for op in _DEVICE_OPS:
            globals()[op] = getattr(device_ops, op)
        return globals()[name]
    raise AttributeError(f"module {__name__!r} has no attribute {name!r}")
