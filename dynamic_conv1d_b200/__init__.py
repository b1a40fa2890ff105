"""B200-native dynamic short convolutions (drop-in for OliverSieberling/dynamic-conv1d).

    from dynamic_conv1d_b200 import headwise_dynamic_convolution, lowrank_dynamic_convolution

Both ops are ``torch.autograd.Function``s over libdynconv.so, a C-ABI library of
hand-written sm_100a CUDA kernels (see ``include/dynconv.h``).  So are the operators around
them in a language model:

    decay_linear_attention[_fused]        linear attention with a decay for each head
    linear_cross_entropy                  the loss over a large vocabulary, without logits
    *_step, convolution_cache             one token at a time, on caches updated in place

Calls never synchronise.  The tensor-core kernels bound every device-side wait
(1.5 s); a wait that gives up makes its kernel return early and sets a device
error word, which ``check_device(t)`` reads (raising ``DynconvError`` with status
DYNCONV_ERR_TIMEOUT).  Call it once per training step (or set DYNCONV_SYNC_CHECK=1
/ ``set_sync_checks(True)`` to check after every call while debugging).
"""
from ._lib import DynconvError, check_device, set_sync_checks
from .headwise import headwise_dynamic_convolution
from .linear_attention import decay_linear_attention, decay_linear_attention_fused, decay_linear_attention_step
from .lowrank import lowrank_dynamic_convolution, lowrank_dynamic_convolution_grouped
from .modules import (
    ConvolvedLinearAttention,
    LayerCache,
    LowRankDynamicShortConvolution,
    QKVLowRankDynamicShortConvolution,
)
from .parallel import data_parallel, shard_rows
from .sequence_parallel import headwise_dynamic_convolution_sp, lowrank_dynamic_convolution_sp
from .step import (
    convolution_cache,
    headwise_dynamic_convolution_step,
    lowrank_dynamic_convolution_grouped_step,
    lowrank_dynamic_convolution_step,
)
from .vocab_loss import linear_cross_entropy

__all__ = [
    "headwise_dynamic_convolution",
    "lowrank_dynamic_convolution",
    "lowrank_dynamic_convolution_grouped",
    "headwise_dynamic_convolution_step",
    "lowrank_dynamic_convolution_step",
    "lowrank_dynamic_convolution_grouped_step",
    "convolution_cache",
    "decay_linear_attention",
    "decay_linear_attention_fused",
    "decay_linear_attention_step",
    "linear_cross_entropy",
    "LowRankDynamicShortConvolution",
    "QKVLowRankDynamicShortConvolution",
    "ConvolvedLinearAttention",
    "LayerCache",
    "data_parallel",
    "lowrank_dynamic_convolution_sp",
    "headwise_dynamic_convolution_sp",
    "shard_rows",
    "check_device",
    "set_sync_checks",
    "DynconvError",
]
