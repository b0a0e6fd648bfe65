"""Wayfinder causal learned-address retrieval + sparse attention on B200 (sm_100a).

Public API (names and arguments of the reference's ``routing_attention``):
  causal_topk, fused_sparse_attention, sparse_meat_attention, SparseMeatConfig,
  LearnedAddressSparseAttention, LearnedAddressModule, RetrievalConfig,
  TransformerLM (the decoder harness); HostFusedSparseAttention runs the fused
  op on pinned host tensors with upload, compute and download overlapped.

The decoder's other operators, each with its backward: fused_linear (bias,
activation and residual in the product's epilogue), layer_norm and token_logprobs
(log probability, entropy and top alternatives of given tokens); and its two ends,
token_embedding and linear_token_logprobs (log probabilities without the logits).

The compute runs in ``libwayfinder_sm100.so`` (C ABI: ``include/wayfinder.h``);
there is no CPU path.  Kernel faults that do not stop a kernel (an out-of-range
index, a bounded wait that timed out) raise ``RuntimeError`` at the next call on
the device, or at ``check_status()``, which waits for the device's queued work.
"""

from ._lib import check_status, load_library
from .attention import (
    KeyVectorSparseAttention,
    LearnedAddressModule,
    LearnedAddressSparseAttention,
    RetrievalConfig,
    RoutingSparseAttention,
    retrieval_config_from_dict,
)
from .router import MultiScaleRouter, PerLayerRouter, RouterMLP
from .causal_topk import causal_topk, causal_topk_available, promote_compute_dtype
from .decoder import DenseSDPAAttention, TransformerBlock, TransformerLM
from .graphs import CapturedForward
from .layer_norm import layer_norm
from .embedding import token_embedding
from .linear import fused_linear
from .linear_logprobs import LinearLogprobs, linear_token_logprobs
from .token_logprobs import TokenLogprobs, token_logprobs
from .host_pipeline import HostFusedSparseAttention, host_fused_sparse_attention
from .fused_sparse import (
    SparseMeatConfig,
    fused_sparse_attention,
    fused_sparse_attention_available,
    sparse_meat_attention,
)

__all__ = [
    "load_library",
    "check_status",
    "causal_topk",
    "causal_topk_available",
    "promote_compute_dtype",
    "fused_sparse_attention",
    "fused_sparse_attention_available",
    "sparse_meat_attention",
    "HostFusedSparseAttention",
    "CapturedForward",
    "host_fused_sparse_attention",
    "SparseMeatConfig",
    "fused_linear",
    "layer_norm",
    "token_logprobs",
    "TokenLogprobs",
    "linear_token_logprobs",
    "LinearLogprobs",
    "token_embedding",
    "LearnedAddressModule",
    "LearnedAddressSparseAttention",
    "KeyVectorSparseAttention",
    "RoutingSparseAttention",
    "RouterMLP",
    "PerLayerRouter",
    "MultiScaleRouter",
    "RetrievalConfig",
    "retrieval_config_from_dict",
    "DenseSDPAAttention",
    "TransformerBlock",
    "TransformerLM",
]
