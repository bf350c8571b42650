"""A stand-in for the engine's attention-backend contract, where the engine is not
installed: the names that ``my_vllm_b200.contract`` takes from it, as far as
``B200PagedBackend`` uses them, so that the backend and its kernels can be run,
tested and timed there. It drives no engine: nothing of its scheduler, its layers
or its registry's policies is here.

``add()`` puts it in the place of ``my_vllm_b200.contract``; ``nanovllm`` itself
stays absent, so what needs the engine still finds that out.
"""

from __future__ import annotations

import enum
import importlib.util
import sys
from dataclasses import dataclass
from typing import Any

import torch

ENGINE_CONTRACT = False
CONTRACT = "my_vllm_b200.contract"


class BatchType(enum.Enum):
    PURE_PREFILL = "pure_prefill"
    PURE_DECODE = "pure_decode"
    MIXED = "mixed"


class AttentionRoute(enum.Enum):
    WARMUP = "warmup"
    PREFILL = "prefill"
    DECODE = "decode"
    MIXED_SPLIT = "mixed_split"


@dataclass(frozen=True)
class CommonAttentionMetadata:
    """A step's batch: prefill sequences first, then decode ones of one token."""

    num_prefill_seqs: int
    num_decode_seqs: int
    num_prefill_tokens: int
    num_decode_tokens: int
    query_start_loc: torch.Tensor
    seq_lens: torch.Tensor
    slot_mapping: torch.Tensor
    block_tables: torch.Tensor | None
    max_q_len: int
    max_kv_len: int
    block_counts: tuple[int, ...] | None = None
    num_kv_blocks: int = 0
    num_prefill_kv_blocks: int = 0
    trusted: bool = False

    @property
    def num_seqs(self) -> int:
        return self.num_prefill_seqs + self.num_decode_seqs

    @property
    def num_query_tokens(self) -> int:
        return self.num_prefill_tokens + self.num_decode_tokens


@dataclass(frozen=True)
class AttentionPlan:
    batch_type: BatchType
    route: AttentionRoute
    common: CommonAttentionMetadata
    metadata: Any


class AttentionBackend:
    def __init__(self, num_q_heads, num_kv_heads, head_dim, block_size, dtype):
        if num_kv_heads <= 0 or num_q_heads % num_kv_heads:
            raise ValueError("num_q_heads must be divisible by num_kv_heads")
        self.num_q_heads, self.num_kv_heads, self.head_dim = num_q_heads, num_kv_heads, head_dim
        self.block_size, self.dtype = block_size, dtype
        self.softmax_scale = head_dim ** -0.5


class AttentionBackendRegistry:
    _BACKENDS: dict[str, type] = {}

    @classmethod
    def registered_names(cls) -> tuple[str, ...]:
        return tuple(cls._BACKENDS)

    @classmethod
    def register(cls, name: str, backend: type) -> None:
        if name in cls._BACKENDS:
            raise ValueError(f"backend {name!r} is already registered")
        cls._BACKENDS[name] = backend


def _classify_batch(common: CommonAttentionMetadata) -> BatchType:
    if common.num_decode_seqs == 0:
        return BatchType.PURE_PREFILL
    return BatchType.MIXED if common.num_prefill_seqs else BatchType.PURE_DECODE


def _validate_common_metadata(common: CommonAttentionMetadata, *, require_cuda: bool) -> None:
    """Types and shapes alone: no value is read from the device."""
    if common.num_seqs <= 0 or common.num_decode_tokens != common.num_decode_seqs:
        raise ValueError("a batch needs sequences, its decode ones of one token each")
    for name, n in (("query_start_loc", common.num_seqs + 1), ("seq_lens", common.num_seqs),
                    ("slot_mapping", common.num_query_tokens)):
        t = getattr(common, name)
        if t.dtype != torch.int32 or t.ndim != 1 or t.numel() != n:
            raise ValueError(f"{name} must be a 1-D int32 tensor of {n} values")
        if require_cuda and not t.is_cuda:
            raise ValueError(f"{name} must be a CUDA tensor")


def _torch_sdpa_varlen(q, k, v, common: CommonAttentionMetadata) -> torch.Tensor:
    """Causal attention of each sequence's own rows, in fp32 products and sums."""
    out = torch.empty_like(q)
    group = q.size(1) // k.size(1)
    starts = common.query_start_loc.tolist()
    for a, b in zip(starts, starts[1:]):
        x = q[a:b].float().transpose(0, 1)
        keys, values = (t[a:b].float().transpose(0, 1).repeat_interleave(group, 0) for t in (k, v))
        scores = x @ keys.transpose(1, 2) * q.size(2) ** -0.5
        later = torch.ones(b - a, b - a, dtype=torch.bool, device=q.device).triu(1)
        p = torch.softmax(scores.masked_fill(later, float("-inf")), -1)
        out[a:b] = (p @ values).transpose(0, 1).to(q.dtype)
    return out


def add() -> bool:
    """Stand in for the contract where the engine cannot be imported; whether it does."""
    if importlib.util.find_spec("nanovllm") is not None:
        return False
    import my_vllm_b200

    sys.modules[CONTRACT] = my_vllm_b200.contract = sys.modules[__name__]
    return True
