"""B200PagedBackend over a 4-bit cache: its plans, checks and routes (prefill,
decode, both at once, a captured decode step). Runs on the engine's contract
where the engine is installed, else on a stand-in with the same names."""

import dataclasses
import enum
import importlib
import sys
import types

import pytest
import torch

import my_vllm_b200
from conftest import ENGINE_INSTALLED
from int4_cases import Case, assert_within, decode_tolerance, prefill_tolerance
from my_vllm_b200 import ops

NAMES = ("nanovllm", "nanovllm.layers", "nanovllm.layers.attention_backend", "nanovllm.utils",
         "nanovllm.utils.context", "my_vllm_b200.contract", "my_vllm_b200.backend")


def _stand_in():
    class BatchType(enum.Enum):
        PURE_PREFILL, PURE_DECODE, MIXED = range(3)

    class AttentionRoute(enum.Enum):
        WARMUP, PREFILL, DECODE, MIXED_SPLIT = "warmup", "prefill", "decode", "mixed_split"

    common = dataclasses.make_dataclass("CommonAttentionMetadata", [
        "num_prefill_seqs", "num_decode_seqs", "num_prefill_tokens", "num_decode_tokens",
        "query_start_loc", "seq_lens", "slot_mapping", "block_tables", "max_q_len", "max_kv_len",
        "block_counts", "num_kv_blocks", "num_prefill_kv_blocks", "trusted"])
    common.num_seqs = property(lambda c: c.num_prefill_seqs + c.num_decode_seqs)
    common.num_query_tokens = property(lambda c: c.num_prefill_tokens + c.num_decode_tokens)

    class AttentionBackend:
        def __init__(self, num_q_heads, num_kv_heads, head_dim, block_size, dtype):
            self.num_q_heads, self.num_kv_heads, self.head_dim = num_q_heads, num_kv_heads, head_dim
            self.block_size, self.dtype, self.softmax_scale = block_size, dtype, head_dim ** -0.5

    def classify(c):
        if not c.num_decode_seqs:
            return BatchType.PURE_PREFILL
        return BatchType.MIXED if c.num_prefill_seqs else BatchType.PURE_DECODE

    modules = {name: types.ModuleType(name) for name in NAMES[:5]}
    modules["nanovllm.layers.attention_backend"].__dict__.update(
        AttentionBackend=AttentionBackend, AttentionBackendRegistry=type("Registry", (), {}),
        AttentionPlan=dataclasses.make_dataclass("AttentionPlan", ["batch_type", "route", "common",
                                                                   "metadata"]),
        AttentionRoute=AttentionRoute, _classify_batch=classify, _torch_sdpa_varlen=None,
        _validate_common_metadata=lambda common, *, require_cuda: None)
    modules["nanovllm.utils.context"].__dict__.update(BatchType=BatchType,
                                                      CommonAttentionMetadata=common)
    return modules


@pytest.fixture(scope="module")
def backend():
    if ENGINE_INSTALLED:
        yield importlib.import_module("my_vllm_b200.backend")
        return
    held = {name: sys.modules.pop(name, None) for name in NAMES}
    sys.modules.update(_stand_in())
    try:
        yield importlib.import_module("my_vllm_b200.backend")
    finally:
        for name, module in held.items():
            sys.modules.pop(name, None)
            if module is not None:
                sys.modules[name] = module
            elif name.startswith("my_vllm_b200."):
                my_vllm_b200.__dict__.pop(name.split(".")[1], None)


def _make(backend, hq=8, hkv=2, bs=16, dtype=torch.bfloat16, kv=ops.INT4_DTYPE):
    return backend.B200PagedBackend(hq, hkv, 128, bs, dtype, kv_cache_dtype=kv)


def _common(backend, c, dev):
    """The batch of a Case whose first sequences have several new tokens."""
    n = sum(q > 1 for q in c.q_lens)
    counts = tuple((k + c.bs - 1) // c.bs for k in c.kv_lens)
    return backend.CommonAttentionMetadata(
        num_prefill_seqs=n, num_decode_seqs=len(c.q_lens) - n, num_prefill_tokens=sum(c.q_lens[:n]),
        num_decode_tokens=len(c.q_lens) - n, query_start_loc=c.starts.to(dev),
        seq_lens=c.lens.to(dev), slot_mapping=torch.zeros(sum(c.q_lens), dtype=torch.int32,
                                                          device=dev),
        block_tables=c.tables.to(dev), max_q_len=max(c.q_lens), max_kv_len=max(c.kv_lens),
        block_counts=counts, num_kv_blocks=sum(counts), num_prefill_kv_blocks=sum(counts[:n]),
        trusted=True)


def test_construction_and_plans(backend):
    b = _make(backend)
    assert b.kv_cache_dtype == torch.uint8
    with pytest.raises(TypeError, match="4-bit"):
        _make(backend, kv=torch.int8)
    c = Case([1] * 3, [40, 700, 5], 8, 2, 16, torch.bfloat16)
    common = _common(backend, c, "cpu")
    want = ops.plan_decode(3, 8, 2, 128, 16, 700, total_kv_tokens=16 * (3 + 44 + 1), kv_int4=True)
    if not ENGINE_INSTALLED:  # the engine's own validator wants the metadata on the GPU
        assert b.build_metadata(common).decode_plan == want
    assert ops.prefill_workspace_bytes(kv_int4=True) > 0


@pytest.mark.gpu
@pytest.mark.parametrize("q,kv", [([40, 9], [40, 200]), ([1, 1, 1], [300, 17, 64]),
                                  ([30, 2, 1, 1], [90, 2, 41, 500])])
def test_routes(backend, cuda_device, q, kv):
    dev = cuda_device
    c = Case(q, kv, 8, 2, 16, torch.bfloat16, seed=len(q))
    b = _make(backend)
    common = _common(backend, c, dev)
    plan = b.build_plan(common)
    empty = torch.empty(0, device=dev)
    args = (c.q.to(dev), empty, empty, c.k.to(dev), c.v.to(dev), plan)
    out = b.forward(*args)
    b.check_status()
    ref, bounds = c.reference()
    n = common.num_prefill_tokens
    tol = prefill_tolerance(ref, bounds, c.dtype)
    tol[n:] = decode_tolerance(ref, bounds, c.dtype)[n:]
    assert_within(out, ref, tol)
    with pytest.raises(ValueError, match="cache"):
        b.forward(args[0], empty, empty, args[3].view(torch.int8), args[4].view(torch.int8), plan)
    with pytest.raises(ValueError, match="72"):
        b.forward(args[0], empty, empty, args[3][..., :64], args[4][..., :64], plan)


@pytest.mark.gpu
def test_captured_decode_step(backend, cuda_device):
    dev = cuda_device
    b = _make(backend)
    cases = [Case([1] * 4, kv, 8, 2, 16, torch.bfloat16, seed=sum(kv))
             for kv in ([30, 400, 3, 64], [1, 17, 640, 200])]
    pages = max(c.k.size(0) for c in cases)
    k, v = (torch.zeros(ops.int4_cache_shape(pages, 16, 2), dtype=torch.uint8, device=dev)
            for _ in range(2))
    q = torch.zeros(4, 8, 128, dtype=torch.bfloat16, device=dev)
    state = b.create_full_decode_graph_state(4, 4 * 40, dev)
    empty, graph = torch.empty(0, device=dev), None
    for c in cases:
        k[: c.k.size(0)].copy_(c.k)
        v[: c.v.size(0)].copy_(c.v)
        q.copy_(c.q)
        plan = b.build_plan(_common(backend, c, dev))
        b.plan_full_decode_graph(state, plan)
        if graph is None:
            b.activate_full_decode_graph(state)
            b.forward(q, empty, empty, k, v, plan)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = b.forward(q, empty, empty, k, v, plan)
            b.deactivate_full_decode_graph()
        out.fill_(9.0)
        graph.replay()
        b.check_status()
        ref, bounds = c.reference()
        assert_within(out, ref, decode_tolerance(ref, bounds, c.dtype))
