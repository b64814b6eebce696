"""The paged-cache and logits operators under tracing with sizes that may
change, and under forward-mode differentiation.  No call here reaches CUDA."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as forward_ad
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.symbolic_shapes import DimDynamic, ShapeEnv, StatelessSymbolicContext

from flux_b200 import operators as ops

pytestmark = pytest.mark.skipif(not ops.native_paged_cache_is_available(),
                                reason="libfluxb200_torch.so is not built (python -m flux_b200.build)")


class Symbolic:
    """Fake CUDA tensors whose sizes of the given values are symbols."""

    def __enter__(self):
        self.env = ShapeEnv()
        self.mode = FakeTensorMode(shape_env=self.env)
        self.mode.__enter__()
        return self

    def __exit__(self, *exc):
        return self.mode.__exit__(*exc)

    def __call__(self, *shape, dtype=torch.float32, dynamic=(0,)):
        sizes = [DimDynamic.DYNAMIC if d in dynamic else DimDynamic.STATIC for d in range(len(shape))]
        context = StatelessSymbolicContext(dynamic_sizes=sizes)
        with torch._C._DisableTorchDispatch():  # a tensor of its own, which the mode then takes
            real = torch.empty(shape, dtype=dtype, device="meta")
        fake = self.mode.from_tensor(real, symbolic_context=context, static_shapes=False)
        return fake


def is_symbol(size):
    return isinstance(size, torch.SymInt) and size.node.maybe_as_int() is None


def test_attention_keeps_a_symbolic_batch():
    with Symbolic() as empty:
        query, table = empty(7, 6, 1, 64), empty(7, 3, dtype=torch.int32, dynamic=(0, 1))
        k, v = (empty(5, 2, 16, 64, dynamic=(0,)) for _ in range(2))
        lengths = empty(7, dtype=torch.int64)
        out = ops.paged_gqa_decode_attention_native(query, k, v, table, lengths, 0.125)
        assert is_symbol(out.shape[0]) and tuple(out.shape[1:]) == (6, 1, 64) and out.dtype == torch.float32
        for bad, message in ((dict(query=empty(7, 6, 2, 64)), "query must be"),
                             (dict(query=empty(7, 5, 1, 64)), "divisible by KV heads"),
                             (dict(lengths=empty(7, dtype=torch.int32)), "lengths must be"),
                             (dict(page_table=empty(7, 3)), "int32"),
                             (dict(page_table=empty(9, 3, dtype=torch.int32)), "one row per sequence"),
                             (dict(value_pages=empty(5, 2, 16, 32)), "same shape")):
            args = dict(query=query, key_pages=k, value_pages=v, page_table=table, lengths=lengths, scale=0.125)
            with pytest.raises(RuntimeError, match=message):
                ops.paged_gqa_decode_attention_native(**{**args, **bad})


def test_write_keeps_a_symbolic_number_of_tokens():
    with Symbolic() as empty:
        packed, positions = empty(7, 640, dtype=torch.bfloat16), empty(7, dtype=torch.int64)
        k, v = (empty(5, 2, 16, 64, dtype=torch.bfloat16) for _ in range(2))
        cos, sin = empty(50, 64), empty(50, 64)
        out = ops.paged_qkv_rope_cache_native(packed, cos, sin, k, v, empty(2, 3, dtype=torch.int32), positions, positions)
        assert is_symbol(out.shape[0]) and tuple(out.shape[1:]) == (6, 1, 64) and out.dtype == torch.bfloat16
        with pytest.raises(RuntimeError, match="packed_qkv must be"):
            ops.paged_qkv_rope_cache_native(empty(7, 641), cos, sin, k, v, empty(2, 3, dtype=torch.int32), positions, positions)
        with pytest.raises(RuntimeError, match="one token per page_table row"):
            ops.paged_qkv_rope_cache_native(packed, cos, sin, k, v, empty(2, 3, dtype=torch.int32), positions)


def test_logits_keep_a_symbolic_batch():
    with Symbolic() as empty:
        logits, tokens = empty(7, 100, dtype=torch.float16), empty(7, 9, dtype=torch.int64, dynamic=(0, 1))
        vec, penalties = empty(7, dtype=torch.int64), empty(7, 3)
        out = ops.logits_process_native(logits, tokens, vec, vec, penalties, empty(100, dynamic=()),
                                        empty(7, 4, dtype=torch.int32))
        assert is_symbol(out.shape[0]) and out.shape[1] == 100 and out.dtype == torch.float16
        into = empty(7, 100, dtype=torch.float16)
        assert ops.logits_process_native_out(logits, into, tokens, vec, vec, penalties).shape == into.shape
        with pytest.raises(RuntimeError, match="go together"):
            ops.logits_process_native(logits, tokens)
        with pytest.raises(RuntimeError, match="bias must be"):
            ops.logits_process_native(logits, bias=empty(99, dynamic=()))


def test_page_operations_keep_a_symbolic_list():
    with Symbolic() as empty:
        k, v = (empty(3, 5, 2, 16, 64, dynamic=(1,)) for _ in range(2))
        table, lengths = empty(4, 3, dtype=torch.int32), empty(4, dtype=torch.int64)
        counts, ids = empty(5, dtype=torch.int32), empty(7, dtype=torch.int64)
        status = ops.cache_sequences_reserve_native(table, lengths, counts, ids, ids, 16)
        assert is_symbol(status.shape[0]) and status.dtype == torch.int32
        status = ops.cache_sequences_fork_native(k, v, table, lengths, counts, ids, ids)
        assert is_symbol(status.shape[0]) and status.dtype == torch.int32
        ops.cache_sequences_free_native(table, lengths, counts, ids)
        ops.cache_pages_copy_native(k, v, ids, ids)
        assert ops.cache_pages_compact_native(k, v, table, counts).shape == ()
        with pytest.raises(RuntimeError, match="page_counts must be"):
            ops.cache_sequences_reserve_native(table, lengths, ids, ids, ids, 16)


def test_a_traced_step_serves_other_batches():
    """One trace with symbolic sizes: the batch of the trace is not in it."""
    from torch.fx.experimental.proxy_tensor import make_fx

    def step(query, k, v, table, lengths, logits):
        out = ops.paged_gqa_decode_attention_native(query, k, v, table, lengths, 0.125)
        return out + 1, ops.logits_process_native(logits) * 2

    args = (torch.zeros(7, 6, 1, 64), torch.zeros(5, 2, 16, 64), torch.zeros(5, 2, 16, 64),
            torch.zeros((7, 3), dtype=torch.int32), torch.zeros(7, dtype=torch.int64), torch.zeros(7, 100))
    graph = make_fx(step, tracing_mode="symbolic")(*args)
    values = [n.meta["val"] for n in graph.graph.nodes if n.op == "call_function" and "val" in n.meta]
    assert values and all(is_symbol(v.shape[0]) for v in values if isinstance(v, torch.Tensor))


def test_forward_mode_derivatives_are_refused():
    x, t = torch.zeros(2, 100), torch.ones(2, 100)
    k, v = torch.zeros(5, 2, 16, 64), torch.zeros(5, 2, 16, 64)
    table, lengths = torch.zeros((2, 3), dtype=torch.int32), torch.zeros(2, dtype=torch.int64)
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="inference-only"):
            ops.logits_process_native(forward_ad.make_dual(x, t))
        q = torch.zeros(2, 6, 1, 64)
        with pytest.raises(RuntimeError, match="inference-only"):
            ops.paged_gqa_decode_attention_native(forward_ad.make_dual(q, q + 1), k, v, table, lengths, 0.125)
        with pytest.raises(RuntimeError, match="inference-only"):
            ops.paged_gqa_decode_attention_native(q, k, forward_ad.make_dual(v, v + 1), table, lengths, 0.125)
        with pytest.raises(RuntimeError, match="CUDA tensors are required"):
            ops.logits_process_native(x)
    with pytest.raises(RuntimeError, match="CUDA tensors are required"):
        ops.logits_process_native(x)
