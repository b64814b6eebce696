"""GPU checks of the paged-cache and logits operators at the ends of what they
accept: the longest tables, the largest finite values, scores without a limit."""

from __future__ import annotations

import pytest
import torch

from tests import paged_reference as ref
from tests.test_gpu_paged import _assert_attention, _ops, _randn

pytestmark = pytest.mark.gpu

TYPES = ref.TYPES


@pytest.mark.parametrize("page", [32, 31])
@pytest.mark.parametrize("query,pages,group", [("f32", "f32", 1), ("f32", "f32", 4), ("f32", "f32", 5), ("f32", "f32", 16),
                                               ("f32", "bf16", 3), ("f32", "f16", 9), ("bf16", "bf16", 2), ("f16", "f16", 16)])
def test_attention_over_the_longest_table(page, query, pages, group):
    """2^31 - 1 rows, or what whole pages give of them: all but a few entries are holes, the last one is none."""
    dim, columns = 16, (2 ** 31 - 1) // page
    k, v = (_randn((5, 1, page, dim), TYPES[pages], seed) for seed in (1, 2))
    q = _randn((1, group, 1, dim), TYPES[query], 3)
    used = {0: 3, columns // 2: 0, columns - 2: 4, columns - 1: 1}
    table = torch.full((1, columns), -1, dtype=torch.int32, device="cuda")
    for entry, p in used.items():
        table[0, entry] = p
    short = torch.tensor([list(used.values())], dtype=torch.int32)
    lengths = torch.tensor([2 ** 40], device="cuda")
    out = torch.full((1, group, 1, dim), float("nan"), dtype=TYPES[query], device="cuda")
    ops = _ops()
    kc, vc = k.cuda(), v.cuda()
    workspace = torch.empty(ops.paged_gqa_decode_attention_workspace_floats(q, kc), device="cuda")
    ops.paged_gqa_decode_attention_native_out(q.cuda(), kc, vc, table, lengths, 0.25, out, workspace)
    _assert_attention(out, q, k, v, short, torch.tensor([4 * page]), 0.25)
    lengths.fill_(columns * page - 1)  # without the last row
    out = ops.paged_gqa_decode_attention_native(q.cuda(), kc, vc, table, lengths, 0.25)
    _assert_attention(out, q, k, v, short, torch.tensor([4 * page - 1]), 0.25)
