"""GPU checks of the paged-cache and logits operators at the ends of what they
accept: the longest tables, the largest finite values, scores without a limit."""

from __future__ import annotations

import pytest
import torch

from tests import paged_reference as ref
from tests.test_gpu_paged import _assert_attention, _attend_case, _ops, _randn

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


TOP = torch.finfo(torch.float32).max


@pytest.mark.parametrize("dim", [16, 64, 128, 256])
@pytest.mark.parametrize("group", [1, 4, 5, 8, 9, 16])
@pytest.mark.parametrize("where", ["values", "keys", "queries"])
def test_attention_with_the_largest_finite_values(group, dim, where):
    """Elements up to the largest float32, among them those that round up to infinity in fewer bits, beside operands
    so small that every product and sum stays in range."""
    case = [_randn((40, 2, 16, dim), torch.float32, 1), _randn((40, 2, 16, dim), torch.float32, 2),
            _randn((2, 2 * group, 1, dim), torch.float32, 3)]
    k, v, q = case
    lengths, scale = torch.tensor([1, 300]), 0.25
    table = ref.table_for([1, 300], 16, 40)
    near = torch.tensor([TOP, -TOP, TOP * (1 - 2.0 ** -13), TOP * (1 - 2.0 ** -10), -TOP * (1 - 2.0 ** -12), TOP * 0.999])
    if where == "values":
        v *= 2.0 ** 10
        first = int(table[0, 0])
        v[first, :, 0, :6], v[first, :, 0, -1] = near, -TOP  # all the weight: the output is the value
        p = int(table[1, 3])
        v[p, :, 5, 3:9] = near
        k[p, :, 5] = 0  # about the mean weight, far below 1
    elif where == "keys":
        k *= 2.0 ** 100
        q *= 2.0 ** -100
        for b in range(2):
            k[int(table[b, 0]), :, 0, :6] = near
        q[..., :6] = q[..., :6].sign() * 2.0 ** -126
    else:
        q[..., :6] = near * (1 + torch.arange(2 * group).view(1, -1, 1, 1) % 2 * -2.0 ** -11)
        k[..., :6] = k[..., :6].sign() * 2.0 ** -126
    assert all(t.isfinite().all() for t in (k, v, q))
    out = _ops().paged_gqa_decode_attention_native(q.cuda(), k.cuda(), v.cuda(), table.cuda(), lengths.cuda(), scale)
    _assert_attention(out, q, k, v, table, lengths, scale)


@pytest.mark.parametrize("group", [1, 3, 4, 5, 8, 9, 16])
def test_attention_with_the_largest_queries_on_16_bit_pages(group):
    """Float32 queries up to the largest, where bfloat16 ends earlier."""
    k, v = (_randn((40, 2, 16, 64), torch.bfloat16, seed) for seed in (1, 2))
    q = _randn((2, 2 * group, 1, 64), torch.float32, 3)
    table, lengths = ref.table_for([1, 300], 16, 40), torch.tensor([1, 300])
    q[..., :4] = torch.tensor([TOP, -TOP, TOP * (1 - 2.0 ** -9), -TOP * (1 - 2.0 ** -10)])
    k[..., :4] = k[..., :4].sign() * 2.0 ** -126
    out = _ops().paged_gqa_decode_attention_native(q.cuda(), k.cuda(), v.cuda(), table.cuda(), lengths.cuda(), 0.25)
    _assert_attention(out, q, k, v, table, lengths, 0.25)



@pytest.mark.parametrize("group", [3, 8, 12])
@pytest.mark.parametrize("size", [1e-34, 1e-35, 1e-37, 1e30, 1e36])
def test_attention_with_tiny_and_huge_queries_on_float16_pages(group, size):
    """Float32 queries down to the smallest normal ones, with a scale that makes up for it."""
    case = _attend_case([300, 5], 16, 2, group, 64, "f32", "f16", seed=5, scale=0.125 / size)
    q, k, v, kc, vc, table, lengths, scale = case
    q *= size
    out = _ops().paged_gqa_decode_attention_native(q.cuda(), kc, vc, table.cuda(), lengths.cuda(), scale)
    _assert_attention(out, q, k, v, table, lengths, scale)
    zero = _ops().paged_gqa_decode_attention_native(0 * q.cuda(), kc, vc, table.cuda(), lengths.cuda(), scale)
    _assert_attention(zero, 0 * q, k, v, table, lengths, scale)

@pytest.mark.parametrize("dim,group", [(64, 4), (128, 8), (256, 3), (64, 16), (128, 9)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows", [(1 << 21) + 64 * 255, (1 << 16) + 64, 1 << 16, 1 << 14])
def test_attention_sums_over_millions_of_rows(dtype, dim, group, rows):
    """Values of one sign, equal weights, whole units in one CTA each: what is lost at every step would add up."""
    page, batch = 64, 112  # 448 units
    v = (_randn((1, 4, page, dim), torch.float32, 2).abs() + 0.5).to(dtype)
    k = torch.zeros_like(v)
    q = _randn((batch, 4 * group, 1, dim), dtype, 3)
    table = torch.zeros((1, rows // page), dtype=torch.int32, device="cuda").expand(batch, -1).contiguous()
    lengths = torch.full((batch,), rows, device="cuda")
    out = _ops().paged_gqa_decode_attention_native(q.cuda(), k.cuda(), v.cuda(), table, lengths, 0.1).cpu().double()
    expected = v[0].double().mean(1).repeat_interleave(group, 0).view(1, 4 * group, 1, dim)
    # 2 terms of a run's tiles truncated by less than 2^-23 each, then float32 sums of the runs (of 256 tiles beyond
    # 65536 rows), and the weights' terms; one rounding to 16 bits
    run = 256 if rows > 1 << 16 else rows // page
    tolerance = 2 * run * 2.0 ** -23 + rows // page / run * ref.U32 + 2.0 ** -16 + 1.01 * ref.half_step(dtype)
    error = ((out - expected).abs() / expected).max().item()
    assert error <= tolerance, (error, tolerance)


@pytest.mark.parametrize("query", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("group", [3, 8, 12])
@pytest.mark.parametrize("columns", [600, 1100])
def test_attention_joins_runs_of_any_maximum(query, group, columns):
    """More tiles in one CTA than are summed in one go, whose scores rise, fall, or are hidden for long."""
    page, pages, batch, rows = 64, 40, 160, 600 * 64
    k, v = (_randn((pages, 3, page, 64), TYPES[query], seed) for seed in (1, 2))
    k *= torch.linspace(0.1, 3, pages).view(-1, 1, 1, 1).to(k.dtype)
    q = _randn((batch, 3 * group, 1, 64), TYPES[query], 3)
    order = torch.arange(600) * pages // 600
    table = torch.stack([order, order.flip(0), torch.where(order < 20, -1, order), torch.where(order < 35, order, -1)])
    table = torch.nn.functional.pad(table, (0, columns - 600), value=-1).int().repeat(batch // 4, 1)
    lengths = torch.full((batch,), rows - 17)
    out = _ops().paged_gqa_decode_attention_native(q.cuda(), k.cuda(), v.cuda(), table.cuda(), lengths.cuda(), 0.125)
    pick = [0, 1, 2, 3, 156, 157, 158, 159]
    _assert_attention(out[pick], q[pick], k, v, table[pick], lengths[pick], 0.125)


INF = float("inf")


@pytest.mark.parametrize("query,pages,group", [("f32", "f32", 1), ("f32", "f32", 4), ("f32", "f32", 5), ("f32", "f32", 16),
                                               ("f32", "bf16", 3), ("f32", "f16", 9), ("bf16", "bf16", 2), ("f16", "f16", 16)])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("length", [1, 100])
def test_attention_with_an_infinity_in_a_key_row(query, pages, group, sign, length):
    """A score of -inf has weight 0 (zeros where all scores are); one of +inf gives NaN.  Float32 queries meet 16-bit
    keys as terms, one of which may be 0: NaN either way."""
    k, v = (_randn((8, 1, 16, 64), TYPES[pages], seed) for seed in (1, 2))
    q = _randn((1, group, 1, 64), TYPES[query], 3).abs() + 0.5
    q = q.to(TYPES[query])
    table = torch.arange(7, dtype=torch.int32).view(1, -1)
    k[0, 0, 0, 5] = sign * INF
    out = _ops().paged_gqa_decode_attention_native(q.cuda(), k.cuda(), v.cuda(), table.cuda(),
                                                   torch.tensor([length], device="cuda"), 0.125).cpu()
    if sign > 0:
        assert out.isnan().all()
    elif query == pages and length == 1:
        assert not out.any()
    elif query == pages:
        k[0, 0, 0] = -(q[0, 0, 0].float() * 1e4).to(k.dtype)  # as far below the others as to have no weight
        _assert_attention(out, q, k, v, table, torch.tensor([length]), 0.125)
    else:
        assert out.isnan().all() or out.isfinite().all()


@pytest.mark.parametrize("query,pages,group", [("f32", "f32", 4), ("f32", "f32", 5), ("f32", "f32", 16), ("f32", "f16", 9),
                                               ("bf16", "bf16", 2)])
@pytest.mark.parametrize("size", [INF, -INF, float("nan")])
def test_attention_with_an_infinity_in_a_value_row(query, pages, group, size):
    """Not finite where the row counts, in its own dim only."""
    k, v = (_randn((8, 1, 16, 64), TYPES[pages], seed) for seed in (1, 2))
    q = _randn((1, group, 1, 64), TYPES[query], 3)
    v[3, 0, 7, 9] = size
    table = torch.arange(7, dtype=torch.int32).view(1, -1)
    out = _ops().paged_gqa_decode_attention_native(q.cuda(), k.cuda(), v.cuda(), table.cuda(),
                                                   torch.tensor([100], device="cuda"), 0.125).cpu()
    assert not out[..., 9].isfinite().any() and out[..., :9].isfinite().all() and out[..., 10:].isfinite().all()


@pytest.mark.parametrize("vocab,history", [(33, 40), (8193, 9000), (30001, 40000)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_logits_penalties_are_those_of_float32(dtype, vocab, history):
    """Bit for bit: a division or a product, a product, two differences and a sum, each rounded once in float32.  16-bit
    logits, whose quotient may be off by one step of float32, are rounded once more from there."""
    g = torch.Generator().manual_seed(vocab)
    repetition = torch.tensor([1.1, 1.3, 0.7, 3.0, 1e-20, 1e20, 1.0000001, 1.9999998])
    rows = repetition.shape[0]
    x = (torch.randn((rows, vocab), generator=g) * 3).to(dtype)
    x[3, :9] = torch.tensor([float("inf"), -float("inf"), 3.3e38, -3.3e38, 0.0, -0.0, 1e-30, 1e30, 2.0 ** 120])
    tokens_of_row_3 = torch.arange(9)
    tokens = torch.randint(vocab, (rows, history), generator=g)
    tokens[3, :9] = tokens_of_row_3
    lengths = torch.full((rows,), history - 3)
    prompts = torch.tensor([0, 5, history, 7, history, history, 11, 9])
    bias = torch.randn(vocab, generator=g)
    penalties = torch.stack((repetition, torch.rand(rows, generator=g), torch.rand(rows, generator=g)), 1)
    out = _ops().logits_process_native(x.cuda(), tokens.cuda(), prompts.cuda(), lengths.cuda(), penalties.cuda(), bias.cuda())
    column = torch.arange(history)
    inside = (column < lengths.unsqueeze(1)).float()
    emitted = inside * (column >= prompts.unsqueeze(1))
    zero = torch.zeros((rows, vocab))
    seen, count = zero.scatter_add(1, tokens, inside) > 0, zero.scatter_add(1, tokens, emitted)
    r, presence, frequency = penalties.unsqueeze(2).unbind(1)
    y = x.float()
    y = torch.where(seen, torch.where(y > 0, y / r, y * r), y)
    y = torch.where(count > 0, y - frequency * count - presence, y) + bias
    if dtype == torch.float32:
        assert torch.equal(out.cpu(), y)
        return
    got, size = out.cpu().double(), torch.maximum(x.double().abs() / r.double(), y.double().abs())
    finite = y.isfinite()
    assert torch.equal(got[~finite], y.double()[~finite])
    error = (got - y.double()).abs() - ref.half_step(dtype) * y.double().abs() - 2.0 ** -22 * size
    assert (error[finite] <= 0).all()
