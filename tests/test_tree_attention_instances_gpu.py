"""Attention over the paged cache in every kernel it has: few rows to a unit (up to 16) and many, fewer units than CTAs
and more, parts joined from registers, in one step and in two, and the branches of the softmax in each."""
import random

import pytest
import torch

from flashlite_b200 import flash_attn_wmma as fa

from test_tree_attention_gpu import Case

pytestmark = pytest.mark.gpu

# tokens of a request, heads, key heads: 4 and 40 rows to a unit
ROWS = [(2, 2, 1), (10, 4, 1)]


@pytest.mark.parametrize("words", [0, 1])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 128])
def test_more_units_of_many_rows_than_ctas(cuda, dim, dtype, words):
    """Each CTA has its share of several units of 18 to 72 rows: whole ones, later and first parts, some of one tile."""
    rng = random.Random(dim + words)
    lengths = [(rng.choice([0, 5, 60, 128, 300, 700]), rng.randint(9, 31)) for _ in range(40)]
    c = Case(cuda, lengths, 16, 8, dim, 16, dtype, words=words, seed=dim, poison=True)
    first = c.check()
    for _ in range(20):
        again = c.run()
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
    assert fa.device_error() == 0


@pytest.mark.parametrize("dim", [64, 128])
def test_row_tiles_of_more_than_128_rows(cuda, dim):
    """Prompts of several row tiles, more of them than CTAs."""
    rng = random.Random(dim)
    Case(cuda, [(rng.choice([0, 17, 200]), rng.randint(100, 200)) for _ in range(10)], 16, 8, dim, 32, seed=dim).check()


@pytest.mark.parametrize("dim", [64, 128])
def test_many_parts_of_many_rows(cuda, dim):
    """Two units of 128 and 88 rows whose caches are cut into dozens of parts: joined in groups, then among the groups."""
    c = Case(cuda, [(6000, 54)], 4, 1, dim, 32, seed=dim)
    first = c.check()
    for _ in range(10):
        again = c.run()
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


@pytest.mark.parametrize("words", [0, 1])
def test_many_parts_among_more_units_than_ctas(cuda, words):
    """One long cache among short ones, 160 units of 40 rows in all: the even division cuts its units into dozens of
    parts."""
    rng = random.Random(words)
    lengths = [(rng.randint(0, 100), 5) for _ in range(39)]
    lengths.insert(11, (16000, 5))
    c = Case(cuda, lengths, 32, 4, 64, 64, words=words, seed=words)
    first = c.check()
    for _ in range(10):
        again = c.run()
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


@pytest.mark.parametrize("parts", [300, 700, 1500])
@pytest.mark.parametrize("tokens,heads", [(9, 4), (30, 4)])
def test_parts_joined_from_registers(cuda, tokens, heads, parts):
    """36 and 120 rows, units of a few parts each."""
    c = Case(cuda, [(parts, tokens)] * 12, heads * 4, 4, 128, 16, seed=parts)
    first = c.check()
    for _ in range(10):
        again = c.run()
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


@pytest.mark.parametrize("tokens,heads,kv_heads", ROWS)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("words", [0, 1])
@pytest.mark.parametrize("sm_scale", [0.3, -0.2, 1e-3])
def test_scales(cuda, sm_scale, words, dim, tokens, heads, kv_heads):
    Case(cuda, [(200, tokens), (3, tokens)], heads, kv_heads, dim, 32, words=words).check(sm_scale)


@pytest.mark.parametrize("tokens,heads,kv_heads", ROWS)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype,low,score", [(torch.float16, 60000.0, 1.0), (torch.bfloat16, 2.0 ** 64, 2.0 ** -30),
                                             (torch.bfloat16, 2.0 ** 64, 1.296875 / 2)])
@pytest.mark.parametrize("n", [300, 5000])
def test_equal_lowest_scores_average(cuda, n, dtype, low, score, dim, tokens, heads, kv_heads):
    """Equal scores as low as a type (and, last, fp32 in base 2) holds them are scores, not masks: a row gives the mean of the values it sees,
    whether or not the unit is cut into parts. Equal probabilities: only sums in fp32 and the result's rounding are off."""
    c = Case(cuda, [(n, tokens)], heads, kv_heads, dim, 16, dtype)
    c.q[:] = 0
    c.q[..., 0] = -low
    c.k[:] = 0
    c.k[..., 0] = low * score
    out, lse = c.run(sm_scale=1.0)
    s = -float(c.q[0, 0, 0].double().abs() * c.k[0, 0, 0, 0].double())
    rows = torch.tensor([c.table[0][p // 16] * 16 + p % 16 for p in range(n + tokens)], device=cuda)
    v = c.v.double().reshape(-1, kv_heads, dim)[rows]
    for t in range(tokens):
        want = v[:n + t + 1].mean(0)[0]
        u = 2.0 ** -11 if dtype == torch.float16 else 2.0 ** -8
        assert float((out[t].double() - want).abs().max()) <= u * float(want.abs().max()) + 2.0 ** -16 * 4
    assert float((lse.double() / s - 1).abs().max()) <= 2.0 ** -20
    assert fa.device_error() == 0


@pytest.mark.parametrize("tokens,heads,kv_heads", ROWS)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("words", [0, 1])
@pytest.mark.parametrize("sm_scale", [4.0, -4.0])
def test_scores_far_past_a_million(cuda, sm_scale, words, dim, tokens, heads, kv_heads):
    """Scores of up to 2^22, 2^12 and more apart: the largest takes all, and its value comes out as it is."""
    ctx, rng = 500, random.Random(dim)
    c = Case(cuda, [(ctx, tokens)], heads, kv_heads, dim, 16, words=words, seed=3)
    n = ctx + tokens
    order = list(range(n))
    rng.shuffle(order)
    c.q[:] = 0
    c.q[..., 0] = torch.tensor([1024.0 if rng.random() < 0.5 else -1024.0 for _ in range(tokens * heads)],
                               device=cuda).view(tokens, heads)
    c.k[:] = 0
    for p in range(n):
        c.k[c.table[0][p // 16], p % 16, :, 0] = float(2 * order[p])
    out, lse = c.run(sm_scale=sm_scale)
    for t in range(tokens):
        seen = list(range(ctx)) + [ctx + j for j in range(tokens)
                                   if (j <= t if not words else j < 32 and (int(c.mask[t, 0]) >> j) & 1)]
        for h in range(heads):
            a = float(c.q[t, h, 0]) * sm_scale
            best = max(seen, key=lambda p: a * order[p])
            assert torch.equal(out[t, h], c.v[c.table[0][best // 16], best % 16, h * kv_heads // heads])
            want = a * 2 * order[best]
            assert abs(float(lse[t, h]) - want) <= 2.0 ** -20 * abs(want) + 1e-6
    assert fa.device_error() == 0


@pytest.mark.parametrize("lengths,heads,kv_heads,dim,changes", [
    # few rows: 157 parts of a unit, joined in two steps; then fewer, and none
    ([(20011, 3)], 4, 1, 64, [[20011], [20011], [3000], [200], [20000]]),
    # many rows, few units: dozens of parts; then parts joined from registers
    ([(6000, 20)], 4, 1, 128, [[6000], [6000], [300], [6000], [90]]),
    # many rows, more units than CTAs
    ([(300 + 40 * b, 12) for b in range(40)], 32, 8, 64, [[300 + 40 * b for b in range(40)], [40 * b for b in range(40)],
                                                         [1500] + [7] * 39, [300 + 40 * b for b in range(40)]]),
])
def test_cut_units_in_a_captured_call(cuda, lengths, heads, kv_heads, dim, changes):
    """A captured call runs again with the same call number: its arrival counts have to start from none each time."""
    c = Case(cuda, lengths, heads, kv_heads, dim, 16, seed=dim)
    i = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    # rows long enough for every change
    need = max(max(ch) for ch in changes) + max(t for _, t in lengths)
    cols = -(-need // 16) + 1
    table = i([(r + r * (cols // len(r) + 1))[:cols] for r in [[x for x in row if x < 10 ** 6] for row in c.table]])
    ctx, cu = i(c.context), i(c.cu)
    call = lambda: fa.tree_attention(c.q, c.k, c.v, table, ctx, cu, return_lse=True)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = call()
    for lens in changes:
        ctx.copy_(i(lens))
        want, wlse = call()
        for _ in range(3):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want) and torch.equal(lse, wlse), lens
    assert fa.device_error() == 0
