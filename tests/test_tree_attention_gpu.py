"""Attention over the paged cache against the formula in 64 bits.

Tolerance, with u the type's unit roundoff, W = sum_j p_j |v_j| of the row and R its largest sum_d |q_d k_jd| scale:
the kernel rounds each probability once to the storage type (u W), sums products in fp32 (2^-16 W covers a few
thousand of them at 2^-24 each, and the base-2 exponential's 2^-22), computes the scores in fp32 (2^-20 R each,
which moves a probability by that factor and its normaliser too: 2^-19 R W) and rounds the result once (u |o|).
fp16 probabilities below the normal range move by at most 2^-25 of the largest: covered by 2^-16 W + 2^-24. The
log-sum-exp is held in fp32: 2^-20 (1 + R + |lse|)."""
import random

import pytest
import torch

from flashlite_b200 import flash_attn_wmma as fa
from oracle import serving_oracle as orc

pytestmark = pytest.mark.gpu


class Case:
    """Random q and caches for requests of given (cached, new) lengths, blocks in random order."""

    def __init__(self, device, lengths, heads, kv_heads, dim, page, dtype=torch.float16, layout="bnhd", words=0, seed=0,
                 spread=1.0, poison=False, tail=0):
        rng = random.Random(seed)
        g = torch.Generator(device=device).manual_seed(seed)
        self.context = [c for c, _ in lengths]
        self.cu = [0]
        for _, t in lengths:
            self.cu.append(self.cu[-1] + t)
        tokens = self.cu[-1] + tail
        counts = [-(-(c + t) // page) for c, t in lengths]
        blocks = sum(counts) + 3
        order = list(range(blocks))
        rng.shuffle(order)
        cols = max(counts + [1]) + 1
        self.table, at = [], 0
        for n in counts:
            self.table.append(order[at:at + n] + [10 ** 6] * (cols - n))  # unused entries name no block
            at += n
        shape = (blocks, page, kv_heads, dim)
        kc, vc = (torch.randn(shape, generator=g, device=device) * spread for _ in range(2))
        if poison:  # everything outside the requests' tokens
            used = torch.zeros(blocks, page, dtype=torch.bool)
            for b, (c, t) in enumerate(lengths):
                for p in range(c + t):
                    used[self.table[b][p // page], p % page] = True
            kc[~used.to(device)] = float("nan")
            vc[~used.to(device)] = float("inf")
        self.layout = layout
        self.k, self.v = (x.to(dtype) if layout == "bnhd" else x.to(dtype).transpose(1, 2).contiguous() for x in (kc, vc))
        self.q = (torch.randn(tokens, heads, dim, generator=g, device=device) * spread).to(dtype)
        self.mask = None
        if words:
            rows = [[rng.getrandbits(32) for _ in range(words)] for _ in range(tokens)]
            self.mask = torch.tensor([[w - (1 << 32) if w >> 31 else w for w in r] for r in rows], dtype=torch.int32,
                                     device=device)
        self.device = device

    def run(self, **more):
        i = lambda x: torch.tensor(x, dtype=torch.int32, device=self.device)  # noqa: E731
        return fa.tree_attention(self.q, self.k, self.v, i(self.table), i(self.context), i(self.cu), tree_mask=self.mask,
                                 layout=self.layout, return_lse=True, **more)

    def check(self, sm_scale=0.0):
        out, lse = self.run(sm_scale=sm_scale)
        # masked places may hold anything: the oracle sees what the rows see
        want, wlse, weight, reach = orc.tree_attention(self.q, self.k, self.v, self.table, self.context, self.cu, self.mask,
                                                       sm_scale, self.layout)
        compare(out, lse, want, wlse, weight, reach)
        assert fa.device_error() == 0
        return out, lse


def compare(out, lse, want, wlse, weight, reach):
    u = orc.UNIT[out.dtype]
    out, lse = out.double().cpu(), lse.double().cpu()
    assert torch.equal(out.isnan(), want.isnan())
    assert torch.equal(lse == -float("inf"), wlse == -float("inf"))
    bound = u * want.abs() + (1.1 * u + 2.0 ** -16 + 2.0 ** -19 * reach[..., None]) * weight + 2.0 ** -24
    off = torch.nan_to_num((out - want).abs() - bound, nan=-1.0)
    assert bool((off <= 0).all()), float(off.max())
    live = wlse > -float("inf")
    off = (lse - wlse).abs()[live] - 2.0 ** -20 * (1 + reach + wlse.abs())[live]
    assert off.numel() == 0 or bool((off <= 0).all()), float(off.max())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lengths", [[(0, 1)], [(1, 1)], [(63, 1)], [(64, 1)], [(127, 1)], [(128, 1)], [(777, 1)],
                                     [(5, 1), (0, 1), (300, 1), (64, 1)], [(1000, 1)] * 9])
def test_one_token(cuda, dtype, dim, lengths):
    Case(cuda, lengths, 8, 2, dim, 16, dtype, poison=True).check()


@pytest.mark.parametrize("layout", ["bnhd", "bhnd"])
@pytest.mark.parametrize("page", [8, 16, 32, 64, 128, 256])
@pytest.mark.parametrize("dim", [64, 128])
def test_pages(cuda, dim, page, layout):
    Case(cuda, [(page - 1, 3), (page, 1), (3 * page + 5, 7), (2, 0), (page + 1, 2 * page)], 6, 2, dim, page, layout=layout,
         poison=True, seed=page).check()


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (8, 8), (3, 1), (5, 1), (14, 2), (32, 4), (40, 8), (100, 1), (128, 1)])
@pytest.mark.parametrize("dim", [64, 128])
def test_head_groups(cuda, heads, kv_heads, dim):
    Case(cuda, [(70, 1), (33, 5), (0, 3)], heads, kv_heads, dim, 16, seed=heads).check()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("nodes,words", [(1, 1), (7, 1), (32, 1), (33, 2), (61, 2), (130, 5), (40, 1)])
def test_random_masks(cuda, dtype, nodes, words):
    """Any bits, rows that see none of the new tokens among them; 40 tokens with one word: the others unseen."""
    Case(cuda, [(90, nodes), (0, nodes), (129, max(1, nodes // 2))], 8, 2, 64, 16, dtype, words=words, seed=nodes,
         poison=True).check()


@pytest.mark.parametrize("dim", [64, 128])
def test_rows_that_see_nothing(cuda, dim):
    """No cached token and an empty mask: 0 and -inf, beside rows that do see something."""
    c = Case(cuda, [(0, 6), (4, 3), (0, 2)], 4, 2, dim, 16, words=1)
    c.mask[:] = 0
    c.mask[2] = 0b101
    out, lse = c.check()
    assert bool((out[[0, 1, 3, 4, 5, 9, 10]] == 0).all()) and bool((lse[[0, 1, 3, 4, 5, 9, 10]] == -float("inf")).all())
    assert bool((lse[2] > -float("inf")).all())


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("tree", [False, True])
def test_values_in_masked_places(cuda, dim, tree, bad):
    """NaN or infinite keys and values of a token that a row does not see leave the row as it is."""
    n = 40
    c = Case(cuda, [(50, n), (3, n)], 8, 2, dim, 16, words=2 if tree else 0, seed=7)
    victim = 17
    if tree:
        for t in range(2 * n):
            if t % n != victim and t % 3:
                c.mask[t, 0] &= ~(1 << victim)
    clean, clean_lse = c.run()
    for b, ctx in enumerate(c.context):
        p = ctx + victim
        c.k[c.table[b][p // 16], p % 16] = bad
        c.v[c.table[b][p // 16], p % 16] = bad
    out, lse = c.run()
    unseen = torch.tensor([(((int(c.mask[t, 0]) >> victim) & 1) == 0) if tree else (t % n) < victim for t in range(2 * n)],
                          device=cuda)
    assert int(unseen.sum()) > 10
    assert torch.equal(out[unseen], clean[unseen]) and torch.equal(lse[unseen], clean_lse[unseen])
    assert bool((~torch.isfinite(out[~unseen])).any(-1).all())


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_a_seen_value_that_is_not_finite(cuda, bad):
    """An infinite or NaN element of a value that rows see comes out in that element alone."""
    for dim, tree in ((64, False), (128, True)):
        c = Case(cuda, [(20, 6)], 4, 2, dim, 16, words=1 if tree else 0)
        if tree:
            c.mask[:] = 0b111111
        clean, _ = c.run()
        p = 20 + 2
        c.v[c.table[0][p // 16], p % 16, :, 5] = bad
        out, _ = c.run()
        rows = slice(0, 6) if tree else slice(2, 6)
        hit = out[rows, :, 5]
        assert bool(hit.isnan().all() if bad != bad else (hit == bad).all())
        out[rows, :, 5] = clean[rows, :, 5]
        assert torch.equal(out, clean)


@pytest.mark.parametrize("spread", [0.05, 8.0])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_flat_and_peaked_rows(cuda, dtype, spread):
    Case(cuda, [(900, 4), (130, 9)], 8, 2, 64, 16, dtype, spread=spread).check()
    Case(cuda, [(900, 4), (130, 9)], 8, 2, 128, 16, dtype, spread=spread).check()


@pytest.mark.parametrize("sm_scale", [0.3, -0.2, 1e-3])
def test_scales(cuda, sm_scale):
    Case(cuda, [(200, 3)], 4, 4, 64, 32).check(sm_scale)
    Case(cuda, [(200, 3)], 4, 4, 128, 32).check(sm_scale)


def test_lowest_scores(cuda):
    """Scores at the type's lowest value are scores, not masks: rows of equal ones average their values."""
    c = Case(cuda, [(30, 2)], 2, 1, 64, 16)
    c.q[:] = 0
    c.q[..., 0] = -60000.0
    c.k[:] = 0
    c.k[..., 0] = 60000.0
    c.check(1.0)


@pytest.mark.parametrize("dim", [64, 128])
def test_chunks_of_prompts(cuda, dim):
    """More query rows than one tile holds, causal, with and without cached tokens."""
    Case(cuda, [(0, 150), (77, 260), (3, 1)], 8, 4, dim, 32, seed=3).check()
    Case(cuda, [(40, 131)], 3, 1, dim, 16, torch.bfloat16, seed=4).check()


def test_long_cache_few_rows(cuda):
    """One request, a cache long enough to be divided among the whole GPU."""
    Case(cuda, [(20011, 3)], 4, 1, 64, 64).check()
    Case(cuda, [(9001, 1), (12, 1), (7777, 2)], 2, 2, 128, 16, torch.bfloat16).check()


def test_many_short_requests(cuda):
    rng = random.Random(1)
    Case(cuda, [(rng.randint(0, 40), rng.randint(0, 2)) for _ in range(700)], 4, 2, 64, 16).check()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,tokens", [(8, 1), (4, 6), (8, 9)])
def test_ragged_batches(cuda, dim, dtype, heads, tokens):
    """More units than CTAs, each with its share of several: the pipeline runs on from unit to unit, through caches of
    no tile to a dozen, whatever the parity of what it has done before."""
    rng = random.Random(heads * tokens)
    lengths = [(rng.choice([0, 5, 128, 300, 700, 1500]), rng.randint(0, tokens)) for _ in range(90)]
    Case(cuda, lengths, heads, 8 if heads == 8 else 4, dim, 16, dtype, words=1 if tokens > 1 else 0, seed=tokens,
         poison=True).check()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("page", [16, 256])
def test_caches_of_one_page_among_longer_ones(cuda, dim, page):
    """Tiles of a single page, which one of two loading warps fetches alone, by the dozen in each CTA, then tiles of many:
    the other warp must neither wait for what has come and gone nor miss its turn. Many runs, as it is a matter of time."""
    rng = random.Random(page + dim)
    lengths = [(rng.choice([3, 9, 15, 15, 15, 900]), 1) for _ in range(900)]
    c = Case(cuda, lengths, 4, 4, dim, page)
    first = c.check()
    for _ in range(100):
        again = c.run()
    assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
    assert fa.device_error() == 0


def test_repeatable(cuda):
    """The same bits every time: no sum depends on the order in which parts finish."""
    c = Case(cuda, [(9000, 4), (501, 4), (33, 4)], 8, 2, 128, 16)
    first = c.run()
    for _ in range(5):
        again = c.run()
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_padding_rows(cuda):
    """Rows of q past the last request (a fixed-size batch): 0 and -inf."""
    c = Case(cuda, [(100, 3), (5, 2)], 4, 2, 64, 16, tail=4)
    out, lse = c.check()
    assert bool((out[5:] == 0).all()) and bool((lse[5:] == -float("inf")).all())


def test_strides(cuda):
    """q as a slice of a fused projection, caches as slices of one allocation, tables as slices of a wider one."""
    c = Case(cuda, [(100, 3), (37, 5)], 8, 2, 64, 16)
    want, wlse = c.run()
    fused = torch.randn(8, 12, 64, device=cuda).half()
    fused[:, :8] = c.q
    c.q = fused[:, :8]
    both = torch.stack([c.k, c.v], 1)
    c.k, c.v = both[:, 0], both[:, 1]
    i = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    table = torch.zeros(2, 40, dtype=torch.int32, device=cuda)
    table[:, 5:5 + len(c.table[0])] = i(c.table)
    out, lse = fa.tree_attention(c.q, c.k, c.v, table[:, 5:5 + len(c.table[0])], i(c.context), i(c.cu), return_lse=True)
    assert torch.equal(out, want) and torch.equal(lse, wlse)
    buf = torch.empty_like(want)
    got, none = fa.tree_attention(c.q, c.k, c.v, table[:, 5:5 + len(c.table[0])], i(c.context), i(c.cu), out=buf)
    assert got.data_ptr() == buf.data_ptr() and none is None and torch.equal(buf, want)


def test_lengths_and_blocks_out_of_range_are_recorded(cuda):
    """A cache longer than the table's row, a block number that names none: recorded, and nothing is read there."""
    c = Case(cuda, [(30, 1), (10, 1)], 2, 1, 64, 16)
    good, _ = c.run()
    c.context[0] = 10 ** 6
    out, _ = c.run()
    assert fa.device_error() == 2
    assert torch.equal(out[1], good[1])
    c.context[0] = 30
    c.table[0][0] = -5
    out, _ = c.run()
    assert fa.device_error() == 2
    assert torch.equal(out[1], good[1])


def test_concurrent_streams(cuda):
    """Two calls in flight on two streams do not share their working memory."""
    a = Case(cuda, [(6000, 2), (100, 2)], 8, 2, 64, 16, seed=1)
    b = Case(cuda, [(5000, 3)], 4, 1, 64, 32, seed=2)
    wa, wb = a.run(), b.run()
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(8):
        with torch.cuda.stream(s1):
            ga = a.run()
        with torch.cuda.stream(s2):
            gb = b.run()
        torch.cuda.synchronize()
        assert torch.equal(ga[0], wa[0]) and torch.equal(gb[0], wb[0])


def test_captured_into_a_graph(cuda):
    """Lengths are read on the device: a captured call follows them."""
    c = Case(cuda, [(300, 2), (40, 2)], 4, 2, 64, 16)
    i = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    table, ctx, cu = i(c.table), i(c.context), i(c.cu)
    call = lambda: fa.tree_attention(c.q, c.k, c.v, table, ctx, cu, return_lse=True)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = call()
    for lengths in ([300, 40], [20, 7], [299, 0]):
        ctx.copy_(i(lengths))
        graph.replay()
        want, wlse = call()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(lse, wlse)
