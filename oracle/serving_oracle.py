"""64-bit CPU statements of the serving operators and rotary positions: the
formulas, token by token and request by request. Test infrastructure only;
never imported by the package. The reference has no counterpart."""
from __future__ import annotations

import math

import torch

#: Unit roundoff of the storage types (half of the spacing above 1).
UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def rotate(x, table, positions, interleaved=False, inverse=False):
    """``x`` [tokens, heads, D] (any type) with ``positions`` [tokens]; returns (y, magnitude), float64, where
    magnitude is the sum of the absolute products that make up each element of y."""
    x = x.double().cpu()
    table = table.double().cpu()
    rot = table.shape[1]
    y, mag = x.clone(), x.abs()
    for t, p in enumerate(positions.tolist()):
        for j in range(rot // 2):
            a, b = (2 * j, 2 * j + 1) if interleaved else (j, j + rot // 2)
            c, s = float(table[p, j]), float(table[p, rot // 2 + j])
            s = -s if inverse else s
            x0, x1 = x[t, :, a], x[t, :, b]
            y[t, :, a], y[t, :, b] = x0 * c - x1 * s, x1 * c + x0 * s
            mag[t, :, a], mag[t, :, b] = (x0 * c).abs() + (x1 * s).abs(), (x1 * c).abs() + (x0 * s).abs()
    return y, mag


def plan(context, cu, table, held, free, num_free, tokens, page, parents=None, words=0):
    """Lists in, lists out: (table, slots, positions, admitted, num_free, held, mask rows as unsigned words)."""
    table = [list(r) for r in table]
    held = list(held)
    slots, positions, admitted = [-1] * tokens, [0] * tokens, []
    masks = [[0] * words for _ in range(tokens)]
    upto, used = 0, 0
    for b, ctx in enumerate(context):
        count = cu[b + 1] - cu[b]
        have = max(held[b], -(-ctx // page))
        want = max(have, -(-(ctx + count) // page))
        fits = want <= len(table[b])
        need = want - have if fits else 0
        ok = fits and (need == 0 or upto + need <= num_free)
        admitted.append(ok)
        if ok:
            for j in range(need):
                table[b][have + j] = free[num_free - 1 - (upto + j)]
            if need:
                used = upto + need
        held[b] = want if ok else have
        upto += need
        for i in range(count):
            t = cu[b] + i
            if ok:
                slots[t] = table[b][(ctx + i) // page] * page + (ctx + i) % page
            positions[t] = ctx + i
            if parents is not None:
                chain, node = [], i
                while node >= 0:
                    chain.append(node)
                    node = parents[cu[b] + node]
                positions[t] = ctx + len(chain) - 1
                for n in chain:
                    masks[t][n // 32] |= 1 << (n % 32)
    return table, slots, positions, admitted, num_free - used, held, masks


def visible(i, count, mask_row=None):
    """Which of its request's ``count`` new tokens token i sees."""
    if mask_row is None:
        return [j for j in range(count) if j <= i]
    return [j for j in range(count) if j // 32 < len(mask_row) and (int(mask_row[j // 32]) >> (j % 32)) & 1]


def tree_attention(q, k_cache, v_cache, table, context, cu, tree_mask=None, sm_scale=0.0, layout="bnhd"):
    """(out, lse, weight, reach) in float64: weight = sum_j p_j |v_j| (what rounding p and out scales with), reach =
    the largest sum_d |q_d k_jd| * scale of the row (what the scores' rounding scales with)."""
    q, k_cache, v_cache = q.double().cpu(), k_cache.double().cpu(), v_cache.double().cpu()
    if layout == "bhnd":
        k_cache, v_cache = k_cache.transpose(1, 2), v_cache.transpose(1, 2)
    page, kv_heads = k_cache.shape[1], k_cache.shape[2]
    tokens, heads, dim = q.shape
    scale = sm_scale if sm_scale else 1.0 / math.sqrt(dim)
    out = torch.zeros(tokens, heads, dim, dtype=torch.float64)
    weight = torch.zeros_like(out)
    lse = torch.full((tokens, heads), -math.inf, dtype=torch.float64)
    reach = torch.zeros(tokens, heads, dtype=torch.float64)
    for b, ctx in enumerate(context):
        count = cu[b + 1] - cu[b]
        place = list(range(ctx + count))
        rows = torch.tensor([int(table[b][p // page]) * page + p % page for p in place], dtype=torch.long)
        kb = k_cache.reshape(-1, kv_heads, dim)[rows]
        vb = v_cache.reshape(-1, kv_heads, dim)[rows]
        for i in range(count):
            t = cu[b] + i
            seen = list(range(ctx)) + [ctx + j for j in
                                       visible(i, count, None if tree_mask is None else tree_mask[t].tolist())]
            if not seen:
                continue
            ks = kb[seen].repeat_interleave(heads // kv_heads, dim=1)
            vs = vb[seen].repeat_interleave(heads // kv_heads, dim=1)
            s = torch.einsum("hd,jhd->hj", q[t], ks) * scale
            lse[t] = torch.logsumexp(s, 1)
            p = (s - lse[t][:, None]).exp()
            out[t] = torch.einsum("hj,jhd->hd", p, vs)
            weight[t] = torch.einsum("hj,jhd->hd", p, vs.abs())
            reach[t] = torch.einsum("hd,jhd->hj", q[t].abs(), ks.abs()).amax(1) * abs(scale)
    return out, lse, weight, reach
