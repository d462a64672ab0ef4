"""Cases for the serving operators and the rotary positions of flashlite_b200.

Three operators, which one step of a serving loop runs one after the other:

* ``plan``: from the requests' lengths, the block table's new entries, the slot
  and the position of every new token and, for trees of drafted tokens, the
  packed ancestor masks.
* ``rotary``: rotary positions of queries and keys; as a training step uses
  them (forward and gradient) and as a serving step does (rotated keys and the
  values go straight to their slots of the paged cache).
* ``attention``: the new tokens' attention over the paged cache, with the
  visibility of a tree of drafted tokens or causal among the new tokens.

``run`` computes them in plain torch, or, with ``own`` true, by the calls a
user makes of the framework. Lengths go by the case; data go by the seed.
"""
import math
import random

import torch

own = False

DEV = "cuda"
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


# --------------------------------------------------------------------------
# cases
# --------------------------------------------------------------------------
def listed():
    return [
        # One decode step's bookkeeping for a small batch: latency alone.
        dict(name="plan_decode_small", op="plan", requests=7, context=900, tokens=1, page=16, tree=False),
        # A verification step of a large batch, each request with a tree of 61 drafted tokens.
        dict(name="plan_tree", op="plan", requests=192, context=6000, tokens=61, page=32, tree=True),
        # Mixed prompts entering at once: over a hundred thousand new slots.
        dict(name="plan_prompts", op="plan", requests=509, context=2500, tokens=513, page=16, tree=False),
        # Query and key positions of one training step, forward and gradient: 2 x 8 heads x 4096 x 64.
        dict(name="rotary_train", op="rotary", batch=2, length=4096, heads=8, kv_heads=8, dim=64, rot=64,
             interleaved=False, layout="bhnd", dtype="fp16", scaling="none"),
        # A long-context training step with shared key heads, part of the head rotated, interleaved pairs.
        dict(name="rotary_train_long", op="rotary", batch=3, length=16381, heads=32, kv_heads=8, dim=128, rot=96,
             interleaved=True, layout="bnhd", dtype="bf16", scaling="by_parts"),
        # One decode step of a few requests: rotate and append, latency alone.
        dict(name="append_decode", op="append", tokens=5, heads=8, kv_heads=8, dim=64, rot=64, interleaved=False,
             page=16, blocks=512, layout="bnhd", dtype="fp16", scaling="none"),
        # A prompt of odd length entering the cache.
        dict(name="append_prompt", op="append", tokens=8191, heads=32, kv_heads=8, dim=128, rot=128,
             interleaved=False, page=32, blocks=640, layout="bnhd", dtype="bf16", scaling="linear"),
        # The smallest attention call: one request, one token, a short cache.
        dict(name="attention_single", op="attention", requests=1, tokens=1, context=777, heads=8, kv_heads=8,
             dim=64, page=16, layout="bnhd", dtype="fp16", tree=False),
        # Decode of a ragged batch with shared key heads.
        dict(name="attention_decode", op="attention", requests=64, tokens=1, context=8192, heads=32, kv_heads=8,
             dim=128, page=16, layout="bnhd", dtype="bf16", tree=False),
        # Verification of trees of drafted tokens, ragged batch.
        dict(name="attention_tree", op="attention", requests=16, tokens=61, context=5000, heads=32, kv_heads=8,
             dim=128, page=64, layout="bhnd", dtype="fp16", tree=True),
        # One request with a very long cache and a small tree.
        dict(name="attention_long", op="attention", requests=1, tokens=8, context=131072, heads=8, kv_heads=8,
             dim=64, page=128, layout="bnhd", dtype="fp16", tree=True),
        # Chunks of prompts over what is cached already: bound by the products.
        dict(name="attention_chunk", op="attention", requests=4, tokens=509, context=8192, heads=32, kv_heads=8,
             dim=128, page=32, layout="bnhd", dtype="bf16", tree=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["plan", "rotary", "append", "attention", "attention", "attention"])
    if op == "plan":
        tree = rng.random() < 0.5
        requests = _log(rng, 1, 600)
        tokens = _log(rng, 1, 64 if tree else 512)
        return dict(op=op, requests=requests, context=_log(rng, 1, 8000), tokens=tokens,
                    page=rng.choice([8, 16, 32, 64, 128]), tree=tree)
    dim = rng.choice([64, 128])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 1, 2, 3, 4, 5, 7, 8])
    dtype = rng.choice(["fp16", "bf16"])
    layout = rng.choice(["bnhd", "bhnd"])
    if op in ("rotary", "append"):
        rot = rng.choice([dim, dim, dim // 2, dim // 4 * 3])
        more = dict(heads=heads, kv_heads=kv_heads, dim=dim, rot=rot, interleaved=rng.random() < 0.5, layout=layout,
                    scaling=rng.choice(["none", "linear", "ntk", "by_parts"]))
        most = 3 * 16381 * 40 * 128 // ((heads + 2 * kv_heads) * dim)
        if op == "rotary":
            batch = rng.choice([1, 2, 3, 4])
            length = _log(rng, 1, min(16384, most // batch))
            return dict(op=op, batch=batch, length=length, dtype=rng.choice([dtype, dtype, "fp32"]), **more)
        tokens = _log(rng, 1, min(16384, most))
        page = rng.choice([8, 16, 32, 64, 128])
        return dict(op=op, tokens=tokens, page=page, blocks=-(-tokens // page) * 2 + 3, dtype=dtype, **more)
    tree = rng.random() < 0.5
    requests = _log(rng, 1, 64)
    tokens = _log(rng, 1, 64) if tree or rng.random() < 0.6 else _log(rng, 64, 512)
    # at most the bytes of attention_decode and the products of attention_chunk
    most = min(64 * 8192 * 8 * 128 / (requests * kv_heads * dim), 4 * 509 * 8192 * 32 * 128 / (requests * tokens * heads * dim))
    context = _log(rng, 1, max(1, min(131072, int(most))))
    return dict(op=op, requests=requests, tokens=tokens, context=context, heads=heads, kv_heads=kv_heads, dim=dim,
                page=rng.choice([16, 32, 64, 128]), layout=layout, dtype=dtype, tree=tree)


def _lengths(case):
    """(cached, new) tokens of each request: the largest is the case's own, the others spread below it."""
    n = case["requests"]
    golden = 0.6180339887498949
    cached = [case["context"]] + [int(case["context"] * (0.125 + 0.875 * (b * golden % 1.0))) for b in range(1, n)]
    new = [case["tokens"]] * n
    if case["op"] == "plan" and not case["tree"] and case["tokens"] > 1:  # prompts differ in length
        new = [case["tokens"]] + [1 + int((case["tokens"] - 1) * (b * golden * golden % 1.0)) for b in range(1, n)]
    return cached, new


def _parents(case, new):
    """A tree for each request: node i hangs below one of the nodes before it, or below the cached tokens (-1)."""
    r = random.Random(case["tokens"] * 1000 + case["requests"])
    return [[r.choice([-1] + list(range(max(0, i - 9), i))) if i else -1 for i in range(t)] for t in new]


def _visible(parents):
    """0/1 rows: node i sees its ancestors and itself."""
    rows = []
    for i, p in enumerate(parents):
        row = list(rows[p]) if p >= 0 else [0] * len(parents)
        row[i] = 1
        rows.append(row)
    return rows


# --------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------
def _table(positions, rot, scaling, base=10000.0):
    """[positions, rot] fp32: rot/2 cosines, then rot/2 sines, for contexts `factor` times the trained length."""
    factor, original = 8.0, 2048
    j = torch.arange(rot // 2, dtype=torch.float64, device=DEV)
    scale = 1.0
    if scaling == "ntk":
        base = base * factor ** (rot / (rot - 2))
    freq = base ** (-2.0 * j / rot)
    if scaling == "linear":
        freq = freq / factor
    elif scaling == "by_parts":  # fast pairs keep their frequency, slow ones are stretched, a ramp between
        turns = original * freq / (2 * math.pi)
        keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0.0, 1.0)
        freq = freq * keep + freq / factor * (1.0 - keep)
        scale = 0.1 * math.log(factor) + 1.0
    angle = torch.arange(positions, dtype=torch.float64, device=DEV)[:, None] * freq
    return torch.cat([angle.cos() * scale, angle.sin() * scale], 1).float()


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device=DEV)


def _cumulated(values):
    out = [0]
    for v in values:
        out.append(out[-1] + v)
    return out


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    state = dict(case=case)
    op = case["op"]
    if op == "plan":
        cached, new = _lengths(case)
        page = case["page"]
        have = [-(-c // page) for c in cached]
        want = [-(-(c + t) // page) for c, t in zip(cached, new)]
        width = max(want)
        total = sum(want)
        order = torch.randperm(total + 17, generator=g, device=DEV).to(torch.int32)
        table = torch.zeros(len(cached), width, dtype=torch.int32, device=DEV)
        column = torch.arange(width, device=DEV)[None]
        held = column < _ints(have, torch.int64)[:, None]
        table[held] = order[: sum(have)]
        free = order[sum(have):].contiguous()
        state.update(context_lens=_ints(cached), cu_seqlens=_ints(_cumulated(new)), block_table=table,
                     held_blocks=_ints(have), free_blocks=free, num_free=_ints([free.numel()]), total=sum(new), page=page, parents=None, words=0)
        if case["tree"]:
            state.update(parents=_ints(sum(_parents(case, new), [])), words=-(-case["tokens"] // 32))
        return state
    dtype = TYPES[case["dtype"]]
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32).to(dtype)

    if op == "rotary":
        batch, length = case["batch"], case["length"]
        shape = (lambda h: (batch, length, h, dim)) if case["layout"] == "bnhd" else (lambda h: (batch, h, length, dim))
        state.update(q=normal(*shape(heads)), k=normal(*shape(kv_heads)), dq=normal(*shape(heads)),
                     dk=normal(*shape(kv_heads)), table=_table(length, case["rot"], case["scaling"]),
                     positions=torch.arange(length, dtype=torch.int32, device=DEV))
        return state
    page = case["page"]
    paged = (lambda n: (n, page, kv_heads, dim)) if case["layout"] == "bnhd" else (lambda n: (n, kv_heads, page, dim))
    if op == "append":
        t = case["tokens"]
        start = 4 * case["page"] + 5
        slots = torch.randperm(case["blocks"] * page, generator=g, device=DEV)
        if t > 64:  # a prompt fills whole blocks, which lie anywhere
            block = torch.randperm(case["blocks"], generator=g, device=DEV)
            at = torch.arange(t, device=DEV)
            slots = block[at // page] * page + at % page
        state.update(q=normal(t, heads, dim), k=normal(t, kv_heads, dim), v=normal(t, kv_heads, dim),
                     table=_table(start + t, case["rot"], case["scaling"]),
                     positions=torch.arange(start, start + t, dtype=torch.int32, device=DEV), slots=slots[:t].contiguous(),
                     k_cache=torch.zeros(paged(case["blocks"]), dtype=dtype, device=DEV),
                     v_cache=torch.zeros(paged(case["blocks"]), dtype=dtype, device=DEV))
        return state
    cached, new = _lengths(case)
    width = max(-(-(c + t) // page) for c, t in zip(cached, new))
    counts = [-(-(c + t) // page) for c, t in zip(cached, new)]
    blocks = sum(counts) + 3
    order = torch.randperm(blocks, generator=g, device=DEV).to(torch.int32)
    table = torch.zeros(len(cached), width, dtype=torch.int32, device=DEV)
    table[torch.arange(width, device=DEV)[None] < _ints(counts, torch.int64)[:, None]] = order[: sum(counts)]
    state.update(q=normal(sum(new), heads, dim), k_cache=normal(*paged(blocks)), v_cache=normal(*paged(blocks)),
                 block_table=table, context_lens=_ints(cached), cu_seqlens=_ints(_cumulated(new)),
                 most=max(new), tree_mask=None)
    if case["tree"]:
        words = -(-case["tokens"] // 32)
        rows = []
        for parents in _parents(case, new):
            for row in _visible(parents):
                value = sum(1 << j for j, on in enumerate(row) if on)
                rows.append([(w - (1 << 32) if w >> 31 else w) for w in ((value >> (32 * i)) & 0xFFFFFFFF for i in range(words))])
        state.update(tree_mask=_ints(rows))
    return state


# --------------------------------------------------------------------------
# the plain forms
# --------------------------------------------------------------------------
def _plan(s):
    ctx, cu, table, page = s["context_lens"].long(), s["cu_seqlens"].long(), s["block_table"], s["page"]
    new = cu[1:] - cu[:-1]
    have = s["held_blocks"].long()
    want = torch.maximum(have, (ctx + new + page - 1) // page)
    fits = want <= table.shape[1]
    need = torch.where(fits, want - have, 0)
    upto = need.cumsum(0)
    free = s["num_free"].long()
    admitted = fits & ((need == 0) | (upto <= free))
    used = torch.where(admitted & (need > 0), upto, 0).amax()
    column = torch.arange(table.shape[1], device=table.device)[None]
    fresh = admitted[:, None] & (column >= have[:, None]) & (column < want[:, None])
    source = free - 1 - ((upto - need)[:, None] + column - have[:, None])
    table.copy_(torch.where(fresh, s["free_blocks"][source.clamp(0, s["free_blocks"].numel() - 1)], table))
    token = torch.arange(s["total"], device=table.device)
    request = torch.searchsorted(cu[1:], token, right=True).clamp(max=new.numel() - 1)
    index = token - cu[request]
    place = ctx[request] + index
    slot = table[request, (place // page).clamp(max=table.shape[1] - 1)].long() * page + place % page
    slots = torch.where(admitted[request], slot, -1)
    left, held = (free - used).int(), torch.where(admitted, want, have).int()
    if s["parents"] is None:
        return table, slots, place.int(), admitted, left, held, None
    width = 32 * s["words"]
    above = torch.zeros(new.numel(), width, width, device=table.device)
    inner = s["parents"] >= 0
    above[request[inner], index[inner], s["parents"][inner].long()] = 1.0
    closure = above + torch.eye(width, device=table.device)
    for _ in range(max(1, (width - 1).bit_length())):
        closure = (closure @ closure).clamp(max=1.0)
    rows = closure[request, index].long()
    positions = ctx[request] + rows.sum(1) - 1
    bits = (rows.view(-1, s["words"], 32) << torch.arange(32, device=table.device)).sum(2)
    mask = torch.where(bits >= 1 << 31, bits - (1 << 32), bits).int()
    return table, slots, positions.int(), admitted, left, held, mask


def _rotated(x, cos, sin, rot, interleaved):
    """x [..., dim] with cos and sin [..., rot/2] that broadcast against it, in 32 bits, rounded once."""
    f = x.float()
    part = f[..., :rot]
    if interleaved:
        a, b = part[..., 0::2], part[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = part[..., : rot // 2], part[..., rot // 2:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, f[..., rot:]], -1).to(x.dtype)


def _angles(s, head_axis, sign=1.0):
    rows = s["table"][s["positions"].long()]
    half = rows.shape[1] // 2
    return rows[:, :half].unsqueeze(head_axis), sign * rows[:, half:].unsqueeze(head_axis)


def _rotary(s):
    c = s["case"]
    axis = 0 if c["layout"] == "bhnd" else 1
    cos, sin = _angles(s, axis)
    turn = lambda x, sn: _rotated(x, cos, sn, c["rot"], c["interleaved"])  # noqa: E731
    return turn(s["q"], sin), turn(s["k"], sin), turn(s["dq"], -sin), turn(s["dk"], -sin)


def _append(s):
    c = s["case"]
    cos, sin = _angles(s, 1)
    q = _rotated(s["q"], cos, sin, c["rot"], c["interleaved"])
    k = _rotated(s["k"], cos, sin, c["rot"], c["interleaved"])
    block, at = s["slots"] // c["page"], s["slots"] % c["page"]
    for cache, x in ((s["k_cache"], k), (s["v_cache"], s["v"])):
        if c["layout"] == "bnhd":
            cache[block, at] = x
        else:
            cache[block, :, at] = x
    return q, s["k_cache"], s["v_cache"]


def _gathered(cache, table, layout):
    """[requests, heads, keys, dim] in 32 bits of the pages that the table names."""
    x = cache[table.long()]
    x = x.permute(0, 3, 1, 2, 4) if layout == "bnhd" else x.permute(0, 2, 1, 3, 4)
    return x.float().reshape(x.shape[0], x.shape[1], -1, x.shape[4])


def _attention(s):
    c = s["case"]
    cu, ctx = s["cu_seqlens"].long(), s["context_lens"].long()
    n, most, heads, kv_heads, dim = ctx.numel(), s["most"], c["heads"], c["kv_heads"], c["dim"]
    new = cu[1:] - cu[:-1]
    i = torch.arange(most, device=cu.device)
    token = (cu[:-1, None] + i).clamp(max=s["q"].shape[0] - 1)
    q = s["q"][token].float().view(n, most, kv_heads, heads // kv_heads, dim).permute(0, 2, 3, 1, 4).flatten(2, 3)
    k, v = _gathered(s["k_cache"], s["block_table"], c["layout"]), _gathered(s["v_cache"], s["block_table"], c["layout"])
    key = torch.arange(k.shape[2], device=cu.device)
    draft = key - ctx[:, None]  # [n, keys]: which of its request's new tokens a key is
    if s["tree_mask"] is None:
        seen = draft[:, None, :] <= i[None, :, None]
    else:
        words = s["tree_mask"][token]
        at = draft.clamp(0, 32 * words.shape[2] - 1)
        bits = torch.gather(words, 2, (at // 32)[:, None, :].expand(-1, most, -1)) >> (at % 32)[:, None, :]
        seen = (draft < 0)[:, None, :] | ((bits & 1) == 1)
    seen = seen & (draft < new[:, None])[:, None, :]
    seen = seen[:, None, None].expand(-1, 1, heads // kv_heads, -1, -1).flatten(2, 3)
    scores = (q @ k.transpose(2, 3)) * (1.0 / math.sqrt(dim))
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(3, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = (scores - top).exp()
    total = p.sum(3, keepdim=True)
    out = (p @ v) / torch.where(total > 0, total, 1.0)
    lse = (top + total.log()).squeeze(3)
    live = (i < new[:, None])
    out = out.view(n, kv_heads, heads // kv_heads, most, dim).permute(0, 3, 1, 2, 4).reshape(n, most, heads, dim)
    lse = lse.view(n, kv_heads, heads // kv_heads, most).permute(0, 3, 1, 2).reshape(n, most, heads)
    rows = live.flatten().nonzero().squeeze(1) if most > 1 else slice(None)
    return out.flatten(0, 1)[rows].to(s["q"].dtype), lse.flatten(0, 1)[rows]


# --------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------
def run(state):
    s, c = state, state["case"]
    if not own:
        return {"plan": _plan, "rotary": _rotary, "append": _append, "attention": _attention}[c["op"]](s)
    from flashlite_b200 import flash_attn_wmma as fa

    if c["op"] == "plan":
        slots, positions, admitted, left, held, mask = fa.plan_cache_step(
            s["context_lens"], s["cu_seqlens"], s["block_table"], s["held_blocks"], s["free_blocks"], s["num_free"],
            s["total"], s["page"], parents=s["parents"], mask_words=s["words"])
        return s["block_table"], slots, positions, admitted, left, held, mask
    if c["op"] == "rotary":
        more = dict(interleaved=c["interleaved"], layout=c["layout"])
        q, k = fa.rotary(s["q"], s["k"], s["table"], s["positions"], **more)
        dq, dk = fa.rotary_backward(s["dq"], s["dk"], s["table"], s["positions"], **more)
        return q, k, dq, dk
    if c["op"] == "append":
        q = fa.rotary_append(s["q"], s["k"], s["v"], s["table"], s["positions"], s["slots"], s["k_cache"], s["v_cache"],
                             interleaved=c["interleaved"], layout=c["layout"])
        return q, s["k_cache"], s["v_cache"]
    out, lse = fa.tree_attention(s["q"], s["k_cache"], s["v_cache"], s["block_table"], s["context_lens"], s["cu_seqlens"],
                                 tree_mask=s["tree_mask"], layout=c["layout"], return_lse=True)
    return out, lse


# --------------------------------------------------------------------------
# what a pass cannot do without
# --------------------------------------------------------------------------
def work(case):
    op = case["op"]
    if op == "plan":
        cached, new = _lengths(case)
        n, t = len(cached), sum(new)
        fresh = sum(-(-(c + x) // case["page"]) + (-c // case["page"]) for c, x in zip(cached, new))
        words = -(-case["tokens"] // 32) if case["tree"] else 0
        # lengths and offsets read, fresh blocks read and written, a slot and a position for each token, parents and masks
        return {"bytes": n * (4 + 4 + 4 + 4 + 1) + 8 * fresh + 12 * t + (4 + 4 * words) * t * case["tree"], "flops": 4 * t}
    size = 4 if case["dtype"] == "fp32" else 2
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    if op == "rotary":
        t = case["batch"] * case["length"]
        return {"bytes": 4 * t * (heads + kv_heads) * dim * size + case["length"] * (4 * case["rot"] + 4),
                "flops": 2 * 3 * t * (heads + kv_heads) * case["rot"]}
    if op == "append":
        t = case["tokens"]
        return {"bytes": 2 * t * (heads + 2 * kv_heads) * dim * size + t * (4 * case["rot"] + 12),
                "flops": 3 * t * (heads + kv_heads) * case["rot"]}
    cached, new = _lengths(case)
    if case["tree"]:
        inner = sum(sum(map(sum, _visible(p))) for p in _parents(case, new))
    else:
        inner = sum(t * (t + 1) // 2 for t in new)
    pairs = inner + sum(c * t for c, t in zip(cached, new))
    keys = sum(c + t for c, t in zip(cached, new))
    return {"bytes": 2 * keys * kv_heads * dim * size + sum(new) * heads * (2 * dim * size + 4), "flops": 4 * pairs * heads * dim}


# --------------------------------------------------------------------------
# the definitions in 64 bits
# --------------------------------------------------------------------------
def _exact_rotation(x, table, where, rot, interleaved, transposed):
    """Each pair (x0, x1) as a complex number times cos + i sin (the gradient: times its conjugate). x: [tokens, heads, dim]."""
    row = table.double()[where.long()]
    turn = torch.complex(row[:, : rot // 2], row[:, rot // 2:])[:, None]
    turn = turn.conj() if transposed else turn
    y = x.double().clone()
    first = torch.arange(0, rot, 2, device=x.device) if interleaved else torch.arange(rot // 2, device=x.device)
    second = first + (1 if interleaved else rot // 2)
    z = torch.complex(y[..., first], y[..., second]) * turn
    y[..., first], y[..., second] = z.real, z.imag
    return y


def exact(case, seed):
    op = case["op"]
    if op == "plan":  # whole numbers only
        return None
    s = prepare(case, seed)
    if op == "rotary":
        where = s["positions"].repeat(case["batch"])

        def one(x, transposed):
            y = x.transpose(1, 2) if case["layout"] == "bhnd" else x
            z = _exact_rotation(y.reshape(-1, y.shape[2], y.shape[3]), s["table"], where, case["rot"], case["interleaved"], transposed)
            z = z.view(y.shape)
            return z.transpose(1, 2) if case["layout"] == "bhnd" else z

        return one(s["q"], False), one(s["k"], False), one(s["dq"], True), one(s["dk"], True)
    if op == "append":
        q = _exact_rotation(s["q"], s["table"], s["positions"], case["rot"], case["interleaved"], False)
        k = _exact_rotation(s["k"], s["table"], s["positions"], case["rot"], case["interleaved"], False)
        page = case["page"]

        def filled(cache, x):
            flat = cache.double()
            flat = flat.transpose(1, 2) if case["layout"] == "bhnd" else flat
            flat = flat.reshape(-1, flat.shape[2], flat.shape[3]).index_copy(0, s["slots"], x.double())
            flat = flat.view(-1, page, flat.shape[1], flat.shape[2])
            return flat.transpose(1, 2) if case["layout"] == "bhnd" else flat

        return q, filled(s["k_cache"], k), filled(s["v_cache"], s["v"])
    cached, new = _lengths(case)
    trees = _parents(case, new)
    heads, kv_heads, dim, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    outs, lses, at = [], [], 0
    for b, (c, t) in enumerate(zip(cached, new)):
        place = torch.arange(c + t, device=DEV)
        block = s["block_table"][b].long()[place // page]
        if case["layout"] == "bnhd":
            k, v = s["k_cache"][block, place % page], s["v_cache"][block, place % page]
        else:
            k, v = s["k_cache"][block, :, place % page], s["v_cache"][block, :, place % page]
        inner = torch.tensor(_visible(trees[b]), device=DEV) > 0 if case["tree"] else torch.ones(t, t, device=DEV).tril() > 0
        bias = torch.zeros(t, c + t, dtype=torch.float64, device=DEV)
        bias[:, c:][~inner] = -math.inf
        q = s["q"][at:at + t].double()
        out, lse = torch.empty_like(q), torch.empty(t, heads, dtype=torch.float64, device=DEV)
        for h in range(kv_heads):
            mine = slice(h * (heads // kv_heads), (h + 1) * (heads // kv_heads))
            score = torch.einsum("tgd,ld->tgl", q[:, mine], k[:, h].double()) / math.sqrt(dim) + bias[:, None]
            lse[:, mine] = torch.logsumexp(score, 2)
            out[:, mine] = torch.einsum("tgl,ld->tgd", (score - lse[:, mine, None]).exp(), v[:, h].double())
        outs.append(out)
        lses.append(lse)
        at += t
    return torch.cat(outs), torch.cat(lses)
