"""Operators around the paged key/value cache, each with cases of real use, a plain form and a definition in 64 bits.

Five operators of one decoder layer that serves from a paged cache:

  rotary      pos_encoding_ops.rotary_embedding: positions rotated in the half or the interleaved
              layout, over all or the first part of every head, with a plain or a stretched table
  qk_norm     pos_encoding_ops.qk_norm_rotary_embedding: RMS norm of every query and key head and the
              rotation in the same pass
  tree        attention_ops.tree_cached_kv_attention: drafted tokens of a tree (or chain) over the cache
  accumulate  attention_ops.cached_kv_attention_accumulate: attention over the cache that also adds
              every position's weight to a weight cache
  evict       cache_ops.evict_cached_kv: keeps the heaviest and the latest positions of every head,
              and moves them to the front of the sequence's blocks

Layouts, with x = 16 bytes of elements: key cache [blocks, kv heads, head size / x, block, x], value
cache [blocks, kv heads, head size, block], weight cache [blocks, kv heads, block] in float32.
Block 0 of every cache is nobody's: tables are padded with it.
"""
import functools
import math

import numpy as np
import torch

own = False

DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}
BYTES = {"float16": 2, "bfloat16": 2, "float32": 4}
EPSILON = 1e-6
BASE = 10000.0


@functools.lru_cache(maxsize=None)
def _package():
    import __graft_entry__
    return __graft_entry__.load_package()


# ---- cases ------------------------------------------------------------------------------------


def listed():
    return [
        # one step of a small batch that generates: the launch is all there is
        dict(name="rotary_step", op="rotary", dtype="float16", tokens=8, heads=32, kv_heads=32, head_size=128,
             rot_dim=128, interleaved=False, scaling="none", max_position=8192),
        # a long prompt of a model that rotates half of every head, pairs interleaved, far positions
        dict(name="rotary_prompt_part", op="rotary", dtype="bfloat16", tokens=16381, heads=32, kv_heads=8, head_size=128,
             rot_dim=64, interleaved=True, scaling="yarn", max_position=131072),
        # a generating batch of a model that norms its query and key heads
        dict(name="qk_norm_step", op="qk_norm", dtype="bfloat16", tokens=256, heads=32, kv_heads=8, head_size=128,
             rot_dim=128, interleaved=False, scaling="none", max_position=32768),
        # its prompts, forty heads of each
        dict(name="qk_norm_prompt", op="qk_norm", dtype="float16", tokens=8192, heads=40, kv_heads=40, head_size=128,
             rot_dim=128, interleaved=False, scaling="linear", max_position=32768),
        # one user, a tree of 26 drafted tokens: latency
        dict(name="tree_one", op="tree", dtype="float16", seqs=1, drafted=26, chain=False, even=True, heads=32, kv_heads=32,
             head_size=128, block=16, context=1024),
        # trees of up to 64 tokens in a batch of shared key/value heads, contexts of all lengths
        dict(name="tree_batch", op="tree", dtype="bfloat16", seqs=24, drafted=64, chain=False, even=False, heads=32, kv_heads=8,
             head_size=128, block=16, context=4096),
        # a serving batch that checks chains of five, one key/value head to each query head
        dict(name="tree_chain_batch", op="tree", dtype="float16", seqs=64, drafted=5, chain=True, even=False, heads=40,
             kv_heads=40, head_size=128, block=16, context=2048),
        # two long documents, short trees
        dict(name="tree_long", op="tree", dtype="bfloat16", seqs=2, drafted=12, chain=False, even=True, heads=32, kv_heads=8,
             head_size=128, block=32, context=40009),
        # one user, one token a step, weights kept for a later eviction: latency
        dict(name="accumulate_one", op="accumulate", dtype="float16", seqs=1, drafted=1, chain=True, even=True, heads=32,
             kv_heads=32, head_size=128, block=16, context=2048),
        # the same in a serving batch
        dict(name="accumulate_batch", op="accumulate", dtype="bfloat16", seqs=96, drafted=1, chain=True, even=False, heads=32,
             kv_heads=8, head_size=128, block=16, context=4096),
        # one short sequence over its budget
        dict(name="evict_one", op="evict", dtype="float16", seqs=1, heads=12, head_size=64, block=16, context=1025,
             budget=512, recent=64),
        # a batch brought back from 8 k positions to 2 k
        dict(name="evict_batch", op="evict", dtype="bfloat16", seqs=32, heads=8, head_size=128, block=16, context=8192,
             budget=2048, recent=512),
    ]


def _spread(rng, low, high):
    """A whole number of [low, high], even over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _heads(rng):
    kv = rng.choice([1, 2, 3, 4, 5, 8, 12, 16, 32])
    group = rng.choice([g for g in (1, 1, 2, 4, 5, 8) if g * kv <= 40])
    return kv * group, kv


def draw(rng):
    op = rng.choice(["rotary", "qk_norm", "tree", "tree", "accumulate", "evict"])
    dtype = rng.choice(["float16", "bfloat16", "float16", "bfloat16", "float32"])
    heads, kv_heads = _heads(rng)
    head_size = rng.choice([64, 80, 96, 128])
    if op in ("rotary", "qk_norm"):
        most = int(16384 * 40 * 128 / (40 * head_size)) // (2 if dtype == "float32" else 1)
        rot_dim = rng.choice([head_size, head_size, head_size // 2, 32, 24])
        return dict(op=op, dtype=dtype, tokens=_spread(rng, 1, most // 2), heads=heads, kv_heads=kv_heads, head_size=head_size,
                    rot_dim=rot_dim, interleaved=rng.random() < 0.5, scaling=rng.choice(["none", "linear", "ntk", "yarn"]),
                    max_position=rng.choice([2048, 8192, 32768, 131072]))
    block = rng.choice([8, 16, 32])
    if op == "evict":
        context = _spread(rng, 2, 16384)
        budget = max(1, int(context * rng.uniform(0.1, 1.1)))
        most = 1.5e9 / (kv_heads * head_size * BYTES[dtype] * 2 * context)
        return dict(op=op, dtype=dtype, seqs=_spread(rng, 1, max(1, min(64, int(most)))), heads=kv_heads, head_size=head_size,
                    block=block, context=context, budget=budget, recent=int(budget * rng.uniform(0, 1)))
    context = _spread(rng, 70, 40000)
    drafted = _spread(rng, 1, 64 if op == "tree" else 4)
    most = min(1.0e9 / (kv_heads * head_size * BYTES[dtype] * 2 * context),
               2.5e10 / (4.0 * heads * drafted * context * head_size) / (8 if dtype == "float32" else 1))
    return dict(op=op, dtype=dtype, seqs=_spread(rng, 1, max(1, min(128, int(most)))), drafted=drafted,
                chain=op != "tree" or rng.random() < 0.3, even=rng.random() < 0.4, heads=heads, kv_heads=kv_heads,
                head_size=head_size, block=block, context=context)


def _lengths(case):
    """Context lengths (drafted tokens among them) and numbers of drafted tokens of a case's sequences."""
    n, longest, most = case["seqs"], case["context"], case.get("drafted", 1)
    if case.get("even", True):
        return [longest] * n, [most] * n
    # a fixed irregular spread over a quarter to the whole, the first at the full size
    drafted = [most if i == 0 else max(1, most - (i * 7) % max(1, most // 2 + 1)) for i in range(n)]
    lens = [max(d, int(longest * (1.0 - 0.75 * ((i * 0.6180339887) % 1.0)))) for i, d in enumerate(drafted)]
    return lens, drafted


# ---- what a pass cannot do without ----------------------------------------------------------------


def work(case):
    size = BYTES[case["dtype"]]
    if case["op"] in ("rotary", "qk_norm"):
        heads, tokens = case["heads"] + case["kv_heads"], case["tokens"]
        touched = case["head_size"] if case["op"] == "qk_norm" else case["rot_dim"]
        table = min(tokens, case["max_position"]) * case["rot_dim"] * 4
        weights = 2 * case["head_size"] * size if case["op"] == "qk_norm" else 0
        flops = tokens * heads * (3 * case["rot_dim"] + (4 * case["head_size"] if case["op"] == "qk_norm" else 0))
        return {"bytes": 2 * tokens * heads * touched * size + table + 8 * tokens + weights, "flops": flops}
    if case["op"] == "evict":
        heads, n = case["heads"], case["seqs"]
        kept = min(case["context"], case["budget"])
        moved = kept if case["budget"] < case["context"] else 0
        token = 2 * case["head_size"] * size
        return {"bytes": n * heads * (case["context"] * 4 + moved * (2 * token + 4) + 4 * case["budget"])
                + n * -(-case["context"] // case["block"]) * 4, "flops": n * heads * case["context"]}
    lens, drafted = _lengths(case)
    heads, kv, dim = case["heads"], case["kv_heads"], case["head_size"]
    total = sum(drafted)
    moved = sum(lens) * kv * 2 * dim * size + 2 * total * heads * dim * size
    moved += sum(-(-c // case["block"]) for c in lens) * 4 + 8 * len(lens)
    if not case["chain"]:
        moved += sum(t * t for t in drafted)
    if case["op"] == "accumulate":
        moved += sum(lens) * kv * 8
    return {"bytes": moved, "flops": 4.0 * heads * dim * sum(c * t for c, t in zip(lens, drafted))}


# ---- inputs -----------------------------------------------------------------------------------------


def _angles(case, positions):
    """(angles [len(positions), rot_dim / 2] in 64 bits, amplitude) of the positions, with the case's stretching by 4."""
    dim, factor, scaling = case["rot_dim"], 4.0, case["scaling"]
    pair = torch.arange(0, dim, 2, dtype=torch.float64, device=positions.device)
    base = BASE * factor ** (dim / (dim - 2)) if scaling == "ntk" else BASE
    freq = base ** (-pair / dim)
    amplitude = 1.0
    if scaling == "linear":
        freq = freq / factor
    if scaling == "yarn":
        # frequencies of over 32 turns in the first length stay, those of under one are divided, a ramp between
        length = case["max_position"] / factor
        edge = [dim * math.log(length / (turns * 2 * math.pi)) / (2 * math.log(BASE)) for turns in (32.0, 1.0)]
        low, high = max(math.floor(edge[0]), 0), min(math.ceil(edge[1]), dim - 1)
        ramp = ((pair / 2 - low) / max(high - low, 1e-3)).clamp(0, 1)
        freq = freq * (1 - ramp) + freq / factor * ramp
        amplitude = 0.1 * math.log(factor) + 1.0
    return positions.double()[:, None] * freq[None], amplitude


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 7919 + 17)
    return g


def prepare(case, seed):
    g, dtype = _generator(seed), DTYPES[case["dtype"]]
    state = {"case": case}
    randn = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    if case["op"] in ("rotary", "qk_norm"):
        tokens, dim, q, k = case["tokens"], case["head_size"], case["heads"], case["kv_heads"]
        # query and key as the projection leaves them: columns of one [tokens, (q + 2 k) heads] result
        qkv = randn(tokens, (q + 2 * k) * dim).to(dtype)
        state.update(query=qkv[:, :q * dim], key=qkv[:, q * dim:(q + k) * dim])
        state["positions"] = torch.randint(0, case["max_position"], (tokens,), generator=g, device="cuda")
        angle, amplitude = _angles(case, torch.arange(case["max_position"], device="cuda"))
        state["table"] = torch.cat((angle.cos() * amplitude, angle.sin() * amplitude), dim=1).float()
        if case["op"] == "qk_norm":
            state["weights"] = [(1.0 + 0.2 * randn(dim)).to(dtype) for _ in range(2)]
        return state
    n, block, dim = case["seqs"], case["block"], case["head_size"]
    kv = case["kv_heads"] if "kv_heads" in case else case["heads"]
    lens, drafted = _lengths(case)
    mixed = np.random.RandomState(int(seed) % (1 << 31)).permutation(n)
    lens, drafted = [lens[i] for i in mixed], [drafted[i] for i in mixed]
    held = [-(-c // block) for c in lens]
    order = (torch.randperm(sum(held), generator=g, device="cuda") + 1).int()
    starts = np.concatenate(([0], np.cumsum(held)))
    at = torch.zeros(n, max(held), dtype=torch.int64)
    for i, (s, h) in enumerate(zip(starts, held)):
        at[i, :h] = torch.arange(int(s) + 1, int(s) + h + 1)
    at = at.cuda()
    state["tables"] = torch.cat((order.new_zeros(1), order))[at]
    state["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    blocks, x = sum(held) + 1, 16 // BYTES[case["dtype"]]
    state["key_cache"] = randn(blocks, kv, dim // x, block, x).to(dtype)
    state["value_cache"] = randn(blocks, kv, dim, block).to(dtype)
    if case["op"] in ("accumulate", "evict"):
        # a few positions carry most of the weight; about one in five never had any
        weight = torch.exp(2.0 * randn(blocks, kv, block))
        never = torch.rand(blocks, kv, block, generator=g, device="cuda") < 0.2
        state["weight_cache"] = torch.where(never, torch.zeros_like(weight), weight)
    if case["op"] == "evict":
        state["kept"] = torch.zeros(n, kv, case["budget"], dtype=torch.int32, device="cuda")
        return state
    total, most = sum(drafted), max(drafted)
    state["query"] = (1.5 * randn(total, (case["heads"] + 2 * kv) * dim)).to(dtype)[:, :case["heads"] * dim].unflatten(1, (case["heads"], dim))
    state["starts"] = torch.tensor(np.concatenate(([0], np.cumsum(drafted))), dtype=torch.int32, device="cuda")
    state["most"], state["mask"] = most, None
    if not case["chain"]:
        # trees grown token by token: each hangs on the context or on any token before it
        r = np.random.RandomState(int(seed) % (1 << 31) + 1)
        sees = np.zeros((n, most + 1, most), dtype=bool)  # the row behind the last: the context's end, sees nothing drafted
        for t in range(most):
            parent = r.randint(-1, t, size=n) if t else np.full(n, -1)
            sees[:, t] = sees[np.arange(n), parent]
            sees[:, t, t] = True
        state["mask"] = torch.from_numpy(np.concatenate([sees[i, :t] for i, t in enumerate(drafted)])).cuda()
    state["out"] = torch.zeros(total, case["heads"], dim, dtype=dtype, device="cuda")
    return state


# ---- the operators ----------------------------------------------------------------------------------


def run(state):
    case = state["case"]
    return {"rotary": _rotary, "qk_norm": _rotary, "tree": _attend, "accumulate": _attend, "evict": _evict}[case["op"]](state, case)


def _rotary(state, case):
    query, key, dim = state["query"], state["key"], case["head_size"]
    if own:
        ops = _package().pos_encoding_ops
        if case["op"] == "rotary":
            ops.rotary_embedding(state["positions"], query, key, dim, state["table"], case["interleaved"])
        else:
            ops.qk_norm_rotary_embedding(state["positions"], query, key, dim, state["weights"][0], state["weights"][1],
                                         EPSILON, state["table"], case["interleaved"])
        return query, key
    half = case["rot_dim"] // 2
    row = state["table"][state["positions"]][:, None]
    weights = state.get("weights", (None, None))
    _rotate_plain(query, dim, half, row, weights[0], case["interleaved"])
    _rotate_plain(key, dim, half, row, weights[1], case["interleaved"])
    return query, key


def _rotate_plain(rows, dim, half, row, weight, interleaved):
    v = rows.unflatten(1, (-1, dim)).float()
    if weight is not None:
        v = v * torch.rsqrt(v.square().mean(-1, keepdim=True) + EPSILON) * weight.float()
    cos, sin = row[..., :half], row[..., half:]
    part, rest = v[..., :2 * half], v[..., 2 * half:]
    a, b = (part[..., 0::2], part[..., 1::2]) if interleaved else (part[..., :half], part[..., half:])
    a, b = a * cos - b * sin, b * cos + a * sin
    part = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    rows.copy_(torch.cat((part, rest), -1).flatten(1))


def _attend(state, case):
    scale = case["head_size"] ** -0.5
    out, query, tables, lens, starts = (state[k] for k in ("out", "query", "tables", "lens", "starts"))
    if own:
        ops = _package().attention_ops
        if case["op"] == "tree":
            ops.tree_cached_kv_attention(out, query, state["key_cache"], state["value_cache"], scale, tables, lens, starts,
                                         state["mask"], case["block"], case["context"], state["most"])
            return out
        ops.cached_kv_attention_accumulate(out, query, state["key_cache"], state["value_cache"], state["weight_cache"], scale,
                                           tables, lens, starts, case["block"], case["context"], state["most"])
        return out, state["weight_cache"]
    kv, dim, most = case["kv_heads"], case["head_size"], state["most"]
    n, group, total = tables.shape[0], case["heads"] // kv, query.shape[0]
    at = tables.long()
    k = state["key_cache"][at].permute(0, 2, 1, 4, 3, 5).reshape(n, kv, -1, dim).float()
    v = state["value_cache"][at].permute(0, 2, 1, 4, 3).reshape(n, kv, -1, dim).float()
    places = k.shape[2]
    drafted = (starts[1:] - starts[:-1])[:, None]
    step = torch.arange(most, device=out.device)
    rows = (starts[:-1, None] + step).clamp(max=total - 1).long()
    q = query[rows].float().unflatten(2, (kv, group)).permute(0, 2, 1, 3, 4).reshape(n, kv, most * group, dim)
    place = torch.arange(places, device=out.device)
    drafted_place = place - (lens[:, None] - drafted)  # [n, places], negative in the context
    if state["mask"] is None:
        sees = drafted_place[:, None] <= step[:, None]
    else:
        wide = torch.nn.functional.pad(state["mask"], (0, 1))[rows]
        sees = wide.gather(2, drafted_place.clamp(0, most).long()[:, None].expand(-1, most, -1)) | (drafted_place[:, None] < 0)
    sees = sees & (place < lens[:, None])[:, None] & (step < drafted)[..., None]
    logits = (torch.matmul(q, k.transpose(2, 3)) * scale).unflatten(2, (most, group))
    logits = logits.masked_fill(~sees[:, None, :, None], -math.inf)
    top = logits.amax(-1, keepdim=True).clamp(min=-1e30)
    p = torch.exp(logits - top)
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-30)
    o = torch.matmul(p.flatten(2, 3), v).unflatten(2, (most, group)).permute(0, 2, 1, 3, 4).flatten(2, 3)
    token = torch.arange(total, device=out.device)
    seq = torch.searchsorted(starts[1:], token, right=True)
    out.copy_(o[seq, token - starts[seq]])
    if case["op"] == "tree":
        return out
    weight = state["weight_cache"]
    old = weight[at].transpose(1, 2).flatten(2)
    new = torch.where((drafted_place >= 0)[:, None], torch.zeros_like(old), old) + p.sum((2, 3))
    new = torch.where((place < lens[:, None])[:, None], new, old)
    weight[at] = new.unflatten(2, (-1, case["block"])).transpose(1, 2)
    return out, weight


def _evict(state, case):
    tables, lens, kept = state["tables"], state["lens"], state["kept"]
    keys, values, weight = state["key_cache"], state["value_cache"], state["weight_cache"]
    if own:
        _package().cache_ops.evict_cached_kv(keys, values, weight, tables, lens, kept, case["recent"], case["context"])
        return kept, keys, values, weight
    n, heads, budget, block = tables.shape[0], case["heads"], case["budget"], case["block"]
    at = tables.long()
    w = weight[at].transpose(1, 2).flatten(2)
    place = torch.arange(w.shape[2], device=w.device)
    length = lens[:, None, None]
    w = torch.where(place >= length - case["recent"], math.inf, w)
    w = torch.where(place >= length, -math.inf, w)
    order = torch.sort(w, dim=2, descending=True, stable=True).indices[..., :budget]
    order = torch.nn.functional.pad(order, (0, budget - order.shape[2]))
    slot = torch.arange(budget, device=w.device)
    held = slot < length  # [n, 1, budget]
    order = torch.where(held, order, 1 << 30).sort(2).values
    kept.copy_(torch.where(held, order, -1))
    # a place that keeps nothing is written over with itself
    moves = held & (length > budget)
    to = slot.expand_as(order)
    source = torch.where(moves, order, to)
    last = at.shape[1] - 1
    head = torch.arange(heads, device=w.device)[:, None]
    seq = torch.arange(n, device=w.device)[:, None, None]
    inside = to // block <= last
    from_block = torch.where(inside, at[seq, (source // block).clamp(max=last)], 0)
    to_block = torch.where(inside, at[seq, (to // block).clamp(max=last)], 0)
    a, b = source % block, to % block
    a = torch.where(inside, a, 0)
    b = torch.where(inside, b, 0)
    new_keys, new_values, new_weight = keys[from_block, head, :, a], values[from_block, head, :, a], weight[from_block, head, a]
    keys[to_block, head, :, b] = new_keys
    values[to_block, head, :, b] = new_values
    weight[to_block, head, b] = new_weight
    return kept, keys, values, weight


# ---- the definitions in 64 bits -----------------------------------------------------------------------


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] in ("rotary", "qk_norm"):
        return _exact_rotary(state, case)
    if case["op"] == "evict":
        return _exact_evict(state, case)
    return _exact_attention(state, case)


def _exact_rotary(state, case):
    """Every pair (a, b) as the complex number a + b i, times amplitude e^(i angle)."""
    angle, amplitude = _angles(case, state["positions"])
    turn = torch.polar(torch.full_like(angle, amplitude), angle)
    dim, part, answers = case["head_size"], case["rot_dim"], []
    for k, rows in enumerate((state["query"], state["key"])):
        whole = torch.empty(rows.shape, dtype=torch.float64, device=rows.device)
        for h in range(rows.shape[1] // dim):
            v = rows[:, h * dim:(h + 1) * dim].double()
            if case["op"] == "qk_norm":
                v = v / torch.sqrt((v * v).sum(1, keepdim=True) / dim + EPSILON) * state["weights"][k].double()
            pairs = v[:, :part].reshape(-1, part // 2, 2) if case["interleaved"] else v[:, :part].reshape(-1, 2, part // 2).transpose(1, 2)
            turned = torch.view_as_real(torch.complex(pairs[..., 0].contiguous(), pairs[..., 1].contiguous()) * turn)
            v[:, :part] = (turned if case["interleaved"] else turned.transpose(1, 2)).reshape(-1, part)
            whole[:, h * dim:(h + 1) * dim] = v
        answers.append(whole)
    return tuple(answers)


def _exact_attention(state, case):
    """Sequence by sequence: the positions in a row, the visible ones chosen by an additive mask."""
    block, kv, dim = case["block"], case["kv_heads"], case["head_size"]
    group = case["heads"] // kv
    starts, lens = state["starts"].tolist(), state["lens"].tolist()
    out = torch.zeros(state["out"].shape, dtype=torch.float64, device="cuda")
    weight = state["weight_cache"].double() if case["op"] == "accumulate" else None
    for i, length in enumerate(lens):
        first, rows = starts[i], starts[i + 1] - starts[i]
        place = torch.arange(length, device="cuda")
        blocks, offset = state["tables"][i].long()[place // block], place % block
        bias = torch.zeros(rows, length, dtype=torch.float64, device="cuda")
        if state["mask"] is None:
            bias[:, length - rows:] = torch.triu(torch.full((rows, rows), -math.inf, dtype=torch.float64, device="cuda"), 1)
        else:
            bias[:, length - rows:][~state["mask"][first:first + rows, :rows]] = -math.inf
        for h in range(kv):
            k = state["key_cache"][blocks, h, :, offset].double().reshape(length, dim)
            v = state["value_cache"][blocks, h, :, offset].double()
            q = state["query"][first:first + rows, h * group:(h + 1) * group].double().reshape(-1, dim)
            p = torch.softmax((q @ k.T) / math.sqrt(dim) + bias.repeat_interleave(group, 0), 1)
            out[first:first + rows, h * group:(h + 1) * group] = (p @ v).reshape(rows, group, dim)
            if weight is not None:
                before = weight[blocks, h, offset]
                before[length - rows:] = 0
                weight[blocks, h, offset] = before + p.sum(0)
    return out if weight is None else (out, weight)


def _exact_evict(state, case):
    """Head by head on the host: places ordered by weight, then by place."""
    block, budget, recent = case["block"], case["budget"], case["recent"]
    lens, tables = state["lens"].tolist(), state["tables"].long().cpu()
    weight = state["weight_cache"].cpu().numpy()
    kept = np.full(tuple(state["kept"].shape), -1, dtype=np.int32)
    keys, values, weights = (state[k].clone() for k in ("key_cache", "value_cache", "weight_cache"))
    for i, length in enumerate(lens):
        place = np.arange(length)
        where = tables[i].numpy()[place // block]
        for h in range(case["heads"]):
            if length <= budget:
                kept[i, h, :length] = place
                continue
            old = place[:length - recent]
            w = weight[where[old], h, old % block]
            best = np.lexsort((old, -w))[:budget - recent]
            chosen = np.sort(np.concatenate((old[best], place[length - recent:])))
            kept[i, h] = chosen
            a = torch.from_numpy(where[chosen]).cuda(), torch.from_numpy(chosen % block).cuda()
            b = torch.from_numpy(where[:budget]).cuda(), torch.from_numpy(place[:budget] % block).cuda()
            for new, was in ((keys, state["key_cache"]), (values, state["value_cache"])):
                new[b[0], h, :, b[1]] = was[a[0], h, :, a[1]]
            weights[b[0], h, b[1]] = state["weight_cache"][a[0], h, a[1]]
    return torch.from_numpy(kept).cuda(), keys, values, weights
