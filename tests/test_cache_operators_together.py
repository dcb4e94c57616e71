"""The operators around the paged cache as a decoder layer uses them, one after the other: head norms and
rotation, the cache write, attention of a drafted tree, the accepted path kept, single tokens with their
weights accumulated, eviction, and on.  The oracle is dense attention in float64 over each token's own
history, from the very numbers that the cache holds.

Tolerances: the rows that enter an attention are taken as the operators left them (their own tests bound
their roundings), so what is left is attention's: weights rounded to fp16 (2^-11 each, on sum p |v| and
the result), fp32 sums (covered by 2^-14 of the same for contexts of a few hundred), half a step of the
result."""
import math

import numpy as np
import pytest
import torch

H = 2.0 ** -11


def make_cpu_mask_cases():
    return [[-1], [-1, 0, 0, 1, -1], [-1, -1, -1], [-1, 0, 1, 2, 3]]


def test_tree_mask_lists_ancestors(pkg):
    from vllm_amd.worker import tree_mask
    parents = make_cpu_mask_cases()
    mask = tree_mask(parents, device="cpu")
    assert mask.shape == (14, 5) and mask.dtype == torch.bool
    row = 0
    for p in parents:
        for i in range(len(p)):
            line, t = set(), i
            while t >= 0:
                line.add(t)
                t = p[t]
            assert set(mask[row + i].nonzero().flatten().tolist()) == line
        row += len(p)
    with pytest.raises(ValueError, match="earlier"):
        tree_mask([[0]], device="cpu")
    with pytest.raises(ValueError, match="earlier"):
        tree_mask([[-2]], device="cpu")
    assert tree_mask([], device="cpu").shape == (0, 1)


def test_keep_path_refuses_paths_that_do_not_rise(pkg):
    from vllm_amd.worker import keep_path
    with pytest.raises(ValueError, match="rise"):
        keep_path([], [], torch.zeros(1, 1, dtype=torch.int32), [0], [[2, 1]])


def test_keep_path_refuses_what_is_not_in_the_tables(pkg):
    """On the host: an index that is not there would end a program on the GPU."""
    from vllm_amd.worker import keep_path
    keys, values = [torch.zeros(4, 1, 8, 16, 8).half()], [torch.zeros(4, 1, 64, 16).half()]
    tables = torch.zeros(1, 2, dtype=torch.int32)
    for first, paths in (([30], [[0, 2]]), ([-1], [[1]]), ([0, 0], [[0], [1]]), ([], [[1]])):
        with pytest.raises(ValueError, match="block table"):
            keep_path(keys, values, tables, first, paths)


@pytest.mark.parametrize("scaling", ["none", "linear", "ntk", "yarn"])
def test_cos_sin_cache_against_its_definition(pkg, scaling):
    """Angles by hand in float64; a float32 table rounds cos and sin once (2^-24 of an amplitude below 1.2)."""
    from vllm_amd.layers import rotary_cos_sin_cache
    dim, positions, factor, base = 64, 4096, 4.0, 10000.0
    table = rotary_cos_sin_cache(dim, positions, base, scaling, factor).double().numpy()
    at = np.array([0, 1, 77, 1023, 4095])
    for i in (0, 1, 9, 13, 17, 31):
        f = base ** (-2 * i / dim)
        amplitude = 1.0
        if scaling == "linear":
            f /= factor
        if scaling == "ntk":
            f = (base * factor ** (dim / (dim - 2))) ** (-2 * i / dim)
        if scaling == "yarn":
            low = max(math.floor(dim * math.log(1024 / (32 * 2 * math.pi)) / (2 * math.log(base))), 0)
            high = min(math.ceil(dim * math.log(1024 / (2 * math.pi)) / (2 * math.log(base))), dim - 1)
            r = min(max((i - low) / (high - low), 0.0), 1.0)
            f = f * (1 - r) + f / factor * r
            amplitude = 0.1 * math.log(factor) + 1.0
        # the angle itself may differ in its last bits: 4095 * 2^-50 at most
        assert np.abs(table[at, i] - amplitude * np.cos(at * f)).max() <= 1.2 * 2.0 ** -24 + 1e-11
        assert np.abs(table[at, dim // 2 + i] - amplitude * np.sin(at * f)).max() <= 1.2 * 2.0 ** -24 + 1e-11
    if scaling == "ntk":  # the slowest pair is stretched by the factor, the fastest not at all
        assert abs(np.arctan2(table[1, dim - 1], table[1, dim // 2 - 1]) * factor / base ** (-(dim - 2) / dim) - 1) < 1e-3
        assert abs(table[1, 0] - math.cos(1.0)) < 1e-6
    with pytest.raises(ValueError, match="even"):
        rotary_cos_sin_cache(63, 8)
    with pytest.raises(ValueError, match="not supported"):
        rotary_cos_sin_cache(64, 8, scaling="other")
    with pytest.raises(ValueError, match="factor"):
        rotary_cos_sin_cache(64, 8, scaling="linear", factor=0.5)


def test_rotary_module_keeps_its_table(pkg):
    from vllm_amd.layers import RotaryEmbedding
    m = RotaryEmbedding(64, 32, 128, qk_norm=True).half()
    assert m.cos_sin_cache.dtype == torch.float32 and m.query_weight.dtype == torch.float16
    assert m.to(torch.bfloat16).cos_sin_cache.dtype == torch.float32


class Engine:
    """Two sequences in a paged cache, and their history as the cache holds it."""

    def __init__(self, pkg, seed, heads=4, kv=2, dim=64, block=16, interleaved=True):
        from vllm_amd.layers import RotaryEmbedding
        self.pkg, self.heads, self.kv, self.dim, self.block = pkg, heads, kv, dim, block
        self.gen = torch.Generator(device="cuda").manual_seed(seed)
        self.rotary = RotaryEmbedding(dim, dim // 2, 4096, interleaved=interleaved, qk_norm=True).half().cuda()
        blocks = 64
        self.kc = torch.full((blocks, kv, dim // 8, block, 8), math.nan, dtype=torch.float16, device="cuda")
        self.vc = torch.full((blocks, kv, dim, block), math.nan, dtype=torch.float16, device="cuda")
        self.wc = torch.full((blocks, kv, block), math.nan, device="cuda")
        free = torch.randperm(blocks, generator=torch.Generator().manual_seed(seed)).int()
        self.tables = free.view(2, -1).cuda()
        self.lens = [0, 0]                  # positions in the cache
        self.true = [0, 0]                  # positions of the text
        self.keys, self.values = [[], []], [[], []]   # per sequence [position][kv head, dim], float64
        self.weights = [np.zeros((kv, 0)), np.zeros((kv, 0))]

    def slots(self, s, positions):
        at = torch.as_tensor(positions, device="cuda")
        return (self.tables[s, at // self.block].long() * self.block + at % self.block).int()

    def project(self, positions):
        """A fused projection's rows, normed and rotated in place: query, key, value views."""
        n, width = len(positions), (self.heads + 2 * self.kv) * self.dim
        qkv = torch.randn(n, width, generator=self.gen, device="cuda").half()
        q, k, v = qkv.split([self.heads * self.dim, self.kv * self.dim, self.kv * self.dim], 1)
        self.rotary(torch.tensor(positions, device="cuda"), q, k)
        return q.unflatten(1, (self.heads, self.dim)), k.unflatten(1, (self.kv, self.dim)), v.unflatten(1, (self.kv, self.dim))

    def dense(self, q, keys, values):
        """q [heads, dim], keys / values: per kv head [n, dim] -> [heads, dim], bound"""
        out, bound = np.zeros((self.heads, self.dim)), np.zeros((self.heads, self.dim))
        ps = []
        for h in range(self.heads):
            g = h // (self.heads // self.kv)
            s = keys[g] @ q[h] * self.dim ** -0.5
            p = np.exp(s - s.max())
            p /= p.sum()
            out[h] = p @ values[g]
            bound[h] = (H + 2.0 ** -14) * (p @ np.abs(values[g]) + np.abs(out[h]))
            ps.append(p)
        return out, bound + H * (np.abs(out) + bound) + 2.0 ** -25, ps

    def history(self, s):
        return ([np.stack([k[g] for k in self.keys[s]]) for g in range(self.kv)],
                [np.stack([v[g] for v in self.values[s]]) for g in range(self.kv)])

    def check(self, got, want, bound, what):
        g = got.double().cpu().numpy()
        assert (np.abs(g - want) <= bound).all(), f"{what}: {np.nanmax(np.abs(g - want) / bound)} of the bound"

    def draft(self, parents):
        """Writes drafted trees behind the contexts and attends to them; returns the rows per sequence."""
        from vllm_amd.worker import tree_mask
        starts = np.concatenate(([0], np.cumsum([len(p) for p in parents])))
        positions, slots = [], []
        for s, tree in enumerate(parents):
            depth = []
            for p in tree:
                depth.append(0 if p < 0 else depth[p] + 1)
            positions += [self.true[s] + d for d in depth]
            slots.append(self.slots(s, [self.lens[s] + i for i in range(len(tree))]))
        q, k, v = self.project(positions)
        self.pkg.cache_ops.reshape_and_cache(k, v, self.kc, self.vc, torch.cat(slots))
        lens = [n + len(t) for n, t in zip(self.lens, parents)]
        out = torch.empty(len(positions), self.heads, self.dim, dtype=torch.float16, device="cuda")
        self.pkg.attention_ops.tree_cached_kv_attention(
            out, q, self.kc, self.vc, self.dim ** -0.5, self.tables, torch.tensor(lens, dtype=torch.int32, device="cuda"),
            torch.tensor(starts, dtype=torch.int32, device="cuda"), tree_mask(parents), self.block, max(lens), max(len(t) for t in parents))
        qn, kn, vn = (t.double().cpu().numpy() for t in (q, k, v))
        for s, tree in enumerate(parents):
            hk, hv = self.history(s)
            for i in range(len(tree)):
                line, t = [], i
                while t >= 0:
                    line.append(t)
                    t = tree[t]
                rows = [starts[s] + t for t in line]
                want, bound, _ = self.dense(qn[starts[s] + i], [np.concatenate((hk[g], kn[rows, g])) for g in range(self.kv)],
                                            [np.concatenate((hv[g], vn[rows, g])) for g in range(self.kv)])
                self.check(out[starts[s] + i], want, bound, f"drafted token {i} of sequence {s}")
        return kn, vn, starts

    def accept(self, paths, kn, vn, starts):
        from vllm_amd.worker import keep_path
        keep_path([self.kc], [self.vc], self.tables, self.lens, paths)
        for s, path in enumerate(paths):
            for t in path:
                self.keys[s].append(kn[starts[s] + t])
                self.values[s].append(vn[starts[s] + t])
            self.lens[s] += len(path)
            self.true[s] += len(path)

    def step(self, tokens=1):
        """`tokens` new tokens of every sequence (a chain), their weights accumulated; checked against the history."""
        positions = [p for s in range(2) for p in range(self.true[s], self.true[s] + tokens)]
        q, k, v = self.project(positions)
        slots = torch.cat([self.slots(s, range(self.lens[s], self.lens[s] + tokens)) for s in range(2)])
        self.pkg.cache_ops.reshape_and_cache(k, v, self.kc, self.vc, slots)
        kn, vn, qn = (t.double().cpu().numpy() for t in (k, v, q))
        lens = [n + tokens for n in self.lens]
        out = torch.empty(2 * tokens, self.heads, self.dim, dtype=torch.float16, device="cuda")
        lens_t = torch.tensor(lens, dtype=torch.int32, device="cuda")
        self.pkg.attention_ops.cached_kv_attention_accumulate(
            out, q, self.kc, self.vc, self.wc, self.dim ** -0.5, self.tables, lens_t,
            torch.tensor([0, tokens, 2 * tokens], dtype=torch.int32, device="cuda"), self.block, max(lens), tokens)
        if tokens == 1 and self.heads == self.kv:  # the same rows through the decode operator
            other = torch.empty_like(out)
            self.pkg.attention_ops.single_query_cached_kv_attention(other, q, self.kc, self.vc, self.dim ** -0.5, self.tables,
                                                                    lens_t, self.block, max(lens))
        for s in range(2):
            self.weights[s] = np.concatenate((self.weights[s], np.zeros((self.kv, tokens))), 1)
            for i in range(tokens):
                self.keys[s].append(kn[s * tokens + i])
                self.values[s].append(vn[s * tokens + i])
                hk, hv = self.history(s)
                want, bound, ps = self.dense(qn[s * tokens + i], hk, hv)
                self.check(out[s * tokens + i], want, bound, f"token {i} of sequence {s}")
                if tokens == 1 and self.heads == self.kv:
                    self.check(other[s], want, bound + 2e-6 * np.abs(want), f"decode, sequence {s}")
                for h, p in enumerate(ps):
                    self.weights[s][h // (self.heads // self.kv), :len(p)] += p
        self.lens = lens
        self.true = [n + tokens for n in self.true]

    def check_weights(self):
        for s in range(2):
            at = torch.arange(self.lens[s], device="cuda")
            got = self.wc[self.tables[s, at // self.block].long(), :, at % self.block].double().cpu().numpy().T
            # fp32 logits and sums: 2^-14 of a weight covers contexts of a few hundred (see above)
            assert (np.abs(got - self.weights[s]) <= 2.0 ** -14 * self.weights[s] + 1e-9).all()


def evict_and_rebuild(e, budget, recent):
    kept = torch.empty(2, e.kv, budget, dtype=torch.int32, device="cuda")
    e.pkg.cache_ops.evict_cached_kv(e.kc, e.vc, e.wc, e.tables, torch.tensor(e.lens, dtype=torch.int32, device="cuda"), kept, recent, max(e.lens))
    kept = kept.cpu().numpy()
    for s in range(2):
        n = e.lens[s]
        if n <= budget:
            assert (kept[s] == np.where(np.arange(budget) < n, np.arange(budget), -1)).all()
            continue
        for g in range(e.kv):  # the heaviest and the latest, up to weights that fp32 cannot tell apart
            stay = kept[s, g]
            assert (np.diff(stay) > 0).all() and set(range(n - recent, n)) <= set(stay.tolist())
            old = e.weights[s][g, :n - recent]
            gone = np.setdiff1d(np.arange(n - recent), stay)
            assert old[gone].max() <= old[stay[stay < n - recent]].min() * (1 + 2.0 ** -12)
        e.keys[s] = [np.stack([e.keys[s][kept[s, g, j]][g] for g in range(e.kv)]) for j in range(budget)]
        e.values[s] = [np.stack([e.values[s][kept[s, g, j]][g] for g in range(e.kv)]) for j in range(budget)]
        e.weights[s] = np.stack([e.weights[s][g, kept[s, g]] for g in range(e.kv)])
        e.lens[s] = budget


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv,interleaved", [(4, 2, True), (3, 3, False), (8, 1, True)])
def test_drafts_accepted_then_weights_then_eviction(pkg, heads, kv, interleaved):
    e = Engine(pkg, seed=heads, heads=heads, kv=kv, interleaved=interleaved)
    e.step(40)                                          # the prompt, as a chain
    trees = [[-1, 0, 0, 1, -1, 4, 2], [-1, -1, 1]]
    e.accept([[0, 2, 6], [1, 2]], *e.draft(trees))
    e.weights = [np.concatenate((w, np.zeros((kv, n - w.shape[1]))), 1) for w, n in zip(e.weights, e.lens)]
    for s in range(2):                                  # accepted tokens were never weighed: theirs start from 0
        at = torch.arange(40, e.lens[s], device="cuda")
        e.wc[e.tables[s, at // e.block].long(), :, at % e.block] = 0
    e.accept([[0, 1], [0]], *e.draft([[-1, 0], [-1]]))
    e.weights = [np.concatenate((w, np.zeros((kv, n - w.shape[1]))), 1) for w, n in zip(e.weights, e.lens)]
    for s in range(2):
        at = torch.arange(40, e.lens[s], device="cuda")
        e.wc[e.tables[s, at // e.block].long(), :, at % e.block] = 0
    for _ in range(6):
        e.step()
    e.check_weights()
    evict_and_rebuild(e, 30, 8)
    e.check_weights()
    for _ in range(20):                                 # past the end of a block, and over the budget again
        e.step()
    e.check_weights()
    evict_and_rebuild(e, 33, 0)
    e.step(3)
    e.check_weights()
    e.accept([[1], [0]], *e.draft([[-1, -1], [-1, 0]]))


class HostCacheOps:
    """gather_cached_kv and reshape_and_cache on host tensors."""

    @staticmethod
    def gather_cached_kv(key, value, kc, vc, slots):
        block = vc.shape[3]
        b, o = slots.long() // block, slots.long() % block
        key.copy_(kc[b, :, :, o].flatten(2))
        value.copy_(vc[b, :, :, o])

    @staticmethod
    def reshape_and_cache(key, value, kc, vc, slots):
        block = vc.shape[3]
        b, o = slots.long() // block, slots.long() % block
        kc[b, :, :, o] = key.unflatten(2, (kc.shape[2], kc.shape[4]))
        vc[b, :, :, o] = value


@pytest.mark.parametrize("paths", [[[0, 2, 6], [1, 2]], [[0, 1], []], [[], [3]], [[], []]], ids=str)
def test_keep_path_starts_accepted_weights_from_zero(pkg, paths):
    """Two layers: keys and values of the path move, its weights are 0 whatever their blocks held before, all others stay."""
    from vllm_amd.worker import keep_path
    gen = torch.Generator().manual_seed(3)
    kv, dim, block, first = 2, 8, 4, [6, 3]
    tables = torch.randperm(10, generator=gen).int().view(2, 5)
    kcs = [torch.randn(10, kv, dim // 4, block, 4, generator=gen) for _ in range(2)]
    vcs = [torch.randn(10, kv, dim, block, generator=gen) for _ in range(2)]
    wcs = [torch.rand(10, kv, block, generator=gen) for _ in range(2)]
    for s in range(2):
        for pos in range(first[s], 20):
            for w in wcs:
                w[int(tables[s, pos // block]), :, pos % block] = math.nan
    want = [w.clone() for w in wcs]
    old = [v.clone() for v in vcs]
    for s, path in enumerate(paths):
        for i in range(len(path)):
            for w in want:
                w[int(tables[s, (first[s] + i) // block]), :, (first[s] + i) % block] = 0.0
    keep_path(kcs, vcs, tables, first, paths, HostCacheOps, weight_caches=wcs)
    for w, e in zip(wcs, want):
        assert torch.equal(w.view(torch.int32), e.view(torch.int32))
    for v, o in zip(vcs, old):
        for s, path in enumerate(paths):
            for i, t in enumerate(path):
                to, src = first[s] + i, first[s] + t
                assert torch.equal(v[int(tables[s, to // block]), :, :, to % block], o[int(tables[s, src // block]), :, :, src % block])


def test_keep_path_refuses_weights_that_do_not_fit(pkg):
    from vllm_amd.worker import keep_path
    keys, values = [torch.zeros(4, 1, 8, 16, 8).half()], [torch.zeros(4, 1, 64, 16).half()]
    tables = torch.zeros(1, 2, dtype=torch.int32)
    for weights in ([], [torch.zeros(4, 1, 16)] * 2, [torch.zeros(4, 2, 16)], [torch.zeros(4, 1, 8)], [torch.zeros(3, 1, 16)]):
        with pytest.raises(ValueError, match="weight"):
            keep_path(keys, values, tables, [0], [[0]], HostCacheOps, weight_caches=weights)
    # in place already, but past the table: nothing moves, weights would be written
    with pytest.raises(ValueError, match="block table"):
        keep_path(keys, values, tables, [31], [[0, 1]], HostCacheOps, weight_caches=[torch.zeros(4, 1, 16)])
    with pytest.raises(ValueError, match="block table"):
        keep_path(keys, values, tables, [-1], [[0]], HostCacheOps, weight_caches=[torch.zeros(4, 1, 16)])


@pytest.mark.gpu
def test_accepted_drafts_do_not_outlive_heavier_positions(pkg):
    """The weight cache holds NaN wherever nothing was weighed, and eviction keeps NaN before all else: the entries of
    accepted tokens have to start from 0 with the path."""
    from vllm_amd.worker import keep_path
    e = Engine(pkg, seed=11)
    e.step(40)
    paths = [[0, 2, 6], [0, 1]]
    kn, vn, starts = e.draft([[-1, 0, 0, 1, -1, 4, 2], [-1, 0, 0]])
    keep_path([e.kc], [e.vc], e.tables, e.lens, paths, weight_caches=[e.wc])
    for s, path in enumerate(paths):
        for t in path:
            e.keys[s].append(kn[starts[s] + t])
            e.values[s].append(vn[starts[s] + t])
        e.lens[s] += len(path)
        e.true[s] += len(path)
    e.weights = [np.concatenate((w, np.zeros((e.kv, n - w.shape[1]))), 1) for w, n in zip(e.weights, e.lens)]
    e.check_weights()
    for _ in range(3):
        e.step()
    e.check_weights()
    evict_and_rebuild(e, 30, 2)
    e.step(2)
    e.check_weights()


def test_rotary_module_keeps_its_table_where_weights_are_emptied(pkg):
    """A model that is made without memory first, then given empty memory and its checkpoint: the table is in none."""
    from vllm_amd.layers import RotaryEmbedding, rotary_cos_sin_cache
    want = rotary_cos_sin_cache(32, 128)
    with torch.device("meta"):
        m = RotaryEmbedding(64, 32, 128, qk_norm=True)
    assert m.query_weight.is_meta
    m = m.to_empty(device="cpu")
    assert not m.query_weight.is_meta and "cos_sin_cache" not in m.state_dict()
    assert torch.equal(m.cos_sin_cache, want)
    assert torch.equal(RotaryEmbedding(64, 32, 128).to_empty(device="cpu").double().cos_sin_cache, want)
    assert torch.equal(RotaryEmbedding(64, 32, 128, qk_norm=True).to("meta").to_empty(device="cpu").cos_sin_cache, want)
