"""evict_cached_kv against a plain selection and copy on the host.  Nothing is computed but an order, so everything is equal
to the bit: the positions, the three caches, and every byte that the call has no business with."""
import ctypes
import math

import numpy as np
import pytest
import torch


class Case:

    def __init__(self, lens, budget, recent, heads=2, dim=64, block=16, dtype=torch.float16, weights="spread", seed=0, spare=2):
        gen = torch.Generator().manual_seed(seed)
        self.lens, self.budget, self.recent, self.heads, self.dim, self.block, self.dtype = lens, budget, recent, heads, dim, block, dtype
        x = 16 // torch.empty(0, dtype=dtype).element_size()
        held = [-(-c // block) for c in lens]
        blocks = sum(held) + spare
        order = torch.randperm(blocks, generator=gen).tolist()
        self.tables = torch.full((len(lens), max(held + [1]) + 1), -7, dtype=torch.int32)
        at = 0
        for i, h in enumerate(held):
            self.tables[i, :h] = torch.tensor(order[at:at + h], dtype=torch.int32)
            at += h
        bits = {2: torch.int16, 4: torch.int32}[torch.empty(0, dtype=dtype).element_size()]
        info = torch.iinfo(bits)
        self.kc = torch.randint(info.min, info.max, (blocks, heads, dim // x, block, x), generator=gen).to(bits)  # any bits at all
        self.vc = torch.randint(info.min, info.max, (blocks, heads, dim, block), generator=gen).to(bits)
        if weights == "spread":
            self.wc = torch.exp(3 * torch.randn(blocks, heads, block, generator=gen))
            self.wc[torch.rand(self.wc.shape, generator=gen) < 0.2] = 0.0
        elif weights == "few":       # many equal ones, both zeros, negative ones
            self.wc = torch.tensor([0.0, -0.0, 1.0, 1.0, -2.0, 0.5])[torch.randint(0, 6, (blocks, heads, block), generator=gen)]
        elif weights == "equal":
            self.wc = torch.full((blocks, heads, block), 0.25)
        elif weights == "close":     # neighbours in the last bit
            self.wc = (torch.randint(0, 5, (blocks, heads, block), generator=gen, dtype=torch.int32) + 0x3f800000).view(torch.float32)
        else:                        # specials
            self.wc = torch.tensor([math.nan, -math.nan, math.inf, -math.inf, 0.0, -0.0, 1e-45, -1e-45, 3e38, 1.0])[
                torch.randint(0, 10, (blocks, heads, block), generator=gen)]
        self.lens_t = torch.tensor(lens, dtype=torch.int32)

    def expect(self):
        kept = np.full((len(self.lens), self.heads, self.budget), -1, dtype=np.int32)
        kc, vc, wc = self.kc.clone(), self.vc.clone(), self.wc.view(torch.int32).clone()
        for i, n in enumerate(self.lens):
            for h in range(self.heads):
                place = np.arange(n)
                if n <= self.budget:
                    kept[i, h, :n] = place
                    continue
                block, off = self.tables[i].numpy()[place // self.block], place % self.block
                w = self.wc.numpy()[block, h, off][:n - self.recent].astype(np.float64)
                w = np.where(np.isnan(w), np.inf, w), np.isnan(w)
                order = np.lexsort((place[:n - self.recent], -w[0], ~w[1]))  # NaN, then by value, then by place
                stay = np.sort(np.concatenate((order[:self.budget - self.recent], place[n - self.recent:]))).astype(np.int64)
                kept[i, h] = stay
                to = place[:self.budget]
                src, dst = (block[stay], off[stay]), (block[to], off[to])
                kc[dst[0], h, :, dst[1]] = self.kc[src[0], h, :, src[1]]
                vc[dst[0], h, :, dst[1]] = self.vc[src[0], h, :, src[1]]
                wc[dst[0], h, dst[1]] = self.wc.view(torch.int32)[src[0], h, src[1]]
        return torch.from_numpy(kept), kc, vc, wc

    def device(self):
        return dict(kc=self.kc.cuda().view(self.dtype), vc=self.vc.cuda().view(self.dtype), wc=self.wc.cuda(), tables=self.tables.cuda(),
                    lens=self.lens_t.cuda(), kept=torch.full((len(self.lens), self.heads, self.budget), -99, dtype=torch.int32, device="cuda"))

    def call(self, pkg, d, max_ctx=None):
        pkg.cache_ops.evict_cached_kv(d["kc"], d["vc"], d["wc"], d["tables"], d["lens"], d["kept"], self.recent,
                                      max(self.lens) if max_ctx is None else max_ctx)

    def check(self, d, want=None):
        want = self.expect() if want is None else want
        assert torch.equal(d["kept"].cpu(), want[0])
        assert torch.equal(d["kc"].cpu().view(want[1].dtype), want[1]), "key cache"
        assert torch.equal(d["vc"].cpu().view(want[2].dtype), want[2]), "value cache"
        assert torch.equal(d["wc"].cpu().view(torch.int32), want[3]), "weight cache"


def run(pkg, case):
    d = case.device()
    case.call(pkg, d)
    case.check(d)


@pytest.mark.gpu
@pytest.mark.parametrize("lens,budget,recent", [
    ([1], 1, 0), ([2], 1, 0), ([2], 1, 1), ([0, 5, 3], 4, 2), ([17, 16, 15], 16, 0), ([33, 100, 64], 20, 20),
    ([130, 64, 65, 63], 64, 10), ([257], 3, 1), ([300], 299, 0), ([300], 299, 299), ([1000, 40], 500, 100), ([129], 128, 127),
], ids=str)
@pytest.mark.parametrize("block", [8, 16, 32])
def test_lengths(pkg, lens, budget, recent, block):
    run(pkg, Case(lens, budget, recent, block=block, seed=budget))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("block", [8, 16, 32])
@pytest.mark.parametrize("dim", [64, 80, 96, 128, 8, 200])
def test_head_and_block_sizes(pkg, dim, block, dtype):
    run(pkg, Case([150, 70], 45, 7, heads=3, dim=dim, block=block, dtype=dtype, seed=dim))


@pytest.mark.gpu
@pytest.mark.parametrize("weights", ["few", "equal", "close", "special"])
@pytest.mark.parametrize("recent", [0, 30])
def test_ties_and_special_weights(pkg, weights, recent):
    run(pkg, Case([700, 333, 90], 90, recent, weights=weights))


@pytest.mark.gpu
@pytest.mark.parametrize("n", [8191, 8192, 8193, 16383, 16384, 16385, 20000, 40000])
def test_long_contexts(pkg, n):
    """About as many positions as the selection holds in LDS, and more."""
    run(pkg, Case([n, 5000], n // 3, n // 10, heads=1))
    run(pkg, Case([n], 100, 0, heads=1, weights="few"))


@pytest.mark.gpu
def test_only_the_lightest_at_the_front_go(pkg):
    """What is lost lies at the very end or start of a block, or is one position in the last block."""
    for drop in (0, 15, 16, 47, 48, 62):
        c = Case([64], 63, 1, heads=1)
        c.wc[:] = 1.0
        c.wc[int(c.tables[0, drop // 16]), 0, drop % 16] = 0.0
        run(pkg, c)


@pytest.mark.gpu
def test_contradictory_sequences_are_left_alone(pkg):
    c = Case([100, 90, 80], 30, 5)
    want = c.expect()

    def untouched(d, bad):
        kept, kc, vc, wc = (t.clone() for t in want)
        for i in bad:
            kept[i] = -1
            held = c.tables[i][c.tables[i] >= 0].long()
            kc[held], vc[held], wc[held] = c.kc[held], c.vc[held], c.wc.view(torch.int32)[held]
        c.check(d, (kept, kc, vc, wc))

    d = c.device()
    c.call(pkg, d, max_ctx=95)
    untouched(d, [0])
    for value in (-1, 1 << 20, 2 ** 31 - 1):
        d = c.device()
        d["tables"][1, 3] = value
        c.call(pkg, d)
        untouched(d, [1])
    d = c.device()
    d["lens"][2] = -3
    c.call(pkg, d)
    untouched(d, [2])


@pytest.mark.gpu
def test_twice_and_in_a_graph(pkg):
    """The second call on what the first left; and a captured call on fresh contents each time."""
    c = Case([400, 300], 100, 20, heads=2)
    want = c.expect()
    d = c.device()
    fresh = {k: v.clone() for k, v in d.items()}
    graph = torch.cuda.CUDAGraph()
    c.call(pkg, d)
    c.check(d, want)
    with torch.cuda.graph(graph):
        c.call(pkg, d)
    side = torch.cuda.Stream()
    for _ in range(3):
        for k in d:
            d[k].copy_(fresh[k])
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            graph.replay()
        torch.cuda.current_stream().wait_stream(side)
        torch.randn(1 << 20, device="cuda").sum().item()
        c.check(d, want)
    # on the result, with the new lengths, nothing more happens
    d["lens"].fill_(100)
    c.call(pkg, d)
    c.check(d, (torch.arange(100, dtype=torch.int32).expand(2, 2, 100), *want[1:]))


@pytest.mark.gpu
def test_blocks_past_32_bit_offsets(pkg):
    """The same batch at the end of caches of over 2^32 bytes: the same positions and the same bits."""
    c = Case([300, 200], 70, 10, heads=4, dim=128)
    want = c.expect()
    blocks = c.kc.shape[0]
    n = (1 << 32) // (4 * 128 * 16 * 2) + 64
    d = c.device()
    for k in ("kc", "vc", "wc"):
        t = torch.empty((n,) + tuple(d[k].shape[1:]), dtype=d[k].dtype, device="cuda")
        t[n - blocks:] = d[k]
        d[k] = t
    d["tables"] = torch.where(d["tables"] >= 0, d["tables"] + (n - blocks), d["tables"])
    c.call(pkg, d)
    for k in ("kc", "vc", "wc"):
        d[k] = d[k][n - blocks:].contiguous()
    c.check(d, want)


def test_c_entry_refuses_without_a_gpu(pkg):
    c = pkg._capi
    p = ctypes.c_void_p(4096)

    def call(**kw):
        a = dict(k=p, v=p, w=p, bt=p, cl=p, kept=p, S=2, H=2, D=64, B=16, nb=8, mb=4, mc=64, budget=10, recent=2, dt=c.PA_DTYPE_F16,
                 ws=ctypes.c_void_p(1 << 20), wb=1 << 20)
        a.update(kw)
        return c.lib.pa_evict_cached_kv(a["k"], a["v"], a["w"], a["bt"], a["cl"], a["kept"], a["S"], a["H"], a["D"], a["B"], a["nb"],
                                        a["mb"], a["mc"], a["budget"], a["recent"], a["dt"], a["ws"], a["wb"], None)

    assert call(dt=5) == c.PA_ERR_UNSUPPORTED and "data type" in c.last_error()
    assert call(B=24) == c.PA_ERR_UNSUPPORTED and "block size" in c.last_error()
    assert call(S=-1) == c.PA_ERR_INVALID_ARGUMENT and "negative" in c.last_error()
    assert call(budget=0) == c.PA_ERR_INVALID_ARGUMENT and "budget" in c.last_error()
    assert call(recent=11) == c.PA_ERR_INVALID_ARGUMENT and "num_recent" in c.last_error()
    assert call(recent=-1) == c.PA_ERR_INVALID_ARGUMENT
    assert call(D=66) == c.PA_ERR_INVALID_ARGUMENT and "head size" in c.last_error()
    assert call(w=None) == c.PA_ERR_INVALID_ARGUMENT and "null" in c.last_error()
    assert call(v=ctypes.c_void_p(4100)) == c.PA_ERR_INVALID_ARGUMENT and "aligned" in c.last_error()
    assert call(mc=65) == c.PA_ERR_INVALID_ARGUMENT and "cannot hold" in c.last_error()
    assert call(ws=None) == c.PA_ERR_INVALID_ARGUMENT and "workspace" in c.last_error()
    assert call(wb=10) == c.PA_ERR_INVALID_ARGUMENT and "workspace" in c.last_error()
    assert call(nb=1 << 28) == c.PA_ERR_INVALID_ARGUMENT and "slots" in c.last_error()
    assert call(S=0) == c.PA_OK and call(H=0) == c.PA_OK
    assert c.lib.pa_evict_workspace_bytes(2, 2) > 0 and c.lib.pa_evict_workspace_bytes(0, 2) == 0


def test_module_refuses_cpu_tensors(pkg):
    c = Case([20], 10, 2)
    with pytest.raises(RuntimeError, match="must be on the GPU"):
        pkg.cache_ops.evict_cached_kv(c.kc.view(c.dtype), c.vc.view(c.dtype), c.wc, c.tables, c.lens_t, torch.zeros(1, 2, 10, dtype=torch.int32), 2, 20)


@pytest.mark.gpu
def test_module_refuses_what_does_not_fit(pkg):
    c = Case([20], 10, 2)
    for match, kw in (
        ("one data type", dict(vc=lambda t: t.view(torch.bfloat16))),
        ("contiguous", dict(vc=lambda t: t.transpose(0, 1))),
        ("shape", dict(kc=lambda t: t[:1])),
        ("weight_cache", dict(wc=lambda t: t.double())),
        ("weight_cache", dict(wc=lambda t: t[:, :1])),
        ("int32", dict(kept=lambda t: t.long())),
        ("match", dict(kept=lambda t: t[:, :1].contiguous())),
        ("match", dict(lens=lambda t: t.repeat(2))),
        ("budget", dict(kept=lambda t: t[..., :0].contiguous())),
    ):
        d = c.device()
        for k, f in kw.items():
            d[k] = f(d[k])
        with pytest.raises(RuntimeError, match=match):
            c.call(pkg, d)
    d = c.device()
    with pytest.raises(RuntimeError, match="num_recent"):
        pkg.cache_ops.evict_cached_kv(d["kc"], d["vc"], d["wc"], d["tables"], d["lens"], d["kept"], 11, 20)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("block", [8, 16, 32])
@pytest.mark.parametrize("recent", [0, 777])
def test_contexts_past_the_selection_s_lds_beside_shorter_ones(pkg, dtype, block, recent):
    """Weights that are held on chip and moved at once, and weights that are read again and moved by waves of their own, in
    one launch: three heads, sequences above, at and below the border, and one that keeps what it has."""
    run(pkg, Case([16400, 2500, 16384, 17011, 900], 2000, recent, heads=3, dim=64, block=block, dtype=dtype, seed=block))
    run(pkg, Case([20100, 16385], 16390, recent, heads=3, dim=8, block=block, dtype=dtype, weights="few", seed=recent))
