"""tree_cached_kv_attention and cached_kv_attention_accumulate against a float64 evaluation of the definition.

The oracle takes, row by row, only the positions that the row sees: what lies elsewhere may be anything.

Tolerances, counted from the arithmetic (u = 2^-23, which also covers a product instruction that
truncates; h = half a step of the type, 0 where weights stay fp32):
  logits      an fp32 sum of head_size products and two roundings behind it:
              e = (head_size + 4) u |scale| sum |q k| + 4 u |s|, and 4 u of exp2; a weight's relative
              error is at most E = 2 (e + 4 u) for the largest e of the row
  weights     rounded to the type, h each, and added up as rounded (fp16 below 2^-20 of the row's
              largest loses bits: 2^-31 of it at most)
  sums        one product instruction per 32 (fp32: 4) positions after another, then waves and partitions:
              S = (n / 32 or 4 + 64 + 32) u
  result      |out - want| <= (h + E + S) (sum p |v| + |want|) + n 2^-31 max |v|, then half a step
  weight      |w - want| <= (E + S) want + u |old + want|
"""
import ctypes
import math

import numpy as np
import pytest
import torch

HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
U = 2.0 ** -23


class Case:
    """One batch: caches filled with garbage (NaN) wherever no context lies, tables of scattered blocks."""

    def __init__(self, lens, drafted, heads=4, kv=2, dim=64, block=16, dtype=torch.float16, scale=None, masked=True, seed=0,
                 pad_rows=3, q_pad=8, q_shift=0, extra_cols=2, v_mean=0.0):
        gen = torch.Generator().manual_seed(seed)
        self.lens, self.drafted, self.heads, self.kv, self.dim, self.block, self.dtype = lens, drafted, heads, kv, dim, block, dtype
        self.scale = dim ** -0.5 if scale is None else scale
        n, x = len(lens), 16 // torch.empty(0, dtype=dtype).element_size()
        held = [-(-c // block) for c in lens]
        width = max(held + [1]) + extra_cols
        blocks = sum(held) + 2
        order = torch.randperm(blocks, generator=gen).tolist()
        self.tables = torch.full((n, width), 2 ** 30, dtype=torch.int32)  # entries past the context are never read
        self.keys, self.values = [], []
        kc = torch.full((blocks, kv, dim // x, block, x), math.nan).to(dtype)
        vc = torch.full((blocks, kv, dim, block), math.nan).to(dtype)
        at = 0
        for i, c in enumerate(lens):
            k = torch.randn(c, kv, dim, generator=gen).to(dtype)
            v = (torch.randn(c, kv, dim, generator=gen) + v_mean).to(dtype)
            self.keys.append(k)
            self.values.append(v)
            for b in range(held[i]):
                phys = order[at + b]
                self.tables[i, b] = phys
                part = slice(b * block, min(c, (b + 1) * block))
                m = part.stop - part.start
                kc[phys, :, :, :m] = k[part].view(m, kv, dim // x, x).permute(1, 2, 0, 3)
                vc[phys, :, :, :m] = v[part].permute(1, 2, 0)
            at += held[i]
        total = sum(drafted)
        self.starts = torch.tensor(np.concatenate(([0], np.cumsum(drafted))), dtype=torch.int32)
        stride = heads * dim + q_pad
        self.q_store = (1.5 * torch.randn((total + pad_rows) * stride + q_shift, generator=gen)).to(dtype)
        self.q_view = ((total + pad_rows, heads, dim), (stride, dim, 1), q_shift)
        self.max_query = max(drafted + [1])
        self.mask = None
        if masked:
            self.mask = torch.rand(total + pad_rows, self.max_query + 1, generator=gen) < 0.5
        self.kc, self.vc = kc, vc
        self.lens_t = torch.tensor(lens, dtype=torch.int32)

    @property
    def query(self):
        return self.q_store.as_strided(*self.q_view)

    def sees(self, i, t):
        c, n = self.lens[i], self.drafted[i]
        s = np.ones(c, dtype=bool)
        s[c - n:] = np.arange(n) <= t if self.mask is None else self.mask[int(self.starts[i]) + t, :n].numpy()
        return s

    def oracle(self):
        """(out, bound before the last rounding, weights [seq][kv, positions], their bounds)"""
        rows = sum(self.drafted)
        out, bound = np.zeros((rows, self.heads, self.dim)), np.zeros((rows, self.heads, self.dim))
        h = 0.0 if self.dtype == torch.float32 else HALF[self.dtype]
        per = 4 if self.dtype == torch.float32 else 32
        q = self.query.double().numpy()
        weights, wbound = [], []
        for i, c in enumerate(self.lens):
            w, wb = np.zeros((self.kv, c)), np.zeros((self.kv, c))
            k, v = self.keys[i].double().numpy(), self.values[i].double().numpy()
            for t in range(self.drafted[i]):
                r = int(self.starts[i]) + t
                see = self.sees(i, t)
                if not see.any():
                    continue
                for hd in range(self.heads):
                    g = hd // (self.heads // self.kv)
                    kk, vv = k[see, g], v[see, g]
                    s = self.scale * (kk @ q[r, hd])
                    e = (self.dim + 4) * U * abs(self.scale) * (np.abs(kk) @ np.abs(q[r, hd])) + 4 * U * np.abs(s)
                    rel = 2 * (e.max() + 4 * U) + (c / per + 96) * U
                    p = np.exp(s - s.max())
                    p /= p.sum()
                    out[r, hd] = p @ vv
                    bound[r, hd] = (h + rel) * (p @ np.abs(vv) + np.abs(out[r, hd])) + c * 2.0 ** -31 * np.abs(vv).max()
                    w[g, see] += p
                    wb[g, see] += rel * p
            weights.append(w)
            wbound.append(wb)
        return out, bound, weights, wbound

    def device(self):
        d = {k: getattr(self, k).cuda() for k in ("kc", "vc", "tables", "lens_t", "starts")}
        d["query"] = self.q_store.cuda().as_strided(*self.q_view)
        d["mask"] = None if self.mask is None else self.mask.cuda()
        d["out"] = torch.full(self.q_view[0], 7.0, dtype=self.dtype, device="cuda")
        return d

    def attend(self, pkg, d, max_ctx=None, max_query=None):
        pkg.attention_ops.tree_cached_kv_attention(
            d["out"], d["query"], d["kc"], d["vc"], self.scale, d["tables"], d["lens_t"], d["starts"], d["mask"], self.block,
            max(self.lens + [1]) if max_ctx is None else max_ctx, self.max_query if max_query is None else max_query)
        return d["out"]

    def accumulate(self, pkg, d, max_ctx=None):
        pkg.attention_ops.cached_kv_attention_accumulate(
            d["out"], d["query"], d["kc"], d["vc"], d["weights"], self.scale, d["tables"], d["lens_t"], d["starts"], self.block,
            max(self.lens + [1]) if max_ctx is None else max_ctx, self.max_query)
        return d["out"]

    def check_out(self, got, oracle, what=""):
        rows = sum(self.drafted)
        want, bound = oracle[0], oracle[1]
        g = got[:rows].double().cpu().numpy()
        limit = bound + HALF[self.dtype] * (np.abs(want) + bound) + 2.0 ** -25
        ok = np.abs(g - want) <= limit
        assert ok.all(), f"{what}: {(~ok).sum()} of {ok.size} elements off, first at {np.argwhere(~ok)[0]}, worst {np.nanmax(np.abs(g - want) / limit)} of the bound"
        assert bool((got[rows:] == 7.0).all()), "rows behind the last sequence were written"


def run(pkg, case):
    d = case.device()
    case.check_out(case.attend(pkg, d), case.oracle())


# lens (drafted included), drafted, heads, kv heads
SHAPES = [
    ([1], [1], 1, 1),                         # the smallest there is
    ([40, 7, 1, 33], [1, 1, 1, 1], 4, 4),     # single tokens
    ([70, 5], [5, 5], 4, 1),                  # 20 rows; a context of drafted tokens only
    ([100, 31, 32, 64], [16, 3, 0, 1], 2, 1),  # a sequence without queries
    ([65, 300, 129], [13, 26, 8], 6, 2),      # 78 rows
    ([90, 200], [64, 33], 5, 5),              # 64 rows
    ([150, 260], [50, 7], 8, 1),              # 400 rows: several workgroups
    ([20, 129], [17, 1], 3, 1),
    ([0, 17, 0], [0, 2, 0], 2, 2),
    ([500, 333], [300, 333], 4, 2),           # the next stretch of a prompt, and a whole one
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("masked", [True, False])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"{s[2]}over{s[3]}_" + "_".join(f"{t}of{c}" for c, t in zip(s[0], s[1])))
def test_shapes(pkg, shape, masked, dtype):
    lens, drafted, heads, kv = shape
    run(pkg, Case(lens, drafted, heads, kv, dtype=dtype, masked=masked, seed=len(lens) + heads))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("block", [8, 16, 32])
@pytest.mark.parametrize("dim", [64, 80, 96, 128])
@pytest.mark.parametrize("rows", [3, 9, 20, 40])  # times two query heads: each form of the launch
def test_head_and_block_sizes(pkg, dim, block, dtype, rows):
    run(pkg, Case([rows + 77, rows + 2], [rows, rows - 1], 4, 2, dim=dim, block=block, dtype=dtype, seed=dim + block))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dim", [64, 128])
def test_long_contexts_in_partitions(pkg, dim, dtype):
    """One sequence of many partitions beside ones that fill few or a part of one."""
    run(pkg, Case([9001, 255, 257, 3], [5, 2, 5, 3], 2, 1, dim=dim, dtype=dtype, v_mean=0.5))


@pytest.mark.gpu
@pytest.mark.parametrize("seqs,kv,most", [(40, 8, 3), (37, 8, 20), (256, 2, 3), (257, 1, 2)])
def test_batches_of_more_workgroups_than_the_chip(pkg, seqs, kv, most):
    """Sequences of all lengths, equal and empty ones among them: up to 256 of them are taken by their length."""
    drafted = [i * 7 % (most + 1) for i in range(seqs)]
    lens = [max(t, i * 37 % 90 if i % 5 else 41) for i, t in enumerate(drafted)]
    for masked in (True, False):
        c = Case(lens, drafted, 2 * kv, kv, masked=masked, seed=seqs)
        oracle = c.oracle()
        d = c.device()
        c.check_out(c.attend(pkg, d), oracle)
    d = c.device()
    d["weights"] = torch.zeros(c.kc.shape[0], kv, 16, device="cuda")
    c.check_out(c.accumulate(pkg, d), oracle)
    got = d["weights"].double().cpu().numpy()
    for i, n in enumerate(lens):
        for pos in range(n if drafted[i] else 0):
            w = got[int(c.tables[i, pos // 16]), :, pos % 16]
            assert (np.abs(w - oracle[2][i][:, pos]) <= oracle[3][i][:, pos] + U * oracle[2][i][:, pos] + 1e-30).all()
    # one that contradicts itself in their midst: its own rows only
    d["lens_t"][20] = 10 ** 6
    out = c.accumulate(pkg, d)
    wrong = torch.zeros(sum(drafted), dtype=torch.bool)
    wrong[int(c.starts[20]):int(c.starts[21])] = True
    assert torch.equal(torch.isnan(out[:sum(drafted)]).flatten(1).all(1).cpu(), wrong)
    assert torch.equal(torch.isnan(out[:sum(drafted)]).flatten(1).any(1).cpu(), wrong)


@pytest.mark.gpu
@pytest.mark.parametrize("parts_ctx", [16384, 12289])
def test_more_partitions_than_half_a_wave(pkg, parts_ctx):
    run(pkg, Case([parts_ctx], [1], 1, 1, dim=64))


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [0.0, -0.2, 3.0])
def test_scales(pkg, scale):
    """0: all weights alike; negative; one so large that the softmax picks single positions."""
    for masked in (True, False):
        run(pkg, Case([70, 40], [6, 40], 4, 2, scale=scale, masked=masked, dtype=torch.bfloat16))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("pad,shift", [(0, 0), (3, 0), (8, 1), (5, 3)])
def test_query_strides_and_alignments(pkg, dtype, pad, shift):
    run(pkg, Case([50, 20], [6, 9], 4, 2, dim=80, dtype=dtype, q_pad=pad, q_shift=shift))


@pytest.mark.gpu
def test_rising_logits(pkg):
    """Keys that grow along the context: the running maximum is raised again and again, far past its slack."""
    for dtype in (torch.float16, torch.bfloat16, torch.float32):
        c = Case([700], [4], 2, 1, dtype=dtype, masked=False)
        for b in range(-(-700 // 16)):
            c.kc[int(c.tables[0, b])] *= 1.0 + b
        c.keys[0] = torch.cat([(c.keys[0][16 * b:16 * b + 16] * (1.0 + b)) for b in range(-(-700 // 16))])
        run(pkg, c)


@pytest.mark.gpu
@pytest.mark.parametrize("masked", [True, False])
def test_a_long_chain_over_a_long_context(pkg, masked):
    """Many rows and many partitions: positions behind a workgroup's last row are left out of a chain."""
    run(pkg, Case([2100], [700], 2, 2, masked=masked, dtype=torch.bfloat16))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("drafted", [[3], [40]])
@pytest.mark.parametrize("scale", [1e9, -1e9])
def test_logits_far_beyond_the_slack(pkg, dtype, drafted, scale):
    """Logits of 10^10, whose last bit is worth hundreds: the softmax picks one position where the gap to the next is
    more than the logits' own error (e of the file's head), and is finite everywhere."""
    c = Case([300], drafted, 4, 2, dtype=dtype, masked=False, scale=scale)
    out = c.attend(pkg, c.device())[:drafted[0]].double().cpu().numpy()
    assert np.isfinite(out).all()
    q, sure = c.query.double().numpy(), 0
    for t in range(drafted[0]):
        n = 300 - drafted[0] + t + 1
        for h in range(4):
            k, v = c.keys[0][:n, h // 2].double().numpy(), c.values[0][:n, h // 2].double().numpy()
            s = scale * (k @ q[t, h])
            e = ((c.dim + 4) * U * abs(scale) * (np.abs(k) @ np.abs(q[t, h])) + 4 * U * np.abs(s)).max()
            order = np.argsort(-s)
            if s[order[0]] - s[order[1]] > 2 * e + 100:
                sure += 1
                assert (np.abs(out[t, h] - v[order[0]]) <= 4 * HALF[dtype] * np.abs(v[order[0]]) + 2.0 ** -24).all()
    assert sure > 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_logits_at_the_type_s_end(pkg, dtype):
    """All logits near -10^36: no row passes for one that sees nothing."""
    c = Case([40], [2], 2, 1, dtype=dtype, masked=False, scale=1.0)
    c.kc[:] = torch.where(torch.isnan(c.kc), c.kc, torch.full_like(c.kc, -1e18))
    c.q_store[:] = 1.5e16
    out = c.attend(pkg, c.device())[:2].double().cpu().numpy()
    for t in range(2):
        want = c.values[0][:39 + t].double().mean(0).numpy()  # equal logits: the mean
        for h in range(2):
            assert (np.abs(out[t, h] - want[0]) <= 2.0 ** -6 * np.abs(c.values[0].double().numpy()).max()).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_rows_that_see_nothing_are_zero(pkg, dtype):
    c = Case([9, 40], [9, 3], 4, 2, dtype=dtype)
    c.mask[:] = False
    d = c.device()
    out = c.attend(pkg, d)
    assert not out[:9].any()           # no context, nothing seen
    c.check_out(out, c.oracle())       # the second sequence still sees its context


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads", [2, 12])
def test_infinities_and_nan_in_places_not_seen(pkg, dtype, heads):
    """Drafted positions hold infinities and NaN in keys and values; rows that do not see them are exact, rows that
    see them show them."""
    c = Case([60], [10], heads, 2, dtype=dtype, seed=5)
    specials = {51: math.inf, 53: -math.inf, 55: math.nan, 58: torch.finfo(dtype).max}
    c.mask[:] = True
    c.mask[:6, [1, 3, 5, 8]] = False   # rows 0..5 see none of them
    c.mask[6, [3, 5, 8]] = False       # row 6 sees +inf
    c.mask[7, [1, 5, 8]] = False       # row 7 sees -inf
    c.mask[8, [1, 3, 8]] = False       # row 8 sees NaN
    c.mask[9, [1, 3, 5]] = False       # row 9 sees the type's largest
    clean = c.oracle()
    d = c.device()
    for pos, val in specials.items():
        d["vc"][int(c.tables[0, pos // 16]), :, ::2, pos % 16] = val
    out = c.attend(pkg, d)
    rows = slice(0, 6)
    g, want, bound = out[rows].double().cpu().numpy(), clean[0][rows], clean[1][rows]
    assert (np.abs(g - want) <= bound + HALF[dtype] * (np.abs(want) + bound) + 2.0 ** -25).all()
    assert bool((out[6, :, ::2] == math.inf).all()) and bool((out[7, :, ::2] == -math.inf).all())
    assert bool(torch.isnan(out[8, :, ::2]).all()) and bool(torch.isfinite(out[6:9, :, 1::2]).all())
    assert not torch.isnan(out[9]).any()
    # keys: a NaN logit in a place that is not seen
    d = c.device()
    d["kc"][int(c.tables[0, 55 // 16]), :, :, 55 % 16] = math.nan
    out = c.attend(pkg, d)
    g = out[rows].double().cpu().numpy()
    assert (np.abs(g - want) <= bound + HALF[dtype] * (np.abs(want) + bound) + 2.0 ** -25).all()
    assert bool(torch.isnan(out[8]).all())


@pytest.mark.gpu
def test_the_same_block_twice_and_in_two_sequences(pkg):
    """Sequences that share their first blocks, and a table that names one block twice."""
    c = Case([64, 64], [2, 2], 2, 2, masked=False)
    for i, src in ((0, 1), (1, 0)):
        dst = int(c.tables[0, i])
        c.tables[1, i] = dst
        for s in (c.keys, c.values):
            s[1][16 * i:16 * i + 16] = s[0][16 * i:16 * i + 16]
    c.tables[0, 2] = c.tables[0, 0]
    for s in (c.keys, c.values):
        s[0][32:48] = s[0][0:16]
    run(pkg, c)


@pytest.mark.gpu
def test_contradictions_give_nan(pkg):
    """Each of these sequences gets NaN rows, its neighbours their results."""
    c = Case([60, 70, 30], [4, 5, 2], 4, 2, masked=False)
    oracle = c.oracle()

    def rows_of(i):
        return slice(int(c.starts[i]), int(c.starts[i + 1]))

    def check(d, bad, **kw):
        out = c.attend(pkg, d, **kw)
        for i in range(3):
            if i in bad:
                assert bool(torch.isnan(out[rows_of(i)]).all())
            else:
                g, w, b = out[rows_of(i)].double().cpu().numpy(), oracle[0][rows_of(i)], oracle[1][rows_of(i)]
                assert (np.abs(g - w) <= b + HALF[c.dtype] * (np.abs(w) + b) + 2.0 ** -25).all()
        assert bool((out[11:] == 7.0).all())

    check(c.device(), [1], max_ctx=64)             # a longer context than the call says
    check(c.device(), [1], max_query=4)            # more queries than the call says
    for bad in (-1, 1 << 20, 2 ** 31 - 1):         # a block that is not there
        d = c.device()
        d["tables"][0, 1] = bad
        check(d, [0])
    d = c.device()
    d["lens_t"][2] = 1                             # fewer positions than new tokens
    check(d, [2])
    d = c.device()
    d["lens_t"][2] = -5
    check(d, [2])


@pytest.mark.gpu
def test_query_starts_outside_the_rows(pkg):
    """Starts that run backwards or past the rows: nothing outside the output is touched."""
    c = Case([60, 70], [4, 5], 2, 1, masked=False)
    d = c.device()
    d["starts"].copy_(torch.tensor([0, 400, 5]))
    out = c.attend(pkg, d)
    assert bool(torch.isnan(out).all())
    d = c.device()
    d["starts"].copy_(torch.tensor([-3, 2, 1]))
    out = c.attend(pkg, d)
    assert bool(torch.isnan(out[:2]).all()) and bool((out[2:] == 7.0).all())


@pytest.mark.gpu
def test_empty_calls(pkg):
    c = Case([5], [2], 2, 2)
    d = c.device()
    d["query"], d["out"], d["mask"] = d["query"][:0], d["out"][:0], d["mask"][:0]
    c.attend(pkg, d)
    d = c.device()
    d["tables"], d["lens_t"], d["starts"] = d["tables"][:0], d["lens_t"][:0], d["starts"][:1]
    assert bool((c.attend(pkg, d) == 7.0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", [([40, 7, 1, 33], [1, 1, 1, 1], 4, 4), ([2050, 300], [1, 1], 8, 2), ([90, 64, 5], [3, 64, 5], 4, 2),
                                   ([1500, 0], [40, 0], 16, 2), ([9001], [2], 2, 1)], ids=str)
def test_accumulated_weights(pkg, shape, dtype):
    lens, drafted, heads, kv = shape
    c = Case(lens, drafted, heads, kv, dtype=dtype, masked=False, block=16 if heads != 8 else 32)
    oracle = c.oracle()
    d = c.device()
    gen = torch.Generator().manual_seed(1)
    old = torch.rand(c.kc.shape[0], kv, c.block, generator=gen) * 3
    touched = torch.zeros(old.shape, dtype=torch.bool)
    want, bound = old.double().clone(), torch.zeros(old.shape, dtype=torch.float64)
    for i, length in enumerate(lens):
        for pos in range(length):
            at = (int(c.tables[i, pos // c.block]), slice(None), pos % c.block)
            touched[at] = drafted[i] > 0
            if drafted[i] == 0:
                continue
            before = 0 if pos >= length - drafted[i] else old[at].double()
            want[at] = before + torch.from_numpy(oracle[2][i][:, pos])
            bound[at] = torch.from_numpy(oracle[3][i][:, pos]) + U * want[at]
    # what a block held before it was handed out does not matter
    stale = old.clone()
    for i, length in enumerate(lens):
        for pos in range(length - drafted[i], length):
            stale[int(c.tables[i, pos // c.block]), :, pos % c.block] = math.nan
    d["weights"] = stale.cuda()
    c.check_out(c.accumulate(pkg, d), oracle)
    got = d["weights"].cpu()
    same = ~touched
    assert torch.equal(got[same].view(torch.int32), stale[same].view(torch.int32))
    assert ((got.double() - want).abs()[touched] <= bound[touched] + 1e-30).all()
    # the sums are made in one order: the same call gives the same bits
    again = c.device()
    again["weights"] = stale.cuda()
    c.accumulate(pkg, again)
    assert torch.equal(again["weights"].cpu().view(torch.int32), got.view(torch.int32)) and torch.equal(again["out"], d["out"])


@pytest.mark.gpu
def test_accumulate_skips_contradictory_sequences(pkg):
    c = Case([60, 70], [1, 1], 2, 2, masked=False)
    d = c.device()
    d["weights"] = torch.ones(c.kc.shape[0], 2, 16, device="cuda")
    d["lens_t"][0] = 1000
    c.accumulate(pkg, d)
    assert bool(torch.isnan(d["out"][0]).all()) and bool(torch.isfinite(d["out"][1]).all())
    for b in range(4):
        assert bool((d["weights"][int(c.tables[0, b])] == 1).all())


@pytest.mark.gpu
@pytest.mark.parametrize("length", [60, 9000])
def test_a_bad_block_spoils_its_sequence_s_weights_alone(pkg, length):
    c = Case([length, 70], [1, 1], 2, 2, masked=False)
    d = c.device()
    d["weights"] = torch.ones(c.kc.shape[0], 2, 16, device="cuda")
    d["tables"][0, 1] = 2 ** 31 - 1
    c.accumulate(pkg, d)
    assert bool(torch.isnan(d["out"][0]).all()) and bool(torch.isfinite(d["out"][1]).all())
    w = d["weights"]
    assert bool(torch.isnan(w[int(c.tables[0, 0])]).all()) and bool((w[int(c.tables[0, 1])] == 1).all())
    assert bool((w[int(c.tables[1, 0])] >= 1).all())


@pytest.mark.gpu
def test_two_graphs_replayed_in_turn(pkg):
    """Two captured calls of other sizes, replayed on a stream of their own with eager calls between."""
    cases = [Case([700, 33], [5, 3], 4, 2, seed=1), Case([90, 1200], [1, 1], 2, 1, masked=False, seed=2)]
    devs = [c.device() for c in cases]
    devs[1]["weights"] = torch.zeros(cases[1].kc.shape[0], 1, 16, device="cuda")
    calls = [lambda: cases[0].attend(pkg, devs[0]), lambda: cases[1].accumulate(pkg, devs[1])]
    for f in calls:
        f()
    torch.cuda.synchronize()
    want = [d["out"].clone() for d in devs]
    weights = devs[1]["weights"].clone()
    graphs = []
    for f in calls:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            f()
        graphs.append(g)
    side = torch.cuda.Stream()
    for _ in range(4):
        for d in devs:
            d["out"].fill_(7.0)
        devs[1]["weights"].zero_()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            graphs[1].replay()
            graphs[0].replay()
        torch.cuda.current_stream().wait_stream(side)
        torch.randn(1 << 20, device="cuda").sum().item()
        for d, w in zip(devs, want):
            assert torch.equal(d["out"], w)
        assert torch.equal(devs[1]["weights"], weights)


@pytest.mark.gpu
def test_captured_with_the_most_logits_a_workgroup_holds(pkg):
    """Over 64 KiB of them, weighed in the launch itself: the same bits eagerly and replayed."""
    c = Case([4096, 4000, 9], [1, 1, 1], 8, 2, masked=False)
    d = c.device()
    d["weights"] = torch.zeros(c.kc.shape[0], 2, 16, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.accumulate(pkg, d)
    graph.replay()
    first = d["weights"].clone()
    e = c.device()
    e["weights"] = torch.zeros_like(first)
    c.accumulate(pkg, e)
    c.check_out(e["out"], c.oracle())
    for _ in range(3):
        d["weights"].zero_()
        d["out"].fill_(7.0)
        torch.randn(1 << 20, device="cuda").sum().item()
        graph.replay()
        assert torch.equal(d["out"], e["out"]) and torch.equal(d["weights"], e["weights"]) and torch.equal(first, e["weights"])


@pytest.mark.gpu
@pytest.mark.parametrize("drafted", [[1, 1], [5, 9], [40, 33]])
def test_blocks_past_32_bit_offsets(pkg, drafted):
    """The same batch at the start of a small cache and at the end of one of over 2^32 bytes: the same bits."""
    c = Case([130, 75], drafted, 4, 4, dim=128, block=16, masked=False)
    small = c.device()
    blocks = c.kc.shape[0]
    n = (1 << 32) // (4 * 128 * 16 * 2) + 64          # blocks of 16 KiB: offsets past 2^32 bytes
    big = dict(small)
    for k in ("kc", "vc"):
        t = torch.empty((n,) + tuple(small[k].shape[1:]), dtype=small[k].dtype, device="cuda")
        t[n - blocks:] = small[k]
        big[k] = t
    big["tables"] = torch.where(small["tables"] < blocks, small["tables"] + (n - blocks), small["tables"])
    for call in ((c.attend, c.accumulate) if max(drafted) < 10 else (c.attend,)):
        outs = []
        for d, total in ((small, blocks), (big, n)):
            d["weights"] = torch.zeros(total, 4, 16, device="cuda")
            d["out"] = torch.zeros_like(d["out"])
            outs.append(call(pkg, d).clone())
        assert torch.equal(outs[0], outs[1])
        assert torch.equal(small["weights"], big["weights"][n - blocks:])


def test_c_entry_refuses_without_a_gpu(pkg):
    c = pkg._capi
    p = ctypes.c_void_p(4096)

    def call(acc=False, **kw):
        a = dict(out=p, q=p, kc=p, vc=p, w=p, scale=1.0, bt=p, cl=p, qs=p, mask=None, ms=0, S=2, T=4, H=4, KV=2, D=64, B=16, nb=8,
                 mb=4, mc=64, mq=2, st=256, dt=c.PA_DTYPE_F16, ws=None, wb=0)
        a.update(kw)
        mid = (a["S"], a["T"], a["H"], a["KV"], a["D"], a["B"], a["nb"], a["mb"], a["mc"], a["mq"], a["st"], a["dt"], a["ws"], a["wb"], None)
        if acc:
            return c.lib.pa_cached_kv_attention_accumulate(a["out"], a["q"], a["kc"], a["vc"], a["w"], a["scale"], a["bt"], a["cl"], a["qs"], *mid)
        return c.lib.pa_tree_cached_kv_attention(a["out"], a["q"], a["kc"], a["vc"], a["scale"], a["bt"], a["cl"], a["qs"], a["mask"], a["ms"], *mid)

    big = ctypes.c_void_p(1 << 30)
    for acc in (False, True):
        assert call(acc, dt=9) == c.PA_ERR_UNSUPPORTED and "data type" in c.last_error()
        assert call(acc, D=100) == c.PA_ERR_UNSUPPORTED and "head size: 100" in c.last_error()
        assert call(acc, B=64) == c.PA_ERR_UNSUPPORTED and "block size: 64" in c.last_error()
        assert call(acc, T=-1) == c.PA_ERR_INVALID_ARGUMENT and "negative" in c.last_error()
        assert call(acc, KV=3) == c.PA_ERR_INVALID_ARGUMENT and "multiple" in c.last_error()
        assert call(acc, KV=0) == c.PA_ERR_INVALID_ARGUMENT
        assert call(acc, q=None) == c.PA_ERR_INVALID_ARGUMENT and "null" in c.last_error()
        assert call(acc, kc=ctypes.c_void_p(4104)) == c.PA_ERR_INVALID_ARGUMENT and "aligned" in c.last_error()
        assert call(acc, scale=math.inf) == c.PA_ERR_INVALID_ARGUMENT and "finite" in c.last_error()
        assert call(acc, scale=math.nan) == c.PA_ERR_INVALID_ARGUMENT
        assert call(acc, scale=-3e38) == c.PA_ERR_INVALID_ARGUMENT and "finite" in c.last_error()  # times log2(e) it is not
        assert call(acc, st=200) == c.PA_ERR_INVALID_ARGUMENT and "shorter" in c.last_error()
        assert call(acc, mc=65) == c.PA_ERR_INVALID_ARGUMENT and "cannot hold" in c.last_error()
        assert call(acc, mq=65) == c.PA_ERR_INVALID_ARGUMENT and "exceeds" in c.last_error()
        assert call(acc, nb=0) == c.PA_ERR_INVALID_ARGUMENT
        assert call(acc, mb=1 << 20, mc=1 << 20, ws=big, wb=64) == c.PA_ERR_INVALID_ARGUMENT and "workspace" in c.last_error()
        for zero in ("S", "T", "H"):
            assert call(acc, **{zero: 0}) == c.PA_OK
        assert call(acc, mq=0) == c.PA_OK
    assert call(True, w=None) == c.PA_ERR_INVALID_ARGUMENT and "null" in c.last_error()
    assert call(mask=p, ms=-1) == c.PA_ERR_INVALID_ARGUMENT and "mask" in c.last_error()
    assert c.lib.pa_tree_workspace_bytes(0, 4, 2, 64, 64, 1, 0, c.PA_DTYPE_F16) == 0
    assert c.lib.pa_tree_workspace_bytes(2, 4, 3, 64, 64, 1, 1, c.PA_DTYPE_F16) == 0
    # contexts in partitions: the logits alone are 2 sequences x 4 heads x 3 tokens x 8192 positions
    assert c.lib.pa_tree_workspace_bytes(2, 4, 2, 64, 8192, 3, 1, c.PA_DTYPE_F16) >= 2 * 4 * 3 * 8192 * 4


def test_modules_refuse_cpu_tensors(pkg):
    c = Case([20], [2], 2, 2)
    out = torch.zeros(5, 2, 64, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="must be on the GPU"):
        pkg.attention_ops.tree_cached_kv_attention(out, c.query, c.kc, c.vc, 1.0, c.tables, c.lens_t, c.starts, c.mask, 16, 20, 2)
    with pytest.raises(RuntimeError, match="must be on the GPU"):
        pkg.attention_ops.cached_kv_attention_accumulate(out, c.query, c.kc, c.vc, torch.zeros(c.kc.shape[0], 2, 16), 1.0, c.tables,
                                                         c.lens_t, c.starts, 16, 20, 2)


@pytest.mark.gpu
def test_modules_refuse_what_does_not_fit(pkg):
    c = Case([20], [2], 2, 2)

    def call(acc=False, mc=20, mq=2, **kw):
        d = c.device()
        d["weights"] = torch.zeros(c.kc.shape[0], 2, 16, device="cuda")
        for k, f in kw.items():
            d[k] = f(d[k])
        if acc:
            pkg.attention_ops.cached_kv_attention_accumulate(d["out"], d["query"], d["kc"], d["vc"], d["weights"], 1.0, d["tables"], d["lens_t"], d["starts"], 16, mc, mq)
        else:
            pkg.attention_ops.tree_cached_kv_attention(d["out"], d["query"], d["kc"], d["vc"], 1.0, d["tables"], d["lens_t"], d["starts"], d["mask"], 16, mc, mq)

    call()
    for match, kw in (
        ("one data type", dict(kc=lambda t: t.float())),
        ("one data type", dict(out=lambda t: t.float())),
        ("int32", dict(tables=lambda t: t.long())),
        ("int32", dict(starts=lambda t: t.long())),
        ("do not match", dict(starts=lambda t: t[:1])),
        ("do not match", dict(lens_t=lambda t: t.repeat(2))),
        ("contiguous", dict(kc=lambda t: t.transpose(0, 1))),
        ("shaped like query", dict(out=lambda t: t[:2])),
        ("dense", dict(query=lambda t: t.transpose(1, 2))),
        ("multiple", dict(query=lambda t: torch.zeros(5, 3, 64, dtype=t.dtype, device="cuda"), out=lambda t: torch.zeros(5, 3, 64, dtype=t.dtype, device="cuda"))),
        ("tree_mask", dict(mask=lambda t: t.int())),
        ("tree_mask", dict(mask=lambda t: t[:, :1])),
        ("tree_mask", dict(mask=lambda t: t[:1])),
        ("tree_mask", dict(mask=lambda t: t.t().contiguous().t())),
        ("one device", dict(mask=lambda t: t.cpu())),
        ("value_cache shape", dict(vc=lambda t: t[:, :, :32].contiguous())),
        ("key_cache shape", dict(kc=lambda t: t[:-1])),
    ):
        with pytest.raises(RuntimeError, match=match):
            call(**kw)
    for match, kw in (("weight_cache", dict(weights=lambda t: t.half())), ("weight_cache", dict(weights=lambda t: t[:-1])),
                      ("weight_cache", dict(weights=lambda t: t[..., :8].contiguous())), ("one device", dict(weights=lambda t: t.cpu()))):
        with pytest.raises(RuntimeError, match=match):
            call(acc=True, **kw)
    with pytest.raises(RuntimeError, match="cannot hold"):
        call(mc=1000)
    with pytest.raises(RuntimeError, match="exceeds"):
        call(mc=1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads", [2, 12, 30])                    # 10, 60 and 150 rows: each kernel
@pytest.mark.parametrize("length", [300, 517, 600, 1030, 1200])   # 2, 3 (the draft in two of them), 3, 5 and 5 partitions
def test_infinities_that_are_seen_come_through_every_number_of_partitions(pkg, length, heads, dtype):
    """As test_infinities_and_nan_in_places_not_seen, where the rows' shares of the context are joined."""
    c = Case([length], [10], heads, 2, dtype=dtype, seed=length)
    c.mask[:] = True
    c.mask[:6, [1, 3, 5]] = False   # rows 0..5 see none of them
    c.mask[6, [3, 5]] = False       # row 6 sees +inf
    c.mask[7, [1, 5]] = False       # row 7 sees -inf
    c.mask[8, [1, 3]] = False       # row 8 sees NaN
    c.mask[9, 5] = False            # row 9 sees both infinities
    want, bound = c.oracle()[:2]
    d = c.device()
    for i, val in ((1, math.inf), (3, -math.inf), (5, math.nan)):
        pos = length - 10 + i
        d["vc"][int(c.tables[0, pos // 16]), :, ::2, pos % 16] = val
    out = c.attend(pkg, d)[:10].double().cpu().numpy()
    limit = bound + HALF[dtype] * (np.abs(want) + bound) + 2.0 ** -25
    assert (np.abs(out[:6] - want[:6]) <= limit[:6]).all()
    assert (np.abs(out[6:, :, 1::2] - want[6:, :, 1::2]) <= limit[6:, :, 1::2]).all()
    assert (out[6, :, ::2] == math.inf).all() and (out[7, :, ::2] == -math.inf).all()
    assert np.isnan(out[8:, :, ::2]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", [([1500, 40, 700], [40, 33, 64], 4, 2), ([2000], [1], 8, 8), ([900] * 6, [20, 64, 3, 64, 1, 50], 16, 2)], ids=str)
def test_the_same_call_gives_the_same_bits(pkg, shape, dtype):
    """Nothing depends on which wave or workgroup comes first."""
    lens, drafted, heads, kv = shape
    c = Case(lens, drafted, heads, kv, dim=128, dtype=dtype)
    first = c.attend(pkg, c.device()).clone()
    d = c.device()
    for _ in range(20):
        d["out"].fill_(7.0)
        assert torch.equal(c.attend(pkg, d), first)


@pytest.mark.gpu
def test_bounds_past_the_tables_are_refused_before_memory_is_asked_for(pkg):
    """The workspace goes by the bounds: these would take more than the card has."""
    c = Case([20], [2], 2, 2)
    d = c.device()
    d["weights"] = torch.zeros(c.kc.shape[0], 2, 16, device="cuda")
    for most in (1 << 27, 1 << 30, 2 ** 31 - 1):
        before = torch.cuda.memory_reserved()
        with pytest.raises(RuntimeError, match="cannot hold"):
            pkg.attention_ops.cached_kv_attention_accumulate(d["out"], d["query"], d["kc"], d["vc"], d["weights"], 1.0, d["tables"],
                                                             d["lens_t"], d["starts"], 16, most, most)
        with pytest.raises(RuntimeError, match="cannot hold"):
            pkg.attention_ops.tree_cached_kv_attention(d["out"], d["query"], d["kc"], d["vc"], 1.0, d["tables"], d["lens_t"],
                                                       d["starts"], None, 16, most, most)
        assert torch.cuda.memory_reserved() == before
    # a call without rows: nothing to do, whatever its bounds
    pkg.attention_ops.cached_kv_attention_accumulate(d["out"][:0], d["query"][:0], d["kc"], d["vc"], d["weights"], 1.0, d["tables"],
                                                     d["lens_t"], d["starts"], 16, 1 << 30, 1 << 29)
    pkg.attention_ops.tree_cached_kv_attention(d["out"], d["query"], d["kc"], d["vc"], 1.0, d["tables"][:0], d["lens_t"][:0],
                                               d["starts"][:1], None, 16, 1 << 30, 1 << 29)


def test_workspace_of_bounds_that_are_refused(pkg):
    """No call takes them: no size is made up for them from sums that have overflowed."""
    c = pkg._capi
    for acc in (0, 1):
        for most in ((1 << 30) + 1, 2 ** 31 - 300, 2 ** 31 - 1):
            assert c.lib.pa_tree_workspace_bytes(1, 1, 1, 64, most, 1, acc, c.PA_DTYPE_F16) == 0
        assert c.lib.pa_tree_workspace_bytes(2 ** 31 - 1, 1024, 1024, 64, 1 << 30, 1, acc, c.PA_DTYPE_F16) == 0
        assert c.lib.pa_tree_workspace_bytes(1, 1024, 1, 64, 1 << 30, 1 << 30, acc, c.PA_DTYPE_F16) == 0
    p = ctypes.c_void_p(4096)
    for seqs, heads, query in ((2 ** 31 - 1, 1024, 1), (2 ** 31 - 1, 1024, 1 << 30), (64, 1024, 1 << 30)):
        rc = c.lib.pa_tree_cached_kv_attention(p, p, p, p, 1.0, p, p, p, None, 0, seqs, 4, heads, 1024, 64, 8, 8, 1 << 27, 1 << 30, query,
                                               heads * 64, c.PA_DTYPE_F16, None, 0, None)
        assert rc == c.PA_ERR_INVALID_ARGUMENT and "too many" in c.last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("seqs,kv,most", [(40, 8, 3), (37, 8, 20), (256, 2, 3), (255, 1, 40)])
@pytest.mark.parametrize("bound", [100, 2500])
def test_many_sequences_as_they_come_and_by_their_length(pkg, seqs, kv, most, bound):
    """The same batch under a tight bound of its contexts and under one that makes a launch take the longest first."""
    drafted = [i * 11 % (most + 1) for i in range(seqs)]
    lens = [max(t, i * 53 % 97 if i % 7 else 41) for i, t in enumerate(drafted)]
    c = Case(lens, drafted, 2 * kv, kv, dtype=torch.bfloat16, seed=bound, extra_cols=160)
    d = c.device()
    c.check_out(c.attend(pkg, d, max_ctx=bound), c.oracle())
    c.mask = None
    oracle = c.oracle()
    d = c.device()
    d["weights"] = torch.zeros(c.kc.shape[0], kv, 16, device="cuda")
    c.check_out(c.accumulate(pkg, d, max_ctx=bound), oracle)
    got = d["weights"].double().cpu().numpy()
    for i, n in enumerate(lens):
        for pos in range(n if drafted[i] else 0):
            w = got[int(c.tables[i, pos // 16]), :, pos % 16]
            assert (np.abs(w - oracle[2][i][:, pos]) <= oracle[3][i][:, pos] + U * oracle[2][i][:, pos] + 1e-30).all()
    d["lens_t"][20] = 10 ** 6                # its own rows only
    out = c.accumulate(pkg, d, max_ctx=bound)
    wrong = torch.zeros(sum(drafted), dtype=torch.bool)
    wrong[int(c.starts[20]):int(c.starts[21])] = True
    assert torch.equal(torch.isnan(out[:sum(drafted)]).flatten(1).any(1).cpu(), wrong)


@pytest.mark.gpu
@pytest.mark.parametrize("drafted", [[5, 3], [12, 40]])
def test_masks_of_any_byte_and_stride(pkg, drafted):
    """uint8 masks of any non-zero value, rows of a wider tensor from an odd address, and one row for all tokens."""
    c = Case([70, 90], drafted, 4, 2, seed=9)
    gen = torch.Generator().manual_seed(4)
    values = torch.tensor([1, 2, 64, 128, 255], dtype=torch.uint8)[torch.randint(0, 5, c.mask.shape, generator=gen)] * c.mask
    wide = torch.randint(0, 256, (c.mask.shape[0], c.mask.shape[1] + 13), generator=gen, dtype=torch.uint8)
    wide[:, 7:7 + c.mask.shape[1]] = values
    d = c.device()
    d["mask"] = wide.cuda()[:, 7:7 + c.mask.shape[1]]
    c.check_out(c.attend(pkg, d), c.oracle())
    c.mask = c.mask[:1].expand(c.mask.shape[0], -1).contiguous()
    d = c.device()
    d["mask"] = c.mask[:1].cuda().expand(c.mask.shape[0], -1)
    c.check_out(c.attend(pkg, d), c.oracle())


@pytest.mark.gpu
def test_two_threads_on_two_streams(pkg):
    """Calls of two sizes from two host threads, on a stream each: the bits of the same calls one after the other."""
    import threading
    cases = [Case([4096, 300], [1, 1], 8, 2, masked=False, seed=1), Case([4600, 17, 900], [1, 1, 1], 8, 2, masked=False, seed=2)]
    devs = [c.device() for c in cases]
    want = []
    for c, d in zip(cases, devs):
        d["weights"] = torch.zeros(c.kc.shape[0], 2, 16, device="cuda")
        c.accumulate(pkg, d)
        want.append((d["out"].clone(), d["weights"].clone()))
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        c, d = cases[i], devs[i]
        stream = torch.cuda.Stream()
        try:
            with torch.cuda.stream(stream):
                for _ in range(30):
                    d["weights"].zero_()
                    d["out"].fill_(7.0)
                    c.accumulate(pkg, d)
                    if not (torch.equal(d["out"], want[i][0]) and torch.equal(d["weights"], want[i][1])):
                        wrong.append(i)
            stream.synchronize()
        except Exception as e:
            wrong.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@pytest.mark.gpu
@pytest.mark.parametrize("length,drafted", [(400, 300), (700, 40), (64, 5)])
def test_a_bad_block_within_a_chain(pkg, length, drafted):
    """The last block is not there: rows that reach it are NaN, rows before it NaN or their results."""
    c = Case([length], [drafted], 4, 2, masked=False)
    want, bound = c.oracle()[:2]
    d = c.device()
    last = (length - 1) // 16
    d["tables"][0, last] = c.kc.shape[0]
    out = c.attend(pkg, d)[:drafted].double().cpu().numpy()
    reach = np.arange(drafted) + length - drafted >= last * 16
    assert np.isnan(out[reach]).all()
    rest = out[~reach]
    limit = (bound + HALF[c.dtype] * (np.abs(want) + bound) + 2.0 ** -25)[~reach]
    assert (np.isnan(rest) | (np.abs(rest - want[~reach]) <= limit)).all()
    assert (np.isnan(rest).all((1, 2)) | ~np.isnan(rest).any((1, 2))).all()
