"""rotary_embedding and qk_norm_rotary_embedding: both pair layouts, parts of a head, head norms.

The definition is evaluated here in float64 with numpy.  Tolerances, counted from the arithmetic:
  * one rounding to the storage type at the end, half a step: eps / 2 relative to the value
    (2^-11 fp16, 2^-8 bf16, 2^-24 fp32);
  * the table is exact as given (the oracle reads the same float32 or 16-bit numbers);
  * fp32 in between: the rotation is a product and a fused multiply-add, off by at most 2 * 2^-24
    of |a cos| + |b sin|; the norm adds the sum of squares (n terms, pairwise over lanes: at most
    (n / 16 + 8) * 2^-24 relative, halved by the root), the mean, the root, the reciprocal and two
    products: 8 * 2^-24 more.
"""
import ctypes

import numpy as np
import pytest
import torch

HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}
U = 2.0 ** -24


def make_table(max_position, rot_dim, dtype, base=10000.0):
    freq = base ** (-np.arange(0, rot_dim, 2) / max(rot_dim, 1))
    angle = np.arange(max_position)[:, None] * freq[None]
    return torch.from_numpy(np.concatenate((np.cos(angle), np.sin(angle)), 1)).to(dtype)


def oracle(positions, rows, head_size, table, interleaved, weight=None, epsilon=0.0):
    """(result, bound of the error before the last rounding), both float64 [tokens, heads, head_size]."""
    x = rows.double().cpu().numpy().reshape(rows.shape[0], -1, head_size).copy()
    err = np.zeros_like(x)
    if weight is not None:
        x *= 1.0 / np.sqrt((x * x).mean(-1, keepdims=True) + epsilon)
        x *= weight.double().cpu().numpy()
        err = np.abs(x) * U * ((head_size / 16 + 8) / 2 + 8)
    rot = table.shape[1]
    row = table.double().cpu().numpy()[positions.cpu().numpy()][:, None]
    c, s = row[..., :rot // 2], row[..., rot // 2:]
    ia = slice(0, rot, 2) if interleaved else slice(0, rot // 2)
    ib = slice(1, rot, 2) if interleaved else slice(rot // 2, rot)
    a, b = x[..., ia].copy(), x[..., ib].copy()
    ea, eb = err[..., ia].copy(), err[..., ib].copy()
    x[..., ia], x[..., ib] = a * c - b * s, b * c + a * s
    err[..., ia] = ea * abs(c) + eb * abs(s) + 2 * U * (abs(a * c) + abs(b * s))
    err[..., ib] = eb * abs(c) + ea * abs(s) + 2 * U * (abs(b * c) + abs(a * s))
    return x, err


def assert_rows(got, want, err, what):
    g = got.double().cpu().numpy().reshape(want.shape)
    bound = err + HALF_STEP[got.dtype] * (np.abs(want) + err) + TINY[got.dtype]
    bad = ~(np.abs(g - want) <= bound)
    assert not bad.any(), f"{what}: {bad.sum()} elements, worst {np.abs(g - want)[bad].max()} at {np.argwhere(bad)[0]}"


def rows_of(gen, tokens, heads, head_size, dtype, pad, shift, device):
    """[tokens, heads * head_size] with a row stride of `pad` more, `shift` elements into its storage."""
    n = heads * head_size
    base = torch.randn(tokens * (n + pad) + shift, generator=gen).to(dtype).to(device)
    return base, base[shift:].as_strided((tokens, n), (n + pad, 1), shift)


CASES = [
    # tokens, heads, kv heads, head size, rot_dim, row padding, storage shift
    (1, 1, 1, 64, 64, 0, 0),
    (7, 12, 12, 64, 32, 8, 0),
    (33, 32, 8, 128, 128, 64, 0),
    (5, 40, 40, 128, 64, 0, 0),
    (19, 5, 1, 80, 80, 0, 0),
    (3, 4, 2, 96, 24, 0, 0),       # 12 pairs: narrower vectors
    (9, 3, 3, 80, 20, 16, 0),      # 10 pairs
    (4, 2, 1, 66, 6, 0, 0),        # odd numbers of pairs and of the rest
    (11, 4, 4, 64, 64, 1, 0),      # odd row stride: element by element
    (6, 4, 2, 128, 96, 2, 1),      # odd start
    (2, 3, 1, 256, 256, 3, 0),     # long head, odd stride: more elements than lanes
    (2, 2, 2, 512, 64, 0, 0),      # a rest of more vectors than pairs
    (3, 2, 1, 2, 2, 0, 0),         # one pair
    (300, 2, 1, 64, 64, 0, 0),
    (5, 7, 0, 64, 64, 0, 0),       # no key heads
]


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "x".join(map(str, c)))
def test_against_float64(pkg, case, dtype, norm, interleaved):
    tokens, heads, kv, d, rot, pad, shift = case
    gen = torch.Generator().manual_seed(hash(case) % 1000)
    qb, q = rows_of(gen, tokens, heads, d, dtype, pad, shift, "cuda")
    kb, k = rows_of(gen, tokens, kv, d, dtype, pad, shift, "cuda")
    table_dtype = torch.float32 if (tokens + heads) % 2 else dtype
    table = make_table(512, rot, table_dtype).cuda()
    pos = torch.randint(0, 512, (tokens,), generator=gen).cuda()
    wq, wk = ((1 + 0.3 * torch.randn(d, generator=gen)).to(dtype).cuda() for _ in range(2))
    before = [qb.clone(), kb.clone()]
    want = [oracle(pos, r, d, table, interleaved, w if norm else None, 1e-5) for r, w in ((q, wq), (k, wk))]
    ops = pkg.pos_encoding_ops
    if norm:
        ops.qk_norm_rotary_embedding(pos, q, k, d, wq, wk, 1e-5, table, interleaved)
    else:
        ops.rotary_embedding(pos, q, k, d, table, interleaved)
    for got, (w, e), name in ((q, want[0], "query"), (k, want[1], "key")):
        if got.numel():
            assert_rows(got, w, e, name)
    # what lies between and around the rows is as it was; without the norm so is the unrotated part
    for base, was, rows in ((qb, before[0], q), (kb, before[1], k)):
        touched = torch.zeros(base.shape, dtype=torch.bool, device="cuda")
        mark = touched[shift:].as_strided(rows.shape, rows.stride(), shift)
        mark.unflatten(1, (-1, d))[..., :d if norm else rot] = True
        assert torch.equal(base[~touched], was[~touched])


@pytest.mark.gpu
def test_agrees_with_the_neox_operator_to_its_rounding(pkg):
    """Half layout, one number of heads, a table of the rows' type: the operator that was there, but for its roundings
    (each product and the sum are rounded: at most 3 half steps of |a cos| + |b sin|)."""
    gen = torch.Generator().manual_seed(3)
    q, k = (torch.randn(37, 12 * 64, generator=gen).half().cuda() for _ in range(2))
    table = make_table(128, 64, torch.float16).cuda()
    pos = torch.randint(0, 128, (37,), generator=gen).cuda()
    q2, k2 = q.clone(), k.clone()
    x = q.double().cpu().view(37, 12, 64)
    pkg.pos_encoding_ops.rotary_embedding_neox(pos, q, k, 64, table)
    pkg.pos_encoding_ops.rotary_embedding(pos, q2, k2, 64, table, False)
    mass = (x[..., :32].abs() + x[..., 32:].abs()).repeat(1, 1, 2).view(37, -1)
    assert ((q.double() - q2.double()).cpu().abs() <= 4 * 2.0 ** -11 * mass + 2.0 ** -24).all()


@pytest.mark.gpu
@pytest.mark.parametrize("norm", [False, True])
def test_padded_and_unknown_positions(pkg, norm):
    gen = torch.Generator().manual_seed(4)
    q, k = torch.randn(4, 2 * 64, generator=gen).half().cuda(), torch.randn(4, 64, generator=gen).half().cuda()
    w = torch.ones(64, dtype=torch.float16, device="cuda")
    table = make_table(16, 32, torch.float32).cuda()
    pos = torch.tensor([-1, 15, 16, 1 << 40]).cuda()
    q0, k0 = q.clone(), k.clone()
    if norm:
        pkg.pos_encoding_ops.qk_norm_rotary_embedding(pos, q, k, 64, w, w, 1e-6, table, True)
    else:
        pkg.pos_encoding_ops.rotary_embedding(pos, q, k, 64, table, True)
    assert torch.equal(q[0], q0[0]) and torch.equal(k[0], k0[0])
    assert torch.isfinite(q[1]).all() and torch.isfinite(k[1]).all() and not torch.equal(q[1], q0[1])
    for rows in (q.view(4, 2, 64)[2:], k.view(4, 1, 64)[2:]):
        assert torch.isnan(rows[..., :32]).all() and torch.isfinite(rows[..., 32:]).all()


@pytest.mark.gpu
def test_head_of_zeros_stays_zero(pkg):
    q, k = torch.zeros(2, 128, dtype=torch.bfloat16, device="cuda"), torch.zeros(2, 64, dtype=torch.bfloat16, device="cuda")
    w = torch.ones(64, dtype=torch.bfloat16, device="cuda")
    pkg.pos_encoding_ops.qk_norm_rotary_embedding(torch.arange(2).cuda(), q, k, 64, w, w, 1e-6, make_table(4, 64, torch.float32).cuda(), False)
    assert not q.any() and not k.any()


@pytest.mark.gpu
def test_captured_and_on_a_side_stream(pkg):
    gen = torch.Generator().manual_seed(5)
    src = torch.randn(16, 6 * 64, generator=gen).half().cuda()
    table, pos = make_table(64, 64, torch.float32).cuda(), torch.arange(16).cuda()
    w = torch.ones(64, dtype=torch.float16, device="cuda")
    want = src.clone()
    pkg.pos_encoding_ops.qk_norm_rotary_embedding(pos, want[:, :256], want[:, 256:], 64, w, w, 1e-6, table, False)
    qkv = src.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        pkg.pos_encoding_ops.qk_norm_rotary_embedding(pos, qkv[:, :256], qkv[:, 256:], 64, w, w, 1e-6, table, False)
    for _ in range(3):
        qkv.copy_(src)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(qkv, want)


def test_c_entry_refuses_without_a_gpu(pkg):
    c = pkg._capi
    p = [ctypes.c_void_p(4096 * (i + 1)) for i in range(6)]

    def call(norm=False, **kw):
        a = dict(T=2, H=2, KV=1, D=64, rot=32, maxp=8, qs=128, ks=64, dtype=c.PA_DTYPE_F16, table=c.PA_DTYPE_F32,
                 pos=p[0], q=p[1], k=p[2], tab=p[3], wq=p[4], wk=p[5])
        a.update(kw)
        tail = (a["tab"], a["T"], a["H"], a["KV"], a["D"], a["rot"], a["maxp"], a["qs"], a["ks"], 0, a["dtype"], a["table"], None)
        if norm:
            return c.lib.pa_qk_norm_rotary_embedding(a["pos"], a["q"], a["k"], a["wq"], a["wk"], 1e-6, *tail)
        return c.lib.pa_rotary_embedding(a["pos"], a["q"], a["k"], *tail)

    for norm in (False, True):
        assert call(norm, dtype=7) == c.PA_ERR_UNSUPPORTED and "data type" in c.last_error()
        assert call(norm, dtype=c.PA_DTYPE_F32, table=c.PA_DTYPE_F16) == c.PA_ERR_UNSUPPORTED and "cos_sin_cache" in c.last_error()
        assert call(norm, rot=33) == c.PA_ERR_INVALID_ARGUMENT and "even" in c.last_error()
        assert call(norm, rot=66) == c.PA_ERR_INVALID_ARGUMENT
        assert call(norm, T=-1) == c.PA_ERR_INVALID_ARGUMENT and "negative" in c.last_error()
        assert call(norm, pos=None) == c.PA_ERR_INVALID_ARGUMENT and "null" in c.last_error()
        assert call(norm, qs=100) == c.PA_ERR_INVALID_ARGUMENT and "shorter" in c.last_error()
        assert call(norm, k=ctypes.c_void_p(4096 * 2 + 64)) == c.PA_ERR_INVALID_ARGUMENT and "overlap" in c.last_error()
        assert call(norm, qs=192, ks=192, k=ctypes.c_void_p(4096 * 2 + 200)) == c.PA_ERR_INVALID_ARGUMENT and "overlap" in c.last_error()
        assert call(norm, T=0) == c.PA_OK and c.last_error() == ""
    assert call(True, wq=None) == c.PA_ERR_INVALID_ARGUMENT and "weight" in c.last_error()


def test_modules_refuse_cpu_tensors(pkg):
    q, k = torch.zeros(2, 128), torch.zeros(2, 64)
    pos, tab, w = torch.zeros(2, dtype=torch.int64), torch.zeros(4, 64), torch.ones(64)
    with pytest.raises(RuntimeError, match="must be on the GPU"):
        pkg.pos_encoding_ops.rotary_embedding(pos, q, k, 64, tab, False)
    with pytest.raises(RuntimeError, match="must be on the GPU"):
        pkg.pos_encoding_ops.qk_norm_rotary_embedding(pos, q, k, 64, w, w, 1e-6, tab, False)


@pytest.mark.gpu
def test_modules_refuse_what_does_not_fit(pkg):
    q, k = torch.zeros(2, 128, device="cuda").half(), torch.zeros(2, 64, device="cuda").half()
    pos, tab = torch.zeros(2, dtype=torch.int64, device="cuda"), torch.zeros(4, 64, device="cuda")
    w = torch.ones(64, device="cuda").half()
    rot, norm = pkg.pos_encoding_ops.rotary_embedding, pkg.pos_encoding_ops.qk_norm_rotary_embedding
    for bad, match in (
        (lambda: rot(pos.int(), q, k, 64, tab, False), "int64"),
        (lambda: rot(pos[:1], q, k, 64, tab, False), "shorter"),
        (lambda: rot(pos, q, k.float(), 64, tab, False), "one data type"),
        (lambda: rot(pos, q, k, 64, tab.double(), False), "cos_sin_cache"),
        (lambda: rot(pos, q, k, 48, tab[:, :48].contiguous(), False), "no multiple"),
        (lambda: rot(pos, q, k, 32, tab, False), "rot_dim"),
        (lambda: rot(pos, q, k[:1], 64, tab, False), "num_kv_heads"),
        (lambda: rot(pos, q, q[:, :64], 64, tab, False), "overlap"),
        (lambda: rot(pos, q.t(), k, 64, tab, False), "num_heads|dense"),
        (lambda: norm(pos, q, k, 64, w.float(), w, 1e-6, tab, False), "weights"),
        (lambda: norm(pos, q, k, 64, w[:32], w, 1e-6, tab, False), "weights"),
        (lambda: norm(pos, q, k, 64, w, w, -1.0, tab, False), "epsilon"),
    ):
        with pytest.raises(RuntimeError, match=match):
            bad()
