"""The block operators on the GPU where their forms end: sizes that take each
tile, repeated and far-apart rows, offsets past 32 bits, scales of 0 and near it, many small
weights, hidden NaN under every tile of the attention, mostly empty batches,
and splits with workspaces of their own in captured graphs."""
import numpy as np
import pytest
import torch

import block_reference as R
from test_gpu_block import NAN, attention_case, near, rnd, run_attention, weights

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ products

# n m from below 2^20 to above 2^24: tiles of 64 with k in one, two and four shares, of 128 and of 256; odd edges of each.
@pytest.mark.parametrize("pair", [("f32", "f32"), ("f32", "q8_0"), ("f16", "f16"), ("bf16", "bf16"), ("bf16", "q8_0")],
                         ids="-".join)
@pytest.mark.parametrize("shape", [(2049, 96, 2100), (4100, 64, 4099), (1030, 160, 1100), (700, 64, 130)], ids=str)
def test_linear_of_every_tile(eg2, gpu, pair, shape):
    (kind, wkind), (n, k, m) = pair, shape
    if wkind != "q8_0":
        k += 6  # a last slice that is not whole
    rng = np.random.default_rng(n)
    x, x64 = rnd(rng, (n, k), kind)
    w, w64 = weights(rng, m, k, wkind, gpu)
    b = rng.standard_normal(m).astype(np.float32)
    y = torch.full((n, m), NAN, dtype=R.TYPES[kind], device=gpu)
    eg2.ops.linear(x.to(gpu), w, y, bias=torch.from_numpy(b).to(gpu), act="silu")
    near(y, *R.linear(x64, w64, b, "silu", None, R.TYPES[kind]))


@pytest.mark.parametrize("pair", [("f32", "f32"), ("bf16", "bf16"), ("f16", "q8_0")], ids="-".join)
@pytest.mark.parametrize("shape", [(2049, 96, 1100), (4100, 64, 2051)], ids=str)
def test_linear_gated_of_large_tiles(eg2, gpu, pair, shape):
    (kind, wkind), (n, k, m) = pair, shape
    rng = np.random.default_rng(m)
    x, x64 = rnd(rng, (n, k), kind)
    (g, g64), (u, u64) = weights(rng, m, k, wkind, gpu), weights(rng, m, k, wkind, gpu)
    y = torch.full((n, m), NAN, dtype=R.TYPES[kind], device=gpu)
    eg2.ops.linear_gated(x.to(gpu), g, u, y, act="gelu")
    near(y, *R.linear_gated(x64, g64, u64, None, None, "gelu", R.TYPES[kind]))


@pytest.mark.parametrize("pair", [("f32", "f32"), ("f32", "q8_0"), ("bf16", "bf16"), ("bf16", "q8_0")], ids="-".join)
@pytest.mark.parametrize("n", [3, 200])
def test_repeated_rows(eg2, gpu, pair, n):
    """One row of weights for every column and one row of x for every row: strides of 0."""
    kind, wkind = pair
    rng = np.random.default_rng(n)
    x, x64 = rnd(rng, (1, 96), kind)
    w, w64 = weights(rng, 1, 96, wkind, gpu)
    y = torch.full((n, 150), NAN, dtype=R.TYPES[kind], device=gpu)
    eg2.ops.linear(x.to(gpu).expand(n, -1), w.expand(150, -1), y)
    near(y, *R.linear(np.repeat(x64, n, 0), np.repeat(w64, 150, 0), None, "none", None, R.TYPES[kind]))


@pytest.fixture(scope="module")
def far(gpu):
    """bf16 values past 2^32 elements; only what a test writes is defined."""
    return torch.empty(40 << 27, dtype=torch.bfloat16, device=gpu)


@pytest.mark.parametrize("stride", [1 << 20, 1 << 27])
def test_rows_past_32_bits(eg2, gpu, far, stride):
    """Rows of x, the weights, y and the residual whose offsets pass 2^32 elements."""
    rng = np.random.default_rng(1)
    rows = far.numel() // stride
    n, m = min(rows, 4200), 40
    wide = far.view(-1, stride)[:n]
    x, x64 = rnd(rng, (n, 72), "bf16")
    w, w64 = weights(rng, m, 72, "bf16", gpu)
    r, r64 = rnd(rng, (n, m), "bf16")
    wide[:, :72], wide[:, 80:80 + m], wide[:m, 200:272] = x.to(gpu), r.to(gpu), w
    eg2.ops.linear(wide[:, :72], wide[:m, 200:272], wide[:, 130:130 + m], act="relu", residual=wide[:, 80:80 + m])
    near(wide[:, 130:130 + m], *R.linear(x64, w64, None, "relu", r64, torch.bfloat16))


@pytest.mark.parametrize("stride", [1 << 20, 1 << 27])
def test_heads_past_32_bits(eg2, gpu, far, stride):
    rng = np.random.default_rng(2)
    rows = min(far.numel() // stride, 4200)
    wide = far.view(-1, stride)[:rows]
    x, x64 = rnd(rng, (rows, 3, 64), "bf16")
    heads = wide[:, :192].unflatten(1, (3, 64))
    heads.copy_(x.to(gpu))
    eg2.ops.heads_norm_rope(heads[:, :2], heads[:, 2:], None, None, None, None, 1e-6, heads[:, :2], heads[:, 2:], 0.5)
    scale = np.array([0.5, 0.5, 1.0])[None, :, None]
    want, off = R.heads_norm_rope(x64, None, None, None, 1e-6, 1.0, torch.bfloat16)
    near(heads, want * scale, off * scale)  # halves are exact


@pytest.mark.parametrize("stride", [1 << 20, 1 << 27])
@pytest.mark.parametrize("q_len", [1, 24])
def test_attention_cache_past_32_bits(eg2, gpu, far, stride, q_len):
    """Keys and values at the end of a cache whose last rows lie past 2^32 elements (a tile's rows past 2^32 bytes)."""
    rng = np.random.default_rng(3)
    rows = far.numel() // stride
    n = min(rows, 700)
    wide = far.view(-1, stride)
    (k, k64), (v, v64), (q, q64) = rnd(rng, (n, 1, 64), "bf16"), rnd(rng, (n, 1, 64), "bf16"), rnd(rng, (q_len, 2, 64), "bf16")
    keys, values = (wide[:, a:a + 64].unsqueeze(1) for a in (0, 64))
    keys[rows - n:], values[rows - n:] = k.to(gpu), v.to(gpu)
    off = torch.tensor([0, q_len], dtype=torch.int32, device=gpu)
    at = torch.tensor([rows - n, rows], dtype=torch.int32, device=gpu)
    out = torch.full((q_len, 2, 64), 77.0, dtype=torch.bfloat16, device=gpu)
    eg2.ops.window_attention(q.to(gpu), keys, values, off, at, out, 0.125, -1, 0, 0, longest=n)
    near(out, *R.window_attention(q64, k64, v64, [0, q_len], [0, n], 0.125, -1, 0, 0, None, torch.bfloat16))


# ------------------------------------------------------------------ attention

@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows", [2400, 1200, 600])  # of 8 heads: tiles of 128 (fp32 64), 64 and 32 rows
@pytest.mark.parametrize("d", [64, 128, 200, 256])
def test_attention_hidden_places_in_every_tile(eg2, gpu, kind, rows, d):
    """NaN behind the keys, and a NaN and an infinite key or value that some rows of a tile see: those rows
    are NaN (or what the infinity makes of them), the others as if it were not there."""
    rng = np.random.default_rng(rows + d)
    (q, q64), (k, k64), (v, v64), qo, ko, kl = attention_case(rng, kind, [rows], [rows], 8, 1, d, cap=rows + 50)
    k[rows:], v[rows:] = NAN, NAN
    j, i = rows // 3, 2 * rows // 3
    for at in (j, i):
        k64[at], v64[at] = 0, 0  # of the rows that do not see it
    v[j, 0, ::7], v[i, 0, 1::5] = NAN, float("inf")
    k[i] = NAN
    left, right, sinks = 40, 0, 2
    got = run_attention(eg2, gpu, q, k, v, qo, ko, kl, d ** -0.5, left, right, sinks, rows).double().cpu().numpy()
    seen = {t: at for at in (j, i) for t in range(at, at + left + 1)}
    for t0, t1 in ((0, 70), (j - 50, j + 100), (i - 50, i + 100), (rows - 70, rows)):
        want, off = R.window_attention(q64[t0:t1], k64[:t1], v64[:t1], [0, t1 - t0], [0, t1], d ** -0.5, left, right, sinks,
                                       None, R.TYPES[kind])
        for t in range(t0, t1):
            if t not in seen:
                assert (np.abs(got[t] - want[t - t0]) <= off[t - t0]).all(), t
            elif seen[t] == i:
                assert np.isnan(got[t]).all(), t
            else:
                assert np.isnan(got[t][:, ::7]).all(), t
    for t in range(j, j + left + 1):  # the value's other columns are as before
        assert np.isfinite(got[t][:, 1::7]).all(), t


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("scale", [0.0, -0.0, 1e-44, -1e-36])
def test_attention_scales_near_zero(eg2, gpu, kind, scale):
    """Weights that are all but equal, also with large products of queries and keys (fp32: 1e37)."""
    rng = np.random.default_rng(4)
    big = 1e17 if kind == "f32" else 30.0
    q, k = rnd(rng, (33, 2, 64), kind, big), rnd(rng, (50, 1, 64), kind, big)
    v, v64 = rnd(rng, (50, 1, 64), kind)
    qo, ko = np.array([0, 33], np.int32), np.array([0, 50], np.int32)
    got = run_attention(eg2, gpu, q[0], k[0], v, qo, ko, None, scale, 20, 0, 1)
    s = np.float64(np.float32(scale))
    want, off = R.window_attention(q[1], k[1], v64, qo, ko, s, 20, 0, 1, None, R.TYPES[kind])
    # a scale below 2^-126 counts to its last bit: at most half a step of 2^-149 times the products, of two factors
    top = np.abs(q[1]).max() * np.abs(k[1]).max() * 64
    near(got, want, off + np.abs(v64).max() * 4 * np.expm1(2.0 ** -148 * top))


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows", [1, 40, 700, 2400])
def test_attention_many_small_weights(eg2, gpu, kind, rows):
    """One key far above 4000 others, whose weights of 2^-16 (below fp16's normal numbers) still add up to 6 %."""
    rng = np.random.default_rng(5)
    k = torch.zeros(4000, 1, 64, dtype=R.TYPES[kind])
    k[37, 0, 0] = 11.0
    q = torch.zeros(rows, 8, 64, dtype=R.TYPES[kind])
    q[:, :, 0] = 1.0
    v = torch.from_numpy(rng.uniform(0.5, 1.5, (4000, 1, 64)).astype(np.float32)).to(R.TYPES[kind])
    qo, ko = np.array([0, rows], np.int32), np.array([0, 4000], np.int32)
    got = run_attention(eg2, gpu, q, k, v, qo, ko, None, 1.0, -1, -1, 0, 4000)
    want, off = R.window_attention(q[:1].double().numpy(), k.double().numpy(), v.double().numpy(), [0, 1], ko, 1.0, -1, -1, 0,
                                   None, R.TYPES[kind])
    near(got, np.broadcast_to(want[:1], got.shape), np.broadcast_to(off[:1], got.shape))


def test_attention_of_a_mostly_empty_batch(eg2, gpu):
    """The most sequences and heads, one of them with a query."""
    rng = np.random.default_rng(6)
    batch, kv = 65535, 64
    (q, q64), (k, k64), (v, v64) = rnd(rng, (1, kv, 8), "bf16"), rnd(rng, (900, kv, 8), "bf16"), rnd(rng, (900, kv, 8), "bf16")
    for at in (0, 40000, batch - 1):
        qo = (np.arange(batch + 1) > at).astype(np.int32)
        ko = qo * 900
        got = run_attention(eg2, gpu, q, k, v, qo, ko, None, 0.3, -1, 0, 0, 900)
        near(got, *R.window_attention(q64, k64, v64, [0, 1], [0, 900], 0.3, -1, 0, 0, None, torch.bfloat16))


def test_attention_of_many_sequences(eg2, gpu):
    """5000 sequences of no, one and a few rows: the search for a tile's sequence in several rounds."""
    rng = np.random.default_rng(7)
    lens = rng.integers(0, 4, 5000)
    (q, q64), (k, k64), (v, v64), qo, ko, _ = attention_case(rng, "f32", list(lens), list(lens), 1, 1, 8)
    got = run_attention(eg2, gpu, q, k, v, qo, ko, None, 0.3, -1, 0, 0)
    near(got, *R.window_attention(q64, k64, v64, qo, ko, 0.3, -1, 0, 0, None, q.dtype))


def split_call(gpu, seed):
    rng = np.random.default_rng(seed)
    d = {name: rnd(rng, shape, "bf16")[0].to(gpu) for name, shape in
         (("q", (3, 4, 128)), ("k", (6000, 2, 128)), ("v", (6000, 2, 128)), ("out", (3, 4, 128)))}
    d["qo"] = torch.tensor([0, 1, 3], dtype=torch.int32, device=gpu)
    d["ko"] = torch.tensor([0, 2000, 6000], dtype=torch.int32, device=gpu)
    return d


def run_split(eg2, d, **more):
    eg2.ops.window_attention(d["q"], d["k"], d["v"], d["qo"], d["ko"], d["out"], 0.1, 1500, 0, 4, longest=4000, **more)


def test_attention_workspace_of_the_caller(eg2, gpu):
    need = eg2.ops.window_attention_workspace(2, 3, 6000, 4, 2, 128, torch.bfloat16, 1500, 0, 4, 4000)
    assert need > 0
    d = split_call(gpu, 1)
    run_split(eg2, d)
    want = d["out"].clone()
    space = torch.full((need + 4096,), 0xFF, dtype=torch.uint8, device=gpu)  # of NaN
    run_split(eg2, d, workspace=space[:need])
    assert torch.equal(d["out"], want) and (space[need:] == 0xFF).all()
    with pytest.raises(eg2.HipError):
        run_split(eg2, d, workspace=space[:need - 1])
    with pytest.raises(eg2.HipError):
        run_split(eg2, d, workspace=space[8:need + 8])
    with pytest.raises(ValueError):
        run_split(eg2, d, workspace=space[:need].cpu())


def test_two_captured_splits_replay_at_once(eg2, gpu):
    """Two graphs of split calls, each with its own workspace, on two streams, their inputs changed between replays."""
    calls = [split_call(gpu, seed) for seed in (1, 2)]
    want = []
    for d in calls:
        run_split(eg2, d)
        want.append(d["out"].clone())
    torch.cuda.synchronize()
    graphs, streams = [torch.cuda.CUDAGraph() for _ in calls], [torch.cuda.Stream() for _ in calls]
    for g, d in zip(graphs, calls):
        with torch.cuda.graph(g):
            run_split(eg2, d)
    first = [{n: d[n].clone() for n in ("q", "k", "v")} for d in calls]
    for turn in range(4):
        for i, d in enumerate(calls):
            for n in ("q", "k", "v"):
                d[n].copy_(first[i ^ (turn & 1)][n])
            d["out"].fill_(NAN)
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for i, d in enumerate(calls):
            assert torch.equal(d["out"], want[i ^ (turn & 1)]), (turn, i)
