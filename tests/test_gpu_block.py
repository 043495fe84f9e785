"""The block operators (eg2_hip_linear, _linear_gated, _heads_norm_rope,
_window_attention) on the GPU against their definitions in 64 bits
(block_reference.py, which derives every bound): types, sizes from one to past
a tile and odd ones, strides, alignment, masks that leave rows empty, what lies in hidden
places, buffers behind the results, streams, captured graphs, and the whole block."""
import numpy as np
import pytest
import torch

import block_reference as R

pytestmark = pytest.mark.gpu
NAN = float("nan")


def rnd(rng, shape, dtype, scale=1.0):
    """(tensor of dtype on the host, its values in 64 bits)"""
    t = torch.from_numpy((rng.standard_normal(shape) * scale).astype(np.float32)).to(R.TYPES[dtype])
    return t, t.double().numpy()


def weights(rng, m, k, kind, gpu):
    w = (rng.standard_normal((m, k)) / np.sqrt(k)).astype(np.float32)
    if kind == "q8_0":
        raw, values = R.quantize(w)
        return torch.from_numpy(raw).to(gpu), values
    t = torch.from_numpy(w).to(R.TYPES[kind])
    return t.to(gpu), t.double().numpy()


def near(got, want, off):
    got = got.double().cpu().numpy()
    bad = ~(np.abs(got - want) <= off)
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4], np.abs(got - want)[bad][:4], off[bad][:4])


def inside(t, gpu, pad=3):
    """A copy of a host matrix as the middle of a larger NaN buffer: (view, buffer)."""
    rows, cols = t.shape
    buf = torch.full((rows + 2, cols + 2 * pad), NAN, dtype=t.dtype, device=gpu)
    buf[1:-1, pad:-pad] = t.to(gpu)
    return buf[1:-1, pad:-pad], buf


# ------------------------------------------------------------------ products

PAIRS = [("f32", "f32"), ("f32", "f16"), ("f32", "bf16"), ("f32", "q8_0"), ("f16", "f16"), ("f16", "q8_0"),
         ("bf16", "bf16"), ("bf16", "q8_0")]
SHAPES = [(1, 32, 1), (1, 768, 768), (2, 64, 130), (5, 2048, 96), (16, 96, 64), (17, 32, 65), (33, 160, 257),
          (64, 512, 128), (130, 800, 200), (257, 256, 300), (300, 64, 1000)]


def run_linear(eg2, gpu, rng, pair, shape, act="none", bias=True, residual=True):
    (kind, wkind), (n, k, m) = pair, shape
    x, x64 = rnd(rng, (n, k), kind)
    w, w64 = weights(rng, m, k, wkind, gpu)
    b = rng.standard_normal(m).astype(np.float32) if bias else None
    r, r64 = rnd(rng, (n, m), kind) if residual else (None, None)
    y = torch.full((n, m), NAN, dtype=R.TYPES[kind], device=gpu)
    eg2.ops.linear(x.to(gpu), w, y, bias=torch.from_numpy(b).to(gpu) if bias else None, act=act,
                   residual=r.to(gpu) if residual else None)
    near(y, *R.linear(x64, w64, b, act, r64, R.TYPES[kind]))


@pytest.mark.parametrize("pair", PAIRS, ids="-".join)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_linear(eg2, gpu, pair, shape):
    rng = np.random.default_rng(sum(shape))
    run_linear(eg2, gpu, rng, pair, shape, act=["none", "gelu", "silu", "relu"][sum(shape) % 4])


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", [(1, 1, 1), (3, 7, 5), (1, 1150, 769), (70, 33, 65), (67, 1150, 130), (129, 71, 131),
                                   (40, 1151, 77), (300, 516, 258)], ids=str)
def test_linear_odd_sizes(eg2, gpu, kind, shape):
    run_linear(eg2, gpu, np.random.default_rng(shape[1]), (kind, kind), shape, act="silu")


@pytest.mark.parametrize("pair", [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("bf16", "q8_0")], ids="-".join)
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("act", ["none", "gelu", "silu", "relu"])
def test_linear_epilogues(eg2, gpu, pair, bias, residual, act):
    for shape in ((3, 64, 40), (70, 64, 130)):
        run_linear(eg2, gpu, np.random.default_rng(5), pair, shape, act, bias, residual)


@pytest.mark.parametrize("pair", PAIRS, ids="-".join)
@pytest.mark.parametrize("shape", [(1, 64, 33), (5, 2048, 96), (33, 160, 257), (130, 800, 200), (260, 128, 300)], ids=str)
def test_linear_gated(eg2, gpu, pair, shape):
    rng = np.random.default_rng(sum(shape) + 1)
    (kind, wkind), (n, k, m) = pair, shape
    x, x64 = rnd(rng, (n, k), kind)
    (g, g64), (u, u64) = weights(rng, m, k, wkind, gpu), weights(rng, m, k, wkind, gpu)
    for act, bias in (("gelu", True), ("silu", False), ("relu", True), ("none", False)):
        gb, ub = (rng.standard_normal(m).astype(np.float32) if bias else None for _ in range(2))
        y = torch.full((n, m), NAN, dtype=R.TYPES[kind], device=gpu)
        eg2.ops.linear_gated(x.to(gpu), g, u, y, act=act, gate_bias=torch.from_numpy(gb).to(gpu) if bias else None,
                             up_bias=torch.from_numpy(ub).to(gpu) if bias else None)
        near(y, *R.linear_gated(x64, g64, u64, gb, ub, act, R.TYPES[kind]))


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n", [3, 65])
@pytest.mark.parametrize("pad", [1, 2, 8])
def test_products_with_strides_write_nothing_beside(eg2, gpu, kind, n, pad):
    """Every operand is the middle of a larger buffer of NaN, at each alignment."""
    rng = np.random.default_rng(n + pad)
    k, m = 96, 70
    (x, x64), (w, w64), (r, r64) = rnd(rng, (n, k), kind), rnd(rng, (m, k), kind, 0.1), rnd(rng, (n, m), kind)
    xv, _ = inside(x, gpu, pad)
    wv, _ = inside(w, gpu, pad)
    rv, _ = inside(r, gpu, pad)
    yv, buf = inside(torch.zeros((n, m), dtype=x.dtype), gpu, pad)
    eg2.ops.linear(xv, wv, yv, residual=rv)
    near(yv, *R.linear(x64, w64, None, "none", r64, x.dtype))
    yv.fill_(NAN)
    assert torch.isnan(buf).all()
    eg2.ops.linear_gated(xv, wv, wv, yv, act="silu")
    near(yv, *R.linear_gated(x64, w64, w64, None, None, "silu", x.dtype))
    yv.fill_(NAN)
    assert torch.isnan(buf).all()
    # one row of x for every row of y, and the residual in place
    one = xv[:1].expand(n, k)
    acc = rv.clone()
    eg2.ops.linear(one, wv, acc, residual=acc)
    near(acc, *R.linear(np.repeat(x64[:1], n, 0), w64, None, "none", r64, x.dtype))


def test_q8_rows_apart(eg2, gpu):
    """Q8_0 rows inside wider rows of blocks, that start on 2 bytes only."""
    rng = np.random.default_rng(8)
    for kind in ("f32", "f16", "bf16"):
        for n in (3, 70):
            raw, values = R.quantize((rng.standard_normal((50, 160)) * 0.1).astype(np.float32))
            buf = torch.full((50 * 34 * 7 + 2,), 0x7f, dtype=torch.uint8, device=gpu)
            view = buf[2:].view(50, 34 * 7)[:, 34:34 * 6]
            view.copy_(torch.from_numpy(raw))
            x, x64 = rnd(rng, (n, 160), kind)
            y = torch.empty((n, 50), dtype=x.dtype, device=gpu)
            eg2.ops.linear(x.to(gpu), view, y)
            near(y, *R.linear(x64, values, None, "none", None, x.dtype))


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n", [4, 70])
def test_non_finite_operands_stay_in_their_rows_and_columns(eg2, gpu, kind, n):
    rng = np.random.default_rng(11)
    k, m = 100, 70
    (x, x64), (w, w64) = rnd(rng, (n, k), kind), rnd(rng, (m, k), kind, 0.1)
    x[1, 5], w[3, 7], w[60, 99] = float("inf"), NAN, float("-inf")
    y = torch.empty((n, m), dtype=x.dtype, device=gpu)
    eg2.ops.linear(x.to(gpu), w.to(gpu), y)
    want = x.double() @ w.double().t()
    got = y.cpu().double()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf])
    clean = np.ones((n, m), bool)
    clean[1], clean[:, 3], clean[:, 60] = False, False, False
    want, off = R.linear(np.nan_to_num(x64), np.nan_to_num(w64), None, "none", None, x.dtype)
    assert (np.abs(got.numpy() - want) <= off)[clean].all()


def test_activations_over_their_range(eg2, gpu):
    """x = 1 weight each: the activation of every value, to the bounds of one product."""
    z = np.concatenate([np.linspace(-30, 30, 4001), [-1e4, -200.0, -88.0, 88.0, 200.0, 1e4, 0.0]]).astype(np.float32)
    x = torch.from_numpy(z[:, None].copy()).to(gpu)
    w = torch.ones((1, 1), device=gpu)
    for act in ("gelu", "silu", "relu", "none"):
        y = torch.empty((len(z), 1), device=gpu)
        eg2.ops.linear(x, w, y, act=act)
        z64 = z.astype(np.float64)
        with np.errstate(over="ignore"):
            want = R.activation(z64, act)
        # t = the argument of exp: off by 4 u |t|, where the result is not below 2^-100; exp, the sum and the quotient 4 u
        t = np.abs(2 * 0.8 * (z64 + 0.044715 * z64 ** 3))
        off = np.abs(want) * (4 * np.minimum(t, 100) + 8) * R.U + 2.0 ** -100
        assert (np.abs(y[:, 0].double().cpu().numpy() - want) <= off).all(), act


def test_rows_do_not_depend_on_the_others(eg2, gpu):
    """An output's bits follow from its own row and column."""
    rng = np.random.default_rng(4)
    for kind in ("f32", "bf16"):
        for n in (6, 200):
            x, _ = rnd(rng, (n, 320), kind)
            w, _ = rnd(rng, (200, 320), kind)
            y, z = (torch.empty((n, 200), dtype=x.dtype, device=gpu) for _ in range(2))
            eg2.ops.linear(x.to(gpu), w.to(gpu), y)
            x[1:], w[:150] = 1e30 if kind == "bf16" else NAN, 0.0
            eg2.ops.linear(x.to(gpu), w.to(gpu), z)
            assert torch.equal(y[0, 150:], z[0, 150:])


# ------------------------------------------------------------------ heads

def angles(rotary, positions=700):
    t = np.arange(positions)[:, None] * 1e4 ** (-np.arange(rotary // 2) * 2 / max(rotary, 1))[None]
    return np.concatenate([np.cos(t), np.sin(t)], 1).astype(np.float32)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("geometry", [(3, 1, 256, 256), (4, 2, 128, 64), (1, 0, 64, 64), (16, 4, 128, 128), (2, 2, 80, 80),
                                      (3, 1, 2, 2), (1, 1, 6, 4), (2, 1, 512, 512), (1, 1, 510, 254), (5, 1, 96, 0)], ids=str)
@pytest.mark.parametrize("rows", [1, 37])
def test_heads_norm_rope(eg2, gpu, kind, geometry, rows):
    heads, kv, d, rotary = geometry
    rng = np.random.default_rng(d + rows)
    x, x64 = rnd(rng, (rows, (heads + kv) * d), kind, 3.0)
    qw, kw = (rng.standard_normal(d).astype(np.float32) for _ in range(2))
    table, pos = (angles(rotary), rng.integers(0, 700, rows).astype(np.int32)) if rotary else (None, None)
    for shift in (0, 1):  # the second time off every alignment
        buf = torch.full((rows, (heads + kv) * d + 8 + shift), NAN, dtype=x.dtype, device=gpu)
        view = buf[:, shift:shift + x.shape[1]]
        view.copy_(x)
        q, k = view[:, :heads * d].unflatten(1, (heads, d)), None
        k_out = None
        if kv:
            k = view[:, heads * d:].unflatten(1, (kv, d))
            k_out = k if shift else torch.empty((rows, kv, d), dtype=x.dtype, device=gpu)
        q_out = torch.empty((rows, heads, d), dtype=x.dtype, device=gpu)
        eg2.ops.heads_norm_rope(q, k, torch.from_numpy(qw).to(gpu), torch.from_numpy(kw).to(gpu) if kv and shift else None,
                                torch.from_numpy(table).to(gpu) if rotary else None,
                                torch.from_numpy(pos).to(gpu) if rotary else None, 1e-6, q_out, k_out, q_scale=0.0625)
        q64, k64 = x64[:, :heads * d].reshape(rows, heads, d), x64[:, heads * d:].reshape(rows, kv, d)
        t64 = table.astype(np.float64) if rotary else None
        near(q_out, *R.heads_norm_rope(q64, qw, t64, pos, 1e-6, 0.0625, x.dtype))
        if kv:
            near(k_out, *R.heads_norm_rope(k64, kw if shift else None, t64, pos, 1e-6, 1.0, x.dtype))
        assert torch.isnan(buf[:, shift + x.shape[1]:]).all()


def test_heads_with_unknown_positions_are_nan(eg2, gpu):
    q = torch.randn(4, 2, 64, device=gpu)
    k = torch.randn(4, 1, 64, device=gpu)
    pos = torch.tensor([0, -1, 700, 699], dtype=torch.int32, device=gpu)
    qo, ko = torch.zeros_like(q), torch.zeros_like(k)
    eg2.ops.heads_norm_rope(q, k, None, None, torch.from_numpy(angles(64)).to(gpu), pos, 1e-6, qo, ko)
    for t in (qo, ko):
        assert torch.isnan(t[1:3]).all() and torch.isfinite(t[[0, 3]]).all()


def test_heads_of_zeros_and_of_nan(eg2, gpu):
    """A head of zeros stays zero; a NaN stays in its head."""
    q = torch.randn(3, 2, 128, device=gpu).bfloat16()
    q[0, 0] = 0.0
    q[1, 1, 7] = NAN
    out = torch.empty_like(q)
    eg2.ops.heads_norm_rope(q, None, None, None, torch.from_numpy(angles(128)).to(gpu),
                            torch.arange(3, dtype=torch.int32, device=gpu), 1e-6, out, None)
    assert (out[0, 0] == 0).all() and torch.isnan(out[1, 1]).all()
    assert torch.isfinite(out[[0, 2]]).all() and torch.isfinite(out[1, 0]).all()


# ------------------------------------------------------------------ attention

def attention_case(rng, kind, q_lens, k_lens, heads, kv, d, cap=None):
    """Host tensors, their 64-bit values and the offsets; cap: a cache of cap rows a sequence."""
    rows, key_rows = sum(q_lens), cap * len(k_lens) if cap else sum(k_lens)
    q, k, v = rnd(rng, (rows, heads, d), kind), rnd(rng, (key_rows, kv, d), kind), rnd(rng, (key_rows, kv, d), kind)
    qo = np.concatenate([[0], np.cumsum(q_lens)]).astype(np.int32)
    ko = (np.arange(len(k_lens) + 1) * cap if cap else np.concatenate([[0], np.cumsum(k_lens)])).astype(np.int32)
    return q, k, v, qo, ko, np.array(k_lens, np.int32) if cap else None


def run_attention(eg2, gpu, q, k, v, qo, ko, kl, scale, left, right, sinks, longest=0, **more):
    dev = lambda a: None if a is None else torch.from_numpy(np.ascontiguousarray(a)).to(gpu)  # noqa: E731
    out = torch.full(q.shape, 77.0, dtype=q.dtype, device=gpu)
    eg2.ops.window_attention(q.to(gpu), k.to(gpu), v.to(gpu), dev(qo), dev(ko), out, scale, left, right, sinks,
                             k_lengths=dev(kl), longest=longest, **more)
    return out


def check_attention(eg2, gpu, case, kind, left, right, sinks, longest=0):
    (q, q64), (k, k64), (v, v64), qo, ko, kl = case
    scale = q.shape[2] ** -0.5
    got = run_attention(eg2, gpu, q, k, v, qo, ko, kl, scale, left, right, sinks, longest)
    near(got, *R.window_attention(q64, k64, v64, qo, ko, scale, left, right, sinks, kl, R.TYPES[kind]))


WINDOWS = [(-1, -1, 0), (-1, 0, 0), (5, 5, 0), (5, 5, 3), (20, 0, 4), (0, 0, 0), (0, 0, 1), (64, -1, 2), (-1, 3, 0)]


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("geometry", [(3, 1, 256), (4, 2, 64), (2, 2, 80), (4, 1, 128)], ids=str)
@pytest.mark.parametrize("window", WINDOWS, ids=str)
def test_attention_packed(eg2, gpu, kind, geometry, window):
    rng = np.random.default_rng(geometry[2] + window[0])
    lens = [1, 33, 0, 70, 16, 5]
    check_attention(eg2, gpu, attention_case(rng, kind, lens, lens, *geometry), kind, *window)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d", [8, 16, 24, 40, 72, 96, 136, 192, 200, 248])
def test_attention_head_sizes(eg2, gpu, kind, d):
    rng = np.random.default_rng(d)
    check_attention(eg2, gpu, attention_case(rng, kind, [3, 40], [50, 40], 3, 1, d), kind, 30, 2, 2)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("window", [(-1, 0, 0), (100, 0, 4), (3, 0, 16), (0, 0, 0), (700, 2, 1)], ids=str)
@pytest.mark.parametrize("heads", [(16, 4, 128), (3, 1, 256), (7, 1, 64), (8, 8, 80), (40, 1, 64)], ids=str)
def test_attention_single_tokens_over_caches(eg2, gpu, kind, window, heads):
    """One query each; caches that hold none, one, a few and many keys; with and without the hint."""
    rng = np.random.default_rng(heads[2])
    lens = [1, 0, 5, 64, 333, 600]
    case = attention_case(rng, kind, [1] * 6, lens, *heads, cap=601)
    for longest in (0, 600, 100000):
        check_attention(eg2, gpu, case, kind, *window, longest=longest)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("window", [(-1, 0, 0), (50, 0, 4), (4, 4, 0)], ids=str)
def test_attention_more_or_fewer_queries_than_keys(eg2, gpu, kind, window):
    """Prompts in pieces over a cache; queries before the first key see nothing (causal) and come out as 0."""
    rng = np.random.default_rng(3)
    check_attention(eg2, gpu, attention_case(rng, kind, [20, 9, 130, 3, 1], [150, 9, 40, 0, 3], 4, 2, 64), kind, *window)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_attention_long_split(eg2, gpu, kind):
    """Many keys for few rows, split over the GPU and joined."""
    rng = np.random.default_rng(9)
    case = attention_case(rng, kind, [1, 2], [5000, 3111], 4, 2, 128)
    for window in ((-1, 0, 0), (1000, 0, 4), (4000, 0, 300)):
        check_attention(eg2, gpu, case, kind, *window, longest=5000)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("q_len", [1, 40])
def test_attention_hidden_places_may_hold_anything(eg2, gpu, kind, q_len):
    """NaN and infinities behind a sequence's keys, in keys that no row sees, and in one
    that only some rows see: those are NaN, the others as if it were not there."""
    rng = np.random.default_rng(12)
    (q, q64), (k, k64), (v, v64), qo, ko, kl = attention_case(rng, kind, [q_len] * 2, [100, 77], 4, 2, 64, cap=128)
    left, right, sinks = 20, 0, 2
    plain = R.window_attention(q64, k64, v64, qo, ko, 0.125, left, right, sinks, kl, q.dtype)
    for b, n in enumerate((100, 77)):
        for t in (k, v):
            t[128 * b + n:128 * (b + 1)] = NAN  # behind the keys
            t[128 * b + 2:128 * b + n - q_len - 20] = float("inf")  # before every window, after the sinks
    near(run_attention(eg2, gpu, q, k, v, qo, ko, kl, 0.125, left, right, sinks, 100), *plain)
    if q_len > 1:
        for value in (NAN, float("inf")):
            for t, other in ((k, v), (v, k)):
                keep = t[70].clone()
                t[70, 0] = value  # key 70 of sequence 0: seen by the queries at 70 .. 90 of heads 0 and 1
                got = run_attention(eg2, gpu, q, k, v, qo, ko, kl, 0.125, left, right, sinks, 100)
                t[70] = keep
                sees = np.zeros(plain[0].shape, bool)
                sees[10:31, :2] = True
                g = got.double().cpu().numpy()
                assert (np.abs(g - plain[0]) <= plain[1])[~sees].all(), (value, t is k)
                if value != value:
                    assert np.isnan(g)[10:31, :2].all(), t is k


def test_attention_rows_outside_every_sequence_are_left(eg2, gpu):
    rng = np.random.default_rng(2)
    for kind in ("f32", "bf16"):
        (q, q64), (k, k64), (v, v64), qo, ko, kl = attention_case(rng, kind, [7, 30, 9], [7, 30, 9], 2, 1, 64)
        qo = np.array([7, 37], np.int32)  # the middle one alone
        got = run_attention(eg2, gpu, q, k, v, qo, ko[1:3], None, 0.1, 4, 4, 1)
        assert (got[:7] == 77).all() and (got[37:] == 77).all()
        want, off = R.window_attention(q64, k64, v64, qo, ko[1:3], 0.1, 4, 4, 1, None, q.dtype)
        near(got[7:37], want[7:37], off[7:37])


def test_attention_offsets_past_the_buffers_are_clipped(eg2, gpu):
    """Offsets and lengths that claim more rows than there are: only the rows there are are read and written."""
    rng = np.random.default_rng(6)
    (q, q64), (k, k64), (v, v64), _, _, _ = attention_case(rng, "f32", [40], [60], 2, 1, 64)
    got = run_attention(eg2, gpu, q, k, v, np.array([0, 100], np.int32), np.array([-5, 4000], np.int32),
                        np.array([5000], np.int32), 0.125, 8, 0, 1)
    near(got, *R.window_attention(q64, k64, v64, [0, 40], [0, 60], 0.125, 8, 0, 1, None, q.dtype))


def test_attention_strides(eg2, gpu):
    """q, k and v as parts of fused rows, heads before rows, and a K/V head shared by every sequence row."""
    rng = np.random.default_rng(7)
    for kind in ("f32", "f16", "bf16"):
        for lens in ([50], [1, 1, 1]):
            (q, q64), (k, k64), (v, v64), qo, ko, _ = attention_case(rng, kind, lens, lens, 4, 2, 64)
            rows = q.shape[0]
            fused = torch.full((rows, 10, 64), NAN, dtype=q.dtype, device=gpu)
            fused[:, 1:5], fused[:, 5:7], fused[:, 7:9] = q, k, v
            out = torch.full((4, rows, 72), 77.0, dtype=q.dtype, device=gpu)
            view = out[:, :, :64].transpose(0, 1)
            off = torch.from_numpy(qo).to(gpu)
            eg2.ops.window_attention(fused[:, 1:5], fused[:, 5:7], fused[:, 7:9], off, off, view, 0.125, 9, 0, 2)
            near(view, *R.window_attention(q64, k64, v64, qo, qo, 0.125, 9, 0, 2, None, q.dtype))
            assert (out[:, :, 64:] == 77).all()


def test_attention_large_scores(eg2, gpu):
    """Scores of thousands: the maximum is taken out before exp."""
    rng = np.random.default_rng(5)
    for kind in ("f32", "bf16"):
        (q, q64), (k, k64), (v, v64), qo, ko, _ = attention_case(rng, kind, [33], [33], 2, 1, 64)
        # one key per row far above the rest: q = 40 k
        q = (k * 40).expand(-1, 2, -1).contiguous()
        q64 = q.double().numpy()
        got = run_attention(eg2, gpu, q, k, v, qo, ko, None, 1.0, -1, -1, 0)
        want, _ = R.window_attention(q64, k64, v64, qo, ko, 1.0, -1, -1, 0, None, q.dtype)
        # the weights beside the largest are below e^-100: every row is its own value
        assert np.abs(want - np.repeat(v64, 2, 1)).max() < 1e-30
        near(got, want, R.rounding(want, q.dtype) + 8 * R.U * np.abs(want))


# ------------------------------------------------------------------ streams, graphs, together

def block(eg2, s):
    """One pre-norm transformer block by the package's operators: the fp32 row norm by name, the rest by these."""
    o, E = eg2.ops, eg2
    n = s["x"].shape[0]
    o.op("eg2_norm", E.EgNorm(s["h"].data_ptr(), s["x"].data_ptr(), s["norm1"].data_ptr(), n, 192, 1.0), n, 64)
    s["h16"].copy_(s["h"])
    o.linear(s["h16"], s["w_qkv"], s["qkv"], bias=s["b_qkv"])
    heads = s["qkv"].view(n, 5, 64)
    o.heads_norm_rope(heads[:, :3], heads[:, 3:4], s["qn"], s["kn"], s["table"], s["pos"], 1e-6, heads[:, :3],
                      heads[:, 3:4], q_scale=0.125)
    o.window_attention(heads[:, :3], heads[:, 3:4], heads[:, 4:5], s["off"], s["off"], s["a"], 1.0, left=16, right=16,
                       sinks=2, workspace=s["ws"])
    o.linear(s["a"].view(n, 192), s["w_o"], s["y16"], residual=s["x16"])
    s["y"].copy_(s["y16"])
    o.op("eg2_norm", E.EgNorm(s["h"].data_ptr(), s["y"].data_ptr(), s["norm2"].data_ptr(), n, 192, 1.0), n, 64)
    s["h16"].copy_(s["h"])
    o.linear_gated(s["h16"], s["w_g"], s["w_u"], s["f"])
    o.linear(s["f"], s["w_d"], s["y16"], residual=s["y16"])


def block_state(eg2, gpu, kind, lens, seed):
    rng = np.random.default_rng(seed)
    n, dt = sum(lens), R.TYPES[kind]
    t = lambda a: torch.from_numpy(a.astype(np.float32)).to(gpu)  # noqa: E731
    w = lambda m, k: (t(rng.standard_normal((m, k)) / np.sqrt(k))).to(dt)  # noqa: E731
    s = {"x": t(rng.standard_normal((n, 192))), "norm1": t(1 + 0.1 * rng.standard_normal(192)),
         "norm2": t(1 + 0.1 * rng.standard_normal(192)), "qn": t(1 + 0.1 * rng.standard_normal(64)),
         "kn": t(1 + 0.1 * rng.standard_normal(64)), "table": torch.from_numpy(angles(64)).to(gpu),
         "w_qkv": w(320, 192), "b_qkv": t(0.1 * rng.standard_normal(320)), "w_o": w(192, 192), "w_g": w(320, 192),
         "w_u": w(320, 192), "w_d": w(192, 320)}
    s["x16"] = s["x"].to(dt)
    s["x"] = s["x16"].float()
    s["pos"] = torch.from_numpy(np.concatenate([np.arange(x) for x in lens]).astype(np.int32)).to(gpu)
    s["off"] = torch.from_numpy(np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)).to(gpu)
    s["h"], s["y"] = torch.empty_like(s["x"]), torch.empty_like(s["x"])
    for name, cols in (("h16", 192), ("qkv", 320), ("y16", 192), ("f", 320)):
        s[name] = torch.empty((n, cols), dtype=dt, device=gpu)
    s["a"] = torch.empty((n, 3, 64), dtype=dt, device=gpu)
    need = eg2.ops.window_attention_workspace(len(lens), n, n, 3, 1, 64, dt, 16, 16, 2)
    s["ws"] = torch.empty(max(16, need), dtype=torch.uint8, device=gpu)
    return s


def block_reference(s, lens, dt):
    """The block in 64 bits, rounded to dt where the operators hand over."""
    r = lambda a: torch.from_numpy(a).to(dt).double().numpy()  # noqa: E731
    d = lambda name: s[name].double().cpu().numpy()  # noqa: E731
    norm = lambda x, w: r(x / np.sqrt((x * x).mean(1, keepdims=True) + 1e-6) * w)  # noqa: E731
    x, t64, pos = d("x16"), d("table"), s["pos"].cpu().numpy()
    qkv = r(R.linear(norm(x, d("norm1")), d("w_qkv"), d("b_qkv"), "none", None, dt)[0]).reshape(-1, 5, 64)
    q = r(R.heads_norm_rope(qkv[:, :3], d("qn"), t64, pos, 1e-6, 0.125, dt)[0])
    k = r(R.heads_norm_rope(qkv[:, 3:4], d("kn"), t64, pos, 1e-6, 1.0, dt)[0])
    off = s["off"].cpu().numpy()
    a = r(R.window_attention(q, k, qkv[:, 4:5], off, off, 1.0, 16, 16, 2, None, dt)[0]).reshape(-1, 192)
    y = r(R.linear(a, d("w_o"), None, "none", x, dt)[0])
    f = r(R.linear_gated(norm(y, d("norm2")), d("w_g"), d("w_u"), None, None, "gelu", dt)[0])
    return R.linear(f, d("w_d"), None, "none", y, dt)[0]


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_a_whole_block(eg2, gpu, kind):
    lens = [1, 40, 7, 90]
    s = block_state(eg2, gpu, kind, lens, 1)
    block(eg2, s)
    want = block_reference(s, lens, R.TYPES[kind])
    # Ten hand-overs, each rounded to the type (half a step) and passed on with a gain of about 1:
    # ten half steps, doubled for what the norms and the gate add, of the row's rms (in 2-norm).
    err = np.linalg.norm(s["y16"].double().cpu().numpy() - want) / np.linalg.norm(want)
    assert err <= max(20 * torch.finfo(R.TYPES[kind]).eps / 2, 1e-5), err


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_a_captured_block_replays(eg2, gpu, kind):
    lens = [1, 40, 7, 90]
    s, other = block_state(eg2, gpu, kind, lens, 1), block_state(eg2, gpu, kind, lens, 2)
    block(eg2, s)
    block(eg2, other)
    want = [s["y16"].clone(), other["y16"].clone()]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        block(eg2, s)
    first = {name: s[name].clone() for name in ("x", "x16", "w_qkv", "b_qkv", "w_o", "w_g", "w_u", "w_d", "norm1", "norm2",
                                                  "qn", "kn")}
    for turn in range(4):
        for name in first:
            s[name].copy_((other if turn % 2 else first)[name])
        s["y16"].fill_(NAN)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(s["y16"], want[turn % 2]), turn
        block(eg2, other)  # eager work of its own between the replays
        torch.cuda.synchronize()
        assert torch.equal(other["y16"], want[1])


def test_two_streams_at_once(eg2, gpu):
    """The same calls on two streams, each with its own buffers, give what they give alone."""
    lens = [1, 40, 7, 90]
    states = [block_state(eg2, gpu, "bf16", lens, seed) for seed in (1, 2)]
    for s in states:
        block(eg2, s)
    want = [s["y16"].clone() for s in states]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in states]
    for _ in range(3):
        for s, st in zip(states, streams):
            with torch.cuda.stream(st):
                block(eg2, s)
    torch.cuda.synchronize()
    for s, w in zip(states, want):
        assert torch.equal(s["y16"], w)
