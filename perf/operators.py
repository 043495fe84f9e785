"""The floating-point operators of a transformer block, timed and compared
with their plain form: products with an epilogue (`linear`), the gated half
of a feed-forward block (`linear_gated`), the norms of queries and keys with
the rotation (`heads_norm_rope`), and attention over a sliding window and a
few first keys (`window_attention`).

With `own` false every operator is computed by elementary torch operations in
32 bits and rounded once; with `own` true by the calls of the package's
binding. Sizes are those of the two models of this repository (768 / 1152
wide with 3 query heads and one KV head of 256; 512 / 2048 wide with 4) and
generic ones.
"""
import importlib.util
import math
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
EPS = 1e-6
own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2, "q8_0": 34 / 32}


def _package():
    if "eg2hip" not in sys.modules:
        path = os.path.join(ROOT, "embeddinggemma2-amdkfd_amd", "eg2hip.py")
        spec = importlib.util.spec_from_file_location("eg2hip", path)
        mod = importlib.util.module_from_spec(spec)
        sys.modules["eg2hip"] = mod
        spec.loader.exec_module(mod)
    return sys.modules["eg2hip"]


# ------------------------------------------------------------------ the cases

def listed():
    return [
        # One token through a square projection of the 768-wide model: nothing but latency.
        {"name": "linear 1x768x768 bf16", "op": "linear", "type": "bf16", "weights": "bf16", "n": 1, "k": 768,
         "m": 768, "bias": True, "act": "none", "residual": True},
        # A short text through the 300M model's Q|K|V matrix as the file holds it (Q8_0), 32-bit activations.
        {"name": "linear 45x768x1280 q8_0", "op": "linear", "type": "f32", "weights": "q8_0", "n": 45, "k": 768,
         "m": 1280, "bias": False, "act": "none", "residual": False},
        # A ragged batch through the down projection, with sizes that fit no tile.
        {"name": "linear 333x1150x769 f16", "op": "linear", "type": "f16", "weights": "f16", "n": 333, "k": 1150,
         "m": 769, "bias": True, "act": "silu", "residual": True},
        # A long prompt through a wide projection: the largest product.
        {"name": "linear 4096x2048x8192 bf16", "op": "linear", "type": "bf16", "weights": "bf16", "n": 4096,
         "k": 2048, "m": 8192, "bias": True, "act": "gelu", "residual": False},
        # The 300M model's gate and up projections over a full wave.
        {"name": "gated 2048x768x1152 bf16", "op": "gated", "type": "bf16", "weights": "bf16", "n": 2048, "k": 768,
         "m": 1152, "bias": False, "act": "gelu"},
        # A few single tokens of running sequences through a wide gated block with Q8_0 weights: the weights' bytes.
        {"name": "gated 4x2048x8192 q8_0", "op": "gated", "type": "bf16", "weights": "q8_0", "n": 4, "k": 2048,
         "m": 8192, "bias": False, "act": "silu"},
        # Queries and keys of the 300M model inside its fused Q|K|V rows, an almost full wave.
        {"name": "norm_rope 2011 3+1x256 f32", "op": "norm_rope", "type": "f32", "rows": 2011, "heads": 3,
         "kv_heads": 1, "d": 256, "rotary": 256},
        # A long prompt's heads of 128.
        {"name": "norm_rope 8192 16+4x128 bf16", "op": "norm_rope", "type": "bf16", "rows": 8192, "heads": 16,
         "kv_heads": 4, "d": 128, "rotary": 128},
        # Nine texts in one wave on a sliding-window layer of the 300M model, 32-bit.
        {"name": "attention 9 texts f32", "op": "attention", "type": "f32", "batch": 9, "queries": 113, "keys": 0,
         "ragged": True, "heads": 3, "kv_heads": 1, "d": 256, "left": 256, "right": 256, "sinks": 1},
        # Sixteen texts of 128 on the same layer, 16-bit: the bulk indexer's wave.
        {"name": "attention 16 texts bf16", "op": "attention", "type": "bf16", "batch": 16, "queries": 128, "keys": 0,
         "ragged": False, "heads": 3, "kv_heads": 1, "d": 256, "left": 256, "right": 256, "sinks": 1},
        # One long prompt, causal, a window of half of it and four first tokens that stay visible.
        {"name": "attention causal 8192 bf16", "op": "attention", "type": "bf16", "batch": 1, "queries": 8192,
         "keys": 0, "ragged": False, "heads": 16, "kv_heads": 4, "d": 128, "left": 4095, "right": 0, "sinks": 4},
        # One token each of 24 running sequences over their caches.
        {"name": "attention decode 24 bf16", "op": "attention", "type": "bf16", "batch": 24, "queries": 1,
         "keys": 6000, "ragged": True, "heads": 16, "kv_heads": 4, "d": 128, "left": 2047, "right": 0, "sinks": 4},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["linear", "linear", "gated", "norm_rope", "attention", "attention", "attention"])
    kind = rng.choice(["f32", "f16", "bf16", "bf16"])
    if op in ("linear", "gated"):
        weights = rng.choice([kind, kind, "q8_0"] + (["f16", "bf16"] if kind == "f32" else []))
        n, k, m = _log_int(rng, 1, 4096), _log_int(rng, 64, 4096), _log_int(rng, 64, 8192)
        if weights == "q8_0":
            k = max(64, k // 32 * 32)
        elif rng.random() < 0.6:
            k, m = max(64, k // 64 * 64), max(64, m // 64 * 64)
        # no more operations than the largest listed product (32-bit ones: an eighth)
        cap = 4096 * 2048 * 8192 // (2 if op == "gated" else 1) // (8 if kind == "f32" else 1)
        n = max(1, min(n, cap // (k * m)))
        case = {"op": op, "type": kind, "weights": weights, "n": n, "k": k, "m": m, "bias": rng.random() < 0.5,
                "act": rng.choice(["none", "gelu", "silu", "relu"])}
        if op == "linear":
            case["residual"] = rng.random() < 0.5
        return case
    heads, kv_heads = rng.choice([(3, 1), (4, 2), (4, 1), (8, 8), (16, 4), (7, 1), (32, 8)])
    if op == "norm_rope":
        d = rng.choice([64, 80, 128, 256])
        return {"op": op, "type": kind, "rows": _log_int(rng, 1, 8192 * 20 * 128 // ((heads + kv_heads) * d)),
                "heads": heads, "kv_heads": kv_heads, "d": d, "rotary": rng.choice([d, d, d // 2])}
    d = rng.choice([64, 80, 128, 256])
    form = rng.choice(["texts", "causal", "chunk", "decode"])
    left, sinks = rng.choice([64, 127, 511, 1000, 2047]), rng.choice([0, 1, 4, 16])
    right = left if form == "texts" else 0
    if form == "decode":
        batch, keys = _log_int(rng, 1, 48), _log_int(rng, 64, 8192)
        return {"op": op, "type": kind, "batch": batch, "queries": 1, "keys": keys, "ragged": True, "heads": heads,
                "kv_heads": kv_heads, "d": d, "left": rng.choice([left, -1]), "right": 0, "sinks": sinks}
    batch = 1 if form == "chunk" else _log_int(rng, 1, 16)
    most = min(4096, int(math.sqrt(8192 * 8192 * 16 * 128 / (heads * d * batch * (16 if kind == "f32" else 1)))))
    queries = _log_int(rng, min(16, most), most)
    return {"op": op, "type": kind, "batch": batch, "queries": queries,
            "keys": min(4096, queries + _log_int(rng, 1, 2048)) if form == "chunk" else 0, "ragged": batch > 1,
            "heads": heads, "kv_heads": kv_heads, "d": d, "left": left, "right": right, "sinks": sinks}


def _lengths(case):
    """Queries and keys of each sequence: ragged ones alternate between a third and the whole."""
    b = case["batch"]
    share = [1.0 if not case["ragged"] else 1.0 - (i * 5 % 9) / 13 for i in range(b)]
    q = [case["queries"] if case["keys"] else max(1, int(case["queries"] * s)) for s in share]
    k = [max(case["queries"], int(case["keys"] * s)) for s in share] if case["keys"] else q
    return q, k


# ------------------------------------------------------------------ inputs

def _q8_blocks(g, m, k):
    """[m, 34 k / 32] bytes of Q8_0 blocks: the little-endian fp16 scale, then 32 int8 values."""
    scale = ((torch.rand((m, k // 32, 1), generator=g, device="cuda") + 0.5) / (73.0 * math.sqrt(k))).half()
    values = torch.randint(-127, 128, (m, k // 32, 32), generator=g, device="cuda", dtype=torch.int8)
    return torch.cat([scale.view(torch.uint8), values.view(torch.uint8)], 2).reshape(m, k // 32 * 34).contiguous()


def _weights(g, case, m, k):
    if case["weights"] == "q8_0":
        return _q8_blocks(g, m, k)
    return (torch.randn((m, k), generator=g, device="cuda") / math.sqrt(k)).to(TYPES[case["weights"]])


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt = TYPES[case["type"]]

    def randn(*shape, scale=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * scale).to(dt)

    s = dict(case)
    if case["op"] in ("linear", "gated"):
        n, k, m = case["n"], case["k"], case["m"]
        s["x"] = randn(n, k)
        names = ["w"] if case["op"] == "linear" else ["w", "up"]
        s.update({name: _weights(g, case, m, k) for name in names})
        s.update({name + "_bias": torch.randn((m,), generator=g, device="cuda") * 0.1 if case["bias"] else None
                  for name in names})
        s["r"] = randn(n, m) if case.get("residual") else None
        s["y"] = torch.empty((n, m), dtype=dt, device="cuda")
        return s
    heads, kv_heads, d = case["heads"], case["kv_heads"], case["d"]
    if case["op"] == "norm_rope":
        rows, rotary = case["rows"], case["rotary"]
        qkv = randn(rows, (heads + 2 * kv_heads) * d)  # q and k are parts of the fused projection's rows
        s["q"] = qkv[:, :heads * d].view(rows, heads, d)
        s["k"] = qkv[:, heads * d:(heads + kv_heads) * d].view(rows, kv_heads, d)
        s["q_w"], s["k_w"] = (1.0 + 0.1 * torch.randn((d,), generator=g, device="cuda") for _ in range(2))
        table = torch.arange(8192, device="cuda", dtype=torch.float64)[:, None] * \
            1e4 ** (-torch.arange(rotary // 2, device="cuda", dtype=torch.float64) * 2 / rotary)[None]
        s["table"] = torch.cat([table.cos(), table.sin()], 1).float()
        s["pos"] = torch.randint(0, 8192, (rows,), generator=g, device="cuda", dtype=torch.int32)
        s["q_out"], s["k_out"] = torch.empty_like(s["q"]).contiguous(), torch.empty_like(s["k"]).contiguous()
        return s
    q_len, k_len = _lengths(case)
    cached = case["keys"] > 0
    cap = max(k_len)
    rows, key_rows = sum(q_len), cap * case["batch"] if cached else sum(k_len)
    s["q"] = randn(rows, heads, d)
    s["k"], s["v"] = randn(key_rows, kv_heads, d), randn(key_rows, kv_heads, d)
    ints = {"dtype": torch.int32, "device": "cuda"}
    s["q_offsets"] = torch.tensor([sum(q_len[:i]) for i in range(len(q_len) + 1)], **ints)
    if cached:  # a cache of `cap` rows a sequence, of which each holds its own number
        s["k_offsets"] = torch.tensor([cap * i for i in range(len(k_len) + 1)], **ints)
        s["k_lengths"] = torch.tensor(k_len, **ints)
    else:
        s["k_offsets"], s["k_lengths"] = s["q_offsets"], None
    s["longest_q"], s["longest_k"], s["scale"] = max(q_len), cap, 1.0 / math.sqrt(d)
    s["out"] = torch.empty((rows, heads, d), dtype=dt, device="cuda")
    return s


# ------------------------------------------------------------------ one pass

def _decoded(w):
    """The weights in 32 bits; bytes are Q8_0 blocks."""
    if w.dtype != torch.uint8:
        return w.float()
    b = w.view(w.shape[0], -1, 34)
    d = b[:, :, :2].contiguous().view(torch.float16).float()
    return (b[:, :, 2:].contiguous().view(torch.int8).float() * d).view(w.shape[0], -1)


def _activated(z, act):
    if act == "gelu":
        return 0.5 * z * (1.0 + torch.tanh(0.7978845608028654 * z * (1.0 + 0.044715 * z * z)))
    if act == "silu":
        return z / (1.0 + torch.exp(-z))
    if act == "relu":
        return torch.clamp_min(z, 0.0)
    return z


def _product(x, w, bias):
    z = x.float() @ _decoded(w).t()
    return z if bias is None else z + bias


def _rotated(x, w, table, pos, scale):
    u = x.float()
    u = u * torch.rsqrt((u * u).mean(-1, keepdim=True) + EPS) * w
    half = table.shape[1] // 2
    cs = table[pos.long()][:, None]
    c, s, a, b = cs[..., :half], cs[..., half:], u[..., :half], u[..., half:2 * half]
    return (torch.cat([a * c - b * s, a * s + b * c, u[..., 2 * half:]], -1) * scale).to(x.dtype)


def _attended(s):
    """Padded to the longest sequence: [batch, KV head, group x query, key] scores, those that are not visible -inf."""
    q, k, v = s["q"], s["k"], s["v"]
    rows, heads, d = q.shape
    kv_heads, batch = k.shape[1], s["q_offsets"].numel() - 1
    group = heads // kv_heads
    q0, k0 = s["q_offsets"].long(), s["k_offsets"].long()
    q_len, k_len = q0[1:] - q0[:-1], s["k_lengths"].long() if s["k_lengths"] is not None else k0[1:] - k0[:-1]
    i = torch.arange(s["longest_q"], device=q.device)[None]
    pos = (k_len - q_len)[:, None] + i  # [batch, query]
    if s["longest_q"] == 1 and 0 <= s["left"] and s["left"] + 1 + s["sinks"] < s["longest_k"]:
        # one query each: the first keys and the window alone, a key that is among both once
        first = torch.arange(s["sinks"], device=q.device)[None].expand(batch, -1)
        near = pos - s["left"] + torch.arange(s["left"] + 1, device=q.device)[None]
        key = torch.cat([first, near], 1)
        once = torch.cat([first < (pos - s["left"]), near >= 0], 1)
    else:
        key = torch.arange(s["longest_k"], device=q.device)[None].expand(batch, -1)
        once = torch.ones_like(key, dtype=torch.bool)
    at = (k0[:-1, None] + key).clamp(0, k.shape[0] - 1)
    kk = k[at].float().permute(0, 2, 3, 1).contiguous()  # [batch, KV head, d, key]
    vv = v[at].float().permute(0, 2, 1, 3).contiguous()
    qq = q[(q0[:-1, None] + i).clamp(0, rows - 1)].float()  # [batch, query, head, d]
    qq = qq.view(batch, -1, kv_heads, group, d).permute(0, 2, 3, 1, 4).reshape(batch, kv_heads, -1, d)
    seen = (key < k_len[:, None])[:, None] & once[:, None]
    if s["right"] >= 0:
        seen = seen & (key[:, None] <= pos[:, :, None] + s["right"])
    if s["left"] >= 0:
        seen = seen & ((key[:, None] >= pos[:, :, None] - s["left"]) | (key[:, None] < s["sinks"]))
    seen = seen.expand(batch, s["longest_q"], key.shape[1])[:, None, None]
    score = (torch.matmul(qq, kk) * s["scale"]).view(batch, kv_heads, group, -1, key.shape[1])
    score = score.masked_fill(~seen, -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True).clamp_min(-1e30))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(batch, kv_heads, -1, key.shape[1]), vv).view(batch, kv_heads, group, -1, d)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    o = o.permute(0, 3, 1, 2, 4).reshape(batch, -1, heads, d)
    return o[i < q_len[:, None]].to(q.dtype)


def run(s):
    op = s["op"]
    if own:
        ops = _package().ops
        if op == "linear":
            ops.linear(s["x"], s["w"], s["y"], bias=s["w_bias"], act=s["act"], residual=s["r"])
            return s["y"]
        if op == "gated":
            ops.linear_gated(s["x"], s["w"], s["up"], s["y"], gate_bias=s["w_bias"], up_bias=s["up_bias"],
                             act=s["act"])
            return s["y"]
        if op == "norm_rope":
            ops.heads_norm_rope(s["q"], s["k"], s["q_w"], s["k_w"], s["table"], s["pos"], EPS, s["q_out"], s["k_out"],
                                q_scale=s["d"] ** -0.5)
            return s["q_out"], s["k_out"]
        ops.window_attention(s["q"], s["k"], s["v"], s["q_offsets"], s["k_offsets"], s["out"], s["scale"],
                             left=s["left"], right=s["right"], sinks=s["sinks"], k_lengths=s["k_lengths"],
                             longest=s["longest_k"])
        return s["out"]
    if op == "linear":
        y = _activated(_product(s["x"], s["w"], s["w_bias"]), s["act"])
        return (y if s["r"] is None else y + s["r"].float()).to(s["x"].dtype)
    if op == "gated":
        gate, up = _product(s["x"], s["w"], s["w_bias"]), _product(s["x"], s["up"], s["up_bias"])
        return (_activated(gate, s["act"]) * up).to(s["x"].dtype)
    if op == "norm_rope":
        return (_rotated(s["q"], s["q_w"], s["table"], s["pos"], s["d"] ** -0.5),
                _rotated(s["k"], s["k_w"], s["table"], s["pos"], 1.0))
    return _attended(s)


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    size = BYTES[case["type"]]
    if case["op"] in ("linear", "gated"):
        n, k, m = case["n"], case["k"], case["m"]
        count = 1 if case["op"] == "linear" else 2
        return {"bytes": size * n * (k + m) + count * m * (BYTES[case["weights"]] * k + (4 if case["bias"] else 0)) +
                (size * n * m if case.get("residual") else 0), "flops": 2 * count * n * k * m}
    heads, kv_heads, d = case["heads"], case["kv_heads"], case["d"]
    if case["op"] == "norm_rope":
        values = case["rows"] * (heads + kv_heads) * d
        return {"bytes": 2 * size * values + 4 * min(case["rows"], 8192) * case["rotary"] + 4 * case["rows"] + 8 * d,
                "flops": 8 * values}
    pairs, keys = 0, 0
    for nq, nk in zip(*_lengths(case)):
        used = 0
        for i in range(nq):
            p = nk - nq + i
            hi = min(nk, p + case["right"] + 1) if case["right"] >= 0 else nk
            lo = max(0, p - case["left"]) if case["left"] >= 0 else 0
            pairs += max(0, hi - lo) + max(0, min(case["sinks"], lo, hi))
            used = max(used, hi) if i == nq - 1 else used
        first = max(0, nk - nq - case["left"]) if case["left"] >= 0 else 0
        keys += max(0, used - first) + min(case["sinks"], first)
    return {"bytes": size * d * (2 * heads * sum(_lengths(case)[0]) + 2 * kv_heads * keys),
            "flops": 4 * heads * d * pairs}


# ------------------------------------------------------------------ the same in 64 bits

def _double(w):
    if w.dtype != torch.uint8:
        return w.double()
    rows = w.shape[0]
    blocks = w.reshape(-1, 34)
    bits = blocks[:, 0].int() + 256 * blocks[:, 1].int()  # scales here are positive and normal
    scale = (1.0 + (bits & 1023).double() / 1024) * torch.exp2((bits >> 10).double() - 15)
    sub = (bits & 1023).double() * 2.0 ** -24
    scale = torch.where(bits >= 1024, scale, sub)
    values = blocks[:, 2:].double()
    values = torch.where(values > 127, values - 256, values)
    return (values * scale[:, None]).reshape(rows, -1)


def _exact_act(z, act):
    if act == "gelu":  # 0.5 (1 + tanh u) = 1 / (1 + exp(-2 u))
        return z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
    return {"none": lambda: z, "silu": lambda: z * torch.sigmoid(z), "relu": lambda: torch.relu(z)}[act]()


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "linear":
        z = torch.nn.functional.linear(s["x"].double(), _double(s["w"]),
                                       None if s["w_bias"] is None else s["w_bias"].double())
        y = _exact_act(z, case["act"])
        return y if s["r"] is None else y + s["r"].double()
    if case["op"] == "gated":
        gate, up = (torch.nn.functional.linear(s["x"].double(), _double(s[w]),
                                               None if s[w + "_bias"] is None else s[w + "_bias"].double())
                    for w in ("w", "up"))
        return _exact_act(gate, case["act"]) * up
    if case["op"] == "norm_rope":
        angle = torch.view_as_complex(torch.stack(s["table"].double()[s["pos"].long()].chunk(2, 1), -1))
        got = []
        for x, w, scale in ((s["q"], s["q_w"], case["d"] ** -0.5), (s["k"], s["k_w"], 1.0)):
            u = x.double()
            u = u / (u.square().mean(-1, keepdim=True) + EPS).sqrt() * w.double()
            half = case["rotary"] // 2
            z = torch.complex(u[..., :half].contiguous(), u[..., half:2 * half].contiguous()) * angle[:, None]
            got.append(torch.cat([z.real, z.imag, u[..., 2 * half:]], -1) * scale)
        return tuple(got)
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    row = 0
    for b, (nq, nk) in enumerate(zip(*_lengths(case))):
        start = int(s["k_offsets"][b])
        p = torch.arange(nk - nq, nk, device="cuda")[:, None]
        t = torch.arange(nk, device="cuda")[None]
        hidden = torch.zeros((nq, nk), dtype=torch.bool, device="cuda")
        if case["left"] >= 0:
            hidden |= (t < p - case["left"]) & (t >= case["sinks"])
        if case["right"] >= 0:
            hidden |= t > p + case["right"]
        for h in range(case["heads"]):
            kv = h * case["kv_heads"] // case["heads"]
            k, v = s["k"][start:start + nk, kv].double(), s["v"][start:start + nk, kv].double()
            score = (s["q"][row:row + nq, h].double() @ k.t()) * s["scale"]
            out[row:row + nq, h] = torch.softmax(score.masked_fill(hidden, -math.inf), 1) @ v
        row += nq
    return out
