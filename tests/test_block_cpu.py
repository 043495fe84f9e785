"""Host-side checks of the block operators that need no GPU: the records'
layout, what the entry points refuse (every case fails before a launch), and the
64-bit reference the GPU tests use against a plain masked softmax."""
import ctypes as C
import math
import os

import numpy as np
import pytest
import torch

import block_reference as R

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
INVALID = 1  # hipErrorInvalidValue


def test_records_match_the_c_layout(tmp_path, eg2):
    import subprocess

    recs = {"LinearArgs": "eg2_linear_args", "LinearGatedArgs": "eg2_linear_gated_args",
            "HeadsNormRopeArgs": "eg2_heads_norm_rope_args", "WindowAttentionArgs": "eg2_window_attention_args"}
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "eg2_hip.h"', "int main(void) {"]
    for r, c in recs.items():
        lines.append(f'  printf("{r} %zu\\n", sizeof({c}));')
        for f, _ in getattr(eg2, r)._fields_:
            lines.append(f'  printf("{r}.{f} %zu\\n", offsetof({c}, {f}));')
    lines.append('  printf("types %u\\n", EG2_TYPE_F32 + 100 * EG2_TYPE_F16 + 10000 * EG2_TYPE_Q8_0 + 1000000 * EG2_TYPE_BF16);')
    lines.append('  printf("acts %u\\n", EG2_ACT_NONE + 10 * EG2_ACT_GELU + 100 * EG2_ACT_SILU + 1000 * EG2_ACT_RELU);')
    lines.append("  return 0; }")
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines))
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    out = dict(line.split() for line in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines())
    for r in recs:
        cls = getattr(eg2, r)
        assert int(out[r]) == C.sizeof(cls)
        for f, _ in cls._fields_:
            assert int(out[f"{r}.{f}"]) == getattr(cls, f).offset, (r, f)
    assert int(out["types"]) == eg2.TYPE_F32 + 100 * eg2.TYPE_F16 + 10000 * eg2.TYPE_Q8_0 + 1000000 * eg2.TYPE_BF16
    a = eg2.ACTIVATIONS
    assert int(out["acts"]) == a["none"] + 10 * a["gelu"] + 100 * a["silu"] + 1000 * a["relu"]


def refused(entry, record, **changes):
    for name, value in changes.items():
        assert hasattr(record, name)
        setattr(record, name, value)
    return entry(C.byref(record), None) == INVALID


P = 1 << 20  # a pointer value on every alignment; nothing is launched


def test_linear_refuses(eg2):
    entry = eg2.lib().eg2_hip_linear

    def rec(kind=30, wkind=30):
        return eg2.LinearArgs(P, P, P, P, P + 4096, 64, 64, 48, 48, 4, 64, 48, kind, wkind, 1)

    for change in ({"y": None}, {"x": None}, {"weight": None}, {"n": 0}, {"k": 0}, {"m": 0}, {"n": (1 << 24) + 1},
                   {"k": (1 << 24) + 1}, {"ldy": 47}, {"type": 8}, {"type": 2}, {"weight_type": 2}, {"weight_type": 0},
                   {"weight_type": 1}, {"act": 4}, {"y": P + 1}, {"x": P + 1}, {"weight": P + 1}, {"bias": P + 2},
                   {"residual": P + 1}, {"residual": P}, {"n": 1 << 24, "m": 512, "ldy": 512}, {"ldx": 1 << 31},
                   {"ldw": 1 << 31}, {"ldy": 1 << 31}, {"ldr": 1 << 31}):
        if change == {"residual": P}:
            change = {"residual": P, "ldr": 56}  # y itself with another stride
        assert refused(entry, rec(), **change), change
    assert refused(entry, rec(0), x=P + 2)
    for change in ({"k": 48}, {"ldw": 80}, {"weight": P + 1}):
        assert refused(entry, rec(30, 8), **change), change
    assert entry(None, None) == INVALID


def test_linear_gated_refuses(eg2):
    entry = eg2.lib().eg2_hip_linear_gated

    def rec(kind=1, wkind=1):
        return eg2.LinearGatedArgs(P, P, P, P, P, P, 64, 64, 48, 4, 64, 48, kind, wkind, 1)

    for change in ({"y": None}, {"x": None}, {"gate": None}, {"up": None}, {"n": 0}, {"k": 0}, {"m": 0}, {"ldy": 47},
                   {"type": 8}, {"weight_type": 30}, {"act": 9}, {"up": P + 1}, {"gate": P + 1}, {"gate_bias": P + 2},
                   {"up_bias": P + 2}, {"weight_type": 8, "k": 40}, {"weight_type": 8, "ldw": 72}):
        assert refused(entry, rec(), **change), change
    assert entry(None, None) == INVALID


def test_heads_norm_rope_refuses(eg2):
    entry = eg2.lib().eg2_hip_heads_norm_rope

    def rec():
        return eg2.HeadsNormRopeArgs(P, P, P + 65536, P + 65536, P, P, P, P, 256, 64, 256, 64, 256, 64, 256, 64, 4, 3, 1, 64,
                                     64, 100, 30, 1e-6, 1.0)

    for change in ({"q": None}, {"q_out": None}, {"k": None}, {"k_out": None}, {"table": None}, {"pos": None}, {"rows": 0},
                   {"rows": (1 << 24) + 1}, {"q_heads": 0}, {"q_heads": 4096}, {"k_heads": 5000}, {"d": 0}, {"d": 63},
                   {"d": 514}, {"rotary": 66}, {"rotary": 31}, {"table_rows": 0}, {"type": 8}, {"q": P + 1}, {"k": P + 1},
                   {"q_weight": P + 2}, {"k_weight": P + 1}, {"table": P + 1}, {"pos": P + 2}, {"q": P, "q_row": 512},
                   {"k": P, "k_head": 128}, {"q_row": 1 << 31}, {"k_out_head": 1 << 31}, {"rows": 1 << 24, "q_heads": 2}):
        assert refused(entry, rec(), **change), change
    assert entry(None, None) == INVALID


def attention_record(eg2, **changes):
    r = eg2.WindowAttentionArgs(P, P, P, P, P, P, None, P, 1 << 40, 256, 64, 128, 64, 128, 64, 256, 64, 2, 40, 80, 4, 2, 64,
                                30, 16, 0, 2, 0, 0.125)
    for name, value in changes.items():
        assert hasattr(r, name)
        setattr(r, name, value)
    return r


def test_window_attention_refuses(eg2):
    entry = eg2.lib().eg2_hip_window_attention
    for change in ({"out": None}, {"q": None}, {"k": None}, {"v": None}, {"q_offsets": None}, {"k_offsets": None},
                   {"batch": 0}, {"batch": 65536}, {"rows": 0}, {"rows": 1 << 31}, {"key_rows": 0}, {"key_rows": 1 << 31},
                   {"heads": 0}, {"kv_heads": 0}, {"heads": 5}, {"heads": 4098, "kv_heads": 2}, {"d": 0}, {"d": 60},
                   {"d": 264}, {"type": 8}, {"q": P + 8}, {"k": P + 4}, {"v": P + 2}, {"out": P + 8}, {"q_row": 260},
                   {"k_head": 68}, {"v_row": 132}, {"out_head": 4}, {"q_offsets": P + 2}, {"k_lengths": P + 1},
                   {"scale": math.inf}, {"scale": math.nan}, {"scale": -3e38}, {"q_row": 1 << 31},
                   {"key_rows": (1 << 30) + 1}, {"batch": 65535, "kv_heads": 65, "heads": 65}):
        assert entry(C.byref(attention_record(eg2, **change)), None) == INVALID, change
    assert entry(C.byref(attention_record(eg2, type=0, k_row=130)), None) == INVALID
    assert entry(None, None) == INVALID


def test_window_attention_refuses_a_small_workspace(eg2):
    """Few rows over many keys are split over the GPU and need one."""
    lib = eg2.lib()
    big = {"batch": 1, "rows": 1, "key_rows": 100000, "longest": 100000, "left": -1}
    need = lib.eg2_hip_window_attention_workspace(C.byref(attention_record(eg2, **big)))
    assert lib.eg2_hip_window_attention_workspace(C.byref(attention_record(eg2, d=7))) == 0
    assert lib.eg2_hip_window_attention_workspace(None) == 0
    if not need:
        pytest.skip("the keys are not split")
    for change in ({"workspace": None}, {"workspace_bytes": need - 1}, {"workspace": P + 8}):
        assert lib.eg2_hip_window_attention(C.byref(attention_record(eg2, **big, **change)), None) == INVALID, change


def test_python_refuses(eg2):
    o = eg2.ops
    f = lambda *s: torch.zeros(s)  # noqa: E731
    h = lambda *s: torch.zeros(s, dtype=torch.float16)  # noqa: E731
    i = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    bad = [
        lambda: o.linear(f(4, 8), f(5, 8), f(4, 5)),  # not on a GPU
        lambda: o.linear(f(4, 8), f(5, 9), f(4, 5)),
        lambda: o.linear(f(4, 8), f(5, 8), f(3, 5)),
        lambda: o.linear(f(4, 8), f(5, 8), h(4, 5)),
        lambda: o.linear(h(4, 8), f(5, 8), h(4, 5)),
        lambda: o.linear(f(4, 8), f(8, 5).t(), f(4, 5)),
        lambda: o.linear(f(4, 8), f(5, 8), f(4, 5), bias=f(4)),
        lambda: o.linear(f(4, 8), f(5, 8), f(4, 5), bias=h(5)),
        lambda: o.linear(f(4, 8), f(5, 8), f(4, 5), residual=f(4, 4)),
        lambda: o.linear(f(4, 8), f(5, 8), f(4, 5), act="tanh"),
        lambda: o.linear(f(4, 40), torch.zeros((5, 34), dtype=torch.uint8), f(4, 5)),
        lambda: o.linear(f(4, 64), torch.zeros((5, 34), dtype=torch.uint8), f(4, 5)),
        lambda: o.linear(torch.zeros((4, 8), dtype=torch.float64), f(5, 8), torch.zeros((4, 5), dtype=torch.float64)),
        lambda: o.linear_gated(f(4, 8), f(5, 8), f(6, 8), f(4, 5)),
        lambda: o.linear_gated(f(4, 8), f(5, 8), f(5, 16)[:, :8], f(4, 5)),
        lambda: o.linear_gated(f(4, 8), f(5, 8), f(5, 8), f(4, 5), up_bias=f(6)),
        lambda: o.heads_norm_rope(f(4, 3, 8), f(4, 1, 8), None, None, None, None, 1e-6, f(4, 3, 8), f(4, 1, 8)),
        lambda: o.heads_norm_rope(f(4, 3, 8), f(4, 1, 6), None, None, None, None, 1e-6, f(4, 3, 8), f(4, 1, 6)),
        lambda: o.heads_norm_rope(f(4, 3, 8), f(4, 1, 8), None, None, None, None, 1e-6, f(4, 3, 8), None),
        lambda: o.heads_norm_rope(f(4, 3, 8), None, f(7), None, None, None, 1e-6, f(4, 3, 8), None),
        lambda: o.heads_norm_rope(f(4, 3, 8), None, None, None, f(9, 8), None, 1e-6, f(4, 3, 8), None),
        lambda: o.heads_norm_rope(f(4, 3, 8), None, None, None, f(9, 8), i(3), 1e-6, f(4, 3, 8), None),
        lambda: o.window_attention(f(4, 2, 8), f(4, 1, 8), f(4, 1, 8), i(2), i(2), f(4, 2, 8), 1.0),
        lambda: o.window_attention(f(4, 2, 8), f(4, 1, 8), f(5, 1, 8), i(2), i(2), f(4, 2, 8), 1.0),
        lambda: o.window_attention(f(4, 2, 8), f(4, 1, 8), f(4, 1, 8), i(2), i(3), f(4, 2, 8), 1.0),
        lambda: o.window_attention(f(4, 2, 8), f(4, 1, 8), f(4, 1, 8), f(2), i(2), f(4, 2, 8), 1.0),
        lambda: o.window_attention(f(4, 2, 8), f(4, 1, 8), f(4, 1, 8), i(0), i(0), f(4, 2, 8), 1.0),
        lambda: o.window_attention(f(4, 2, 8), h(4, 1, 8), h(4, 1, 8), i(2), i(2), f(4, 2, 8), 1.0),
    ]
    for call in bad:
        with pytest.raises(ValueError):
            call()


def test_reference_attention_is_a_masked_softmax():
    """The reference's row-by-row selection against one masked softmax, and a planted mistake found."""
    rng = np.random.default_rng(0)
    q, k, v = (rng.standard_normal(s) for s in ((20, 4, 8), (30, 2, 8), (30, 2, 8)))
    for left, right, sinks in ((-1, -1, 0), (5, 0, 2), (3, 3, 0), (0, 0, 1)):
        out, _ = R.window_attention(q, k, v, [0, 20], [0, 30], 0.3, left, right, sinks, None, torch.float32)
        p, s = np.arange(10, 30)[:, None], np.arange(30)[None]
        hidden = np.zeros((20, 30), bool)
        if left >= 0:
            hidden |= (s < p - left) & (s >= sinks)
        if right >= 0:
            hidden |= s > p + right
        for h in range(4):
            sc = torch.from_numpy(q[:, h] @ k[:, h // 2].T * 0.3).masked_fill(torch.from_numpy(hidden), -math.inf)
            want = torch.softmax(sc, 1).numpy() @ v[:, h // 2]
            assert np.abs(out[:, h] - want).max() < 1e-14
        wrong, off = R.window_attention(q, k, v, [0, 20], [0, 30], 0.3, left, right, sinks + 1 if left >= 0 else 0, None,
                                        torch.float32)
        if left >= 0:
            assert (np.abs(wrong - out) > off).any()
    none, _ = R.window_attention(q, k[:4], v[:4], [0, 20], [0, 4], 0.3, 2, 0, 1, None, torch.float32)
    assert (none[:16] == 0).all() and np.abs(none[16:]).min() > 0


def test_reference_quantizer_and_products():
    rng = np.random.default_rng(1)
    w = rng.standard_normal((6, 64)).astype(np.float32)
    raw, values = R.quantize(w)
    assert raw.shape == (6, 68) and np.abs(values - w).max() <= np.abs(w).max() / 127
    d = raw.reshape(6, 2, 34)[:, :, :2].copy().view(np.float16).astype(np.float64)
    assert np.array_equal(raw.reshape(6, 2, 34)[:, :, 2:].view(np.int8) * d, values.reshape(6, 2, 32))
    x = rng.standard_normal((5, 64))
    y, off = R.linear(x, values, None, "gelu", None, torch.bfloat16)
    t = torch.nn.functional.gelu(torch.from_numpy(x @ values.T), approximate="tanh").numpy()
    assert np.abs(y - t).max() < 1e-12 and (off >= R.rounding(y, torch.bfloat16)).all()


@pytest.mark.parametrize("source", ["kernels_window.hip", "kernels_linear_f32.hip", "kernels_linear_bf16.hip"])
def test_only_the_dma_uses_m0(tmp_path, source):
    """The loads to LDS set M0 in inline asm and declare it clobbered: sound only while no
    instruction of the compiler's reads it. Every mention of m0 in the compiled kernels is the asm's own write."""
    import re
    import shutil
    import subprocess

    hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
    if not shutil.which(hipcc):
        pytest.skip("hipcc not available")
    pkg = os.path.join(ROOT, "embeddinggemma2-amdkfd_amd")
    out = tmp_path / "kernels.s"
    subprocess.run([hipcc, "--offload-arch=gfx950", "-O3", "-std=c++17", "-ffp-contract=off",
                    "-fhip-fp32-correctly-rounded-divide-sqrt", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
                    "-mllvm", "-amdgpu-mfma-vgpr-form", "-I" + os.path.join(ROOT, "include"), "-I" + os.path.join(pkg, "csrc"),
                    "--cuda-device-only", "-S", os.path.join(pkg, "csrc", source), "-o", str(out)],
                   check=True, capture_output=True, timeout=600)
    inside, own, other = False, 0, []
    for line in out.read_text().splitlines():
        if "#ASMSTART" in line or "#ASMEND" in line:
            inside = "#ASMSTART" in line
            continue
        code = line.split(";")[0]
        if re.search(r"\bm0\b", code):
            if inside and re.match(r"\s*s_mov_b32 m0, (s\d+|vcc_lo|vcc_hi)\s*$", code):  # any scalar register may hold it
                own += 1
            else:
                other.append(code)
    assert own and not other, (own, other[:5])
