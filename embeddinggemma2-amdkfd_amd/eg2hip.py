"""Python binding of libeg2hip.so (the gfx950 executor and its operators).

Mirrors the reference's executor interface (src/gemma2_kfd.h:7-10):
`Encoder(gguf_path)` wraps ei_gemma2_kfd_create / _free and
`Encoder.batch(ids, offsets)` wraps ei_gemma2_kfd_batch, raising on the
same conditions the C ABI reports with `false` + message. `ops` exposes the
operator-level entry points of include/eg2_hip.h for device buffers (torch
tensors are used only as device allocations and for their streams).

The library must be built (`make -C embeddinggemma2-amdkfd_amd`); there is
no fallback path: a missing library raises immediately.
"""
import ctypes as C
import os
import struct

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libeg2hip.so")

N_EMBD, N_FF, HEAD_DIM, N_CTX, VOCAB = 768, 1152, 256, 2048, 262144
QKV_COLS = N_EMBD + 2 * HEAD_DIM

_vp, _f, _i32 = C.c_void_p, C.POINTER(C.c_float), C.POINTER(C.c_int32)
_u = C.c_uint


class EiStr(C.Structure):
    _fields_ = [("str", C.c_void_p), ("len", C.c_uint64)]


class _KvValue(C.Union):
    _fields_ = [("u64", C.c_uint64), ("i64", C.c_int64), ("f64", C.c_double), ("b", C.c_bool), ("s", EiStr)]


class EiKv(C.Structure):
    _fields_ = [("key", EiStr), ("type", C.c_uint32), ("v", _KvValue), ("arr_type", C.c_uint32),
                ("arr_n", C.c_uint64), ("arr_data", C.c_void_p)]


class EiTensor(C.Structure):
    _fields_ = [("name", EiStr), ("n_dims", C.c_uint32), ("ne", C.c_uint64 * 4), ("type", C.c_uint32),
                ("offset", C.c_uint64), ("data", C.c_void_p), ("n_bytes", C.c_uint64)]


class EiGguf(C.Structure):
    _fields_ = [("map", C.c_void_p), ("map_len", C.c_size_t), ("version", C.c_uint32), ("n_kv", C.c_uint64),
                ("n_tensors", C.c_uint64), ("alignment", C.c_uint64), ("data_off", C.c_uint64),
                ("kv", C.POINTER(EiKv)), ("tensors", C.POINTER(EiTensor))]


class BatchConfig(C.Structure):
    """eg2_batch_config (include/eg2_stream.h)."""
    _fields_ = [("max_batch_tokens", C.c_size_t), ("max_batch_sequence_tokens", C.c_size_t),
                ("max_batch_requests", C.c_size_t), ("lookahead", C.c_uint), ("sort_longest_first", C.c_uint)]


class SynthConfig(C.Structure):
    _fields_ = [("seed", C.c_uint64), ("n_layer", C.c_uint), ("dense_head", C.c_uint), ("weight_std", C.c_float),
                ("embed_std", C.c_float), ("norm_std", C.c_float), ("rope_base_full", C.c_float),
                ("rope_base_swa", C.c_float), ("sliding_window", C.c_uint), ("sliding_window_pattern", C.c_uint),
                ("threads", C.c_uint)]


# The operator records of include/abi.h (kernels/abi.h:3-11) and EgSaxpy.
class EgGather(C.Structure):
    _fields_ = [("out", _vp), ("weight", _vp), ("ids", _vp), ("n", _u)]


class EgMM(C.Structure):
    _fields_ = [("out", _vp), ("x", _vp), ("weight", _vp), ("n", _u), ("k", _u), ("m", _u), ("type", _u)]


class EgNorm(C.Structure):
    _fields_ = [("out", _vp), ("x", _vp), ("weight", _vp), ("rows", _u), ("d", _u), ("scale", C.c_float)]


class EgRope(C.Structure):
    _fields_ = [("x", _vp), ("table", _vp), ("n", _u), ("heads", _u), ("d", _u)]


class EgAttention(C.Structure):
    _fields_ = [("out", _vp), ("q", _vp), ("k", _vp), ("v", _vp), ("bounds", _vp), ("n", _u), ("window", _u)]


class EgElement(C.Structure):
    _fields_ = [("out", _vp), ("x", _vp), ("other", _vp), ("n", _u), ("mode", _u), ("layer", _u),
                ("scale", C.c_float)]


class EgPool(C.Structure):
    _fields_ = [("out", _vp), ("x", _vp), ("offsets", _vp), ("batch", _u)]


class EgNormResidual(C.Structure):
    _fields_ = [("out", _vp), ("x", _vp), ("weight", _vp), ("rows", _u), ("d", _u), ("scale", C.c_float)]


class EgNormRope(C.Structure):
    _fields_ = [("x", _vp), ("weight", _vp), ("table", _vp), ("rows", _u), ("d", _u), ("heads", _u)]


class EgSaxpy(C.Structure):
    _fields_ = [("y", _vp), ("x", _vp), ("a", C.c_float), ("n", _u)]


# The records of the block operators (include/eg2_hip.h) and the ids of their types and activations.
_u64 = C.c_uint64
_torch_types = None  # ops._types()


def _packed(cls):
    """Gives a record class pack(*fields): the record's bytes, in a fraction of the time of its constructor."""
    codes = {_vp: "P", _u64: "Q", _u: "I", C.c_int: "i", C.c_float: "f"}
    packer = struct.Struct("@" + "".join(codes[t] for _, t in cls._fields_) + "0Q")  # 0Q: padded as the record is
    assert packer.size == C.sizeof(cls)
    cls.pack = staticmethod(packer.pack)
    return cls


TYPE_F32, TYPE_F16, TYPE_Q8_0, TYPE_BF16 = 0, 1, 8, 30
ACTIVATIONS = {"none": 0, "gelu": 1, "silu": 2, "relu": 3}


@_packed
class LinearArgs(C.Structure):
    """eg2_linear_args."""
    _fields_ = [("y", _vp), ("x", _vp), ("weight", _vp), ("bias", _vp), ("residual", _vp), ("ldx", _u64),
                ("ldw", _u64), ("ldy", _u64), ("ldr", _u64), ("n", _u), ("k", _u), ("m", _u), ("type", _u),
                ("weight_type", _u), ("act", _u)]


@_packed
class LinearGatedArgs(C.Structure):
    """eg2_linear_gated_args."""
    _fields_ = [("y", _vp), ("x", _vp), ("gate", _vp), ("up", _vp), ("gate_bias", _vp), ("up_bias", _vp),
                ("ldx", _u64), ("ldw", _u64), ("ldy", _u64), ("n", _u), ("k", _u), ("m", _u), ("type", _u),
                ("weight_type", _u), ("act", _u)]


@_packed
class HeadsNormRopeArgs(C.Structure):
    """eg2_heads_norm_rope_args."""
    _fields_ = [("q_out", _vp), ("k_out", _vp), ("q", _vp), ("k", _vp), ("q_weight", _vp), ("k_weight", _vp),
                ("table", _vp), ("pos", _vp), ("q_row", _u64), ("q_head", _u64), ("k_row", _u64), ("k_head", _u64),
                ("q_out_row", _u64), ("q_out_head", _u64), ("k_out_row", _u64), ("k_out_head", _u64), ("rows", _u),
                ("q_heads", _u), ("k_heads", _u), ("d", _u), ("rotary", _u), ("table_rows", _u), ("type", _u),
                ("eps", C.c_float), ("q_scale", C.c_float)]


@_packed
class WindowAttentionArgs(C.Structure):
    """eg2_window_attention_args."""
    _fields_ = [("out", _vp), ("q", _vp), ("k", _vp), ("v", _vp), ("q_offsets", _vp), ("k_offsets", _vp),
                ("k_lengths", _vp), ("workspace", _vp), ("workspace_bytes", _u64), ("q_row", _u64), ("q_head", _u64),
                ("k_row", _u64), ("k_head", _u64), ("v_row", _u64), ("v_head", _u64), ("out_row", _u64),
                ("out_head", _u64), ("batch", _u), ("rows", _u), ("key_rows", _u), ("heads", _u), ("kv_heads", _u),
                ("d", _u), ("type", _u), ("left", C.c_int), ("right", C.c_int), ("sinks", _u), ("longest", _u),
                ("scale", C.c_float)]


# Every symbol declared in include/eg2_hip.h, eg2_ops.h, eg2_stream.h and gemma2_kfd.h.
SIGNATURES = {
    "eg2_op_launch": (C.c_int, [C.c_char_p, _vp, C.c_size_t, _u, _u, _u, _vp]),
    "eg2_op_count": (C.c_uint, []),
    "eg2_op_name": (C.c_char_p, [_u]),
    "eg2_hip_embed_norm_quant": (C.c_int, [_vp, _vp, _u, C.c_float, _vp, C.c_float, _vp, _vp, _vp, _vp]),
    "eg2_hip_residual_norm_quant": (C.c_int, [_vp, _vp, _vp, _vp, C.c_float, _vp, _vp, _u, _vp]),
    "eg2_hip_qk_norm_rope": (C.c_int, [_vp, _vp, _vp, _vp, _vp, C.c_float, _vp, _u, _vp]),
    "eg2_hip_attention": (C.c_int, [_vp, _vp, _vp, _u, _vp, _u, _u, _u, _vp, _vp, _vp, _vp]),
    "eg2_hip_attention_static": (C.c_int, [_vp, _vp, _u, _u, _u, _vp, _vp, _vp]),
    "eg2_hip_attention_scores": (C.c_int, [_vp, _vp, _vp, _u, _u, _u, _vp, _vp]),
    "eg2_hip_attention_softmax": (C.c_int, [_vp, _u, _u, _u, _vp, _vp]),
    "eg2_hip_attention_context": (C.c_int, [_vp, _vp, _vp, _u, _u, _u, _vp, _vp, _vp, _vp]),
    "eg2_attention_plan": (C.c_int, [C.POINTER(C.c_size_t), C.c_size_t, C.c_size_t, C.c_size_t, _vp, _vp,
                                     C.POINTER(C.c_size_t)]),
    "eg2_attention_capacity": (None, [C.c_size_t, C.c_size_t, C.POINTER(C.c_size_t)]),
    "eg2_hip_gelu_quant": (C.c_int, [_vp, _vp, _vp, _u, _vp]),
    "eg2_hip_libm_eval": (C.c_int, [_vp, _u, _vp, _vp, _vp]),
    "eg2_hip_tanh_approx_error": (C.c_int, [_vp, _vp]),
    "eg2_hip_quantize_rows": (C.c_int, [_vp, _u, _vp, _vp, _u, _vp]),
    "eg2_hip_rms_norm_rows": (C.c_int, [_vp, _vp, C.c_float, _u, _vp]),
    "eg2_hip_pool_l2": (C.c_int, [_vp, _vp, _vp, _u, _vp]),
    "eg2_hip_pool_mean": (C.c_int, [_vp, _vp, _vp, _u, _vp]),
    "eg2_hip_l2_prefix": (C.c_int, [_vp, _u, _u, _u, _vp]),
    "eg2_hip_gemm_q8": (C.c_int, [_vp, _vp, _u, _vp, _vp, _u, _vp, _u, _u, _u, _u, _vp]),
    "eg2_hip_gemm_q8_geglu": (C.c_int, [_vp, _vp, _u, _vp, _vp, _u, _vp, _vp, _u, _u, _u, _u, _vp]),
    "eg2_hip_gemm_q8_qkv_rope": (C.c_int, [_vp, _vp, _u, _vp, _vp, _u, _u, _u, _vp, _vp, _vp, _vp, C.c_float, _vp,
                                           _vp]),
    "eg2_hip_linear": (C.c_int, [_vp, _vp]),
    "eg2_hip_linear_gated": (C.c_int, [_vp, _vp]),
    "eg2_hip_heads_norm_rope": (C.c_int, [_vp, _vp]),
    "eg2_hip_window_attention": (C.c_int, [_vp, _vp]),
    "eg2_hip_window_attention_workspace": (C.c_uint64, [_vp]),
    "eg2_hip_error_string": (C.c_char_p, [C.c_int]),
    "eg2_hip_device_check": (C.c_int, [C.c_char_p, C.c_size_t]),
    "eg2_q8_tile_bytes": (C.c_size_t, [C.c_size_t, _u]),
    "eg2_q8_pack_rows": (None, [_vp, C.c_size_t, _u, _vp]),
    "eg2_q8_unpack_rows": (None, [_vp, C.c_size_t, _u, _vp]),
    "eg2_q8_weight_tiles": (None, [_vp, C.c_size_t, _u, _vp, _vp]),
    "eg2_q8_geglu_weight_tiles": (C.c_int, [_vp, _vp, C.c_size_t, _u, _vp, _vp]),
    "eg2_rope_table": (None, [C.c_float, _u, _vp]),
    "eg2_gguf_open": (C.c_int, [C.c_char_p, C.POINTER(EiGguf), C.c_char_p, C.c_size_t]),
    "eg2_gguf_close": (None, [C.POINTER(EiGguf)]),
    "eg2_synth_write_gguf": (C.c_int, [C.c_char_p, C.POINTER(SynthConfig), C.c_char_p, C.c_size_t]),
    "eg2_batch_config_default": (None, [C.POINTER(BatchConfig)]),
    "eg2_pack_waves": (C.c_size_t, [C.POINTER(C.c_size_t), C.c_size_t, C.POINTER(BatchConfig), C.POINTER(C.c_size_t),
                                    C.POINTER(C.c_size_t)]),
    "eg2_normalize_prefix": (C.c_bool, [_f, C.c_uint]),
    "eg2_stream_embed": (C.c_bool, [C.c_void_p, _i32, C.POINTER(C.c_size_t), C.c_size_t, C.POINTER(C.c_uint),
                                    C.POINTER(BatchConfig), _f, C.POINTER(C.c_size_t), C.c_char_p, C.c_size_t]),
    "ei_gemma2_kfd_create": (C.c_void_p, [C.POINTER(EiGguf), C.c_char_p, C.c_size_t]),
    "ei_gemma2_kfd_free": (None, [C.c_void_p]),
    "eg2_kfd_stage": (C.c_bool, [C.c_void_p, _i32, C.POINTER(C.c_size_t), C.c_size_t, C.c_char_p, C.c_size_t]),
    "eg2_kfd_launch_staged": (C.c_bool, [C.c_void_p, C.c_uint, C.c_char_p, C.c_size_t]),
    "eg2_kfd_collect": (C.c_bool, [C.c_void_p, _f, C.c_char_p, C.c_size_t]),
    "eg2_kfd_lanes": (C.c_uint, [C.c_void_p]),
    "eg2_kfd_validate_gguf": (C.c_bool, [C.POINTER(EiGguf), C.c_char_p, C.c_size_t]),
    "eg2_kfd_inject_failure": (None, [C.c_void_p]),
    "eg2_f32_to_chars": (C.c_size_t, [C.c_char_p, C.c_float]),
    "eg2_tokenizer_create": (C.c_void_p, [C.c_void_p, C.c_char_p, C.c_size_t]),
    "eg2_tokenizer_free": (None, [C.c_void_p]),
    "eg2_tokenizer_text_to_id": (C.c_int32, [C.c_void_p, C.c_char_p, C.c_size_t]),
    "eg2_tokenize": (C.c_size_t, [C.c_void_p, C.c_char_p, C.c_size_t, C.c_bool, C.c_bool, _i32, C.c_size_t]),
    "eg2_tokenize_batch": (C.c_size_t, [C.c_void_p, C.c_char_p, C.POINTER(C.c_size_t), C.c_size_t, C.c_bool,
                                        C.c_bool, _i32, C.c_size_t, C.POINTER(C.c_size_t), C.c_uint]),
    "eg2_base64_f32": (C.c_size_t, [_f, C.c_size_t, C.c_char_p]),
    "eg2_embeddings_response_bound": (C.c_size_t, [C.c_size_t, C.c_uint, C.c_size_t]),
    "eg2_embeddings_response": (C.c_size_t, [_f, C.c_size_t, C.c_uint, C.c_int, C.c_int, C.c_char_p, C.c_size_t,
                                             C.c_size_t, C.c_char_p, C.c_size_t]),
    "eg2_kfd_acquire_lane": (C.c_int, [C.c_void_p]),
    "eg2_kfd_try_acquire_lane": (C.c_int, [C.c_void_p]),
    "eg2_kfd_release_lane": (None, [C.c_void_p, C.c_uint]),
    "eg2_kfd_stage_lane": (C.c_bool, [C.c_void_p, C.c_uint, _i32, C.POINTER(C.c_size_t), C.c_size_t, C.c_char_p,
                                      C.c_size_t]),
    "eg2_kfd_launch_lane": (C.c_bool, [C.c_void_p, C.c_uint, C.c_uint, C.c_char_p, C.c_size_t]),
    "eg2_kfd_collect_lane": (C.c_bool, [C.c_void_p, C.c_uint, _f, C.c_char_p, C.c_size_t]),
    "eg2_kfd_lane_ready": (C.c_int, [C.c_void_p, C.c_uint, C.c_char_p, C.c_size_t]),
    "ei_gemma2_kfd_batch": (C.c_bool, [C.c_void_p, _i32, C.POINTER(C.c_size_t), C.c_size_t, _f, C.c_char_p,
                                       C.c_size_t]),
}

_lib = None


def lib():
    """The loaded library (raises if it was not built)."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(f"{LIB_PATH} is not built: run `make -C {HERE}`")
        handle = C.CDLL(LIB_PATH)
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(handle, name)
            fn.restype = res
            fn.argtypes = args
        _lib = handle
    return _lib


class HipError(RuntimeError):
    pass


def check(code, what):
    if code != 0:
        raise HipError(f"{what}: {lib().eg2_hip_error_string(code).decode()} ({code})")


def synth_gguf(path, seed=0, n_layer=24, dense_head=True, weight_std=0.02, embed_std=0.02, norm_std=0.1,
               rope_base_full=10000.0, rope_base_swa=10000.0, sliding_window=0, sliding_window_pattern=6,
               threads=8):
    """Writes a synthetic gemma-embedding GGUF (see eg2_synth_write_gguf)."""
    cfg = SynthConfig(seed, n_layer, 1 if dense_head else 0, weight_std, embed_std, norm_std, rope_base_full,
                      rope_base_swa, sliding_window, sliding_window_pattern, threads)
    err = C.create_string_buffer(512)
    if lib().eg2_synth_write_gguf(os.fsencode(path), C.byref(cfg), err, 512) != 0:
        raise HipError("synthetic GGUF: " + err.value.decode())


class Gguf:
    """A GGUF file parsed into the engine's ei_gguf layout."""

    def __init__(self, path):
        self.g = EiGguf()
        err = C.create_string_buffer(512)
        if lib().eg2_gguf_open(os.fsencode(path), C.byref(self.g), err, 512) != 0:
            raise HipError(err.value.decode())

    def close(self):
        if self.g is not None:
            lib().eg2_gguf_close(C.byref(self.g))
            self.g = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def validate_gguf(gguf):
    """eg2_kfd_validate_gguf on an open Gguf: None, or the rejection message."""
    err = C.create_string_buffer(512)
    if lib().eg2_kfd_validate_gguf(C.byref(gguf.g), err, 512):
        return None
    return err.value.decode()


class Tokenizer:
    """eg2_tokenizer over the tokenizer.ggml.* keys of a GGUF file."""

    def __init__(self, gguf_path):
        self.gguf = Gguf(gguf_path)
        err = C.create_string_buffer(512)
        self.tok = lib().eg2_tokenizer_create(C.byref(self.gguf.g), err, 512)
        if not self.tok:
            raise HipError(err.value.decode())

    def encode(self, text, add_special=True, parse_special=False):
        """Token ids of `text` (bytes or str) as an int32 array."""
        import numpy as np

        b = text.encode() if isinstance(text, str) else bytes(text)
        n = lib().eg2_tokenize(self.tok, b, len(b), add_special, parse_special, None, 0)
        ids = np.zeros(max(n, 1), np.int32)
        lib().eg2_tokenize(self.tok, b, len(b), add_special, parse_special, ids.ctypes.data_as(_i32), n)
        return ids[:n]

    def encode_batch(self, texts, add_special=True, parse_special=False, threads=0):
        """(ids, offsets) of several texts packed back to back."""
        import numpy as np

        bs = [t.encode() if isinstance(t, str) else bytes(t) for t in texts]
        toffs = (C.c_size_t * (len(bs) + 1))(*np.concatenate([[0], np.cumsum([len(b) for b in bs])]).astype(int))
        joined = b"".join(bs)
        cap = 4 * len(joined) + 4 * len(bs) + 16
        ids = np.zeros(cap, np.int32)
        ioffs = (C.c_size_t * (len(bs) + 1))()
        n = lib().eg2_tokenize_batch(self.tok, joined, toffs, len(bs), add_special, parse_special,
                                     ids.ctypes.data_as(_i32), cap, ioffs, threads)
        if n == (1 << 64) - 1:
            raise HipError("token capacity exceeded")
        return ids[:n], np.array(list(ioffs), np.int64)

    def text_to_id(self, text):
        b = text.encode() if isinstance(text, str) else bytes(text)
        return lib().eg2_tokenizer_text_to_id(self.tok, b, len(b))

    def close(self):
        if getattr(self, "tok", None):
            lib().eg2_tokenizer_free(self.tok)
            self.tok = None
        if getattr(self, "gguf", None):
            self.gguf.close()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class Encoder:
    """ei_gemma2_kfd_create / _batch / _free over a GGUF file."""

    def __init__(self, gguf_path):
        self.gguf = Gguf(gguf_path)
        err = C.create_string_buffer(1024)
        self.ctx = lib().ei_gemma2_kfd_create(C.byref(self.gguf.g), err, 1024)
        if not self.ctx:
            raise HipError(err.value.decode())

    def batch(self, ids, offsets):
        """ids: int32 array of offsets[-1] tokens; offsets: batch+1 sizes.
        Returns float32 [batch, 768] (numpy)."""
        import numpy as np

        ids = np.ascontiguousarray(ids, dtype=np.int32)
        offs = (C.c_size_t * len(offsets))(*[int(o) for o in offsets])
        batch = len(offsets) - 1
        out = np.zeros((max(batch, 1), N_EMBD), dtype=np.float32)
        err = C.create_string_buffer(1024)
        ok = lib().ei_gemma2_kfd_batch(self.ctx, ids.ctypes.data_as(_i32), offs, batch,
                                       out.ctypes.data_as(_f), err, 1024)
        if not ok:
            raise HipError(err.value.decode())
        return out[:batch]

    @property
    def lanes(self):
        """Waves the context keeps in flight (eg2_kfd_lanes)."""
        return lib().eg2_kfd_lanes(self.ctx)

    def stage(self, ids, offsets, lane=0):
        """Uploads one wave to a lane (eg2_kfd_stage_lane); launch()/collect()
        with the same lane then run it."""
        import numpy as np

        if not hasattr(self, "_staged"):
            self._staged = {}
        ids = np.ascontiguousarray(ids, dtype=np.int32)
        offs = (C.c_size_t * len(offsets))(*[int(o) for o in offsets])
        batch = len(offsets) - 1
        err = C.create_string_buffer(1024)
        if not lib().eg2_kfd_stage_lane(self.ctx, lane, ids.ctypes.data_as(_i32), offs, batch, err, 1024):
            raise HipError(err.value.decode())
        self._staged[lane] = batch

    def launch(self, repeats=1, lane=0):
        err = C.create_string_buffer(1024)
        if not lib().eg2_kfd_launch_lane(self.ctx, lane, repeats, err, 1024):
            raise HipError(err.value.decode())

    def ready(self, lane=0):
        """eg2_kfd_lane_ready: True once the lane's enqueued work is done,
        False while it runs (never waits)."""
        err = C.create_string_buffer(1024)
        r = lib().eg2_kfd_lane_ready(self.ctx, lane, err, 1024)
        if r < 0:
            raise HipError(err.value.decode())
        return bool(r)

    def collect(self, lane=0):
        import numpy as np

        out = np.zeros((self._staged[lane], N_EMBD), dtype=np.float32)
        err = C.create_string_buffer(1024)
        if not lib().eg2_kfd_collect_lane(self.ctx, lane, out.ctypes.data_as(_f), err, 1024):
            raise HipError(err.value.decode())
        return out

    def stream(self, ids, text_offsets, dims, cfg=None):
        """eg2_stream_embed: texts ids[text_offsets[i]:text_offsets[i+1]] with
        output widths dims[i], packed into waves by the batcher's rules.
        Returns (float32 [n, 768] with zeros past dims[i], wave count)."""
        import numpy as np

        ids = np.ascontiguousarray(ids, dtype=np.int32)
        n = len(text_offsets) - 1
        offs = (C.c_size_t * (n + 1))(*[int(o) for o in text_offsets])
        d = (C.c_uint * n)(*[int(x) for x in dims])
        cfg = cfg or batch_config()
        out = np.zeros((n, N_EMBD), dtype=np.float32)
        waves = C.c_size_t(0)
        err = C.create_string_buffer(1024)
        if not lib().eg2_stream_embed(self.ctx, ids.ctypes.data_as(_i32), offs, n, d, C.byref(cfg),
                                      out.ctypes.data_as(_f), C.byref(waves), err, 1024):
            raise HipError(err.value.decode())
        return out, waves.value

    def close(self):
        if getattr(self, "ctx", None):
            lib().ei_gemma2_kfd_free(self.ctx)
            self.ctx = None
        if getattr(self, "gguf", None) is not None:
            self.gguf.close()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def batch_config(**overrides):
    """The launcher's batching settings (eg2_batch_config_default), with overrides."""
    cfg = BatchConfig()
    lib().eg2_batch_config_default(C.byref(cfg))
    for k, v in overrides.items():
        setattr(cfg, k, v)
    return cfg


def pack_waves(lengths, cfg=None):
    """eg2_pack_waves: the list of waves, each a list of sequence indices in
    execution order."""
    n = len(lengths)
    arr = (C.c_size_t * max(n, 1))(*[int(x) for x in lengths])
    order = (C.c_size_t * max(n, 1))()
    ends = (C.c_size_t * max(n, 1))()
    cfg = cfg or batch_config()
    w = lib().eg2_pack_waves(arr, n, C.byref(cfg), order, ends)
    if n and not w:
        raise HipError("eg2_pack_waves rejected its arguments")
    waves, b = [], 0
    for i in range(w):
        waves.append(list(order[b:ends[i]]))
        b = ends[i]
    return waves


def normalize_prefix(embedding, dims):
    """eg2_normalize_prefix on a copy of a 768-float embedding."""
    import numpy as np

    e = np.ascontiguousarray(embedding, dtype=np.float32).copy()
    if not lib().eg2_normalize_prefix(e.ctypes.data_as(_f), dims):
        raise HipError(f"unsupported dims {dims}")
    return e


def rope_table(base, n_pos=N_CTX):
    import numpy as np

    t = np.zeros((n_pos, HEAD_DIM), dtype=np.float32)
    lib().eg2_rope_table(base, n_pos, t.ctypes.data)
    return t


def q8_tile_bytes(rows, k):
    """Bytes of a Q8_0 row-tile buffer (rows rounded up to 32)."""
    return lib().eg2_q8_tile_bytes(rows, k)


def q8_pack_rows(q):
    """int8 [rows, k] -> the row-tile layout (flat int8, padding rows zero)."""
    import numpy as np

    q = np.ascontiguousarray(q, dtype=np.int8)
    rows, k = q.shape
    tiles = np.zeros(q8_tile_bytes(rows, k), dtype=np.int8)
    lib().eg2_q8_pack_rows(q.ctypes.data, rows, k, tiles.ctypes.data)
    return tiles


def q8_unpack_rows(tiles, rows, k):
    """Row-tile bytes -> int8 [rows, k]."""
    import numpy as np

    tiles = np.ascontiguousarray(tiles).view(np.int8)
    assert tiles.size >= q8_tile_bytes(rows, k)
    q = np.zeros((rows, k), dtype=np.int8)
    lib().eg2_q8_unpack_rows(tiles.ctypes.data, rows, k, q.ctypes.data)
    return q


def q8_weight_tiles(blocks_u8, rows, k):
    """GGUF Q8_0 bytes [rows, k] -> the projection GEMM's weight operands
    (wq: int8 row tiles, flat; wd: float32 block scales [k/32, ldw], ldw =
    rows rounded up to 32)."""
    import numpy as np

    src = np.ascontiguousarray(blocks_u8, dtype=np.uint8)
    wq = np.zeros(q8_tile_bytes(rows, k), dtype=np.int8)
    wd = np.zeros((k // 32, (rows + 31) // 32 * 32), dtype=np.float32)
    lib().eg2_q8_weight_tiles(src.ctypes.data, rows, k, wq.ctypes.data, wd.ctypes.data)
    return wq, wd


def q8_geglu_weight_tiles(gate_u8, up_u8, ff, k):
    """GGUF Q8_0 gate and up bytes [ff, k] -> the operands of the fused
    gate|up + GeGLU GEMM (rows interleaved in 32-row groups; wq int8 row
    tiles, flat; wd float32 [k/32, 2 ff])."""
    import numpy as np

    g = np.ascontiguousarray(gate_u8, dtype=np.uint8)
    u = np.ascontiguousarray(up_u8, dtype=np.uint8)
    if g.size != ff * (k // 32) * 34 or u.size != g.size:
        raise ValueError("gate/up must hold ff x k Q8_0 values each")
    wq = np.zeros(q8_tile_bytes(2 * ff, k), dtype=np.int8)
    wd = np.zeros((k // 32, 2 * ff), dtype=np.float32)
    if lib().eg2_q8_geglu_weight_tiles(g.ctypes.data, u.ctypes.data, ff, k, wq.ctypes.data, wd.ctypes.data):
        raise ValueError("ff and k must be multiples of 32")
    return wq, wd


def f32_to_chars(value):
    """eg2_f32_to_chars: the shortest round-trip text of a float32 (None
    for a non-finite value)."""
    buf = C.create_string_buffer(32)
    n = lib().eg2_f32_to_chars(buf, C.c_float(value))
    return buf.raw[:n].decode() if n else None


def base64_f32(values):
    """eg2_base64_f32 of a float32 array."""
    import numpy as np

    v = np.ascontiguousarray(values, dtype=np.float32).ravel()
    buf = C.create_string_buffer(4 * ((4 * v.size + 2) // 3) + 1)
    n = lib().eg2_base64_f32(v.ctypes.data_as(_f), v.size, buf)
    return buf.raw[:n].decode()


def embeddings_response(embeddings, dims, api="ollama", encoding="float", model="", prompt_tokens=0):
    """eg2_embeddings_response: the response body for [n, 768] embeddings
    (normalised to their first `dims` values on a copy)."""
    import numpy as np

    e = np.array(embeddings, dtype=np.float32, copy=True, order="C").reshape(-1, N_EMBD)
    m = model.encode() if isinstance(model, str) else bytes(model)
    cap = lib().eg2_embeddings_response_bound(e.shape[0], dims, len(m))
    buf = C.create_string_buffer(cap + 1)
    n = lib().eg2_embeddings_response(e.ctypes.data_as(_f), e.shape[0], dims, {"ollama": 0, "openai": 1}[api],
                                      {"float": 0, "base64": 1}[encoding], m, len(m), prompt_tokens, buf, cap + 1)
    if n == 0:
        raise ValueError("embedding response failed (dims, non-finite value)")
    return buf.raw[:n].decode()


def attention_capacity(tokens, batch):
    """(items, score floats): eg2_attention_capacity."""
    counts = (C.c_size_t * 2)()
    lib().eg2_attention_capacity(tokens, batch, counts)
    return int(counts[0]), int(counts[1])


def attention_plan(offsets, rows=None):
    """(items uint32 [n, 8], tok uint32 [rows, 4], score floats, score item
    count) of the sequences [offsets[s], offsets[s+1]) (eg2_attention_plan):
    the score items, then the context items; rows defaults to offsets[-1],
    and every row must belong to a sequence."""
    import numpy as np

    offs = (C.c_size_t * len(offsets))(*[int(o) for o in offsets])
    total, batch = int(offsets[-1]), len(offsets) - 1
    rows = total if rows is None else rows
    cap_items, cap_scores = attention_capacity(max(total, 1), max(batch, 1))
    items = np.zeros((cap_items, 8), dtype=np.uint32)
    tok = np.zeros((max(rows, total, 1), 4), dtype=np.uint32)
    counts = (C.c_size_t * 3)()
    rc = lib().eg2_attention_plan(offs, batch, cap_items, cap_scores, items.ctypes.data, tok.ctypes.data, counts)
    if rc != 0:
        raise HipError("attention plan exceeds its capacity")
    return items[:counts[0]], tok[:rows], int(counts[1]), int(counts[2])


class AttentionPlan:
    """The attention plan of a packing on the device (work items, their two
    counts, token records) and its scores scratch."""

    GRID = 1024  # workgroups striding over each item list (the executor's choice)

    def __init__(self, offsets, device, rows=None):
        import numpy as np
        import torch

        items, tok, score_floats, score_items = attention_plan(offsets, rows)
        self.n_items = len(items)
        self.items = torch.from_numpy(np.ascontiguousarray(items).view(np.int32).reshape(-1).copy()
                                      if len(items) else np.zeros(8, np.int32)).to(device)
        self.count = torch.tensor([score_items, len(items) - score_items], dtype=torch.int32, device=device)
        self.tok = torch.from_numpy(np.ascontiguousarray(tok).view(np.int32).reshape(-1).copy()).to(device)
        self.scores = torch.zeros(max(1, score_floats), dtype=torch.float32, device=device)
        self.rows = tok.shape[0]
        self.longest = max(int(offsets[i + 1]) - int(offsets[i]) for i in range(len(offsets) - 1))


class ops:
    """Operator entry points on torch device tensors (current torch stream)."""

    @staticmethod
    def _stream():
        import torch

        return C.c_void_p(torch.cuda.current_stream().cuda_stream)

    @staticmethod
    def _p(t):
        return C.c_void_p(t.data_ptr()) if t is not None else None

    @classmethod
    def embed_norm_quant(cls, table, ids, embed_scale, norm_w, eps, x, xq, xd):
        check(lib().eg2_hip_embed_norm_quant(cls._p(table), cls._p(ids), ids.numel(), embed_scale, cls._p(norm_w),
                                             eps, cls._p(x), cls._p(xq), cls._p(xd), cls._stream()),
              "embed_norm_quant")

    @classmethod
    def residual_norm_quant(cls, x, h, post_w, next_w, eps, xq, xd):
        check(lib().eg2_hip_residual_norm_quant(cls._p(x), cls._p(h), cls._p(post_w), cls._p(next_w), eps,
                                                cls._p(xq), cls._p(xd), x.shape[0], cls._stream()),
              "residual_norm_quant")

    @classmethod
    def qk_norm_rope(cls, qkv, q_w, k_w, table, pos, eps, out):
        """Rows [q0 q1 q2 | k | v] of qkv normalised / rotated into out (may be qkv)."""
        check(lib().eg2_hip_qk_norm_rope(cls._p(qkv), cls._p(q_w), cls._p(k_w), cls._p(table), cls._p(pos), eps,
                                         cls._p(out), qkv.shape[0], cls._stream()), "qk_norm_rope")

    @classmethod
    def gemm_q8_qkv_rope(cls, xq, xd, wq, wd, n, q_w, k_w, table, pos, eps, out):
        """The QKV projection of n rows (xq/xd as for gemm_q8, weights of the
        [q|k|v] concatenation) followed by qk_norm_rope, in one kernel, into
        out [n, 1280]."""
        check(lib().eg2_hip_gemm_q8_qkv_rope(cls._p(xq), cls._p(xd), xd.shape[1], cls._p(wq), cls._p(wd),
                                             wd.shape[1], n, 32 * xd.shape[0], cls._p(q_w), cls._p(k_w),
                                             cls._p(table), cls._p(pos), eps, cls._p(out), cls._stream()),
              "gemm_q8_qkv_rope")

    @classmethod
    def attention(cls, qkv, offsets, window, cq, cd):
        """Packed attention over sequences [offsets[s], offsets[s+1]) of the
        rows [q0 q1 q2 | k | v] of qkv (rows a multiple of 4 covered by the
        sequences), the context quantized into cq / cd."""
        import torch

        plan = AttentionPlan(offsets, qkv.device, qkv.shape[0])
        cls.attention_planned(qkv, plan, window, cq, cd)
        torch.cuda.current_stream().synchronize()  # keeps the plan alive until the kernels ran

    @classmethod
    def attention_planned(cls, qkv, plan, window, cq, cd, longest=None):
        """attention() with a prebuilt AttentionPlan (no host work, no sync);
        longest overrides the plan's longest sequence (0 = the softmax form
        for any length)."""
        check(lib().eg2_hip_attention(cls._p(qkv), cls._p(plan.items), cls._p(plan.count), plan.GRID,
                                      cls._p(plan.tok), window, qkv.shape[0],
                                      plan.longest if longest is None else longest, cls._p(plan.scores),
                                      cls._p(cq), cls._p(cd), cls._stream()), "attention")

    @classmethod
    def attention_stage(cls, stage, qkv, plan, window, cq=None, cd=None, longest=None):
        """One of attention_planned's three kernels stages ("scores",
        "softmax", "context"), for timing them one by one."""
        longest = plan.longest if longest is None else longest
        L = lib()
        if stage == "scores":
            rc = L.eg2_hip_attention_scores(cls._p(qkv), cls._p(plan.items), cls._p(plan.count), plan.GRID, window,
                                            qkv.shape[0], cls._p(plan.scores), cls._stream())
        elif stage == "softmax":
            rc = L.eg2_hip_attention_softmax(cls._p(plan.tok), window, qkv.shape[0], longest, cls._p(plan.scores),
                                             cls._stream())
        elif stage == "context":
            rc = L.eg2_hip_attention_context(cls._p(qkv), cls._p(plan.items), cls._p(plan.count), plan.GRID, window,
                                             qkv.shape[0], cls._p(plan.scores), cls._p(cq), cls._p(cd),
                                             cls._stream())
        else:
            raise ValueError(stage)
        check(rc, "attention_" + stage)

    STATIC_ROWS, STATIC_BATCH = 2048, 2048  # EG2_ATTENTION_STATIC_ROWS / _BATCH

    @classmethod
    def attention_static(cls, qkv, offsets_d, window, cq, cd):
        """attention() through the allocation-free entry point: offsets_d is
        a device uint32/int32 tensor of the batch + 1 sequence bounds; the
        plan is built on the device into the library's static array."""
        rows, batch = qkv.shape[0], offsets_d.numel() - 1
        if rows > cls.STATIC_ROWS or batch > cls.STATIC_BATCH or batch < 1 or rows % 4:
            raise ValueError(f"attention_static: rows {rows} (at most {cls.STATIC_ROWS}, a multiple of 4) and "
                             f"batch {batch} (1 to {cls.STATIC_BATCH}) exceed the static scratch's limits")
        check(lib().eg2_hip_attention_static(cls._p(qkv), cls._p(offsets_d), batch, window, rows, cls._p(cq),
                                             cls._p(cd), cls._stream()), "attention_static")

    @classmethod
    def gelu_quant(cls, gu, gq, gd):
        check(lib().eg2_hip_gelu_quant(cls._p(gu), cls._p(gq), cls._p(gd), gu.shape[0], cls._stream()),
              "gelu_quant")

    @classmethod
    def quantize_rows(cls, x, q, d):
        check(lib().eg2_hip_quantize_rows(cls._p(x), x.shape[1], cls._p(q), cls._p(d), x.shape[0], cls._stream()),
              "quantize_rows")

    @classmethod
    def rms_norm_rows(cls, x, w, eps):
        check(lib().eg2_hip_rms_norm_rows(cls._p(x), cls._p(w), eps, x.shape[0], cls._stream()), "rms_norm_rows")

    @classmethod
    def pool_l2(cls, x, offsets, out):
        check(lib().eg2_hip_pool_l2(cls._p(x), cls._p(offsets), cls._p(out), out.shape[0], cls._stream()),
              "pool_l2")

    @classmethod
    def pool_mean(cls, x, offsets, out):
        check(lib().eg2_hip_pool_mean(cls._p(x), cls._p(offsets), cls._p(out), out.shape[0], cls._stream()),
              "pool_mean")

    @classmethod
    def l2_prefix(cls, x, dims):
        check(lib().eg2_hip_l2_prefix(cls._p(x), x.shape[1], dims, x.shape[0], cls._stream()), "l2_prefix")

    @classmethod
    def op(cls, name, record, grid, block):
        """Launches operator `name` (include/eg2_ops.h) with a record from
        this module; `grid` is a workgroup count or an (x, y) pair."""
        gx, gy = (grid, 1) if isinstance(grid, int) else grid
        check(lib().eg2_op_launch(name.encode(), C.byref(record), C.sizeof(record), gx, gy, block, cls._stream()),
              name)

    @classmethod
    def gemm_q8(cls, xq, xd, wq, wd, y, m=None):
        """y[:, :m] = xq . W^T: xq int8 row tiles of y.shape[0] rows with the
        activation scales xd [k/32, ldx]; (wq, wd) the weights from
        q8_weight_tiles (m defaults to y's width)."""
        n = y.shape[0]
        k = 32 * xd.shape[0]
        m = y.shape[1] if m is None else m
        check(lib().eg2_hip_gemm_q8(cls._p(xq), cls._p(xd), xd.shape[1], cls._p(wq), cls._p(wd), wd.shape[1],
                                    cls._p(y), n, m, k, y.shape[1], cls._stream()), "gemm_q8")

    @classmethod
    def gemm_q8_geglu(cls, xq, xd, wq, wd, gq, gd, n):
        """gq/gd = Q8_0 of gelu(gate) * up for n rows of xq (int8 row tiles,
        scales xd [k/32, ldx]); (wq, wd) from q8_geglu_weight_tiles; gd is
        [ff/32, ldg] and gq the row tiles of ff values per row."""
        k = 32 * xd.shape[0]
        ff = 32 * gd.shape[0]
        check(lib().eg2_hip_gemm_q8_geglu(cls._p(xq), cls._p(xd), xd.shape[1], cls._p(wq), cls._p(wd), wd.shape[1],
                                          cls._p(gq), cls._p(gd), gd.shape[1], n, ff, k, cls._stream()),
              "gemm_q8_geglu")

    # ---- block operators: any geometry, fp32 / fp16 / bf16 (include/eg2_hip.h). They run on the current
    # stream of their tensors' device. A call's checks and its record are most of a small call's time: all that must hold
    # is one condition, and what is wrong is looked for only when something is.

    @staticmethod
    def _types():
        """(ids of the activation types, torch's float32, int32, uint8, the current raw stream of a device, torch.cuda)."""
        global _torch_types
        if _torch_types is None:
            import torch

            raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)  # the number alone, without its object
            _torch_types = ({torch.float32: TYPE_F32, torch.float16: TYPE_F16, torch.bfloat16: TYPE_BF16},
                            torch.float32, torch.int32, torch.uint8,
                            raw or (lambda device: torch.cuda.current_stream(device).cuda_stream), torch.cuda)
        return _torch_types

    @staticmethod
    def _refuse(what, **tensors):
        """Raises for tensors that do not fit together."""
        said = ", ".join(f"{name} {tuple(t.shape)} strides {t.stride()} {t.dtype} on {t.device}"
                         for name, t in tensors.items() if t is not None)
        raise ValueError(f"{what}: not tensors of one GPU whose sizes and types fit, with dense last dimensions: {said}")

    @classmethod
    def _vector(cls, t, what, name, n, dtype, device):
        """The address of a dense vector of n values of a type on the device; None: 0."""
        if t is None:
            return 0
        if t.dtype is not dtype or t.shape != (n,) or not t.is_contiguous() or t.get_device() != device:
            raise ValueError(f"{what}: {name} is not {n} dense values of {dtype} on the same GPU: {tuple(t.shape)} {t.dtype} "
                             f"on {t.device}")
        return t.data_ptr()

    @staticmethod
    def _launch(what, entry, record, device):
        _, _, _, _, stream_of, cuda = _torch_types
        stream = stream_of(device)
        if cuda.current_device() == device:
            code = entry(record, stream)
        else:
            with cuda.device(device):
                code = entry(record, stream)
        if code:
            check(code, what)

    @classmethod
    def _product(cls, what, x, w, y, act):
        """(n, k, m, type id, type id and strides of the weights, strides of x and y, activation id, GPU)."""
        ids, _, _, uint8, _, _ = _torch_types or cls._types()
        act_id = ACTIVATIONS.get(act)
        if act_id is None:
            raise ValueError(f"{what}: no activation {act!r}")
        if not x.dim() == w.dim() == y.dim() == 2:
            cls._refuse(what, x=x, weight=w, y=y)
        (n, k), (ldx, x1), (wm, wk), (ldw, w1) = x.shape, x.stride(), w.shape, w.stride()
        (rows, m), (ldy, y1) = y.shape, y.stride()
        dtype, device = x.dtype, x.get_device()
        kind, wkind = ids.get(dtype), ids.get(w.dtype)
        if w.dtype is uint8:  # rows of Q8_0 blocks, 34 bytes for 32 values
            wkind, dense = TYPE_Q8_0, k % 32 == 0 and wk == k // 32 * 34 and (wm == 1 or ldw % 34 == 0)
            ldw = ldw // 34 * 32
        else:
            dense = wk == k and (kind == TYPE_F32 or wkind == kind)
        if (kind is None or wkind is None or not dense or rows != n or wm != m or y.dtype is not dtype or
                (x1 != 1 and k > 1) or (w1 != 1 and wk > 1) or (y1 != 1 and m > 1) or
                not y.get_device() == w.get_device() == device or device < 0):
            cls._refuse(what, x=x, weight=w, y=y)
        return (n, k, m, kind, wkind, ldx if n > 1 else k, ldw if m > 1 else k, ldy if n > 1 else m, act_id, device)

    @classmethod
    def linear(cls, x, weight, y, bias=None, act="none", residual=None):
        """y = act(x . weight^T + bias) + residual (eg2_hip_linear): x [n, k],
        weight [m, k] or uint8 [m, 34 k / 32] of Q8_0 blocks, y [n, m], bias
        float32 [m], residual [n, m] (may be y); act "none", "gelu", "silu" or "relu"."""
        n, k, m, kind, wkind, ldx, ldw, ldy, act, device = cls._product("linear", x, weight, y, act)
        res = ldr = 0
        if residual is not None:
            if (residual.shape != y.shape or residual.dtype is not y.dtype or residual.get_device() != device or
                    (residual.stride(1) != 1 and m > 1)):
                cls._refuse("linear", y=y, residual=residual)
            res, ldr = residual.data_ptr(), residual.stride(0) if n > 1 else m
        if bias is not None:
            bias = cls._vector(bias, "linear", "bias", m, _torch_types[1], device)
        record = LinearArgs.pack(y.data_ptr(), x.data_ptr(), weight.data_ptr(), bias or 0, res, ldx, ldw, ldy, ldr, n, k,
                                 m, kind, wkind, act)
        cls._launch("linear", lib().eg2_hip_linear, record, device)

    @classmethod
    def linear_gated(cls, x, gate, up, y, gate_bias=None, up_bias=None, act="gelu"):
        """y = act(x . gate^T + gate_bias) * (x . up^T + up_bias)
        (eg2_hip_linear_gated): the arguments of linear, gate and up alike."""
        what = "linear_gated"
        n, k, m, kind, wkind, ldx, ldw, ldy, act, device = cls._product(what, x, gate, y, act)
        if (up.shape != gate.shape or up.stride() != gate.stride() or up.dtype is not gate.dtype or
                up.get_device() != device):
            cls._refuse(what, gate=gate, up=up)
        float32 = _torch_types[1]
        record = LinearGatedArgs.pack(y.data_ptr(), x.data_ptr(), gate.data_ptr(), up.data_ptr(),
                                      cls._vector(gate_bias, what, "gate_bias", m, float32, device),
                                      cls._vector(up_bias, what, "up_bias", m, float32, device), ldx, ldw, ldy, n, k, m,
                                      kind, wkind, act)
        cls._launch(what, lib().eg2_hip_linear_gated, record, device)

    @classmethod
    def heads_norm_rope(cls, q, k, q_w, k_w, table, pos, eps, q_out, k_out, q_scale=1.0):
        """Every head of q [rows, heads, d] and k [rows, kv_heads, d] (k and
        k_out may be None) RMS-normalised, times q_w / k_w (float32 [d] or None),
        rotated by table[pos] (float32 [positions, rotary] as rope_table, int32
        [rows]; both None: not rotated) and, of q, scaled, into q_out and k_out,
        which may be q and k (eg2_hip_heads_norm_rope)."""
        what = "heads_norm_rope"
        ids, float32, int32, _, _, _ = _torch_types or cls._types()
        if q.dim() != 3 or q_out.dim() != 3:
            cls._refuse(what, q=q, q_out=q_out)
        dtype, device, shape = q.dtype, q.get_device(), q.shape
        kind = ids.get(dtype)
        (rows, heads, d), (q_row, q_head, q1), (qo_row, qo_head, qo1) = shape, q.stride(), q_out.stride()
        if (kind is None or q_out.shape != shape or q_out.dtype is not dtype or ((q1 != 1 or qo1 != 1) and d > 1) or
                q_out.get_device() != device or device < 0):
            cls._refuse(what, q=q, q_out=q_out)
        kp = kop = k_heads = k_row = k_head = ko_row = ko_head = 0
        if (k is None) != (k_out is None):
            raise ValueError(f"{what}: k and k_out go together")
        if k is not None:
            if k.dim() != 3 or k_out.dim() != 3:
                cls._refuse(what, k=k, k_out=k_out)
            (k_rows, k_heads, k_d), (k_row, k_head, k1), (ko_row, ko_head, ko1) = k.shape, k.stride(), k_out.stride()
            if (k_rows != rows or k_d != d or k_out.shape != k.shape or not k.dtype is k_out.dtype is dtype or
                    ((k1 != 1 or ko1 != 1) and d > 1) or not k.get_device() == k_out.get_device() == device):
                cls._refuse(what, q=q, k=k, k_out=k_out)
            kp, kop = k.data_ptr(), k_out.data_ptr()
        if (table is None) != (pos is None):
            raise ValueError(f"{what}: table and pos go together")
        tp = at = positions = rotary = 0
        if table is not None:
            if table.dim() != 2 or table.dtype is not float32 or not table.is_contiguous() or table.get_device() != device:
                cls._refuse(what, q=q, table=table)
            (positions, rotary), tp = table.shape, table.data_ptr()
            at = cls._vector(pos, what, "pos", rows, int32, device)
        record = HeadsNormRopeArgs.pack(q_out.data_ptr(), kop, q.data_ptr(), kp,
                                        cls._vector(q_w, what, "q_w", d, float32, device),
                                        cls._vector(k_w, what, "k_w", d, float32, device), tp, at, q_row, q_head, k_row,
                                        k_head, qo_row, qo_head, ko_row, ko_head, rows, heads, k_heads, d, rotary,
                                        positions, kind, eps, q_scale)
        cls._launch(what, lib().eg2_hip_heads_norm_rope, record, device)

    @classmethod
    def window_attention(cls, q, k, v, q_offsets, k_offsets, out, scale, left=-1, right=-1, sinks=0, k_lengths=None,
                         longest=0, workspace=None):
        """out = attention of q [rows, heads, d] over k and v [key rows,
        kv_heads, d] of the sequences that the int32 offsets (and lengths of keys) give,
        each query seeing `left` keys before its own, `right` after it (-1: all)
        and the first `sinks` (eg2_hip_window_attention). longest: the longest
        sequence of keys, a hint. workspace: a uint8 tensor of
        window_attention_workspace's bytes; by default one is taken from torch."""
        what = "window_attention"
        ids, _, int32, uint8, _, _ = _torch_types or cls._types()
        if not q.dim() == k.dim() == v.dim() == out.dim() == 3:
            cls._refuse(what, q=q, k=k, v=v, out=out)
        dtype, device, shape, k_shape = q.dtype, q.get_device(), q.shape, k.shape
        kind = ids.get(dtype)
        (rows, heads, d), (key_rows, kv_heads, k_d) = shape, k_shape
        (q_row, q_head, q1), (k_row, k_head, k1) = q.stride(), k.stride()
        (v_row, v_head, v1), (out_row, out_head, out1) = v.stride(), out.stride()
        if (kind is None or k_d != d or v.shape != k_shape or out.shape != shape or
                not k.dtype is v.dtype is out.dtype is dtype or not q1 == k1 == v1 == out1 == 1 or
                not k.get_device() == v.get_device() == out.get_device() == device or device < 0):
            cls._refuse(what, q=q, k=k, v=v, out=out)
        if heads == 1:  # the strides of a dimension of one are anything
            q_head, out_head = d, d
        if kv_heads == 1:
            k_head, v_head = d, d
        if rows == 1:
            q_row, out_row = heads * d, heads * d
        if key_rows == 1:
            k_row, v_row = kv_heads * d, kv_heads * d
        batch = q_offsets.numel() - 1
        if batch < 0 or sinks < 0 or longest < 0:
            raise ValueError(f"{what}: no offsets, or sinks {sinks} or longest {longest} below 0")
        qo = cls._vector(q_offsets, what, "q_offsets", batch + 1, int32, device)
        ko = qo if k_offsets is q_offsets else cls._vector(k_offsets, what, "k_offsets", batch + 1, int32, device)
        kl = 0 if k_lengths is None else cls._vector(k_lengths, what, "k_lengths", batch, int32, device)
        fields = [out.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), qo, ko, kl, 0, 0, q_row, q_head, k_row, k_head,
                  v_row, v_head, out_row, out_head, batch, rows, key_rows, heads, kv_heads, d, kind, left, right, sinks,
                  longest, scale]
        record = WindowAttentionArgs.pack(*fields)
        if workspace is None:
            need = lib().eg2_hip_window_attention_workspace(record)
            if need:  # torch keeps it for this stream until the kernels are done
                import torch

                workspace = torch.empty(need, dtype=uint8, device=q.device)
        if workspace is not None:
            fields[8] = workspace.numel()
            fields[7] = cls._vector(workspace, what, "workspace", fields[8], uint8, device)
            record = WindowAttentionArgs.pack(*fields)
        cls._launch(what, lib().eg2_hip_window_attention, record, device)

    @classmethod
    def window_attention_workspace(cls, batch, rows, key_rows, heads, kv_heads, d, dtype, left=-1, right=-1, sinks=0,
                                   longest=0):
        """Bytes of workspace of a window_attention call of these sizes."""
        kind = cls._types()[0].get(dtype)
        if kind is None:
            raise ValueError(f"window_attention_workspace: {dtype} is not float32, float16 or bfloat16")
        return lib().eg2_hip_window_attention_workspace(
            WindowAttentionArgs.pack(*(0,) * 9, *(0,) * 8, batch, rows, key_rows, heads, kv_heads, d, kind, left, right,
                                     sinks, longest, 1.0))
