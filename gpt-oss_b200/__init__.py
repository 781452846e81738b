"""B200 (sm_100a) engine for the GPT-OSS MoE block: Python binding of the C ABI.

The product is ``libgptoss_moe_b200.so`` (CUDA kernels + ``extern "C"`` layer,
declared in ``include/gptoss_moe_b200.h``).  This module only loads it through
``ctypes`` and wraps the handle in :class:`MoeEngine`, whose methods map one to
one onto the C entry points.  There is no CPU fallback: loading fails loudly
when the library has not been built, and every compute call fails with
``GPTOSS_E_CUDA`` when no sm_100 GPU is present.
"""
from __future__ import annotations

import ctypes
import pathlib
import struct

import numpy as np

PKG_DIR = pathlib.Path(__file__).resolve().parent
LIB_PATH = PKG_DIR / "libgptoss_moe_b200.so"
HEADER_PATH = PKG_DIR.parent / "include" / "gptoss_moe_b200.h"

GPTOSS_OK = 0
GPTOSS_E_INVALID = -1
GPTOSS_E_CUDA = -2
GPTOSS_E_CAPACITY = -3
GPTOSS_E_DEVICE = -4
GPTOSS_E_STATE = -5
GPTOSS_E_COMM = -6

WEIGHTS_BF16 = 0
WEIGHTS_MXFP4 = 1
GEMM_TCGEN05 = 0
GEMM_SIMT = 1
GEMM_PAIR = 2

STAGES = ("route", "permute", "gate_up", "down", "combine", "dispatch", "return")


class MoeConfig(ctypes.Structure):
    """Mirror of gptoss_moe_config_t."""

    _fields_ = [
        ("hidden_dim", ctypes.c_int),
        ("intermediate_dim", ctypes.c_int),
        ("n_experts", ctypes.c_int),
        ("experts_per_token", ctypes.c_int),
        ("n_layers", ctypes.c_int),
        ("max_tokens", ctypes.c_int),
        ("swiglu_limit", ctypes.c_float),
        ("ep_rank", ctypes.c_int),
        ("ep_size", ctypes.c_int),
        ("weight_format", ctypes.c_int),
        ("device", ctypes.c_int),
    ]


class MoeError(RuntimeError):
    def __init__(self, code: int, text: str):
        super().__init__(f"gptoss_moe error {code}: {text}")
        self.code = code


class ModelConfig(ctypes.Structure):
    """gptoss_model_config_t: the reference's Config / .bin header (run.cpp:26-46)."""
    _fields_ = [("vocab_size", ctypes.c_int), ("hidden_dim", ctypes.c_int),
                ("n_experts", ctypes.c_int), ("experts_per_token", ctypes.c_int),
                ("intermediate_dim", ctypes.c_int), ("n_layers", ctypes.c_int),
                ("head_dim", ctypes.c_int), ("n_attn_heads", ctypes.c_int),
                ("n_kv_heads", ctypes.c_int), ("seq_len", ctypes.c_int),
                ("initial_context_length", ctypes.c_int), ("rope_theta", ctypes.c_float),
                ("rope_scaling_factor", ctypes.c_float), ("sliding_window", ctypes.c_int),
                ("swiglu_limit", ctypes.c_float)]


class Sampling(ctypes.Structure):
    """Mirror of gptoss_decode_sampling_t."""
    _fields_ = [(n, ctypes.c_void_p) for n in ("u", "temperature", "top_k", "top_p", "min_p")]


class RopeArgs(ctypes.Structure):
    """Mirror of gptoss_rope_args_t."""
    _fields_ = [(n, ctypes.c_void_p) for n in ("q", "k", "v", "q_out", "k_cache", "v_cache", "pos",
                                               "slots", "inv_freq")] + \
               [(n, ctypes.c_longlong) for n in ("q_stride", "k_stride", "v_stride", "q_out_stride",
                                                 "k_cache_stride", "v_cache_stride", "n_slots")] + \
               [("concentration", ctypes.c_float)] + \
               [(n, ctypes.c_int) for n in ("n_rows", "n_q_heads", "n_kv_heads", "head_dim",
                                            "rotary_dim", "interleaved", "angle_f32", "dtype")]


class AttentionArgs(ctypes.Structure):
    """Mirror of gptoss_attention_args_t."""
    _fields_ = [(n, ctypes.c_void_p) for n in ("q", "k", "v", "out", "q_start", "kv_start", "kv_len",
                                               "sinks", "status")] + \
               [(n, ctypes.c_longlong) for n in ("q_stride", "k_stride", "v_stride", "out_stride",
                                                 "n_kv_rows")] + \
               [("scale", ctypes.c_float)] + \
               [(n, ctypes.c_int) for n in ("n_tokens", "n_seqs", "n_q_heads", "n_kv_heads",
                                            "head_dim", "window", "max_kv_len", "dtype")]


class SampleArgs(ctypes.Structure):
    """Mirror of gptoss_sample_args_t."""
    _fields_ = [(n, ctypes.c_void_p) for n in ("logits", "u", "temperature", "top_k", "top_p",
                                               "min_p", "pos", "next")] + \
               [("stride", ctypes.c_longlong)] + \
               [(n, ctypes.c_int) for n in ("n_rows", "vocab", "dtype")]


_lib = None


def load_library() -> ctypes.CDLL:
    """Load the native library (once).  Raises if it has not been built."""
    global _lib
    if _lib is not None:
        return _lib
    if not LIB_PATH.exists():
        raise RuntimeError(
            f"{LIB_PATH} is missing: build it with `python -c 'import __graft_entry__ as g; "
            "g.build()'` (there is no fallback path)"
        )
    lib = ctypes.CDLL(str(LIB_PATH))
    vp, ip, fp = ctypes.c_void_p, ctypes.POINTER(ctypes.c_int), ctypes.POINTER(ctypes.c_float)
    c_int, c_char_p = ctypes.c_int, ctypes.c_char_p
    sigs = {
        "gptoss_moe_create": (c_int, [ctypes.POINTER(MoeConfig), ctypes.POINTER(vp)]),
        "gptoss_moe_destroy": (c_int, [vp]),
        "gptoss_moe_last_error": (c_char_p, [vp]),
        "gptoss_moe_load_layer_f32": (c_int, [vp, c_int, vp, vp, vp, vp, vp, vp]),
        "gptoss_moe_load_layer_bf16": (c_int, [vp, c_int, vp, vp, vp, vp, vp, vp, c_int]),
        "gptoss_moe_load_layer_mxfp4": (
            c_int,
            [vp, c_int, vp, vp, vp, vp, vp, vp, vp, vp, c_int],
        ),
        "gptoss_moe_forward": (c_int, [vp, c_int, vp, vp, vp, c_int, vp]),
        "gptoss_moe_forward_host": (c_int, [vp, c_int, vp, vp, vp, c_int]),
        "gptoss_moe_forward_host_submit": (c_int, [vp, c_int, vp, vp, vp, c_int, ip]),
        "gptoss_moe_forward_host_wait": (c_int, [vp, c_int]),
        "gptoss_moe_load_ffn_norm": (c_int, [vp, c_int, vp]),
        "gptoss_moe_route": (c_int, [vp, c_int, vp, vp, c_int, vp]),
        "gptoss_moe_permute": (c_int, [vp, vp, c_int, vp]),
        "gptoss_moe_experts": (c_int, [vp, c_int, vp]),
        "gptoss_moe_combine": (c_int, [vp, vp, c_int, vp]),
        "gptoss_moe_rmsnorm": (c_int, [vp, vp, vp, vp, vp, c_int, vp]),
        "gptoss_moe_get_routing": (c_int, [vp, c_int, vp, vp, vp, vp, vp]),
        "gptoss_moe_get_activations": (c_int, [vp, vp, ctypes.c_size_t]),
        "gptoss_moe_set_option": (c_int, [vp, c_char_p, c_int]),
        "gptoss_moe_launch_count": (ctypes.c_longlong, [vp]),
        "gptoss_moe_device_status": (c_int, [vp]),
        "gptoss_moe_stage_ms": (c_int, [vp, c_int, fp]),
        "gptoss_moe_ep_unique_id": (c_int, [vp]),
        "gptoss_moe_ep_init": (c_int, [vp, vp]),
        "gptoss_moe_ep_transport": (c_int, [vp]),
        "gptoss_moe_ep_init_local": (c_int, [ctypes.POINTER(vp), c_int]),
        "gptoss_moe_forward_part": (c_int, [vp, c_int, c_int, vp, vp, vp, c_int, vp]),
        "gptoss_moe_version": (c_char_p, []),
        "gptoss_moe_permute_static": (c_int, [vp, vp, c_int, c_int, c_int, vp, vp, vp, vp, vp]),
        "gptoss_decode_create": (c_int, [ctypes.POINTER(ModelConfig), c_int, c_int,
                                         ctypes.POINTER(vp)]),
        "gptoss_decode_destroy": (c_int, [vp]),
        "gptoss_decode_last_error": (c_char_p, [vp]),
        "gptoss_decode_load_bin": (c_int, [vp, vp]),
        "gptoss_decode_load_weights": (c_int, [vp, vp]),
        "gptoss_decode_step": (c_int, [vp, vp, vp, c_int, vp, vp]),
        "gptoss_decode_get_logits": (c_int, [vp, c_int, vp]),
        "gptoss_decode_moe": (vp, [vp]),
        "gptoss_decode_device_count": (c_int, []),
        "gptoss_decode_create_ep": (c_int, [ctypes.POINTER(ModelConfig), c_int, c_int, c_int, c_int,
                                            ctypes.POINTER(vp)]),
        "gptoss_decode_set_tensor": (c_int, [vp, c_char_p, c_int, vp, c_int, c_int]),
        "gptoss_decode_set_kv": (c_int, [vp, c_int, c_int, c_int, c_int, c_int, vp, vp]),
        "gptoss_decode_get_kv": (c_int, [vp, c_int, c_int, c_int, c_int, c_int, vp, vp]),
        "gptoss_decode_create_prefill": (c_int, [ctypes.POINTER(ModelConfig), c_int, c_int, c_int,
                                                 ctypes.POINTER(vp)]),
        "gptoss_decode_step_sample": (c_int, [vp, vp, vp, c_int, ctypes.POINTER(Sampling), vp, vp]),
        "gptoss_decode_prefill": (c_int, [vp, vp, vp, vp, vp, c_int, ctypes.POINTER(Sampling), vp, vp]),
        "gptoss_decode_rope_table": (c_int, [c_int, ctypes.c_float, ctypes.c_float, c_int, vp, fp]),
        "gptoss_decode_rope_append": (c_int, [vp, vp]),
        "gptoss_decode_prompt_attention": (c_int, [vp, vp]),
        "gptoss_decode_sample": (c_int, [vp, vp]),
    }
    for name, (res, args) in sigs.items():
        fn = getattr(lib, name)
        fn.restype = res
        fn.argtypes = args
    _lib = lib
    return lib


def _ptr(obj):
    """Raw address of a torch tensor, numpy array, int or None."""
    if obj is None:
        return None
    if isinstance(obj, int):
        return ctypes.c_void_p(obj)
    if isinstance(obj, np.ndarray):
        if not obj.flags["C_CONTIGUOUS"]:
            raise ValueError("array must be C-contiguous")
        return ctypes.c_void_p(obj.ctypes.data)
    if hasattr(obj, "data_ptr"):
        if not obj.is_contiguous():
            raise ValueError("tensor must be contiguous")
        return ctypes.c_void_p(obj.data_ptr())
    raise TypeError(f"cannot take the address of {type(obj)}")


def permute_static(slot_expert, slot_weight, n_rows, top_k, n_experts, expert_offsets, sorted_row,
                   sorted_weight, row_of, stream=0):
    """gptoss_moe_permute_static: the permutation stage without an engine handle and
    without any allocation (scratch is a fixed array inside the library).  All
    arguments are device buffers owned by the caller."""
    lib = load_library()
    rc = lib.gptoss_moe_permute_static(_ptr(slot_expert), _ptr(slot_weight), n_rows, top_k,
                                       n_experts, _ptr(expert_offsets), _ptr(sorted_row),
                                       _ptr(sorted_weight), _ptr(row_of), ctypes.c_void_p(stream))
    if rc != GPTOSS_OK:
        raise MoeError(rc, lib.gptoss_moe_last_error(None).decode())


# -- the handle-free operators of a prompt pass and of a drawn token.  A decode step calls them
# for every layer, so the checks are kept cheap: dtypes are compared by identity, devices by
# index, and the argument structs are packed rather than filled field by field.
_DTYPE_CODES = {}
_ROPE_PACK = struct.Struct("@9P7qf8i0q").pack
_ATTENTION_PACK = struct.Struct("@9P5qf8i0q").pack
_SAMPLE_PACK = struct.Struct("@8Pq3i0q").pack


def _dtype_codes():
    """torch dtype -> GPTOSS_DTYPE_*, filled on the first call (the callers pass torch tensors)."""
    if not _DTYPE_CODES:
        import torch

        _DTYPE_CODES.update({torch.bfloat16: 0, torch.float16: 1, torch.float32: 2,
                             "int32": torch.int32, "int64": torch.int64, "float32": torch.float32})
    return _DTYPE_CODES


def _check_op(lib, rc):
    if rc != GPTOSS_OK:
        raise MoeError(rc, (lib.gptoss_decode_last_error(None) or b"").decode())


def _dtype_code(t, what):
    code = _dtype_codes().get(t.dtype)
    if code is None:
        raise TypeError(f"{what}: element type {t.dtype} is not supported")
    return code


def _vector(t, what, dtype, n, device):
    """Address of a contiguous 1-D tensor of n elements (0 for None)."""
    if t is None:
        return 0
    if (t.dtype is not dtype or t.dim() != 1 or t.shape[0] != n or not t.is_contiguous()
            or t.get_device() != device):
        if t.dtype is not dtype:
            raise TypeError(f"{what} must be {dtype}, not {t.dtype}")
        if t.get_device() != device:
            raise ValueError(f"{what} is on {t.device}, expected cuda:{device}")
        raise ValueError(f"{what} must be contiguous with {n} elements, not {tuple(t.shape)}")
    return t.data_ptr()


def _rows(t, what, dtype, device, heads, head_dim):
    """(address, row stride, rows) of a [rows, heads, head_dim] tensor with contiguous heads."""
    if t is None:
        return 0, 0, 0
    if t.dtype is not dtype:
        raise TypeError(f"{what} must be {dtype}, not {t.dtype}")
    if t.get_device() != device:
        raise ValueError(f"{what} is on {t.device}, expected cuda:{device}")
    if t.dim() != 3:
        raise ValueError(f"{what} must be [rows, {heads}, {head_dim}], not {tuple(t.shape)}")
    rows, h, d = t.shape
    if h != heads or d != head_dim:
        raise ValueError(f"{what} must be [rows, {heads}, {head_dim}], not {tuple(t.shape)}")
    s0, s1, s2 = t.stride()
    if (s2 != 1 and d > 1) or (s1 != d and h > 1):
        raise ValueError(f"{what}: the heads of a row must be contiguous (strides {t.stride()})")
    return t.data_ptr(), (s0 if rows > 1 else h * d), rows


def _on_gpu(t, what):
    if not t.is_cuda:
        raise ValueError(f"{what} must be on a GPU, it is on {t.device}")
    return t.get_device()


def rope_table(rotary_dim, theta, scaling_factor=1.0, initial_context_length=4096):
    """gptoss_decode_rope_table: (inv_freq float32 [rotary_dim / 2], concentration)."""
    lib = load_library()
    inv = np.empty(max(rotary_dim // 2, 0), dtype=np.float32)
    conc = ctypes.c_float()
    _check_op(lib, lib.gptoss_decode_rope_table(rotary_dim, theta, scaling_factor,
                                                initial_context_length, _ptr(inv),
                                                ctypes.byref(conc)))
    return inv, float(conc.value)


def rope_append(q, k, v, pos, inv_freq, q_out=None, k_cache=None, v_cache=None, slots=None,
                concentration=1.0, interleaved=False, angle_f32=False, stream=0):
    """gptoss_decode_rope_append: rotary positions on q and k, k and v stored at their cache
    rows.  q [rows, heads, head_dim], k and v [rows, kv heads, head_dim] (any row stride, heads
    contiguous; each may be None) in bf16, fp16 or fp32; k_cache / v_cache [slots, kv heads,
    head_dim]; pos int32 [rows] (< 0: row skipped); slots int64 [rows] or None (row i to cache
    row i); inv_freq float32 [rotary_dim / 2].  q_out may be q, and without slots k_cache may
    be k.  All tensors are on one GPU, `stream` is a stream of it (0: its default stream)."""
    lib = load_library()
    first = q if q is not None else (k if k is not None else v)
    if first is None:
        raise ValueError("q, k and v are all None")
    dev, code, dtype = _on_gpu(first, "input"), _dtype_code(first, "input"), first.dtype
    if first.dim() != 3:
        raise ValueError("the inputs must be [rows, heads, head_dim]")
    rows, _, d = first.shape
    kv = k if k is not None else v
    hq, hkv = (0 if q is None else q.shape[1]), (0 if kv is None else kv.shape[1])
    qp, qs, nq = _rows(q, "q", dtype, dev, hq, d)
    kp, ks, nk = _rows(k, "k", dtype, dev, hkv, d)
    vp, vs, nv = _rows(v, "v", dtype, dev, hkv, d)
    qop, qos, nqo = _rows(q_out, "q_out", dtype, dev, hq, d)
    kcp, kcs, nkc = _rows(k_cache, "k_cache", dtype, dev, hkv, d)
    vcp, vcs, nvc = _rows(v_cache, "v_cache", dtype, dev, hkv, d)
    for name, t, n in (("q", q, nq), ("k", k, nk), ("v", v, nv), ("q_out", q_out, nqo)):
        if n != rows and t is not None:
            raise ValueError(f"{name} has {n} rows, expected {rows}")
    if k_cache is not None and v_cache is not None and nkc != nvc:
        raise ValueError("k_cache and v_cache have different numbers of rows")
    types = _DTYPE_CODES
    half = inv_freq.shape[0]
    args = _ROPE_PACK(qp, kp, vp, qop, kcp, vcp, _vector(pos, "pos", types["int32"], rows, dev),
                      _vector(slots, "slots", types["int64"], rows, dev),
                      _vector(inv_freq, "inv_freq", types["float32"], half, dev),
                      qs, ks, vs, qos, kcs, vcs, nkc or nvc, concentration, rows, hq, hkv, d,
                      2 * half, interleaved, angle_f32, code)
    _check_op(lib, lib.gptoss_decode_rope_append(args, stream))


def prompt_attention(q, k, v, q_start, kv_start, kv_len, out, sinks=None, scale=None, window=0,
                     max_kv_len=0, status=None, stream=0):
    """gptoss_decode_prompt_attention: causal attention of packed query rows over K / V rows.
    q and out [tokens, heads, head_dim], k and v [kv rows, kv heads, head_dim] (any row stride
    that is a multiple of 8, heads contiguous) in bf16 or fp16; q_start int32 [seqs + 1],
    kv_start int64 [seqs], kv_len int32 [seqs]; sinks float32 [heads] or None; scale defaults
    to 1 / sqrt(head_dim); window 0 = none; max_kv_len: the largest kv_len where the caller
    knows it; status: int32 [1] tensor or None."""
    lib = load_library()
    dev, code, dtype = _on_gpu(q, "q"), _dtype_code(q, "q"), q.dtype
    if q.dim() != 3 or k.dim() != 3:
        raise ValueError("q and k must have three dimensions")
    tokens, hq, d = q.shape
    hkv = k.shape[1]
    qp, qs, _ = _rows(q, "q", dtype, dev, hq, d)
    kp, ks, n_kv = _rows(k, "k", dtype, dev, hkv, d)
    vp, vs, n_v = _rows(v, "v", dtype, dev, hkv, d)
    op, os_, n_out = _rows(out, "out", dtype, dev, hq, d)
    if n_v != n_kv or n_out != tokens:
        raise ValueError("k and v, or q and out, have different numbers of rows")
    n = kv_len.shape[0]
    types = _DTYPE_CODES
    args = _ATTENTION_PACK(qp, kp, vp, op, _vector(q_start, "q_start", types["int32"], n + 1, dev),
                           _vector(kv_start, "kv_start", types["int64"], n, dev),
                           _vector(kv_len, "kv_len", types["int32"], n, dev),
                           _vector(sinks, "sinks", types["float32"], hq, dev),
                           _vector(status, "status", types["int32"], 1, dev), qs, ks, vs, os_, n_kv,
                           d ** -0.5 if scale is None else scale, tokens, n, hq, hkv, d, window,
                           max_kv_len, code)
    _check_op(lib, lib.gptoss_decode_prompt_attention(args, stream))


def sample_tokens(logits, u, next_tokens, temperature=None, top_k=None, top_p=None, min_p=None,
                  pos=None, stream=0):
    """gptoss_decode_sample: next_tokens int32 [rows] drawn from logits [rows, vocab] (bf16, fp16
    or fp32, any row stride) with the uniform numbers u float32 [rows].  temperature, top_p,
    min_p float32 [rows], top_k int32 [rows], pos int32 [rows]; None switches one off
    (temperature None = 1; a temperature <= 0 is the argmax)."""
    lib = load_library()
    dev, code = _on_gpu(logits, "logits"), _dtype_code(logits, "logits")
    if logits.dim() != 2 or (logits.shape[1] > 1 and logits.stride(1) != 1):
        raise ValueError("logits must be [rows, vocab] with contiguous rows")
    rows, vocab = logits.shape
    f32, i32 = _DTYPE_CODES["float32"], _DTYPE_CODES["int32"]
    args = _SAMPLE_PACK(logits.data_ptr(), _vector(u, "u", f32, rows, dev),
                        _vector(temperature, "temperature", f32, rows, dev),
                        _vector(top_k, "top_k", i32, rows, dev),
                        _vector(top_p, "top_p", f32, rows, dev),
                        _vector(min_p, "min_p", f32, rows, dev), _vector(pos, "pos", i32, rows, dev),
                        _vector(next_tokens, "next_tokens", i32, rows, dev),
                        logits.stride(0) if rows > 1 else vocab, rows, vocab, code)
    _check_op(lib, lib.gptoss_decode_sample(args, stream))


class MoeEngine:
    """One engine = one gptoss_moe_t handle.  Method names follow the C ABI."""

    def __init__(
        self,
        hidden_dim,
        intermediate_dim,
        n_experts,
        experts_per_token,
        n_layers=1,
        max_tokens=1024,
        swiglu_limit=7.0,
        ep_rank=0,
        ep_size=1,
        weight_format=WEIGHTS_BF16,
        device=0,
    ):
        self.lib = load_library()
        self.cfg = MoeConfig(
            hidden_dim, intermediate_dim, n_experts, experts_per_token, n_layers, max_tokens,
            swiglu_limit, ep_rank, ep_size, weight_format, device,
        )
        self.handle = ctypes.c_void_p()
        rc = self.lib.gptoss_moe_create(ctypes.byref(self.cfg), ctypes.byref(self.handle))
        if rc != GPTOSS_OK:
            text = self.lib.gptoss_moe_last_error(None).decode()
            self.handle = None
            raise MoeError(rc, text)

    @classmethod
    def borrowed(cls, handle, cfg: "MoeConfig"):
        """The engine inside another object (a decode engine): same methods, not owned."""
        self = cls.__new__(cls)
        self.lib = load_library()
        self.cfg = cfg
        self.handle = handle
        self._borrowed = True
        return self

    # -- plumbing
    def _check(self, rc):
        if rc != GPTOSS_OK:
            raise MoeError(rc, self.lib.gptoss_moe_last_error(self.handle).decode())

    def close(self):
        if getattr(self, "handle", None):
            if not getattr(self, "_borrowed", False):
                self.lib.gptoss_moe_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    @property
    def local_experts(self):
        return self.cfg.n_experts // max(1, self.cfg.ep_size)

    # -- weights
    def load_layer_f32(self, layer, w_router, b_router, w_mlp1, b_mlp1, w_mlp2, b_mlp2):
        arrs = [np.ascontiguousarray(a, dtype=np.float32)
                for a in (w_router, b_router, w_mlp1, b_mlp1, w_mlp2, b_mlp2)]
        self._check(self.lib.gptoss_moe_load_layer_f32(self.handle, layer, *[_ptr(a) for a in arrs]))

    def load_layer_bf16(self, layer, w_router, b_router, w_mlp1, b_mlp1, w_mlp2, b_mlp2,
                        on_device):
        args = [_ptr(a) for a in (w_router, b_router, w_mlp1, b_mlp1, w_mlp2, b_mlp2)]
        self._check(self.lib.gptoss_moe_load_layer_bf16(self.handle, layer, *args,
                                                        1 if on_device else 0))

    def load_layer_mxfp4(self, layer, w_router_bf16, b_router, w1_blocks, w1_scales, b_mlp1,
                         w2_blocks, w2_scales, b_mlp2, on_device):
        args = [_ptr(a) for a in (w_router_bf16, b_router, w1_blocks, w1_scales, b_mlp1,
                                  w2_blocks, w2_scales, b_mlp2)]
        self._check(self.lib.gptoss_moe_load_layer_mxfp4(self.handle, layer, *args,
                                                         1 if on_device else 0))

    # -- compute
    def forward(self, layer, t, x, pos, n_tokens, stream=0):
        self._check(self.lib.gptoss_moe_forward(self.handle, layer, _ptr(t), _ptr(x), _ptr(pos),
                                                n_tokens, ctypes.c_void_p(stream)))

    def forward_host(self, layer, t_host, x_host, pos_host, n_tokens):
        self._check(self.lib.gptoss_moe_forward_host(self.handle, layer, _ptr(t_host),
                                                     _ptr(x_host), _ptr(pos_host), n_tokens))

    def forward_host_submit(self, layer, t_host, x_host, pos_host, n_tokens) -> int:
        ticket = ctypes.c_int()
        self._check(self.lib.gptoss_moe_forward_host_submit(
            self.handle, layer, _ptr(t_host), _ptr(x_host), _ptr(pos_host), n_tokens,
            ctypes.byref(ticket)))
        return int(ticket.value)

    def load_ffn_norm(self, layer, scale):
        scale = np.ascontiguousarray(scale, dtype=np.float32)
        self._check(self.lib.gptoss_moe_load_ffn_norm(self.handle, layer, _ptr(scale)))

    def forward_host_wait(self, ticket: int):
        self._check(self.lib.gptoss_moe_forward_host_wait(self.handle, ticket))

    def route(self, layer, t, pos, n_tokens, stream=0):
        self._check(self.lib.gptoss_moe_route(self.handle, layer, _ptr(t), _ptr(pos), n_tokens,
                                              ctypes.c_void_p(stream)))

    def permute(self, t, n_tokens, stream=0):
        self._check(self.lib.gptoss_moe_permute(self.handle, _ptr(t), n_tokens,
                                                ctypes.c_void_p(stream)))

    def experts(self, layer, stream=0):
        self._check(self.lib.gptoss_moe_experts(self.handle, layer, ctypes.c_void_p(stream)))

    def combine(self, x, n_tokens, stream=0):
        self._check(self.lib.gptoss_moe_combine(self.handle, _ptr(x), n_tokens,
                                                ctypes.c_void_p(stream)))

    def rmsnorm(self, out, x, w_dev, pos, n_tokens, stream=0):
        self._check(self.lib.gptoss_moe_rmsnorm(self.handle, _ptr(out), _ptr(x), _ptr(w_dev),
                                                _ptr(pos), n_tokens, ctypes.c_void_p(stream)))

    # -- taps
    def get_routing(self, n_tokens, want_logits=False):
        K, El, E = self.cfg.experts_per_token, self.local_experts, self.cfg.n_experts
        topk_i = np.empty((n_tokens, K), dtype=np.int32)
        topk_v = np.empty((n_tokens, K), dtype=np.float32)
        offsets = np.empty((El + 1,), dtype=np.int32)
        # under expert parallelism the owner's sorted order holds rows of every rank's batch,
        # whatever this rank's own n_tokens is: size for the engine's capacity
        rows_cap = self.cfg.max_tokens * max(1, self.cfg.ep_size) if self.cfg.ep_size > 1 else n_tokens
        sorted_token = np.full((max(1, rows_cap * K),), -1, dtype=np.int32)
        logits = np.empty((n_tokens, E), dtype=np.float32) if want_logits else None
        self._check(self.lib.gptoss_moe_get_routing(self.handle, n_tokens, _ptr(topk_i),
                                                    _ptr(topk_v), _ptr(offsets),
                                                    _ptr(sorted_token), _ptr(logits)))
        out = {"topk_i": topk_i, "topk_v": topk_v, "expert_offsets": offsets,
               "sorted_token": sorted_token[: int(offsets[-1])]}
        if want_logits:
            out["logits"] = logits
        return out

    def get_activations(self, n_rows):
        buf = np.empty((n_rows, self.cfg.intermediate_dim), dtype=np.uint16)
        self._check(self.lib.gptoss_moe_get_activations(self.handle, _ptr(buf), buf.nbytes))
        return buf

    def set_option(self, name, value):
        self._check(self.lib.gptoss_moe_set_option(self.handle, name.encode(), int(value)))

    def launch_count(self):
        return int(self.lib.gptoss_moe_launch_count(self.handle))

    def device_status(self):
        return int(self.lib.gptoss_moe_device_status(self.handle))

    def stage_ms(self, stage):
        ms = ctypes.c_float()
        idx = STAGES.index(stage) if isinstance(stage, str) else stage
        self._check(self.lib.gptoss_moe_stage_ms(self.handle, idx, ctypes.byref(ms)))
        return float(ms.value)

    # -- expert parallelism
    @staticmethod
    def ep_unique_id():
        lib = load_library()
        buf = (ctypes.c_ubyte * 128)()
        rc = lib.gptoss_moe_ep_unique_id(ctypes.cast(buf, ctypes.c_void_p))
        if rc != GPTOSS_OK:
            raise MoeError(rc, "gptoss_moe_ep_unique_id failed")
        return bytes(buf)

    def ep_init(self, unique_id: bytes):
        buf = (ctypes.c_ubyte * 128).from_buffer_copy(unique_id)
        self._check(self.lib.gptoss_moe_ep_init(self.handle, ctypes.cast(buf, ctypes.c_void_p)))

    @staticmethod
    def ep_init_local(engines):
        """gptoss_moe_ep_init_local: engines[r] was created with ep_rank r, ep_size len(engines);
        all of them live in this process."""
        lib = load_library()
        arr = (ctypes.c_void_p * len(engines))(*[e.handle for e in engines])
        rc = lib.gptoss_moe_ep_init_local(arr, len(engines))
        if rc != GPTOSS_OK:
            text = lib.gptoss_moe_last_error(engines[0].handle).decode()
            for e in engines:
                t2 = lib.gptoss_moe_last_error(e.handle).decode()
                if t2:
                    text = t2
            raise MoeError(rc, text or lib.gptoss_moe_last_error(None).decode())

    def forward_part(self, layer, part, t, x, pos, n_tokens, stream=0):
        self._check(self.lib.gptoss_moe_forward_part(self.handle, layer, part, _ptr(t), _ptr(x),
                                                     _ptr(pos), n_tokens, ctypes.c_void_p(stream)))

    @property
    def ep_transport(self) -> int:
        """0 = NCCL send/recv, 1 = peer memory, -1 before ep_init."""
        return int(self.lib.gptoss_moe_ep_transport(self.handle))


class DecodeEngine:
    """Mirror of include/gptoss_decode_b200.h: one greedy decode step for a batch of
    sequences (row i owns KV-cache slot i)."""

    def __init__(self, cfg: dict, max_batch: int, device: int = 0, ep_rank: int = 0,
                 ep_size: int = 1, max_tokens: int | None = None):
        """max_tokens: rows of one prefill pass (default: max_batch)."""
        self.lib = load_library()
        self.cfg = dict(cfg)
        self.max_batch = max_batch
        self.max_tokens = max_batch if max_tokens is None else max_tokens
        c = ModelConfig(**cfg)
        h = ctypes.c_void_p()
        if max_tokens is None:
            rc = self.lib.gptoss_decode_create_ep(ctypes.byref(c), max_batch, device, ep_rank,
                                                  ep_size, ctypes.byref(h))
        elif ep_size > 1:
            raise ValueError("max_tokens is for engines with all experts local")
        else:
            rc = self.lib.gptoss_decode_create_prefill(ctypes.byref(c), max_batch, max_tokens,
                                                       device, ctypes.byref(h))
        if rc != 0:
            raise MoeError(rc, (self.lib.gptoss_decode_last_error(None) or b"").decode())
        self.handle = h

    def _check(self, rc):
        if rc != 0:
            raise MoeError(rc, (self.lib.gptoss_decode_last_error(self.handle) or b"").decode())

    def load_bin(self, image: np.ndarray):
        """image: the whole .bin file as a uint8/float32 array (e.g. np.memmap); tensors
        start 60 bytes in."""
        raw = image.view(np.uint8).reshape(-1)
        first = raw[60:]
        self._check(self.lib.gptoss_decode_load_bin(self.handle,
                                                    ctypes.c_void_p(first.ctypes.data)))

    def set_tensor(self, name: str, layer: int, src):
        """src: float32 numpy array (host) or a CUDA torch tensor (bf16 weights, fp32 others)."""
        on_device = hasattr(src, "data_ptr")
        is_bf16 = on_device and str(src.dtype) == "torch.bfloat16"
        self._check(self.lib.gptoss_decode_set_tensor(self.handle, name.encode(), layer, _ptr(src),
                                                      int(on_device), int(is_bf16)))

    def set_kv(self, layer: int, row0: int, pos0: int, k, v):
        """k, v: CUDA bf16 tensors [rows, positions, n_kv_heads * head_dim]."""
        self._check(self.lib.gptoss_decode_set_kv(self.handle, layer, row0, k.shape[0], pos0,
                                                  k.shape[1], _ptr(k), _ptr(v)))

    def get_kv(self, layer: int, row0: int, pos0: int, k, v):
        """Fills the CUDA bf16 tensors k, v [rows, positions, n_kv_heads * head_dim]."""
        self._check(self.lib.gptoss_decode_get_kv(self.handle, layer, row0, k.shape[0], pos0,
                                                  k.shape[1], _ptr(k), _ptr(v)))

    def moe(self, ep_rank: int = 0, ep_size: int = 1, device: int = 0) -> "MoeEngine":
        """The MoE engine inside, with MoeEngine's methods (weights, options, timers, EP)."""
        c = self.cfg
        cfg = MoeConfig(c["hidden_dim"], c["intermediate_dim"], c["n_experts"],
                        c["experts_per_token"], c["n_layers"], self.max_tokens, c["swiglu_limit"],
                        ep_rank, ep_size, WEIGHTS_BF16, device)
        return MoeEngine.borrowed(ctypes.c_void_p(self.lib.gptoss_decode_moe(self.handle)), cfg)

    @staticmethod
    def _sampling(sampling, n):
        """(struct or None, arrays kept alive) from a dict of u, temperature, top_k, top_p, min_p."""
        if sampling is None:
            return None, None
        unknown = set(sampling) - {"u", "temperature", "top_k", "top_p", "min_p"}
        if unknown:
            raise ValueError(f"unknown sampling settings: {sorted(unknown)}")
        keep = {}
        for name, value in sampling.items():
            if value is not None:
                a = np.ascontiguousarray(value, dtype=np.int32 if name == "top_k" else np.float32)
                if a.shape != (n,):
                    raise ValueError(f"{name} must have {n} entries, not {a.shape}")
                keep[name] = a
        s = Sampling(*[keep[n].ctypes.data if n in keep else None
                       for n in ("u", "temperature", "top_k", "top_p", "min_p")])
        return s, keep

    def step(self, tokens, pos, stream: int = 0, sampling: dict | None = None):
        """One token per row.  sampling: None for the argmax, or a dict with the uniform numbers
        "u" and any of "temperature", "top_k", "top_p", "min_p" (one entry per row)."""
        tokens = np.ascontiguousarray(tokens, dtype=np.int32)
        pos = np.ascontiguousarray(pos, dtype=np.int32)
        if tokens.size < tokens.shape[0] or pos.size < tokens.shape[0]:
            raise ValueError(f"tokens and pos must have an entry for each of the {tokens.shape[0]} rows")
        nxt = np.empty(tokens.shape[0], dtype=np.int32)
        if sampling is None:
            self._check(self.lib.gptoss_decode_step(self.handle, _ptr(tokens), _ptr(pos),
                                                    tokens.shape[0], _ptr(nxt),
                                                    ctypes.c_void_p(stream)))
            return nxt
        s, keep = self._sampling(sampling, tokens.shape[0])
        self._check(self.lib.gptoss_decode_step_sample(self.handle, _ptr(tokens), _ptr(pos),
                                                       tokens.shape[0], ctypes.byref(s), _ptr(nxt),
                                                       ctypes.c_void_p(stream)))
        del keep
        return nxt

    def prefill(self, prompts, rows, pos0=None, stream: int = 0, sampling: dict | None = None):
        """Feeds prompts[i] (token ids) to cache row rows[i] from position pos0[i] (default 0) on
        and returns the token that follows each."""
        prompts = [np.ascontiguousarray(p, dtype=np.int32).reshape(-1) for p in prompts]
        n = len(prompts)
        rows = np.ascontiguousarray(rows, dtype=np.int32)
        pos0 = np.zeros(n, np.int32) if pos0 is None else np.ascontiguousarray(pos0, dtype=np.int32)
        if rows.shape != (n,) or pos0.shape != (n,):
            raise ValueError(f"rows and pos0 must have an entry for each of the {n} prompts")
        tokens = np.concatenate(prompts) if n else np.empty(0, np.int32)
        lens = np.array([p.shape[0] for p in prompts], dtype=np.int32)
        nxt = np.empty(n, dtype=np.int32)
        s, keep = self._sampling(sampling, n)
        self._check(self.lib.gptoss_decode_prefill(
            self.handle, _ptr(tokens), _ptr(rows), _ptr(pos0), _ptr(lens), n,
            None if s is None else ctypes.byref(s), _ptr(nxt), ctypes.c_void_p(stream)))
        del keep
        return nxt

    def logits(self, row: int) -> np.ndarray:
        out = np.empty(self.cfg["vocab_size"], dtype=np.float32)
        self._check(self.lib.gptoss_decode_get_logits(self.handle, row, _ptr(out)))
        return out

    def close(self):
        if getattr(self, "handle", None):
            self.lib.gptoss_decode_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:  # noqa: BLE001
            pass
