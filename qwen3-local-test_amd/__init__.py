"""qwattn: the MI355X full-attention hot path of the qwen4exp / Qwen3-Next engine.

Python mirror of the C ABI in include/qwattn.h, used by the tests and bench.py. Device memory and
streams come from PyTorch (plumbing only); every computation runs in libqwattn.so's HIP kernels.
There is no fallback: if the library is missing, or a call fails, an error is raised, the way the
reference backends throw std::runtime_error (src/vk_common.h:19-23, src/qwen4_vk.cpp:304).

The package directory name carries a hyphen, so it is loaded by path (see load_package in
tests/conftest.py, bench.py and __graft_entry__.py) under the module name `qwattn_amd`.
"""
import ctypes
import functools
import os
import struct

import torch  # loads the HIP runtime that libqwattn.so then shares

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "lib", "libqwattn.so")
HEADER = os.path.join(os.path.dirname(HERE), "include", "qwattn.h")

OK, EINVAL, EHIP, ENOMEM, ERANGE, ESTATE, ETIMEOUT = 0, -1, -2, -3, -4, -5, -6
F32, BF16, F16 = 0, 1, 2
LOG2E = 1.4426950408889634


class QwattnError(RuntimeError):
    """A nonzero status from the C ABI, with qwattn_last_error's text."""

    def __init__(self, code, msg):
        super().__init__(f"{msg} (status {code})")
        self.code = code


class Config(ctypes.Structure):
    _fields_ = [("n_heads", ctypes.c_int), ("n_kv_heads", ctypes.c_int), ("head_dim", ctypes.c_int),
                ("rope_dim", ctypes.c_int), ("rope_theta", ctypes.c_float), ("rms_eps", ctypes.c_float),
                ("max_ctx", ctypes.c_int), ("max_tokens", ctypes.c_int), ("max_splits", ctypes.c_int)]


class MatOut(ctypes.Structure):
    """qwattn_mat_out: one matrix of qwattn_mat_multi and its output."""
    _fields_ = [("w", ctypes.c_void_p), ("s", ctypes.c_void_p), ("rows", ctypes.c_int), ("y", ctypes.c_void_p),
                ("y_stride", ctypes.c_int), ("post", ctypes.c_int), ("post_scale", ctypes.c_float)]


_MAT_OUT = struct.Struct("@PPI4xPIif4x")  # MatOut's layout; packing it costs a quarter of a ctypes.Structure
assert _MAT_OUT.size == ctypes.sizeof(MatOut)


# qwattn_conv, qwattn_delta, qwattn_moe_layer, qwattn_paged_append_args and qwattn_paged_attend_args as the C ABI lays
# them out (a qwattn_paged_cache is the first part of the last two)
_CONV = struct.Struct("@5i4xPPqPPPPPq")
_DELTA = struct.Struct("@8iPPPPqqqPPPPPPPqPPqPN")
_MOE_LAYER = struct.Struct("@3i4xPPPPPP")
_PAGED_CACHE = "PPPqiii4x"
_PAGED_APPEND = struct.Struct("@" + _PAGED_CACHE + "4iPPPqqPPqqPPPPq")
_PAGED_ATTEND = struct.Struct("@" + _PAGED_CACHE + "5if" + "PPPqqPqqPqPN")


_lib = None
_P = ctypes.c_void_p
_I = ctypes.c_int


def load_library():
    """Loads libqwattn.so (built by build.py); raises if it is not built."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise RuntimeError(f"{LIB_PATH} is not built; run __graft_entry__.build() first")
    lib = ctypes.CDLL(LIB_PATH)
    sig = {
        "qwattn_create": [ctypes.POINTER(_P), _I, ctypes.POINTER(Config)],
        "qwattn_destroy": [_P],
        "qwattn_get_config": [_P, ctypes.POINTER(Config)],
        "qwattn_rope_table": [_P, ctypes.POINTER(_P)],
        "qwattn_fill_rope": [_P, _P, _P, _I],
        "qwattn_kv_alloc": [_P, _I, _I],
        "qwattn_kv_grow": [_P, _P, _I],
        "qwattn_kv_slot": [_P, _I, ctypes.POINTER(_P), ctypes.POINTER(_P), ctypes.POINTER(_I)],
        "qwattn_qk_norm_rope_append": [_P, _P, _P, _P, _P, _I, _P, _P, _P, _P, _P, _I, _P, _I, _I, _I],
        "qwattn_attend_partial": [_P, _P, _P, _P, _P, _I, _I, _I, _I, ctypes.POINTER(_I)],
        "qwattn_decode_partial": [_P, _P, _P, _P, _P, _I, _P, _P, _P, _P, _P, _I, _I, _I, _I, ctypes.POINTER(_I)],
        "qwattn_decode": [_P, _P, _P, _P, _P, _I, _P, _P, _P, _P, _P, _I, _P, _I, _I, _I, ctypes.POINTER(_I)],
        "qwattn_combine": [_P, _P, _P, _I, _P, _I, _I],
        "qwattn_attend_prefill": [_P, _P, _P, _I, _P, _P, _I, _P, _I, _P, _I, _I],
        "qwattn_attend_prefill_qg": [_P, _P, _P, _I, _P, _P, _P, _P, _I, _P, _I, _I],
        "qwattn_prefill": [_P, _P, _P, _P, _P, _I, _P, _P, _P, _P, _P, _I, _P, _I, _I],
        "qwattn_layer_attention": [_P, _P, _I, _P, _P, _P, _I, _P, _P, _P, _I, _I, _I],
        "qwattn_sync_status": [_P, _P],
        "qwattn_qsa_pool": [_P, _P, _P, _I, _P, _I, _I, _P, _P, _I, _I, _I],
        "qwattn_qsa_select": [_P, _P, _P, _I, _P, _I, _I, _I, _I, _P, _I, _I, _P, _I, _P, _I],
        "qwattn_qsa_index": [_P, _P, _P, _P, _I, _P, _P, _I, _I, _I, _I, _P, _P, _I, _I, _I, _P, _I, _P, _I],
        "qwattn_mat": [_P, _P, _P, _P, _I, _I, _I, _P, _I, _P, _I, _I, _I, ctypes.c_float],
        "qwattn_mat_multi": [_P, _P, _P, _I, _I, _I, _P, _I, _I],
        "qwattn_q8_unpack": [_P, _I, _I, _P, _P],
        "qwattn_qsa_key_bits": [_P, _P, _P, _I, _I, _I, _I, _P, _I],
        "qwattn_attend_partial_qsa": [_P, _P, _P, _P, _P, _I, _I, _I, _I, _P, _I, _P],
        "qwattn_decode_qsa": [_P, _P, _P, _P, _P, _I, _P, _P, _P, _P, _P, _I, _P, _I, _I, _I, _P, _I, _P],
        "qwattn_attend_prefill_qsa": [_P, _P, _P, _I, _P, _P, _I, _P, _I, _P, _I, _I, _P, _I],
        "qwattn_prefill_qsa": [_P, _P, _P, _P, _P, _I, _P, _P, _P, _P, _P, _I, _P, _I, _I, _P, _I],
        "qwattn_layer_attention_qsa": [_P, _P, _I, _P, _P, _P, _I, _P, _P, _P, _I, _I, _I, _P, _I],
        "qwattn_decode_noalloc": [_I, _P, ctypes.POINTER(Config), _P, _P, _P, _I, _P, _P, _P, _P, _P, _I, _P, _I, _I,
                                  _I, _P, ctypes.POINTER(_I)],
        "qwattn_conv_silu": [_P, _P, _P],
        "qwattn_delta_rule": [_P, _P, _P],
        "qwattn_delta_workspace": [_P, _P],
        "qwattn_moe_route": [_P, _P, _P, _I, _I, _I, _I, _I, _P, _P],
        "qwattn_moe": [_P, _P, _P, _P, _I, ctypes.c_int64, _P, _P, _I, _P, ctypes.c_int64, _I, _P, ctypes.c_size_t],
        "qwattn_moe_workspace": [_P, _I, _I, _I, _P],
        "qwattn_paged_append": [_P, _P, _P],
        "qwattn_paged_attend": [_P, _P, _P],
        "qwattn_paged_workspace": [_P, _P],
        "qwattn_set_wait_limits": [_P, _I, _I],
        "qwattn_set_alloc_fault": [_P, _I],
    }
    for name, args in sig.items():
        f = getattr(lib, name)
        f.argtypes = args
        f.restype = _I
    lib.qwattn_last_error.argtypes = [_P]
    lib.qwattn_last_error.restype = ctypes.c_char_p
    _lib = lib
    return lib


def q8_unpack(blocks, rows, cols):
    """GGUF Q8_0 rows (uint8 [rows, cols/32*34]) to the planar pair qwattn_mat takes: int8 [rows, cols] and
    float32 scales [rows, cols/32] (numpy, host memory), through the library's qwattn_q8_unpack."""
    import numpy as np
    lib = load_library()
    b = np.ascontiguousarray(blocks, dtype=np.uint8)
    w = np.zeros((rows, cols), np.int8)
    s = np.zeros((rows, cols // 32), np.float32)
    rc = lib.qwattn_q8_unpack(ctypes.c_void_p(b.ctypes.data), rows, cols, ctypes.c_void_p(w.ctypes.data),
                              ctypes.c_void_p(s.ctypes.data))
    if rc != OK:
        raise QwattnError(rc, "qwattn_q8_unpack: bad shape")
    return w, s


def header_functions():
    """Names of the functions include/qwattn.h declares."""
    import re
    text = open(HEADER).read()
    return sorted(set(re.findall(r"^\s*(?:int|const char\*)\s+(qwattn_\w+)\s*\(", text, re.M)))


# A decode layer's launches take 25 us on the card, and its three calls took 36 us to issue through ctypes objects,
# torch.cuda.Stream objects and repeated tensor attributes: addresses and streams go to ctypes as plain integers,
# and each tensor attribute is read once. Layers of one token at 4,096 keys: 36.9 -> 24.3 us each.
def _ptr(t):
    return None if t is None else t.data_ptr()


# (None in a torch without GPU support, where the host helpers here still work)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_cuda_device = getattr(torch._C, "_cuda_getDevice", None)


def _stream(stream):
    """The handle of `stream`, or of the current device's current stream."""
    if stream is not None:
        return stream.cuda_stream
    if _raw_stream and _cuda_device and torch.cuda.is_initialized():
        return _raw_stream(_cuda_device())
    return torch.cuda.current_stream().cuda_stream


_F32, _F16, _I8 = torch.float32, torch.float16, torch.int8
_DT = {torch.float32: F32, torch.bfloat16: BF16, torch.float16: F16}


def _check_weights(w, s):
    """(rows, cols) of a projection's weights: int8 [rows, cols] with float32 scales s [rows, cols/32] (planar
    Q8_0), or float32 [rows, cols] with s None; both contiguous, as the C ABI reads them."""
    shape = w.shape
    if len(shape) != 2 or not w.is_contiguous():
        raise ValueError(f"weights must be a contiguous [rows, cols] matrix, got shape {tuple(shape)}")
    rows, cols = shape
    if s is None:
        if w.dtype != _F32:
            raise ValueError(f"float weights must be float32, got {w.dtype} (int8 weights need scales)")
    else:
        if w.dtype != _I8:
            raise ValueError(f"Q8 weights must be int8, got {w.dtype}")
        if s.dtype != _F32 or not s.is_contiguous() or s.shape != (rows, cols // 32):
            raise ValueError(f"Q8 scales must be contiguous float32 [{rows}, {cols // 32}], got {s.dtype} "
                             f"{tuple(s.shape)}")
    return rows, cols


def _check_rows(t, name, width, n=None):
    """A float32 [n, >= width] operand with unit column stride (row stride free); returns (rows, row stride)."""
    shape, stride = t.shape, t.stride()
    if t.dtype != _F32 or len(shape) != 2 or stride[1] != 1:
        raise ValueError(f"{name} must be float32 [n, >= {width}] with unit column stride")
    if shape[1] < width:
        raise ValueError(f"{name} has {shape[1]} columns, needs >= {width}")
    if n is not None and shape[0] < n:
        raise ValueError(f"{name} has {shape[0]} rows, needs >= {n}")
    return shape[0], stride[0]


_ROW_DT = {torch.float32: F32, torch.bfloat16: BF16}


def _check_seq_rows(t, name, shape, dtype):
    """Row stride of a [n_seq, n, ...] operand of the linear-attention operators: `shape`, dtype, its rows (all but the
    first two dims) contiguous, row b * n + t at one stride."""
    if t.dtype is not dtype or t.shape != shape:
        raise ValueError(f"{name} must be {dtype} {tuple(shape)}, got {t.dtype} {tuple(t.shape)}")
    stride, inner = t.stride(), 1
    if len(stride) == 4 and stride[3] == 1 and stride[2] == shape[3] and stride[0] == shape[1] * stride[1]:
        return stride[1]
    for d in range(len(shape) - 1, 1, -1):
        if stride[d] != inner and shape[d] != 1:
            raise ValueError(f"{name}: the elements of a row must be contiguous, got strides {stride}")
        inner *= shape[d]
    row = stride[1] if shape[1] > 1 else stride[0] if shape[0] > 1 else inner
    if shape[0] > 1 and shape[1] > 1 and stride[0] != shape[1] * row:
        raise ValueError(f"{name}: row b * n + t must be at (b * n + t) times one stride, got strides {stride}")
    return row


def _check_head_rows(t, name, shape, dtype):
    """(row stride, head stride) of a [n_seq, n, heads, dim] operand of the paged operators: `shape`, dtype, contiguous
    heads at one stride, row b * n + t at one stride."""
    if t.dtype is not dtype or t.shape != shape:
        raise ValueError(f"{name} must be {dtype} {tuple(shape)}, got {t.dtype} {tuple(t.shape)}")
    n_seq, n, heads, dim = shape
    seq, row, head, one = t.stride()
    head = head if heads > 1 else dim
    row = row if n > 1 else seq if n_seq > 1 else heads * head
    if one != 1 or (n_seq > 1 and n > 1 and seq != n * row):
        raise ValueError(f"{name}: a head must be contiguous and row b * n + t at (b * n + t) times one stride, got strides "
                         f"{t.stride()}")
    return row, head


def _check_matrix(t, name, shape, dtype):
    """Row stride of a [n, width] operand of exactly `shape` and dtype with contiguous rows."""
    stride = t.stride()
    if t.dtype is not dtype or t.shape != shape or (stride[1] != 1 and shape[1] != 1):
        raise ValueError(f"{name} must be {dtype} {shape} with contiguous rows, got {t.dtype} {tuple(t.shape)}")
    return stride[0] if shape[0] > 1 else shape[1]


def _check_whole(t, name, shape, dtype=torch.float32):
    """A contiguous operand of exactly `shape` and dtype."""
    if t.dtype is not dtype or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous {dtype} {tuple(shape)}, got {t.dtype} {tuple(t.shape)}")


BLK = 32  # positions per cache block


def k_block(rows):
    """[cap][NKV][D] K rows -> the blocked K cache layout of include/qwattn.h, flat (cap % 32 == 0):
    head h, block b, key kb, dim d at ((h*(cap/32) + b)*32*D) + ((((d/32)*2 + (kb/4)%2)*4 + (d/8)%4)*16
    + (kb/8)*4 + kb%4)*8 + d%8."""
    cap, nkv, d = rows.shape
    x = rows.reshape(cap // BLK, 4, 2, 4, nkv, d // 32, 4, 8)  # [b][kb/8][kb/4%2][kb%4][h][d/32][d/8%4][d%8]
    return x.permute(4, 0, 5, 2, 6, 1, 3, 7).contiguous().view(-1)


def k_rows(kcache, cap, nkv, d):
    """Inverse of k_block: the flat blocked K cache -> [cap][NKV][D] rows (a copy)."""
    x = kcache.view(nkv, cap // BLK, d // 32, 2, 4, 4, 4, 8)   # [h][b][d/32][s][g][kb/8][kb%4][e]
    return x.permute(1, 5, 3, 6, 0, 2, 4, 7).reshape(cap, nkv, d)


def v_block(rows):
    """[cap][NKV][D] V rows -> the blocked V cache layout, flat: head h, block b, key kb, dim d at
    ((h*(cap/32) + b)*32*D) + (((d/16)*4 + kb/8)*16 + d%16)*8 + kb%8."""
    cap, nkv, d = rows.shape
    x = rows.reshape(cap // BLK, 4, 8, nkv, d // 16, 16)        # [b][kb/8][kb%8][h][d/16][d%16]
    return x.permute(3, 0, 4, 1, 5, 2).contiguous().view(-1)


def v_rows(vcache, cap, nkv, d):
    """Inverse of v_block."""
    x = vcache.view(nkv, cap // BLK, d // 16, 4, 16, 8)         # [h][b][d/16][kb/8][d%16][kb%8]
    return x.permute(1, 3, 5, 0, 2, 4).reshape(cap, nkv, d)


class Attention:
    """One qwattn context: attention shape, rope table, split partials and (optionally) K/V caches."""

    _paged_ws = None  # bytes of paged_attend's workspace, once asked for

    def __init__(self, n_heads, n_kv_heads, head_dim, rope_dim, rope_theta=1e7, rms_eps=1e-6, max_ctx=262144,
                 max_tokens=2048, max_splits=1024, device=0):
        self.lib = load_library()
        self.cfg = Config(n_heads, n_kv_heads, head_dim, rope_dim, rope_theta, rms_eps, max_ctx, max_tokens,
                          max_splits)
        self.device = device
        self._torch_device = torch.device("cuda", device)
        h = ctypes.c_void_p()
        rc = self.lib.qwattn_create(ctypes.byref(h), device, ctypes.byref(self.cfg))
        if rc:
            raise QwattnError(rc, self.lib.qwattn_last_error(None).decode())
        self.h = h
        self.NH, self.NKV, self.D, self.R = n_heads, n_kv_heads, head_dim, rope_dim

    def close(self):
        if getattr(self, "h", None):
            self.lib.qwattn_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def _check(self, rc):
        if rc:
            raise QwattnError(rc, self.lib.qwattn_last_error(self.h).decode())

    # ---- state ---------------------------------------------------------------------------------------
    def rope_table(self):
        """The context's rope table as a [max_ctx, R/2, 2] float32 tensor view (device memory)."""
        p = ctypes.c_void_p()
        self._check(self.lib.qwattn_rope_table(self.h, ctypes.byref(p)))
        n = self.cfg.max_ctx * (self.R // 2) * 2
        return _wrap_device_floats(p.value, n, self.device).view(self.cfg.max_ctx, self.R // 2, 2)

    def fill_rope(self, table, n_pos, stream=None):
        self._check(self.lib.qwattn_fill_rope(self.h, _stream(stream), _ptr(table), n_pos))

    def kv_alloc(self, n_slots, cap):
        self._check(self.lib.qwattn_kv_alloc(self.h, n_slots, cap))

    def kv_grow(self, tokens, stream=None):
        self._check(self.lib.qwattn_kv_grow(self.h, _stream(stream), tokens))

    def kv_slot(self, slot):
        """(K cache, V cache, cap): flat fp16 views of one slot's blocked caches (see k_rows / v_rows)."""
        k, v, cap = ctypes.c_void_p(), ctypes.c_void_p(), ctypes.c_int()
        self._check(self.lib.qwattn_kv_slot(self.h, slot, ctypes.byref(k), ctypes.byref(v), ctypes.byref(cap)))
        n = cap.value * self.NKV * self.D
        kc = _wrap_device_halfs(k.value, n, self.device)
        vc = _wrap_device_halfs(v.value, n, self.device)
        return kc, vc, cap.value

    # ---- kernels -------------------------------------------------------------------------------------
    def qk_norm_rope_append(self, qg, k, v, qn, kn, rope, kcache, vcache, kv_cap, q_out, pos, n, stream=None):
        """q_out None: the key and value rows only (for attend_prefill_qg)."""
        self._check(self.lib.qwattn_qk_norm_rope_append(
            self.h, _stream(stream), _ptr(qg), _ptr(k), _ptr(v), _DT[qg.dtype], _ptr(qn), _ptr(kn), _ptr(rope),
            _ptr(kcache), _ptr(vcache), kv_cap, _ptr(q_out) if q_out is not None else None,
            _DT[q_out.dtype] if q_out is not None else 0, pos, n))

    def attend_partial(self, q, kcache, vcache, kv_cap, pos, n, n_split=0, stream=None):
        used = ctypes.c_int()
        self._check(self.lib.qwattn_attend_partial(self.h, _stream(stream), _ptr(q), _ptr(kcache), _ptr(vcache),
                                                   kv_cap, pos, n, n_split, ctypes.byref(used)))
        return used.value

    def decode_partial(self, qg, k, v, qn, kn, rope, kcache, vcache, kv_cap, pos, n, n_split=0, stream=None):
        """Fused norm + rope + append + split-KV partials (n <= 8, n * NH/NKV <= 32); returns splits."""
        used = ctypes.c_int()
        self._check(self.lib.qwattn_decode_partial(
            self.h, _stream(stream), _ptr(qg), _ptr(k), _ptr(v), _DT[qg.dtype], _ptr(qn), _ptr(kn), _ptr(rope),
            _ptr(kcache), _ptr(vcache), kv_cap, pos, n, n_split, ctypes.byref(used)))
        return used.value

    def decode(self, qg, k, v, qn, kn, rope, kcache, vcache, kv_cap, out, pos, n, n_split=0, stream=None):
        """Norm + rope + append + split-KV attend + combine and gate in one launch (n <= 8, n * NH/NKV <= 32;
        the combine kernel follows only when a KV head or 16-row slice gets fewer splits than rows);
        returns the split count."""
        used = ctypes.c_int()
        self._check(self.lib.qwattn_decode(
            self.h, _stream(stream), _ptr(qg), _ptr(k), _ptr(v), _DT[qg.dtype], _ptr(qn), _ptr(kn), _ptr(rope),
            _ptr(kcache), _ptr(vcache), kv_cap, _ptr(out), pos, n, n_split, ctypes.byref(used)))
        return used.value

    def combine(self, qg, out, n, n_split, stream=None):
        self._check(self.lib.qwattn_combine(self.h, _stream(stream), _ptr(qg), _DT[qg.dtype], _ptr(out), n, n_split))

    def attend_prefill(self, q, kcache, vcache, kv_cap, qg, out, pos, n, stream=None):
        self._check(self.lib.qwattn_attend_prefill(self.h, _stream(stream), _ptr(q), _DT[q.dtype], _ptr(kcache),
                                                   _ptr(vcache), kv_cap, _ptr(qg), _DT[qg.dtype], _ptr(out), pos, n))

    # ---- QSA indexer ------------------------------------------------------------------------------------

    def qsa_pool(self, ik, k_gamma, cr, raw, pooled, cap, pos, n, stream=None):
        """Caches raw indexer keys ik [n, ID] at positions pos.. into raw [cap, ID] and pools the blocks the
        call completes into pooled [cap // cr + 1, ID] (src/qwen4_qsa.h:38-54)."""
        self._check(self.lib.qwattn_qsa_pool(self.h, _stream(stream), _ptr(ik), _DT[ik.dtype], _ptr(k_gamma),
                                             ik.shape[-1], cr, _ptr(raw), _ptr(pooled), cap, pos, n))

    def qsa_select(self, iq, q_gamma, cr, budget, pooled, pos, n, mask=None, key_bits=None, stream=None):
        """Block selection of iq [n, IH, ID] (src/qwen4_qsa.h:58-91) into mask [n, mask_words] uint32 (as
        int32 storage) and/or key_bits [n, kb_words]."""
        self._check(self.lib.qwattn_qsa_select(
            self.h, _stream(stream), _ptr(iq), _DT[iq.dtype], _ptr(q_gamma), iq.shape[1], iq.shape[2], cr, budget,
            _ptr(pooled), pos, n, _ptr(mask), 0 if mask is None else mask.shape[-1], _ptr(key_bits),
            0 if key_bits is None else key_bits.shape[-1]))

    def qsa_index(self, ik, iq, k_gamma, q_gamma, cr, budget, raw, pooled, cap, pos, n, mask=None, key_bits=None,
                  stream=None):
        """qsa_pool then qsa_select in one call (one launch when no block completes); ik and iq in one dtype."""
        self._check(self.lib.qwattn_qsa_index(
            self.h, _stream(stream), _ptr(ik), _ptr(iq), _DT[iq.dtype], _ptr(k_gamma), _ptr(q_gamma), iq.shape[1],
            iq.shape[2], cr, budget, _ptr(raw), _ptr(pooled), cap, pos, n, _ptr(mask),
            0 if mask is None else mask.shape[-1], _ptr(key_bits), 0 if key_bits is None else key_bits.shape[-1]))

    def mat(self, x, y, w, s=None, post=0, post_scale=0.0, stream=None):
        """y [n, >= rows] = x [n, >= cols] W^T (Qwen4Vulkan::mat): W planar Q8 (w int8 [rows, cols] with s
        [rows, cols/32]) or float32 w [rows, cols]; post 1 applies silu(y * post_scale)."""
        rows, cols = _check_weights(w, s)
        n, x_stride = _check_rows(x, "x", cols)
        y_stride = _check_rows(y, "y", rows, n)[1]
        self._check(self.lib.qwattn_mat(self.h, _stream(stream), w.data_ptr(), _ptr(s), int(s is not None), rows, cols,
                                        x.data_ptr(), x_stride, y.data_ptr(), y_stride, n, post, post_scale))

    def mat_multi(self, x, outs, stream=None):
        """Several projections of x in one call (qwattn_mat_multi): outs = [(y, w, s), ...] (s None for float32
        weights, all of one kind and one column count), each as in mat."""
        if not outs:
            raise ValueError("mat_multi: no matrices")
        _, w, s = outs[0]
        q8 = s is not None
        first = _check_weights(w, s)
        cols = first[1]
        n, x_stride = _check_rows(x, "x", cols)
        mats = bytearray()
        for i, (y, w, s) in enumerate(outs):
            if (s is not None) != q8:
                raise ValueError(f"mat_multi: matrix {i} mixes Q8 and float32 weights")
            rows, c = _check_weights(w, s) if i else first
            if c != cols:
                raise ValueError(f"mat_multi: matrix {i} has {c} columns, matrix 0 has {cols}")
            y_stride = _check_rows(y, f"y[{i}]", rows, n)[1]
            mats += _MAT_OUT.pack(w.data_ptr(), s.data_ptr() if q8 else 0, rows & 0xFFFFFFFF, y.data_ptr(),
                                  y_stride & 0xFFFFFFFF, 0, 0.0)  # 32 bits as ctypes.c_int takes them
        self._check(self.lib.qwattn_mat_multi(self.h, _stream(stream), bytes(mats), len(outs), int(q8), cols,
                                              x.data_ptr(), x_stride, n))

    # ---- linear attention and experts -------------------------------------------------------------------

    def _on_device(self, tensors, stream):
        """The stream's handle, once every operand is known to be on this context's GPU (the device's current stream
        where none is given)."""
        device = self.device
        for t in tensors:
            if t is not None and t.get_device() != device:  # (-1: the CPU)
                raise ValueError(f"operands must be on cuda:{self.device}, got one on {t.device}")
        if stream is not None:
            return stream.cuda_stream
        return _raw_stream(device) if _raw_stream else torch.cuda.current_stream(self.device).cuda_stream

    def _workspace(self, size, given, stream):
        """(address, bytes) of the caller's workspace tensor, or of one from torch's allocator, and the tensor itself,
        which must live until the call is made."""
        if given is not None:
            if not given.is_contiguous():
                raise ValueError("the workspace must be contiguous")
            return given.data_ptr(), given.numel() * given.element_size(), given
        if not size:
            return 0, 0, None
        if stream is None:
            t = torch.empty(size, dtype=torch.uint8, device=self._torch_device)
        else:  # from that stream's memory: another stream's may still be in use there
            with torch.cuda.stream(stream):
                t = torch.empty(size, dtype=torch.uint8, device=self._torch_device)
        return t.data_ptr(), size, t

    def conv_silu(self, x, w, state, y, bias=None, lens=None, snap=None, stream=None):
        """Short causal depthwise convolution + SiLU of x [n_seq, n, channels] into y, rows before the first from
        state [n_seq, taps - 1, channels], which becomes the last rows; w [channels, taps], bias [channels]; lens
        [n_seq] int32 shortens sequences; snap [n_seq, n, taps - 1, channels] gets the state after each token."""
        if x.dtype not in _ROW_DT or len(x.shape) != 3 or len(w.shape) != 2:
            raise ValueError(f"x must be float32 or bfloat16 [n_seq, n, channels] and w [channels, taps], got {x.dtype} "
                             f"{tuple(x.shape)} and {tuple(w.shape)}")
        (n_seq, n, ch), taps = x.shape, w.shape[1]
        x_stride = _check_seq_rows(x, "x", x.shape, x.dtype)
        y_stride = _check_seq_rows(y, "y", x.shape, x.dtype)
        _check_whole(w, "w", (ch, taps))
        _check_whole(state, "state", (n_seq, taps - 1, ch))
        if bias is not None:
            _check_whole(bias, "bias", (ch,))
        if lens is not None:
            _check_whole(lens, "lens", (n_seq,), torch.int32)
        if snap is not None:
            _check_whole(snap, "snap", (n_seq, n, taps - 1, ch))
        s = self._on_device((x, w, state, y, bias, lens, snap), stream)
        args = _CONV.pack(n_seq, n, ch, taps, _ROW_DT[x.dtype], _ptr(lens) or 0, x.data_ptr(), x_stride, w.data_ptr(),
                          _ptr(bias) or 0, state.data_ptr(), _ptr(snap) or 0, y.data_ptr(), y_stride)
        self._check(self.lib.qwattn_conv_silu(self.h, s, args))

    def delta_rule(self, q, k, v, a, b, state, out, a_coef=None, dt_bias=None, z=None, gamma=None, lens=None, snap=None,
                   tiled=False, workspace=None, stream=None):
        """The gated delta rule over n tokens of n_seq sequences: q, k [n_seq, n, k_heads, key_dim], v, z and out
        [n_seq, n, v_heads, val_dim] of one dtype, gates a, b [n_seq, n, v_heads], state [n_seq, v_heads, key_dim,
        val_dim] updated in place, snap [n_seq, n, v_heads, key_dim, val_dim] the state after each token; formulas in
        include/qwattn.h. workspace: a tensor of delta_workspace() bytes (None: from torch's allocator)."""
        if v.dtype not in _ROW_DT or len(v.shape) != 4 or len(k.shape) != 4:
            raise ValueError(f"k and v must be float32 or bfloat16 [n_seq, n, heads, dim], got {v.dtype}, "
                             f"{tuple(k.shape)}, {tuple(v.shape)}")
        shape, dtype = v.shape, v.dtype
        n_seq, n, hv, dv = shape
        _, _, hk, dk = k.shape
        qk = (n_seq, n, hk, dk)
        q_stride, k_stride = _check_seq_rows(q, "q", qk, dtype), _check_seq_rows(k, "k", qk, dtype)
        v_stride = _check_seq_rows(v, "v", shape, dtype)
        out_stride = _check_seq_rows(out, "out", shape, dtype)
        z_stride = _check_seq_rows(z, "z", shape, dtype) if z is not None else 0
        gates, heads = (n_seq, n, hv), (hv,)
        _check_whole(a, "a", gates)
        _check_whole(b, "b", gates)
        _check_whole(state, "state", (n_seq, hv, dk, dv))
        if a_coef is not None:
            _check_whole(a_coef, "a_coef", heads)
        if dt_bias is not None:
            _check_whole(dt_bias, "dt_bias", heads)
        if gamma is not None:
            _check_whole(gamma, "gamma", (dv,))
        if snap is not None:
            _check_whole(snap, "snap", (n_seq, n, hv, dk, dv))
        if lens is not None:
            _check_whole(lens, "lens", (n_seq,), torch.int32)
        s = self._on_device((q, k, v, a, b, state, out, a_coef, dt_bias, z, gamma, lens, snap, workspace), stream)
        size = delta_workspace(n_seq, n, hk, hv, dk, dv, dtype, z is not None, snap is not None)
        ws, ws_bytes, keep = self._workspace(size, workspace, stream) if size or workspace is not None else (0, 0, None)
        args = _DELTA.pack(n_seq, n, hk, hv, dk, dv, int(tiled), _ROW_DT[dtype], _ptr(lens) or 0, q.data_ptr(),
                           k.data_ptr(), v.data_ptr(), q_stride, k_stride, v_stride, a.data_ptr(), b.data_ptr(),
                           _ptr(a_coef) or 0, _ptr(dt_bias) or 0, state.data_ptr(), _ptr(snap) or 0, _ptr(z) or 0,
                           z_stride, _ptr(gamma) or 0, out.data_ptr(), out_stride, ws, ws_bytes)
        self._check(self.lib.qwattn_delta_rule(self.h, s, args))

    def moe_route(self, logits, ids, weights, renorm=True, stream=None):
        """The top_k experts of each row of logits [n, >= n_experts] (its columns are the experts) into ids [n, top_k]
        int32 and weights [n, top_k]: softmax weights, divided by the selected ones' sum with renorm."""
        n, stride = _check_rows(logits, "logits", 1)
        if len(ids.shape) != 2 or ids.shape[0] != n:
            raise ValueError(f"ids must be [{n}, top_k], got {tuple(ids.shape)}")
        top_k, experts = ids.shape[1], logits.shape[1]
        _check_whole(ids, "ids", (n, top_k), torch.int32)
        _check_whole(weights, "weights", (n, top_k))
        s = self._on_device((logits, ids, weights), stream)
        self._check(self.lib.qwattn_moe_route(self.h, s, logits.data_ptr(), stride if n > 1 else experts, n, experts, top_k,
                                              int(renorm), ids.data_ptr(), weights.data_ptr()))

    def moe(self, x, ids, weights, gate, up, down, y, workspace=None, stream=None):
        """SwiGLU experts over x [n, hidden] into y: each token's ids [n, top_k] int32 (outside the experts: skipped) with
        weights [n, top_k]; gate, up (int8 [n_experts, ffn, hidden], scales [n_experts, ffn, hidden / 32]) and down
        ([n_experts, hidden, ffn], [n_experts, hidden, ffn / 32]) pairs. workspace as in delta_rule (moe_workspace())."""
        w = gate[0]
        if x.dtype not in _ROW_DT or len(x.shape) != 2 or len(ids.shape) != 2 or len(w.shape) != 3:
            raise ValueError(f"x must be float32 or bfloat16 [n, hidden], ids [n, top_k] and gate [n_experts, ffn, hidden], "
                             f"got {x.dtype} {tuple(x.shape)}, {tuple(ids.shape)}, {tuple(w.shape)}")
        (n, top_k), (experts, ffn, hidden) = ids.shape, w.shape
        wide, narrow = (experts, ffn, hidden), (experts, ffn, hidden // 32)
        _check_whole(w, "gate", wide, _I8)
        _check_whole(gate[1], "gate's scales", narrow)
        _check_whole(up[0], "up", wide, _I8)
        _check_whole(up[1], "up's scales", narrow)
        _check_whole(down[0], "down", (experts, hidden, ffn), _I8)
        _check_whole(down[1], "down's scales", (experts, hidden, ffn // 32))
        dtype, rows = x.dtype, (n, hidden)
        x_stride, y_stride = _check_matrix(x, "x", rows, dtype), _check_matrix(y, "y", rows, dtype)
        _check_whole(ids, "ids", (n, top_k), torch.int32)
        _check_whole(weights, "weights", (n, top_k))
        s = self._on_device((x, ids, weights, *gate, *up, *down, y, workspace), stream)
        size = moe_workspace(experts, hidden, ffn, dtype, n, top_k)
        ws, ws_bytes, keep = self._workspace(size, workspace, stream)
        layer = _MOE_LAYER.pack(experts, hidden, ffn, gate[0].data_ptr(), up[0].data_ptr(), down[0].data_ptr(),
                                gate[1].data_ptr(), up[1].data_ptr(), down[1].data_ptr())
        self._check(self.lib.qwattn_moe(self.h, s, layer, x.data_ptr(), _ROW_DT[dtype], x_stride, ids.data_ptr(),
                                        weights.data_ptr(), top_k, y.data_ptr(), y_stride, n, ws, ws_bytes))

    # ---- batches over a paged cache ---------------------------------------------------------------------

    def _paged_cache(self, kpool, vpool, table, pos, lens, n_seq):
        """The cache's part of the packed arguments, its operands checked."""
        nkv, shape = self.NKV, kpool.shape
        if len(shape) != 3 or shape[1] != nkv or shape[2] % self.D:
            raise ValueError(f"kpool must be [n_pages, {nkv}, page * {self.D}], got {tuple(shape)}")
        _check_whole(kpool, "kpool", shape, _F16)
        _check_whole(vpool, "vpool", shape, _F16)
        if (table.dtype is not torch.int32 or len(table.shape) != 2 or table.shape[0] != n_seq or
                (table.shape[1] != 1 and table.stride(1) != 1)):
            raise ValueError(f"table must be int32 [{n_seq}, pages] with unit column stride, got {table.dtype} {tuple(table.shape)}")
        _check_whole(pos, "pos", (n_seq,), torch.int32)
        if lens is not None:
            _check_whole(lens, "lens", (n_seq,), torch.int32)
        pages = table.shape[1]
        return (kpool.data_ptr(), vpool.data_ptr(), table.data_ptr(), table.stride(0) if n_seq > 1 else pages, shape[0], pages,
                shape[2] // self.D)

    def paged_append(self, k, v, kpool, vpool, table, pos, q=None, q_out=None, qn=None, kn=None, rope=None, lens=None,
                     stream=None):
        """Appends new tokens' keys and values k, v [n_seq, n, KV heads, head_dim] to the pages of their sequences, the
        keys normalized (kn [head_dim] as gamma - 1, None: not) and rotated to positions pos[b] + t; q [n_seq, n, heads,
        head_dim] likewise (qn) into q_out. Pools kpool, vpool float16 [n_pages, KV heads, page * head_dim] in the block
        layout (k_block, v_block), table int32 [n_seq, pages], pos int32 [n_seq]; rope [rows, rope_dim / 2, 2] (None:
        the context's); lens [n_seq] int32 shortens sequences. A token at a position past the table's pages or the rope
        rows is not appended and its query is zero."""
        if k.dtype not in _ROW_DT or len(k.shape) != 4:
            raise ValueError(f"k must be float32 or bfloat16 [n_seq, n, KV heads, head_dim], got {k.dtype} {tuple(k.shape)}")
        dtype, (n_seq, n) = k.dtype, k.shape[:2]
        kv, heads = (n_seq, n, self.NKV, self.D), (n_seq, n, self.NH, self.D)
        k_stride, v_stride = _check_seq_rows(k, "k", kv, dtype), _check_seq_rows(v, "v", kv, dtype)
        q_stride = q_head = out_stride = 0
        if q is not None:
            q_stride, q_head = _check_head_rows(q, "q", heads, dtype)
        if q_out is not None:
            out_stride = _check_seq_rows(q_out, "q_out", heads, dtype)
        if qn is not None:
            _check_whole(qn, "qn", (self.D,))
        if kn is not None:
            _check_whole(kn, "kn", (self.D,))
        if rope is not None:
            _check_whole(rope, "rope", (rope.shape[0], self.R // 2, 2))
        cache = self._paged_cache(kpool, vpool, table, pos, lens, n_seq)
        s = self._on_device((k, v, kpool, vpool, table, pos, q, q_out, qn, kn, rope, lens), stream)
        args = _PAGED_APPEND.pack(*cache, n_seq, n, _ROW_DT[dtype], 0 if rope is None else rope.shape[0], _ptr(lens) or 0,
                                  pos.data_ptr(), _ptr(q) or 0, q_stride, q_head, k.data_ptr(), v.data_ptr(), k_stride, v_stride,
                                  _ptr(qn) or 0, _ptr(kn) or 0, _ptr(rope) or 0, _ptr(q_out) or 0, out_stride)
        self._check(self.lib.qwattn_paged_append(self.h, s, args))

    def paged_workspace(self):
        """Bytes of workspace that every paged_attend call of this context needs."""
        size = ctypes.c_size_t()
        self._check(self.lib.qwattn_paged_workspace(self.h, ctypes.byref(size)))
        return size.value

    def paged_attend(self, q, kpool, vpool, table, pos, out, gate=None, lens=None, window=0, sinks=0, scale=0.0,
                     workspace=None, stream=None):
        """Causal attention of q [n_seq, n, heads, head_dim] (normalized, rotated: paged_append's q_out) over the pages of
        their sequences (as in paged_append, which must have written the rows' own keys) into out, times sigmoid(gate):
        one token a sequence, a few or a chunk. window: a token sees its last `window` positions and the first `sinks`
        (0: all). scale 0: 1 / sqrt(head_dim). Tokens that paged_append left out for lying past the rope rows are to be kept
        out by `lens` or a table of no more pages than those rows have positions. workspace: a tensor of paged_workspace() bytes (None: from torch's
        allocator)."""
        if q.dtype not in _ROW_DT or len(q.shape) != 4:
            raise ValueError(f"q must be float32 or bfloat16 [n_seq, n, heads, head_dim], got {q.dtype} {tuple(q.shape)}")
        dtype, (n_seq, n) = q.dtype, q.shape[:2]
        heads = (n_seq, n, self.NH, self.D)
        q_stride, q_head = _check_head_rows(q, "q", heads, dtype)
        gate_stride, gate_head = _check_head_rows(gate, "gate", heads, dtype) if gate is not None else (0, 0)
        out_stride = _check_seq_rows(out, "out", heads, dtype)
        cache = self._paged_cache(kpool, vpool, table, pos, lens, n_seq)
        s = self._on_device((q, kpool, vpool, table, pos, out, gate, lens, workspace), stream)
        if self._paged_ws is None:
            self._paged_ws = self.paged_workspace()
        ws, ws_bytes, keep = self._workspace(self._paged_ws, workspace, stream)
        args = _PAGED_ATTEND.pack(*cache, n_seq, n, _ROW_DT[dtype], window, sinks, scale, _ptr(lens) or 0, pos.data_ptr(),
                                  q.data_ptr(), q_stride, q_head, _ptr(gate) or 0, gate_stride, gate_head, out.data_ptr(),
                                  out_stride, ws, ws_bytes)
        self._check(self.lib.qwattn_paged_attend(self.h, s, args))

    def qsa_key_bits(self, mask, cr, pos, n, key_bits, stream=None):
        """Per-key visibility bits [n, kb_words] from a block mask [n, mask_words] (shaders/attention.comp:35-43)."""
        self._check(self.lib.qwattn_qsa_key_bits(self.h, _stream(stream), _ptr(mask), mask.shape[-1], cr, pos, n,
                                                 _ptr(key_bits), key_bits.shape[-1]))

    def attend_partial_qsa(self, q, kcache, vcache, kv_cap, pos, n, n_split, key_bits, stream=None):
        """attend_partial over the keys whose bit is set in key_bits [n, kb_words]; returns the split count."""
        used = ctypes.c_int()
        self._check(self.lib.qwattn_attend_partial_qsa(self.h, _stream(stream), _ptr(q), _ptr(kcache), _ptr(vcache),
                                                       kv_cap, pos, n, n_split, _ptr(key_bits), key_bits.shape[-1],
                                                       ctypes.byref(used)))
        return used.value

    def decode_qsa(self, qg, k, v, qn, kn, rope, kcache, vcache, kv_cap, out, pos, n, n_split, key_bits, stream=None):
        """decode over the keys whose bit is set in key_bits [n, kb_words]; returns the split count."""
        used = ctypes.c_int()
        self._check(self.lib.qwattn_decode_qsa(
            self.h, _stream(stream), _ptr(qg), _ptr(k), _ptr(v), _DT[qg.dtype], _ptr(qn), _ptr(kn), _ptr(rope),
            _ptr(kcache), _ptr(vcache), kv_cap, _ptr(out), pos, n, n_split, _ptr(key_bits), key_bits.shape[-1],
            ctypes.byref(used)))
        return used.value

    def attend_prefill_qsa(self, q, kcache, vcache, kv_cap, qg, out, pos, n, key_bits, stream=None):
        """attend_prefill over the keys whose bit is set in key_bits [n, kb_words]."""
        self._check(self.lib.qwattn_attend_prefill_qsa(self.h, _stream(stream), _ptr(q), _DT[q.dtype], _ptr(kcache),
                                                       _ptr(vcache), kv_cap, _ptr(qg), _DT[qg.dtype], _ptr(out), pos,
                                                       n, _ptr(key_bits), key_bits.shape[-1]))

    def prefill_qsa(self, qg, k, v, qn, kn, rope, kcache, vcache, kv_cap, out, pos, n, key_bits, stream=None):
        """prefill (norm + rope + append, MFMA attention) over the keys whose bit is set in key_bits."""
        self._check(self.lib.qwattn_prefill_qsa(
            self.h, _stream(stream), _ptr(qg), _ptr(k), _ptr(v), _DT[qg.dtype], _ptr(qn), _ptr(kn), _ptr(rope),
            _ptr(kcache), _ptr(vcache), kv_cap, _ptr(out), pos, n, _ptr(key_bits), key_bits.shape[-1]))

    def layer_attention_qsa(self, slot, qg, k, v, qn, kn, out, pos, n, key_bits, n_split=0, stream=None):
        self._check(self.lib.qwattn_layer_attention_qsa(
            self.h, _stream(stream), slot, _ptr(qg), _ptr(k), _ptr(v), _DT[qg.dtype], _ptr(qn), _ptr(kn), _ptr(out),
            pos, n, n_split, _ptr(key_bits), key_bits.shape[-1]))

    def attend_prefill_qg(self, qg, qn, rope, kcache, vcache, kv_cap, out, pos, n, stream=None):
        """The MFMA prefill normalizing and rotating the query half of qg itself (the chunk's K/V rows
        already appended)."""
        self._check(self.lib.qwattn_attend_prefill_qg(self.h, _stream(stream), _ptr(qg), _DT[qg.dtype], _ptr(qn),
                                                      _ptr(rope), _ptr(kcache), _ptr(vcache), kv_cap, _ptr(out),
                                                      pos, n))

    def prefill(self, qg, k, v, qn, kn, rope, kcache, vcache, kv_cap, out, pos, n, stream=None):
        """Norm + rope + append of the chunk's K/V rows, then the MFMA prefill normalizing the query rows
        itself (rope_dim 0, 32, 64, 128 or 256; other widths go through the context's fp16 query buffer):
        two launches."""
        self._check(self.lib.qwattn_prefill(
            self.h, _stream(stream), _ptr(qg), _ptr(k), _ptr(v), _DT[qg.dtype], _ptr(qn), _ptr(kn), _ptr(rope),
            _ptr(kcache), _ptr(vcache), kv_cap, _ptr(out), pos, n))

    def attend(self, q, kcache, vcache, kv_cap, qg, out, pos, n, n_split=0, stream=None):
        """Split-KV + combine when n * NH/NKV <= 32, else the prefill kernel (q fp32 unscaled)."""
        if n * (self.NH // self.NKV) <= 32:
            used = self.attend_partial(q, kcache, vcache, kv_cap, pos, n, n_split, stream)
            self.combine(qg, out, n, used, stream)
        else:
            self.attend_prefill(q, kcache, vcache, kv_cap, qg, out, pos, n, stream)

    def sync_status(self, stream=None):
        """Waits for the stream; raises QwattnError(ETIMEOUT) once if a bounded in-kernel wait gave up."""
        self._check(self.lib.qwattn_sync_status(self.h, _stream(stream)))

    def set_wait_limits(self, spin_max=0, epoch_skew=0):
        """Test hook of the decode kernels' bounded waits (0, 0 = production defaults)."""
        self._check(self.lib.qwattn_set_wait_limits(self.h, spin_max, epoch_skew))

    def set_alloc_fault(self, nth):
        """Test hook: the nth K/V buffer allocation of the next kv_alloc / kv_grow fails (0 = off)."""
        self._check(self.lib.qwattn_set_alloc_fault(self.h, nth))

    def layer_attention(self, slot, qg, k, v, qn, kn, out, pos, n, n_split=0, stream=None):
        self._check(self.lib.qwattn_layer_attention(self.h, _stream(stream), slot, _ptr(qg), _ptr(k), _ptr(v),
                                                    _DT[qg.dtype], _ptr(qn), _ptr(kn), _ptr(out), pos, n, n_split))


def decode_noalloc(cfg, qg, k, v, qn, kn, rope, kcache, vcache, kv_cap, out, pos, n, n_split=0, wait_status=None,
                   device=0, stream=None):
    """qwattn_decode without a context or allocation (library-static scratch); returns the split count."""
    lib = load_library()
    used = ctypes.c_int()
    rc = lib.qwattn_decode_noalloc(device, _stream(stream), ctypes.byref(cfg), _ptr(qg), _ptr(k), _ptr(v),
                                   _DT[qg.dtype], _ptr(qn), _ptr(kn), _ptr(rope), _ptr(kcache), _ptr(vcache), kv_cap,
                                   _ptr(out), pos, n, n_split, _ptr(wait_status), ctypes.byref(used))
    if rc:
        raise QwattnError(rc, lib.qwattn_last_error(None).decode())
    return used.value


@functools.lru_cache(maxsize=4096)
def delta_workspace(n_seq, n, k_heads, v_heads, key_dim, val_dim, dtype, gated=False, snap=False):
    """Bytes of workspace that an Attention.delta_rule call of these sizes, or of fewer sequences or tokens, needs at most
    (gated: with z, or without)."""
    lib, size = load_library(), ctypes.c_size_t()
    some = 256  # any address: only whether z and snap are set is looked at
    args = _DELTA.pack(n_seq, n, k_heads, v_heads, key_dim, val_dim, 0, _ROW_DT[dtype], 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0,
                       some if snap else 0, some if gated else 0, 0, 0, 0, 0, 0, 0)
    rc = lib.qwattn_delta_workspace(args, ctypes.byref(size))
    if rc:
        raise QwattnError(rc, lib.qwattn_last_error(None).decode())
    return size.value


@functools.lru_cache(maxsize=4096)
def moe_workspace(n_experts, hidden, ffn, dtype, n, top_k):
    """Bytes of workspace that an Attention.moe call of these sizes, or of fewer rows, needs at most."""
    lib, size = load_library(), ctypes.c_size_t()
    rc = lib.qwattn_moe_workspace(_MOE_LAYER.pack(n_experts, hidden, ffn, 0, 0, 0, 0, 0, 0), _ROW_DT[dtype], n, top_k,
                                  ctypes.byref(size))
    if rc:
        raise QwattnError(rc, lib.qwattn_last_error(None).decode())
    return size.value


class _DeviceArray:
    """Minimal __cuda_array_interface__ exporter so torch can view library-owned device memory."""

    def __init__(self, ptr, n, typestr):
        self.__cuda_array_interface__ = {"shape": (n,), "typestr": typestr, "data": (ptr, False), "version": 3,
                                         "strides": None}


def _wrap_device_floats(ptr, n, device):
    return torch.as_tensor(_DeviceArray(ptr, n, "<f4"), device=f"cuda:{device}")


def _wrap_device_halfs(ptr, n, device):
    return torch.as_tensor(_DeviceArray(ptr, n, "<f2"), device=f"cuda:{device}")
