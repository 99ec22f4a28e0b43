"""Python binding of libkvexp_b200.so (the C ABI in include/kvexp_b200.h).

Mirrors the reference library's public API (namespace kvexp, include/kvexp/*.hpp of
cvs0/compressed-kv-attention): attention_decode, encode_bf16 / decode_bf16 / EncodedTensor,
Backend, plus the GPU-native batched plan.  Arguments may be numpy arrays (host memory), torch
tensors (host or CUDA), raw integer addresses or None.  Errors raise the Python counterpart of the
reference's exception type:

    std::invalid_argument -> ValueError
    std::runtime_error    -> RuntimeError
    std::logic_error      -> LogicError

There is no CPU fallback: importing this module fails when the shared library is missing.
"""
from __future__ import annotations

import ctypes as C
import enum
import os
import struct

import numpy as np

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "lib", "libkvexp_b200.so")

KVX_OK = 0
KVX_ERR_INVALID_ARGUMENT = 1
KVX_ERR_RUNTIME = 2
KVX_ERR_LOGIC = 3
KVX_ERR_CUDA = 4
KVX_ERR_TIMEOUT = 5
KVX_ERR_UNSUPPORTED = 6

K_ENCODE_BLOCK = 128   # kEncodeBlock, include/kvexp/bf16.hpp:12
K_MAX_HEAD_DIM = 256   # kMaxHeadDim, include/kvexp/bf16.hpp:13


class Backend(enum.IntEnum):
    """kvexp::Backend (include/kvexp/attention.hpp:10-14).  All values run the GPU kernels; the
    value selects the reference's shape rule and error text."""
    Scalar = 0
    Avx2 = 1
    Avx512Bf16 = 2


class LogicError(Exception):
    """std::logic_error of the reference (encoder size-model drift)."""


class CudaError(RuntimeError):
    """A CUDA runtime call inside the library failed."""


class DeviceTimeout(RuntimeError):
    """A bounded device-side wait expired (the kernel returned instead of hanging)."""


if not os.path.exists(LIB_PATH):
    raise ImportError(f"{LIB_PATH} is missing: build it with "
                      "`python compressed-kv-attention_b200/build.py` (there is no CPU fallback)")

_lib = C.CDLL(LIB_PATH)

_vp = C.c_void_p
_sz = C.c_size_t


class kvx_block(C.Structure):
    _fields_ = [("offset", C.c_uint32), ("n_escape", C.c_uint16), ("mode", C.c_uint8),
                ("n_tokens", C.c_uint8)]


class kvx_unit(C.Structure):
    _fields_ = [("k", _vp), ("v", _vp), ("k_index", _vp), ("v_index", _vp), ("q", _vp),
                ("out", _vp), ("k_bytes", C.c_uint64), ("v_bytes", C.c_uint64),
                ("n_blocks", C.c_int32), ("seq", C.c_int32), ("lse", _vp)]


def _sig(name, res, args):
    f = getattr(_lib, name)
    f.restype = res
    f.argtypes = args
    return f


_last_error = _sig("kvx_last_error", C.c_char_p, [])
_version = _sig("kvx_version", C.c_char_p, [])
_device_info = _sig("kvx_device_info", C.c_int, [C.POINTER(C.c_int)] * 3 + [C.POINTER(_sz)])
_attention = _sig("kvx_attention_decode", C.c_int,
                  [C.c_int, _vp, _vp, _vp, _vp, _sz, _vp, _sz, _vp, C.c_int, C.c_int, C.c_int,
                   C.c_int, C.c_int])
_attention_units = _sig("kvx_attention_decode_units", C.c_int,
                        [C.c_int, C.c_int, _vp, _vp, _vp, _vp, _vp, _vp, C.c_int, C.c_int,
                         C.c_int, C.c_int])
_encode_bound = _sig("kvx_encode_bound", _sz, [C.c_int, C.c_int, C.c_int])
_encode = _sig("kvx_encode_bf16", C.c_int,
               [_vp, C.c_int, C.c_int, C.c_int, _vp, _sz, C.POINTER(_sz)])
_encode_bits = _sig("kvx_encode_bf16_bits", C.c_int,
                    [_vp, C.c_int, C.c_int, C.c_int, C.c_int, _vp, _sz, C.POINTER(_sz)])
_decode = _sig("kvx_decode_bf16", C.c_int, [_vp, _sz, C.c_int, C.c_int, _vp])
_xkv_index = _sig("kvx_xkv_index", C.c_int,
                  [_vp, _sz, C.c_int, _vp, C.c_int, C.POINTER(C.c_int), C.POINTER(C.c_longlong)])
_plan_create = _sig("kvx_plan_create", C.c_int,
                    [_vp, C.c_int, C.c_int, C.c_int, C.c_int, C.POINTER(_vp)])
_plan_run = _sig("kvx_plan_run", C.c_int, [_vp, _vp])
_plan_run_part = _sig("kvx_plan_run_part", C.c_int, [_vp, C.c_int, _vp])
_plan_check = _sig("kvx_plan_check", C.c_int, [_vp])
_plan_launches = _sig("kvx_plan_launches", C.c_int, [_vp])
_plan_split = _sig("kvx_plan_split_units", C.c_int, [_vp])
_plan_destroy = _sig("kvx_plan_destroy", None, [_vp])
_enc_bounds = _sig("kvx_encode_batch_bounds", C.c_int,
                   [C.c_int, C.c_int, C.c_int, C.c_int, C.POINTER(_sz), C.POINTER(_sz)])
_enc_batch = _sig("kvx_encode_batch", C.c_int,
                  [C.c_int, _vp, C.c_int, C.c_int, C.c_int, _vp, _sz, _vp, _vp, _vp, _vp])
_enc_batch_bits = _sig("kvx_encode_batch_bits", C.c_int,
                       [C.c_int, _vp, C.c_int, C.c_int, C.c_int, C.c_int, _vp, _sz, _vp, _vp,
                        _vp, _vp])
_append_bits = _sig("kvx_cache_append_bits", C.c_int,
                    [_vp, C.c_int, C.c_int, C.c_int, C.c_int, _vp, _sz, _sz, _vp,
                     C.POINTER(_sz), C.POINTER(C.c_int), _vp])
_append = _sig("kvx_cache_append", C.c_int,
               [_vp, C.c_int, C.c_int, C.c_int, _vp, _sz, _sz, _vp, C.POINTER(_sz),
                C.POINTER(C.c_int), _vp])
_synth = _sig("kvx_synth_bf16", C.c_int,
              [_vp, C.c_int, C.c_int, C.c_uint64, C.c_uint64, C.c_int, C.c_uint32, _vp])
_probe = _sig("kvx_hbm_read_probe", C.c_int, [_vp, _sz, C.c_int, C.POINTER(C.c_double)])
_noalloc = _sig("kvx_attention_decode_noalloc", C.c_int,
                [_vp, _vp, _sz, _vp, _vp, _sz, _vp, C.c_int, _vp, C.c_int, C.c_int, C.c_int, _vp])
_fold = _sig("kvx_fold_shards", C.c_int, [_vp, C.c_int, C.c_int, C.c_int, _vp, _vp, _vp])
_expstats = _sig("kvx_exponent_stats", C.c_int, [_vp, C.c_int, C.c_int, C.c_int, _vp, _vp])



class kvx_view(C.Structure):
    _fields_ = [("data", _vp), ("token_stride", C.c_int64), ("head_stride", C.c_int64)]


class kvx_pages(C.Structure):
    _fields_ = [("k", _vp), ("v", _vp), ("page_stride", C.c_int64), ("token_stride", C.c_int64),
                ("head_stride", C.c_int64), ("n_pages", C.c_int32), ("page_tokens", C.c_int32)]


class kvx_rope(C.Structure):
    _fields_ = [("cos", _vp), ("sin", _vp), ("pos", _vp), ("axis", _vp), ("pos_stride", C.c_int64),
                ("n_pos", C.c_int32), ("rot_dim", C.c_int32), ("n_axes", C.c_int32),
                ("interleaved", C.c_int32)]


class kvx_attend(C.Structure):
    _fields_ = [("q", kvx_view), ("out", kvx_view), ("lse", _vp), ("pages", _vp),
                ("prefix_table", _vp), ("prefix", _vp), ("table", _vp), ("lens", _vp), ("table_stride", C.c_int64),
                ("prefix_len", C.c_int32), ("max_len", C.c_int32), ("batch", C.c_int32),
                ("scale", C.c_float)]


# The serving-step calls take these structs many times a token: they go as packed bytes, whose address
# ctypes passes as it is (building the ctypes objects costs several microseconds a call).
_pack_view = struct.Struct("@Pqq").pack
_pack_rope = struct.Struct("@PPPPqiiii").pack
_pack_attend = struct.Struct("@PqqPqqPPPPPPqiiif").pack
assert struct.calcsize("@Pqq") == C.sizeof(kvx_view) and struct.calcsize("@PPPPqiiii") == C.sizeof(kvx_rope)
assert struct.calcsize("@PqqPqqPPPPPPqiiif") == C.sizeof(kvx_attend)
_buf = C.c_char_p

_batch_create = _sig("kvx_batch_create", C.c_int,
                     [C.c_int, C.c_int, C.c_int, C.c_int, C.c_int, C.POINTER(_vp)])
_batch_rotate = _sig("kvx_batch_rotate", C.c_int,
                     [_vp, _buf, _buf, C.c_int, C.c_int, _buf, C.c_int, _vp])
_batch_append = _sig("kvx_batch_append", C.c_int,
                     [_vp, _buf, _buf, _buf, _buf, C.c_int, _buf, _vp, _buf, _vp])
_batch_attend = _sig("kvx_batch_attend", C.c_int, [_vp, _buf, _vp])
_batch_wait_limit = _sig("kvx_batch_wait_limit", C.c_int, [_vp, C.c_int])
_batch_check = _sig("kvx_batch_check", C.c_int, [_vp])
_batch_destroy = _sig("kvx_batch_destroy", None, [_vp])
_prefix_create = _sig("kvx_prefix_create", C.c_int, [_vp, C.c_int, C.c_int, C.POINTER(_vp)])
_prefix_destroy = _sig("kvx_prefix_destroy", None, [_vp])

# Every symbol the C header declares, for load/export checks.
EXPORTED = [
    "kvx_last_error", "kvx_version", "kvx_device_info", "kvx_attention_decode",
    "kvx_attention_decode_units", "kvx_encode_bound", "kvx_encode_bf16", "kvx_decode_bf16",
    "kvx_xkv_index", "kvx_plan_create", "kvx_plan_run", "kvx_plan_run_part", "kvx_plan_check", "kvx_plan_launches", "kvx_plan_split_units",
    "kvx_plan_destroy", "kvx_encode_batch_bounds", "kvx_encode_batch", "kvx_cache_append",
    "kvx_synth_bf16", "kvx_hbm_read_probe", "kvx_attention_decode_noalloc", "kvx_fold_shards",
    "kvx_exponent_stats", "kvx_encode_bf16_bits", "kvx_encode_batch_bits", "kvx_cache_append_bits",
    "kvx_batch_create", "kvx_batch_rotate", "kvx_batch_append", "kvx_batch_attend",
    "kvx_batch_wait_limit", "kvx_batch_check", "kvx_batch_destroy", "kvx_prefix_create", "kvx_prefix_destroy",
]

# Residual code widths the encoder may use (include/kvexp_b200.h KVX_CODE_BITS_*): the reference's
# {2, 4}, or with the library's 3-bit extension.
CODE_BITS_REFERENCE = 0x14
CODE_BITS_ALL = 0x1C


def _check(rc: int) -> None:
    if rc == KVX_OK:
        return
    msg = (_last_error() or b"").decode()
    if rc == KVX_ERR_INVALID_ARGUMENT:
        raise ValueError(msg)
    if rc == KVX_ERR_LOGIC:
        raise LogicError(msg)
    if rc == KVX_ERR_CUDA:
        raise CudaError(msg)
    if rc == KVX_ERR_TIMEOUT:
        raise DeviceTimeout(msg)
    if rc == KVX_ERR_UNSUPPORTED:
        raise NotImplementedError(msg)
    raise RuntimeError(msg)


def _addr(x):
    """Address of a numpy array / torch tensor / int / None."""
    if x is None:
        return None
    if isinstance(x, int):
        return x
    if isinstance(x, np.ndarray):
        if not x.flags["C_CONTIGUOUS"]:
            raise ValueError("arrays must be C-contiguous")
        return x.ctypes.data
    if hasattr(x, "data_ptr"):
        if not x.is_contiguous():
            raise ValueError("tensors must be contiguous")
        return x.data_ptr()
    raise TypeError(f"unsupported buffer type {type(x)!r}")


def _nbytes(x):
    if isinstance(x, np.ndarray):
        return x.nbytes
    if hasattr(x, "data_ptr"):
        return x.numel() * x.element_size()
    raise TypeError("size unknown for raw addresses; pass the byte count")


def version() -> str:
    return _version().decode()


def device_info() -> dict:
    a, b, n = C.c_int(0), C.c_int(0), C.c_int(0)
    mem = _sz(0)
    _check(_device_info(C.byref(a), C.byref(b), C.byref(n), C.byref(mem)))
    return {"sm": (a.value, b.value), "sm_count": n.value, "hbm_bytes": mem.value}


def attention_decode(backend, q, k_raw, v_raw, k_xkv, k_bytes, v_xkv, v_bytes, out, n_q, dim,
                     seq, n_threads, split_tokens=K_ENCODE_BLOCK):
    """kvexp::attention_decode (include/kvexp/attention.hpp:58-61), run on the GPU."""
    _check(_attention(int(backend), _addr(q), _addr(k_raw), _addr(v_raw), _addr(k_xkv),
                      int(k_bytes), _addr(v_xkv), int(v_bytes), _addr(out), int(n_q), int(dim),
                      int(seq), int(n_threads), int(split_tokens)))


def attention_decode_units(backend, qs, kxs, k_bytes, vxs, v_bytes, outs, n_q, dim, seq,
                           split_tokens=K_ENCODE_BLOCK):
    """All (layer, KV head) units of a step in one GPU job (the reference's model_heads loop)."""
    n = len(qs)
    arr = lambda xs: (C.c_void_p * n)(*[_addr(x) for x in xs])
    kb = (_sz * n)(*[int(b) for b in k_bytes])
    vb = (_sz * n)(*[int(b) for b in v_bytes])
    _check(_attention_units(int(backend), n, arr(qs), arr(kxs), kb, arr(vxs), vb, arr(outs),
                            int(n_q), int(dim), int(seq), int(split_tokens)))


class EncodedTensor:
    """kvexp::EncodedTensor (include/kvexp/codec.hpp:38-43): bytes (numpy uint8) + shape."""

    def __init__(self, data, seq_len, head_dim, block_tokens):
        self.bytes = data
        self.seq_len = seq_len
        self.head_dim = head_dim
        self.block_tokens = block_tokens


def encode_bound(seq_len, head_dim, block_tokens=K_ENCODE_BLOCK) -> int:
    return int(_encode_bound(int(seq_len), int(head_dim), int(block_tokens)))


def encode_bf16(kv, seq_len, head_dim, block_tokens=K_ENCODE_BLOCK,
                code_bits=CODE_BITS_REFERENCE) -> EncodedTensor:
    """kvexp::encode_bf16 (include/kvexp/codec.hpp:45-46) on the GPU; byte-identical output.
    code_bits=CODE_BITS_ALL also allows 3-bit blocks (the library's extension)."""
    cap = max(16, encode_bound(seq_len, head_dim, block_tokens))
    out = np.zeros(cap, dtype=np.uint8)
    nb = _sz(0)
    if code_bits == CODE_BITS_REFERENCE:
        _check(_encode(_addr(kv), int(seq_len), int(head_dim), int(block_tokens), out.ctypes.data,
                       cap, C.byref(nb)))
    else:
        _check(_encode_bits(_addr(kv), int(seq_len), int(head_dim), int(block_tokens),
                            int(code_bits), out.ctypes.data, cap, C.byref(nb)))
    return EncodedTensor(out[: nb.value].copy(), seq_len, head_dim, block_tokens)


def decode_bf16(blob, nbytes, seq_len, head_dim, out):
    """kvexp::decode_bf16 (include/kvexp/codec.hpp:48) on the GPU."""
    _check(_decode(_addr(blob), int(nbytes), int(seq_len), int(head_dim), _addr(out)))


def xkv_index(blob, nbytes, head_dim, index, max_blocks):
    """Block index of a device blob into device memory `index`; returns (n_blocks, n_tokens)."""
    nb, nt = C.c_int(0), C.c_longlong(0)
    _check(_xkv_index(_addr(blob), int(nbytes), int(head_dim), _addr(index), int(max_blocks),
                      C.byref(nb), C.byref(nt)))
    return nb.value, nt.value


def attention_decode_noalloc(q, k_xkv, k_bytes, k_index, v_xkv, v_bytes, v_index, n_blocks, out,
                             n_q, dim, seq, stream=None):
    """One decode step over device-resident XKV K/V that allocates no GPU memory (for callers
    whose device memory is all reserved up front; see kvx_attention_decode_noalloc).  Every
    argument is device memory; the indexes come from xkv_index or the GPU encoder."""
    _check(_noalloc(_addr(q), _addr(k_xkv), int(k_bytes), _addr(k_index), _addr(v_xkv),
                    int(v_bytes), _addr(v_index), int(n_blocks), _addr(out), int(n_q), int(dim),
                    int(seq), _addr(stream)))


def fold_shards(parts, n_parts, n_rows, dim, out, lse_out=None, stream=None):
    """Rank-ordered fold of sequence-shard results on the GPU (kvx_fold_shards): parts holds
    n_parts blocks of [n_rows * dim outputs, n_rows lse] FP32; asynchronous on `stream`."""
    _check(_fold(_addr(parts), int(n_parts), int(n_rows), int(dim), _addr(out), _addr(lse_out),
                 stream))


class Plan:
    """A reusable batched decode step (kvx_plan): fixed units, one launch (+ combine) per run."""

    def __init__(self, units, n_q, dim, block_tokens=K_ENCODE_BLOCK):
        arr = (kvx_unit * len(units))(*units)
        h = _vp()
        _check(_plan_create(C.cast(arr, _vp), len(units), int(n_q), int(dim), int(block_tokens),
                            C.byref(h)))
        self._h = h

    def run(self, stream=None):
        _check(_plan_run(self._h, stream))

    def run_part(self, part, stream=None):
        _check(_plan_run_part(self._h, int(part), stream))

    @property
    def n_split(self) -> int:
        return int(_plan_split(self._h))

    def check(self):
        _check(_plan_check(self._h))

    @property
    def launches(self) -> int:
        return int(_plan_launches(self._h))

    def close(self):
        if self._h:
            _plan_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def make_unit(k, v, q, out, *, k_index=None, v_index=None, k_bytes=0, v_bytes=0, n_blocks=0,
              seq, lse=None) -> kvx_unit:
    return kvx_unit(_addr(k), _addr(v), _addr(k_index), _addr(v_index), _addr(q), _addr(out),
                    int(k_bytes), int(v_bytes), int(n_blocks), int(seq), _addr(lse))


def encode_batch_bounds(n_tensors, seq, head_dim, block_tokens=K_ENCODE_BLOCK):
    a, b = _sz(0), _sz(0)
    _check(_enc_bounds(int(n_tensors), int(seq), int(head_dim), int(block_tokens), C.byref(a),
                       C.byref(b)))
    return a.value, b.value


def encode_batch(tensors, seq, head_dim, arena, index, block_tokens=K_ENCODE_BLOCK,
                 stream=None, code_bits=CODE_BITS_REFERENCE):
    """GPU-encode device tensors into `arena`; returns (blob_offsets, blob_bytes) numpy arrays."""
    n = len(tensors)
    ptrs = (C.c_void_p * n)(*[_addr(t) for t in tensors])
    off = np.zeros(n, dtype=np.uint64)
    nb = np.zeros(n, dtype=np.uint64)
    if code_bits == CODE_BITS_REFERENCE:
        _check(_enc_batch(n, C.cast(ptrs, _vp), int(seq), int(head_dim), int(block_tokens),
                          _addr(arena), _nbytes(arena), _addr(index), off.ctypes.data,
                          nb.ctypes.data, stream))
    else:
        _check(_enc_batch_bits(n, C.cast(ptrs, _vp), int(seq), int(head_dim), int(block_tokens),
                               int(code_bits), _addr(arena), _nbytes(arena), _addr(index),
                               off.ctypes.data, nb.ctypes.data, stream))
    return off, nb


def cache_append(kv_new, n_new, head_dim, blob, at, capacity, index,
                 block_tokens=K_ENCODE_BLOCK, stream=None, code_bits=CODE_BITS_REFERENCE):
    """Encode n_new tokens and append them at byte `at` of a device blob; returns
    (bytes_written, blocks_written)."""
    bw, kw = _sz(0), C.c_int(0)
    if code_bits == CODE_BITS_REFERENCE:
        _check(_append(_addr(kv_new), int(n_new), int(head_dim), int(block_tokens), _addr(blob),
                       int(at), int(capacity), _addr(index), C.byref(bw), C.byref(kw), stream))
    else:
        _check(_append_bits(_addr(kv_new), int(n_new), int(head_dim), int(block_tokens),
                            int(code_bits), _addr(blob), int(at), int(capacity), _addr(index),
                            C.byref(bw), C.byref(kw), stream))
    return bw.value, kw.value


def synth_bf16(out, seq, dim, seed, stream_id, profile, rate, stream=None):
    _check(_synth(_addr(out), int(seq), int(dim), int(seed), int(stream_id), int(profile),
                  int(rate), stream))


def hbm_read_probe(buf, nbytes=None, reps=10) -> float:
    g = C.c_double(0)
    _check(_probe(_addr(buf), int(nbytes if nbytes is not None else _nbytes(buf)), int(reps),
                  C.byref(g)))
    return g.value


def exponent_stats(kv, seq_len, head_dim, block_tokens=K_ENCODE_BLOCK):
    """kvx_exponent_stats on a [seq_len, head_dim] BF16 tensor (host numpy or a device tensor):
    returns (best [3, n_blocks, head_dim] int32 for windows of 3 / 7 / 15 exponents,
    entropy [n_blocks, head_dim] float32)."""
    nb = (int(seq_len) + int(block_tokens) - 1) // int(block_tokens)
    best = np.zeros((3, nb, int(head_dim)), dtype=np.int32)
    ent = np.zeros((nb, int(head_dim)), dtype=np.float32)
    _check(_expstats(_addr(kv), int(seq_len), int(head_dim), int(block_tokens), best.ctypes.data,
                     ent.ctypes.data))
    return best, ent


def exponent_report(kv, seq_len, head_dim, block_tokens=K_ENCODE_BLOCK, bit_widths=(2, 3, 4)):
    """The reference analyser's per-tensor report from the GPU statistics: the size policy
    (python/analyze_exponents.py:117-156 `policy_size`: per block the smallest of the raw
    container and each residual width, ties to raw, then fewer escapes, then narrower codes) and
    the mean entropy of the exponent in each (full block, dim) (`block_conditional_entropy`,
    :57-72; nan when there is no full block)."""
    seq, dim, bt = int(seq_len), int(head_dim), int(block_tokens)
    best, ent = exponent_stats(kv, seq, dim, bt)
    col = {2: 0, 3: 1, 4: 2}
    total = 0
    esc_total = 0
    coded = 0
    modes = {}
    for b in range(best.shape[1]):
        n = min(bt, seq - b * bt)
        options = [(0, 8 + 2 * n * dim, 0)]
        for bits in bit_widths:
            n_esc = n * dim - int(best[col[bits], b].sum())
            options.append((bits, 8 + dim + n * dim + (n * dim * bits + 7) // 8 + 2 * n_esc, n_esc))
        mode, size, n_esc = min(options, key=lambda t: (t[1], 0 if t[0] == 0 else 1, t[2], t[0]))
        total += size
        esc_total += n_esc
        modes[mode] = modes.get(mode, 0) + 1
        if mode != 0:
            coded += n * dim
    full = seq // bt
    tight = 2 * seq * dim
    return {
        "container_bytes": total, "tight_bytes": tight, "ratio": total / tight,
        "escape_rate": esc_total / (seq * dim), "coded_element_fraction": coded / (seq * dim),
        "mode_blocks": {str(k): v for k, v in sorted(modes.items())},
        "block_conditional_entropy": float(ent[:full].astype(np.float64).mean()) if full else float("nan"),
    }


# ---- serving step: rotation, paged cache, attention over a shared prefix ---------------------------
#
# These calls take CUDA tensors (torch) of any strides whose last dimension is contiguous, run on
# `stream` (a cudaStream_t address, default the legacy stream) and return at once.

DTYPES = {"bf16": (0, "bfloat16"), "fp16": (1, "float16")}


def _device_tensor(x, name, dtype, ndim, device=None):
    """Checks what the device code takes on trust: a CUDA tensor of this type and rank, on this device
    if one is given, its last dimension contiguous.  Returns its strides."""
    at = x.get_device() if hasattr(x, "get_device") else -1
    if at != device:
        if at < 0:
            raise ValueError(f"{name} must be a CUDA tensor")
        if device is not None:
            raise ValueError(f"{name} is on device {at}, not on device {device}")
    if x.dtype is not dtype:
        raise ValueError(f"{name} must be {dtype}, not {x.dtype}")
    st = x.stride()
    if len(st) != ndim:
        raise ValueError(f"{name} must have {ndim} dimensions, not {len(st)}")
    if st[-1] != 1 and x.shape[-1] > 1:
        raise ValueError(f"{name}: the last dimension must be contiguous")
    return st


class Rope:
    """A rotation's tables (kvx_rope): cos and sin [n_pos, rot_dim / 2] FP32; with several axes
    (time, height, width), axis [rot_dim / 2] uint8 gives each pair's."""

    def __init__(self, cos, sin, axis=None, n_axes=1, interleaved=False):
        import torch
        _device_tensor(cos, "cos", torch.float32, 2)
        self.device = cos.get_device()
        for name, x in (("cos", cos), ("sin", sin)):
            _device_tensor(x, name, torch.float32, 2, self.device)
            if not x.is_contiguous() or x.shape != cos.shape:
                raise ValueError("cos and sin must be contiguous and of one shape")
        if axis is not None:
            _device_tensor(axis, "axis", torch.uint8, 1, self.device)
            if axis.shape[0] != cos.shape[1]:
                raise ValueError("axis must name one axis for each pair")
        elif n_axes != 1:
            raise ValueError("several axes need the axis of each pair")
        self._keep = (cos, sin, axis)
        self._int32 = torch.int32
        self.n_axes = int(n_axes)
        self._tables = _addr(cos), _addr(sin)
        self._axis = _addr(axis) or 0
        self._rest = int(cos.shape[0]), 2 * int(cos.shape[1]), self.n_axes, int(bool(interleaved))

    def _at(self, pos, n_tokens, device):
        """kvx_rope for positions [n_tokens] or [n_axes, n_tokens] int32 on the device of a batch."""
        if self.device != device:
            raise ValueError(f"the rotation's tables are on device {self.device}, not on device {device}")
        shape = pos.shape
        st = _device_tensor(pos, "pos", self._int32, len(shape), device)
        if shape != (self.n_axes, n_tokens) and (shape != (n_tokens,) or self.n_axes != 1):
            raise ValueError("pos must be [n_tokens], or [n_axes, n_tokens]")
        return _pack_rope(*self._tables, pos.data_ptr(), self._axis, st[0] if len(st) == 2 else 0, *self._rest)


class Pages:
    """One layer's page pools (kvx_pages): k and v [n_pages, page_tokens, n_kv_heads, dim] of the
    same type and strides; heads outside tokens in memory is the transposed view of such a pool."""

    def __init__(self, k, v):
        _device_tensor(k, "k", k.dtype, 4)
        self.device = k.get_device()
        for name, x in (("k", k), ("v", v)):
            _device_tensor(x, name, k.dtype, 4, self.device)
            if x.shape != k.shape or x.stride() != k.stride():
                raise ValueError("k and v must have one shape and one set of strides")
        self.k, self.v = k, v
        self.n_heads, self.dim, self.dtype = int(k.shape[2]), int(k.shape[3]), k.dtype
        self.page_tokens = int(k.shape[1])
        c = kvx_pages(k.data_ptr(), v.data_ptr(), k.stride(0), k.stride(1), k.stride(2), int(k.shape[0]),
                      self.page_tokens)
        self._c = bytes(c)
        self._at = C.cast(C.c_char_p(self._c), _vp).value


class Prefix:
    """A shared prefix kept as XKV blobs (kvx_prefix): one kvx_unit (make_unit without queries) for
    each KV head.  `keep` holds what the units point into."""

    def __init__(self, units, dim, keep=None):
        self._h = None
        self._keep = keep
        self.dim, self.n_heads = int(dim), len(units)
        self.seq = int(units[0].seq) if units else 0
        self.nbytes = sum(int(u.k_bytes) + int(u.v_bytes) for u in units)
        arr = (kvx_unit * len(units))(*units)
        h = _vp()
        _check(_prefix_create(C.cast(arr, _vp), len(units), self.dim, C.byref(h)))
        self._h = h

    @classmethod
    def encode(cls, k, v, block_tokens=K_ENCODE_BLOCK, code_bits=CODE_BITS_REFERENCE):
        """Encodes k and v (BF16 CUDA tensors [n_kv_heads, tokens, dim], contiguous) on the GPU."""
        import torch
        for name, x in (("k", k), ("v", v)):
            _device_tensor(x, name, torch.bfloat16, 3, torch.cuda.current_device())
            if not x.is_contiguous() or x.shape != k.shape:
                raise ValueError("k and v must be contiguous and of one shape")
        heads, seq, dim = (int(n) for n in k.shape)
        if heads == 0 or seq == 0:
            raise ValueError("an empty prefix")
        bound, entries = encode_batch_bounds(2 * heads, seq, dim, block_tokens)
        arena = torch.empty(bound, dtype=torch.uint8, device=k.device)
        index = torch.empty(entries * C.sizeof(kvx_block), dtype=torch.uint8, device=k.device)
        torch.cuda.current_stream(k.device).synchronize()
        off, nb = encode_batch([x for h in range(heads) for x in (k[h], v[h])], seq, dim, arena, index,
                               block_tokens, code_bits=code_bits)
        blobs = arena[:int(off[-1] + nb[-1] + 31) & ~15].clone()  # the bound is of incompressible data
        blocks = -(-seq // block_tokens)
        torch.cuda.current_stream(k.device).synchronize()

        def unit(h):
            at = [blobs.data_ptr() + int(off[2 * h + i]) for i in (0, 1)]
            ix = [index.data_ptr() + (2 * h + i) * blocks * C.sizeof(kvx_block) for i in (0, 1)]
            return make_unit(at[0], at[1], None, None, k_index=ix[0], v_index=ix[1], k_bytes=nb[2 * h],
                             v_bytes=nb[2 * h + 1], n_blocks=blocks, seq=seq)

        return cls([unit(h) for h in range(heads)], dim, keep=(blobs, index))

    def close(self):
        if self._h:
            _prefix_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class Batch:
    """The operators of a batch's serving step (kvx_batch) for one head layout and type ("bf16" or
    "fp16"), with scratch for up to max_batch sequences."""

    def __init__(self, max_batch, n_q_heads, n_kv_heads, dim, dtype="bf16"):
        import torch
        if dtype not in DTYPES:
            raise ValueError(f"dtype must be one of {sorted(DTYPES)}")
        code, name = DTYPES[dtype]
        self._type, self._int32, self._int64, self._float32 = getattr(torch, name), torch.int32, torch.int64, torch.float32
        self.n_q_heads, self.n_kv_heads, self.dim = int(n_q_heads), int(n_kv_heads), int(dim)
        h = _vp()
        self._h = None
        _check(_batch_create(int(max_batch), self.n_q_heads, self.n_kv_heads, self.dim, code,
                             C.byref(h)))
        self._h = h
        self.device = torch.cuda.current_device()

    def _view(self, x, name, tokens, heads):
        """(address, token stride, head stride) of a [tokens, heads, dim] tensor."""
        st = _device_tensor(x, name, self._type, 3, self.device)
        if x.shape != (tokens, heads, self.dim):
            raise ValueError(f"{name} must be {(tokens, heads, self.dim)}, not {tuple(x.shape)}")
        return x.data_ptr(), st[0], st[1]

    def _pages(self, pages):
        if pages.n_heads != self.n_kv_heads or pages.dim != self.dim or pages.dtype is not self._type:
            raise ValueError("the page pools have other heads, another head_dim or another type")
        if pages.device != self.device:
            raise ValueError(f"the page pools are on device {pages.device}, not on device {self.device}")
        return pages

    def rotate(self, x, pos, rope, out, inverse=False, stream=None):
        """out = x [tokens, heads, dim] rotated by its positions (inverse: back, which is the
        gradient's rotation); out may be x."""
        n, heads = x.shape[:2]
        rc = _batch_rotate(self._h, _pack_view(*self._view(x, "x", n, heads)),
                           _pack_view(*self._view(out, "out", n, heads)), n, heads, rope._at(pos, n, self.device),
                           1 if inverse else 0, stream)
        if rc:
            _check(rc)

    def append(self, q, k, v, pos, rope, slots, pages, q_out, stream=None):
        """Store new tokens: k [tokens, n_kv_heads, dim] rotated and v at `slots` (int64, page *
        page_tokens + place; negative: not stored), q rotated into q_out (both None: no queries).
        rope None: nothing is rotated."""
        n = k.shape[0]
        if _device_tensor(slots, "slots", self._int64, 1, self.device) and slots.shape[0] != n:
            raise ValueError("slots must be one for each token")
        if (q is None) != (q_out is None):
            raise ValueError("q and q_out go together")
        kv = self.n_kv_heads
        rc = _batch_append(
            self._h, None if q is None else _pack_view(*self._view(q, "q", n, self.n_q_heads)),
            _pack_view(*self._view(k, "k", n, kv)), _pack_view(*self._view(v, "v", n, kv)),
            None if q is None else _pack_view(*self._view(q_out, "q_out", n, self.n_q_heads)), n,
            None if rope is None else rope._at(pos, n, self.device), slots.data_ptr(), self._pages(pages)._c, stream)
        if rc:
            _check(rc)

    def attend(self, q, out, pages, table, lens, max_len, *, prefix_table=None, prefix_len=0, prefix=None,
               scale=None, lse=None, stream=None):
        """out[b, h] = attention of q [batch, n_q_heads, dim] over the shared prefix (prefix_len
        tokens in the pages of prefix_table, int32, or a Prefix) and then the first lens[b] tokens of
        row b of table (int32 [batch, pages]); max_len bounds lens.  lse [batch, n_q_heads] FP32
        receives the log-sum-exp of the scaled scores."""
        n, heads = q.shape[0], self.n_q_heads
        max_len, prefix_len = int(max_len), int(prefix_len)
        at_table = at_lens = at_prefix = at_lse = stride = 0
        if max_len > 0:
            st = _device_tensor(table, "table", self._int32, 2, self.device)
            _device_tensor(lens, "lens", self._int32, 1, self.device)
            if table.shape[0] != n or lens.shape[0] != n:
                raise ValueError("table and lens must have one row for each sequence")
            if table.shape[1] * pages.page_tokens < max_len:
                raise ValueError("table rows hold fewer than max_len tokens")
            at_table, at_lens, stride = table.data_ptr(), lens.data_ptr(), st[0]
        if prefix_table is not None and prefix_len > 0:
            _device_tensor(prefix_table, "prefix_table", self._int32, 1, self.device)
            if prefix_table.shape[0] * pages.page_tokens < prefix_len:
                raise ValueError("prefix_table holds fewer than prefix_len tokens")
            at_prefix = prefix_table.data_ptr()
        if lse is not None:
            _device_tensor(lse, "lse", self._float32, 2, self.device)
            if lse.shape != (n, heads) or not lse.is_contiguous():
                raise ValueError("lse must be contiguous [batch, n_q_heads]")
            at_lse = lse.data_ptr()
        if scale is not None and not scale > 0:
            raise ValueError("scale must be positive")
        rc = _batch_attend(self._h, _pack_attend(
            *self._view(q, "q", n, heads), *self._view(out, "out", n, heads), at_lse, self._pages(pages)._at,
            at_prefix, 0 if prefix is None else prefix._h.value, at_table, at_lens, stride, prefix_len, max_len,
            n, scale or 0.0), stream)
        if rc:
            _check(rc)

    def wait_limit(self, microseconds):
        """How long a kernel may wait for one of its own copies or matrix products (1 s unless set); what depends on
        a wait that ran out is NaN, and check() raises."""
        _check(_batch_wait_limit(self._h, int(microseconds)))

    def check(self):
        """Synchronise and raise what the device reported since the last check."""
        _check(_batch_check(self._h))

    def close(self):
        if self._h:
            _batch_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
