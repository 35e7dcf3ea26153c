"""Python-side mirror of the operator and layer interface, one thin wrapper per C-ABI entry.

Tensors are torch CUDA fp16/int32 tensors; host arrays are numpy. Nothing here computes: every
function forwards to `libet_b200.so`.
"""
import array
import ctypes
import importlib.util
import os
import struct

import numpy as np

from . import check, lib, ptr, raw_stream
from .build import binding_path

__all__ = [
    "skip_layernorm", "softmax_mask", "TileWeight", "tile_spmm_bias", "tile_spmm_cache_clear",
    "RowWeight", "attention_otf", "attention_prune", "qk_scores", "attention_sharedqk", "attention_batch", "attention_static_scores",
    "gen_sparse_tile_mat", "gen_sparse_row_mat", "build_head_ptr", "Encoder", "encoder_buffer_size",
    "encoder_batch_buffer_size", "KIND_TILE", "KIND_PRUNE", "KIND_LENGTH", "KIND_PRUNE_QKV",
    "Model", "attention_check", "prune_dense_to_tiles", "select_rows_magnitude", "compact_rows", "set_tuning_goal",
    "set_attention_scores_fp32", "attention_scores_fp32", "rotary_axes", "AdapterBank", "attention_rules", "attention_rules_scratch_size",
    "skip_rmsnorm", "quantise_rows", "Fp8Weight", "kv_cache_write", "kv_cache_read", "attention_tree",
]

_i = ctypes.c_int


# The entry points that are called per launch, with their argument types declared: ctypes then converts plain numbers by
# itself, which costs a third of building a c_void_p / c_int object for every argument (p = pointer, i = int, s = size_t).
_SIGNATURES = {
    "et_skip_layernorm": "ppppiip", "et_softmax_mask": "ppiiip", "et_tile_linear": "pppiip", "et_row_linear": "pppip",
    "et_tile_spmm_bias": "pppppiiipip", "et_attention_otf": "pppppiiip", "et_attention_prune": "ppppppipiiip",
    "et_qk_scores": "pppiiip", "et_attention_sharedqk": "ppppiiip", "et_attention_static_scores": "pppppiiip",
    "et_attention_batch": "ppppiippppippiiiiiip", "et_encoder_run": "pppp", "et_encoder_run_batch": "pppppipsp",
    "et_model_run_batch": "pppppip", "et_rotary_axes_by": "p", "et_adapter_add_by": "p", "et_attention_rules_by": "p",
    "et_skip_rmsnorm": "p", "et_quantise_rows": "p", "et_fp8_linear": "p", "et_kv_cache_write": "p", "et_kv_cache_read": "p", "et_attention_tree": "p",
}


class _Entries:
    """One attribute per entry point of _SIGNATURES, bound on first use of the library."""
    __slots__ = tuple(_SIGNATURES)

    def __init__(self):
        types = {"p": ctypes.c_void_p, "i": ctypes.c_int, "s": ctypes.c_size_t}
        for name, signature in _SIGNATURES.items():
            fn = lib()[name]   # a function object of its own: argument types of lib().<name> stay undeclared
            fn.argtypes = [types[c] for c in signature]
            fn.restype = ctypes.c_int
            setattr(self, name, fn)


_entries = None


def _lib():
    global _entries
    if _entries is None:
        _entries = _Entries()
    return _entries


def _a(t):
    """Address of a torch tensor, a numpy array, or None."""
    if t is None:
        return None
    try:
        return t.data_ptr()
    except AttributeError:
        return ptr(t).value


def _ints(values):
    """(address, count, owner) of a sequence of whole numbers as C ints."""
    if type(values) is list or type(values) is tuple:
        try:
            a = array.array("i", values)
            return a.buffer_info()[0], len(a), a
        except TypeError:
            pass   # not all of them are ints: as numpy converts them
    a = np.ascontiguousarray(values, dtype=np.int32)
    return a.ctypes.data, len(a), a


def skip_layernorm(in_out, skip, gamma, beta, stream=None):
    """in_out[num, size] <- LN(in_out + skip) * gamma + beta, in place."""
    num, size = in_out.shape
    rc = (_entries or _lib()).et_skip_layernorm(_a(in_out), _a(skip), _a(gamma), _a(beta), num, size, raw_stream(stream))
    if rc:
        check(rc)
    return in_out


def softmax_mask(scores, mask=None, valid_len=None, stream=None):
    """scores[nmat, L, L] <- softmax(scores + mask) per row, in place."""
    nmat, L, L2 = scores.shape
    assert L == L2
    rc = (_entries or _lib()).et_softmax_mask(_a(scores), _a(mask), nmat, L, L if valid_len is None else valid_len,
                                              raw_stream(stream))
    if rc:
        check(rc)
    return scores


def set_tuning_goal(goal):
    """"latency" (default): weights created afterwards are packed for the shortest single launch; "throughput": for
    the least SM time per launch (several independent batches in flight on separate streams)."""
    check(lib().et_set_tuning_goal(_i({"latency": 0, "throughput": 1}[goal])))


def set_attention_scores_fp32(on):
    """Whether attention must accumulate Q K^T in fp32. The tcgen05 kernel always does: kept for callers that set it."""
    check(lib().et_set_attention_scores_fp32(_i(1 if on else 0)))


def attention_scores_fp32():
    return bool(lib().et_attention_scores_fp32())


class TileWeight:
    """Packed, device-resident 16x16 tile-pruned weight (the reference's Linear_tile)."""

    def __init__(self, in_feat, out_feat, size, data, row_ptr, row_offset, bias=None, is_gelu=False):
        self.in_feat, self.out_feat, self.size, self.is_gelu = in_feat, out_feat, size, is_gelu
        data = np.ascontiguousarray(data, dtype=np.float16)
        row_ptr = np.ascontiguousarray(row_ptr, dtype=np.int32)
        row_offset = np.ascontiguousarray(row_offset, dtype=np.int32)
        bias = None if bias is None else np.ascontiguousarray(bias, dtype=np.float16)
        self.ntile = int(row_offset.shape[0])
        self._h = ctypes.c_void_p(0)
        check(lib().et_tile_weight_create(ctypes.byref(self._h), _i(in_feat), _i(out_feat), _i(size),
                                          _i(self.ntile), ptr(data), ptr(row_ptr), ptr(row_offset),
                                          ptr(bias)))

    def run(self, out, x, gelu=None, stream=None):
        tokens = x.shape[0]
        g = self.is_gelu if gelu is None else gelu
        rc = (_entries or _lib()).et_tile_linear(self._h, _a(out), _a(x), tokens, 1 if g else 0, raw_stream(stream))
        if rc:
            check(rc)
        return out

    def check(self):
        code = _i(0)
        check(lib().et_tile_weight_check(self._h, ctypes.byref(code)))

    def info(self):
        arr = (ctypes.c_int * 6)()
        check(lib().et_tile_weight_info(self._h, arr))
        return dict(zip(["nb", "n_chunks", "k_chunks", "stages", "stage_bytes", "packed_bytes"], arr))

    def close(self):
        if self._h:
            lib().et_tile_weight_destroy(self._h)
            self._h = ctypes.c_void_p(0)

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def tile_spmm_bias(Y, X, row_ptr, row_offset, data, bias, K=None, gelu=False, stream=None):
    """Launcher-level entry with device-resident tile arrays (packed form cached by address)."""
    M, N = Y.shape
    K = X.shape[1] if K is None else K
    rc = (_entries or _lib()).et_tile_spmm_bias(_a(Y), _a(X), _a(row_ptr), _a(row_offset), _a(data), M, N, K, _a(bias),
                                                1 if gelu else 0, raw_stream(stream))
    if rc:
        check(rc)
    return Y


def tile_spmm_cache_clear():
    check(lib().et_tile_spmm_cache_clear())


# ---------------------------------------------------------------------------------- row-pruned linear
class RowWeight:
    """Row-pruned linear (the reference's Linear_row): only `row_id` output features are kept."""

    def __init__(self, in_feat, out_feat, size, weight, row_id, bias, nhead):
        weight = np.ascontiguousarray(weight, dtype=np.float16)
        row_id = np.ascontiguousarray(row_id, dtype=np.int32)
        bias = None if bias is None else np.ascontiguousarray(bias, dtype=np.float16)
        self.in_feat, self.out_feat, self.size, self.nhead = in_feat, out_feat, size, nhead
        self._h = ctypes.c_void_p(0)
        check(lib().et_row_weight_create(ctypes.byref(self._h), _i(in_feat), _i(out_feat), _i(size),
                                         ptr(weight), ptr(row_id), _i(len(row_id)), ptr(bias), _i(nhead)))
        nrow, n = _i(0), _i(0)
        rid, hp = ctypes.c_void_p(0), ctypes.c_void_p(0)
        hph = (ctypes.c_int * (nhead + 1))()
        check(lib().et_row_weight_meta(self._h, ctypes.byref(nrow), ctypes.byref(n), ctypes.byref(rid),
                                       ctypes.byref(hp), hph))
        self.nrow, self.row_id_size = nrow.value, n.value
        self.row_id_dev, self.head_ptr_dev = rid, hp          # device addresses (c_void_p)
        self.head_ptr = np.array(list(hph), dtype=np.int32)

    def run(self, out, x, stream=None):
        rc = (_entries or _lib()).et_row_linear(self._h, _a(out), _a(x), x.shape[0], raw_stream(stream))
        if rc:
            check(rc)
        return out

    def close(self):
        if self._h:
            lib().et_row_weight_destroy(self._h)
            self._h = ctypes.c_void_p(0)

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


# ---------------------------------------------------------------------------------- attention
def attention_otf(out, Q, K, V, mask, seq_len, d_model, nhead, stream=None):
    rc = (_entries or _lib()).et_attention_otf(_a(out), _a(Q), _a(K), _a(V), _a(mask), seq_len, d_model, nhead, raw_stream(stream))
    if rc:
        check(rc)
    return out


def attention_prune(out, Q, K, V, v_col_id, v_head_ptr, nnz_col_v, mask, seq_len, d_model, nhead, stream=None):
    rc = (_entries or _lib()).et_attention_prune(_a(out), _a(Q), _a(K), _a(V), _a(v_col_id), _a(v_head_ptr), nnz_col_v, _a(mask),
                                                 seq_len, d_model, nhead, raw_stream(stream))
    if rc:
        check(rc)
    return out


def qk_scores(QK, Q, K, seq_len, d_model, nhead, stream=None):
    rc = (_entries or _lib()).et_qk_scores(_a(QK), _a(Q), _a(K), seq_len, d_model, nhead, raw_stream(stream))
    if rc:
        check(rc)
    return QK


def attention_sharedqk(out, QK, V, mask, seq_len, d_model, nhead, stream=None):
    rc = (_entries or _lib()).et_attention_sharedqk(_a(out), _a(QK), _a(V), _a(mask), seq_len, d_model, nhead, raw_stream(stream))
    if rc:
        check(rc)
    return out


def attention_static_scores(out, Q, K, V, mask, seq_len, d_model, nhead, stream=None):
    """et_attention_otf's result through the library's built-in score buffer: allocates nothing."""
    rc = (_entries or _lib()).et_attention_static_scores(_a(out), _a(Q), _a(K), _a(V), _a(mask), seq_len, d_model, nhead,
                                                         raw_stream(stream))
    if rc:
        check(rc)
    return out


def attention_check():
    """Raises EtError (ET_ERR_DEVICE_TIMEOUT) if a bounded wait of the tensor-core attention kernel gave up on the
    current device since the last check; synchronises."""
    code = _i(0)
    check(lib().et_attention_check(ctypes.byref(code)))


def attention_batch(out, Q, K, V, d_model, nhead, cu_seqlens=None, valid_lens=None, batch=1, uniform_len=0,
                    max_seq_len=0, total_tokens=None, mask=None, mask_ld=0, qk_pitch=None, v_pitch=None, qk_head_ptr=None,
                    v_col_id=None, v_head_ptr=None, stream=None):
    total = Q.shape[0] if total_tokens is None else total_tokens
    rc = (_entries or _lib()).et_attention_batch(
        _a(out), _a(Q), _a(K), _a(V), Q.shape[1] if qk_pitch is None else qk_pitch, V.shape[1] if v_pitch is None else v_pitch,
        _a(qk_head_ptr), _a(v_col_id), _a(v_head_ptr), _a(mask), mask_ld, _a(cu_seqlens), _a(valid_lens), batch, uniform_len,
        max_seq_len, total, d_model, nhead, raw_stream(stream))
    if rc:
        check(rc)
    return out


# ---------------------------------------------------------------------------------- positions, adapters, rules on scores
# et_rotary_axes_args, et_adapter_add_args and et_attention_rules_args as they lie in memory
_rotary_args, _adapter_args, _rules_args = struct.Struct("@8P11i0P").pack, struct.Struct("@7P5i0P").pack, struct.Struct("@8PNPffPPiiiPPP12i").pack
_kept = None


def _torch_kept():
    """(lookup of the current device, of a device's current stream, float16, int32, float32): fetched once, these calls are short."""
    global _kept
    if _kept is None:
        import torch
        raw_stream()   # initialises CUDA
        try:
            _kept = (torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream, torch.float16, torch.int32, torch.float32)
        except AttributeError:
            _kept = (torch.cuda.current_device, lambda device: raw_stream(), torch.float16, torch.int32, torch.float32)
    return _kept


def _refuse(name, t, dtype, dims, device):
    raise ValueError(f"{name}: a {dims}-dimensional {dtype} tensor on the current CUDA device ({device}) expected, the elements of a row neighbours, rows "
                     f"one behind the other; not {t.dtype} {tuple(t.shape)} with strides {t.stride()} on {t.device}")


def _array(name, t, dtype, device, n):
    """Address of a contiguous array of n elements."""
    if t.dtype is dtype and t.get_device() == device and t.dim() == 1 and t.is_contiguous():
        if t.numel() == n:
            return t.data_ptr()
        raise ValueError(f"{name}: {n} elements expected, not {t.numel()}")
    _refuse(name, t, dtype, 1, device)


def _matrix(name, t, dtype, device):
    """(rows, columns) of a contiguous matrix."""
    if t.dtype is not dtype or t.get_device() != device or t.dim() != 2 or not t.is_contiguous():
        _refuse(name, t, dtype, 2, device)
    return t.shape


def rotary_axes(q_out, k_out, q, k, positions, inv_freq, axis, head_dim, interleaved=False, stream=None):
    """Rotary positions over several axes on the heads of q [tokens, heads * head_dim] and k (either may be None); rows may be slices of
    wider ones, q_out may be q and k_out may be k. positions [tokens, axes] int32; inv_freq float32 and axis int32, one for each
    pair of features (twice as many features are turned). Returns (q_out, k_out)."""
    current, stream_of, f16, i32, f32 = _kept or _torch_kept()
    device = current()
    tokens, axes = positions.shape
    pairs = inv_freq.numel()
    if (positions.dtype is not i32 or axis.dtype is not i32 or inv_freq.dtype is not f32 or positions.get_device() != device or axis.get_device() != device
            or inv_freq.get_device() != device or axis.numel() != pairs or not positions.is_contiguous() or not axis.is_contiguous() or not inv_freq.is_contiguous()):
        raise ValueError(f"positions int32 [tokens, axes], inv_freq float32 and axis int32 [pairs], contiguous, on the current CUDA device ({device}) expected, not "
                         + ", ".join(f"{t.dtype} {tuple(t.shape)} {t.stride()} on {t.device}" for t in (positions, inv_freq, axis)))
    nq = nk = q_pitch = k_pitch = q_out_pitch = k_out_pitch = 0
    q_at = k_at = q_out_at = k_out_at = 0
    if q is not None:
        q_at, q_out_at, q_pitch, q_out_pitch, nq = _turned("q", q, q_out, tokens, head_dim, f16, device)
    if k is not None:
        k_at, k_out_at, k_pitch, k_out_pitch, nk = _turned("k", k, k_out, tokens, head_dim, f16, device)
    rc = (_entries or _lib()).et_rotary_axes_by(_rotary_args(
        q_out_at, q_at, k_out_at, k_at, positions.data_ptr(), inv_freq.data_ptr(), axis.data_ptr(), stream_of(device) if stream is None else stream.cuda_stream,
        q_out_pitch, q_pitch, nq, k_out_pitch, k_pitch, nk, head_dim, 2 * pairs, axes, 1 if interleaved else 0, tokens))
    if rc:
        check(rc)
    return q_out, k_out


def _turned(name, x, out, tokens, head_dim, f16, device):
    """(addresses and pitches of x and of its result, heads)."""
    rows, width = shape = x.shape
    pitch, step = x.stride()
    out_pitch, out_step = out.stride()
    if (x.dtype is f16 and out.dtype is f16 and x.get_device() == device and out.get_device() == device and rows == tokens and head_dim > 0 and width % head_dim == 0 and out.shape == shape
            and step == 1 and out_step == 1):
        return (x.data_ptr(), out.data_ptr(), pitch, out_pitch, width // head_dim) if rows > 1 else (x.data_ptr(), out.data_ptr(), width, width, width // head_dim)
    raise ValueError(f"{name}: {tokens} rows of whole float16 heads of {head_dim} on the current CUDA device ({device}), neighbouring elements, and the result alike expected, "
                     f"not {x.dtype} {tuple(x.shape)} on {x.device} and {out.dtype} {tuple(out.shape)} on {out.device}")


class AdapterBank:
    """Low-rank adapters of one projection, for sequences that each have one of them (or none): out = base + scale B (A x)."""

    def __init__(self, in_feat, out_feat, max_rank, slots):
        self.in_feat, self.out_feat, self.max_rank, self.slots = in_feat, out_feat, max_rank, slots
        self._h = ctypes.c_void_p(0)
        check(lib().et_adapter_bank_create(ctypes.byref(self._h), _i(in_feat), _i(out_feat), _i(max_rank), _i(slots)))

    def set(self, slot, A, B, scale=1.0):
        """Fills a slot: A [rank, in_feat], B [out_feat, rank], host arrays. Synchronises the device."""
        A, B = np.ascontiguousarray(A, dtype=np.float16), np.ascontiguousarray(B, dtype=np.float16)
        if A.ndim != 2 or B.ndim != 2 or A.shape[1] != self.in_feat or B.shape[0] != self.out_feat or A.shape[0] != B.shape[1]:
            raise ValueError(f"A [rank, {self.in_feat}] and B [{self.out_feat}, rank] expected, not {A.shape} and {B.shape}")
        check(lib().et_adapter_bank_set(self._h, _i(slot), _i(A.shape[0]), ptr(A), ptr(B), ctypes.c_float(scale)))

    def clear(self, slot):
        """Empties a slot: its sequences get base. Synchronises the device."""
        check(lib().et_adapter_bank_set(self._h, _i(slot), _i(0), None, None, ctypes.c_float(0.0)))

    def add(self, out, base, x, adapter_ids, cu_seqlens=None, stream=None):
        """out = base + the adapter's product for each sequence's tokens. adapter_ids int32 [batch] (-1: none), cu_seqlens int32 [batch + 1]
        or None (one token to a sequence). out may be base; rows may be slices of wider ones."""
        current, stream_of, f16, i32, _ = _kept or _torch_kept()
        device = current()
        rows, width = x.shape
        shape = base.shape
        x_pitch, x_step = x.stride()
        base_pitch, base_step = base.stride()
        out_pitch, out_step = out.stride()
        if (x.dtype is not f16 or base.dtype is not f16 or out.dtype is not f16 or x.get_device() != device or base.get_device() != device or out.get_device() != device
                or width != self.in_feat or shape != out.shape or shape != (rows, self.out_feat) or x_step != 1 or base_step != 1 or out_step != 1):
            raise ValueError(f"float16 x [{rows}, {self.in_feat}], base and out [{rows}, {self.out_feat}] on the current CUDA device ({device}) with neighbouring elements expected, not "
                             f"{x.dtype} {tuple(x.shape)} on {x.device}, {base.dtype} {tuple(base.shape)} on {base.device}, {out.dtype} {tuple(out.shape)} on {out.device}")
        if rows <= 1:
            x_pitch, base_pitch, out_pitch = width, self.out_feat, self.out_feat
        batch = adapter_ids.numel()
        rc = (_entries or _lib()).et_adapter_add_by(_adapter_args(
            self._h.value or 0, out.data_ptr(), base.data_ptr(), x.data_ptr(), 0 if cu_seqlens is None else _array("cu_seqlens", cu_seqlens, i32, device, batch + 1),
            _array("adapter_ids", adapter_ids, i32, device, batch), stream_of(device) if stream is None else stream.cuda_stream, out_pitch, base_pitch, x_pitch, batch, rows))
        if rc:
            check(rc)
        return out

    def close(self):
        if self._h:
            lib().et_adapter_bank_destroy(self._h)
            self._h = ctypes.c_void_p(0)

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def attention_rules_scratch_size(batch, max_k_len):
    """Bytes of scratch that attention_rules needs with documents."""
    f = lib().et_attention_rules_scratch_size
    f.restype = ctypes.c_size_t
    return int(f(_i(batch), _i(max_k_len)))


def attention_rules(out, Q, K, V, head_dim, cu_seqlens=None, k_start=None, k_lens=None, batch=1, max_q_len=0, max_k_len=0, scale=0.0, cap=0.0, slopes=None,
                    distance_bias=None, window=(-1, -1), prefix_lens=None, q_docs=None, k_docs=None, scratch=None, stream=None):
    """Attention with rules on its scores (capped, biased by distance, seen through windows, prefixes and documents) over packed sequences, or of
    tokens over keys kept from before (k_start, k_lens). Q and out [tokens, heads * head_dim], K and V [rows, kv_heads * head_dim], rows may be
    slices of wider ones; see et_attention_rules for each argument. max_q_len, max_k_len: 0 takes the number of rows."""
    current, stream_of, f16, i32, f32 = _kept or _torch_kept()
    device = current()
    q_shape, k_shape = Q.shape, K.shape
    tokens, width = q_shape
    k_rows, kv_width = k_shape
    q_pitch, q_step = Q.stride()
    k_pitch, k_step = K.stride()
    v_pitch, v_step = V.stride()
    out_pitch, out_step = out.stride()
    if (Q.dtype is not f16 or K.dtype is not f16 or V.dtype is not f16 or out.dtype is not f16 or Q.get_device() != device or K.get_device() != device
            or V.get_device() != device or out.get_device() != device or out.shape != q_shape or V.shape != k_shape or head_dim < 1 or width % head_dim or kv_width % head_dim
            or not kv_width or not width or (q_step != 1 or out_step != 1) and width > 1 or (k_step != 1 or v_step != 1) and kv_width > 1):
        raise ValueError(f"float16 rows of whole heads of {head_dim} on the current CUDA device ({device}) with neighbouring elements, out like Q and V like K expected, not "
                         + ", ".join(f"{n} {t.dtype} {tuple(t.shape)} {t.stride()} on {t.device}" for n, t in (("Q", Q), ("out", out), ("K", K), ("V", V))))
    if tokens <= 1:
        q_pitch = out_pitch = width
    if k_rows <= 1:
        k_pitch = v_pitch = kv_width
    nhead, nhead_kv = width // head_dim, kv_width // head_dim
    reach = table = 0
    if distance_bias is not None:
        heads, places = _matrix("distance_bias", distance_bias, f16, device)
        if heads != nhead or places % 2 == 0:
            raise ValueError("distance_bias: [heads, 2 reach + 1] expected")
        reach, table = places // 2, distance_bias.data_ptr()
    scratch_bytes = 0
    if scratch is not None:
        scratch_bytes = scratch.numel() * scratch.element_size()
        if scratch.get_device() != device or not scratch.is_contiguous():
            raise ValueError("scratch must be contiguous, on the current CUDA device")
    rc = (_entries or _lib()).et_attention_rules_by(_rules_args(
        out.data_ptr(), Q.data_ptr(), K.data_ptr(), V.data_ptr(), 0 if cu_seqlens is None else _array("cu_seqlens", cu_seqlens, i32, device, batch + 1),
        0 if k_start is None else _array("k_start", k_start, i32, device, batch), 0 if k_lens is None else _array("k_lens", k_lens, i32, device, batch),
        0 if scratch is None else scratch.data_ptr(), scratch_bytes, stream_of(device) if stream is None else stream.cuda_stream,
        scale, cap, 0 if slopes is None else _array("slopes", slopes, f32, device, nhead), table, reach, window[0], window[1],
        0 if prefix_lens is None else _array("prefix_lens", prefix_lens, i32, device, batch),
        0 if q_docs is None else _array("q_docs", q_docs, i32, device, tokens), 0 if k_docs is None else _array("k_docs", k_docs, i32, device, k_rows),
        out_pitch, q_pitch, k_pitch, v_pitch, nhead, nhead_kv, head_dim, batch, tokens, k_rows, max_q_len or tokens, max_k_len or k_rows))
    if rc:
        check(rc)
    return out


# ---------------------------------------------------------------------------------- layers in 8 bits
# et_skip_rmsnorm_args, et_quantise_rows_args, et_fp8_linear_args, et_kv_cache_args and et_attention_tree_args as they lie in memory
_rmsnorm_args, _quantise_args, _fp8_args, _cache_args, _tree_args = (struct.Struct(f).pack for f in ("@7P6if0P", "@4P4i0P", "@5P4i0P", "@6P7i0P", "@9P12if0P"))
_kept8 = None
_fast = None


def _load_fast():
    """The module that checks and packs the arguments of these calls in C++ (binding.cpp), or False where it has not been built: then, and where it does not take what it is given, the
    checks below do it, which name what is wrong."""
    global _fast
    if _fast is None:
        path = binding_path()   # (none of another Python's or torch's)
        if path is None or not os.path.exists(path):
            _fast = False
            return _fast
        try:
            import torch  # noqa: F401  (its libraries are loaded first)
            spec = importlib.util.spec_from_file_location(__package__ + "._binding", path)
            _binding = importlib.util.module_from_spec(spec)
            spec.loader.exec_module(_binding)
        except ImportError:
            _fast = False
            return _fast
        _binding.bind(*(ctypes.cast(lib()[name], ctypes.c_void_p).value for name in (
            "et_skip_rmsnorm", "et_quantise_rows", "et_fp8_linear", "et_kv_cache_write", "et_kv_cache_read", "et_attention_tree")))
        _fast = _binding
    return _fast


def _torch_kept8():
    """(float16, float32, (float16,), (e4m3, uint8), int8, int64, lookups of the current device and of its stream)."""
    global _kept8
    if _kept8 is None:
        import torch
        current, stream_of, f16, _, f32 = _torch_kept()
        _kept8 = (f16, f32, (f16,), (torch.float8_e4m3fn, torch.uint8), torch.int8, torch.int64, current, stream_of)
    return _kept8


def _rows(name, t, dtypes, shape, device):
    """(address, pitch) of rows with neighbouring elements that may be slices of wider ones."""
    if t.dtype in dtypes and t.get_device() == device and t.shape == shape:
        if t.is_contiguous():
            return t.data_ptr(), shape[1]
        pitch, step = t.stride()
        if step == 1 or shape[1] == 1:
            return t.data_ptr(), pitch if shape[0] > 1 else shape[1]
    raise ValueError(f"{name}: {tuple(shape)} of {' or '.join(str(d) for d in dtypes)} on the current CUDA device ({device}) with neighbouring elements expected, "
                     f"not {t.dtype} {tuple(t.shape)} with strides {t.stride()} on {t.device}")


def _row_scales(scales, rows, width, f32, device):
    if scales.dtype is f32 and scales.get_device() == device and scales.shape == ((width + 127) // 128, rows) and scales.is_contiguous():
        return scales.data_ptr()
    raise ValueError(f"scales: contiguous float32 {((width + 127) // 128, rows)} on the current CUDA device ({device}) expected, not {scales.dtype} {tuple(scales.shape)} on {scales.device}")


def skip_rmsnorm(out, x, skip, gamma, residual=None, scales=None, eps=1e-6, stream=None):
    """h = x + skip (skip may be None), out = h / sqrt(mean(h^2) + eps) * gamma for rows [rows, width] of float16, residual = h where it is given. Without scales
    out is float16; with scales float32 [ceil(width / 128), rows] it is e4m3 (or uint8), a scale for each 128 features of a row. Rows may be slices of wider ones; residual
    (and a float16 out) may be x or skip. Returns out."""
    fast = _fast if _fast is not None else _load_fast()
    if fast:
        rc = fast.skip_rmsnorm(out, x, skip, gamma, residual, scales, eps, None if stream is None else stream.cuda_stream)
        if rc == 0:
            return out
        if rc > 0:
            check(rc)
    f16, f32, f16s, e4m3s, _, _, current, stream_of = _kept8 or _torch_kept8()
    device = current()
    shape = x.shape
    rows, width = shape
    x_at, x_pitch = _rows("x", x, f16s, shape, device)
    skip_at, skip_pitch = (0, 0) if skip is None else _rows("skip", skip, f16s, shape, device)
    residual_at, residual_pitch = (0, 0) if residual is None else _rows("residual", residual, f16s, shape, device)
    if scales is None:
        scales_at = 0
        out_at, out_pitch = _rows("out", out, f16s, shape, device)
    else:
        scales_at = _row_scales(scales, rows, width, f32, device)
        out_at, out_pitch = _rows("out", out, e4m3s, shape, device)
    rc = (_entries or _lib()).et_skip_rmsnorm(_rmsnorm_args(
        out_at, x_at, skip_at, _array("gamma", gamma, f16, device, width), residual_at, scales_at, stream_of(device) if stream is None else stream.cuda_stream,
        out_pitch, x_pitch, skip_pitch, residual_pitch, rows, width, eps))
    if rc:
        check(rc)
    return out


def quantise_rows(out, scales, x, stream=None):
    """Rows of float16 x [rows, width] as e4m3 (or uint8) out with a scale for each 128 features of a row in scales float32 [ceil(width / 128), rows]. Returns (out, scales)."""
    fast = _fast if _fast is not None else _load_fast()
    if fast:
        rc = fast.quantise_rows(out, scales, x, None if stream is None else stream.cuda_stream)
        if rc == 0:
            return out, scales
        if rc > 0:
            check(rc)
    _, f32, f16s, e4m3s, _, _, current, stream_of = _kept8 or _torch_kept8()
    device = current()
    shape = x.shape
    rows, width = shape
    x_at, x_pitch = _rows("x", x, f16s, shape, device)
    out_at, out_pitch = _rows("out", out, e4m3s, shape, device)
    rc = (_entries or _lib()).et_quantise_rows(_quantise_args(
        out_at, _row_scales(scales, rows, width, f32, device), x_at, stream_of(device) if stream is None else stream.cuda_stream, out_pitch, x_pitch, rows, width))
    if rc:
        check(rc)
    return out, scales


class Fp8Weight:
    """Linear with operands in e4m3: codes uint8 [out_feat, in_feat] (the bytes of e4m3) and scales float32 [ceil(out_feat / 128), ceil(in_feat / 128)], host arrays."""

    def __init__(self, in_feat, out_feat, codes, scales, bias=None, is_gelu=False):
        self.in_feat, self.out_feat, self.is_gelu = in_feat, out_feat, is_gelu
        self._h = ctypes.c_void_p(0)
        codes, scales = np.ascontiguousarray(codes), np.ascontiguousarray(scales, dtype=np.float32)
        bias = None if bias is None else np.ascontiguousarray(bias, dtype=np.float16)
        blocks = ((out_feat + 127) // 128, (in_feat + 127) // 128)
        if codes.dtype != np.uint8 or codes.shape != (out_feat, in_feat) or scales.shape != blocks or (bias is not None and bias.shape != (out_feat,)):
            raise ValueError(f"codes uint8 {(out_feat, in_feat)}, scales {blocks} and bias {(out_feat,)} expected, not {codes.dtype} {codes.shape}, {scales.shape}"
                             + ("" if bias is None else f" and {bias.shape}"))
        check(lib().et_fp8_weight_create(ctypes.byref(self._h), _i(in_feat), _i(out_feat), ptr(codes), ptr(scales), ptr(bias)))

    def run(self, out, x, x_scales, gelu=None, stream=None):
        """out [tokens, out_feat] float16 = x . W^T + bias (then tanh-GELU), x [tokens, in_feat] e4m3 (or uint8) with x_scales float32 [ceil(in_feat / 128), tokens]; rows
        may be slices of wider ones."""
        fast = _fast if _fast is not None else _load_fast()
        if fast:
            rc = fast.fp8_linear(self._h.value or 0, self.in_feat, self.out_feat, 1 if (self.is_gelu if gelu is None else gelu) else 0, out, x, x_scales,
                                 None if stream is None else stream.cuda_stream)
            if rc == 0:
                return out
            if rc > 0:
                check(rc)
        _, f32, f16s, e4m3s, _, _, current, stream_of = _kept8 or _torch_kept8()
        device = current()
        tokens = x.shape[0]
        x_at, x_pitch = _rows("x", x, e4m3s, (tokens, self.in_feat), device)
        out_at, out_pitch = _rows("out", out, f16s, (tokens, self.out_feat), device)
        rc = (_entries or _lib()).et_fp8_linear(_fp8_args(
            self._h.value or 0, out_at, x_at, _row_scales(x_scales, tokens, self.in_feat, f32, device), stream_of(device) if stream is None else stream.cuda_stream,
            out_pitch, x_pitch, tokens, 1 if (self.is_gelu if gelu is None else gelu) else 0))
        if rc:
            check(rc)
        return out

    def check(self):
        """Raises EtError (ET_ERR_DEVICE_TIMEOUT) if a device-side wait of one of the weight's launches gave up."""
        code = _i(0)
        check(lib().et_fp8_weight_check(self._h, ctypes.byref(code)))

    def close(self):
        if self._h:
            lib().et_fp8_weight_destroy(self._h)
            self._h = ctypes.c_void_p(0)

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def _cache(codes, scales, i8, f32, device):
    """(pages, heads, rows of a page, head_dim) of a cache."""
    shape = codes.shape
    if (codes.dtype is i8 and scales.dtype is f32 and codes.get_device() == device and scales.get_device() == device and len(shape) == 5 and shape[1] == 2
            and scales.shape == shape[:4] and codes.is_contiguous() and scales.is_contiguous()):
        pages, _, heads, page, head_dim = shape
        return pages, heads, page, head_dim
    raise ValueError(f"contiguous int8 codes [pages, 2, heads, page, head_dim] and float32 scales [pages, 2, heads, page] on the current CUDA device ({device}) expected, "
                     f"not {codes.dtype} {tuple(codes.shape)} on {codes.device} and {scales.dtype} {tuple(scales.shape)} on {scales.device}")


def _cache_call(write, codes, scales, k, v, slots, stream):
    fast = _fast if _fast is not None else _load_fast()
    if fast:
        rc = fast.kv_cache(write, codes, scales, k, v, slots, None if stream is None else stream.cuda_stream)
        if rc == 0:
            return
        if rc > 0:
            check(rc)
    entries = _entries or _lib()
    entry = entries.et_kv_cache_write if write else entries.et_kv_cache_read
    f16, f32, f16s, _, i8, _, current, stream_of = _kept8 or _torch_kept8()
    device = current()
    pages, heads, page, head_dim = _cache(codes, scales, i8, f32, device)
    shape = (k.shape[0], heads * head_dim)
    k_at, k_pitch = _rows("k", k, f16s, shape, device)
    v_at, v_pitch = _rows("v", v, f16s, shape, device)
    rc = entry(_cache_args(codes.data_ptr(), scales.data_ptr(), k_at, v_at, _array("slots", slots, (_kept or _torch_kept())[3], device, shape[0]),
                           stream_of(device) if stream is None else stream.cuda_stream, k_pitch, v_pitch, shape[0], pages, heads, page, head_dim))
    if rc:
        check(rc)


def kv_cache_write(codes, scales, k, v, slots, stream=None):
    """Quantises rows of k and v [tokens, heads * head_dim] float16 into a cache: codes int8 [pages, 2, heads, page, head_dim], scales float32 [pages, 2, heads, page]. Row t
    goes to slots[t] (int32: page number * page + row; below 0: nowhere); slots differ. Returns (codes, scales)."""
    _cache_call(True, codes, scales, k, v, slots, stream)
    return codes, scales


def kv_cache_read(k, v, codes, scales, slots, stream=None):
    """Rows of a cache as float16: k and v [tokens, heads * head_dim], row t from slots[t] (below 0: left as it is). Returns (k, v)."""
    _cache_call(False, codes, scales, k, v, slots, stream)
    return k, v


def attention_tree(out, q, codes, scales, table, k_lens, tree=None, cu_seqlens=None, max_q_len=0, max_k_len=0, scale=0.0, stream=None):
    """Attention of drafted tokens q [tokens, heads * head_dim] float16 over a cache (as kv_cache_write leaves it): table int32 [batch, pages of the longest], k_lens int32 [batch]
    keys, the drafted tokens' own the last of them. A token sees the keys before those and the drafted ones whose bit is set in tree int64 [tokens] (None: those up to
    itself). cu_seqlens int32 [batch + 1], or None: max_q_len tokens each. max_q_len (0: 1 without cu_seqlens, 64 with it) and max_k_len (0: all that the table has)."""
    fast = _fast if _fast is not None else _load_fast()
    if fast:
        rc = fast.attention_tree(out, q, codes, scales, table, k_lens, tree, cu_seqlens, max_q_len, max_k_len, scale, None if stream is None else stream.cuda_stream)
        if rc == 0:
            return out
        if rc > 0:
            check(rc)
    f16, f32, f16s, _, i8, i64, current, stream_of = _kept8 or _torch_kept8()
    i32 = (_kept or _torch_kept())[3]
    device = current()
    pages, heads, page, head_dim = _cache(codes, scales, i8, f32, device)
    shape = q.shape
    tokens, width = shape
    if not head_dim or not heads or width % head_dim:
        raise ValueError(f"q: whole heads of {head_dim} expected, not rows of {width}")
    q_at, q_pitch = _rows("q", q, f16s, shape, device)
    out_at, out_pitch = _rows("out", out, f16s, shape, device)
    batch, most = _matrix("table", table, i32, device)
    rc = (_entries or _lib()).et_attention_tree(_tree_args(
        out_at, q_at, codes.data_ptr(), scales.data_ptr(), table.data_ptr(), _array("k_lens", k_lens, i32, device, batch),
        0 if cu_seqlens is None else _array("cu_seqlens", cu_seqlens, i32, device, batch + 1), 0 if tree is None else _array("tree", tree, i64, device, tokens),
        stream_of(device) if stream is None else stream.cuda_stream, out_pitch, q_pitch, width // head_dim, heads, head_dim, batch, tokens,
        max_q_len or (1 if cu_seqlens is None else 64), max_k_len or min(most * page, 0x7ff00000), pages, page, most, scale))
    if rc:
        check(rc)
    return out


# ---------------------------------------------------------------------------------- format generators
def gen_sparse_tile_mat(nrow, ncol, sparsity, seed, bernoulli=False):
    cap = (nrow // 16) * (ncol // 16)
    row_ptr = np.zeros(nrow // 16 + 1, dtype=np.int32)
    row_offset = np.zeros(max(cap, 1), dtype=np.int32)
    n = _i(0)
    check(lib().et_gen_sparse_tile_mat(_i(nrow), _i(ncol), ctypes.c_float(sparsity), ctypes.c_uint64(seed),
                                       _i(1 if bernoulli else 0), ptr(row_ptr), ptr(row_offset), _i(cap),
                                       ctypes.byref(n)))
    return row_ptr, row_offset[:n.value].copy()


def gen_sparse_row_mat(nrow, sparsity, seed, nhead=0):
    row_id = np.zeros(nrow, dtype=np.int32)
    n = _i(0)
    check(lib().et_gen_sparse_row_mat(_i(nrow), ctypes.c_float(sparsity), ctypes.c_uint64(seed), _i(nhead),
                                      ptr(row_id), _i(nrow), ctypes.byref(n)))
    return row_id[:n.value].copy()


def build_head_ptr(row_id, nhead, out_feat):
    row_id = np.ascontiguousarray(row_id, dtype=np.int32)
    hp = np.zeros(nhead + 1, dtype=np.int32)
    check(lib().et_build_head_ptr(ptr(row_id), _i(len(row_id)), _i(nhead), _i(out_feat), ptr(hp)))
    return hp


# ---------------------------------------------------------------------------------- encoder layers
KIND_TILE, KIND_PRUNE, KIND_LENGTH, KIND_PRUNE_QKV = 0, 1, 2, 3


def encoder_buffer_size(kind, d_model, seq_len, nheads):
    f = lib().et_encoder_buffer_size
    f.restype = ctypes.c_size_t
    return int(f(_i(kind), _i(d_model), _i(seq_len), _i(nheads)))


def encoder_batch_buffer_size(kind, d_model, total_tokens, batch, max_len, nheads):
    f = lib().et_encoder_batch_buffer_size
    f.restype = ctypes.c_size_t
    return int(f(_i(kind), _i(d_model), _i(total_tokens), _i(batch), _i(max_len), _i(nheads)))


class Encoder:
    """One encoder layer (Encoder_tile / Encoder_prune / Encoder_length of the reference).

    q, k, v, o, mlp1, mlp2 are TileWeight (or RowWeight where the kind prunes rows); the encoder takes
    ownership of them. ln = (gamma1, beta1, gamma2, beta2) host arrays; mask host [seq_len, seq_len] or None;
    buffer: device scratch tensor for run() (None if only run_batch is used)."""

    def __init__(self, kind, d_model, seq_len, nheads, buffer, q, k, v, o, mlp1, mlp2, ln, mask=None):
        self.kind, self.d_model, self.seq_len, self.nheads = kind, d_model, seq_len, nheads
        self._buffer = buffer
        self._lin = (q, k, v, o, mlp1, mlp2)
        ln = [np.ascontiguousarray(a, dtype=np.float16) for a in ln]
        mask = None if mask is None else np.ascontiguousarray(mask, dtype=np.float16)
        self._h = ctypes.c_void_p(0)
        L = lib()
        common = (ptr(ln[0]), ptr(ln[1]), ptr(ln[2]), ptr(ln[3]), ptr(mask))
        if kind in (KIND_TILE, KIND_LENGTH):
            check(L.et_encoder_tile_create(ctypes.byref(self._h), _i(kind), _i(d_model), _i(seq_len), _i(nheads),
                                           ptr(buffer), q._h, k._h, v._h, o._h, mlp1._h, mlp2._h, *common))
        elif kind == KIND_PRUNE:
            check(L.et_encoder_prune_create(ctypes.byref(self._h), _i(d_model), _i(seq_len), _i(nheads),
                                            ptr(buffer), q._h, k._h, v._h, o._h, mlp1._h, mlp2._h, *common))
        elif kind == KIND_PRUNE_QKV:
            check(L.et_encoder_prune_qkv_create(ctypes.byref(self._h), _i(d_model), _i(seq_len), _i(nheads),
                                                ptr(buffer), q._h, k._h, v._h, o._h, mlp1._h, mlp2._h, *common))
        else:
            raise ValueError("unknown encoder kind")

    def run(self, out, x, stream=None):
        rc = (_entries or _lib()).et_encoder_run(self._h, _a(out), _a(x), raw_stream(stream))
        if rc:
            check(rc)
        return out

    def run_batch(self, out, x, seq_lens, scratch, valid_lens=None, stream=None):
        lens, n, keep = _ints(seq_lens)
        valid, _, keep_valid = (None, 0, None) if valid_lens is None else _ints(valid_lens)
        rc = (_entries or _lib()).et_encoder_run_batch(self._h, _a(out), _a(x), lens, valid, n, _a(scratch),
                                                       scratch.numel() * scratch.element_size(), raw_stream(stream))
        if rc:
            check(rc)
        return out

    def check(self):
        """Raises EtError (ET_ERR_DEVICE_TIMEOUT) if a device-side wait of one of the layer's kernels gave up."""
        code = _i(0)
        check(lib().et_encoder_check(self._h, ctypes.byref(code)))

    def set_graph_replay(self, on):
        check(lib().et_encoder_set_graph_replay(self._h, _i(1 if on else 0)))

    def set_materialize_scores(self, on):
        check(lib().et_encoder_set_materialize_scores(self._h, _i(1 if on else 0)))

    def close(self):
        if self._h:
            lib().et_encoder_destroy(self._h)
            self._h = ctypes.c_void_p(0)

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class Model:
    """A stack of encoder layers run back to back on packed tokens (et_model_* of the C ABI). Takes ownership of
    the layers of the `Encoder` objects given (they become empty shells). Scratch is owned by the model."""

    def __init__(self, encoders):
        self._encoders = list(encoders)
        arr = (ctypes.c_void_p * len(self._encoders))(*[e._h for e in self._encoders])
        self._h = ctypes.c_void_p(0)
        check(lib().et_model_create(ctypes.byref(self._h), arr, _i(len(self._encoders))))

    @property
    def num_layers(self):
        return int(lib().et_model_num_layers(self._h))

    def reserve(self, total_tokens, batch, max_len):
        check(lib().et_model_reserve(self._h, _i(total_tokens), _i(batch), _i(max_len)))

    def run_batch(self, out, x, seq_lens, valid_lens=None, stream=None):
        lens, n, keep = _ints(seq_lens)
        valid, _, keep_valid = (None, 0, None) if valid_lens is None else _ints(valid_lens)
        rc = (_entries or _lib()).et_model_run_batch(self._h, _a(out), _a(x), lens, valid, n, raw_stream(stream))
        if rc:
            check(rc)
        return out

    def set_layernorm_fusion(self, on):
        check(lib().et_model_set_layernorm_fusion(self._h, _i(1 if on else 0)))

    @property
    def layernorm_fused(self):
        return bool(lib().et_model_layernorm_fused(self._h))

    def check(self):
        """Raises EtError (ET_ERR_DEVICE_TIMEOUT) if a device-side wait of one of the stack's kernels gave up."""
        code = _i(0)
        check(lib().et_model_check(self._h, ctypes.byref(code)))

    def set_graph_replay(self, on):
        check(lib().et_model_set_graph_replay(self._h, _i(1 if on else 0)))

    def close(self):
        if self._h:
            lib().et_model_destroy(self._h)
            self._h = ctypes.c_void_p(0)

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


# ---------------------------------------------------------------------------------- real-weight ingestion
def prune_dense_to_tiles(weight, sparsity):
    """Dense fp16 [out_feat, in_feat] -> (row_ptr, row_offset, data[ntile, 256]) keeping the tiles of largest norm."""
    w = np.ascontiguousarray(weight, dtype=np.float16)
    out_feat, in_feat = w.shape
    cap = (out_feat // 16) * (in_feat // 16)
    row_ptr = np.zeros(out_feat // 16 + 1, dtype=np.int32)
    row_offset = np.zeros(max(cap, 1), dtype=np.int32)
    data = np.zeros((max(cap, 1), 256), dtype=np.float16)
    n = _i(0)
    check(lib().et_prune_dense_to_tiles(ptr(w), _i(out_feat), _i(in_feat), ctypes.c_float(sparsity), ptr(row_ptr),
                                        ptr(row_offset), ptr(data), _i(cap), ctypes.byref(n)))
    return row_ptr, row_offset[:n.value].copy(), data[:n.value].copy()


def select_rows_magnitude(weights, nhead, sparsity):
    """Row ids (ascending) kept per head by summed squared norm over the given dense [out_feat, in_feat] weights."""
    ws = [np.ascontiguousarray(w, dtype=np.float16) for w in weights]
    out_feat, in_feat = ws[0].shape
    arr = (ctypes.c_void_p * len(ws))(*[w.ctypes.data for w in ws])
    row_id = np.zeros(out_feat, dtype=np.int32)
    n = _i(0)
    check(lib().et_select_rows_magnitude(arr, _i(len(ws)), _i(out_feat), _i(in_feat), _i(nhead),
                                         ctypes.c_float(sparsity), ptr(row_id), _i(out_feat), ctypes.byref(n)))
    return row_id[:n.value].copy()


def compact_rows(weight, bias, row_id):
    """(weight[ceil16(n), in_feat], bias[ceil16(n)]) of the kept rows, zero padded."""
    w = np.ascontiguousarray(weight, dtype=np.float16)
    b = None if bias is None else np.ascontiguousarray(bias, dtype=np.float16)
    row_id = np.ascontiguousarray(row_id, dtype=np.int32)
    nrow = (len(row_id) + 15) // 16 * 16
    wc = np.zeros((nrow, w.shape[1]), dtype=np.float16)
    bc = np.zeros(nrow, dtype=np.float16)
    check(lib().et_compact_rows(ptr(w), ptr(b), _i(w.shape[0]), _i(w.shape[1]), ptr(row_id), _i(len(row_id)),
                                ptr(wc), ptr(bc)))
    return wc, bc
