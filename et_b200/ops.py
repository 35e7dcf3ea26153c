"""Python-side mirror of the operator and layer interface, one thin wrapper per C-ABI entry.

Tensors are torch CUDA fp16/int32 tensors; host arrays are numpy. Nothing here computes: every
function forwards to `libet_b200.so`.
"""
import array
import ctypes
import struct

import numpy as np

from . import check, lib, ptr, raw_stream

__all__ = [
    "skip_layernorm", "softmax_mask", "TileWeight", "tile_spmm_bias", "tile_spmm_cache_clear",
    "RowWeight", "attention_otf", "attention_prune", "qk_scores", "attention_sharedqk", "attention_batch", "attention_static_scores",
    "gen_sparse_tile_mat", "gen_sparse_row_mat", "build_head_ptr", "Encoder", "encoder_buffer_size",
    "encoder_batch_buffer_size", "KIND_TILE", "KIND_PRUNE", "KIND_LENGTH", "KIND_PRUNE_QKV",
    "Model", "attention_check", "prune_dense_to_tiles", "select_rows_magnitude", "compact_rows", "set_tuning_goal",
    "set_attention_scores_fp32", "attention_scores_fp32", "rotary_axes", "AdapterBank", "attention_rules", "attention_rules_scratch_size",
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
