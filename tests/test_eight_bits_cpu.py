"""What the operators of a layer in 8 bits refuse, before any CUDA call, what they do with nothing to do, and how their arguments lie in memory."""
import ctypes

import numpy as np
import pytest

from tests.test_operators_cpu import P, lib, numbers, structure  # noqa: F401

I = ctypes.c_int


def with_float(pointers, ints, last):
    fields = structure(pointers, ints)._fields_ + [(last, ctypes.c_float)]
    return type("Args", (ctypes.Structure,), {"_fields_": fields})


NormArgs = with_float("out x skip gamma residual scales stream", "out_pitch x_pitch skip_pitch residual_pitch rows width", "eps")
QuantiseArgs = structure("out scales x stream", "out_pitch x_pitch rows width")
LinearArgs = structure("weight y x x_scales stream", "y_pitch x_pitch tokens gelu")
CacheArgs = structure("codes scales k v slots stream", "k_pitch v_pitch tokens pages heads page head_dim")
TreeArgs = with_float("out q codes scales table k_lens cu_seqlens tree stream", "out_pitch q_pitch nhead nhead_kv head_dim batch q_tokens max_q_len max_k_len pages page table_width", "scale")


@pytest.mark.parametrize("of,packer", [(NormArgs, "_rmsnorm_args"), (QuantiseArgs, "_quantise_args"), (LinearArgs, "_fp8_args"), (CacheArgs, "_cache_args"), (TreeArgs, "_tree_args")])
def test_arguments_are_packed_as_the_structure_lies(of, packer):
    from et_b200 import ops
    values = numbers(of)
    want = of()
    for (name, _), v in zip(of._fields_, values):
        setattr(want, name, v)
    packed = getattr(ops, packer)(*values)
    assert len(packed) == ctypes.sizeof(of) and packed == bytes(want)


@pytest.mark.parametrize("name", ["et_skip_rmsnorm", "et_quantise_rows", "et_kv_cache_write", "et_kv_cache_read", "et_attention_tree", "et_fp8_linear"])
def test_structures_of_arguments_are_needed(lib, name):
    assert getattr(lib, name)(None) == 1 and name.encode() in lib.et_last_error()


def call(lib, name, of, base, change):
    return getattr(lib, name)(ctypes.byref(of(**{**base, **change})))


A, B, C = (ctypes.c_void_p(1 << n) for n in (10, 11, 12))
NORM = dict(out=A, x=P, skip=B, gamma=P, residual=C, scales=None, out_pitch=64, x_pitch=64, skip_pitch=64, residual_pitch=64, rows=0, width=64, eps=1e-6)


@pytest.mark.parametrize("change", [dict(rows=-1), dict(width=0), dict(width=32769), dict(eps=0.0), dict(eps=-1.0), dict(eps=float("nan")), dict(eps=2.0), dict(rows=1, out=None),
                                    dict(rows=1, x=None), dict(rows=1, gamma=None), dict(rows=1, out_pitch=63), dict(rows=1, x_pitch=8), dict(rows=1, skip_pitch=8),
                                    dict(rows=1, residual_pitch=8), dict(rows=1, residual=A), dict(rows=1, residual=P, residual_pitch=128), dict(rows=1, residual=B, residual_pitch=128),
                                    dict(rows=1, out=P, scales=C), dict(rows=1, out=B, out_pitch=128), dict(rows=1, out=B, scales=C)])
def test_norm_refuses(lib, change):
    assert call(lib, "et_skip_rmsnorm", NormArgs, NORM, change) == 1 and b"et_skip_rmsnorm" in lib.et_last_error()


def test_norm_of_nothing(lib):
    assert call(lib, "et_skip_rmsnorm", NormArgs, NORM, {}) == 0


QUANTISE = dict(out=A, scales=B, x=P, out_pitch=64, x_pitch=64, rows=0, width=64)


@pytest.mark.parametrize("change", [dict(rows=-1), dict(width=0), dict(width=32769), dict(rows=1, out=None), dict(rows=1, x=None), dict(rows=1, scales=None), dict(rows=1, out=P),
                                    dict(rows=1, out_pitch=63), dict(rows=1, x_pitch=63)])
def test_quantise_refuses(lib, change):
    assert call(lib, "et_quantise_rows", QuantiseArgs, QUANTISE, change) == 1 and b"et_quantise_rows" in lib.et_last_error()


def test_quantise_nothing(lib):
    assert call(lib, "et_quantise_rows", QuantiseArgs, QUANTISE, {}) == 0


@pytest.mark.parametrize("sizes", [(0, 64), (64, 0), (24, 64), (64, 24), (-16, 64)])
def test_fp8_weight_refuses(lib, sizes):
    w = ctypes.c_void_p(16)
    assert lib.et_fp8_weight_create(ctypes.byref(w), I(sizes[0]), I(sizes[1]), P, P, None) == 1 and not w
    assert lib.et_fp8_weight_create(None, I(64), I(64), P, P, None) == 1


def test_fp8_weight_needs_its_arrays(lib):
    w = ctypes.c_void_p(16)
    assert lib.et_fp8_weight_create(ctypes.byref(w), I(64), I(64), None, P, None) == 1 and lib.et_fp8_weight_create(ctypes.byref(w), I(64), I(64), P, None, None) == 1
    assert lib.et_fp8_weight_destroy(None) == 0 and lib.et_fp8_weight_check(None, ctypes.byref(I(0))) == 1
    assert lib.et_fp8_linear(ctypes.byref(LinearArgs(None, P, P, P, None, 64, 64, 1, 0))) == 1


@pytest.mark.parametrize("codes,scales,bias", [((64, 128), (1, 1), None), ((128, 256), (2, 1), None), ((128, 256), (1, 2), (64,)), ((128 * 256,), (1, 2), None)])
def test_fp8_weight_checks_shapes(lib, codes, scales, bias):
    import et_b200 as et
    with pytest.raises(ValueError):
        et.Fp8Weight(256, 128, np.zeros(codes, np.uint8), np.ones(scales, np.float32), None if bias is None else np.zeros(bias, np.float16))
    with pytest.raises(ValueError):
        et.Fp8Weight(256, 128, np.zeros((128, 256), np.int16), np.ones((1, 2), np.float32))


CACHE = dict(codes=A, scales=P, k=P, v=P, slots=P, k_pitch=128, v_pitch=128, tokens=0, pages=3, heads=2, page=16, head_dim=64)


@pytest.mark.parametrize("name", ["et_kv_cache_write", "et_kv_cache_read"])
@pytest.mark.parametrize("change", [dict(tokens=-1), dict(pages=-1), dict(heads=0), dict(heads=1 << 16), dict(head_dim=0), dict(head_dim=8), dict(head_dim=72), dict(head_dim=272), dict(page=0),
                                    dict(page=8), dict(page=24), dict(pages=1 << 28), dict(tokens=1, codes=None), dict(tokens=1, scales=None), dict(tokens=1, k=None),
                                    dict(tokens=1, slots=None), dict(tokens=1, codes=ctypes.c_void_p(24)), dict(tokens=2, k_pitch=127), dict(tokens=2, v_pitch=0)])
def test_cache_refuses(lib, name, change):
    assert call(lib, name, CacheArgs, CACHE, change) == 1 and name.encode() in lib.et_last_error()


def test_cache_of_nothing(lib):
    assert call(lib, "et_kv_cache_write", CacheArgs, CACHE, {}) == 0 and call(lib, "et_kv_cache_read", CacheArgs, CACHE, dict(pages=0)) == 0


TREE = dict(out=A, q=P, codes=P, scales=P, table=P, k_lens=P, cu_seqlens=None, tree=None, out_pitch=128, q_pitch=128, nhead=2, nhead_kv=1, head_dim=64, batch=1, q_tokens=4, max_q_len=4,
            max_k_len=32, pages=3, page=16, table_width=2, scale=0.0)


@pytest.mark.parametrize("change", [dict(batch=-1), dict(q_tokens=-1), dict(max_q_len=-1), dict(max_k_len=-1), dict(pages=-1), dict(table_width=-1), dict(nhead=0), dict(nhead_kv=0), dict(nhead=3, nhead_kv=2),
                                    dict(head_dim=0), dict(head_dim=72), dict(head_dim=272), dict(page=0), dict(page=20), dict(max_q_len=65), dict(scale=-1.0), dict(scale=float("inf")),
                                    dict(scale=float("nan")), dict(max_k_len=0x7fffffff), dict(out=None), dict(q=None), dict(k_lens=None), dict(codes=None), dict(table=None), dict(q_pitch=127),
                                    dict(out_pitch=120), dict(q_pitch=132), dict(q=ctypes.c_void_p(8)), dict(codes=ctypes.c_void_p(8)), dict(out=P)])
def test_tree_refuses(lib, change):
    assert call(lib, "et_attention_tree", TreeArgs, TREE, change) == 1 and b"et_attention_tree" in lib.et_last_error()


@pytest.mark.parametrize("change", [dict(batch=0), dict(q_tokens=0), dict(max_q_len=0)])
def test_tree_of_nothing(lib, change):
    assert call(lib, "et_attention_tree", TreeArgs, TREE, change) == 0
