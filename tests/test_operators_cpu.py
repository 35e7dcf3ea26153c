"""What the operators for positions, adapters and rules on scores refuse, before any CUDA call, and what they do with nothing to do."""
import ctypes
import math

import pytest


@pytest.fixture(scope="module")
def lib():
    import et_b200
    from et_b200 import build
    build.build()
    return et_b200.lib()


P = ctypes.c_void_p(16)   # an address that nothing reads


def structure(pointers, ints, between=()):
    """A structure of pointers, what lies between, and ints, in the order of the header."""
    fields = [(n, ctypes.c_void_p) for n in pointers.split()] + list(between) + [(n, ctypes.c_int) for n in ints.split()]
    return type("Args", (ctypes.Structure,), {"_fields_": fields})


RotaryArgs = structure("q_out q k_out k positions inv_freq axis stream", "q_out_pitch q_pitch nhead_q k_out_pitch k_pitch nhead_k head_dim rot_dim n_axes interleaved tokens")
AdapterArgs = structure("bank out base x cu ids stream", "out_pitch base_pitch x_pitch batch tokens")


class ScoreRules(ctypes.Structure):
    _fields_ = [("scale", ctypes.c_float), ("cap", ctypes.c_float), ("slopes", ctypes.c_void_p), ("distance_bias", ctypes.c_void_p), ("reach", ctypes.c_int),
                ("window_left", ctypes.c_int), ("window_right", ctypes.c_int), ("prefix_lens", ctypes.c_void_p), ("q_docs", ctypes.c_void_p), ("k_docs", ctypes.c_void_p)]


RulesArgs = structure("out Q K V cu k_start k_lens scratch", "out_pitch q_pitch k_pitch v_pitch nhead nhead_kv head_dim batch q_tokens k_rows max_q_len max_k_len",
                      [("scratch_bytes", ctypes.c_size_t), ("stream", ctypes.c_void_p), ("rules", ScoreRules)])


def both(lib, name, args, by):
    """The code of a call, which is that of its form with one structure."""
    rc = getattr(lib, name)(*args)
    assert getattr(lib, name + "_by")(ctypes.byref(by)) == rc
    return rc


def numbers(of):
    """1, 2, ... in every field, and the bytes that the packer gives for them, which are the structure's."""
    flat, values = [], iter(range(1, 100))
    for name, kind in of._fields_:
        flat += list(kind._fields_) if kind is ScoreRules else [(name, kind)]
    return [float(next(values)) if kind is ctypes.c_float else next(values) for _, kind in flat]


@pytest.mark.parametrize("of,packer", [(RotaryArgs, "_rotary_args"), (AdapterArgs, "_adapter_args"), (RulesArgs, "_rules_args")])
def test_arguments_are_packed_as_the_structure_lies(of, packer):
    from et_b200 import ops
    values = numbers(of)
    packed = getattr(ops, packer)(*values)
    left, want = iter(values), of()
    for name, kind in of._fields_:
        if kind is ScoreRules:
            for inner, _ in kind._fields_:
                setattr(want.rules, inner, next(left))
        else:
            setattr(want, name, next(left))
    assert packed == bytes(want)


def test_structures_of_arguments_are_needed(lib):
    for name in ("et_rotary_axes_by", "et_adapter_add_by", "et_attention_rules_by"):
        assert getattr(lib, name)(None) == 1 and name.encode() in lib.et_last_error()


def rotary(lib, **change):
    a = dict(q_out=P, q=P, q_out_pitch=64, q_pitch=64, nhead_q=1, k_out=P, k=P, k_out_pitch=64, k_pitch=64, nhead_k=1, head_dim=64, rot_dim=64, positions=P, n_axes=1,
             inv_freq=P, axis=P, interleaved=0, tokens=0, stream=None)
    a.update(change)
    return both(lib, "et_rotary_axes", a.values(), RotaryArgs(**a))


@pytest.mark.parametrize("change", [dict(tokens=-1), dict(nhead_q=-1), dict(head_dim=0), dict(head_dim=257), dict(rot_dim=63), dict(rot_dim=66), dict(rot_dim=-2), dict(n_axes=0),
                                    dict(tokens=1, q=None), dict(tokens=1, k_out=None), dict(tokens=1, positions=None), dict(tokens=1, axis=None), dict(tokens=1, q_pitch=63),
                                    dict(tokens=1, k_out_pitch=8), dict(tokens=1, q_out_pitch=128)])
def test_rotary_refuses(lib, change):
    assert rotary(lib, **change) == 1 and b"et_rotary_axes" in lib.et_last_error()


def test_rotary_of_nothing(lib):
    assert rotary(lib) == 0
    assert rotary(lib, tokens=5, nhead_q=0, nhead_k=0) == 0


@pytest.mark.parametrize("sizes", [(0, 64, 8, 1), (24, 64, 8, 1), (64, 40, 8, 1), (64, 64, 0, 1), (64, 64, 129, 1), (64, 64, 8, 0), (-16, 64, 8, 1)])
def test_adapter_bank_refuses(lib, sizes):
    bank = ctypes.c_void_p(16)
    assert lib.et_adapter_bank_create(ctypes.byref(bank), *sizes) == 1 and not bank
    assert lib.et_adapter_bank_create(None, 64, 64, 8, 1) == 1


def test_adapter_without_a_bank(lib):
    assert lib.et_adapter_bank_set(None, 0, 1, P, P, ctypes.c_float(1)) == 1
    assert lib.et_adapter_add(None, P, P, P, 64, 64, 64, None, P, 1, 1, None) == 1 and lib.et_adapter_add_by(ctypes.byref(AdapterArgs(None, P, P, P, None, P, None, 64, 64, 64, 1, 1))) == 1
    assert lib.et_adapter_bank_destroy(None) == 0


def attention(lib, rules=None, **change):
    a = dict(out=P, Q=P, K=P, V=P, out_pitch=128, q_pitch=128, k_pitch=64, v_pitch=64, nhead=2, nhead_kv=1, head_dim=64, cu=None, k_start=None, k_lens=None, batch=1, q_tokens=4,
             k_rows=4, max_q_len=4, max_k_len=4)
    a.update(change)
    values = dict(scale=0.0, cap=0.0, slopes=0, distance_bias=0, reach=0, window_left=-1, window_right=-1, prefix_lens=0, q_docs=0, k_docs=0)
    values.update(rules or {})
    rules = ScoreRules(**values)
    return both(lib, "et_attention_rules", (*a.values(), ctypes.byref(rules), None, ctypes.c_size_t(0), None), RulesArgs(**a, rules=rules))


@pytest.mark.parametrize("change", [dict(batch=-1), dict(q_tokens=-1), dict(max_k_len=-1), dict(nhead=0), dict(nhead_kv=0), dict(nhead=3, nhead_kv=2), dict(head_dim=0), dict(head_dim=257),
                                    dict(nhead=1 << 16), dict(max_q_len=1 << 30), dict(k_start=P), dict(out=None), dict(Q=None), dict(V=None), dict(batch=2), dict(q_pitch=127),
                                    dict(v_pitch=63), dict(rules=dict(cap=-1.0)), dict(rules=dict(cap=math.inf)), dict(rules=dict(cap=1e-39)), dict(rules=dict(scale=3e38)), dict(rules=dict(scale=math.nan)), dict(rules=dict(scale=-1.0)),
                                    dict(rules=dict(slopes=16, distance_bias=16)), dict(rules=dict(distance_bias=16, reach=-1)), dict(rules=dict(q_docs=16)),
                                    dict(rules=dict(q_docs=16, k_docs=16))])
def test_attention_refuses(lib, change):
    assert attention(lib, **change) == 1 and b"et_attention_rules" in lib.et_last_error()


def test_attention_of_nothing(lib):
    for change in (dict(batch=0), dict(q_tokens=0), dict(max_q_len=0)):
        assert attention(lib, **change) == 0


def test_attention_scratch_size(lib):
    import et_b200 as et
    assert et.attention_rules_scratch_size(0, 100) == 0 and et.attention_rules_scratch_size(3, 0) == 0
    assert et.attention_rules_scratch_size(3, 129) == 3 * 3 * 8 and et.attention_rules_scratch_size(1 << 20, 1 << 20) == (1 << 20) * (1 << 14) * 8
