"""Rotary positions, adapters and attention with rules on its scores, on the GPU, against plain 64-bit forms."""
import math

import numpy as np
import pytest

from tests import operators_lib as ol

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def et():
    import et_b200
    return et_b200


def dev(values, dtype="int32"):
    import torch
    return torch.tensor(np.asarray(values), device="cuda").to(getattr(torch, dtype))


def normal(seed, *shape, std=1.0):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * std).half()


# ------------------------------------------------------------------------------------------------ rotary positions
def rotary_inputs(tokens, hq, hk, hd, rot, axes, far, seed=1, pad=0):
    import torch
    r = np.random.default_rng(seed)
    q = normal(seed, tokens, hq * hd + pad)[:, :hq * hd]
    k = normal(seed + 1, tokens, hk * hd + pad)[:, :hk * hd]
    pos = dev(r.integers(-far, far + 1, (tokens, axes)))
    inv = torch.tensor((10000.0 ** (-2.0 * np.arange(rot // 2) / max(rot, 1))).astype(np.float32), device="cuda")
    return q, k, pos, inv, dev(r.integers(0, axes, rot // 2))


def check_rotary(et, q, k, pos, inv, axis, hd, interleaved, q_out=None, k_out=None):
    import torch
    want = [ol.rotary(x, pos, inv, axis, hd, interleaved) for x in (q, k)]
    # products and their difference in fp32 with angles good to a few 2^-24 turns, then half a step of fp16
    big = [x.double().abs().amax().item() if x.numel() else 0.0 for x in (q, k)]
    got = et.rotary_axes(torch.zeros_like(q) if q_out is None else q_out, torch.zeros_like(k) if k_out is None else k_out, q, k, pos, inv, axis, hd, interleaved=interleaved)
    for g, w, b in zip(got, want, big):
        ol.assert_within(g, w, ol.HALF * w.abs() + 2.0 ** -25 + b * 2.0 ** -19, "rotary")


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,hq,hk,hd,rot,axes,far", [
    (1, 12, 12, 64, 64, 1, 10), (64, 12, 12, 64, 64, 3, 2000), (777, 16, 4, 128, 96, 2, 100000), (130, 5, 1, 80, 46, 4, 3000), (33, 3, 3, 72, 72, 2, 2147483646),
    (100, 2, 7, 256, 250, 1, 1000000), (50, 4, 2, 20, 10, 2, 500), (9, 1, 1, 2, 2, 1, 7), (40, 3, 2, 64, 0, 1, 5), (257, 8, 8, 8, 6, 3, 99), (5000, 1, 1, 32, 16, 2, 4000)])
def test_rotary(et, tokens, hq, hk, hd, rot, axes, far, interleaved):
    check_rotary(et, *rotary_inputs(tokens, hq, hk, hd, rot, axes, far), hd, interleaved)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("hd,rot", [(64, 64), (64, 46), (64, 32), (96, 80), (20, 12)])
def test_rotary_in_place_and_in_slices(et, hd, rot, interleaved):
    """In place gives the same bits as to another place, and touches nothing between the slices."""
    import torch
    hq, hk, t = 12, 4, 301
    qkv = normal(5, t, (hq + 2 * hk) * hd + 8)
    _, _, pos, inv, axis = rotary_inputs(t, 1, 1, hd, rot, 2, 5000)
    before = qkv.clone()
    q, k = qkv[:, :hq * hd], qkv[:, hq * hd:(hq + hk) * hd]
    a, b = et.rotary_axes(torch.zeros(t, hq * hd, device="cuda").half(), torch.zeros(t, hk * hd, device="cuda").half(), q, k, pos, inv, axis, hd, interleaved=interleaved)
    et.rotary_axes(q, k, q, k, pos, inv, axis, hd, interleaved=interleaved)
    assert torch.equal(q, a) and torch.equal(k, b) and torch.equal(qkv[:, (hq + hk) * hd:], before[:, (hq + hk) * hd:])
    for n, x in enumerate((before[:, :hq * hd], before[:, hq * hd:(hq + hk) * hd])):
        w = ol.rotary(x, pos, inv, axis, hd, interleaved)
        ol.assert_within((a, b)[n], w, ol.HALF * w.abs() + 2.0 ** -25 + 6 * 2.0 ** -19, "rotary of a slice")


def test_rotary_of_unaligned_rows_one_operand_and_unknown_axes(et):
    import torch
    q, k, pos, inv, axis = rotary_inputs(40, 3, 3, 64, 64, 2, 900, pad=1)   # rows that start anywhere
    check_rotary(et, q, k, pos, inv, axis, 64, False)
    axis = axis.clone()
    axis[3], axis[5] = 2, -1        # no such axis: not turned
    check_rotary(et, q, k, pos, inv, axis, 64, True)
    alone, _ = et.rotary_axes(torch.zeros_like(q), None, q, None, pos, inv, axis, 64)
    both, _ = et.rotary_axes(torch.zeros_like(q), torch.zeros_like(k), q, k, pos, inv, axis, 64)
    assert torch.equal(alone, both)
    nan = q.clone()
    nan[7, 70] = math.nan
    out, _ = et.rotary_axes(torch.zeros_like(q), None, nan, None, pos, inv, axis, 64)
    bad = torch.isnan(out)
    assert bad[7, 64:128].any() and not bad[:7].any() and not bad[8:].any() and not bad[7, :64].any() and not bad[7, 128:].any()


# ------------------------------------------------------------------------------------------------ adapters
def make_bank(et, k, n, max_rank, ranks, seed=1, slots=None):
    """(bank, {slot: (A, B, scale)}): one adapter of each rank, 0: an empty slot."""
    bank = et.AdapterBank(k, n, max_rank, slots or len(ranks))
    held = {}
    for i, r in enumerate(ranks):
        if r:
            A, B = normal(seed + 2 * i, r, k, std=k ** -0.5), normal(seed + 2 * i + 1, n, r, std=0.5 * r ** -0.5)
            held[i] = (A, B, 0.5 + 0.25 * i)
            bank.set(i, A.cpu().numpy(), B.cpu().numpy(), held[i][2])
    return bank, held


def check_adapter(et, bank, held, lengths, ids, k, n, single=False, seed=50, extra=3, pad=0):
    import torch
    cu = np.concatenate([[0], np.cumsum(lengths)])
    rows = int(cu[-1]) + (0 if single else extra)
    x, base = normal(seed, rows, k + pad)[:, :k], normal(seed + 1, rows, n + pad)[:, :n]
    want, bound = ol.adapter(base, x, cu, ids, held)
    out = torch.full((rows, n + pad), 7.0, device="cuda").half()[:, :n]
    cu_dev = None if single else dev(cu)
    bank.add(out, base, x, dev(ids), cu_seqlens=cu_dev)
    inside = slice(0, int(cu[-1]))
    ol.assert_within(out[inside], want[inside], bound[inside], "adapter")
    assert (out[int(cu[-1]):] == 7.0).all(), "rows behind the last sequence were written"
    place = base.clone()
    bank.add(place, place, x, dev(ids), cu_seqlens=cu_dev)
    assert torch.equal(place[inside], out[inside]) and torch.equal(place[int(cu[-1]):], base[int(cu[-1]):])


@pytest.mark.parametrize("k,n,max_rank,ranks", [(768, 768, 16, [16, 8, 0, 1]), (1024, 4096, 32, [32, 17, 4]), (16, 16, 4, [4, 3]), (4096, 1024, 64, [64, 33, 16, 5]),
                                               (768, 2304, 8, [8]), (208, 368, 128, [128, 100, 65, 2]), (1008, 48, 48, [48, 20])])
@pytest.mark.parametrize("lengths", [[1], [5, 0, 1, 64], [300, 1, 128, 77], [33] * 40, [1000]])
def test_adapters_of_sequences(et, k, n, max_rank, ranks, lengths):
    bank, held = make_bank(et, k, n, max_rank, ranks)
    ids = [(i * 7) % (len(ranks) + 1) - 1 for i in range(len(lengths))]   # -1: none
    ids[-1] = 0
    check_adapter(et, bank, held, lengths, ids, k, n)


@pytest.mark.parametrize("k,n,max_rank,ranks", [(768, 768, 16, [16, 8, 0]), (1024, 368, 32, [32, 17]), (256, 2304, 64, [64, 40]), (208, 48, 128, [128, 100]), (96, 16, 4, [4])])
def test_adapters_of_many_tokens(et, k, n, max_rank, ranks):
    """Enough tokens for the form in which base and out move by TMA: whole tiles, ends of sequences inside one, sequences of one token, without an adapter, empty."""
    bank, held = make_bank(et, k, n, max_rank, ranks)
    lengths = [3001, 2500, 31, 0, 4096, 1, 33, 640]
    check_adapter(et, bank, held, lengths, [0, 1, -1, 0, 0, 1, 0, -1], k, n, pad=8)


@pytest.mark.parametrize("k,n,max_rank,ranks,lengths", [
    (64, 80, 16, [16, 3], [20000, 5, 17000, 3003, 1, 0, 8192]),                              # more than one wave of tiles
    (144, 64, 32, [20, 32], [9 + i * 7 % 32 for i in range(600)]),                           # many short sequences
    (1024, 4096, 64, [64, 50], [1800, 1, 1799]), (4096, 1024, 128, [128, 65], [5003]),       # few tokens, wide: the columns of a tile are shared
    (768, 2304, 8, [8, 5], [128] * 64 + [7] * 3), (80, 1008, 48, [48, 33], [8192]), (32, 16, 100, [100, 1], [72, 8130])])
def test_adapters_of_many_tokens_in_other_shapes(et, k, n, max_rank, ranks, lengths):
    bank, held = make_bank(et, k, n, max_rank, ranks)
    check_adapter(et, bank, held, lengths, [(i + i // 3) % (len(ranks) + 1) - 1 if i else 0 for i in range(len(lengths))], k, n, pad=8)
    et.attention_check()


@pytest.mark.parametrize("rank", [5, 48, 128])
def test_adapter_rows_of_many_tokens_do_not_mix(et, rank):
    """Infinities, what is no number and values whose A x is beyond fp16 stay in their rows; so does a sequence's adapter of infinities."""
    import torch
    k, n = 256, 320
    bank, held = make_bank(et, k, n, rank, [rank, rank])
    lengths, ids = [4500, 3, 4000, 900], [0, 1, -1, 0]
    cu = np.concatenate([[0], np.cumsum(lengths)])
    x, base = normal(1, 9403, k), normal(2, 9403, n)
    x[77], x[4400, 9], x[4502, 0], base[8600, 5] = 60000.0, math.inf, math.nan, math.inf
    x[9000] = 1.0e-7
    want, bound = ol.adapter(base, x, cu, ids, held)
    out = bank.add(torch.zeros_like(base), base, x, dev(ids), cu_seqlens=dev(cu))
    odd = torch.zeros_like(out, dtype=torch.bool)
    odd[4400] = odd[4502] = True
    odd[8600, 5] = True
    assert not torch.isfinite(out[4400]).any() and torch.isnan(out[4502]).all() and torch.isinf(out[8600, 5])
    over = want.abs() > 65504 * (1 - 2.0 ** -10)   # the result itself is beyond the type
    look = ~odd & ~over
    ol.assert_within(torch.where(look, out, 0.0), torch.where(look, want, 0.0), torch.where(look, bound, 0.0), "rows")
    huge = A, B = torch.full((rank, k), 60000.0).half(), torch.ones(n, rank).half()
    bank.set(1, A.numpy(), B.numpy(), 1.0)
    again = bank.add(torch.zeros_like(base), base, x, dev(ids), cu_seqlens=dev(cu))
    same = torch.ones(9403, dtype=torch.bool, device="cuda")
    same[4500:4503] = False
    same[4400] = False
    assert torch.equal(again[same], out[same]) and huge


@pytest.mark.parametrize("batch", [1, 3, 64, 300])
@pytest.mark.parametrize("k,n,max_rank,ranks", [(1024, 1024, 16, [16] * 5), (768, 2304, 64, [64, 1, 0, 40]), (4096, 1024, 128, [128, 16]), (32, 48, 8, [8, 8])])
def test_adapters_of_single_tokens(et, k, n, max_rank, ranks, batch):
    bank, held = make_bank(et, k, n, max_rank, ranks)
    check_adapter(et, bank, held, [1] * batch, [(i * 5) % (len(ranks) + 1) - 1 for i in range(batch)], k, n, single=True)


@pytest.mark.parametrize("lengths", [[1] * 64, [40, 300, 1], [5000, 4100, 77]])
def test_adapters_in_a_graph_and_on_two_streams(et, lengths):
    """Captured twice, replayed side by side with direct calls; a slot that is filled anew, ids and lengths that change are those of the replay."""
    import torch
    k, n, total = 256, 320, sum(lengths)
    bank, held = make_bank(et, k, n, 16, [16, 9])
    single = max(lengths) == 1
    x, base = normal(5, total, k), normal(6, total, n)
    cu = np.concatenate([[0], np.cumsum(lengths)])
    ids = dev([i % 2 for i in range(len(lengths))])
    cu_dev = None if single else dev(cu)
    first = bank.add(torch.zeros_like(base), base, x, ids, cu_seqlens=cu_dev)
    torch.cuda.synchronize()
    outs, graphs, streams = [torch.zeros_like(base) for _ in range(2)], [], [torch.cuda.Stream() for _ in range(2)]
    for out in outs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            bank.add(out, base, x, ids, cu_seqlens=cu_dev)
        graphs.append(g)
    direct = torch.zeros_like(base)
    for _ in range(4):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        bank.add(direct, base, x, ids, cu_seqlens=cu_dev)
    torch.cuda.synchronize()
    assert all(torch.equal(t, first) for t in (*outs, direct))
    A, B = normal(90, 4, k, std=k ** -0.5), normal(91, n, 4)
    bank.set(1, A.cpu().numpy(), B.cpu().numpy(), 2.0)
    held[1] = (A, B, 2.0)
    ids.copy_(dev([1 - i % 2 for i in range(len(lengths))]))
    if not single:
        cu = np.array([0, 3, 3, total])
        cu_dev.copy_(dev(cu))
    graphs[0].replay()
    torch.cuda.synchronize()
    want, bound = ol.adapter(base, x, cu, ids.tolist(), held)
    ol.assert_within(outs[0], want, bound, "replayed")
    et.attention_check()


def test_adapter_rows_in_slices_and_strange_ids(et):
    bank, held = make_bank(et, 256, 512, 16, [16, 8])
    check_adapter(et, bank, held, [40, 2, 9], [0, 1, 0], 256, 512, pad=24)
    check_adapter(et, bank, held, [40, 2, 9, 3], [2, -5, 1 << 30, 1], 256, 512)       # no such slots: nothing is added
    check_adapter(et, bank, held, [1] * 5, [2, 1, -(1 << 31), 0, 9], 256, 512, single=True)


def test_adapter_slots_are_replaced_and_cleared(et):
    bank, held = make_bank(et, 256, 512, 16, [16, 8])
    A, B = normal(90, 3, 256, std=0.1), normal(91, 512, 3)
    bank.set(0, A.cpu().numpy(), B.cpu().numpy(), -1.5)
    held[0] = (A, B, -1.5)
    check_adapter(et, bank, held, [70, 8], [0, 1], 256, 512)
    bank.clear(0)
    del held[0]
    check_adapter(et, bank, held, [70, 8], [0, 1], 256, 512)


@pytest.mark.parametrize("single", [False, True])
def test_adapter_of_large_values_does_not_overflow_and_rows_do_not_mix(et, single):
    """A x far above fp16's largest value, brought back by B; a row that is not finite stays alone."""
    import torch
    k, n, r = 512, 256, 16
    bank = et.AdapterBank(k, n, r, 1)
    A, B = normal(1, r, k, std=8.0), normal(2, n, r, std=2.0 ** -14)
    bank.set(0, A.cpu().numpy(), B.cpu().numpy(), 0.25)
    lengths = [1] * 20 if single else [20]
    x, base = normal(3, 20, k, std=500.0), normal(4, 20, n)
    cu, ids = np.concatenate([[0], np.cumsum(lengths)]), [0] * len(lengths)
    assert (x.double() @ A.double().t()).abs().max() > 65504
    want, bound = ol.adapter(base, x, cu, ids, {0: (A, B, 0.25)})
    out = bank.add(torch.zeros_like(base), base, x, dev(ids), cu_seqlens=None if single else dev(cu))
    ol.assert_within(out, want, bound, "large adapter")
    x[3, 5] = math.inf
    again = bank.add(torch.zeros_like(base), base, x, dev(ids), cu_seqlens=None if single else dev(cu))
    assert not torch.isfinite(again[3]).any() and torch.equal(again[:3], out[:3]) and torch.equal(again[4:], out[4:])


def test_adapter_refusals_on_the_device(et):
    import torch
    bank, _ = make_bank(et, 64, 64, 8, [8])
    x, ids = normal(1, 4, 64), dev([0])
    wide = normal(2, 4, 68)
    for call, error in ((lambda: bank.add(x, x, x, dev([0] * 5)), et.EtError),                              # more single tokens than rows
                        (lambda: bank.add(x, x, wide[:, :64], ids, cu_seqlens=dev([0, 4])), et.EtError),    # rows off 16 bytes
                        (lambda: bank.add(x, x, x.float(), ids), ValueError), (lambda: bank.add(x, x, x, ids.long()), ValueError),
                        (lambda: bank.add(x, x, x, ids, cu_seqlens=dev([0])), ValueError), (lambda: bank.add(x.cpu(), x, x, ids), ValueError),
                        (lambda: bank.set(1, np.zeros((8, 64)), np.zeros((64, 8))), et.EtError), (lambda: bank.set(0, np.zeros((9, 64)), np.zeros((64, 9))), et.EtError),
                        (lambda: bank.set(0, np.zeros((8, 60)), np.zeros((64, 8))), ValueError)):
        with pytest.raises(error):
            call()


# ------------------------------------------------------------------------------------------------ attention
def run_attention(et, Q, K, V, hd, seqs, cu=None, k_start=None, k_lens=None, prefixes=None, window=(-1, -1), cap=0.0, slopes=None, table=None, docs=None, scale=0.0,
                  max_q=None, max_k=None, out=None):
    """Runs the operator and compares it with the 64-bit form. docs: (of the queries, of the keys)."""
    import torch
    batch = len(seqs)
    max_q, max_k = max_q or max([s[1] for s in seqs] + [1]), max_k or max([s[3] for s in seqs] + [1])
    if out is None:
        out = torch.full(Q.shape, 7.0, device="cuda").half()
    scratch = torch.full((max(1, et.attention_rules_scratch_size(batch, max_k)),), 255, dtype=torch.uint8, device="cuda") if docs else None
    et.attention_rules(out, Q, K, V, hd, cu_seqlens=None if cu is None else dev(cu), k_start=None if k_start is None else dev(k_start), k_lens=None if k_lens is None else dev(k_lens),
                       batch=batch, max_q_len=max_q, max_k_len=max_k, scale=scale, cap=cap, slopes=slopes, distance_bias=table, window=window,
                       prefix_lens=None if prefixes is None else dev(prefixes), q_docs=docs[0] if docs else None, k_docs=docs[1] if docs else None, scratch=scratch)
    et.attention_check()   # no wait has given up
    want, bound = ol.attention(Q, K, V, hd, seqs, scale=scale or None, cap=cap, slopes=slopes, table=table, window=window, prefixes=prefixes,
                               q_docs=docs[0] if docs else None, k_docs=docs[1] if docs else None)
    ol.assert_within(out, want, bound, "attention")
    outside = torch.isnan(want).all(1)
    assert (out[outside] == 7.0).all(), "rows of no sequence were written"
    return out


def packed(seed, lengths, hq, hk, hd, extra=0, std=1.0):
    """Q, K, V as slices of one fused buffer, and the sequences."""
    cu = np.concatenate([[0], np.cumsum(lengths)]).astype(int)
    qkv = normal(seed, int(cu[-1]) + extra, (hq + 2 * hk) * hd)
    qkv[:, :hq * hd] *= std
    return (*qkv.split([hq * hd, hk * hd, hk * hd], 1), cu, [(int(cu[b]), n, int(cu[b]), n, 0) for b, n in enumerate(lengths)])


LENGTHS = {"one": [1], "short": [5, 1, 0, 17], "uneven": [300, 129, 64, 1, 128, 255], "long": [1500]}
RULES = {
    "plain": {}, "cap": {"cap": 30.0}, "slopes": {"slopes": True}, "table": {"reach": 128}, "small table": {"reach": 3}, "table of one": {"reach": 0}, "wide table": {"reach": 700},
    "causal": {"window": (-1, 0)}, "window": {"window": (64, 64)}, "narrow": {"window": (0, 0)}, "only behind": {"window": (0, -1)}, "ahead": {"window": (200, 100)},
    "prefix": {"window": (-1, 0), "prefix": True}, "window prefix": {"window": (40, 3), "prefix": True}, "documents": {"docs": 40}, "causal documents": {"docs": 90, "window": (-1, 0)},
    "cap slopes causal": {"cap": 20.0, "slopes": True, "window": (-1, 0)}, "cap table documents": {"cap": 10.0, "reach": 50, "docs": 200},
    "all": {"cap": 50.0, "slopes": True, "docs": 60, "window": (100, 20), "prefix": True},
}


def rules_of(name, lengths, hq, seed=3):
    import torch
    r = np.random.default_rng(seed)
    rule = dict(RULES[name])
    args = {"window": rule.get("window", (-1, -1)), "cap": rule.get("cap", 0.0)}
    if rule.get("slopes"):
        args["slopes"] = torch.tensor(2.0 ** (-8.0 * np.arange(1, hq + 1) / hq), device="cuda").float()
    if "reach" in rule:
        args["table"] = normal(seed, hq, 2 * rule["reach"] + 1)
    if rule.get("prefix"):
        args["prefixes"] = [int(r.integers(0, n + 10)) for n in lengths]
    if rule.get("docs"):
        total = sum(lengths)
        ids = np.repeat(np.arange(total // rule["docs"] + 1), rule["docs"])[:total]
        ids[r.random(total) < 0.02] = -1                      # padding anywhere
        some = r.random(total) < 0.02
        ids[some] = r.integers(0, 3, int(some.sum()))          # and tokens of documents that lie elsewhere
        args["docs"] = (dev(ids),) * 2
    return args


@pytest.mark.parametrize("rule", RULES)
@pytest.mark.parametrize("lengths", LENGTHS)
@pytest.mark.parametrize("hq,hk,hd", [(4, 4, 64), (8, 2, 128)])
def test_attention_of_whole_sequences(et, hq, hk, hd, lengths, rule):
    lengths = LENGTHS[lengths]
    args = rules_of(rule, lengths, hq)
    Q, K, V, cu, seqs = packed(1, lengths, hq, hk, hd, std=3.0 if args["cap"] else 1.0)
    run_attention(et, Q, K, V, hd, seqs, cu=cu, **args)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("batch,longest", [(48, 701), (128, 150), (300, 90)])
@pytest.mark.parametrize("rule", ["plain", "window", "documents", "cap table documents", "all"])
def test_attention_of_ragged_batches_of_several_waves(et, batch, longest, rule, hd):
    """CTAs take over many short items, each with a last block of its own size, in order of length (up to 128 sequences) or as they come."""
    r = np.random.default_rng(batch)
    lengths = [int(n) for n in r.integers(0, longest + 1, batch)]
    Q, K, V, cu, seqs = packed(5, lengths, 12, 4, hd)
    run_attention(et, Q, K, V, hd, seqs, cu=cu, **rules_of(rule, lengths, 12))


@pytest.mark.parametrize("hq,hk,hd", [(3, 1, 16), (2, 2, 32), (6, 3, 48), (4, 1, 80), (2, 1, 96), (5, 5, 112), (2, 2, 20), (3, 1, 7), (2, 1, 192), (4, 2, 256)])
@pytest.mark.parametrize("rule", ["plain", "all", "cap table documents"])
def test_attention_of_other_heads(et, hq, hk, hd, rule):
    lengths = [200, 1, 333]
    Q, K, V, cu, seqs = packed(2, lengths, hq, hk, hd)
    run_attention(et, Q, K, V, hd, seqs, cu=cu, **rules_of(rule, lengths, hq))


@pytest.mark.parametrize("hd", [64, 128])
def test_attention_of_equal_lengths_key_padding_and_rows_left_alone(et, hd):
    Q, K, V, cu, seqs = packed(3, [150] * 5, 4, 2, hd, extra=9)
    run_attention(et, Q, K, V, hd, seqs, window=(-1, 0))                       # no cu_seqlens; nine rows behind the last sequence
    lens = [150, 0, 1, 129, 500]
    run_attention(et, Q, K, V, hd, [(s[0], 150, s[2], min(n, 150), 0) for s, n in zip(seqs, lens)], cu=cu, k_lens=lens, cap=5.0)


@pytest.mark.parametrize("hd", [64, 128, 40])
@pytest.mark.parametrize("rule", ["plain", "causal", "all", "window", "cap table documents"])
def test_attention_over_kept_keys(et, hd, rule):
    """Prompts that go on from kept keys: queries at the end of longer sequences, places anywhere, some shared, one query more than there are keys."""
    import torch
    nq, nk = [100, 1, 0, 260, 30, 7], [400, 300, 50, 260, 20, 0]
    starts = [500, 37, 0, 500, 1200, 3]
    cu = np.concatenate([[0], np.cumsum(nq)]).astype(int)
    Q, K, V = normal(4, int(cu[-1]), 8 * hd), normal(5, 1300, 2 * hd), normal(6, 1300, 2 * hd)
    args = rules_of(rule, nk, 8)
    if "docs" in args:
        args["docs"] = (dev(np.arange(int(cu[-1])) // 100 - 1), dev(np.arange(1300) // 150 % 5 - 1))
    seqs = [(int(cu[b]), nq[b], starts[b], nk[b], nk[b] - nq[b]) for b in range(6)]
    run_attention(et, Q, K, V, hd, seqs, cu=cu, k_start=starts, k_lens=nk, **args)
    assert torch.isfinite(Q).all()


@pytest.mark.parametrize("hq,hk,hd", [(12, 12, 64), (16, 4, 128), (8, 1, 96), (16, 1, 64), (32, 1, 128), (6, 2, 40), (5, 5, 16), (20, 1, 256)])
@pytest.mark.parametrize("lens", [[1], [300], [64, 0, 1, 17, 1000, 63, 65], [9000], [33] * 150])
@pytest.mark.parametrize("rule", ["plain", "cap slopes causal", "window prefix", "table", "documents", "window"])
def test_attention_of_single_tokens(et, hq, hk, hd, lens, rule):
    room = max(lens) + 5
    starts = [b * room for b in range(len(lens))][::-1]
    Q, K, V = normal(7, len(lens), hq * hd), normal(8, room * len(lens), hk * hd), normal(9, room * len(lens), hk * hd)
    args = rules_of(rule, lens, hq)
    if "docs" in args:
        args["docs"] = (dev(np.arange(len(lens)) % 3 - (len(lens) > 2)), dev(np.arange(room * len(lens)) // 40 % 3))
    run_attention(et, Q, K, V, hd, [(b, 1, starts[b], n, n - 1) for b, n in enumerate(lens)], k_start=starts, k_lens=lens, max_q=1, **args)


@pytest.mark.parametrize("hq,hk,hd", [(4, 4, 64), (16, 2, 128), (40, 1, 64), (6, 3, 32)])
@pytest.mark.parametrize("rule", ["causal", "all", "cap table documents"])
def test_attention_of_a_few_tokens(et, hq, hk, hd, rule):
    """Up to four new tokens of a sequence over its kept keys, which see one another as the rules say: several tiles of rows, sequences with fewer."""
    nq, nk = [4, 1, 0, 3, 2], [700, 64, 9, 3, 1]
    starts = [0, 700, 800, 900, 1000]
    cu = np.concatenate([[0], np.cumsum(nq)]).astype(int)
    Q, K, V = normal(4, int(cu[-1]), hq * hd), normal(5, 1010, hk * hd), normal(6, 1010, hk * hd)
    args = rules_of(rule, nk, hq)
    if "docs" in args:
        args["docs"] = (dev(np.arange(int(cu[-1])) % 4 - 1), dev(np.arange(1010) // 100 % 4))
    run_attention(et, Q, K, V, hd, [(int(cu[b]), nq[b], starts[b], nk[b], nk[b] - nq[b]) for b in range(5)], cu=cu, k_start=starts, k_lens=nk, max_q=4, **args)


@pytest.mark.parametrize("hd", [64, 128, 24])
def test_attention_of_values_that_are_not_numbers(et, hd):
    """What a row sees and is not a number makes it not a number, in all its features or in those of V, and no other row."""
    import torch
    Q, K, V, cu, seqs = packed(3, [600, 300], 4, 2, hd)
    K[610, 3] = math.nan                 # of the second sequence, first K/V head: its first two query heads
    V[20, hd + 5] = math.inf             # of the first sequence, second K/V head: its last two query heads, one feature each
    out = run_attention(et, Q, K, V, hd, seqs, cu=cu, window=(-1, 0))
    bad = torch.zeros(900, 4, hd, dtype=torch.bool, device="cuda")
    bad[610:, :2] = True
    bad[20:600, 2:, 5] = True
    assert torch.equal(~torch.isfinite(out.view(900, 4, hd)), bad)
    Q[:] = math.nan
    out = et.attention_rules(torch.zeros_like(out), Q, K, V, hd, cu_seqlens=dev(cu), batch=2, max_q_len=600, max_k_len=600, window=(-1, 0))
    assert torch.isnan(out).all()


@pytest.mark.parametrize("hd", [64, 128])
def test_attention_of_scores_that_keep_growing(et, hd):
    """Every block's scores are far above those of the block before: the reference moves each time; and far below: it stays."""
    import torch
    n = 1000
    Q, K, V = normal(1, 200, 2 * hd, std=0.1), normal(2, n, 2 * hd, std=0.1), normal(3, n, 2 * hd)
    Q[:, 0] = Q[:, hd] = 8.0
    ramp = (torch.arange(n, device="cuda") // 50).half() * 4
    for sign in (1, -1):
        K[:, 0] = K[:, hd] = sign * ramp
        for rows in (200, 1):
            run_attention(et, Q[:rows], K, V, hd, [(0, rows, 0, n, n - rows)], k_start=[0], k_lens=[n], max_q=rows)
            run_attention(et, Q[:rows], K, V, hd, [(0, rows, 0, n, n - rows)], k_start=[0], k_lens=[n], max_q=rows, slopes=torch.tensor([0.5, 0.01], device="cuda"), window=(-1, 0))


@pytest.mark.parametrize("single", [False, True])
@pytest.mark.parametrize("hd", [64, 128])
def test_attention_never_looks_at_what_is_not_seen(et, hd, single):
    """Not a number, infinity and the lowest value behind the last key, in other documents and behind the window."""
    import torch
    hq, hk = 8, 2
    lens, room = [200, 131, 64], 260
    starts = [b * room for b in range(3)]
    K, V = normal(8, room * 3, hk * hd), normal(9, room * 3, hk * hd)
    for b, n in enumerate(lens):
        K[starts[b] + n:starts[b] + room] = math.nan
        V[starts[b] + n:starts[b] + room] = math.nan
        V[starts[b] + n + 1] = math.inf
    nq = [1] * 3 if single else [20, 131, 64]
    cu = np.concatenate([[0], np.cumsum(nq)]).astype(int)
    Q = normal(7, int(cu[-1]), hq * hd)
    seqs = [(int(cu[b]), nq[b], starts[b], n, n - nq[b]) for b, n in enumerate(lens)]
    call = dict(cu=None if single else cu, k_start=starts, k_lens=lens)
    run_attention(et, Q, K, V, hd, seqs, **call)
    run_attention(et, Q, K, V, hd, seqs, cap=3.0, **call)
    # keys 50 .. 54 belong to another document and hold anything
    for value in (math.nan, math.inf, -65504.0):
        K2, V2 = K.clone(), V.clone()
        k_docs = np.zeros(room * 3, dtype=int)
        for s in starts:
            K2[s + 50:s + 55], V2[s + 50:s + 55], k_docs[s + 50:s + 55] = value, value, 3
        out = run_attention(et, Q, K2, V2, hd, seqs, docs=(dev(np.zeros(len(Q), dtype=int)), dev(k_docs)), **call)
        assert torch.isfinite(out).all()
        out = run_attention(et, Q, K2, V2, hd, seqs, docs=(dev(np.zeros(len(Q), dtype=int)), dev(k_docs)), cap=4.0, slopes=torch.ones(hq, device="cuda"), **call)
        assert torch.isfinite(out).all()
        # the last 40 keys only: what lies before the window is not seen
        out = run_attention(et, Q[-1:], K2, V2, hd, [(0, 1, starts[0], 200, 199)], k_start=starts[:1], k_lens=lens[:1], window=(40, 0))
        assert torch.isfinite(out).all()
        # and without documents it is seen: rows that see it are not finite, except where the value is only low
        out = run_attention(et, Q, K2, V2, hd, seqs, window=(-1, 0), **call)
        if math.isnan(value):
            assert torch.isnan(out[-1]).all()


@pytest.mark.parametrize("hd", [64, 128])
def test_attention_of_rows_that_see_nothing(et, hd):
    import torch
    lengths = [140, 300]
    Q, K, V, cu, seqs = packed(3, lengths, 4, 4, hd)
    none = dev(np.full(440, -1))
    assert (run_attention(et, Q, K, V, hd, seqs, cu=cu, docs=(none, none)) == 0).all()
    other = dev(np.arange(440) % 2), dev(np.arange(440) % 2 + 5)
    assert (run_attention(et, Q, K, V, hd, seqs, cu=cu, docs=other) == 0).all()
    assert (run_attention(et, Q, K, V, hd, [(q0, n, k0, 0, 0) for q0, n, k0, _, _ in seqs], cu=cu, k_lens=[0, 0]) == 0).all()
    some = dev(np.where(np.arange(440) % 3 == 0, -1, 1))
    out = run_attention(et, Q, K, V, hd, seqs, cu=cu, docs=(some, some))
    assert (out[::3] == 0).all() and (out[1::3] != 0).any(1).all()
    out = run_attention(et, Q[:2], K, V, hd, [(0, 1, 0, 0, -1), (1, 1, 0, 7, 6)], k_start=[0, 0], k_lens=[0, 7], max_q=1)
    assert (out[0] == 0).all()
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("hd", [64, 128, 40])
@pytest.mark.parametrize("rule", [{}, {"window": (70, 5)}, {"window": (-1, 0), "slopes": True}, {"cap": 20.0, "prefixes": [100, 3]}])
def test_attention_of_documents_in_any_order(et, hd, rule):
    """Numbers in any order, as many as keys, up to the largest; several numbers below 0 on both sides, which see and are seen by nothing."""
    import torch
    lengths = [500, 203]
    Q, K, V, cu, seqs = packed(1, lengths, 4, 2, hd)
    rule = {**rule, **({"slopes": torch.rand(4, device="cuda")} if rule.get("slopes") else {})}
    r = np.random.default_rng(3)
    n = len(Q)
    for docs in (r.integers(-4, 5, n), r.permutation(n) // 2, r.choice([-(1 << 31), -2, -1, 0, (1 << 31) - 1], n), np.arange(n) // 40 - 3, -1 - np.arange(n) % 3):
        other = np.where(r.random(n) < 0.5, docs, r.permutation(docs))
        for pair in ((docs, docs), (docs, other)):
            out = run_attention(et, Q, K, V, hd, seqs, cu=cu, docs=(dev(pair[0]), dev(pair[1])), **rule)
            assert (out[torch.as_tensor(pair[0] < 0, device="cuda")] == 0).all()
    et.attention_check()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("rule", [{}, {"window": (-1, 0)}, {"slopes": True}, {"reach": 30}])
def test_attention_of_scores_around_half_a_cap(et, hd, rule):
    """Rows whose scores end just below, at and above half a cap, far above it and near 0, side by side; one that is not a number."""
    import torch
    n, cap = 300, 8.0
    Q, K, V = torch.zeros(n, 2 * hd, device="cuda").half(), torch.zeros(n, 2 * hd, device="cuda").half(), normal(3, n, 2 * hd)
    K[:, 0] = K[:, hd] = torch.linspace(-1, 1, n, device="cuda").half()
    K[:, 1] = K[:, hd + 1] = 1.0 / 64
    rows = torch.arange(n, device="cuda")
    size = torch.tensor([0.001, 1.0, 3.99, 4.0, 4.01, 9.0, 100.0], device="cuda")[(rows // 32) % 7] * torch.where(rows % 5 == 0, 0.5, 1.0)
    Q[:, 0] = Q[:, hd] = (size * math.sqrt(hd)).half()
    Q[:, 1] = 1.0
    r = {**rule, **({"slopes": torch.tensor([0.02, 0.5], device="cuda")} if "slopes" in rule else {}), **({"table": normal(4, 2, 61)} if "reach" in rule else {})}
    r.pop("reach", None)
    out = run_attention(et, Q, K, V, hd, [(0, n, 0, n, 0)], cu=[0, n], cap=cap, **r)
    K[290, hd + 1] = math.nan   # of the second head, at the end
    Q[40, hd + 1] = 0.0
    again = et.attention_rules(torch.zeros_like(out), Q, K, V, hd, cu_seqlens=dev([0, n]), batch=1, max_q_len=n, max_k_len=n, cap=cap, window=r.get("window", (-1, -1)),
                               slopes=r.get("slopes"), distance_bias=r.get("table"))
    assert torch.equal(again[:, :hd], out[:, :hd]) and torch.isnan(again[290:, hd:]).all()
    assert torch.isnan(again[:290, hd:]).all() if "window" not in r else torch.equal(again[41:290, hd:], out[41:290, hd:])


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("single", [False, True])
def test_attention_of_large_scores(et, hd, single):
    """Scores of hundreds: one key takes all; capped ones are flat again; a scale of its own."""
    lens = [700]
    Q, K, V = normal(7, 1 if single else 130, 4 * hd, std=30.0), normal(8, 700, 4 * hd), normal(9, 700, 4 * hd)
    n = len(Q)
    seqs = [(0, n, 0, 700, 700 - n)]
    for args in ({}, {"cap": 50.0}, {"cap": 0.01}, {"scale": 1e-4}, {"scale": 0.5, "cap": 8.0}, {"cap": 1000.0}):
        run_attention(et, Q, K, V, hd, seqs, k_start=[0], k_lens=lens, **args)


def test_attention_limits_of_the_caller_hold(et):
    """Keys beyond max_k_len or beyond the rows that there are are not seen, whatever the lengths say; so are places outside."""
    for hd in (64, 24):
        Q, K, V = normal(1, 4, 4 * hd), normal(2, 300, 2 * hd), normal(3, 300, 2 * hd)
        lens, starts = [290, 290, 290, 50], [0, 100, 299, 400]
        seqs = [(0, 1, 0, 256, 289), (1, 1, 100, 200, 289), (2, 1, 299, 1, 289), (3, 1, 0, 0, 49)]
        run_attention(et, Q, K, V, hd, seqs, k_start=starts, k_lens=lens, max_q=1, max_k=256)
        run_attention(et, Q[:3], K, V, hd, [(0, 3, 100, 200, 287)], k_start=[100], k_lens=[290], max_k=290, window=(-1, 0))


@pytest.mark.parametrize("hd", [64, 128])
def test_attention_of_a_cache_beyond_32_bits(et, hd):
    """Rows whose elements lie beyond 2^31 of the first."""
    import torch
    pitch, rows = 2048, (1 << 31) // 2048 + 3000
    cache = torch.empty(rows, pitch, dtype=torch.float16, device="cuda")
    start = rows - 700
    cache[start:] = normal(1, 700, pitch)
    K, V = cache[:, :2 * hd], cache[:, 2 * hd:4 * hd]
    last = [(0, 1, start, 700, 699)]
    Q = normal(2, 60, 4 * hd)
    out = torch.zeros_like(Q)
    near_K, near_V = K[start:].clone(), V[start:].clone()
    for q, n in ((Q[:1], 1), (Q, 60)):
        et.attention_rules(out[:n], q, K, V, hd, k_start=dev([start]), k_lens=dev([700]), batch=1, max_q_len=n, max_k_len=700, window=(-1, 0))
        want, bound = ol.attention(q, near_K, near_V, hd, [(0, n, 0, 700, 700 - n)], window=(-1, 0))
        ol.assert_within(out[:n], want, bound, "far rows")
    assert last


def test_attention_in_strange_layouts(et):
    """Pitches and starts that are no multiple of 16 bytes; out in a wider buffer."""
    import torch
    for hd, pad in ((64, 1), (64, 4), (128, 8), (64, 8)):
        q, kv = normal(1, 210, 4 * hd + pad)[:, pad:], normal(2, 210, 4 * hd + pad)
        wide = torch.full((210, 6 * hd + pad), 7.0, device="cuda").half()
        run_attention(et, q, kv[:, :2 * hd], kv[:, 2 * hd:4 * hd], hd, [(0, 100, 0, 100, 0), (100, 110, 100, 110, 0)], cu=[0, 100, 210], window=(30, 30), out=wide[:, hd + pad:5 * hd + pad])
        assert (wide[:, :hd + pad] == 7.0).all() and (wide[:, 5 * hd + pad:] == 7.0).all()


def test_attention_is_the_same_every_time_and_in_a_graph(et):
    """Captured twice and replayed on another stream next to direct calls, with lengths that change in between: every result has the bits of a call of its own."""
    import torch
    hd, hq, hk = 64, 12, 12
    lengths = [33, 500, 1, 260, 129, 77]
    Q, K, V, cu, _ = packed(1, lengths, hq, hk, hd)
    slopes = torch.rand(hq, device="cuda")
    cu_dev, docs = dev(cu), dev(np.arange(len(Q)) // 50)
    scratch = [torch.empty(et.attention_rules_scratch_size(6, 512), dtype=torch.uint8, device="cuda") for _ in range(2)]
    kw = dict(cu_seqlens=cu_dev, batch=6, max_q_len=512, max_k_len=512, slopes=slopes, cap=20.0, q_docs=docs, k_docs=docs)
    first = et.attention_rules(torch.zeros_like(Q), Q, K, V, hd, scratch=scratch[0], **kw)
    single = dict(k_start=dev([0, 100]), k_lens=dev([700, 33]), batch=2, max_q_len=1, max_k_len=800, slopes=slopes)
    token = et.attention_rules(torch.zeros_like(Q[:2]), Q[:2], K, V, hd, **single)
    outs, graphs = [torch.zeros_like(Q) for _ in range(2)], []
    tokens = [torch.zeros_like(Q[:2]) for _ in range(2)]
    torch.cuda.synchronize()
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            et.attention_rules(outs[i], Q, K, V, hd, scratch=scratch[i], **kw)
            et.attention_rules(tokens[i], Q[:2], K, V, hd, **single)
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                outs[i].zero_()
                graphs[i].replay()
    torch.cuda.synchronize()
    for i in range(2):
        assert torch.equal(outs[i], first) and torch.equal(tokens[i], token)
    cu_dev.copy_(dev([0, 100, 100, 400, 900, 999, 1000]))
    docs.copy_(dev(np.arange(len(Q)) // 90))
    again = et.attention_rules(torch.zeros_like(Q), Q, K, V, hd, scratch=scratch[1], **kw)
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], again) and not torch.equal(again, first)
    et.attention_check()


def test_a_layer_of_them_together(et):
    """Q|K|V by a pruned linear, each sequence's adapter, rotary positions in place, attention with rules: as one program runs them, captured too."""
    import torch
    from tests import oracle_lib, util
    orc = oracle_lib.load()
    d, H, hd = 768, 12, 64
    lengths, ids = [200, 31, 128, 1], [0, -1, 1, 0]
    t = sum(lengths)
    rp, ro, data, bias = util.make_tile_linear(orc, d, 3 * d, 0.5, 5, bias_std=0.02, std=1.0 / math.sqrt(d / 2))
    linear = et.TileWeight(d, 3 * d, t, data, rp, ro, bias)
    bank, held = make_bank(et, d, 3 * d, 16, [16, 8])
    x = normal(11, t, d)
    cu = np.concatenate([[0], np.cumsum(lengths)]).astype(int)
    cu_dev, ids_dev = dev(cu), dev(ids)
    _, _, pos, inv, axis = rotary_inputs(t, 1, 1, hd, hd, 2, 300)
    table = normal(12, H, 65)
    qkv, out = torch.zeros(t, 3 * d, device="cuda").half(), torch.zeros(t, d, device="cuda").half()
    q, k, v = qkv.split(d, 1)

    def layer():
        linear.run(qkv, x)
        bank.add(qkv, qkv, x, ids_dev, cu_seqlens=cu_dev)
        et.rotary_axes(q, k, q, k, pos, inv, axis, hd)
        et.attention_rules(out, q, k, v, hd, cu_seqlens=cu_dev, batch=4, max_q_len=200, max_k_len=200, distance_bias=table, window=(64, 64), cap=30.0)

    layer()
    torch.cuda.synchronize()
    first = out.clone()
    # each step from what the one before it left, within that step's own bound
    plain = linear.run(torch.zeros_like(qkv), x)
    want, bound = ol.adapter(plain, x, cu, ids, held)
    added = bank.add(torch.zeros_like(plain), plain, x, ids_dev, cu_seqlens=cu_dev)
    ol.assert_within(added, want, bound, "adapter")
    turned = [ol.rotary(added[:, i * d:(i + 1) * d], pos, inv, axis, hd, False) for i in range(2)]
    for got, w in zip((q, k), turned):
        ol.assert_within(got, w, ol.HALF * w.abs() + 2.0 ** -25 + added.abs().max().item() * 2.0 ** -19, "rotary")
    want, bound = ol.attention(q, k, v, hd, [(int(cu[b]), n, int(cu[b]), n, 0) for b, n in enumerate(lengths)], cap=30.0, table=table, window=(64, 64))
    ol.assert_within(first, want, bound, "attention")
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            layer()
        out.zero_()
        for _ in range(3):
            g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, first)
    linear.check()
    et.attention_check()


def test_attention_refusals_on_the_device(et):
    import torch
    Q = normal(1, 8, 128)
    ok = dict(batch=1, max_q_len=8, max_k_len=8)
    ids = dev(np.zeros(8, dtype=int))
    out = torch.zeros_like(Q)
    for args, error in ((dict(cap=-1.0), et.EtError), (dict(scale=-1.0), et.EtError), (dict(scale=math.nan), et.EtError), (dict(q_docs=ids), et.EtError),
                        (dict(q_docs=ids, k_docs=ids), et.EtError),                                     # no scratch
                        (dict(k_start=dev([0])), et.EtError), (dict(batch=2), et.EtError), (dict(cu_seqlens=dev([0])), ValueError), (dict(slopes=Q[0]), ValueError),
                        (dict(distance_bias=Q[:2]), ValueError), (dict(prefix_lens=dev([1, 2])), ValueError), (dict(k_lens=dev([1]).long()), ValueError),
                        (dict(slopes=torch.ones(2, device="cuda"), distance_bias=normal(2, 2, 5)), et.EtError)):
        with pytest.raises(error):
            et.attention_rules(out, Q, Q, Q, 64, **{**ok, **args})
    for bad in (Q.float(), Q.cpu(), Q.t(), Q[:, :100]):
        with pytest.raises(ValueError):
            et.attention_rules(out, bad, Q, Q, 64, **ok)
    heads = normal(3, 4, 8).t()   # four heads of one feature, a row's elements apart; one of keys
    for bad in ((out[:, :4], heads, Q[:, :1], Q[:, :1]), (heads, out[:, :4], Q[:, :1], Q[:, :1]), (out[:, :1], out[:, :1], heads, heads)):
        with pytest.raises((ValueError, et.EtError)):
            et.attention_rules(*bad, 1, **ok)
    for hd in (0, -64):
        with pytest.raises((ValueError, et.EtError)):
            et.attention_rules(out, Q, Q, Q, hd, **ok)
        with pytest.raises((ValueError, et.EtError)):
            et.rotary_axes(out, None, Q, None, dev(np.zeros((8, 1), dtype=int)), torch.ones(32, device="cuda"), dev(np.zeros(32, dtype=int)), hd)
    assert (out == 0).all()


# Keys of one CTA with a block to each warp, of two CTAs whose second has the last key alone, of a cluster of sixteen.
@pytest.mark.parametrize("n", [49, 65, 993])
@pytest.mark.parametrize("nq", [1, 4, 6])   # single tokens and a few; six are whole sequences to the library
@pytest.mark.parametrize("cap", [0.0, 5.0])
@pytest.mark.parametrize("hq,hk,hd", [(4, 2, 64), (16, 2, 128), (16, 2, 64), (4, 2, 24)])
def test_tokens_over_kept_keys_of_values_that_are_not_numbers(et, hq, hk, hd, cap, nq, n):
    """A query, a block of keys or the last key that is not a number makes exactly the heads of the queries that see it not a number."""
    import torch
    Q, K, V = normal(1, nq, hq * hd), normal(2, n, hk * hd), normal(3, n, hk * hd)

    def odd(q, k, v, window=(-1, -1)):
        """Which elements are not finite."""
        out = et.attention_rules(torch.zeros_like(q), q, k, v, hd, k_start=dev([0]), k_lens=dev([n]), batch=1, max_q_len=nq, max_k_len=n, cap=cap, window=window)
        et.attention_check()
        return ~torch.isfinite(out).view(nq, hq, hd)

    expect = torch.zeros(nq, hq, hd, dtype=torch.bool, device="cuda")
    assert not odd(Q, K, V).any()
    assert odd(torch.full_like(Q, math.nan), K, V).all()
    one = Q.clone()
    one[nq - 1, hd + 1] = math.nan                       # the last query's second head
    expect[nq - 1, 1] = True
    assert torch.equal(odd(one, K, V), expect)
    for first, last in ((0, 16), (32, 48), (n - 1, n)):  # whole blocks, and the last key
        bad = K.clone()
        bad[first:last, hd:2 * hd] = math.nan            # of the second K/V head
        expect = torch.zeros_like(expect)
        expect[:, hq // 2:] = True
        assert torch.equal(odd(Q, bad, V), expect)
        expect[:] = False
        expect[max(0, first - (n - nq)):, hq // 2:] = True
        assert torch.equal(odd(Q, bad, V, window=(-1, 0)), expect)
        assert odd(Q, torch.full_like(K, math.nan), V).all()


@pytest.mark.parametrize("n", [49, 65, 993])
@pytest.mark.parametrize("nq", [1, 4])
@pytest.mark.parametrize("cap", [0.0, 5.0])
@pytest.mark.parametrize("hq,hk,hd", [(4, 2, 64), (16, 2, 128)])
def test_tokens_over_kept_keys_keep_their_bits_beside_masked_keys_that_are_not_numbers(et, hq, hk, hd, cap, nq, n):
    import torch
    Q, K, V = normal(1, nq, hq * hd), normal(2, n, hk * hd), normal(3, n, hk * hd)
    seqs, call = [(0, nq, 0, n, n - nq)], dict(k_start=[0], k_lens=[n], cap=cap, max_q=nq)
    for first, last in ((0, 16), (32, 48), (n - 1, n)):
        bad, k_docs = K.clone(), np.zeros(n, dtype=int)
        bad[first:last], k_docs[first:last] = math.nan, 3
        docs = (dev(np.zeros(nq, dtype=int)), dev(k_docs))
        assert torch.equal(run_attention(et, Q, bad, V, hd, seqs, docs=docs, **call), run_attention(et, Q, K, V, hd, seqs, docs=docs, **call))
    bad = K.clone()
    bad[:16] = math.nan
    near = dict(window=(n - nq - 16, 0))                 # the first sixteen keys are before it
    assert torch.equal(run_attention(et, Q, bad, V, hd, seqs, **near, **call), run_attention(et, Q, K, V, hd, seqs, **near, **call))


@pytest.mark.parametrize("n", [49, 65, 993])
@pytest.mark.parametrize("nq", [1, 4, 6])
@pytest.mark.parametrize("hd", [64, 128, 24])
def test_tokens_over_kept_keys_of_values_beside_scores_far_below(et, hd, nq, n):
    """A value that is not finite counts however small its key's weight is: beside 0 it is not a number."""
    import torch
    Q, K, V = normal(1, nq, 4 * hd, std=0.1), normal(2, n, 2 * hd, std=0.1), normal(3, n, 2 * hd)
    Q[:, ::hd] = 30.0
    K[:, ::hd] = 0.0
    seqs, call = [(0, nq, 0, n, n - nq)], dict(k_start=[0], k_lens=[n], max_q=nq)
    for first, last in ((32, 48), (n - 1, n)):
        for value in (math.inf, math.nan):
            far, bad = K.clone(), V.clone()
            far[first:last, hd] = -30.0 * math.sqrt(hd)  # scores of -900 for the second K/V head's queries
            bad[first, hd + 5] = value
            out = run_attention(et, Q, far, bad, hd, seqs, **call)
            expect = torch.zeros(nq, 4, hd, dtype=torch.bool, device="cuda")
            expect[:, 2:, 5] = True
            assert torch.equal(~torch.isfinite(out).view(nq, 4, hd), expect)


@pytest.mark.parametrize("cap", [512.0, 600.0, 1.0e4, 1.0e6, 1.0e9, 1.0e30])
@pytest.mark.parametrize("bias", ["none", "slopes", "table"])
@pytest.mark.parametrize("hd", [64, 128, 24])
@pytest.mark.parametrize("nq", [1, 4, 150])
def test_attention_of_caps_far_above_the_scores(et, nq, hd, bias, cap):
    """Such a cap changes next to nothing: the error does not grow with it."""
    import torch
    n = 333
    Q, K, V = normal(7, nq, 4 * hd, std=4.0), normal(8, n, 2 * hd), normal(9, n, 2 * hd)
    seqs = [(0, nq, 0, n, n - nq)]
    rules = {"slopes": torch.rand(4, device="cuda") * 0.02} if bias == "slopes" else {"table": normal(4, 4, 61)} if bias == "table" else {}
    scores = torch.einsum("qhd,khd->hqk", Q.double().view(nq, 4, hd), K.double().view(n, 2, hd).repeat_interleave(2, 1)) * hd ** -0.5
    assert 8 < scores.abs().max() < 32
    out = et.attention_rules(torch.zeros_like(Q), Q, K, V, hd, k_start=dev([0]), k_lens=dev([n]), batch=1, max_q_len=nq, max_k_len=n, cap=cap, slopes=rules.get("slopes"),
                             distance_bias=rules.get("table"))
    et.attention_check()
    want, _ = ol.attention(Q, K, V, hd, seqs, cap=cap, **rules)
    # The bound without a cap, a tenth wider. The cap moves a score by s^3 / 3 c^2 <= 0.042 (s <= 32, c >= 512) and a weight, which the bound is linear in, by 4.3 %
    # (relative to the sum of the weights, in which scores of 8 and more hardly differ, less). Its own rounding, 2^-21 of a score, is 1.6e-5 of a weight: 3.2 % of the half step 2^-11 that each
    # has in the bound. Up to c = 512 the quotient's rounding of 2^-22 c is as much as 1.3e-4: that one is counted as the oracle does.
    _, bound = ol.attention(Q, K, V, hd, seqs, cap=cap if cap <= 512 else 0.0, **rules)
    ol.assert_within(out, want, 1.1 * bound, f"cap {cap}")


@pytest.mark.parametrize("hd", [64, 128, 24])
@pytest.mark.parametrize("nq", [1, 4, 150])
@pytest.mark.parametrize("std", [100.0, 1000.0])
def test_attention_of_wide_caps_and_scores_around_them(et, nq, hd, std):
    Q, K, V = normal(7, nq, 4 * hd, std=std), normal(8, 333, 2 * hd), normal(9, 333, 2 * hd)
    for cap in (520.0, 2000.0):
        for rules in ({}, {"table": normal(4, 4, 61)}):
            run_attention(et, Q, K, V, hd, [(0, nq, 0, 333, 333 - nq)], k_start=[0], k_lens=[333], cap=cap, **rules)


def test_attention_waits_for_long_rows_that_are_computed_again(et):
    """An infinite value in a long sequence, seen by every query: its rows take a second, CTAs have more items, and no wait gives up meanwhile."""
    import torch
    hd, hq, nq, n = 64, 300, 32, 60000
    Q, K, V = normal(1, nq, hq * hd), normal(2, n, hd), normal(3, n, hd)
    V[n // 2, 5] = math.inf
    out = et.attention_rules(torch.zeros_like(Q), Q, K, V, hd, k_start=dev([0]), k_lens=dev([n]), batch=1, max_q_len=nq, max_k_len=n)
    et.attention_check()
    odd = ~torch.isfinite(out).view(nq, hq, hd)
    assert odd[:, :, 5].all() and int(odd.sum()) == nq * hq
    for h in (0, 299):
        want, bound = ol.attention(Q[:, h * hd:(h + 1) * hd], K, V.where(torch.isfinite(V), 0), hd, [(0, nq, 0, n, n - nq)])
        want[:, 5] = math.nan
        ol.assert_within(out[:, h * hd:(h + 1) * hd], want, bound, "rows computed again")


def test_attention_of_many_items_with_rows_computed_again(et):
    """More such items than a CTA keeps: every short sequence has a value that is not finite, of which only some queries know."""
    import torch
    hd, hq, lengths = 64, 16, [40, 200] * 200
    Q, K, V, cu, seqs = packed(3, lengths, hq, hq, hd)
    V[torch.as_tensor(cu[:-1] + 20, device="cuda", dtype=torch.long), hd + 7] = math.nan
    for window in ((-1, 0), (-1, -1)):
        out = run_attention(et, Q, K, V, hd, seqs, cu=cu, window=window)
        odd = torch.zeros(len(Q), hq, hd, dtype=torch.bool, device="cuda")
        at = torch.cat([torch.arange(n, device="cuda") for n in lengths])
        odd[at >= (20 if window[1] == 0 else 0), 1, 7] = True
        assert torch.equal(torch.isnan(out.view(-1, hq, hd)), odd)


@pytest.mark.parametrize("hq,hk,hd", [(8, 8, 64), (8, 2, 32), (8, 4, 128)])
@pytest.mark.parametrize("why", ["lengths", "documents", "positions"])
@pytest.mark.parametrize("batch,every", [(400, 10), (120, 4), (400, 3)])
def test_attention_of_many_items_that_see_nothing(et, hq, hk, hd, why, batch, every):
    """A few sequences with keys and then many without one that a query sees: CTAs take several such items in a row behind one that has blocks."""
    r = np.random.default_rng(batch)
    lengths = [int(n) for n in r.integers(30, 300 if batch < 200 else 130, batch)]
    full = [b < batch // every for b in range(batch)] if every != 3 else [b % 3 == 0 for b in range(batch)]
    Q, K, V, cu, seqs = packed(3, lengths, hq, hk, hd)
    if why == "lengths":
        lens = [n if f else 0 for n, f in zip(lengths, full)]
        run_attention(et, Q, K, V, hd, [(q0, n, q0, k, 0) for (q0, n, _, _, _), k in zip(seqs, lens)], cu=cu, k_lens=lens)
    elif why == "documents":
        ids = np.concatenate([np.full(n, 5 if f else -1) for n, f in zip(lengths, full)])
        run_attention(et, Q, K, V, hd, seqs, cu=cu, docs=(dev(ids), dev(ids)))
    else:   # more queries than kept keys: those before the first key see nothing, and behind the last one is nothing
        lens = [n if f else 1 for n, f in zip(lengths, full)]
        run_attention(et, Q, K, V, hd, [(q0, n, q0, k, k - n) for (q0, n, _, _, _), k in zip(seqs, lens)], cu=cu, k_start=[s[0] for s in seqs], k_lens=lens, window=(-1, 0))


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("batch", [400, 120])
def test_attention_of_items_that_all_have_rows_computed_again(et, batch, hd):
    """Every item of every CTA: a CTA's list is full before its items are at an end, and the others start by themselves."""
    import torch
    hq, lengths = 24, [(40, 130, 75)[b % 3] for b in range(batch)]
    Q, K, V, cu, seqs = packed(3, lengths, hq, hq, hd)
    rows = torch.as_tensor(cu[:-1] + 20, device="cuda", dtype=torch.long)
    for h in range(hq):
        V[rows, h * hd + 7] = math.nan
    out = run_attention(et, Q, K, V, hd, seqs, cu=cu, window=(-1, 0))
    at = torch.cat([torch.arange(n, device="cuda") for n in lengths])
    odd = torch.zeros(len(Q), hq, hd, dtype=torch.bool, device="cuda")
    odd[:, :, 7] = (at >= 20)[:, None]
    assert torch.equal(torch.isnan(out.view(-1, hq, hd)), odd)
