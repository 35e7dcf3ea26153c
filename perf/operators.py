"""Operators of newer encoders and of serving them, as measurable cases.

A case is a dict of plain values with an "op":
  rotary     rotary positions over several axes, on the heads of Q and K
  adapter    low-rank adapters of many requests, added to a shared projection's result
  attention  attention with rules on its scores: a tanh cap, a bias by distance (slopes or a table), a window, a prefix, documents;
             whole sequences, or single tokens over keys kept from before

Widths, heads and lengths are those of the benchmark's and the tests' BERT-base and BERT-large layers (hidden 768 or 1024, heads of
64), and beside them the generic ones of grouped heads of 128. All tensors are fp16 as everywhere in this library.
"""
import math
import random

import numpy as np
import torch

own = False


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one new token of each of 64 requests through the rotation of a base layer
        {"name": "rotary 64 tokens", "op": "rotary", "tokens": 64, "hq": 12, "hk": 12, "hd": 64, "rot": 64, "axes": 3, "interleaved": False, "fused": True, "far": 2000},
        # a long video (time, height, width) through a large layer
        {"name": "rotary video 32768", "op": "rotary", "tokens": 32768, "hq": 16, "hk": 16, "hd": 64, "rot": 64, "axes": 3, "interleaved": False, "fused": False, "far": 100},
        # images (height, width), an odd number of patches, part of each head rotated, Q and K as slices of one fused Q|K|V buffer
        {"name": "rotary image 5003", "op": "rotary", "tokens": 5003, "hq": 32, "hk": 8, "hd": 128, "rot": 96, "axes": 2, "interleaved": True, "fused": True, "far": 500000},
        # one token of each of 64 requests, 24 fine-tunes of one projection
        {"name": "adapter 64 tokens", "op": "adapter", "batch": 64, "lo": 1, "hi": 1, "k": 1024, "n": 1024, "rank": 16, "slots": 24, "none": 0.0, "shape": 1},
        # whole prompts of 32 requests through the first linear of a large FFN
        {"name": "adapter prompts 32", "op": "adapter", "batch": 32, "lo": 128, "hi": 1024, "k": 1024, "n": 4096, "rank": 32, "slots": 8, "none": 0.0, "shape": 2},
        # a few short sentences through a fused Q|K|V projection, some of them without an adapter
        {"name": "adapter ragged 9", "op": "adapter", "batch": 9, "lo": 1, "hi": 300, "k": 768, "n": 2304, "rank": 8, "slots": 4, "none": 0.25, "shape": 3},
        # a bidirectional encoder with a learned bias for each distance up to 128
        {"name": "attention table 32x512", "op": "attention", "single": False, "batch": 32, "lo": 512, "hi": 512, "hq": 12, "hk": 12, "hd": 64, "cap": 0.0, "bias": "table", "reach": 128,
         "left": -1, "right": -1, "prefix": 0.0, "docs": 0, "shape": 4},
        # sentences of any length in layers that look 64 tokens to each side
        {"name": "attention window ragged 48", "op": "attention", "single": False, "batch": 48, "lo": 1, "hi": 701, "hq": 12, "hk": 12, "hd": 64, "cap": 0.0, "bias": "", "reach": 0,
         "left": 64, "right": 64, "prefix": 0.0, "docs": 0, "shape": 5},
        # documents of about 700 tokens packed into long rows, a slope for each head
        {"name": "attention documents 2x8192", "op": "attention", "single": False, "batch": 2, "lo": 8192, "hi": 8192, "hq": 16, "hk": 16, "hd": 64, "cap": 0.0, "bias": "slopes", "reach": 0,
         "left": -1, "right": -1, "prefix": 0.0, "docs": 700, "shape": 6},
        # the largest: prompts with a prefix seen by all and capped scores, grouped heads of 128
        {"name": "attention prefix cap 4x4096", "op": "attention", "single": False, "batch": 4, "lo": 4096, "hi": 4096, "hq": 16, "hk": 4, "hd": 128, "cap": 50.0, "bias": "", "reach": 0,
         "left": -1, "right": 0, "prefix": 0.25, "docs": 0, "shape": 7},
        # the smallest call: the next token of one short request
        {"name": "attention token 1x300", "op": "attention", "single": True, "batch": 1, "lo": 300, "hi": 300, "hq": 12, "hk": 12, "hd": 64, "cap": 0.0, "bias": "slopes", "reach": 0,
         "left": -1, "right": 0, "prefix": 0.0, "docs": 0, "shape": 8},
        # the next tokens of 64 requests over up to 8192 kept ones
        {"name": "attention tokens 64x8192", "op": "attention", "single": True, "batch": 64, "lo": 64, "hi": 8192, "hq": 16, "hk": 4, "hd": 128, "cap": 30.0, "bias": "", "reach": 0,
         "left": -1, "right": 0, "prefix": 0.0, "docs": 0, "shape": 9},
    ]


def _between(rng, lo, hi):
    """Log-uniform whole number in [lo, hi]."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["rotary", "adapter", "adapter", "attention", "attention", "attention"])
    if op == "rotary":
        hd = rng.choice([64, 64, 128, 96, 80])
        hk = rng.choice([1, 2, 4, 8, 12])
        hq = hk * rng.choice([1, 1, 2, 4])
        tokens = _between(rng, 1, min(32768, 32768 * 16 * 64 // ((hq + hk) * hd // 2)))
        rot = hd if rng.random() < 0.5 else 2 * rng.randint(hd // 8, hd // 2)
        return {"op": op, "tokens": tokens, "hq": hq, "hk": hk, "hd": hd, "rot": rot, "axes": rng.randint(1, 4),
                "interleaved": rng.random() < 0.5, "fused": rng.random() < 0.5, "far": _between(rng, 10, 1000000)}
    if op == "adapter":
        d = rng.choice([768, 1024])
        k, n = rng.choice([(d, d), (d, 3 * d), (d, 4 * d), (4 * d, d)])
        if 3 * d in (k, n) and d == 1024 or 4 * d in (k, n) and d == 768:
            k, n = (k, d) if k != d else (d, d)
        batch = _between(rng, 1, 128)
        if rng.random() < 0.4:
            lo = hi = 1
        else:
            hi = _between(rng, 2, max(2, min(2048, 32768 // batch)))
            lo = max(1, hi // _between(rng, 1, 16))
        return {"op": op, "batch": batch, "lo": lo, "hi": hi, "k": k, "n": n, "rank": rng.choice([4, 8, 16, 16, 32, 64, rng.randint(1, 64)]),
                "slots": _between(rng, 1, 64), "none": rng.choice([0.0, 0.0, 0.3]), "shape": rng.randrange(1 << 30)}
    single = rng.random() < 0.4
    hd = rng.choice([64, 64, 64, 128, 128, 96, 32])
    hk = rng.choice([1, 2, 4, 8, 12]) if hd > 64 else rng.choice([4, 8, 12, 16])
    hq = hk * rng.choice([1, 2, 4, 8]) if hk <= 4 else hk
    bias = rng.choice(["", "", "slopes", "table"])
    left, right = rng.choice([(-1, -1), (-1, 0), (-1, 0), (_between(rng, 16, 1024), 0), (64, 64), (_between(rng, 8, 512),) * 2])
    if single:
        right = 0 if right else right
        hi = _between(rng, 16, 16384)
        batch = _between(rng, 1, min(128, max(1, 64 * 8192 * 4 * 128 // (hi * hk * hd))))
    else:
        hi = _between(rng, 8, 8192)
        batch = _between(rng, 1, min(64, max(1, 4 * 4096 * 4096 * 16 * 128 // (2 * hi * hi * hq * hd)), max(1, 32768 // hi)))
    lo = hi if rng.random() < 0.4 else max(1, hi // _between(rng, 2, 32))
    return {"op": op, "single": single, "batch": batch, "lo": lo, "hi": hi, "hq": hq, "hk": hk, "hd": hd, "cap": rng.choice([0.0, 0.0, 30.0, 50.0]), "bias": bias,
            "reach": rng.choice([32, 128, 128, rng.randint(1, 600)]) if bias == "table" else 0, "left": left, "right": right,
            "prefix": rng.choice([0.0, 0.0, 0.3]) if right >= 0 else 0.0, "docs": rng.choice([0, 0, _between(rng, 16, 2048)]) if not single else 0,
            "shape": rng.randrange(1 << 30)}


# ------------------------------------------------------------------------------------------------ what a case's sizes are
def _lengths(case):
    r = random.Random(case["shape"])
    lengths = [r.randint(case["lo"], case["hi"]) for _ in range(case["batch"])]
    lengths[r.randrange(case["batch"])] = case["hi"]
    return lengths


def _prefixes(case, lengths):
    r = random.Random(case["shape"] + 1)
    return [int(n * case["prefix"] * 2 * r.random()) for n in lengths]


def _documents(case, lengths):
    """The document of every token: runs of about the case's length, numbered through; the last few tokens of a row are padding (-1)."""
    r = random.Random(case["shape"] + 2)
    ids, number = [], 0
    for n in lengths:
        row, pad = [], r.randint(0, min(n // 4, case["docs"] // 4))
        while len(row) < n - pad:
            row += [number] * min(r.randint(max(1, case["docs"] // 2), case["docs"] * 3 // 2), n - pad - len(row))
            number += 1
        ids.append(np.array(row + [-1] * pad, dtype=np.int32))
    return ids


def _adapters(case):
    r = random.Random(case["shape"] + 3)
    return [-1 if r.random() < case["none"] else r.randrange(case["slots"]) for _ in range(case["batch"])]


def _pairs(case):
    """Pairs of a query and a key that it sees, of one head."""
    lengths, total = _lengths(case), 0
    prefixes = _prefixes(case, lengths)
    documents = _documents(case, lengths) if case["docs"] else None
    for b, n in enumerate(lengths):
        q = np.arange(n - 1, n) if case["single"] else np.arange(n)
        lo = np.zeros_like(q) if case["left"] < 0 else np.maximum(q - case["left"], 0)
        hi = np.full_like(q, n) if case["right"] < 0 else np.minimum(q + case["right"] + 1, n)
        first, last = np.zeros_like(q), np.full_like(q, n)
        if documents is not None:
            d = documents[b]
            edges = np.flatnonzero(np.diff(d)) + 1
            at = np.searchsorted(edges, q, side="right")
            bounds = np.concatenate([[0], edges, [n]])
            first, last = bounds[at], np.where(d[q] < 0, bounds[at], bounds[at + 1])
        window = np.maximum(np.minimum(hi, last) - np.maximum(lo, first), 0)
        pre = np.minimum(prefixes[b], last)
        ahead = np.maximum(pre - first, 0)
        both = np.maximum(np.minimum(np.minimum(hi, last), pre) - np.maximum(lo, first), 0)
        total += int((window + ahead - both).sum())
    return total


def work(case):
    """What a pass cannot do without: inputs read once, outputs written once, two operations per product and sum."""
    if case["op"] == "rotary":
        width = (case["hq"] + case["hk"]) * case["hd"]
        return {"bytes": case["tokens"] * (4 * width + 4 * case["axes"]) + 4 * case["rot"], "flops": 3 * case["tokens"] * (case["hq"] + case["hk"]) * case["rot"]}
    if case["op"] == "adapter":
        lengths, ids = _lengths(case), _adapters(case)
        tokens, adapted = sum(lengths), sum(n for n, a in zip(lengths, ids) if a >= 0)
        weights = len({a for a in ids if a >= 0}) * case["rank"] * (case["k"] + case["n"])
        return {"bytes": 2 * (adapted * case["k"] + 2 * tokens * case["n"] + weights), "flops": 2 * adapted * case["rank"] * (case["k"] + case["n"])}
    lengths = _lengths(case)
    queries = len(lengths) if case["single"] else sum(lengths)
    keys = sum(lengths)
    if case["single"] and case["left"] >= 0 and not case["prefix"]:
        keys = sum(min(n, case["left"] + 1) for n in lengths)
    table = 2 * case["hq"] * (2 * case["reach"] + 1) if case["bias"] == "table" else 0
    return {"bytes": 2 * case["hd"] * (2 * queries * case["hq"] + 2 * keys * case["hk"]) + table, "flops": 4 * case["hd"] * case["hq"] * _pairs(case)}


# ------------------------------------------------------------------------------------------------ inputs
def _inputs(case, seed):
    """Tensors of a case, from the seed alone."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = np.random.default_rng(seed)
    dev = torch.device("cuda")

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, generator=g, device=dev, dtype=torch.float32) * std).half()

    def ints(values):
        return torch.tensor(np.asarray(values, dtype=np.int32), device=dev)

    s = {"case": case}
    if case["op"] == "rotary":
        t, hd = case["tokens"], case["hd"]
        wq, wk = case["hq"] * hd, case["hk"] * hd
        if case["fused"]:   # as the fused projection leaves them
            qkv = normal(t, wq + 2 * wk)
            s["q"], s["k"] = qkv[:, :wq], qkv[:, wq:wq + wk]
        else:
            s["q"], s["k"] = normal(t, wq), normal(t, wk)
        # places on a grid that starts anywhere: the first axis far along, the others inside a picture
        side = max(1, int(math.sqrt(t)))
        i = np.arange(t)
        places = [int(r.integers(0, case["far"] + 1)) + i // max(1, t // 64)] + [i // side % side, i % side, i][:case["axes"] - 1]
        s["positions"] = ints(np.stack(places, 1))
        pairs = case["rot"] // 2
        s["axis"] = ints(np.arange(pairs) * case["axes"] // pairs)
        s["inv_freq"] = torch.tensor((10000.0 ** (-2.0 * np.arange(pairs) / case["rot"])).astype(np.float32), device=dev)
        s["q_out"], s["k_out"] = torch.zeros(t, wq, dtype=torch.float16, device=dev), torch.zeros(t, wk, dtype=torch.float16, device=dev)
        return s
    if case["op"] == "adapter":
        lengths = _lengths(case)
        cu = np.concatenate([[0], np.cumsum(lengths)])
        s["lengths"], s["ids"] = lengths, _adapters(case)
        s["cu"] = ints(cu) if case["hi"] > 1 else None
        s["ids_dev"] = ints(s["ids"])
        s["x"], s["base"] = normal(int(cu[-1]), case["k"]), normal(int(cu[-1]), case["n"])
        s["scales"] = [float(v) for v in r.uniform(0.5, 2.0, case["slots"]).astype(np.float32)]
        s["a"] = normal(case["slots"], case["rank"], case["k"], std=case["k"] ** -0.5)
        s["b"] = normal(case["slots"], case["n"], case["rank"], std=0.5 * case["rank"] ** -0.5)
        s["out"] = torch.zeros_like(s["base"])
        return s
    lengths = _lengths(case)
    hd, hq, hk = case["hd"], case["hq"], case["hk"]
    s["lengths"] = lengths
    s["prefixes"] = _prefixes(case, lengths) if case["prefix"] else None
    if s["prefixes"]:
        s["prefix_dev"] = ints(s["prefixes"])
    sharp = 3.0 if case["cap"] else 1.0   # capped layers have large scores
    if case["single"]:   # keys and values where they were kept: a place of the largest length for every request
        room = (case["hi"] + 63) // 64 * 64
        s["starts"], s["places"] = [b * room for b in range(case["batch"])], room * case["batch"]
        s["q"] = normal(case["batch"], hq * hd, std=sharp)
        s["k"], s["v"] = normal(s["places"], hk * hd), normal(s["places"], hk * hd)
        s["starts_dev"], s["lengths_dev"] = ints(s["starts"]), ints(lengths)
        s["q_at"] = list(range(case["batch"]))
    else:
        cu = np.concatenate([[0], np.cumsum(lengths)])
        qkv = normal(int(cu[-1]), (hq + 2 * hk) * hd)
        qkv[:, :hq * hd] *= sharp
        s["q"], s["k"], s["v"] = qkv[:, :hq * hd], qkv[:, hq * hd:(hq + hk) * hd], qkv[:, (hq + hk) * hd:]
        s["cu"] = ints(cu) if case["lo"] != case["hi"] else None
        s["starts"] = s["q_at"] = [int(v) for v in cu[:-1]]
    if case["bias"] == "slopes":
        s["slopes"] = torch.tensor((2.0 ** (-8.0 * np.arange(1, hq + 1) / hq)).astype(np.float32), device=dev)
    if case["bias"] == "table":
        s["table"] = normal(hq, 2 * case["reach"] + 1)
    if case["docs"]:
        s["documents"] = ints(np.concatenate(_documents(case, lengths)))
    s["out"] = torch.zeros(s["q"].shape, dtype=torch.float16, device=dev)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        import et_b200 as et
        if case["op"] == "adapter":
            bank = et.AdapterBank(case["k"], case["n"], case["rank"], case["slots"])
            a, b = s["a"].cpu().numpy(), s["b"].cpu().numpy()
            for i in range(case["slots"]):
                bank.set(i, a[i], b[i], s["scales"][i])
            s["bank"] = bank
        if case["op"] == "attention" and case["docs"]:
            s["scratch"] = torch.empty(et.attention_rules_scratch_size(case["batch"], case["hi"]), dtype=torch.uint8, device="cuda")
    return s


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    case = s["case"]
    if own:
        return _run_own(s)
    return {"rotary": _plain_rotary, "adapter": _plain_adapter, "attention": _plain_attention}[case["op"]](s)


def _run_own(s):
    import et_b200 as et
    case = s["case"]
    if case["op"] == "rotary":
        return et.rotary_axes(s["q_out"], s["k_out"], s["q"], s["k"], s["positions"], s["inv_freq"], s["axis"], case["hd"], interleaved=case["interleaved"])
    if case["op"] == "adapter":
        return s["bank"].add(s["out"], s["base"], s["x"], s["ids_dev"], cu_seqlens=s["cu"])
    rules = dict(cap=case["cap"], slopes=s.get("slopes"), distance_bias=s.get("table"), window=(case["left"], case["right"]), prefix_lens=s.get("prefix_dev"))
    if case["single"]:
        return et.attention_rules(s["out"], s["q"], s["k"], s["v"], case["hd"], k_start=s["starts_dev"], k_lens=s["lengths_dev"], batch=case["batch"],
                                  max_q_len=1, max_k_len=case["hi"], **rules)
    return et.attention_rules(s["out"], s["q"], s["k"], s["v"], case["hd"], cu_seqlens=s["cu"], batch=case["batch"], max_q_len=case["hi"], max_k_len=case["hi"],
                              q_docs=s.get("documents"), k_docs=s.get("documents"), scratch=s.get("scratch"), **rules)


def _plain_rotary(s):
    """(x, y) -> (x cos a - y sin a, x sin a + y cos a) for each pair of features, a = place on the pair's axis x its frequency."""
    case = s["case"]
    angle = s["positions"][:, s["axis"].long()].double() * s["inv_freq"].double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def turn(x):
        x = x.reshape(x.shape[0], -1, case["hd"]).float()
        rot = case["rot"]
        if case["interleaved"]:
            a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        else:
            a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        out = x.clone()
        u, v = a * cos - b * sin, a * sin + b * cos
        if case["interleaved"]:
            out[..., 0:rot:2], out[..., 1:rot:2] = u, v
        else:
            out[..., :rot // 2], out[..., rot // 2:rot] = u, v
        return out.flatten(1).half()

    return turn(s["q"]), turn(s["k"])


def _plain_adapter(s):
    """base + scale (x A^T) B^T with the A, B and scale of each sequence's adapter."""
    out, at = s["base"].clone(), 0
    for n, i in zip(s["lengths"], s["ids"]):
        if i >= 0:
            low = s["x"][at:at + n].float() @ s["a"][i].float().t()
            out[at:at + n] = (s["base"][at:at + n].float() + s["scales"][i] * (low @ s["b"][i].float().t())).half()
        at += n
    return out


def _plain_attention(s):
    """softmax(cap tanh(q k / (sqrt(hd) cap)) + bias by distance, over the keys that a query sees) v; zeros where it sees none."""
    case = s["case"]
    hd, hq, hk = case["hd"], case["hq"], case["hk"]
    out = torch.zeros(s["q"].shape, dtype=torch.float16, device=s["q"].device)
    for b, n in enumerate(s["lengths"]):
        rows = 1 if case["single"] else n
        q_at, k_at = s["q_at"][b], s["starts"][b]
        k = s["k"][k_at:k_at + n].reshape(n, hk, hd).float().permute(1, 2, 0)
        v = s["v"][k_at:k_at + n].reshape(n, hk, hd).float().permute(1, 0, 2)
        keys = torch.arange(n, device=k.device)
        step = max(1, (1 << 27) // (n * hq))
        for r0 in range(0, rows, step):
            r1 = min(rows, r0 + step)
            q = s["q"][q_at + r0:q_at + r1].reshape(r1 - r0, hk, hq // hk, hd).float().permute(1, 2, 0, 3).reshape(hk, -1, hd)
            places = torch.arange(r0, r1, device=k.device) + (n - 1 if case["single"] else 0)
            away = keys[None, :] - places[:, None]
            scores = ((q * hd ** -0.5) @ k).view(hq, r1 - r0, n)
            if case["cap"]:
                scores = case["cap"] * torch.tanh(scores / case["cap"])
            if case["bias"] == "slopes":
                scores = scores - s["slopes"][:, None, None] * away.abs().float()
            if case["bias"] == "table":
                scores = scores + s["table"].float()[:, away.clamp(-case["reach"], case["reach"]) + case["reach"]]
            seen = torch.ones_like(away, dtype=torch.bool)
            if case["left"] >= 0:
                seen &= away >= -case["left"]
            if case["right"] >= 0:
                seen &= away <= case["right"]
            if s["prefixes"]:
                seen |= keys[None, :] < s["prefixes"][b]
            if case["docs"]:
                d = s["documents"][k_at:k_at + n]
                seen &= (d[r0:r1, None] == d[None, :]) & (d[None, :] >= 0)
            scores = torch.where(seen, scores, -math.inf)
            top = scores.amax(-1, keepdim=True)
            p = torch.exp(scores - torch.where(top > -math.inf, top, 0.0))
            total = p.sum(-1, keepdim=True)
            o = (p.view(hk, -1, n) @ v).view(hq, r1 - r0, hd) / torch.where(total > 0, total, 1.0)
            out[q_at + r0:q_at + r1] = o.permute(1, 0, 2).reshape(r1 - r0, hq * hd).half()
    return out


# ------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "rotary":
        pairs, hd = case["rot"] // 2, case["hd"]
        first = torch.arange(pairs, device="cuda") * (2 if case["interleaved"] else 1)
        second = first + (1 if case["interleaved"] else pairs)
        angle = torch.gather(s["positions"], 1, s["axis"].long().expand(case["tokens"], pairs)).to(torch.float64) * s["inv_freq"].to(torch.float64)
        turn = torch.polar(torch.ones_like(angle), angle)
        result = []
        for name, heads in (("q", case["hq"]), ("k", case["hk"])):
            out = s[name].to(torch.float64)
            for h in range(heads):
                z = torch.complex(out[:, h * hd + first], out[:, h * hd + second]) * turn
                out[:, h * hd + first], out[:, h * hd + second] = z.real, z.imag
            result.append(out)
        return tuple(result)
    if case["op"] == "adapter":
        token_slot = torch.tensor(np.repeat(s["ids"], s["lengths"]), device="cuda")
        out = s["base"].to(torch.float64)
        for i in range(case["slots"]):
            rows = torch.nonzero(token_slot == i).flatten()
            if len(rows):
                full = s["b"][i].to(torch.float64) @ s["a"][i].to(torch.float64)
                out[rows] += s["scales"][i] * (s["x"][rows].to(torch.float64) @ full.t())
        return out
    if 4 * case["hd"] * case["hq"] * sum(n * (1 if case["single"] else n) for n in s["lengths"]) > 4e12:
        return None
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    hd, group = case["hd"], case["hq"] // case["hk"]
    for b, n in enumerate(s["lengths"]):
        k_rows = slice(s["starts"][b], s["starts"][b] + n)
        at = torch.arange(n, device="cuda")
        offset = n - 1 if case["single"] else 0
        for r0 in range(0, 1 if case["single"] else n, 4096):
            r1 = min(r0 + 4096, 1 if case["single"] else n)
            q_rows = slice(s["q_at"][b] + r0, s["q_at"][b] + r1)
            distance = at - (at[r0:r1] + offset).unsqueeze(1) if not case["single"] else (at - offset).unsqueeze(0)
            hidden = torch.zeros(distance.shape, dtype=torch.bool, device="cuda")
            if case["left"] >= 0:
                hidden |= distance < -case["left"]
            if case["right"] >= 0:
                hidden |= distance > case["right"]
            if s["prefixes"]:
                hidden &= at >= s["prefixes"][b]
            if case["docs"]:
                d = s["documents"]
                hidden |= d[q_rows].unsqueeze(1) != d[k_rows]
                hidden |= d[k_rows] < 0
            for h in range(case["hq"]):
                q = s["q"][q_rows, h * hd:(h + 1) * hd].to(torch.float64)
                k = s["k"][k_rows, h // group * hd:(h // group + 1) * hd].to(torch.float64)
                v = s["v"][k_rows, h // group * hd:(h // group + 1) * hd].to(torch.float64)
                x = q @ k.t() / math.sqrt(hd)
                if case["cap"]:
                    x = torch.tanh(x / case["cap"]) * case["cap"]
                if case["bias"] == "slopes":
                    x -= s["slopes"][h].to(torch.float64) * distance.abs()
                if case["bias"] == "table":
                    x += s["table"][h].to(torch.float64)[torch.clamp(distance, min=-case["reach"], max=case["reach"]) + case["reach"]]
                x.masked_fill_(hidden, -math.inf)
                log_total = torch.logsumexp(x, 1, keepdim=True)
                p = torch.exp(x - torch.where(torch.isinf(log_total), 0.0, log_total))
                out[q_rows, h * hd:(h + 1) * hd] = p @ v
    return out
