"""Operators of a layer served in 8 bits, as measurable cases.

A case is a dict of plain values with an "op":
  norm    residual's addition and root-mean-square norm, with an output in fp16, or in e4m3 with a scale for each 128 features of a token; or no
          norm, rows brought to e4m3 alone (the input of a linear behind attention or an activation)
  linear  matrix product of e4m3 activations (a scale for each 128 features of a token) and e4m3 weights (a scale for each 128 x 128), bias, GELU
  cache   keys and values quantised to int8 with a scale for each row and head as they are written into pages, and whole sequences read back in fp16
  tree    attention of drafted tokens over such a cache: each sees what was kept before and, of the drafted ones, those on its way to the root

Widths, heads and lengths are those of the benchmark's and the tests' layers (hidden 768 or 1024, heads of 64) and beside them generic
ones of larger models (4096 features, grouped heads of 128).
"""
import math
import random

import numpy as np
import torch

own = False

BLOCK = 128      # features, and weights' rows, that share a scale
E4M3_MAX = 448.0


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one new token of each of 64 requests before the Q|K|V projection of a large layer
        {"name": "norm 64x1024", "op": "norm", "tokens": 64, "width": 1024, "skip": True, "codes": True, "pitched": False, "norm": True},
        # whole prompts in a wide layer
        {"name": "norm 16384x4096", "op": "norm", "tokens": 16384, "width": 4096, "skip": True, "codes": True, "pitched": False, "norm": True},
        # an odd number of tokens in a base layer whose next linear takes fp16, rows as slices of wider ones
        {"name": "norm half 5003x768", "op": "norm", "tokens": 5003, "width": 768, "skip": True, "codes": False, "pitched": True, "norm": True},
        # the smallest product: one request's next token through an attention's output projection
        {"name": "linear 1x1024", "op": "linear", "tokens": 1, "k": 1024, "n": 1024, "bias": True, "gelu": False},
        # 64 requests' next tokens through a wide projection: reading the weights once
        {"name": "linear 64x4096", "op": "linear", "tokens": 64, "k": 4096, "n": 4096, "bias": False, "gelu": False},
        # a few sentences through a fused Q|K|V projection of a base layer
        {"name": "linear 1111x768", "op": "linear", "tokens": 1111, "k": 768, "n": 2304, "bias": True, "gelu": False},
        # the largest: prompts through the first linear of a wide FFN
        {"name": "linear gelu 16384x4096", "op": "linear", "tokens": 16384, "k": 4096, "n": 4096, "bias": True, "gelu": True},
        # one new token of each of 16 short requests, and their sequences for a layer that takes fp16
        {"name": "cache 16 tokens", "op": "cache", "batch": 16, "lo": 1, "hi": 48, "fresh": 1, "hk": 12, "hd": 64, "page": 16, "shape": 1},
        # the next 2048 tokens of four long prompts, with what is in the cache of them already
        {"name": "cache prompts 4x8192", "op": "cache", "batch": 4, "lo": 5000, "hi": 8192, "fresh": 2048, "hk": 8, "hd": 128, "page": 64, "shape": 2},
        # the smallest tree: eight drafted tokens of one short request
        {"name": "tree 8 over 300", "op": "tree", "batch": 1, "lo": 300, "hi": 300, "drafts": 8, "ragged": False, "hq": 12, "hk": 12, "hd": 64, "page": 16, "shape": 3},
        # the next tokens of 64 requests over up to 8192 kept ones, nothing drafted
        {"name": "tokens 64x8192", "op": "tree", "batch": 64, "lo": 64, "hi": 8192, "drafts": 1, "ragged": False, "hq": 16, "hk": 4, "hd": 128, "page": 64, "shape": 4},
        # trees of up to 48 drafted tokens of 16 requests over long contexts
        {"name": "tree 48 over 16x12000", "op": "tree", "batch": 16, "lo": 1000, "hi": 12000, "drafts": 48, "ragged": True, "hq": 32, "hk": 8, "hd": 128, "page": 32, "shape": 5},
    ]


def _between(rng, lo, hi):
    """Log-uniform whole number in [lo, hi]."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["norm", "linear", "linear", "cache", "tree", "tree"])
    if op == "norm":
        width = rng.choice([768, 1024, 4096, 2048, 16 * rng.randint(4, 400)])
        norm = rng.random() < 0.75
        return {"op": op, "tokens": _between(rng, 1, 16384 * 4096 // max(width, 1024)), "width": width, "skip": norm and rng.random() < 0.8, "codes": not norm or rng.random() < 0.7,
                "pitched": rng.random() < 0.3, "norm": norm}
    if op == "linear":
        k, n = (rng.choice([768, 1024, 1024, 2048, 4096, 16 * rng.randint(8, 256)]) for _ in range(2))
        if rng.random() < 0.3:
            k, n = rng.choice([(768, 2304), (1024, 4096), (4096, 1024)])
        return {"op": op, "tokens": _between(rng, 1, min(32768, 16384 * 4096 * 4096 // (k * n))), "k": k, "n": n, "bias": rng.random() < 0.5, "gelu": rng.random() < 0.3}
    hd = rng.choice([64, 64, 128, 128, 96, 80, 32])
    page = rng.choice([16, 32, 64, 64, 128])
    if op == "cache":
        hk = rng.choice([1, 2, 4, 8, 12])
        hi = _between(rng, 8, 8192)
        batch = _between(rng, 1, max(1, min(64, 4 * 8192 * 8 * 128 // (hi * hk * hd))))
        return {"op": op, "batch": batch, "lo": max(1, hi // _between(rng, 1, 16)), "hi": hi, "fresh": _between(rng, 1, max(2, hi // 2)), "hk": hk, "hd": hd, "page": page,
                "shape": rng.randrange(1 << 30)}
    hk = rng.choice([1, 2, 4, 8]) if hd > 64 else rng.choice([2, 4, 8, 12])
    hq = hk * (rng.choice([1, 2, 4, 8]) if hk <= 4 else 1)
    drafts = 1 if rng.random() < 0.3 else _between(rng, 2, 64)
    hi = _between(rng, max(16, drafts), 16384)
    batch = _between(rng, 1, max(1, min(128, 16 * 6500 * 48 * 32 * 128 // (2 * hi * drafts * hq * hd), 32 * 8192 * 8 * 128 // (hi * hk * hd))))
    return {"op": op, "batch": batch, "lo": hi if rng.random() < 0.3 else max(1, hi // _between(rng, 2, 32)), "hi": hi, "drafts": drafts,
            "ragged": drafts > 1 and rng.random() < 0.5, "hq": hq, "hk": hk, "hd": hd, "page": page, "shape": rng.randrange(1 << 30)}


# ------------------------------------------------------------------------------------------------ what a case's sizes are
def _blocks(n):
    return (n + BLOCK - 1) // BLOCK


def _lengths(case):
    """Keys of every sequence, the new ones among them."""
    r = random.Random(case["shape"])
    lengths = [r.randint(case["lo"], case["hi"]) for _ in range(case["batch"])]
    lengths[r.randrange(case["batch"])] = case["hi"]
    return lengths


def _new(case, lengths):
    """New tokens of every sequence: those written, or those drafted."""
    r = random.Random(case["shape"] + 1)
    if case["op"] == "cache":
        return [min(n, case["fresh"]) for n in lengths]
    return [min(n, r.randint(1, case["drafts"]) if case["ragged"] else case["drafts"]) for n in lengths]


def _trees(case, counts):
    """For every drafted token the bits of those that it sees: itself, and those between it and the root."""
    r = random.Random(case["shape"] + 2)
    rows = []
    for n in counts:
        bits = []
        for i in range(n):
            parent = r.randint(max(-1, i - 6), i - 1)
            bits.append((bits[parent] if parent >= 0 else 0) | 1 << i)
        rows += bits
    return [b - (1 << 64) if b >> 63 else b for b in rows]


def work(case):
    """What a pass cannot do without: inputs read once, outputs written once, two operations per product and sum."""
    if case["op"] == "norm":
        n = case["tokens"] * case["width"]
        out = n + 4 * case["tokens"] * _blocks(case["width"]) if case["codes"] else 2 * n
        return {"bytes": 2 * n + (4 * n if case["skip"] else 0) + out + (2 * case["width"] if case["norm"] else 0), "flops": (6 if case["norm"] else 2) * n}
    if case["op"] == "linear":
        t, k, n = case["tokens"], case["k"], case["n"]
        return {"bytes": t * k + n * k + 2 * t * n + 4 * t * _blocks(k) + 4 * _blocks(n) * _blocks(k) + (2 * n if case["bias"] else 0), "flops": 2 * t * n * k}
    lengths = _lengths(case)
    new = _new(case, lengths)
    if case["op"] == "cache":
        row = 2 * case["hk"]   # heads of K and V
        return {"bytes": row * sum(new) * (2 * case["hd"] + case["hd"] + 4) + row * sum(lengths) * (case["hd"] + 4 + 2 * case["hd"]),
                "flops": 3 * row * case["hd"] * (sum(new) + sum(lengths))}
    bits = _trees(case, new)
    drafted = sum(bin(b & (1 << 64) - 1).count("1") for b in bits)
    pairs = sum((n - d) * d for n, d in zip(lengths, new)) + drafted
    return {"bytes": 2 * case["hk"] * sum(lengths) * (case["hd"] + 4) + 4 * sum(new) * case["hq"] * case["hd"], "flops": 4 * case["hd"] * case["hq"] * pairs}


# ------------------------------------------------------------------------------------------------ inputs
def _by_blocks(x):
    """Rows in blocks of 128 features, the last one filled up with zeros."""
    x = torch.nn.functional.pad(x, (0, -x.shape[-1] % BLOCK))
    return x.reshape(*x.shape[:-1], -1, BLOCK)


def _to_rows(x):
    """(codes, what they are multiplied by) of rows, a scale for each 128 features: scales [blocks, rows]."""
    blocks = _by_blocks(x)
    scales = blocks.abs().amax(-1) / E4M3_MAX
    codes = torch.where(scales[..., None] > 0, blocks / scales[..., None], 0.0).to(torch.float8_e4m3fn)
    return codes.flatten(1)[:, :x.shape[1]], scales.t().contiguous()


def _to_int8(x):
    """(codes, scales) of rows of a head [..., features]."""
    scales = x.abs().amax(-1, keepdim=True) / 127.0
    return torch.where(scales > 0, (x / scales).round(), 0.0).to(torch.int8), scales[..., 0]


def _inputs(case, seed):
    """Tensors of a case, from the seed alone."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = np.random.default_rng(seed)
    dev = torch.device("cuda")

    def normal(*shape, std=1.0, spread=0.0):
        """Features of different sizes, as layers have them."""
        x = torch.randn(*shape, generator=g, device=dev, dtype=torch.float32) * std
        if spread:
            x *= torch.exp(spread * torch.randn(shape[-1], generator=g, device=dev))
        return x

    def ints(values):
        return torch.tensor(np.asarray(values, dtype=np.int32), device=dev)

    s = {"case": case}
    if case["op"] == "norm":
        t, w = case["tokens"], case["width"]
        wide = w + (256 if case["pitched"] else 0)
        s["x"] = normal(t, wide, spread=0.7).half()[:, :w]
        s["skip"] = normal(t, w, std=0.5).half() if case["skip"] else None
        s["gamma"] = (1.0 + 0.1 * torch.randn(w, generator=g, device=dev)).half()
        s["residual"] = torch.zeros(t, w, dtype=torch.float16, device=dev) if case["skip"] else None
        s["out"] = torch.zeros(t, w, dtype=torch.float8_e4m3fn if case["codes"] else torch.float16, device=dev)
        s["scales"] = torch.zeros(_blocks(w), t, dtype=torch.float32, device=dev) if case["codes"] else None
        return s
    if case["op"] == "linear":
        t, k, n = case["tokens"], case["k"], case["n"]
        s["x"], s["x_scales"] = _to_rows(normal(t, k, spread=0.7))
        w = _by_blocks(torch.nn.functional.pad(normal(n, k, std=k ** -0.5), (0, 0, 0, -n % BLOCK)))   # [rows, blocks of columns, 128]
        w = w.reshape(_blocks(n), BLOCK, _blocks(k), BLOCK)
        s["w_scales"] = w.abs().amax((1, 3)) / E4M3_MAX
        s["w"] = (w / s["w_scales"][:, None, :, None]).to(torch.float8_e4m3fn).view(_blocks(n) * BLOCK, -1)[:n, :k].contiguous()
        s["bias"] = normal(n, std=0.2).half() if case["bias"] else None
        s["out"] = torch.zeros(t, n, dtype=torch.float16, device=dev)
        return s
    lengths = _lengths(case)
    new = _new(case, lengths)
    hk, hd, page = case["hk"], case["hd"], case["page"]
    counts = [-(-n // page) for n in lengths]
    pages = sum(counts) + 3
    ids = r.permutation(pages)
    table = np.zeros((case["batch"], max(counts)), dtype=np.int32)
    at = 0
    for b, c in enumerate(counts):   # a sequence's pages lie anywhere
        table[b, :c] = ids[at:at + c]
        at += c
    held = normal(pages * 2 * hk * page, hd, spread=0.3)
    codes, scales = _to_int8(held.half().float())
    s["codes"], s["scales"] = codes.view(pages, 2, hk, page, hd), scales.view(pages, 2, hk, page)
    del held
    if case["op"] == "cache":
        def slots(first):
            return ints(np.concatenate([table[b, np.arange(f, n) // page] * page + np.arange(f, n) % page for b, (f, n) in enumerate(zip(first, lengths))]))
        s["slots"], s["all_slots"] = slots([n - f for n, f in zip(lengths, new)]), slots([0] * len(lengths))
        kv = normal(sum(new), 2 * hk * hd, spread=0.3).half()   # as the fused projection leaves them
        s["k"], s["v"] = kv[:, :hk * hd], kv[:, hk * hd:]
        s["k_out"], s["v_out"] = (torch.zeros(sum(lengths), hk * hd, dtype=torch.float16, device=dev) for _ in range(2))
        return s
    s["q"] = normal(sum(new), case["hq"] * hd).half()
    s["out"] = torch.zeros_like(s["q"])
    s["lengths"], s["new"] = lengths, new
    s["k_lens"], s["table"] = ints(lengths), ints(table)
    s["tree"] = torch.tensor(_trees(case, new), dtype=torch.int64, device=dev) if case["drafts"] > 1 else None
    cu = np.concatenate([[0], np.cumsum(new)])
    s["cu"] = ints(cu) if min(new) != max(new) else None
    s["cu_host"] = [int(v) for v in cu]
    # of every sequence and place in its tree: the row of its token (the last one where it has fewer), and whether there is one
    place = np.arange(max(new))
    s["rows"] = torch.tensor(cu[:-1, None] + np.minimum(place, np.asarray(new)[:, None] - 1), device=dev)
    s["real"] = torch.tensor(place < np.asarray(new)[:, None], device=dev)
    s["kept"] = torch.tensor(np.asarray(lengths) - np.asarray(new), device=dev)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        import et_b200 as et
        if case["op"] == "linear":
            s["weight"] = et.Fp8Weight(case["k"], case["n"], s["w"].view(torch.uint8).cpu().numpy(), s["w_scales"].cpu().numpy(),
                                       None if s["bias"] is None else s["bias"].cpu().numpy(), is_gelu=case["gelu"])
    return s


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    case = s["case"]
    if own:
        return _run_own(s)
    return {"norm": _plain_norm, "linear": _plain_linear, "cache": _plain_cache, "tree": _plain_tree}[case["op"]](s)


def _run_own(s):
    import et_b200 as et
    case = s["case"]
    if case["op"] == "norm":
        if case["norm"]:
            et.skip_rmsnorm(s["out"], s["x"], s["skip"], s["gamma"], residual=s["residual"], scales=s["scales"])
        else:
            et.quantise_rows(s["out"], s["scales"], s["x"])
        return [t for t in (s["out"], s["scales"], s["residual"]) if t is not None]
    if case["op"] == "linear":
        return s["weight"].run(s["out"], s["x"], s["x_scales"])
    if case["op"] == "cache":
        et.kv_cache_write(s["codes"], s["scales"], s["k"], s["v"], s["slots"])
        return et.kv_cache_read(s["k_out"], s["v_out"], s["codes"], s["scales"], s["all_slots"])
    return et.attention_tree(s["out"], s["q"], s["codes"], s["scales"], s["table"], s["k_lens"], tree=s["tree"], cu_seqlens=s["cu"], max_q_len=max(s["new"]), max_k_len=case["hi"])


def _plain_norm(s):
    """h = x + skip, h / sqrt(mean of h^2 + 1e-6) gamma, in fp16 or in codes with their scales; and h."""
    h = s["x"].float()
    if s["skip"] is not None:
        h = h + s["skip"].float()
    y = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + 1e-6) * s["gamma"].float() if s["case"]["norm"] else h
    out = list(_to_rows(y)) if s["case"]["codes"] else [y.half()]
    return out + ([h.half()] if s["skip"] is not None else [])


def _plain_linear(s):
    """The values that the codes stand for, multiplied in 32 bits."""
    k, n = s["case"]["k"], s["case"]["n"]
    x = s["x"].float() * s["x_scales"].t().repeat_interleave(BLOCK, 1)[:, :k]
    w = s["w"].float() * s["w_scales"].repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]
    y = x @ w.t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    if s["case"]["gelu"]:
        y = 0.5 * y * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (y + 0.044715 * y ** 3)))
    return y.half()


def _plain_cache(s):
    """New rows go to their slots in codes; the rows of all sequences come back as values."""
    hk, hd, page = s["case"]["hk"], s["case"]["hd"], s["case"]["page"]
    for side, x in enumerate((s["k"], s["v"])):
        codes, scales = _to_int8(x.float().view(-1, hk, hd))
        at = s["slots"].long()
        s["codes"][at // page, side, :, at % page] = codes
        s["scales"][at // page, side, :, at % page] = scales
    at = s["all_slots"].long()
    return tuple((s["codes"][at // page, side, :, at % page].float() * s["scales"][at // page, side, :, at % page, None]).flatten(1).half() for side in (0, 1))


def _plain_tree(s):
    """softmax(q k / sqrt(hd)) v over the keys kept before and the drafted ones whose bit is set."""
    case = s["case"]
    hq, hk, hd, page = case["hq"], case["hk"], case["hd"], case["page"]
    batch, most = s["rows"].shape
    longest = max(s["lengths"])
    held = s["codes"][s["table"].long()].float() * s["scales"][s["table"].long()][..., None]   # [batch, pages, 2, heads, page, features]
    k, v = held.permute(2, 0, 3, 1, 4, 5).reshape(2, batch, hk, -1, hd)[:, :, :, :longest]
    q = s["q"][s["rows"]].float().view(batch, most, hk, hq // hk, hd).permute(0, 2, 3, 1, 4).reshape(batch, hk, -1, hd)
    scores = ((q * hd ** -0.5) @ k.transpose(2, 3)).view(batch, hq, most, longest)
    ahead = torch.arange(longest, device=q.device) - s["kept"][:, None]   # place among the drafted tokens, below 0: kept before
    bits = s["tree"][s["rows"]] if s["tree"] is not None else torch.ones_like(s["rows"])
    seen = (bits[:, :, None] >> ahead.clamp(0, 63)[:, None]) & 1 == 1
    seen = torch.where((ahead < 0)[:, None], True, seen & (ahead < 64)[:, None]) & (torch.arange(longest, device=q.device) < s["k_lens"][:, None])[:, None]
    scores = torch.where(seen[:, None], scores, -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    o = (p.view(batch, hk, -1, longest) @ v).view(batch, hq, most, hd) / p.sum(-1, keepdim=True)
    o = o.permute(0, 2, 1, 3).flatten(2)
    return o[s["real"]].half()


# ------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "norm":
        h = s["x"].double() + (s["skip"].double() if case["skip"] else 0.0)
        y = h / torch.sqrt((h ** 2).sum(1, keepdim=True) / case["width"] + 1e-6) * s["gamma"].double() if case["norm"] else h
        out = [y]
        if case["codes"]:
            scales = torch.stack([c.abs().max(1).values / E4M3_MAX for c in y.split(BLOCK, 1)])
            out = [torch.cat([c / f[:, None] for c, f in zip(y.split(BLOCK, 1), scales)], 1).float().to(torch.float8_e4m3fn).double(), scales]
        return out + ([h] if case["skip"] else [])
    if case["op"] == "linear":
        y = torch.zeros(case["tokens"], case["n"], dtype=torch.float64, device="cuda")
        for i in range(_blocks(case["k"])):
            at = slice(i * BLOCK, (i + 1) * BLOCK)
            part = s["x"][:, at].double() @ s["w"][:, at].double().t()
            part *= s["x_scales"][i].double()[:, None]
            part *= torch.repeat_interleave(s["w_scales"][:, i].double(), BLOCK)[:case["n"]]
            y += part
        if case["bias"]:
            y += s["bias"].double()
        return torch.nn.functional.gelu(y, approximate="tanh") if case["gelu"] else y
    page, hd = case["page"], case["hd"]
    if case["op"] == "cache":
        result = []
        for side, x in enumerate((s["k"], s["v"])):
            flat = s["codes"][:, side].permute(0, 2, 1, 3).reshape(-1, case["hk"], hd).double() * s["scales"][:, side].permute(0, 2, 1).reshape(-1, case["hk"], 1).double()
            x = x.double().reshape(-1, case["hk"], hd)
            step = x.abs().max(2, keepdim=True).values / 127
            flat[s["slots"].long()] = torch.round(x / step) * step
            result.append(flat[s["all_slots"].long()].flatten(1))
        return tuple(result)
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    group = case["hq"] // case["hk"]
    for b, (n, d) in enumerate(zip(s["lengths"], s["new"])):
        at = torch.arange(n, device="cuda")
        ids = s["table"][b].long()[at // page]
        rows = slice(s["cu_host"][b], s["cu_host"][b + 1])
        hidden = torch.zeros(d, n, dtype=torch.bool, device="cuda")
        if s["tree"] is not None:
            words = [int(w) & (1 << 64) - 1 for w in s["tree"][rows].tolist()]
            hidden[:, n - d:] = torch.tensor([[not w >> j & 1 for j in range(d)] for w in words], device="cuda")
        for h in range(case["hk"]):
            k, v = (s["codes"][ids, side, h, at % page].double() * s["scales"][ids, side, h, at % page, None].double() for side in (0, 1))
            q = s["q"][rows, h * group * hd:(h + 1) * group * hd].double().reshape(d, group, hd)
            x = torch.einsum("dgf,nf->dgn", q, k) / math.sqrt(hd)
            x = x.masked_fill(hidden[:, None], -math.inf)
            out[rows, h * group * hd:(h + 1) * group * hd] = (torch.softmax(x, -1) @ v).flatten(1)
    return out
