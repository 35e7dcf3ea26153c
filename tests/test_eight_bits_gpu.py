"""Layers in 8 bits (norms with e4m3 output, products of e4m3 codes, a cache in int8 pages, attention of drafted tokens over it) against their definitions in 64 bits.

Bounds: a result in fp16 is off by 2^-11 of itself (half a step; below 2^-14 by 2^-25), a code in e4m3 by 2^-4 of its value (below 2^-6 scales by 2^-10 of the scale). What fp32
arithmetic adds stands beside each test."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
HALF, TINY = 2.0 ** -11, 2.0 ** -25


@pytest.fixture(scope="module")
def et():
    import et_b200
    return et_b200


def test_arguments_are_checked_and_packed_in_cpp(et):
    from et_b200 import ops
    assert ops._load_fast(), "et_b200/_binding.so is missing: run `python et_b200/build.py`"


@pytest.fixture(params=["checked in C++", "checked in Python"])
def both_ways(request, et, monkeypatch):
    """What a call gives does not depend on who looks at its arguments."""
    from et_b200 import ops
    ops._load_fast()
    if request.param == "checked in Python":
        monkeypatch.setattr(ops, "_fast", False)


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *shape, std=1.0):
    return torch.randn(*shape, generator=g, device="cuda") * std


def blocks(n):
    return (n + 127) // 128


def rows_of(x, pitch, shift=0):
    """The same rows as slices of wider ones, whose first starts `shift` elements behind an allocation."""
    wide = torch.full((x.shape[0] * pitch + shift,), 77, dtype=x.dtype, device="cuda") if x.dtype != torch.float8_e4m3fn else torch.zeros(x.shape[0] * pitch + shift, dtype=x.dtype, device="cuda")
    v = wide[shift:].view(x.shape[0], pitch)[:, :x.shape[1]]
    v.copy_(x)
    return v


def within(got, want, bound):
    off = (got.double() - want).abs()
    bad = ~(off <= bound)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {float((off / bound)[bad].max() if bad.any() else 0):.3g} times the bound"


# ------------------------------------------------------------------------------------------------ norm
def spread(scales, width):
    """The scale of every feature of a row."""
    return scales.t().repeat_interleave(128, 1)[:, :width]


# fp32: the sum of squares is off by 2^-24 for each of at most 138 additions in a chain, its root by half of that, and four more roundings: below 2^-17
FP32 = 2.0 ** -17


def check_codes(codes, scales, y):
    """codes and scales against the values y in 64 bits."""
    rows, width = y.shape
    top = torch.nn.functional.pad(y.abs(), (0, -width % 128)).view(rows, -1, 128).amax(-1).t()
    within(scales, top / 448, top / 448 * FP32)
    value = codes.float().double() * spread(scales.double(), width)
    within(value, y, y.abs() * (2.0 ** -4 + 2 * FP32) + spread(scales.double(), width) * (2.0 ** -10 * 1.001))


@pytest.mark.parametrize("rows,width,pitch,shift", [(1, 16, 16, 0), (3, 64, 64, 0), (7, 128, 136, 0), (5, 768, 1024, 8), (64, 1024, 1024, 0), (33, 1040, 1040, 0), (9, 2048, 2056, 0), (4, 4096, 4096, 0),
                                                    (3, 8200, 8208, 0), (2, 16384, 16384, 0), (2, 32768, 32768, 0), (6, 100, 100, 0), (5, 129, 131, 1), (4, 768, 769, 0), (3, 1, 1, 0)])
@pytest.mark.parametrize("codes", [True, False])
@pytest.mark.parametrize("skipped", [True, False])
def test_norm(et, rows, width, pitch, shift, codes, skipped):
    g = gen(rows * 1000 + width)
    x = rows_of((normal(g, rows, width) * torch.exp(0.7 * normal(g, width))).half(), pitch, shift)
    skip = rows_of(normal(g, rows, width, std=0.5).half(), pitch, shift) if skipped else None
    gamma = (1 + 0.1 * normal(g, width)).half()
    residual = rows_of(torch.zeros(rows, width, dtype=torch.float16, device="cuda"), pitch, shift) if skipped else None
    out = rows_of(torch.zeros(rows, width, dtype=torch.float8_e4m3fn if codes else torch.float16, device="cuda"), pitch, shift)
    scales = torch.full((blocks(width), rows), -1.0, device="cuda") if codes else None
    assert et.skip_rmsnorm(out, x, skip, gamma, residual=residual, scales=scales, eps=1e-5) is out
    h = x.double() + (skip.double() if skipped else 0)
    y = h / ((h * h).mean(1, keepdim=True) + 1e-5).sqrt() * gamma.double()
    if codes:
        check_codes(out, scales, y)
    else:
        within(out, y, y.abs() * (HALF + FP32) + TINY)
    if skipped:
        within(residual, h, h.abs() * HALF * 1.001 + TINY)   # (the sum in fp32 first: 2^-24)


@pytest.mark.parametrize("place", ["x", "skip"])
@pytest.mark.parametrize("codes", [True, False])
@pytest.mark.parametrize("width", [1024, 4096, 100])
def test_norm_in_place(both_ways, et, place, codes, width):
    g = gen(width)
    x, skip, gamma = normal(g, 9, width).half(), normal(g, 9, width).half(), normal(g, width).half()
    fresh, scales = torch.zeros_like(x), (torch.zeros(blocks(width), 9, device="cuda") if codes else None)
    out = torch.zeros(9, width, dtype=torch.uint8 if codes else torch.float16, device="cuda")
    et.skip_rmsnorm(out, x, skip, gamma, residual=fresh, scales=scales)
    x2, skip2, out2, scales2 = x.clone(), skip.clone(), torch.zeros_like(out), (torch.zeros_like(scales) if codes else None)
    et.skip_rmsnorm(out2, x2, skip2, gamma, residual=x2 if place == "x" else skip2, scales=scales2)
    assert torch.equal(x2 if place == "x" else skip2, fresh) and torch.equal(out, out2) and (not codes or torch.equal(scales, scales2))
    if not codes:
        x3, skip3 = x.clone(), skip.clone()
        et.skip_rmsnorm(x3 if place == "x" else skip3, x3, skip3, gamma)
        assert torch.equal(x3 if place == "x" else skip3, out)


@pytest.mark.parametrize("rows,width,pitch", [(1, 16, 16), (5, 127, 127), (64, 1024, 1024), (1000, 768, 776), (3, 16400, 16400), (2, 8192, 8192)])
def test_quantise(both_ways, et, rows, width, pitch):
    g = gen(width)
    x = rows_of((normal(g, rows, width) * torch.exp(2 * normal(g, width))).half(), pitch)
    x[0, :64] = 0
    out, scales = torch.zeros(rows, width, dtype=torch.float8_e4m3fn, device="cuda"), torch.zeros(blocks(width), rows, device="cuda")
    et.quantise_rows(out, scales, x)
    check_codes(out, scales, x.double())
    assert (out[0, :64].view(torch.uint8) & 127 == 0).all()


@pytest.mark.parametrize("width", [256, 250])
def test_rows_of_zeros_and_of_what_is_not_finite(et, width):
    x = normal(gen(1), 6, width).half()
    x[1] = 0
    x[2, 5] = float("inf")
    x[3, 200] = float("nan")
    x[4] = 65504.0
    out, scales = torch.zeros(6, width, dtype=torch.float8_e4m3fn, device="cuda"), torch.zeros(2, 6, device="cuda")
    et.quantise_rows(out, scales, x)
    value = out.float() * spread(scales, width)
    assert (value[1] == 0).all() and (scales[:, 1] == 0).all()
    assert value[2, 5].isnan() and (value[2, 128:].isfinite()).all() and value[3, 200].isnan() and (value[3, :128].isfinite()).all()
    assert ((value[4] - 65504.0).abs() < 0.01).all() and value[0].isfinite().all() and value[5].isfinite().all()
    y = torch.zeros(6, width, dtype=torch.float16, device="cuda")
    et.skip_rmsnorm(y, x, None, torch.ones(width, dtype=torch.float16, device="cuda"))
    # (a finite value over an infinite norm is 0, as in the formula)
    assert (y[1] == 0).all() and y[2, 5].isnan() and (y[2, 6:] == 0).all() and y[3].isnan().all() and (y[4] == 1).all() and y[5].isfinite().all()


# ------------------------------------------------------------------------------------------------ linear
class Linear:
    def __init__(self, et, k, n, seed=0, bias=True, gelu=False):
        g = gen(seed + k * 7 + n)
        self.k, self.n, self.gelu = k, n, gelu
        self.codes = (normal(g, n, k) * 60).clamp(-448, 448).to(torch.float8_e4m3fn)
        self.scales = torch.exp(normal(g, blocks(n), blocks(k))) * (0.02 / k ** 0.5)
        self.bias = normal(g, n, std=0.3).half() if bias else None
        self.w = self.codes.double() * self.scales.double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
        self.handle = et.Fp8Weight(k, n, self.codes.view(torch.uint8).cpu().numpy(), self.scales.cpu().numpy(), None if self.bias is None else self.bias.cpu().numpy(), is_gelu=gelu)

    def inputs(self, tokens, seed=1):
        g = gen(seed + tokens)
        return (normal(g, tokens, self.k) * 60).clamp(-448, 448).to(torch.float8_e4m3fn), torch.exp(normal(g, blocks(self.k), tokens)) * 0.02

    def check(self, out, x, x_scales):
        x = x.double() * spread(x_scales.double(), self.k)
        y, size = x @ self.w.t(), x.abs() @ self.w.abs().t()
        if self.bias is not None:
            y, size = y + self.bias.double(), size + self.bias.double().abs()
        # products are exact; 32 of them are added at once, then blocks in fp32 with two roundings of a scale: below 2^-18 of the sum of sizes
        slack = size * 2.0 ** -18
        if self.gelu:
            u = y
            y = torch.nn.functional.gelu(y, approximate="tanh")
            slack = slack * 1.13 + u.abs() / 2 * 2.0 ** -10.9   # its slope is at most 1.13; tanh is good to 2^-10.98
        within(out, y, y.abs() * HALF + TINY + slack)
        self.handle.check()


@pytest.mark.parametrize("k,n", [(16, 16), (128, 128), (144, 48), (768, 768), (1024, 400), (1040, 1024), (4096, 256)])
@pytest.mark.parametrize("tokens", [1, 2, 16, 17, 32, 33, 64, 65, 128, 129, 256, 257, 300, 777])
def test_linear(et, k, n, tokens):
    lin = Linear(et, k, n)
    x, s = lin.inputs(tokens)
    out = torch.full((tokens, n), 7.0, dtype=torch.float16, device="cuda")
    assert lin.handle.run(out, x, s) is out
    lin.check(out, x, s)


@pytest.mark.parametrize("tokens", [1, 40, 100, 300, 5000])
@pytest.mark.parametrize("bias", [True, False])
def test_linear_gelu(both_ways, et, tokens, bias):
    lin = Linear(et, 768, 528, bias=bias, gelu=True)
    x, s = lin.inputs(tokens)
    out = torch.zeros(tokens, 528, dtype=torch.float16, device="cuda")
    lin.handle.run(out, x, s)
    lin.check(out, x, s)
    lin.gelu = False
    lin.handle.run(out, x, s, gelu=False)
    lin.check(out, x, s)


@pytest.mark.parametrize("k,n,tokens", [(4096, 4096, 2100), (768, 2304, 9000), (1024, 1024, 20000), (8192, 128, 64), (20000, 64, 5), (20000, 512, 600)])
def test_linear_large(et, k, n, tokens):
    lin = Linear(et, k, n)
    x, s = lin.inputs(tokens)
    out = torch.zeros(tokens, n, dtype=torch.float16, device="cuda")
    lin.handle.run(out, x, s)
    lin.check(out, x, s)


@pytest.mark.parametrize("tokens", [1, 50, 400])
def test_linear_of_slices(both_ways, et, tokens):
    lin = Linear(et, 272, 176)
    x, s = lin.inputs(tokens)
    wide = torch.full((tokens, 200), 3.0, dtype=torch.float16, device="cuda")
    out = wide[:, :176]
    lin.handle.run(out, rows_of(x, 288, 16), s)
    lin.check(out, x, s)
    assert (wide[:, 176:] == 3).all()


def test_linear_rows_do_not_mix(et):
    """A row that is not finite stays alone, whatever the kernel."""
    lin = Linear(et, 256, 256)
    for tokens in (5, 100, 700):
        x, s = lin.inputs(tokens)
        clean, out = (torch.zeros(tokens, 256, dtype=torch.float16, device="cuda") for _ in range(2))
        lin.handle.run(clean, x, s)
        x.view(torch.uint8)[3, 7] = 0x7f
        s[1, 4] = float("inf")
        lin.handle.run(out, x, s)
        rest = [i for i in range(tokens) if i not in (3, 4)]
        assert out[3].isnan().all() and not out[4].isfinite().any() and torch.equal(out[rest], clean[rest])


def test_linear_refuses(both_ways, et):
    lin = Linear(et, 64, 64)
    x, s = lin.inputs(4)
    out = torch.zeros(4, 64, dtype=torch.float16, device="cuda")
    for args in [(out, x.float().half(), s), (out[:3], x, s), (out, x[:, :32], s), (out, x, s.t()), (out, x, s[:, :3]), (out.float(), x, s), (out, x.cpu(), s)]:
        with pytest.raises(ValueError):
            lin.handle.run(*args)
    with pytest.raises(et.EtError):
        lin.handle.run(out, rows_of(x, 72), s)
    with pytest.raises(et.EtError):
        lin.handle.run(rows_of(out, 68), x, s)
    assert lin.handle.run(torch.zeros(0, 64, dtype=torch.float16, device="cuda"), x[:0], s[:, :0].contiguous()).shape == (0, 64)


# ------------------------------------------------------------------------------------------------ cache
def quantised(x):
    """(codes, scales) of rows in numpy's fp32."""
    x = x.float().cpu().numpy()
    s = (np.abs(x).max(-1, keepdims=True) / np.float32(127)).astype(np.float32)
    with np.errstate(invalid="ignore", divide="ignore"):
        c = np.where(s > 0, np.rint((x / s).astype(np.float32)), 0).astype(np.int8)
    return torch.from_numpy(c).cuda(), torch.from_numpy(s[..., 0]).cuda()


@pytest.mark.parametrize("heads,hd,page,pages,tokens,shift,extra", [(1, 16, 16, 2, 1, 0, 0), (2, 64, 16, 40, 77, 0, 0), (3, 80, 32, 9, 100, 8, 64), (4, 128, 64, 30, 1000, 0, 0), (12, 64, 16, 70, 500, 0, 768),
                                                                    (1, 256, 48, 5, 33, 0, 0), (5, 96, 128, 3, 64, 0, 3), (2, 32, 16, 9, 20, 1, 0)])
def test_cache(both_ways, et, heads, hd, page, pages, tokens, shift, extra):
    g = gen(heads * hd)
    width = heads * hd
    rows = lambda: rows_of((normal(g, tokens, width) * torch.exp(normal(g, tokens, 1))).half(), width + extra, shift)  # noqa: E731
    k, v = rows(), rows()
    k[0, :hd] = 0
    codes = torch.randint(-127, 128, (pages, 2, heads, page, hd), generator=g, device="cuda", dtype=torch.int8)
    scales = torch.rand(pages, 2, heads, page, generator=g, device="cuda")
    want_codes, want_scales = codes.clone(), scales.clone()
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:tokens].int()
    slots[tokens // 2::7] = -1
    if tokens > 3:
        slots[1], slots[2] = pages * page, -2147483648
    real = ((slots >= 0) & (slots < pages * page)).nonzero().flatten()
    at = slots[real].long()
    for side, x in enumerate((k, v)):
        c, s = quantised(x[real].view(-1, heads, hd))
        want_codes[at // page, side, :, at % page] = c
        want_scales[at // page, side, :, at % page] = s
    assert et.kv_cache_write(codes, scales, k, v, slots) == (codes, scales)
    assert torch.equal(codes, want_codes) and torch.equal(scales, want_scales)
    k2, v2 = (rows_of(torch.full((tokens, width), 5.0, dtype=torch.float16, device="cuda"), width + extra, shift) for _ in range(2))
    et.kv_cache_read(k2, v2, codes, scales, slots)
    gone = torch.ones(tokens, dtype=torch.bool, device="cuda")
    gone[real] = False
    for side, x in enumerate((k2, v2)):
        want = (codes[at // page, side, :, at % page].float() * scales[at // page, side, :, at % page, None]).half().flatten(1)
        assert torch.equal(x[real], want) and (x[gone] == 5).all()
    # a value is off by half a step of its row's largest / 127, and by what fp16 rounds
    within(k2[real], k[real].double(), (want_scales[at // page, 0, :, at % page].double() * 0.5001).repeat_interleave(hd, 1) + k[real].double().abs() * HALF * 1.1 + TINY)


def test_cache_rows_that_are_not_finite(et):
    codes, scales = torch.zeros(1, 2, 1, 16, 64, dtype=torch.int8, device="cuda"), torch.zeros(1, 2, 1, 16, device="cuda")
    x = normal(gen(3), 3, 64).half()
    x[1, 3], x[2, 9] = float("inf"), float("nan")
    slots = torch.tensor([4, 0, 9], dtype=torch.int32, device="cuda")
    et.kv_cache_write(codes, scales, x, x, slots)
    k, v = torch.zeros_like(x), torch.zeros_like(x)
    et.kv_cache_read(k, v, codes, scales, slots)
    assert k[0].isfinite().all() and k[1].isnan().all() and k[2].isnan().all() and v[2].isnan().all()


# ------------------------------------------------------------------------------------------------ attention of drafted tokens
class Cache:
    """Sequences of given lengths in pages that lie anywhere, with rows of very different sizes."""

    def __init__(self, lengths, hk, hd, page, seed=0, ratio=1.0, spare=2):
        g = gen(seed)
        counts = [-(-n // page) for n in lengths]
        self.pages, self.page, self.hk, self.hd, self.lengths = sum(counts) + spare, page, hk, hd, lengths
        order = torch.randperm(self.pages, generator=g, device="cuda").int()
        self.table = torch.full((len(lengths), max(counts + [1])), 0, dtype=torch.int32, device="cuda")
        at = 0
        for b, c in enumerate(counts):
            self.table[b, :c] = order[at:at + c]
            at += c
        self.codes = torch.randint(-127, 128, (self.pages, 2, hk, page, hd), generator=g, device="cuda", dtype=torch.int8)
        self.scales = torch.exp(ratio * torch.randn(self.pages, 2, hk, page, generator=g, device="cuda")) / 73
        self.k_lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")

    def rows(self, b, side, head, limit=None):
        """(values, whether the page is there) of a sequence's keys in 64 bits."""
        at = torch.arange(min(self.lengths[b], limit if limit is not None else 1 << 30), device="cuda")
        ids = self.table[b, at // self.page].long()
        there = (ids >= 0) & (ids < self.pages)
        ids = ids.clamp(0, self.pages - 1)
        return self.codes[ids, side, head, at % self.page].double() * self.scales[ids, side, head, at % self.page, None].double(), there


def seen_by(cache, b, n, tree, limit=None):
    """[n, keys] of what a sequence's drafted tokens see; tree: their words, or None."""
    length = cache.lengths[b]
    place = torch.arange(min(length, limit if limit is not None else 1 << 30)) - (length - n)
    rows = []
    for i in range(n):
        word = (int(tree[i]) & (1 << 64) - 1) if tree is not None else (2 << i) - 1
        rows.append([p < 0 or (p < 64 and bool(word >> p & 1)) for p in place.tolist()])
    return torch.tensor(rows, dtype=torch.bool, device="cuda").view(n, len(place))


def check_tree(out, q, cache, counts, tree=None, scale=0.0, limit=None):
    hk, hd = cache.hk, cache.hd
    group = q.shape[1] // hd // hk
    row = 0
    for b, n in enumerate(counts):
        if n == 0:
            continue
        words = None if tree is None else tree[row:row + n].tolist()
        seen = seen_by(cache, b, n, words, limit)
        for h in range(hk):
            (k, there), (v, _) = cache.rows(b, 0, h, limit), cache.rows(b, 1, h, limit)
            can = seen & there
            qq = q[row:row + n].double().view(n, -1, hd)[:, h * group:(h + 1) * group]
            f = scale or hd ** -0.5
            s = torch.einsum("ngf,kf->ngk", qq, k) * f
            size = torch.einsum("ngf,kf->ngk", qq.abs(), k.abs()) * f
            s = s.masked_fill(~can[:, None], -float("inf"))
            p = torch.where(can[:, None], (s - s.amax(-1, keepdim=True)).exp(), 0.0).nan_to_num(0.0) if s.shape[-1] else s
            p = p / p.sum(-1, keepdim=True).clamp_min(1e-300)
            vv = torch.where(there[:, None], v, 0.0)
            want, around = p @ vv, p @ vv.abs()
            # A weight times its value's scale is rounded to fp16: 2^-11 of it, or 2^-25 where the largest is 1 or more. A score is off by 2^-20 of the sum of its terms' sizes (fp32, and
            # factors rounded twice), an exponential by 2^-21 more; both enter the weight and the sum.
            worst = torch.where(can[:, None], size, 0.0).amax(-1, keepdim=True) if s.shape[-1] else torch.zeros(n, group, 1, device="cuda")
            largest = (p * vv.abs().amax(-1)).amax(-1, keepdim=True) if s.shape[-1] else worst
            bound = around * (HALF + 2 * (worst * 2.0 ** -20 + 2.0 ** -21)) + want.abs() * HALF + s.shape[-1] * TINY * largest * 2 + TINY
            within(out[row:row + n].view(n, -1, hd)[:, h * group:(h + 1) * group], want, bound)
        row += n


def random_tree(counts, seed):
    r = np.random.default_rng(seed)
    words = []
    for n in counts:
        bits = []
        for i in range(n):
            parent = int(r.integers(max(-1, i - 5), i))
            bits.append((bits[parent] if parent >= 0 else 0) | 1 << i)
        words += bits
    return torch.tensor([w - (1 << 64) if w >> 63 else w for w in words], dtype=torch.int64, device="cuda")


def queries(counts, hq, hd, seed=5):
    return normal(gen(seed), max(1, sum(counts)), hq * hd).half()[:sum(counts)]


def starts(counts):
    return torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32, device="cuda")


HEADS = [(1, 1, 16), (4, 4, 32), (4, 2, 48), (12, 12, 64), (8, 1, 64), (5, 1, 80), (6, 2, 96), (16, 4, 128), (32, 2, 128), (3, 3, 112), (8, 4, 144), (4, 2, 256)]


@pytest.mark.parametrize("hq,hk,hd", HEADS)
@pytest.mark.parametrize("page", [16, 48, 128])
def test_single_tokens(et, hq, hk, hd, page):
    lengths = [1, 16, 17, 100, 333, 64, 2, 515]
    cache = Cache(lengths, hk, hd, page, seed=hq + hd)
    q = queries([1] * 8, hq, hd)
    out = torch.full_like(q, 9.0)
    assert et.attention_tree(out, q, cache.codes, cache.scales, cache.table, cache.k_lens) is out
    check_tree(out, q, cache, [1] * 8)


@pytest.mark.parametrize("hq,hk,hd", HEADS)
@pytest.mark.parametrize("drafts", [2, 7, 33, 64])
def test_trees(et, hq, hk, hd, drafts):
    lengths = [drafts, drafts + 1, 300, 64 + drafts, 777]
    counts = [drafts] * 5
    cache = Cache(lengths, hk, hd, 32, seed=hq + hd + drafts)
    q, tree = queries(counts, hq, hd), random_tree(counts, drafts)
    out = torch.full_like(q, 9.0)
    et.attention_tree(out, q, cache.codes, cache.scales, cache.table, cache.k_lens, tree=tree, max_q_len=drafts, max_k_len=777)
    check_tree(out, q, cache, counts, tree)


def run_kernel(et, kernel, log_csize, out, q, cache, tree, cu, most, max_k_len=0):
    """attention_tree by one of its kernels (0: few rows, 1: many) with clusters of 2^log_csize."""
    import ctypes
    from et_b200 import ops
    p = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
    batch, width = cache.table.shape
    packed = ops._tree_args(p(out), p(q), p(cache.codes), p(cache.scales), p(cache.table), p(cache.k_lens), p(cu), p(tree), torch.cuda.current_stream().cuda_stream,
                            out.stride(0), q.stride(0), q.shape[1] // cache.hd, cache.hk, cache.hd, batch, q.shape[0], most, max_k_len or width * cache.page, cache.pages, cache.page, width, 0.0)
    et.check(et.lib().et_debug_attention_tree(ctypes.create_string_buffer(packed, len(packed)), kernel, log_csize))


@pytest.mark.parametrize("kernel", [0, 1])
@pytest.mark.parametrize("log_csize", [0, 1, 2, 3, 4])
@pytest.mark.parametrize("hq,hk,hd,most", [(2, 2, 16, 5), (6, 2, 32, 21), (8, 1, 48, 17), (4, 4, 64, 40), (8, 2, 80, 9), (4, 1, 96, 64), (3, 3, 112, 1), (8, 2, 128, 33), (2, 1, 256, 20)])
def test_each_kernel_with_every_cluster(et, kernel, log_csize, hq, hk, hd, most):
    if kernel == 1 and hd > 128:
        return
    counts = [most, 1, 0, (most + 1) // 2, most]
    lengths = [700 + most, 1, 40, most, 2 * most + 63]
    cache = Cache(lengths, hk, hd, 48, seed=hd)
    cache.table[4, 0] = -7
    q, tree = queries(counts + [2], hq, hd) * 2, random_tree(counts + [2], 2)
    out = torch.full_like(q, 9.0)
    run_kernel(et, kernel, log_csize, out, q, cache, tree, starts(counts), most)
    assert (out[sum(counts):] == 9).all()
    check_tree(out[:sum(counts)], q[:sum(counts)], cache, counts, tree[:sum(counts)])
    again = torch.zeros_like(q)
    run_kernel(et, kernel, log_csize, again, q, cache, tree, starts(counts), most)
    assert torch.equal(again[:sum(counts)], out[:sum(counts)])
    # what is not seen, in this kernel and cluster: anything, and a value that is not finite for those that see it
    used = torch.zeros(cache.pages, cache.page, dtype=torch.bool, device="cuda")
    for b, n in enumerate(lengths):
        at = torch.arange(n, device="cuda")
        ids = cache.table[b, at // 48].long()
        used[ids.clamp(0), at % 48] |= ids >= 0
    cache.scales.masked_fill_(~used[:, None, None], float("nan"))
    run_kernel(et, kernel, log_csize, again, q, cache, tree, starts(counts), most)
    assert torch.equal(again[:sum(counts)], out[:sum(counts)])
    page = int(cache.table[0, 10])     # key 500 of the first sequence, which all its tokens see
    cache.scales[page, 1, :, 500 - 480] = float("inf")
    run_kernel(et, kernel, log_csize, again, q, cache, tree, starts(counts), most)
    assert not again[:most].isfinite().any() and torch.equal(again[most:sum(counts)], out[most:sum(counts)])
    et.attention_check()


@pytest.mark.parametrize("hq,hk,hd", [(12, 12, 64), (16, 4, 128), (8, 1, 80)])
@pytest.mark.parametrize("tree", [True, False])
def test_ragged(both_ways, et, hq, hk, hd, tree):
    counts = [5, 0, 1, 40, 64, 3, 17]
    lengths = [200, 30, 1, 41, 64, 2000, 90]
    cache = Cache(lengths, hk, hd, 16, seed=3)
    q = queries(counts + [4], hq, hd)          # four rows behind the last sequence
    words = random_tree(counts + [4], 8) if tree else None
    out = torch.full_like(q, 9.0)
    et.attention_tree(out, q, cache.codes, cache.scales, cache.table, cache.k_lens, tree=words, cu_seqlens=starts(counts), max_q_len=64)
    assert (out[sum(counts):] == 9).all()
    check_tree(out[:sum(counts)], q[:sum(counts)], cache, counts, None if words is None else words[:sum(counts)])


@pytest.mark.parametrize("hq,hk,hd", [(12, 12, 64), (16, 4, 128), (32, 4, 128)])
@pytest.mark.parametrize("drafts", [1, 8, 48])
def test_long_contexts(et, hq, hk, hd, drafts):
    lengths = [5000, 9001, 333]
    counts = [drafts] * 3
    cache = Cache(lengths, hk, hd, 64, seed=9)
    q, tree = queries(counts, hq, hd) * 2, random_tree(counts, 1) if drafts > 1 else None
    out = torch.zeros_like(q)
    et.attention_tree(out, q, cache.codes, cache.scales, cache.table, cache.k_lens, tree=tree, max_q_len=drafts, max_k_len=9001, scale=0.11)
    check_tree(out, q, cache, counts, tree, scale=0.11)


@pytest.mark.parametrize("batch", [40, 200])
def test_many_sequences(et, batch):
    r = np.random.default_rng(batch)
    lengths = [int(v) for v in r.integers(1, 700, batch)]
    counts = [min(n, 3) for n in lengths]
    cache = Cache(lengths, 2, 64, 16, seed=batch)
    q = queries(counts, 8, 64)
    out = torch.zeros_like(q)
    et.attention_tree(out, q, cache.codes, cache.scales, cache.table, cache.k_lens, cu_seqlens=starts(counts), max_q_len=3, max_k_len=700)
    check_tree(out, q, cache, counts)


@pytest.mark.parametrize("drafts,hq,hk,hd", [(1, 4, 4, 64), (1, 8, 2, 128), (40, 8, 2, 128), (33, 4, 4, 64)])
def test_scales_of_very_different_sizes(et, drafts, hq, hk, hd):
    """Values' scales over 40 powers of two: a key with a large weight and a tiny value keeps its precision."""
    lengths, counts = [900, 130], [drafts, drafts]
    cache = Cache(lengths, hk, hd, 16, seed=2)
    cache.scales[:, 1] = torch.exp2(torch.randint(-30, 9, cache.scales[:, 1].shape, generator=gen(4), device="cuda").float())
    cache.scales[:, 1, :, ::5] = 0
    q = queries(counts, hq, hd) * 6
    out = torch.zeros_like(q)
    et.attention_tree(out, q, cache.codes, cache.scales, cache.table, cache.k_lens, max_q_len=drafts)
    check_tree(out, q, cache, counts)
    # one key that all weight lies on, whose value is tiny beside the others'
    cache = Cache(lengths, hk, hd, 16, seed=2, ratio=0.0)
    cache.scales[:, 1] *= 64
    page, head0 = int(cache.table[0, 3]), 0
    cache.codes[page, 0, :, 5] = 0
    q = queries(counts, hq, hd)
    cache.codes[page, 0, head0, 5] = (q[0, :hd].float().sign() * 127).to(torch.int8)
    cache.scales[page, 0, head0, 5] = 40.0 / 127 / float(q[0, :hd].float().abs().mean()) / hd ** 0.5 * 1.0
    cache.scales[page, 1, head0, 5] = 2.0 ** -12
    et.attention_tree(out, q, cache.codes, cache.scales, cache.table, cache.k_lens, max_q_len=drafts)
    check_tree(out, q, cache, counts)


@pytest.mark.parametrize("drafts,hq,hk,hd", [(1, 4, 4, 64), (5, 8, 2, 128), (40, 8, 2, 128), (33, 4, 4, 64), (2, 4, 4, 256)])
def test_what_is_not_seen_takes_no_part(et, drafts, hq, hk, hd):
    lengths, counts = [100, 65 + drafts], [drafts, drafts]
    cache = Cache(lengths, hk, hd, 32, seed=6)
    q, tree = queries(counts, hq, hd), random_tree(counts, 3)
    args = lambda: (cache.codes, cache.scales, cache.table, cache.k_lens)  # noqa: E731
    clean, out = torch.zeros_like(q), torch.zeros_like(q)
    et.attention_tree(clean, q, *args(), tree=tree, max_q_len=drafts)
    # rows behind the last key and pages of nobody
    used = torch.zeros(cache.pages, cache.page, dtype=torch.bool, device="cuda")
    for b, n in enumerate(lengths):
        at = torch.arange(n, device="cuda")
        used[cache.table[b, at // 32].long(), at % 32] = True
    for bad in (float("nan"), float("inf")):
        cache.scales.masked_fill_(~used[:, None, None], bad)
        et.attention_tree(out, q, *args(), tree=tree, max_q_len=drafts)
        assert torch.equal(out, clean)
    if drafts > 1:   # a drafted token that only some see
        at = lengths[0] - drafts + drafts // 2
        page = int(cache.table[0, at // 32])
        for side, bad in ((1, float("inf")), (0, float("nan")), (1, float("nan"))):
            keep = cache.scales[page, side, :, at % 32].clone()
            cache.scales[page, side, :, at % 32] = bad
            et.attention_tree(out, q, *args(), tree=tree, max_q_len=drafts)
            cache.scales[page, side, :, at % 32] = keep
            sees = torch.tensor([bool(int(w) >> (drafts // 2) & 1) for w in tree[:drafts].tolist()], device="cuda")
            sees = torch.cat([sees, torch.zeros(drafts, dtype=torch.bool, device="cuda")])
            assert sees.any() and not out[sees].isfinite().any() and torch.equal(out[~sees], clean[~sees])


@pytest.mark.parametrize("drafts,hq,hk,hd", [(3, 4, 4, 64), (40, 8, 2, 128)])
def test_rows_that_see_nothing(et, drafts, hq, hk, hd):
    lengths, counts = [drafts, 50, 0], [drafts, drafts, drafts]
    cache = Cache(lengths, hk, hd, 16, seed=6)
    q, tree = queries(counts, hq, hd), random_tree(counts, 3)
    tree[1], tree[2] = 0, 1
    out = torch.full_like(q, 9.0)
    et.attention_tree(out, q, cache.codes, cache.scales, cache.table, cache.k_lens, tree=tree, max_q_len=drafts)
    assert (out[1] == 0).all() and (out[2 * drafts:] == 0).all() and (out[2] != 0).any()
    check_tree(out[:2 * drafts], q[:2 * drafts], cache, counts[:2], tree[:2 * drafts])


@pytest.mark.parametrize("drafts,hq,hk,hd", [(1, 4, 4, 64), (5, 8, 2, 128), (40, 8, 2, 128), (33, 4, 4, 64)])
def test_pages_that_there_are_not(et, drafts, hq, hk, hd):
    lengths, counts = [300, 200], [drafts, drafts]
    cache = Cache(lengths, hk, hd, 16, seed=8)
    cache.table[0, 2], cache.table[0, 7], cache.table[1, 0], cache.table[1, 5] = -1, cache.pages, -2147483648, 2147483647
    q = queries(counts, hq, hd)
    out = torch.zeros_like(q)
    et.attention_tree(out, q, cache.codes, cache.scales, cache.table, cache.k_lens, max_q_len=drafts)
    check_tree(out, q, cache, counts)


@pytest.mark.parametrize("drafts", [1, 40])
def test_keys_beyond_a_limit(both_ways, et, drafts):
    lengths, counts = [300, 200], [drafts, drafts]
    cache = Cache(lengths, 2, 64, 16, seed=8)
    q = queries(counts, 8, 64)
    out = torch.zeros_like(q)
    et.attention_tree(out, q, cache.codes, cache.scales, cache.table, cache.k_lens, max_q_len=drafts, max_k_len=150)
    check_tree(out, q, cache, counts, limit=150)
    narrow = cache.table[:, :7].contiguous()
    et.attention_tree(out, q, cache.codes, cache.scales, narrow, cache.k_lens, max_q_len=drafts)
    check_tree(out, q, cache, counts, limit=112)


@pytest.mark.parametrize("drafts,hq,hk,hd", [(1, 4, 4, 64), (40, 8, 2, 128)])
def test_queries_that_are_not_finite(et, drafts, hq, hk, hd):
    lengths, counts = [90, 70], [drafts, drafts]
    cache = Cache(lengths, hk, hd, 16, seed=8)
    q = queries(counts, hq, hd)
    clean, out = torch.zeros_like(q), torch.zeros_like(q)
    et.attention_tree(clean, q, cache.codes, cache.scales, cache.table, cache.k_lens, max_q_len=drafts)
    q[0, 3], q[0, hd + 1], q[0, 2 * hd] = float("nan"), float("inf"), -float("inf")
    et.attention_tree(out, q, cache.codes, cache.scales, cache.table, cache.k_lens, max_q_len=drafts)
    assert out[0, :3 * hd].isnan().all() and torch.equal(out[0, 3 * hd:], clean[0, 3 * hd:]) and torch.equal(out[1:], clean[1:])


def test_tree_of_slices(both_ways, et):
    for drafts, hq, hk, hd in ((1, 4, 4, 64), (5, 8, 2, 128), (40, 8, 2, 128)):
        counts = [drafts] * 3
        cache = Cache([64, 65, 400], hk, hd, 16, seed=8)
        q = rows_of(queries(counts, hq, hd), hq * hd + 72, 8)
        wide = torch.full((3 * drafts, hq * hd + 8), 3.0, dtype=torch.float16, device="cuda")
        et.attention_tree(wide[:, :hq * hd], q, cache.codes, cache.scales, cache.table, cache.k_lens, max_q_len=drafts)
        check_tree(wide[:, :hq * hd], q, cache, counts)
        assert (wide[:, hq * hd:] == 3).all()


def test_offsets_beyond_32_bits(et):
    """A cache of more than 2^31 codes (and, in another head, beyond 2^32 bytes) whose last pages are read and written."""
    hk, hd, page = 8, 128, 64
    pages = 2 ** 32 // (2 * hk * hd * page) + 600
    codes = torch.zeros(pages, 2, hk, page, hd, dtype=torch.int8, device="cuda")
    scales = torch.zeros(pages, 2, hk, page, device="cuda")
    n = 500
    slots = ((pages - 600 + torch.arange(n, device="cuda") // page * 70) * page + torch.arange(n, device="cuda") % page).int()
    k, v = normal(gen(1), n, hk * hd).half(), normal(gen(2), n, hk * hd).half()
    et.kv_cache_write(codes, scales, k, v, slots)
    k2, v2 = torch.zeros_like(k), torch.zeros_like(v)
    et.kv_cache_read(k2, v2, codes, scales, slots)
    assert (k2 - k).abs().max() < 0.03 and (v2 - v).abs().max() < 0.03
    for drafts in (1, 40):
        cache = Cache([n], hk, hd, page)
        cache.codes, cache.scales, cache.pages = codes, scales, pages
        cache.table = (pages - 600 + torch.arange(8, device="cuda") * 70).int().view(1, 8)
        q = queries([drafts], 2 * hk, hd)
        out = torch.zeros_like(q)
        et.attention_tree(out, q, codes, scales, cache.table, cache.k_lens, max_q_len=drafts)
        check_tree(out, q, cache, [drafts])


@pytest.mark.parametrize("drafts", [1, 48])
def test_pages_of_more_than_31_bits(both_ways, et, drafts):
    """One page of 16 million keys: the last ones lie beyond 2^31 codes of their page. The others' scores are 160 below these, so that their weights are 0 even in fp32."""
    hd, group, page, n = 128, 4, (1 << 24) + 64, 64
    codes = torch.zeros(1, 2, 1, page, hd, dtype=torch.int8, device="cuda")
    scales = torch.zeros(1, 2, 1, page, device="cuda")
    k, v = (4 + 0.05 * normal(gen(1), n, hd)).half(), normal(gen(2), n, hd).half()
    et.kv_cache_write(codes, scales, k, v, (page - n + torch.arange(n, device="cuda")).int())
    last = Cache([n], 1, hd, n, spare=0)
    last.codes.copy_(codes[:, :, :, page - n:])
    last.scales.copy_(scales[:, :, :, page - n:])
    k2, v2 = torch.zeros_like(k), torch.zeros_like(v)
    et.kv_cache_read(k2, v2, codes, scales, (page - n + torch.arange(n, device="cuda")).int())
    assert (k2 - k).abs().max() < 0.03 and (v2 - v).abs().max() < 0.03 and codes[:, :, :, :page - n].count_nonzero() == 0
    q = (4 + 0.05 * normal(gen(3), drafts, group * hd)).half()
    out = torch.zeros_like(q)
    table = torch.zeros(1, 128, dtype=torch.int32, device="cuda")   # (of more keys than 31 bits count)
    et.attention_tree(out, q, codes, scales, table, torch.tensor([page], dtype=torch.int32, device="cuda"), max_q_len=drafts)
    check_tree(out, q, last, [drafts])


def test_tree_refuses(both_ways, et):
    cache = Cache([64, 65], 2, 64, 16)
    q = queries([2, 2], 4, 64)
    out = torch.zeros_like(q)
    good = dict(codes=cache.codes, scales=cache.scales, table=cache.table, k_lens=cache.k_lens, max_q_len=2)
    et.attention_tree(out, q, **good)
    for change in (dict(codes=cache.codes.view(torch.uint8)), dict(scales=cache.scales[:, :1]), dict(table=cache.table.long()), dict(k_lens=cache.k_lens[:1]), dict(tree=torch.zeros(3, dtype=torch.int64, device="cuda")),
                   dict(tree=torch.zeros(4, dtype=torch.int32, device="cuda")), dict(cu_seqlens=cache.k_lens), dict(codes=cache.codes.transpose(2, 3)), dict(table=cache.table[:, ::2])):
        with pytest.raises(ValueError):
            et.attention_tree(out, q, **{**good, **change})
    for a, b in ((out[:, :60], q[:, :60]), (out.float(), q), (out[:3], q), (out, q.cpu())):
        with pytest.raises(ValueError):
            et.attention_tree(a, b, **good)
    with pytest.raises(et.EtError):
        et.attention_tree(out, q, **{**good, "max_q_len": 65})
    with pytest.raises(et.EtError):
        et.attention_tree(q, q, **good)


# ------------------------------------------------------------------------------------------------ together
class Layer:
    """Attention's half of a layer in 8 bits and the first linear of its FFN: norm, Q|K|V, cache, attention, rows to codes, output, norm, FFN1."""

    def __init__(self, et, d=256, hq=4, hk=2, hd=64, page=16, pages=40):
        self.et, self.d, self.hq, self.hk, self.hd, self.page = et, d, hq, hk, hd, page
        self.qkv, self.o, self.ffn = Linear(et, d, (hq + 2 * hk) * hd, 1), Linear(et, hq * hd, d, 2), Linear(et, d, 2 * d, 3, gelu=True)
        self.gamma = [(1 + 0.1 * normal(gen(i), d)).half() for i in (1, 2)]
        self.codes, self.scales = torch.zeros(pages, 2, hk, page, hd, dtype=torch.int8, device="cuda"), torch.zeros(pages, 2, hk, page, device="cuda")

    def buffers(self, tokens):
        d, dev = self.d, "cuda"
        f8 = lambda w: (torch.zeros(tokens, w, dtype=torch.float8_e4m3fn, device=dev), torch.zeros(blocks(w), tokens, device=dev))  # noqa: E731
        f16 = lambda w: torch.zeros(tokens, w, dtype=torch.float16, device=dev)  # noqa: E731
        return dict(x8=f8(d), qkv=f16((self.hq + 2 * self.hk) * self.hd), a=f16(self.hq * self.hd), a8=f8(self.hq * self.hd), o=f16(d), h=f16(d), h8=f8(d), f=f16(2 * d))

    def run(self, x, slots, table, k_lens, b, tree=None, cu=None, most=1, stream=None):
        et, at = self.et, self.hq * self.hd
        et.skip_rmsnorm(b["x8"][0], x, None, self.gamma[0], scales=b["x8"][1], stream=stream)
        self.qkv.handle.run(b["qkv"], *b["x8"], stream=stream)
        et.kv_cache_write(self.codes, self.scales, b["qkv"][:, at:at + self.hk * self.hd], b["qkv"][:, at + self.hk * self.hd:], slots, stream=stream)
        et.attention_tree(b["a"], b["qkv"][:, :at], self.codes, self.scales, table, k_lens, tree=tree, cu_seqlens=cu, max_q_len=most, stream=stream)
        et.quantise_rows(*b["a8"], b["a"], stream=stream)
        self.o.handle.run(b["o"], *b["a8"], stream=stream)
        et.skip_rmsnorm(b["h8"][0], b["o"], x, self.gamma[1], residual=b["h"], scales=b["h8"][1], stream=stream)
        self.ffn.handle.run(b["f"], *b["h8"], stream=stream)
        return b["f"], b["h"]

    def plain(self, x, counts, lengths, seen):
        """The layer in 64 bits without any rounding: x of all tokens of all sequences, of which the last counts[b] are asked for."""
        norm = lambda h, g: h / ((h * h).mean(1, keepdim=True) + 1e-6).sqrt() * g.double()  # noqa: E731
        qkv = norm(x.double(), self.gamma[0]) @ self.qkv.w.t() + self.qkv.bias.double()
        at, kv = self.hq * self.hd, self.hk * self.hd
        outs, first = [], 0
        for b, (n, length) in enumerate(zip(counts, lengths)):
            rows = qkv[first:first + length]
            q, k, v = rows[length - n:, :at].view(n, self.hq, self.hd), rows[:, at:at + kv].view(length, self.hk, self.hd), rows[:, at + kv:].view(length, self.hk, self.hd)
            k, v = (t.repeat_interleave(self.hq // self.hk, 1) for t in (k, v))
            s = torch.einsum("qhf,khf->hqk", q, k) * self.hd ** -0.5
            s = s.masked_fill(~seen[b][None], -float("inf"))
            a = torch.einsum("hqk,khf->qhf", torch.softmax(s, -1), v).reshape(n, at)
            h = x[first + length - n:first + length].double() + a @ self.o.w.t() + self.o.bias.double()
            f = norm(h, self.gamma[1]) @ self.ffn.w.t() + self.ffn.bias.double()
            outs.append((torch.nn.functional.gelu(f, approximate="tanh"), h))
            first += length
        return torch.cat([o[0] for o in outs]), torch.cat([o[1] for o in outs])


def test_a_layer_of_them_together(both_ways, et):
    """A prompt goes in a token at a time into the cache, then a tree of drafted tokens: against the layer without roundings. Codes of e4m3 are off by 2^-4 at most, by some 2^-5.5 in the mean square;
    three linears behind one another, each with both operands' roundings averaged over its products, leave a few percent of the results' size."""
    layer = Layer(et)
    lengths, counts = [37, 70], [9, 5]
    x = normal(gen(11), sum(lengths), layer.d).half()
    table = torch.stack([torch.arange(0, 8), torch.arange(8, 16)]).int().cuda()
    place = torch.cat([torch.arange(n) for n in lengths])
    seq = torch.tensor(sum(([b] * n for b, n in enumerate(lengths)), []))
    slots = (table.cpu()[seq, place // 16] * 16 + place % 16).int().cuda()
    drafted = torch.cat([torch.arange(n) >= n - c for n, c in zip(lengths, counts)]).cuda()
    tree = random_tree(counts, 4)
    # the kept tokens: their keys alone are asked for (their own results are not)
    kept = (~drafted).nonzero().flatten()
    kept_lens = torch.tensor([n - c for n, c in zip(lengths, counts)], dtype=torch.int32, device="cuda")
    half = [0, int(kept_lens[0]), len(kept)]
    for b in (0, 1):
        rows = kept[half[b]:half[b + 1]]
        for i in range(0, len(rows), 50):
            part = rows[i:i + 50]
            layer.run(x[part], slots[part], table[b:b + 1], torch.tensor([i + len(part)], dtype=torch.int32, device="cuda"), layer.buffers(len(part)), most=len(part))
    new = drafted.nonzero().flatten()
    b = layer.buffers(len(new))
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    got, h = layer.run(x[new], slots[new], table, lens, b, tree=tree, cu=starts(counts), most=9)
    seen, row = [], 0
    for n, c in zip(lengths, counts):
        words = [int(w) & (1 << 64) - 1 for w in tree[row:row + c].tolist()]
        seen.append(torch.tensor([[j < n - c or bool(w >> (j - n + c) & 1) for j in range(n)] for w in words], device="cuda"))
        row += c
    want, want_h = layer.plain(x, counts, lengths, seen)
    assert (got.double() - want).norm() < 0.1 * want.norm() and (h.double() - want_h).norm() < 0.05 * want_h.norm()
    for w in (layer.qkv, layer.o, layer.ffn):
        w.handle.check()
    et.attention_check()
    first = [t.clone() for t in (got, h, layer.codes, layer.scales)]
    # the same on a stream of its own, and captured and replayed over other inputs and back: the same bits
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    xs, ss, b2 = x[new].clone(), slots[new].clone(), layer.buffers(len(new))
    with torch.cuda.stream(stream):
        again = layer.run(xs, ss, table, lens, b2, tree=tree, cu=starts(counts), most=9)
    stream.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(first, (*again, layer.codes, layer.scales)))
    cu, graph = starts(counts), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer.run(xs, ss, table, lens, b2, tree=tree, cu=cu, most=9)
    keep = xs.clone()
    for t in out:
        t.zero_()
    xs.mul_(0.5)
    graph.replay()
    torch.cuda.synchronize()
    assert not torch.equal(out[0], first[0])
    xs.copy_(keep)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(first, (*out, layer.codes, layer.scales)))


def test_two_streams_at_once(et):
    """The same operators on two streams, over and over, give what each gives alone."""
    layers = [Layer(et), Layer(et)]
    work = []
    for i, layer in enumerate(layers):
        n = 20 + 30 * i
        x = normal(gen(20 + i), n, layer.d).half()
        slots = torch.arange(n, device="cuda").int()
        table = torch.arange(4, device="cuda").int().view(1, 4)
        lens = torch.tensor([n], dtype=torch.int32, device="cuda")
        work.append((x, slots, table, lens, layer.buffers(n), n))
    alone = []
    for layer, (x, slots, table, lens, b, n) in zip(layers, work):
        alone.append([t.clone() for t in layer.run(x, slots, table, lens, b, most=n)])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in layers]
    for _ in range(30):
        for layer, (x, slots, table, lens, b, n), st in zip(layers, work, streams):
            layer.run(x, slots, table, lens, b, most=n, stream=st)
    torch.cuda.synchronize()
    for want, (_, _, _, _, b, _), layer in zip(alone, work, layers):
        assert torch.equal(b["f"], want[0]) and torch.equal(b["h"], want[1])
        for w in (layer.qkv, layer.o, layer.ffn):
            w.handle.check()


def test_norm_refuses(both_ways, et):
    x, gamma = torch.zeros(4, 256, dtype=torch.float16, device="cuda"), torch.ones(256, dtype=torch.float16, device="cuda")
    codes, scales = torch.zeros(4, 256, dtype=torch.uint8, device="cuda"), torch.zeros(2, 4, device="cuda")
    et.skip_rmsnorm(codes, x, None, gamma, scales=scales)
    for args in [(x, x.float(), None, gamma), (x[:3], x, None, gamma), (codes, x, None, gamma), (x, x, x[:, :128], gamma), (x, x, None, gamma[:128]), (x, x, None, gamma.float()), (x, x.t(), None, gamma),
                 (x, x.cpu(), None, gamma)]:
        with pytest.raises(ValueError):
            et.skip_rmsnorm(*args)
    for bad in (scales.t(), scales[:1], scales.half()):
        with pytest.raises(ValueError):
            et.skip_rmsnorm(codes, x, None, gamma, scales=bad)
        with pytest.raises(ValueError):
            et.quantise_rows(codes, bad, x)
    with pytest.raises(et.EtError):
        et.skip_rmsnorm(x.clone(), x, None, gamma, eps=0.0)
    out = x.clone()
    with pytest.raises(et.EtError):
        et.skip_rmsnorm(out, x, None, gamma, residual=out)


def test_cache_refuses_tensors(both_ways, et):
    codes, scales = torch.zeros(2, 2, 3, 16, 32, dtype=torch.int8, device="cuda"), torch.zeros(2, 2, 3, 16, device="cuda")
    k, slots = torch.zeros(5, 96, dtype=torch.float16, device="cuda"), torch.arange(5, dtype=torch.int32, device="cuda")
    et.kv_cache_write(codes, scales, k, k, slots)
    for args in [(codes.view(torch.uint8), scales, k, k, slots), (codes, scales.half(), k, k, slots), (codes, scales[:1], k, k, slots), (codes, scales, k[:, :64], k, slots), (codes, scales, k, k[:4], slots),
                 (codes, scales, k, k, slots.long()), (codes, scales, k, k, slots[:4]), (codes.transpose(3, 4), scales, k, k, slots), (codes, scales, k.cpu(), k, slots)]:
        for call in (lambda c, s, a, b, i: et.kv_cache_write(c, s, a, b, i), lambda c, s, a, b, i: et.kv_cache_read(a, b, c, s, i)):
            with pytest.raises(ValueError):
                call(*args)


def test_other_threads_run_while_a_launch_waits(both_ways, et):
    """A launch that waits for room in the device's queue does not hold Python's lock."""
    import threading
    import time
    x = torch.zeros(1, 128, dtype=torch.float16, device="cuda")
    out, scales = torch.zeros(1, 128, dtype=torch.uint8, device="cuda"), torch.zeros(1, 1, device="cuda")
    et.quantise_rows(out, scales, x)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    begin = time.perf_counter()
    with torch.cuda.stream(stream):
        torch.cuda._sleep(2_000_000_000)      # a second or so

    def launches():
        for _ in range(4000):                 # more than the queue takes
            et.quantise_rows(out, scales, x, stream=stream)

    thread = threading.Thread(target=launches)
    thread.start()
    last, longest = time.perf_counter(), 0.0
    while thread.is_alive():
        time.sleep(0.001)
        now = time.perf_counter()
        longest, last = max(longest, now - last), now
    torch.cuda.synchronize()
    took = time.perf_counter() - begin
    assert longest < 0.5 * took, f"this thread stood still for {longest:.2f} of {took:.2f} s"
