"""More of the operators in 8 bits: what stands before them in a stream, every plan of the linear, codes bit for bit, long caches."""
import ctypes

import numpy as np
import pytest

from tests.test_eight_bits_gpu import HALF, TINY, Cache, Linear, blocks, check_tree, et, gen, normal, queries, rows_of, run_kernel, spread, within  # noqa: F401

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


# ------------------------------------------------------------------------------------------------ behind a long kernel
@pytest.mark.parametrize("k,n,tokens", [(4096, 256, 20), (2048, 1024, 700)])
def test_linear_behind_a_long_kernel(et, k, n, tokens):
    """A linear starts while the kernel before it still runs, here for longer (5 s and more) than a bounded wait lasts (4.2 s). Its waits for the operand may begin only then."""
    lin = Linear(et, k, n)
    x, s = lin.inputs(tokens)
    want, out = (torch.zeros(tokens, n, dtype=torch.float16, device="cuda") for _ in range(2))
    lin.handle.run(want, x, s)
    lin.handle.check()
    cache = Cache([1 << 20], 1, 16, 1 << 20, spare=0)
    cache.table = torch.zeros(1, 2047, dtype=torch.int32, device="cuda")   # (the same page over and over)
    q = queries([1], 1, 16)
    a = torch.zeros_like(q)

    def long(keys):
        cache.k_lens.fill_(keys)
        run_kernel(et, 0, 0, a, q, cache, None, None, 1, keys)             # one CTA

    begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    long(1 << 22)
    begin.record()
    long(1 << 22)
    end.record()
    end.synchronize()
    keys = min(0x7ff00000, int((1 << 22) * 6500 / begin.elapsed_time(end)))
    torch.cuda.synchronize()
    begin.record()
    long(keys)
    lin.handle.run(out, x, s)
    end.record()
    end.synchronize()
    assert begin.elapsed_time(end) > 5000
    lin.handle.check()
    et.attention_check()
    assert torch.equal(out, want)


# ------------------------------------------------------------------------------------------------ GELU
@pytest.mark.parametrize("tokens", [3, 60, 5000])
def test_gelu_far_to_the_left(et, tokens):
    """Results behind -3 keep fp16's digits. Features are whole steps of 2^-6 from -7.5 to 7.5, exact in fp32. The exponent, at most 28 where fp16 has a result, is off by 2^-21.4 of itself (three
    roundings, two constants), so the exponential by 2^-17; the reciprocal is off by 0.051^4 = 2^-17.1 and some roundings."""
    k, n = 64, 960
    values = (torch.arange(n, device="cuda") - 480).double() / 64
    codes = torch.zeros(n, k, dtype=torch.float8_e4m3fn, device="cuda")
    rest = values.clone()
    for i in range(4):   # as sums of e4m3 numbers
        codes[:, i] = rest.float().to(torch.float8_e4m3fn)
        rest -= codes[:, i].double()
    assert (rest == 0).all()
    weight = et.Fp8Weight(k, n, codes.view(torch.uint8).cpu().numpy(), np.ones((blocks(n), 1), np.float32), is_gelu=True)
    x = torch.zeros(tokens, k, dtype=torch.float8_e4m3fn, device="cuda")
    x[:, :4] = 1.0
    out = torch.zeros(tokens, n, dtype=torch.float16, device="cuda")
    weight.run(out, x, torch.ones(1, tokens, device="cuda"))
    want = torch.nn.functional.gelu(values, approximate="tanh").expand(tokens, n)
    within(out, want, want.abs() * (HALF + 2.0 ** -15.9) + TINY)
    # far out: nothing is left, or all of it
    weight.run(out, x, torch.full((1, tokens), 2.0 ** 10, device="cuda"))
    assert (out[:, :470] == 0).all() and torch.equal(out[:, 490:].double(), (values[490:] * 1024).half().double().expand(tokens, -1))
    weight.check()


# ------------------------------------------------------------------------------------------------ codes
@pytest.mark.parametrize("rows,width", [(4096, 1024), (1024, 1000), (333, 250), (60000, 128)])
def test_codes_are_those_of_the_quotient(et, rows, width):
    """code = e4m3(x / scale), scale = largest / 448, with fp32's rounded quotients: bit for bit, ties among them."""
    g = gen(width)
    x = (normal(g, rows, width) * torch.exp(3 * normal(g, rows, 1))).clamp(-60000, 60000).half()
    x[::3] = (x[::3] * 16).round().clamp(-60000, 60000)          # whole numbers: quotients meet the middles between codes often
    x[5] = torch.arange(width, device="cuda").half() * 2.0 ** -24  # below fp16's normal numbers
    x[6] = 0
    out, scales = torch.zeros(rows, width, dtype=torch.float8_e4m3fn, device="cuda"), torch.zeros(blocks(width), rows, device="cuda")
    et.quantise_rows(out, scales, x)
    top = torch.nn.functional.pad(x.float().abs(), (0, -width % 128)).view(rows, -1, 128).amax(-1).t()
    assert torch.equal(scales, top / torch.full_like(top, 448))   # (torch divides by a number as it multiplies by its reciprocal)
    s = spread(scales, width)
    want = torch.where(s > 0, x.float() / s, torch.zeros_like(s)).to(torch.float8_e4m3fn)
    assert torch.equal(out.float(), want.float())   # (of zeros either sign)


def test_codes_of_every_number(et):
    """Each of fp16's numbers under scales of all sizes that it is not above."""
    numbers = torch.arange(0, 0x7c00, device="cuda", dtype=torch.int32).to(torch.int16).view(torch.float16)
    for top in (1.0, 447.0, 449.0, 5.0, 7.0, 0.3, 65504.0, 1.375, 2047.0, 3.0):
        some = numbers[numbers <= top]
        some = torch.nn.functional.pad(some, (0, -len(some) % 127)).view(-1, 127)
        x = torch.cat([torch.full((len(some), 1), top, dtype=torch.float16, device="cuda"), some], 1)
        out, scales = torch.zeros(x.shape, dtype=torch.float8_e4m3fn, device="cuda"), torch.zeros(1, len(x), device="cuda")
        et.quantise_rows(out, scales, x)
        assert torch.equal(out.float(), (x.float() / scales[0][:, None]).to(torch.float8_e4m3fn).float())


# ------------------------------------------------------------------------------------------------ long caches
@pytest.mark.parametrize("kernel", [0, 1])
@pytest.mark.parametrize("hd", [64, 128])
def test_many_small_weights_beside_large_ones(et, kernel, hd):
    """Keys whose weights are 2^-25.4 of those of four (one for each warp that has a reference of its own), whose values are large in one feature and 0 in the others: there the small ones are all of
    the result, although each is below half of fp16's smallest step beside 1."""
    n, page = 60000, 64
    cache = Cache([n], 1, hd, page, spare=0, ratio=0.0)
    cache.codes[:, 0], cache.codes[:, 1] = 0, 100
    cache.scales[:, 0], cache.scales[:, 1] = 1.0, 2.0 ** -7
    first = int(cache.table[0, 0])
    cache.codes[first, 0, 0, ::16], cache.codes[first, 1, 0, ::16] = 1, 0
    cache.codes[first, 1, 0, ::16, 7] = -127
    cache.scales[first, 0, 0, ::16] = 25.4 * np.log(2.0) / hd ** 0.5       # with q = 1: the score is 25.4 log 2
    q = torch.ones(3, 2 * hd, dtype=torch.float16, device="cuda")
    out = torch.zeros_like(q)
    run_kernel(et, kernel, 0, out, q, cache, None, None, 3)
    et.attention_check()
    for i in range(3):
        small, v = (n - 6 + i) * 2.0 ** -25.4, torch.full((hd,), 100 / 128, dtype=torch.float64, device="cuda")
        want, lost = v * small / (small + 4), v * (n * 2.0 ** -32) / 4
        want[7] = (100 / 128 * small - 127 / 128 * 4) / (small + 4)
        # rounded once, and each weight by half a step, which is 2^-11 of it or 2^-32 of the largest
        within(out[i].view(2, hd), want, want.abs() * (2 * HALF) + lost + TINY)


# ------------------------------------------------------------------------------------------------ every plan of the linear
def run_plan(et, plan, lin, out, x, s, gelu=False):
    """The linear by one of its plans: (features of a pair's tile, 0, 0), or (0, tokens of a tile, log2 of the CTAs that share its K)."""
    from et_b200 import ops
    packed = ops._fp8_args(lin.handle._h.value, out.data_ptr(), x.data_ptr(), s.data_ptr(), torch.cuda.current_stream().cuda_stream, out.stride(0), x.stride(0), x.shape[0], 1 if gelu else 0)
    et.check(et.lib().et_debug_fp8_linear(ctypes.create_string_buffer(packed, len(packed)), *plan))


PLANS = [(128, 0, 0), (256, 0, 0)] + [(0, tokens, log) for tokens in (16, 32, 64, 128) for log in range(4) if tokens >> log >= 4]


def checked(et, plan, lin, tokens, gelu):
    """One call, X and Y as slices of wider rows: against 64 bits, nothing beside the slices, the same bits again."""
    x, s = lin.inputs(tokens)
    x = rows_of(x, lin.k + 48, 16)
    wide = torch.full((tokens, lin.n + 24), 3.0, dtype=torch.float16, device="cuda")
    out = wide[:, :lin.n]
    run_plan(et, plan, lin, out, x, s, gelu)
    lin.gelu = gelu
    lin.check(out, x, s)
    assert (wide[:, lin.n:] == 3).all()
    again = torch.zeros_like(out)
    run_plan(et, plan, lin, again, x, s, gelu)
    assert torch.equal(again, out)
    return x, s, out


@pytest.mark.parametrize("gelu", [False, True])
@pytest.mark.parametrize("plan", PLANS)
@pytest.mark.parametrize("k,n,tokens", [(1040, 400, 1), (1024, 272, 130), (1168, 144, 61), (2192, 16, 257)])
def test_every_plan(et, plan, gelu, k, n, tokens):
    """Features, tokens and K that fill no tile. (K of 8 blocks and more: as many as the widest split.)"""
    checked(et, plan, Linear(et, k, n), tokens, gelu)


@pytest.mark.parametrize("gelu", [False, True])
@pytest.mark.parametrize("plan", PLANS)
def test_every_plan_with_more_tiles_than_places(et, plan, gelu):
    """Several tiles to a pair (of odd numbers of blocks, so that rings and places go on where the tile before left them), and more CTAs than SMs."""
    k, n, tokens = (1040, 2960, 2500) if plan[0] else (1040, 2960, 900)
    checked(et, plan, Linear(et, k, n), tokens, gelu)


@pytest.mark.parametrize("plan", PLANS)
def test_long_k_by_every_plan(et, plan):
    """More blocks to a CTA than its scales' buffer (16) and its rings hold."""
    checked(et, plan, Linear(et, 6416, 144), 70, False)


@pytest.mark.parametrize("plan", PLANS)
def test_a_row_that_is_not_finite_stays_alone_by_every_plan(et, plan):
    lin = Linear(et, 1040, 272)
    x, s, clean = checked(et, plan, lin, 300, False)
    x.view(torch.uint8)[3, 7] = 0x7f
    s[1, 4] = float("inf")
    s[8, 299] = float("nan")
    out = torch.zeros_like(clean)
    run_plan(et, plan, lin, out, x, s)
    rest = [i for i in range(300) if i not in (3, 4, 299)]
    assert out[3].isnan().all() and not out[4].isfinite().any() and out[299].isnan().all() and torch.equal(out[rest], clean[rest])
