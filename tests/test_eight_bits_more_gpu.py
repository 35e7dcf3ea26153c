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
    """A linear starts while the kernel before it still runs, here for longer (6 s and more) than a bounded wait lasts (4.2 s). Its waits for the operand may begin only then."""
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
    assert begin.elapsed_time(end) > 6000
    lin.handle.check()
    et.attention_check()
    assert torch.equal(out, want)
