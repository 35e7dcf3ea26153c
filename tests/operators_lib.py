"""Plain 64-bit forms of the operators for positions, adapters and rules on scores, with the bounds that go with them."""
import math

import torch

HALF = 2.0 ** -11   # half a step of fp16, relative


def rotary(x, positions, inv_freq, axis, head_dim, interleaved):
    """[tokens, heads * head_dim] turned, in 64 bits."""
    x = x.double().reshape(x.shape[0], -1, head_dim)
    pairs = inv_freq.shape[0]
    known = (axis >= 0) & (axis < positions.shape[1])
    angle = torch.where(known, positions[:, axis.clamp(0, positions.shape[1] - 1).long()].double() * inv_freq.double(), 0.0)[:, None]
    i = torch.arange(pairs, device=x.device)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + pairs)
    out = x.clone()
    out[..., a] = x[..., a] * angle.cos() - x[..., b] * angle.sin()
    out[..., b] = x[..., a] * angle.sin() + x[..., b] * angle.cos()
    return out.flatten(1)


def adapter(base, x, cu, ids, slots):
    """(base + scale B (A x), the bound of its error). slots: {id: (A, B, scale)}.

    The bound: half a step of the result; A x rounded to fp16, each value by at most half a step of itself or, far below the row's largest, by a
    2^-25 of it (a row is scaled to [1, 2)); fp32 sums of K and of rank products."""
    out = base.double().clone()
    bound = torch.zeros_like(out)
    for b, i in enumerate(ids):
        if i not in slots:
            continue
        A, B, scale = slots[i]
        rows = slice(cu[b], cu[b + 1])
        xr, A, B = x[rows].double(), A.double(), B.double()
        low = xr @ A.t()
        size = xr.abs() @ A.abs().t()
        k, r = A.shape[1], A.shape[0]
        low_err = HALF * low.abs() + 2.0 ** -25 * low.abs().amax(1, keepdim=True) + k * 2.0 ** -24 * size
        out[rows] += scale * (low @ B.t())
        bound[rows] = abs(scale) * ((low_err + (r + 2) * 2.0 ** -24 * low.abs()) @ B.abs().t())
    return out, bound + HALF * out.abs() * (1 + 2.0 ** -10) + 2.0 ** -25


def attention(Q, K, V, head_dim, seqs, scale=None, cap=0.0, slopes=None, table=None, window=(-1, -1), prefixes=None, q_docs=None, k_docs=None):
    """(result, bound) in 64 bits. seqs: (first query row, queries, first key row, keys, position of the first query) of each sequence; rows in no
    sequence are not a number. What a query does not see takes no part, whatever it holds; a query that sees something that is not finite has bound infinity.

    The bound, of a result sum p v: the weights are rounded to fp16 (half a step, or 2^-25 of the reference weight 1 when far below it) after exponentials
    with a relative error of 2^-20 at most, of scores with fp32 errors (head_dim products, then the cap's exponential and quotient, an
    absolute error of some 2^-21 of the cap, then the bias); the result is rounded to fp16."""
    hd = head_dim
    H, Hk = Q.shape[1] // hd, K.shape[1] // hd
    scale = hd ** -0.5 if scale is None else scale
    out = torch.full(Q.shape, math.nan, dtype=torch.float64, device=Q.device)
    bound = torch.zeros_like(out)
    for b, (q0, nq, k0, nk, at) in enumerate(seqs):
        if nq == 0:
            continue
        q = Q[q0:q0 + nq].double().view(nq, H, hd).permute(1, 0, 2)
        k = K[k0:k0 + nk].double().view(nk, Hk, hd).permute(1, 0, 2).repeat_interleave(H // Hk, 0)
        v = V[k0:k0 + nk].double().view(nk, Hk, hd).permute(1, 0, 2).repeat_interleave(H // Hk, 0)
        odd = ~(torch.isfinite(k).all(-1) & torch.isfinite(v).all(-1))   # [H, nk]
        k, v = torch.where(torch.isfinite(k), k, 0.0), torch.where(torch.isfinite(v), v, 0.0)
        key = torch.arange(nk, device=Q.device)
        away = key[None] - (torch.arange(nq, device=Q.device) + at)[:, None]
        seen = torch.ones_like(away, dtype=torch.bool)
        if window[0] >= 0:
            seen &= away >= -window[0]
        if window[1] >= 0:
            seen &= away <= window[1]
        if prefixes is not None:
            seen |= (key < prefixes[b])[None]
        if q_docs is not None:
            seen &= (q_docs[q0:q0 + nq, None] == k_docs[None, k0:k0 + nk]) & (q_docs[q0:q0 + nq, None] >= 0)
        s = q @ k.transpose(1, 2) * scale
        err = hd * 2.0 ** -24 * (q.abs() @ k.abs().transpose(1, 2)) * scale + 2.0 ** -22 * s.abs()
        if cap:
            s = cap * torch.tanh(s / cap)
            err = err + 2.0 ** -21 * cap
        if slopes is not None:
            bias = slopes.double()[:, None, None] * away.abs()
            s = s - bias
            err = err + 2.0 ** -22 * bias.abs()
        if table is not None:
            reach = table.shape[1] // 2
            bias = table.double()[:, away.clamp(-reach, reach) + reach]
            s = s + bias
            err = err + 2.0 ** -22 * bias.abs()
        s = s.masked_fill(~seen, -math.inf)
        top = s.amax(-1, keepdim=True) if nk else torch.full((H, nq, 1), -math.inf, device=Q.device, dtype=torch.float64)
        p = torch.exp(s - torch.where(torch.isinf(top), 0.0, top))
        total = p.sum(-1, keepdim=True)
        p = p / torch.where(total > 0, total, 1.0)
        err = err + 2.0 ** -22 * torch.where(seen, (top - s).clamp(min=0), 0.0)   # the difference to the maximum is rounded too
        e = torch.where(seen, HALF + 2.0 ** -20 + err, 0.0)
        o = p @ v
        # weights and their sum are both off: the sum's error moves the whole result
        bd = (p * e) @ v.abs() + (p * (e - HALF).clamp(min=0)).sum(-1, keepdim=True) * o.abs()
        tiny = seen.double() @ v.abs() * 2.0 ** -25 / torch.where(total > 0, total, 1.0)
        bd = bd + tiny + HALF * o.abs() + 2.0 ** -25
        bd = torch.where((seen[None] & odd[:, None]).any(-1, keepdim=True), math.inf, bd)
        out[q0:q0 + nq] = o.permute(1, 0, 2).reshape(nq, H * hd)
        bound[q0:q0 + nq] = bd.permute(1, 0, 2).reshape(nq, H * hd)
    return out, bound


def assert_within(got, want, bound, what=""):
    """Every element within its bound; where that is infinite the result may be anything; rows that are in no sequence (want not a number) are not looked at."""
    got, look = got.double(), ~torch.isnan(want) & ~torch.isinf(bound)
    d = torch.where(look, (got - want).abs(), torch.zeros_like(want))
    bad = look & ~(d <= bound)
    if bad.any():
        at = torch.nonzero(bad)[0].tolist()
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} beyond their bound, first at {at}: {got[tuple(at)].item()} for {want[tuple(at)].item()} "
                             f"(bound {bound[tuple(at)].item():.3g})")
