"""Plain 64-bit forms of the batch operators over a paged cache and the tolerances of their tests.

Everything here runs on the CPU in float64, from the definitions in include/genllm_paged.h."""
import math

import torch

from hybrid import half_step

PAGE = 16


def e4m3(x):
    """x rounded to four significant bits (steps of 2^-9 below 2^-6), ties to even, by integers of the step; NaN for
    what is not finite."""
    _, e = torch.frexp(x)
    unit = torch.ldexp(torch.ones_like(x), (e - 1).clamp(min=-6) - 3)
    return torch.where(torch.isfinite(x), torch.round(x / unit) * unit, torch.nan)


def exponent(top):
    """The least e from -100 on with top <= 448 * 2^e."""
    e = -100
    while top > math.ldexp(448.0, e):
        e += 1
    return e


def values(pool, scales):
    """A pool [n, 16, H, D] of codes and its E8M0 bytes [n, H], as numbers."""
    e = scales.cpu().view(torch.uint8).double() - 127
    two = torch.where(e == 128, torch.nan, torch.ldexp(torch.ones_like(e), e.int()))
    return pool.cpu().view(torch.float8_e4m3fn).double() * two[:, None, :, None]


def scatter(x, pool, scales, ids, start, lens=None):
    """What writing x [B, S, H, D] makes of the codes (float64) and exponents of a pool, both on the CPU, in place."""
    B, S, H, D = x.shape
    x = x.cpu().double()
    for b in range(B):
        n = S if lens is None else min(max(int(lens[b]), 0), S)
        at = int(start[b])
        if at < 0:
            continue
        for page in range(at // PAGE, (at + n + PAGE - 1) // PAGE if n else at // PAGE):
            if page >= ids.shape[1] or not 0 <= int(ids[b, page]) < pool.shape[0]:
                continue
            block = int(ids[b, page])
            lo, hi = max(at, page * PAGE), min(at + n, (page + 1) * PAGE)
            new = slice(lo - page * PAGE, hi - page * PAGE)
            for h in range(H):
                y = x[b, lo - at : hi - at, h]
                had = int(scales[block, h])
                fine = y[torch.isfinite(y)].abs()
                e = exponent(float(fine.max()) if fine.numel() else 0.0)
                if new.start > 0:
                    e = max(e, had)
                    rest = [i for i in range(PAGE) if not new.start <= i < new.stop]
                    pool[block, rest, h] = e4m3(pool[block, rest, h] * 2.0 ** (had - e))
                pool[block, new, h] = e4m3(y / 2.0 ** e)
                scales[block, h] = e


def rows(table, ids, n, H, D):
    """Tokens 0..n-1 of a sequence from a pool's values [blocks, 16, H, D]; NaN where an id is none."""
    out = torch.full((n, H, D), torch.nan, dtype=torch.float64)
    for page in range(-(-n // PAGE)):
        block = int(ids[page])
        if 0 <= block < table.shape[0]:
            out[page * PAGE : (page + 1) * PAGE] = table[block][: n - page * PAGE]
    return out


def attend(q, k, v, pos, scale, causal=True, window=None, sinks=0):
    """One sequence: q [ql, Hq, D] at positions pos.., k and v [n, H, D].  Returns o, sum_t w_t |v_t|, sum_t |v_t| and
    the largest sum_d |q_d k_d| scale of a row, [ql, Hq, ...], in float64."""
    ql, Hq, D = q.shape
    n, H, _ = k.shape
    q = q.cpu().double()
    out, weight, plain = (torch.zeros(ql, Hq, D).double() for _ in range(3))
    size = torch.zeros(ql, Hq, 1).double()
    t = torch.arange(n)
    for i in range(ql):
        p = pos + i
        see = (t <= p) if causal else torch.ones(n, dtype=torch.bool)
        if window is not None:
            see &= (t > p - window) | (t < sinks)
        if not bool(see.any()):
            continue
        for h in range(Hq):
            kk, vv = k[see, h * H // Hq], v[see, h * H // Hq]
            w = torch.softmax(kk @ q[i, h] * scale, 0)
            out[i, h], weight[i, h], plain[i, h] = w @ vv, w @ vv.abs(), vv.abs().sum(0)
            size[i, h] = (kk.abs() @ q[i, h].abs()).max() * scale
    return out, weight, plain, size


def assert_attended(got, want, weight, plain, size, n, p_step, label):
    """got is want rounded once to its type, after what probabilities and sums in fewer bits leave.

    p_step: half a step of the probabilities.  p_t (1 + d_t), |d_t| <= p_step, weighed and summed from the same values:
    sum w_t d_t (v_t - o), at most p_step (sum w_t |v_t| + |o|).  The same holds for what changes a score by x: d = x.
    fp32 leaves in a score at most 256 + 8 half steps of sum |q k| scale (256 sums of products; factor, maximum, exp2's
    argument and value), in a weighted sum n half steps of sum w_t |v_t|.  A probability below 2^-14 of fp16's has steps of
    2^-24 whatever its size, so is off by up to 2^-25, of a sum of probabilities of at least one (the largest is one or
    more): sum_t 2^-25 (|v_t| + |o|)."""
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got.cpu()), nan), f"{label}: NaN elsewhere"
    g, w, a, b, z = (x.detach().cpu().double().nan_to_num(0, 0, 0) for x in (got, want, weight, plain, size))
    part = p_step + (264 * z + 2 * n) * 2.0 ** -24
    bound = half_step(got.dtype) * (1 + 2.0 ** -6) * w.abs() + part * (a + w.abs()) + torch.finfo(got.dtype).smallest_normal
    if p_step == 2.0 ** -11:
        bound = bound + 2.0 ** -25 * (b + n * w.abs())
    worst = ((g - w).abs() / bound).max().item() if g.numel() else 0.0
    print(f"[{label}] worst error {worst:.3f} of its bound", flush=True)
    assert worst <= 1.0, f"{label}: {worst} times the bound"
