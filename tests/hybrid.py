"""Plain 64-bit forms of the hybrid layers' operators and the tolerances of their tests.

Everything here runs on the CPU in float64, from the definitions in
include/genllm_paged.h."""
import math

import torch

ULP32 = 2.0 ** -24  # half a step of fp32, relative


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def softplus(x):
    return torch.logaddexp(x, torch.zeros_like(x))


def delta_rule(q, k, v, a, b, state, scale, a_log=None, dt_bias=None, l2_eps=None, lens=None):
    """The rule token by token: (out, state) in float64; state [B, Hv, Dk, Dv].  Rows past an entry's length are zero."""
    q, k, v, a, beta, s = (x.detach().cpu().double() for x in (q, k, v, a, b, state))
    B, S, Hk, Dk = q.shape
    Hv, Dv = v.shape[2:]
    if a_log is not None:
        a = -torch.exp(a_log.cpu().double()) * softplus(a + dt_bias.cpu().double())
        beta = torch.sigmoid(beta)
    if l2_eps is not None:
        q = q / torch.sqrt((q * q).sum(-1, keepdim=True) + l2_eps)
        k = k / torch.sqrt((k * k).sum(-1, keepdim=True) + l2_eps)
    q, k = q.repeat_interleave(Hv // Hk, 2), k.repeat_interleave(Hv // Hk, 2)
    s, out = s.clone(), torch.zeros(B, S, Hv, Dv, dtype=torch.float64)
    for i in range(B):
        n = S if lens is None else min(max(int(lens[i]), 0), S)
        for t in range(n):
            m = s[i] * torch.exp(a[i, t])[:, None, None]
            u = beta[i, t][:, None] * (v[i, t] - (m * k[i, t][:, :, None]).sum(1))
            s[i] = m + k[i, t][:, :, None] * u[:, None, :]
            out[i, t] = scale * (s[i] * q[i, t][:, :, None]).sum(1)
    return out, s


def causal_conv(x, w, state=None, bias=None, silu=True, lens=None):
    """(out, state) in float64; state [B, W-1, C].  Rows past an entry's length are zero."""
    x, w = x.detach().cpu().double(), w.cpu().double()
    B, S, C = x.shape
    W = w.shape[1]
    out = torch.zeros(B, S, C, dtype=torch.float64)
    new = state.cpu().double().clone() if state is not None else torch.zeros(B, W - 1, C, dtype=torch.float64)
    for i in range(B):
        n = S if lens is None else min(max(int(lens[i]), 0), S)
        if n == 0:
            continue
        line = torch.cat([new[i], x[i, :n]])
        for t in range(n):
            y = sum(w[:, j] * line[t + j] for j in range(W))
            if bias is not None:
                y = y + bias.cpu().double()
            out[i, t] = y / (1 + torch.exp(-y)) if silu else y
        new[i] = line[n:]
    return out, new


def pair_axes(sections, interleaved):
    n, r = len(sections), []
    for i in range(sum(sections)):
        if interleaved:
            r.append(i % n if i // n < sections[i % n] else 0)
        else:
            r.append(next(a for a in range(n) if i < sum(sections[: a + 1])))
    return r


def norm_rope_axes(x, gamma, eps, cos, sin, positions, sections, interleaved):
    """[S, H, D] in float64."""
    y = x.detach().cpu().double().clone()
    cos, sin, pos = cos.cpu().double(), sin.cpu().double(), positions.cpu().long()
    if gamma is not None:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * gamma.cpu().double()
    half = sum(sections)
    for i, axis in enumerate(pair_axes(sections, interleaved)):
        at = pos[axis]
        ok = (at >= 0) & (at < cos.shape[0])
        c = torch.where(ok, cos[at.clamp(0, cos.shape[0] - 1), i], torch.nan)[:, None]
        s = torch.where(ok, sin[at.clamp(0, cos.shape[0] - 1), i], torch.nan)[:, None]
        y0, y1 = y[..., i].clone(), y[..., i + half].clone()
        y[..., i], y[..., i + half] = y0 * c - y1 * s, y0 * s + y1 * c
    return y


def assert_rounded(got, want, label, slack=2.0 ** -14):
    """got is want rounded once to its type: half a step of each value, and `slack` of the largest value of its row for
    what 32-bit sums of terms that cancel leave (and the products of two 8-bit parts, 2^-17 of each term)."""
    assert torch.equal(torch.isnan(got.cpu()), torch.isnan(want)), f"{label}: NaN elsewhere"
    g, w = got.detach().cpu().double().nan_to_num(0, 0, 0), want.nan_to_num(0, 0, 0)
    assert torch.equal(torch.isinf(got.cpu()), torch.isinf(want)), f"{label}: infinities elsewhere"
    row = w.abs().amax(-1, keepdim=True)
    bound = half_step(got.dtype) * (1 + 2.0 ** -6) * w.abs() + slack * row + torch.finfo(got.dtype).tiny
    worst = ((g - w).abs() / bound).max().item() if g.numel() else 0.0
    print(f"[{label}] worst error {worst:.3f} of its bound", flush=True)
    assert worst <= 1.0, f"{label}: {worst} times the bound"


def assert_state(got, want, tokens, label):
    """A state after `tokens` tokens, in the 2-norm of each head's matrix: a token leaves about 36 roundings in an element
    (the sums over a row group, beta and alpha, the update), independent of each other, and what earlier tokens left
    does not grow: 6 sqrt(tokens) half steps of fp32, and one for the state itself."""
    g, w = got.detach().cpu().double(), want
    off = (g - w).flatten(-2).norm(dim=-1)
    norm = w.flatten(-2).norm(dim=-1)
    bound = (6 * math.sqrt(tokens) + 1) * ULP32 * norm + 1e-30
    worst = (off / bound).max().item() if off.numel() else 0.0
    print(f"[{label}] state error {(off / norm.clamp(min=1e-30)).max().item():.2e}, {worst:.3f} of its bound", flush=True)
    assert worst <= 1.0, f"{label}: state {worst} times the bound"
