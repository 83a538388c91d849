"""What the performance of the hybrid layers' operators is measured on.

Beside the paged attention layers a hybrid model has layers whose memory is one
matrix per head, and prompts whose tokens have positions on several axes:

  delta  the gated delta rule (paged.gated_delta_rule): a prompt, or a turn on top of
         a kept state, in chunks; one token, or a few drafted ones, per sequence
  conv   the short causal convolution in front of it (paged.causal_conv), which
         keeps the last inputs of each sequence as its state
  rope   the norm of every q and k head with the rotation by positions on several
         axes in the same pass (paged.qk_norm_rope_axes), for the attention layers

Where `own` is true, run() calls these entry points.  Otherwise it computes the
same in plain torch operations in 32 bits (64 for the running sums of the
decays), rounded once at the end.

The head shapes are generic (16 key / 32 value heads of 128, 64-wide heads, odd
head ratios); the attention layers' are the repository's: 8 / 2 heads of 256
with 64 rotated dims (Qwen3.5), 32 / 8 of 128 (Qwen3-4B).
"""
import math

import torch

own = False

CHUNK = 64
L2_EPS = 1e-6
EPS = 1e-6
THETA = 1e6
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def _delta(name, b, s, hk, hv, dk, dv, dtype="bf16", raw=True, l2=True, ragged=False, slots=0):
    return {"name": name, "kind": "delta", "b": b, "s": s, "hk": hk, "hv": hv, "dk": dk, "dv": dv, "dtype": dtype,
            "raw": raw, "l2": l2, "ragged": ragged, "slots": slots}


def _conv(name, b, s, c, w, dtype="bf16", bias=False, ragged=False, slots=0):
    return {"name": name, "kind": "conv", "b": b, "s": s, "c": c, "w": w, "dtype": dtype, "bias": bias,
            "ragged": ragged, "slots": slots}


def _rope(name, s, hq, hk, d, rope, dtype="bf16", interleaved=True, norm=True):
    return {"name": name, "kind": "rope", "s": s, "hq": hq, "hk": hk, "d": d, "rope": rope, "dtype": dtype,
            "interleaved": interleaved, "norm": norm}


def listed():
    return [
        # a whole prompt through one layer
        _delta("delta_prompt_2k", 1, 2048, 16, 32, 128, 128),
        # a long document through one layer: the largest call
        _delta("delta_prompt_8k", 1, 8192, 16, 32, 128, 128),
        # a padded batch of prompts of unlike length, one of them empty, on 64-wide keys and fp16
        _delta("delta_batch_f16", 4, 700, 4, 8, 64, 128, "f16", ragged=True, slots=6),
        # the next turn of a conversation, on top of the state that the last one left
        _delta("delta_turn_77", 1, 77, 16, 32, 128, 128),
        # one token of one conversation
        _delta("delta_token", 1, 1, 16, 32, 128, 128),
        # one token each of 64 conversations, whose states lie in a pool
        _delta("delta_tokens_64", 64, 1, 16, 32, 128, 128, slots=96),
        # four drafted tokens each of 8 conversations, gates computed by the caller
        _delta("delta_draft_f16", 8, 4, 4, 8, 128, 128, "f16", raw=False, slots=8),
        # the convolution over the q, k and v channels of a whole prompt
        _conv("conv_prompt_2k", 1, 2048, 8192, 4),
        # the same for one token each of 64 conversations
        _conv("conv_tokens_64", 64, 1, 8192, 4, slots=96),
        # a padded batch on an odd number of channels, with a bias
        _conv("conv_batch_f16", 3, 333, 1003, 3, "f16", bias=True, ragged=True),
        # a prompt of text and image patches in an attention layer (Qwen3.5)
        _rope("rope_image_2k", 2048, 8, 2, 256, 64),
        # one token each of 16 conversations (Qwen3-4B's heads), the axes' sections one after another
        _rope("rope_tokens_f16", 16, 32, 8, 128, 128, "f16", interleaved=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    kind = rng.choice(["delta", "delta", "delta", "delta", "conv", "rope"])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    if kind == "delta":
        hk, hv = rng.choice([(16, 32), (16, 32), (4, 8), (6, 6), (10, 10), (2, 6), (1, 3)])
        dk, dv = rng.choice([(128, 128), (128, 128), (64, 64), (64, 128), (128, 64)])
        if rng.random() < 0.5:  # prompts and turns
            b = rng.choice([1, 1, 2, 3, 5])
            s = _log(rng, 17, 8192 // b)
        else:  # tokens and drafts
            b, s = _log(rng, 1, 100), rng.choice([1, 1, 1, 2, 3, 5, 8])
        slots = rng.choice([0, b + rng.randrange(0, 9)])
        return _delta("", b, s, hk, hv, dk, dv, dtype, rng.random() < 0.7, rng.random() < 0.8, b > 1 and rng.random() < 0.4,
                      slots)
    if kind == "conv":
        c = rng.choice([8192, 4096, 2560, 1536, 640, 1003, _log(rng, 64, 8192)])
        b = rng.choice([1, 1, 2, 3, _log(rng, 4, 100)])
        s = rng.choice([1, 1, _log(rng, 2, max(2, 8192 // b))])
        return _conv("", b, s, c, rng.choice([4, 4, 3, 2]), dtype, rng.random() < 0.4, b > 1 and rng.random() < 0.4,
                     rng.choice([0, b + rng.randrange(0, 9)]))
    hq, hk, d = rng.choice([(8, 2, 256), (32, 8, 128), (16, 4, 128), (16, 4, 256), (12, 4, 128), (16, 1, 128)])
    return _rope("", _log(rng, 1, 8192), hq, hk, d, 64 if d == 256 else rng.choice([128, 128, 64]), dtype,
                 rng.random() < 0.5, rng.random() < 0.8)


# ------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, shape, dtype=torch.float32, std=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)


def _uniform(g, shape, lo, hi):
    return torch.rand(shape, generator=g, device="cuda") * (hi - lo) + lo


def _lens(c):
    """The lengths of a padded batch: from the whole width down to nothing."""
    b, s = c["b"], c["s"]
    return [s - i * s // (b - 1) for i in range(b)] if c["ragged"] else [s] * b


def _ids(g, c):
    return torch.randperm(c["slots"], generator=g, device="cuda")[: c["b"]].to(torch.int32) if c["slots"] else None


def _sections(c):
    """Pairs of the time, height and width axes (11, 11, 10 of 32; 16, 24, 24 of 64)."""
    pairs = c["rope"] // 2
    if c["interleaved"]:
        return (pairs - 2 * (pairs // 3) - (pairs % 3 == 2), pairs // 3 + (pairs % 3 == 2), pairs // 3)
    return (pairs - 2 * (3 * pairs // 8), 3 * pairs // 8, 3 * pairs // 8)


def prepare(case, seed):
    c, g = dict(case), _gen(seed)
    t = TYPES[c["dtype"]]
    if c["kind"] == "rope":
        return _prepare_rope(c, g, t)
    st = {"case": c, "lens": torch.tensor(_lens(c), dtype=torch.int32, device="cuda") if c["ragged"] else None}
    b, s = c["b"], c["s"]
    st["ids"] = _ids(g, c)
    n = c["slots"] or b
    if c["kind"] == "conv":
        ch, w = c["c"], c["w"]
        st["x"] = _normal(g, (b, s, ch), t)
        st["w"] = _normal(g, (ch, w), t, 0.5)
        st["bias"] = _normal(g, (ch,), t, 0.3) if c["bias"] else None
        st["state"] = _normal(g, (n, w - 1, ch), t)
        st["out"] = torch.zeros((b, s, ch), dtype=t, device="cuda")
        return st
    hk, hv, dk, dv = c["hk"], c["hv"], c["dk"], c["dv"]
    # q, k and v are channels of one tensor, the convolution's output
    qkv = torch.nn.functional.silu(_normal(g, (b, s, 2 * hk * dk + hv * dv), std=1.5))
    if not c["l2"]:  # keys that the caller has scaled
        qkv[..., : 2 * hk * dk] *= 1.0 / math.sqrt(0.9 * dk)
    qkv = qkv.to(t)
    q, k, v = torch.split(qkv, [hk * dk, hk * dk, hv * dv], dim=-1)
    st["q"], st["k"], st["v"] = q.view(b, s, hk, dk), k.view(b, s, hk, dk), v.view(b, s, hv, dv)
    # decays from nearly none to most of the state in a token, as the layers' heads learn them
    a_log = torch.log(_uniform(g, (hv,), 1.0, 16.0))
    dt = torch.exp(_uniform(g, (hv,), math.log(1e-3), math.log(0.1)))
    dt_bias = dt + torch.log(-torch.expm1(-dt))  # softplus(dt_bias) = dt
    ab = _normal(g, (b, s, 2 * hv))
    if c["raw"]:
        ab = ab.to(t)
        st["a"], st["b"] = ab[..., :hv], ab[..., hv:]
        st["a_log"], st["dt_bias"] = a_log, dt_bias
    else:
        st["a"] = -torch.exp(a_log) * torch.nn.functional.softplus(ab[..., :hv] + dt_bias)
        st["b"] = torch.sigmoid(ab[..., hv:])
        st["a_log"] = st["dt_bias"] = None
    st["state"] = _normal(g, (n, hv, dk, dv), std=0.2)
    st["out"] = torch.zeros((b, s, hv, dv), dtype=t, device="cuda")
    st["scale"] = 1.0 / math.sqrt(dk)
    return st


def _prepare_rope(c, g, t):
    s, hq, hk, d = c["s"], c["hq"], c["hk"], c["d"]
    st = {"case": c, "sections": _sections(c)}
    # q and k as one projection leaves them, token by token; the attention op takes them head by head
    qk = _normal(g, (s, (hq + hk) * d), t)
    st["q"], st["k"] = qk[:, : hq * d].view(s, hq, d), qk[:, hq * d :].view(s, hk, d)
    st["q_out"] = torch.zeros((hq, s, d), dtype=t, device="cuda").transpose(0, 1)
    st["k_out"] = torch.zeros((hk, s, d), dtype=t, device="cuda").transpose(0, 1)
    st["gamma_q"] = _uniform(g, (d,), 0.5, 1.5) if c["norm"] else None
    st["gamma_k"] = _uniform(g, (d,), 0.5, 1.5) if c["norm"] else None
    # text and images in turn: the axes run together over text, apart over an image's rows and columns
    rows = s + 64
    at = torch.arange(s, device="cuda")
    image = (at // 97) % 2 == 1
    side = 1 + int(torch.randint(4, 16, (1,), generator=g, device="cuda"))
    start = at // 97 * 97
    p = torch.stack([at, at, at])
    p[0] = torch.where(image, start, at)
    p[1] = torch.where(image, start + (at - start) // side, at)
    p[2] = torch.where(image, start + (at - start) % side, at)
    st["pos"] = (p + int(torch.randint(0, 64, (1,), generator=g, device="cuda"))).clamp(max=rows - 1).to(torch.int32)
    half = c["rope"] // 2
    f = THETA ** (-torch.arange(half, dtype=torch.float64, device="cuda") / half)
    ang = torch.arange(rows, dtype=torch.float64, device="cuda")[:, None] * torch.cat([f, f])[None, :]
    st["cos"], st["sin"] = torch.cos(ang).float(), torch.sin(ang).float()
    return st


# --------------------------------------------------------------- plain forms
def _axes(sections, interleaved, device):
    """The axis of every rotated pair."""
    pairs, n = sum(sections), len(sections)
    i = torch.arange(pairs, device=device)
    sec = torch.tensor(sections, device=device)
    if interleaved:
        return torch.where(i // n < sec[i % n], i % n, 0)
    return (i[:, None] >= torch.cumsum(sec, 0)[None, :]).sum(1)


def _plain_rope(st):
    c, half = st["case"], st["case"]["rope"] // 2
    axis = _axes(st["sections"], c["interleaved"], "cuda")
    rows = st["pos"].long()[axis].t()  # [s, pairs]
    pair = torch.arange(half, device="cuda")
    cos, sin = st["cos"][rows, pair][:, None, :], st["sin"][rows, pair][:, None, :]
    for x, gamma, out in ((st["q"], st["gamma_q"], st["q_out"]), (st["k"], st["gamma_k"], st["k_out"])):
        y = x.float()
        if gamma is not None:
            y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + EPS) * gamma
        x0, x1 = y[..., :half], y[..., half : 2 * half]
        out.copy_(torch.cat([x0 * cos - x1 * sin, x0 * sin + x1 * cos, y[..., 2 * half :]], -1))
    return [st["q_out"], st["k_out"]]


def _valid(st):
    """[b, s] truth values: the tokens of a padded batch that are there."""
    c = st["case"]
    at = torch.arange(c["s"], device="cuda")[None, :]
    return at < (st["lens"][:, None] if st["lens"] is not None else torch.full((c["b"], 1), c["s"], device="cuda"))


def _slots(st):
    return st["ids"].long() if st["ids"] is not None else torch.arange(st["case"]["b"], device="cuda")


def _plain_conv(st):
    c = st["case"]
    w, s, ids = c["w"], c["s"], _slots(st)
    full = torch.cat([st["state"][ids], st["x"]], 1).float()
    y = sum(full[:, j : j + s] * st["w"][:, j].float() for j in range(w))
    if st["bias"] is not None:
        y = y + st["bias"].float()
    y = y * torch.sigmoid(y)
    st["out"].copy_(torch.where(_valid(st)[..., None], y.to(st["out"].dtype), st["out"]))
    n = st["lens"].long() if st["lens"] is not None else torch.full((c["b"],), s, device="cuda")
    last = n[:, None] + torch.arange(w - 1, device="cuda")[None, :]  # the last w - 1 inputs before each end
    st["state"][ids] = torch.gather(full, 1, last[..., None].expand(-1, -1, c["c"])).to(st["state"].dtype)
    return [st["out"], st["state"]]


def _gates(st):
    a, b = st["a"].float(), st["b"].float()
    if st["a_log"] is not None:
        x = a + st["dt_bias"]
        a = -torch.exp(st["a_log"]) * (torch.clamp(x, min=0) + torch.log1p(torch.exp(-x.abs())))
        b = torch.sigmoid(b)
    return a, b


def _plain_delta(st):
    c = st["case"]
    b, s, hv, g = c["b"], c["s"], c["hv"], c["hv"] // c["hk"]
    valid, ids = _valid(st), _slots(st)
    decay, beta = _gates(st)
    decay, beta = torch.where(valid[..., None], decay, 0.0), torch.where(valid[..., None], beta, 0.0)
    q, k, v = st["q"].float(), st["k"].float(), st["v"].float()
    if c["l2"]:
        q, k = (x / torch.sqrt((x * x).sum(-1, keepdim=True) + L2_EPS) for x in (q, k))
    q, k = (x.repeat_interleave(g, 2) for x in (q * st["scale"], k))
    q, k, v = (x.transpose(1, 2) for x in (q, k, v))  # [b, hv, s, d]
    decay, beta = decay.transpose(1, 2), beta.transpose(1, 2)  # [b, hv, s]
    state = st["state"][ids]
    if s <= 16:  # token by token
        o = []
        for t in range(s):
            state = state * torch.exp(decay[:, :, t, None, None])
            u = beta[:, :, t, None, None] * (v[:, :, t, None, :] - k[:, :, t, None, :] @ state)
            state = state + k[:, :, t, :, None] * u
            o.append(q[:, :, t, None, :] @ state)
        o = torch.cat(o, 2)
    else:
        o, state = _plain_chunks(q, k, v, decay, beta, state)
    st["out"].copy_(torch.where(valid[..., None, None], o[:, :, :s].transpose(1, 2).to(st["out"].dtype), st["out"]))
    st["state"][ids] = state
    return [st["out"], st["state"]]


def _plain_chunks(q, k, v, decay, beta, state):
    """Chunks of 64 tokens: the products inside a chunk for all chunks at once, then the state from chunk to chunk."""
    b, h, s, _ = q.shape
    n = -(-s // CHUNK)
    pad = n * CHUNK - s
    q, k, v = (torch.nn.functional.pad(x, (0, 0, 0, pad)).reshape(b, h, n, CHUNK, -1) for x in (q, k, v))
    decay, beta = (torch.nn.functional.pad(x, (0, pad)).reshape(b, h, n, CHUNK) for x in (decay, beta))
    sums = torch.cumsum(decay.double(), -1)
    at = torch.arange(CHUNK, device="cuda")
    lower = at[:, None] >= at[None, :]
    fade = torch.where(lower, torch.exp((sums[..., :, None] - sums[..., None, :]).clamp(max=0.0)).float(), 0.0)
    kk = beta[..., None] * (k @ k.transpose(-1, -2)) * fade
    inv = torch.eye(CHUNK, device="cuda").expand(b, h, n, CHUNK, CHUNK).clone()
    for i in range(1, CHUNK):  # the inverse of 1 + the part of kk below the diagonal, row by row
        inv[..., i, :] -= (kk[..., i, None, :i] @ inv[..., :i, :])[..., 0, :]
    since = torch.exp(sums).float()[..., None]
    until = torch.exp(sums[..., -1:] - sums).float()[..., None]
    u0 = inv @ (beta[..., None] * v)
    w = inv @ (beta[..., None] * since * k)
    qk = (q @ k.transpose(-1, -2)) * fade
    qs, ks, end = q * since, (k * until).transpose(-1, -2), since[..., -1, :, None]
    o = []
    for i in range(n):
        u = u0[:, :, i] - w[:, :, i] @ state
        o.append(qs[:, :, i] @ state + qk[:, :, i] @ u)
        state = state * end[:, :, i] + ks[:, :, i] @ u
    return torch.cat(o, 2), state


# --------------------------------------------------------- the framework's calls
def _own(st):
    from genllm_amd import paged

    c = st["case"]
    if c["kind"] == "rope":
        paged.qk_norm_rope_axes(st["q"], st["k"], st["q_out"], st["k_out"], st["gamma_q"], st["gamma_k"], EPS, st["cos"],
                                st["sin"], st["pos"], st["sections"], interleaved=c["interleaved"])
        return [st["q_out"], st["k_out"]]
    if c["kind"] == "conv":
        paged.causal_conv(st["x"], st["w"], st["out"], st["state"], bias=st["bias"], silu=True, seq_lens=st["lens"],
                          state_ids=st["ids"])
        return [st["out"], st["state"]]
    paged.gated_delta_rule(st["q"], st["k"], st["v"], st["a"], st["b"], st["state"], st["out"], st["scale"],
                           a_log=st["a_log"], dt_bias=st["dt_bias"], l2_eps=L2_EPS if c["l2"] else None,
                           seq_lens=st["lens"], state_ids=st["ids"])
    return [st["out"], st["state"]]


def run(state):
    if own:
        return _own(state)
    return {"delta": _plain_delta, "conv": _plain_conv, "rope": _plain_rope}[state["case"]["kind"]](state)


# ------------------------------------------------------------------ exact
def exact(case, seed):
    """The definitions in 64 bits: the rule token by token, the convolution tap by tap, the rotation as complex numbers."""
    st = prepare(case, seed)
    return {"delta": _exact_delta, "conv": _exact_conv, "rope": _exact_rope}[case["kind"]](st)


def _exact_rope(st):
    c, r = st["case"], []
    half = c["rope"] // 2
    counts = list(st["sections"])
    if c["interleaved"]:
        axis = [i % 3 if i % 3 and i // 3 < counts[i % 3] else 0 for i in range(half)]
    else:
        axis = [0] * counts[0] + [1] * counts[1] + [2] * counts[2]
    pos = st["pos"].long()
    turn = torch.stack([torch.complex(st["cos"][pos[a], i].double(), st["sin"][pos[a], i].double())
                        for i, a in enumerate(axis)], -1)[:, None, :]
    for x, gamma in ((st["q"], st["gamma_q"]), (st["k"], st["gamma_k"])):
        y = x.double()
        if gamma is not None:
            y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * gamma.double()
        z = torch.complex(y[..., :half], y[..., half : c["rope"]]) * turn
        y[..., :half], y[..., half : c["rope"]] = z.real, z.imag
        r.append(y)
    return r


def _exact_conv(st):
    c = st["case"]
    out, new = st["out"].double(), st["state"].double()
    lens = _lens(c)
    for i in range(c["b"]):
        slot = int(st["ids"][i]) if st["ids"] is not None else i
        line = torch.cat([new[slot], st["x"][i, : lens[i]].double()], 0)
        y = torch.zeros((lens[i], c["c"]), dtype=torch.float64, device="cuda")
        for j in range(c["w"]):
            y += line[j : j + lens[i]] * st["w"][:, j].double()
        if st["bias"] is not None:
            y += st["bias"].double()
        out[i, : lens[i]] = y / (1 + torch.exp(-y))
        new[slot] = line[line.shape[0] - (c["w"] - 1) :]
    return [out, new]


def _exact_delta(st):
    c = st["case"]
    a, beta = st["a"].double(), st["b"].double()
    if st["a_log"] is not None:
        a = -torch.exp(st["a_log"].double()) * torch.logaddexp(a + st["dt_bias"].double(), torch.zeros_like(a))
        beta = 1 / (1 + torch.exp(-beta))
    q, k, v = st["q"].double(), st["k"].double(), st["v"].double()
    if c["l2"]:
        q, k = (x * torch.rsqrt(x.square().sum(-1, keepdim=True) + L2_EPS) for x in (q, k))
    head = torch.arange(c["hv"], device="cuda") // (c["hv"] // c["hk"])
    q, k = q[:, :, head], k[:, :, head]
    slots = _slots(st)
    pool, out = st["state"].double(), st["out"].double()
    m, there, alpha = pool[slots], _valid(st), torch.exp(a)
    for t in range(c["s"]):
        new = m * alpha[:, t, :, None, None]
        u = beta[:, t, :, None] * (v[:, t] - (new * k[:, t, :, :, None]).sum(-2))
        new = new + k[:, t, :, :, None] * u[:, :, None, :]
        o = st["scale"] * (new * q[:, t, :, :, None]).sum(-2)
        m = torch.where(there[:, t, None, None, None], new, m) if c["ragged"] else new
        out[:, t] = torch.where(there[:, t, None, None], o, out[:, t]) if c["ragged"] else o
    pool[slots] = m
    return [out, pool]


# ------------------------------------------------------------------- work
def work(case):
    c = case
    if c["kind"] == "rope":
        n = c["s"] * (c["hq"] + c["hk"]) * c["d"]
        # the tables' rows once for every token (no token shares its row for certain), three positions
        return {"bytes": 4 * n + c["s"] * (2 * 4 * c["rope"] // 2 + 12), "flops": 6 * n}
    tokens = sum(_lens(c))
    there = sum(x > 0 for x in _lens(c))
    if c["kind"] == "conv":
        return {"bytes": 2 * (2 * tokens * c["c"] + c["c"] * (c["w"] + c["bias"]) + 2 * there * (c["w"] - 1) * c["c"]),
                "flops": tokens * c["c"] * (2 * c["w"] + 4)}
    state = c["hv"] * c["dk"] * c["dv"]
    per_token = 2 * (2 * c["hk"] * c["dk"] + 2 * c["hv"] * c["dv"]) + (4 if c["raw"] else 8) * c["hv"]
    return {"bytes": tokens * per_token + 8 * there * state, "flops": 6 * tokens * state}
