"""What the performance of the batch operators over a paged cache is measured on.

A server keeps many sequences in one pool of pages and runs them together; with the
pool in 8 bits it holds twice as many, and with a window a step reads only the end
of each:

  scatter  a batch's new K and V rows quantised into their pages (paged.kv_scatter_f8):
           e4m3 codes and one power-of-two scale for each page of 16 tokens and head,
           which grows with the page
  gather   rows read back from such pages as elements (paged.kv_gather_f8), to move a
           sequence elsewhere or to hand it to a kernel that takes plain rows
  attend   attention of a padded batch of queries over the pages
           (paged.paged_attention_batch): pools in 8 bits or in the elements' 16, whole
           causal contexts, or a sliding window with a few first tokens that stay visible

Where `own` is true, run() calls these entry points.  Otherwise it computes the same
in plain torch operations in 32 bits, rounded once at the end.

The head shapes are the repository's (32 / 8 and 16 / 8 heads of 128: Qwen3; 8 / 2 of
256: Qwen3.5) and generic ones.
"""
import math

import torch

own = False

PAGE = 16
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def _rows(name, kind, b, s, hk, d, dtype="bf16", past=0, ragged=False):
    """New rows written to, or rows read from, positions that begin somewhere in 0..past."""
    return {"name": name, "kind": kind, "b": b, "s": s, "hk": hk, "d": d, "dtype": dtype, "past": past, "ragged": ragged}


def _attend(name, b, s, n, hq, hk, d, dtype="bf16", f8=True, window=0, sinks=0, ragged=False):
    """s queries at the end of contexts of up to n tokens."""
    return {"name": name, "kind": "attend", "b": b, "s": s, "n": n, "hq": hq, "hk": hk, "d": d, "dtype": dtype, "f8": f8,
            "window": window, "sinks": sinks, "ragged": ragged}


def listed():
    return [
        # a whole prompt goes into the cache
        _rows("scatter_prompt_2k", "scatter", 1, 2048, 8, 128),
        # the new token of each of 64 conversations, anywhere in its last page
        _rows("scatter_tokens_64", "scatter", 64, 1, 8, 128, past=1000),
        # a whole conversation leaves the cache
        _rows("gather_context_8k", "gather", 1, 8192, 8, 128),
        # parts of three conversations, unlike in length, on 256-wide heads and fp16
        _rows("gather_batch_f16", "gather", 3, 700, 2, 256, "f16", past=500, ragged=True),
        # one token of one conversation of 8K tokens (Qwen3-4B's heads)
        _attend("decode_8k", 1, 1, 8192, 32, 8, 128),
        # one token each of 64 conversations, the shortest of a page, the longest of 4K
        _attend("decode_batch_64", 64, 1, 4096, 32, 8, 128, ragged=True),
        # one token at the end of 128K: the most keys
        _attend("decode_long_128k", 1, 1, 131072, 16, 8, 128),
        # four drafted tokens each of six short conversations: the smallest call
        _attend("draft_batch_f16", 6, 4, 700, 16, 4, 128, "f16", ragged=True),
        # a prompt over its own rows (Qwen3-1.7B's heads)
        _attend("prompt_2k", 1, 2048, 2048, 16, 8, 128),
        # the next 512 tokens of two long prompts that are taken in chunks: the most work
        _attend("chunk_512_of_8k", 2, 512, 8192, 32, 8, 128),
        # one token each of 32 conversations that see their last 1024 tokens and the first four, in 16 bits
        _attend("window_tokens_32", 32, 1, 16384, 32, 8, 128, f8=False, window=1024, sinks=4, ragged=True),
        # a prompt in which every token sees the last 512 and the first four (Qwen3.5's heads)
        _attend("window_prompt_4k", 1, 4096, 4096, 8, 2, 256, f8=False, window=512, sinks=4),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


HEADS = [(32, 8, 128), (32, 8, 128), (16, 8, 128), (8, 2, 256), (16, 4, 64), (12, 4, 128), (16, 1, 128), (5, 5, 64), (14, 2, 64)]


def draw(rng):
    kind = rng.choice(["scatter", "gather", "attend", "attend", "attend", "attend"])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    hq, hk, d = rng.choice(HEADS)
    if kind != "attend":
        b = rng.choice([1, 1, 2, 3, _log(rng, 4, 100)])
        s = rng.choice([1, _log(rng, 2, 8192 // b)]) if b > 1 else _log(rng, 2, 8192)
        return _rows("", kind, b, s, hk, d, dtype, rng.choice([0, _log(rng, 1, 1000)]), b > 1 and rng.random() < 0.5)
    f8 = rng.random() < 0.7
    if rng.random() < 0.6:  # tokens and drafts
        b, s = rng.choice([1, _log(rng, 2, 64)]), rng.choice([1, 1, 1, 2, 3, 5, 8])
        n = _log(rng, max(s, 40), 131072 // b if f8 and b > 1 else 65536 // b)
    else:  # prompts and chunks
        b = rng.choice([1, 1, 2, 3])
        s = _log(rng, 20, 1000 // b)
        n = s if rng.random() < 0.5 else _log(rng, s, 8192)
    window = rng.choice([0, 0, _log(rng, 16, 2048)])
    return _attend("", b, s, n, hq, hk, d, dtype, f8, window, rng.choice([0, 1, 4, 20]) if window else 0, b > 1 and rng.random() < 0.6)


# ------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, shape, dtype=torch.float32, std=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)


def _lens(c, most):
    """Lengths of a batch: from the whole width down to one."""
    b = c["b"]
    return [max(1, most - i * most // b) for i in range(b)] if c["ragged"] else [most] * b


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _gains(g, c):
    """What the channels of a head are scaled by: about one, a few far above it."""
    e = torch.rand((c["hk"], c["d"]), generator=g, device="cuda") + 0.5
    return torch.where(torch.rand(e.shape, generator=g, device="cuda") < 0.03, 4 * e, e)


def _tables(g, c, pages):
    """Pages of each sequence, scattered over a pool that is a little larger: [b, pages], and the blocks of the pool."""
    blocks = c["b"] * pages + 7
    at = torch.randperm(blocks, generator=g, device="cuda")[: c["b"] * pages]
    return at.view(c["b"], pages).to(torch.int32), blocks


def _pool_f8(g, c, blocks, gains):
    """Codes and scales of a pool that holds rows; the head is outside of the page's tokens."""
    x = _normal(g, (blocks, c["hk"], PAGE, c["d"])) * gains[:, None, :]
    e = _exponent(x.abs().amax((2, 3)))
    codes = (x * _power(-e)[:, :, None, None]).to(torch.float8_e4m3fn)
    return codes.transpose(1, 2), (e + 127).to(torch.uint8)


def prepare(case, seed):
    c, g = dict(case), _gen(seed)
    t = TYPES[c["dtype"]]
    b, s, hk, d = c["b"], c["s"], c["hk"], c["d"]
    gain_k, gain_v = _gains(g, c), 0.2 * _gains(g, c)
    st = {"case": c}
    if c["kind"] != "attend":
        lens = _lens(c, s)
        start = torch.randint(0, c["past"] + 1, (b,), generator=g, device="cuda").tolist() if c["past"] else [0] * b
        pages = -(-(c["past"] + s) // PAGE)
        st["k_ids"], blocks = _tables(g, c, pages)
        st["v_ids"], _ = _tables(g, c, pages)
        st["k_pool"], st["k_scales"] = _pool_f8(g, c, blocks, gain_k)
        st["v_pool"], st["v_scales"] = _pool_f8(g, c, blocks, gain_v)
        st["start"], st["lens"] = _ints(start), _ints(lens) if c["ragged"] else None
        if c["kind"] == "scatter":
            # k as the rotation leaves it; v a part of the fused projection
            st["k"] = (_normal(g, (b, s, hk, d)) * gain_k).to(t)
            kv = (_normal(g, (b, s, 2, hk, d)) * gain_v).to(t)
            st["v"] = kv[:, :, 1]
        else:
            st["k_out"], st["v_out"] = (torch.zeros((b, s, hk, d), dtype=t, device="cuda") for _ in range(2))
        return st
    n = _lens(c, c["n"])
    q_lens = [min(x, max(1, s - i % 3 * (s // 4))) if c["ragged"] else s for i, x in enumerate(n)]
    pages = -(-c["n"] // PAGE)
    st["k_ids"], blocks = _tables(g, c, pages)
    st["v_ids"], _ = _tables(g, c, pages)
    if c["f8"]:
        st["k_pool"], st["k_scales"] = _pool_f8(g, c, blocks, gain_k)
        st["v_pool"], st["v_scales"] = _pool_f8(g, c, blocks, gain_v)
    else:
        st["k_pool"] = (_normal(g, (blocks, PAGE, hk, d)) * gain_k).to(t)
        st["v_pool"] = (_normal(g, (blocks, PAGE, hk, d)) * gain_v).to(t)
        st["k_scales"] = st["v_scales"] = None
    st["n"], st["q_lens"] = _ints(n), _ints(q_lens) if c["ragged"] else None
    # q head by head, as the rotation leaves it; out token by token, as the next projection takes it
    st["q"] = _normal(g, (b, c["hq"], s, d), t, 1.5).transpose(1, 2)
    st["out"] = torch.zeros((b, s, c["hq"], d), dtype=t, device="cuda")
    st["scale"] = 1.0 / math.sqrt(d)
    return st


# --------------------------------------------------------------- plain forms
def _exponent(amax):
    """The least e with amax <= 448 * 2^e, at least -100."""
    m, e = torch.frexp(amax)
    return torch.where(amax > 0, e - 9 + (m > 0.875), torch.full_like(e, -100)).clamp(min=-100).to(torch.int32)


def _power(e):
    """2^e in 32 bits, exactly."""
    return (e.to(torch.int32).clamp(-126, 127) + 127 << 23).view(torch.float32)


def _values(codes, scales):
    """[..., 16, hk, d] in 32 bits."""
    return codes.float() * _power(scales.to(torch.int32) - 127)[..., None, :, None]


def _pages(st, width):
    """The pages from each start on that `width` tokens may reach: (place in the table [b, w], is there, token's place [b, w, 16])."""
    start = st["start"].long()
    w = -(-width // PAGE) + 1
    at = start[:, None] // PAGE + torch.arange(w, device="cuda")
    place = at[:, :, None] * PAGE + torch.arange(PAGE, device="cuda") - start[:, None, None]
    n = st["lens"].long() if st["lens"] is not None else torch.full_like(start, width)
    return at.clamp(max=st["k_ids"].shape[1] - 1), place, (place >= 0) & (place < n[:, None, None])


def _plain_scatter(st):
    s, row = st["case"]["s"], torch.arange(st["case"]["b"], device="cuda")[:, None]
    at, place, new = _pages(st, s)
    some = new.any(-1)
    kept = (st["start"].long()[:, None] % PAGE > 0) & (torch.arange(at.shape[1], device="cuda") == 0)
    for x, pool, scales, ids in ((st["k"], st["k_pool"], st["k_scales"], st["k_ids"]), (st["v"], st["v_pool"], st["v_scales"], st["v_ids"])):
        y = x.float()[row[:, :, None], place.clamp(0, s - 1)]  # [b, w, 16, hk, d]
        y = torch.where(new[..., None, None], y, 0.0)
        ids = ids[row, at].long()
        old, old_e = pool[ids], scales[ids].to(torch.int32) - 127
        e = _exponent(y.abs().amax((2, 4)))
        e = torch.where(kept[..., None], torch.maximum(e, old_e), e)
        codes = (y * _power(-e)[:, :, None, :, None]).to(pool.dtype)
        again = (old.float() * _power(torch.where(kept[..., None], old_e - e, 0))[:, :, None, :, None]).to(pool.dtype)
        codes = torch.where(new[..., None, None], codes.view(torch.uint8), again.view(torch.uint8)).view(pool.dtype)
        pool[ids[some]] = codes[some]
        scales[ids[some]] = (e[some] + 127).to(torch.uint8)
    return [st["k_pool"], st["v_pool"], st["k_scales"], st["v_scales"]]


def _plain_gather(st):
    s, row = st["case"]["s"], torch.arange(st["case"]["b"], device="cuda")[:, None]
    pos = st["start"].long()[:, None] + torch.arange(s, device="cuda")
    n = st["lens"].long()[:, None] if st["lens"] is not None else s
    there = (torch.arange(s, device="cuda") < n).expand(pos.shape)[..., None, None]
    for out, pool, scales, ids in ((st["k_out"], st["k_pool"], st["k_scales"], st["k_ids"]), (st["v_out"], st["v_pool"], st["v_scales"], st["v_ids"])):
        at = ids[row, pos // PAGE].long()
        x = pool[at, pos % PAGE].float() * _power(scales[at].to(torch.int32) - 127)[..., None]
        out.copy_(torch.where(there, x.to(out.dtype), out))
    return [st["k_out"], st["v_out"]]


def _plain_attend(st):
    c = st["case"]
    b, s, hq, hk, d = c["b"], c["s"], c["hq"], c["hk"], c["d"]
    n = st["n"].long()[:, None]
    q_lens = st["q_lens"].long()[:, None] if st["q_lens"] is not None else torch.full_like(n, s)
    i, t = torch.arange(s, device="cuda"), torch.arange(st["k_ids"].shape[1] * PAGE, device="cuda")
    pos = (n - q_lens + i)[..., None]  # [b, s, 1]
    seen = (t <= pos) & (t < n[..., None])
    if c["window"]:
        seen &= (t > pos - c["window"]) | (t < c["sinks"])
    kv = []
    for pool, scales, ids in ((st["k_pool"], st["k_scales"], st["k_ids"]), (st["v_pool"], st["v_scales"], st["v_ids"])):
        at = ids.long()
        x = _values(pool[at], scales[at]) if scales is not None else pool[at].float()
        kv.append(x.reshape(b, -1, hk, d).transpose(1, 2))  # [b, hk, t, d]
    q = st["q"].float().reshape(b, s, hk, hq // hk, d).permute(0, 2, 3, 1, 4).reshape(b, hk, -1, d)
    x = (q @ kv[0].transpose(-1, -2)).view(b, hk, hq // hk, s, -1) * st["scale"]
    x = x.masked_fill_(~seen[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    p = x.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    o = (p.view(b, hk, -1, p.shape[-1]) @ kv[1]).view(b, hk, hq // hk, s, d) / torch.where(total == 0, 1.0, total)
    o = o.permute(0, 3, 1, 2, 4).reshape(b, s, hq, d).to(st["out"].dtype)
    st["out"].copy_(torch.where((i < q_lens)[..., None, None], o, st["out"]))
    return [st["out"]]


# --------------------------------------------------------- the framework's calls
def _own(st):
    from genllm_amd import paged

    c = st["case"]
    if c["kind"] == "scatter":
        paged.kv_scatter_f8(st["k"], st["v"], st["k_pool"], st["v_pool"], st["k_scales"], st["v_scales"], st["k_ids"], st["v_ids"],
                            st["start"], seq_lens=st["lens"])
        return [st["k_pool"], st["v_pool"], st["k_scales"], st["v_scales"]]
    if c["kind"] == "gather":
        paged.kv_gather_f8(st["k_pool"], st["v_pool"], st["k_scales"], st["v_scales"], st["k_ids"], st["v_ids"], st["start"],
                           st["k_out"], st["v_out"], seq_lens=st["lens"])
        return [st["k_out"], st["v_out"]]
    paged.paged_attention_batch(st["q"], st["out"], st["k_pool"], st["v_pool"], st["k_ids"], st["v_ids"], st["n"], st["scale"],
                                q_lens=st["q_lens"], k_scales=st["k_scales"], v_scales=st["v_scales"],
                                window=c["window"] or None, sinks=c["sinks"])
    return [st["out"]]


def run(state):
    if own:
        return _own(state)
    return {"scatter": _plain_scatter, "gather": _plain_gather, "attend": _plain_attend}[state["case"]["kind"]](state)


# ------------------------------------------------------------------ exact
def exact(case, seed):
    """The definitions in 64 bits, sequence by sequence."""
    st = prepare(case, seed)
    return {"scatter": _exact_scatter, "gather": _exact_gather, "attend": _exact_attend}[case["kind"]](st)


def _two(e):
    """2^e in 64 bits, exactly (pow need not be)."""
    return (e.long() + 1023 << 52).view(torch.float64)


def _step(y):
    """y rounded to four significant bits, ties to even; steps of 2^-9 below 2^-6."""
    unit = _two((torch.frexp(y)[1] - 1).clamp(min=-6) - 3)
    return torch.round(y / unit) * unit


def _exact_scatter(st):
    c, r = st["case"], []
    start, lens = st["start"].tolist(), _lens(st["case"], st["case"]["s"])
    for x, pool, scales, ids in ((st["k"], st["k_pool"], st["k_scales"], st["k_ids"]), (st["v"], st["v_pool"], st["v_scales"], st["v_ids"])):
        codes, powers = pool.double(), scales.to(torch.int32) - 127
        for i in range(c["b"]):
            p, end = start[i], start[i] + lens[i]
            while p < end:
                block, slot, stop = int(ids[i, p // PAGE]), p % PAGE, min(end, (p // PAGE + 1) * PAGE)
                y = x[i, p - start[i] : stop - start[i]].double()
                e = torch.full_like(powers[block], -100) if slot == 0 else powers[block].clone()
                # the least power that holds the largest value, from 3 binades below it on
                top = y.abs().amax((0, 2))
                e = torch.where(top > 448 * _two(e), torch.maximum(e, torch.frexp(top)[1] - 12), e)
                while bool((top > 448 * _two(e)).any()):
                    e += top > 448 * _two(e)
                if slot:
                    codes[block] = _step(codes[block] * _two(powers[block] - e)[:, None])
                codes[block, slot : slot + stop - p] = _step(y / _two(e)[:, None])
                powers[block] = e
                p = stop
        r.append(codes)
    return r + [None, None]


def _exact_rows(pool, scales, ids, first, last):
    """Tokens first..last-1 of one sequence, [n, hk, d]."""
    pos = torch.arange(first, last, device="cuda")
    block = ids[pos // PAGE].long()
    x = pool[block, pos % PAGE].double()
    return x * _two(scales[block].to(torch.int32) - 127)[..., None] if scales is not None else x


def _exact_gather(st):
    start, lens, r = st["start"].tolist(), _lens(st["case"], st["case"]["s"]), []
    for out, pool, scales, ids in ((st["k_out"], st["k_pool"], st["k_scales"], st["k_ids"]), (st["v_out"], st["v_pool"], st["v_scales"], st["v_ids"])):
        y = out.double()
        for i, m in enumerate(lens):
            y[i, :m] = _exact_rows(pool, scales, ids[i], start[i], start[i] + m)
        r.append(y)
    return r


def _exact_attend(st):
    c = st["case"]
    g, y = c["hq"] // c["hk"], st["out"].double()
    n = st["n"].tolist()
    q_lens = st["q_lens"].tolist() if st["q_lens"] is not None else [c["s"]] * c["b"]
    for i in range(c["b"]):
        k = _exact_rows(st["k_pool"], st["k_scales"], st["k_ids"][i], 0, n[i])
        v = _exact_rows(st["v_pool"], st["v_scales"], st["v_ids"][i], 0, n[i])
        ago = torch.arange(n[i] - q_lens[i], n[i], device="cuda")[:, None] - torch.arange(n[i], device="cuda")[None, :]
        hidden = ago < 0
        if c["window"]:
            hidden |= (ago >= c["window"]) & (torch.arange(n[i], device="cuda") >= c["sinks"])[None, :]
        for h in range(c["hq"]):
            x = st["q"][i, : q_lens[i], h].double() @ k[:, h // g].T * st["scale"]
            x[hidden] = -math.inf
            y[i, : q_lens[i], h] = torch.exp(x - torch.logsumexp(x, -1, keepdim=True)) @ v[:, h // g]
    return [y]


# ------------------------------------------------------------------- work
def work(case):
    c = case
    if c["kind"] != "attend":
        n = sum(_lens(c, c["s"])) * c["hk"] * c["d"]
        # K and V: elements on one side, codes and a byte for a page and head on the other
        return {"bytes": 2 * (3 * n + n // (PAGE * c["d"])), "flops": 4 * n}
    n = _lens(c, c["n"])
    rows = pairs = keys = 0
    for i, x in enumerate(n):
        m = min(x, max(1, c["s"] - i % 3 * (c["s"] // 4))) if c["ragged"] else c["s"]
        rows += m
        if c["window"]:
            pairs += sum(min(p + 1, c["window"] + min(c["sinks"], max(0, p + 1 - c["window"]))) for p in range(x - m, x))
            first = max(0, x - m - c["window"] + 1)
            keys += x - first + min(c["sinks"], first)
        else:
            pairs += m * x - m * (m - 1) // 2
            keys += x
    size = 1 + 1 / (PAGE * c["d"]) if c["f8"] else 2
    return {"bytes": 2 * 2 * rows * c["hq"] * c["d"] + 2 * keys * c["hk"] * c["d"] * size, "flops": 4 * pairs * c["hq"] * c["d"]}
