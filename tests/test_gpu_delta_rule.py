"""The gated delta rule on the GPU against the rule token by token in 64 bits."""
import math

import pytest
import torch

from genllm_amd import paged
from hybrid import assert_rounded, assert_state, delta_rule, half_step

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def inputs(seed, B, S, Hk, Hv, Dk, Dv, dtype=BF16, raw=True, l2=True, n=None, layout="token", device="cuda"):
    g = torch.Generator().manual_seed(seed)

    def rows(H, D, scale=1.0):
        x = torch.nn.functional.silu(torch.randn(B, S, H, D, generator=g) * 1.5) * scale
        if layout == "head":  # [B, H, S, D] in memory
            return x.transpose(1, 2).contiguous().to(device, dtype).transpose(1, 2)
        if layout == "wide":  # channels of a wider tensor
            y = torch.empty(B, S, H * D + 24, device=device, dtype=dtype).fill_(7.0)
            y[..., 8 : 8 + H * D] = x.reshape(B, S, H * D).to(device, dtype)
            return y[..., 8 : 8 + H * D].view(B, S, H, D)
        return x.to(device, dtype)

    ks = 1.0 if l2 else 1.0 / math.sqrt(0.9 * Dk)
    x = {"q": rows(Hk, Dk, ks), "k": rows(Hk, Dk, ks), "v": rows(Hv, Dv)}
    a_log = torch.log(torch.rand(Hv, generator=g) * 15 + 1)
    dt = torch.exp(torch.rand(Hv, generator=g) * math.log(100.0) + math.log(1e-3))
    dt_bias = dt + torch.log(-torch.expm1(-dt))
    ab = torch.randn(B, S, 2 * Hv, generator=g)
    if raw:
        ab = ab.to(dtype)
        x["a"], x["b"] = ab.to(device)[..., :Hv], ab.to(device)[..., Hv:]
        x["a_log"], x["dt_bias"] = a_log.to(device), dt_bias.to(device)
    else:
        x["a"] = (-torch.exp(a_log) * torch.nn.functional.softplus(ab[..., :Hv] + dt_bias)).to(device)
        x["b"] = torch.sigmoid(ab[..., Hv:]).to(device)
    x["state"] = (torch.randn(n or B, Hv, Dk, Dv, generator=g) * 0.3).to(device)
    x["scale"] = 1.0 / math.sqrt(Dk)
    x["l2_eps"] = 1e-6 if l2 else None
    return x


def out_like(x, layout="token", fill=0.0):
    B, S, Hv, Dv = x["v"].shape
    if layout == "head":
        return torch.full((B, Hv, S, Dv), fill, dtype=x["v"].dtype, device="cuda").transpose(1, 2)
    return torch.full((B, S, Hv, Dv), fill, dtype=x["v"].dtype, device="cuda")


def call(x, out, **kw):
    paged.gated_delta_rule(x["q"], x["k"], x["v"], x["a"], x["b"], x["state"], out, x["scale"], a_log=x.get("a_log"),
                           dt_bias=x.get("dt_bias"), l2_eps=x["l2_eps"], **kw)


def reference(x, ids=None, lens=None):
    s = x["state"].cpu().double()
    s = s[ids] if ids is not None else s[: x["q"].shape[0]]
    return delta_rule(x["q"], x["k"], x["v"], x["a"], x["b"], s, x["scale"], x.get("a_log"), x.get("dt_bias"),
                      x["l2_eps"], lens)


def check(x, label, layout="token", **kw):
    want, new = reference(x)
    out = out_like(x, layout)
    call(x, out, **kw)
    torch.cuda.synchronize()
    assert_rounded(out, want, label)
    assert_state(x["state"], new, x["q"].shape[1], label)


# lengths around the chunk's and the kernels' limits
@pytest.mark.parametrize("S", [1, 2, 3, 7, 8, 9, 15, 16, 17, 31, 33, 63, 64, 65, 100, 127, 128, 129, 200, 321])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_lengths(S, dtype):
    check(inputs(S, 1, S, 2, 4, 128, 128, dtype), f"S={S} {dtype}")


@pytest.mark.parametrize("Dk,Dv", [(64, 64), (64, 128), (128, 64), (128, 128)])
@pytest.mark.parametrize("Hk,Hv", [(1, 1), (1, 3), (2, 2), (3, 6)])
@pytest.mark.parametrize("S", [1, 5, 90])
def test_heads(Dk, Dv, Hk, Hv, S):
    check(inputs(Dk + Dv + Hv + S, 2, S, Hk, Hv, Dk, Dv, F16 if S == 5 else BF16), f"{Hk}/{Hv} of {Dk}x{Dv}, S={S}")


@pytest.mark.parametrize("raw,l2", [(True, True), (True, False), (False, True), (False, False)])
@pytest.mark.parametrize("S", [1, 4, 150])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_gate_and_norm_forms(raw, l2, S, dtype):
    check(inputs(40 + S, 2, S, 2, 4, 128, 64, dtype, raw, l2), f"raw={raw} l2={l2} S={S}")


@pytest.mark.parametrize("layout", ["head", "wide"])
@pytest.mark.parametrize("S", [1, 3, 77])
def test_strides(layout, S):
    check(inputs(50 + S, 3, S, 2, 4, 64, 128, layout=layout), f"{layout} S={S}", layout)


@pytest.mark.parametrize("S", [1, 6, 70, 140])
def test_padded_batch_over_a_pool(S):
    """Lengths from past the end down to nothing, states anywhere in the pool, an entry without a sequence: rows behind
    an entry's end and every other state keep their bits."""
    x = inputs(60 + S, 6, S, 2, 4, 64, 64, n=9)
    ids = torch.tensor([7, 0, -1, 3, 8, 2], dtype=torch.int32)
    lens = torch.tensor([S, max(1, S // 2), S, 0, 10 * S, -4], dtype=torch.int32)
    before = x["state"].clone()
    want, new = reference(x, ids.long().clamp(min=0), lens)
    out = out_like(x, fill=3.25)
    call(x, out, seq_lens=lens.cuda(), state_ids=ids.cuda())
    torch.cuda.synchronize()
    for i in range(6):
        n = 0 if ids[i] < 0 else min(max(int(lens[i]), 0), S)
        assert bool((out[i, n:] == 3.25).all()), f"entry {i}: rows behind its end were written"
        if n:
            assert_rounded(out[i, :n], want[i, :n], f"entry {i}")
            assert_state(x["state"][ids[i]], new[i], n, f"entry {i}")
    used = [int(j) for j, n in zip(ids, lens) if j >= 0 and n > 0]
    for j in range(9):
        if j not in used:
            assert torch.equal(x["state"][j], before[j]), f"state {j} was touched"


@pytest.mark.parametrize("S", [1, 80])
def test_wrong_and_repeated_states(S):
    """A state that is not there, or an earlier entry's: NaN in the entry's rows, and the states as the others leave them."""
    x = inputs(70 + S, 5, S, 1, 2, 64, 64, n=6)
    ids = torch.tensor([4, 6, 4, 1, 1 << 30], dtype=torch.int32)
    lens = torch.tensor([S, S, max(1, S - 3), S, S], dtype=torch.int32)
    before = x["state"].clone()
    want, new = reference(x, ids.long().clamp(max=5), lens)
    out = out_like(x, fill=1.5)
    call(x, out, seq_lens=lens.cuda(), state_ids=ids.cuda())
    torch.cuda.synchronize()
    for i in (0, 3):
        assert_rounded(out[i], want[i], f"entry {i}")
        assert_state(x["state"][ids[i]], new[i], S, f"entry {i}")
    for i in (1, 2, 4):
        n = int(lens[i])
        assert bool(torch.isnan(out[i, :n]).all()) and bool((out[i, n:] == 1.5).all()), f"entry {i}"
    for j in (0, 2, 3, 5):
        assert torch.equal(x["state"][j], before[j])


@pytest.mark.parametrize("S,t", [(4, 2), (70, 40), (150, 64), (150, 77), (200, 131)])
@pytest.mark.parametrize("what", ["v", "k", "q", "b", "a"])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_nan_and_infinity_stay_behind_their_token(S, t, what, bad):
    """Outputs before a NaN or infinite input keep their values; other heads (and, for v, other columns) keep all of them."""
    x = inputs(80 + S, 1, S, 2, 4, 64, 64, raw=False)
    want, _ = reference(x)
    x[what] = x[what].clone()
    if what in "ab":
        x[what][0, t, 1] = -bad if what == "a" and bad != math.inf else bad
    else:
        x[what][0, t, 1, 5] = bad
    out = out_like(x)
    call(x, out)
    torch.cuda.synchronize()
    hit = {"a": [1], "b": [1], "v": [1], "q": [2, 3], "k": [2, 3]}[what]
    for h in range(4):
        if h not in hit:
            assert_rounded(out[:, :, h], want[:, :, h], f"head {h}")
    for h in hit:
        assert_rounded(out[:, :t, h], want[:, :t, h], f"head {h} before")
        if what == "v":
            keep = [c for c in range(64) if c != 5]
            assert_rounded(out[:, :, h][..., keep], want[:, :, h][..., keep], f"head {h}, other columns")
            assert not bool(torch.isfinite(out[0, t, h, 5]))
            assert not bool(torch.isfinite(out[0, t:, h, 5]).any()) or bad == math.inf
        elif what == "q":
            assert_rounded(out[:, t + 1 :, h], want[:, t + 1 :, h], f"head {h} after")
            assert not bool(torch.isfinite(out[0, t, h]).any())
        else:
            assert not bool(torch.isfinite(out[0, t, h]).all())


@pytest.mark.parametrize("S", [3, 90])
def test_decays_that_clear_the_state(S):
    """-inf and very negative log decays: nothing of the state before is left, and what follows is as exact as ever."""
    x = inputs(90 + S, 1, S, 1, 3, 64, 64, raw=False)
    x["a"][0, 1, 0] = -math.inf
    x["a"][0, S // 2, 1] = -1e30
    x["a"][0, 1:, 2] = -1000.0
    check(x, f"clearing, S={S}")


@pytest.mark.parametrize("S", [5, 130])
def test_equal_keys_and_full_writes(S):
    """Every key the same and beta 1: a chunk's triangle is all ones below its diagonal."""
    x = inputs(95 + S, 1, S, 1, 2, 128, 64, raw=False)
    x["k"][:] = x["k"][:, :1].clone()
    x["b"][:] = 1.0
    x["a"][:] = 0.0
    check(x, f"equal keys, S={S}")


def test_zero_keys_and_closed_gates():
    x = inputs(97, 1, 100, 1, 2, 64, 64, raw=False)
    x["k"][:, 10:40] = 0
    x["b"][:, 30:70] = 0
    check(x, "zero keys")


@pytest.mark.parametrize("parts", [(200,), (1,) * 5 + (195,), (64, 64, 72), (130, 70), (8, 100, 92)])
def test_turns_add_up(parts):
    """A prompt cut into calls anywhere leaves what one call leaves."""
    x = inputs(99, 1, 200, 2, 4, 128, 128)
    want, new = reference(x)
    out = out_like(x)
    at = 0
    for n in parts:
        y = dict(x, **{c: x[c][:, at : at + n] for c in ("q", "k", "v", "a", "b")})
        call(y, out[:, at : at + n])
        at += n
    torch.cuda.synchronize()
    assert_rounded(out, want, f"{parts}")
    assert_state(x["state"], new, 200, f"{parts}")


@pytest.mark.parametrize("S", [2, 75])
def test_far_states(S):
    """States behind 2^31 elements of the pool."""
    n = 2100
    pool = torch.empty(n, 8, 128, 128 * 8, dtype=torch.float32, device="cuda").view(n * 8, 8, 128, 128)
    x = inputs(101, 2, S, 4, 8, 128, 128)
    ids = torch.tensor([n * 8 - 1, 3], dtype=torch.int32)
    pool[ids.long().cuda()] = x["state"]
    want, new = reference(x)
    out = out_like(x)
    x["state"] = pool
    call(x, out, state_ids=ids.cuda())
    torch.cuda.synchronize()
    assert_rounded(out, want, "far")
    assert_state(pool[ids.long().cuda()], new, S, "far")


@pytest.mark.parametrize("S", [1, 100])
def test_graph_replays(S):
    """A captured call, replayed with new inputs in its buffers: each replay is the eager call's bits."""
    x = inputs(110, 2, S, 2, 4, 128, 128)
    need = paged.gated_delta_workspace_bytes(2, S, 2, 4, 128, 128)
    ws = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
    out = out_like(x)
    call(x, out, workspace=ws)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        call(x, out, workspace=ws)
    for i in range(4):
        y = inputs(120 + i, 2, S, 2, 4, 128, 128)
        for c in ("q", "k", "v", "a", "b", "state"):
            x[c].copy_(y[c])
        ws.fill_(255 if i % 2 else 0)
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        got, left = out.clone(), x["state"].clone()
        y["a_log"], y["dt_bias"] = x["a_log"], x["dt_bias"]
        eager = out_like(y)
        call(y, eager)
        torch.cuda.synchronize()
        assert torch.equal(got, eager) and torch.equal(left, y["state"]), f"replay {i}"


@pytest.mark.parametrize("S", [1, 130])
def test_other_stream_and_repeats(S):
    """On a stream of the caller's, twice: the same bits, whatever runs on the current stream."""
    x = inputs(130, 1, S, 2, 4, 128, 128)
    first = x["state"].clone()
    want, new = reference(x)
    outs = []
    stream = torch.cuda.Stream()
    for _ in range(2):
        x["state"].copy_(first)
        out = out_like(x)
        torch.cuda.synchronize()
        call(x, out, stream=stream)
        junk = torch.full((1 << 22,), 255, dtype=torch.uint8, device="cuda")
        stream.synchronize()
        outs.append((out, x["state"].clone()))
        del junk
    assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])
    assert_rounded(outs[0][0], want, "stream")
    assert_state(outs[0][1], new, S, "stream")


@pytest.mark.parametrize("S", [1, 2, 28, 29])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_many_heads(S, dtype):
    """Enough heads for the wider waves, on both sides of the line between tokens and chunks."""
    check(inputs(160 + S, 64, S, 2, 4, 64 if S > 2 else 128, 128, dtype), f"many heads, S={S}")


@pytest.mark.parametrize("S", [4, 90, 150])
def test_padding_holds_nan(S):
    """What lies behind an entry's end never counts."""
    x = inputs(170 + S, 3, S, 2, 4, 64, 64)
    lens = torch.tensor([S, S // 2, 3], dtype=torch.int32)
    want, new = reference(x, None, lens)
    for c in ("q", "k", "v", "a", "b"):
        x[c] = x[c].clone()
        for i in range(3):
            x[c][i, int(lens[i]) :] = math.nan
    out = out_like(x, fill=-1.0)
    call(x, out, seq_lens=lens.cuda())
    torch.cuda.synchronize()
    for i in range(3):
        n = int(lens[i])
        assert_rounded(out[i, :n], want[i, :n], f"entry {i}")
        assert_state(x["state"][i], new[i], n, f"entry {i}")
        assert bool((out[i, n:] == -1.0).all())


@pytest.mark.parametrize("B,S,Hv,lens", [(1, 6400, 64, None), (3, 1600, 96, None), (2, 3300, 96, [3300, 1000])])
def test_more_than_one_launch_holds(B, S, Hv, lens):
    """Calls whose chunks or entries go through several launches: the bits of shorter calls, cut at whole chunks (the
    state passes between calls as it passes between launches)."""
    x = inputs(180 + B, B, S, Hv // 2, Hv, 64, 64)
    first = x["state"].clone()
    ln = torch.tensor(lens, dtype=torch.int32) if lens else None
    whole = out_like(x, fill=2.0)
    call(x, whole, **(dict(seq_lens=ln.cuda()) if lens else {}))
    end = x["state"].clone()
    x["state"].copy_(first)
    parts, at = out_like(x, fill=2.0), 0
    for n in (64, 640, 320, S - 1024):
        y = dict(x, **{c: x[c][:, at : at + n] for c in ("q", "k", "v", "a", "b")})
        call(y, parts[:, at : at + n], **(dict(seq_lens=(ln - at).cuda()) if lens else {}))
        at += n
    torch.cuda.synchronize()
    assert torch.equal(whole, parts) and torch.equal(end, x["state"])
    assert bool(torch.isfinite(end).all())


@pytest.mark.parametrize("S", [1, 5, 70, 200])
def test_out_is_v(S):
    x = inputs(190 + S, 2, S, 2, 4, 64, 128)
    want, new = reference(x)
    call(x, x["v"])
    torch.cuda.synchronize()
    assert_rounded(x["v"], want, "out is v")
    assert_state(x["state"], new, S, "out is v")


def test_out_is_v_where_tokens_run_alone():
    """A chunk that runs token by token, written over its own v."""
    x = inputs(195, 1, 150, 1, 2, 64, 64, raw=False)
    x["v"][0, 80, 0, 3] = math.nan
    want, _ = reference(x)
    call(x, x["v"])
    torch.cuda.synchronize()
    keep = [c for c in range(64) if c != 3]
    assert_rounded(x["v"][..., keep], want[..., keep], "other columns")
    assert_rounded(x["v"][:, :80], want[:, :80], "before")
    assert bool(torch.isnan(x["v"][0, 80:, 0, 3]).all())


def test_two_streams_and_a_shared_workspace_in_order():
    """Two calls at once, each with its own workspace; then two graphs that share one, replayed in turn."""
    xs = [inputs(200 + i, 1, 300, 2, 4, 128, 128) for i in range(2)]
    refs = [reference(x) for x in xs]
    firsts = [x["state"].clone() for x in xs]
    outs = [out_like(x) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    for x, out, s in zip(xs, outs, streams):
        call(x, out, stream=s)
    torch.cuda.synchronize()
    for x, out, (want, new) in zip(xs, outs, refs):
        assert_rounded(out, want, "at once")
        assert_state(x["state"], new, 300, "at once")
    eager = [(o.clone(), x["state"].clone()) for o, x in zip(outs, xs)]
    ws = torch.empty(paged.gated_delta_workspace_bytes(1, 300, 2, 4, 128, 128), dtype=torch.uint8, device="cuda")
    graphs = []
    for x, out in zip(xs, outs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call(x, out, workspace=ws)
        graphs.append(g)
    for _ in range(3):
        for x, f, out in zip(xs, firsts, outs):
            x["state"].copy_(f)
            out.zero_()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for x, out, (o, s) in zip(xs, outs, eager):
            assert torch.equal(out, o) and torch.equal(x["state"], s)


def test_large_and_small_values():
    """Keys, values and states far from 1: the normalised keys' scale does not matter, the values' goes through."""
    for scale in (1e-18, 1e18):
        x = inputs(210, 1, 100, 1, 2, 64, 64)
        x["v"].mul_(scale)
        x["state"].mul_(scale)
        x["k"].mul_(2.0 ** 20 if scale > 1 else 2.0 ** -5)
        x["q"].mul_(2.0 ** -5)
        check(x, f"values of {scale}")


# more chains of 16 columns than CUs: two per workgroup
@pytest.mark.parametrize("Dk,Dv", [(64, 64), (64, 128), (128, 64), (128, 128)])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("layout", ["token", "wide"])
def test_paired_chains(Dk, Dv, dtype, layout):
    """A padded batch over a pool: a whole entry, a short one, one behind its first chunk, an empty one, one without a
    sequence, a repeated state."""
    Hv = 16 * 64 // Dv
    S, B = 140, 6
    x = inputs(230 + Dk + Dv, B, S, Hv // 2, Hv, Dk, Dv, dtype, n=8, layout=layout)
    ids = torch.tensor([5, 0, 7, 2, -1, 0], dtype=torch.int32)
    lens = torch.tensor([S, 30, 65, 0, S, 100], dtype=torch.int32)
    before = x["state"].clone()
    want, new = reference(x, ids.long().clamp(min=0), lens)
    out = out_like(x, fill=3.25)
    call(x, out, seq_lens=lens.cuda(), state_ids=ids.cuda())
    torch.cuda.synchronize()
    for i in range(3):
        n = int(lens[i])
        assert bool((out[i, n:] == 3.25).all())
        assert_rounded(out[i, :n], want[i, :n], f"entry {i}")
        assert_state(x["state"][ids[i]], new[i], n, f"entry {i}")
    assert bool((out[3:5] == 3.25).all())
    assert bool(torch.isnan(out[5, :100]).all()) and bool((out[5, 100:] == 3.25).all())
    for j in (1, 2, 3, 4, 6):
        assert torch.equal(x["state"][j], before[j])


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("column", [5, 20])
def test_paired_chains_where_tokens_run_alone(dtype, column):
    """A NaN in one chain of a pair sends the chunk of both token by token, written over v; then whole chunks again."""
    x = inputs(260 + column, 2, 200, 20, 40, 64, 64, dtype, raw=False)
    x["v"][1, 70, 3, column] = math.nan
    x["k"][0, 150, 7] = math.inf
    want, _ = reference(x)
    call(x, x["v"])
    torch.cuda.synchronize()
    got = x["v"]
    assert bool(torch.isnan(got[1, 70:, 3, column]).all())
    keep = [c for c in range(64) if c != column]
    assert_rounded(got[1, :, 3][:, keep], want[1, :, 3][:, keep], "other columns")
    assert_rounded(got[1, :70, 3], want[1, :70, 3], "before")
    others = [h for h in range(40) if h != 3]
    assert_rounded(got[1][:, others], want[1][:, others], "other heads")
    assert_rounded(got[0, :150], want[0, :150], "before the key")
    others = [h for h in range(40) if h not in (14, 15)]
    assert_rounded(got[0][:, others], want[0][:, others], "heads of other keys")
    assert not bool(torch.isfinite(got[0, 150, 14:16]).any())


def test_paired_chains_replayed():
    x = inputs(270, 3, 100, 24, 24, 64, 64)
    first, out = x["state"].clone(), out_like(x)
    call(x, out)
    want, new = out.clone(), x["state"].clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call(x, out)
    for _ in range(4):
        x["state"].copy_(first)
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(x["state"], new)


@pytest.mark.parametrize("S", [5, 100, 200])
@pytest.mark.parametrize("factor", [4, 16, 256])
def test_keys_far_above_one(S, factor):
    """Keys that are not normalised: a token's part grows by 1 - |k|^2 with every later one, as in the rule, and the
    inverse of a whole chunk would overflow.  Only the last tokens have a value, so that the rule itself stays finite."""
    x = inputs(160 + S, 1, S, 1, 2, 64, 64, raw=False, l2=False)
    x["k"][:] = x["k"][:, :1] * factor
    x["b"][:] = 1.0
    x["a"][:] = 0.0
    x["v"][:, : S - 3] = 0
    x["state"][:] = 0
    check(x, f"keys of {factor}, S={S}")


@pytest.mark.parametrize("S", [6, 64, 150])
@pytest.mark.parametrize("grow", [0.5, 5.0])
def test_growing_states(S, grow):
    """Positive log decays: the state grows, and by more than fp32 holds where nothing has been written yet."""
    x = inputs(165 + S, 1, S, 1, 2, 64, 64, raw=False)
    n = min(30, S // 2)
    x["a"][:, :n] = grow
    x["v"][:, :n] = 0
    x["state"][:] = 0
    check(x, f"growing by {grow}, S={S}")


def test_large_betas():
    for beta in (-3.0, 100.0, 1e30):
        x = inputs(170, 1, 80, 1, 2, 64, 64, raw=False)
        x["b"][0, 70, 0] = beta
        x["v"][0, 71:] = 0
        x["b"][0, 71:] = 0
        x["a"][0, 71:] = 0
        check(x, f"beta {beta}")


def test_nothing_to_do():
    x = inputs(140, 2, 4, 1, 2, 64, 64)
    before = x["state"].clone()
    y = dict(x, **{c: x[c][:, :0] for c in ("q", "k", "v", "a", "b")})
    call(y, out_like(x)[:, :0])
    y = dict(x, **{c: x[c][:0] for c in ("q", "k", "v", "a", "b")})
    call(y, out_like(x)[:0])
    torch.cuda.synchronize()
    assert torch.equal(before, x["state"])


def test_python_refusals():
    x = inputs(150, 1, 4, 2, 4, 64, 64)
    out = out_like(x)
    for key, bad in [("k", x["k"].half()), ("v", x["v"][..., ::2]), ("a", x["a"].float()), ("state", x["state"].half()),
                     ("state", x["state"].transpose(2, 3)), ("a_log", None), ("dt_bias", x["dt_bias"][:2])]:
        with pytest.raises(ValueError):
            call(dict(x, **{key: bad}), out)
    with pytest.raises(ValueError):
        call(x, out[:, :3])
    with pytest.raises(ValueError):
        call(x, out, seq_lens=torch.tensor([4], dtype=torch.int64, device="cuda"))
    with pytest.raises(paged.GenllmError):
        call(dict(x, q=torch.zeros(4 * 128 + 4, dtype=BF16, device="cuda")[4:].view(1, 4, 2, 64)), out)  # 8-byte aligned
    assert half_step(BF16) == 2.0 ** -8
