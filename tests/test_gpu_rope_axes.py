"""q/k norms with the rotation on several axes on the GPU against their definition in 64 bits."""
import pytest
import torch

from genllm_amd import paged
from hybrid import assert_rounded, norm_rope_axes

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16
EPS = 1e-6
# a pair's two products and their sum, the norm's factor and gamma: a few half steps of fp32 of the row's largest value
SLACK = 2.0 ** -20


def inputs(seed, S, Hq, Hk, D, rope, axes, dtype=BF16, rows=300):
    g = torch.Generator().manual_seed(seed)
    qk = torch.randn(S, (Hq + Hk) * D, generator=g).to(dtype).cuda()
    cos, sin = paged.rope_cache(1e6, rope, rows)
    return {"q": qk[:, : Hq * D].view(S, Hq, D), "k": qk[:, Hq * D :].view(S, Hk, D),
            "gamma_q": (torch.rand(D, generator=g) + 0.5).cuda(), "gamma_k": (torch.rand(D, generator=g) + 0.5).cuda(),
            "cos": torch.from_numpy(cos).cuda(), "sin": torch.from_numpy(sin).cuda(),
            "pos": torch.randint(0, rows, (axes, S), generator=g, dtype=torch.int32).cuda()}


def check(x, sections, interleaved, label, norm=True, head_major=True):
    gq, gk = (x["gamma_q"], x["gamma_k"]) if norm else (None, None)
    outs = []
    for c in "qk":
        S, H, D = x[c].shape
        o = torch.zeros(H, S, D, dtype=x[c].dtype, device="cuda").transpose(0, 1) if head_major else torch.zeros_like(x[c])
        outs.append(o)
    paged.qk_norm_rope_axes(x["q"], x["k"], outs[0], outs[1], gq, gk, EPS, x["cos"], x["sin"], x["pos"], sections, interleaved)
    torch.cuda.synchronize()
    for c, o, gamma in zip("qk", outs, (gq, gk)):
        want = norm_rope_axes(x[c], gamma, EPS, x["cos"], x["sin"], x["pos"], sections, interleaved)
        assert_rounded(o, want, f"{label} {c}", SLACK)


@pytest.mark.parametrize("S", [1, 2, 5, 33, 200])
@pytest.mark.parametrize("Hq,Hk,D,rope,sections,interleaved", [
    (8, 2, 256, 64, (11, 11, 10), True), (8, 2, 256, 256, (32, 48, 48), False), (32, 8, 128, 128, (16, 24, 24), False),
    (32, 8, 128, 128, (22, 21, 21), True), (5, 1, 128, 64, (32,), False), (3, 3, 64, 64, (10, 22), False),
    (1, 1, 64, 16, (2, 2, 2, 2), True), (7, 2, 256, 48, (0, 24), False), (4, 4, 64, 32, (6, 5, 5), True)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_shapes(S, Hq, Hk, D, rope, sections, interleaved, dtype):
    check(inputs(S + D + rope, S, Hq, Hk, D, rope, len(sections), dtype), sections, interleaved, f"S={S} D={D}/{rope}",
          head_major=S != 5)


@pytest.mark.parametrize("S", [3, 70])
def test_without_norm(S):
    check(inputs(1, S, 8, 2, 256, 64, 3), (11, 11, 10), True, "no norm", norm=False)


@pytest.mark.parametrize("S", [1, 150])
def test_equal_axes_are_the_one_axis_rope(S):
    """The same position on every axis: the framework's own rotation, bit for bit."""
    x = inputs(2, S, 8, 2, 128, 128, 3)
    x["pos"][:] = torch.arange(S, dtype=torch.int32, device="cuda") + 9
    out = torch.zeros(8, S, 128, dtype=BF16, device="cuda")
    paged.qk_norm_rope_axes(x["q"], None, out.transpose(0, 1), None, None, None, EPS, x["cos"], x["sin"], x["pos"],
                            (22, 21, 21), True)
    want = torch.zeros_like(out)
    paged.apply_rope(want, x["q"].transpose(0, 1).contiguous(), x["cos"], x["sin"], 9)
    torch.cuda.synchronize()
    assert torch.equal(out, want)


def test_in_place_and_q_alone():
    x = inputs(3, 50, 8, 2, 256, 64, 3)
    q, k = x["q"].clone(), x["k"].clone()
    paged.qk_norm_rope_axes(x["q"], x["k"], x["q"], x["k"], x["gamma_q"], x["gamma_k"], EPS, x["cos"], x["sin"], x["pos"],
                            (11, 11, 10), True)
    torch.cuda.synchronize()
    for c, was, gamma in (("q", q, x["gamma_q"]), ("k", k, x["gamma_k"])):
        assert_rounded(x[c], norm_rope_axes(was, gamma, EPS, x["cos"], x["sin"], x["pos"], (11, 11, 10), True), c, SLACK)


@pytest.mark.parametrize("S", [4, 130])
def test_positions_outside_the_tables(S):
    """NaN in the pairs of the axis whose position is outside, and nowhere else."""
    x = inputs(4, S, 8, 2, 256, 64, 3)
    x["pos"][1, 2] = 300
    x["pos"][0, 3] = -1
    x["pos"][2, 0] = -(1 << 31)
    x["pos"][2, 1] = (1 << 31) - 1
    check(x, (11, 11, 10), True, "outside")


def test_special_rows():
    x = inputs(5, 6, 8, 2, 256, 64, 3)
    x["q"][1] = 0
    x["q"][2, 3, 7] = float("nan")
    x["q"][3, 4] = 2.0 ** -60
    check(x, (11, 11, 10), True, "special")


def test_graph_replays():
    x = inputs(6, 20, 8, 2, 256, 64, 3)
    outs = [torch.zeros_like(x["q"]), torch.zeros_like(x["k"])]
    args = (x["q"], x["k"], *outs, x["gamma_q"], x["gamma_k"], EPS, x["cos"], x["sin"], x["pos"], (11, 11, 10), True)
    paged.qk_norm_rope_axes(*args)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        paged.qk_norm_rope_axes(*args)
    for i in range(3):
        y = inputs(7 + i, 20, 8, 2, 256, 64, 3)
        for c in ("q", "k", "pos"):
            x[c].copy_(y[c])
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in outs]
        paged.qk_norm_rope_axes(*args)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, outs))


@pytest.mark.parametrize("S,Hq,Hk,D", [(700, 40, 8, 256), (3000, 12, 4, 128), (1, 70, 9, 256), (5, 200, 60, 64)])
def test_many_rows(S, Hq, Hk, D):
    """Several rows per lane, and tokens with more heads than a workgroup has rows."""
    check(inputs(20, S, Hq, Hk, D, 64, 3, rows=64), (11, 11, 10), True, f"{S} x {Hq}+{Hk} of {D}")


def test_other_stream():
    x = inputs(21, 40, 8, 2, 256, 64, 3)
    outs = [torch.zeros_like(x["q"]), torch.zeros_like(x["k"])]
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    paged.qk_norm_rope_axes(x["q"], x["k"], *outs, x["gamma_q"], x["gamma_k"], EPS, x["cos"], x["sin"], x["pos"],
                            (11, 11, 10), True, stream=stream)
    stream.synchronize()
    for c, o in zip("qk", outs):
        want = norm_rope_axes(x[c], x["gamma_" + c], EPS, x["cos"], x["sin"], x["pos"], (11, 11, 10), True)
        assert_rounded(o, want, c, SLACK)


def test_python_refusals():
    x = inputs(8, 4, 2, 1, 64, 64, 3)
    o, p = torch.zeros_like(x["q"]), torch.zeros_like(x["k"])

    def go(**kw):
        a = dict(q=x["q"], k=x["k"], q_out=o, k_out=p, gamma_q=None, gamma_k=None, eps=EPS, cos=x["cos"], sin=x["sin"],
                 positions=x["pos"], sections=(12, 10, 10))
        paged.qk_norm_rope_axes(**dict(a, **kw))

    go()
    for kw in (dict(q_out=o.half()), dict(k_out=p[:3]), dict(sin=x["sin"][:5]), dict(positions=x["pos"].long()),
               dict(sections=(16, 16)), dict(gamma_q=x["gamma_q"].half())):
        with pytest.raises(ValueError):
            go(**kw)
    for kw in (dict(sections=(12, 10, 9)), dict(sections=(2, 15, 15), interleaved=True), dict(eps=-1.0)):
        with pytest.raises(paged.GenllmError):
            go(**kw)
