"""The rotation on views of one buffer that share no element, and in place on them."""
import pytest
import torch

from genllm_amd import paged
from hybrid import assert_rounded, norm_rope_axes
from test_gpu_rope_axes import EPS, SLACK, inputs

pytestmark = pytest.mark.gpu

SECTIONS = (11, 11, 10)


@pytest.mark.parametrize("S", [1, 40])
@pytest.mark.parametrize("order", ["token", "head"])
@pytest.mark.parametrize("in_place", [False, True])
def test_one_buffer(S, order, in_place):
    x = inputs(30 + S, S, 8, 2, 256, 64, 3)
    H = 10 if in_place else 20
    buf = torch.full((S, H, 256) if order == "token" else (H, S, 256), 5.0, dtype=torch.bfloat16, device="cuda")
    rows = buf if order == "token" else buf.transpose(0, 1)
    rows[:, :8], rows[:, 8:10] = x["q"], x["k"]
    q, k = rows[:, :8], rows[:, 8:10]
    qo, ko = (q, k) if in_place else (rows[:, 10:18], rows[:, 18:])
    paged.qk_norm_rope_axes(q, k, qo, ko, x["gamma_q"], x["gamma_k"], EPS, x["cos"], x["sin"], x["pos"], SECTIONS, True)
    torch.cuda.synchronize()
    for c, o in (("q", qo), ("k", ko)):
        want = norm_rope_axes(x[c], x["gamma_" + c], EPS, x["cos"], x["sin"], x["pos"], SECTIONS, True)
        assert_rounded(o, want, f"{order} {c}", SLACK)
    if not in_place:
        assert torch.equal(q, x["q"]) and torch.equal(k, x["k"])
