"""The hybrid layers' operators as a model runs them: a linear layer's convolution and delta rule over a prompt and the
tokens after it, and an attention layer's norm and rotation on several axes in front of the paged cache."""
import math

import pytest
import torch

from genllm_amd import paged
from hybrid import assert_rounded, assert_state, causal_conv, delta_rule, norm_rope_axes

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_linear_layer_prompt_then_tokens(dtype):
    """conv -> split -> delta rule over a ragged batch of prompts, then three tokens each with both states kept."""
    B, S, Hk, Hv, D, W = 3, 150, 2, 4, 64, 4
    C = 2 * Hk * D + Hv * D
    g = torch.Generator().manual_seed(1)
    w = (torch.randn(C, W, generator=g) * 0.5).to(dtype).cuda()
    a_log = torch.log(torch.rand(Hv, generator=g) * 15 + 1).cuda()
    dt_bias = (torch.rand(Hv, generator=g) * -4 - 1).cuda()
    ids = torch.tensor([3, 0, 4], dtype=torch.int32).cuda()
    lens = torch.tensor([150, 41, 3], dtype=torch.int32).cuda()
    conv_state = torch.zeros(5, W - 1, C, dtype=dtype, device="cuda")
    state = torch.zeros(5, Hv, D, D, device="cuda")
    ref_conv, ref_state = torch.zeros(B, W - 1, C).double(), torch.zeros(B, Hv, D, D).double()
    for step, n in enumerate((S, 1, 1, 1)):
        x = torch.randn(B, n, C, generator=g).to(dtype).cuda()
        ab = torch.randn(B, n, 2 * Hv, generator=g).to(dtype).cuda()
        ln = lens if step == 0 else None
        y = torch.zeros_like(x)
        paged.causal_conv(x, w, y, conv_state, seq_lens=ln, state_ids=ids)
        want_y, ref_conv = causal_conv(x, w, ref_conv, lens=ln)
        q, k, v = (t.view(B, n, -1, D) for t in torch.split(y, [Hk * D, Hk * D, Hv * D], -1))
        out = torch.zeros(B, n, Hv, D, dtype=dtype, device="cuda")
        paged.gated_delta_rule(q, k, v, ab[..., :Hv], ab[..., Hv:], state, out, D ** -0.5, a_log=a_log, dt_bias=dt_bias,
                               l2_eps=1e-6, seq_lens=ln, state_ids=ids)
        torch.cuda.synchronize()
        # each operator from what it was given: the rule from the convolution's rounded outputs
        want, ref_state = delta_rule(q, k, v, ab[..., :Hv], ab[..., Hv:], ref_state, D ** -0.5, a_log, dt_bias, 1e-6, ln)
        for i in range(B):
            m = int(lens[i]) if step == 0 else 1
            assert_rounded(y[i, :m], want_y[i, :m], f"conv step {step}", 2.0 ** -16)
            assert_rounded(out[i, :m], want[i, :m], f"rule step {step}")
        assert torch.equal(conv_state[ids.long()].cpu().double(), ref_conv)
        assert_state(state[ids.long()], ref_state, S + step, f"state step {step}")


def test_attention_layer_with_an_image_prompt():
    """norm + rotation on three axes -> page scatter -> prefill, then a decoded token, against attention in 64 bits."""
    S, Hq, Hkv, D, rope = 70, 8, 2, 256, 64
    sections = (11, 11, 10)
    g = torch.Generator().manual_seed(2)
    cos, sin = (torch.from_numpy(t).cuda() for t in paged.rope_cache(1e6, rope, 128))
    gq, gk = (torch.rand(D, generator=g) + 0.5).cuda(), (torch.rand(D, generator=g) + 0.5).cuda()
    pages = 5
    k_pool = torch.zeros(8, 16, Hkv, D, dtype=torch.bfloat16, device="cuda")
    v_pool = torch.zeros_like(k_pool)
    k_ids = torch.tensor([6, 1, 4, 0, 3], dtype=torch.int32, device="cuda")
    v_ids = torch.tensor([2, 7, 5, 1, 0], dtype=torch.int32, device="cuda")
    keys, values, at = [], [], 0
    for n in (S, 1):
        q = torch.randn(n, Hq, D, generator=g).bfloat16().cuda()
        k = torch.randn(n, Hkv, D, generator=g).bfloat16().cuda()
        v = torch.randn(n, Hkv, D, generator=g).bfloat16().cuda()
        pos = torch.stack([torch.full((n,), 3 + at), 3 + at + torch.arange(n) // 8, 3 + at + torch.arange(n) % 8]).int().cuda()
        qr, kr = torch.zeros_like(q), torch.zeros_like(k)
        paged.qk_norm_rope_axes(q, k, qr, kr, gq, gk, 1e-6, cos, sin, pos, sections, True)
        paged.kv_scatter(kr, v, k_pool, v_pool, k_ids, v_ids, at)
        out = torch.zeros_like(q)
        form = paged.paged_prefill if n > 4 else paged.paged_decode
        form(qr, out, k_pool, v_pool, k_ids, v_ids, -(-(at + n) // 16), at + n, Hkv, D ** -0.5, q_layout="token")
        torch.cuda.synchronize()
        for x, r, gamma in ((q, qr, gq), (k, kr, gk)):
            assert_rounded(r, norm_rope_axes(x, gamma, 1e-6, cos, sin, pos, sections, True), "rotation", 2.0 ** -20)
        keys.append(kr.cpu().double())
        values.append(v.cpu().double())
        K, V = torch.cat(keys), torch.cat(values)
        want = torch.zeros(n, Hq, D, dtype=torch.float64)
        for h in range(Hq):
            s = qr.cpu().double()[:, h] @ K[:, h // (Hq // Hkv)].t() * D ** -0.5
            see = torch.arange(at + n)[None, :] <= at + torch.arange(n)[:, None]
            want[:, h] = torch.softmax(s.masked_fill(~see, -math.inf), -1) @ V[:, h // (Hq // Hkv)]
        # the attention kernels round the probabilities to bf16: 2^-8 of each, against the row's largest value
        assert_rounded(out, want, f"attention of {n}", 2.0 ** -7)
        at += n
    assert at <= 16 * pages
