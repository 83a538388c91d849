"""Batch operators over tables that have no page yet."""
import pytest
import torch

from genllm_amd import paged

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("S", [1, 20, 60])
@pytest.mark.parametrize("f8", [True, False])
@pytest.mark.parametrize("causal", [True, False])
def test_attention_without_pages(S, f8, causal):
    """No entry has a key, whatever its length says: zeros."""
    H, D = 2, 128
    ids = torch.zeros(3, 0, dtype=torch.int32, device="cuda")
    (kp, ks), (vp, vs) = (paged.f8_pool(4, H, D) if f8 else (torch.ones(4, 16, H, D, dtype=BF, device="cuda"), None) for _ in "kv")
    q = torch.ones(3, S, 4, D, dtype=BF, device="cuda")
    out = torch.full_like(q, 2.5)
    paged.paged_attention_batch(q, out, kp, vp, ids, ids, ints([0, S, 100]), 1.0, q_lens=ints([S, S, S - 1]), k_scales=ks, v_scales=vs, causal=causal)
    torch.cuda.synchronize()
    assert bool((out[:2] == 0).all()) and bool((out[2, : S - 1] == 0).all()) and bool((out[2, S - 1 :] == 2.5).all())


def test_rows_without_pages():
    """Rows written past the table are dropped, rows read past it are NaN."""
    H, D = 2, 64
    ids = torch.zeros(2, 0, dtype=torch.int32, device="cuda")
    (kp, ks), (vp, vs) = (paged.f8_pool(4, H, D) for _ in "kv")
    x = torch.ones(2, 20, H, D, dtype=BF, device="cuda")
    paged.kv_scatter_f8(x, x, kp, vp, ks, vs, ids, ids, ints([0, 30]))
    torch.cuda.synchronize()
    assert not any(bool(t.view(torch.uint8).any()) for t in (kp, vp, ks, vs))
    out = [torch.full_like(x, 2.5) for _ in "kv"]
    paged.kv_gather_f8(kp, vp, ks, vs, ids, ids, ints([0, 30]), *out, seq_lens=ints([20, 3]))
    torch.cuda.synchronize()
    for y in out:
        assert bool(torch.isnan(y[0]).all()) and bool(torch.isnan(y[1, :3]).all()) and bool((y[1, 3:] == 2.5).all())
