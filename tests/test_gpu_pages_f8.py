"""Rows quantised into 8-bit pages and read back: bit for bit against the definition in 64 bits."""
import math

import pytest
import torch

from genllm_amd import paged
from batch import PAGE, scatter, values

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


class Pages:
    """K and V pools of one batch with scattered tables, on the GPU, and what the definition makes of them."""

    def __init__(self, B, P, H, D, layout="head", seed=0):
        g = torch.Generator().manual_seed(seed)
        n = B * P + 3
        self.ids = [torch.randperm(n, generator=g)[: B * P].view(B, P).int() for _ in "kv"]
        self.pools, self.scales, self.want, self.exps = [], [], [], []
        for _ in "kv":
            codes = torch.randint(0, 256, (n, 16, H, D), generator=g, dtype=torch.uint8)
            byte = torch.randint(100, 140, (n, H), generator=g, dtype=torch.uint8)
            if layout == "head":
                pool, scale = paged.f8_pool(n, H, D)
                assert not bool(pool.view(torch.uint8).any()) and not bool(scale.any())
            else:
                pool, scale = torch.empty(n, 16, H, D, dtype=torch.uint8, device="cuda"), torch.empty(n, H, dtype=torch.uint8, device="cuda")
                if layout == "apart":  # rows with other memory between them
                    pool = torch.zeros(n, 16, H + 1, D + 32, dtype=torch.uint8, device="cuda")[:, :, :H, 16 : 16 + D]
            pool.view(torch.uint8).copy_(codes)
            scale.copy_(byte)
            self.pools.append(pool), self.scales.append(scale)
            self.want.append(codes.view(torch.float8_e4m3fn).double()), self.exps.append(byte.int() - 127)
        self.dev = [i.cuda() for i in self.ids]

    def write(self, k, v, start, lens=None, **kw):
        dev = lambda x: None if x is None else torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
        paged.kv_scatter_f8(k, v, *self.pools, *self.scales, *self.dev, dev(start), seq_lens=dev(lens), **kw)
        for i, x in enumerate((k, v)):
            scatter(x, self.want[i], self.exps[i], self.ids[i], start, lens)

    def check(self, label):
        torch.cuda.synchronize()
        for i, kind in enumerate("KV"):
            got = self.pools[i].view(torch.uint8).cpu().view(torch.float8_e4m3fn).double()
            assert torch.equal(self.scales[i].cpu().int() - 127, self.exps[i]), f"{label}: {kind} scales"
            assert torch.equal(torch.isnan(got), torch.isnan(self.want[i])), f"{label}: {kind} NaN"
            assert torch.equal(got.nan_to_num(0), self.want[i].nan_to_num(0)), f"{label}: {kind} codes"

    def read(self, start, S, dtype, lens=None):
        H, D = self.pools[0].shape[2:]
        out = [torch.full((len(start), S, H, D), 2.5, dtype=dtype, device="cuda") for _ in "kv"]
        dev = lambda x: None if x is None else torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
        paged.kv_gather_f8(*self.pools, *self.scales, *self.dev, dev(start), *out, seq_lens=dev(lens))
        torch.cuda.synchronize()
        for i, kind in enumerate("KV"):
            table = values(self.pools[i], self.scales[i])
            for b, at in enumerate(start):
                n = S if lens is None else min(max(lens[b], 0), S)
                for s in range(S):
                    page, slot = (at + s) // PAGE, (at + s) % PAGE
                    row = out[i][b, s].cpu()
                    if s >= n or at < 0:
                        assert bool((row == 2.5).all()), f"{kind} entry {b} row {s} was written"
                        continue
                    block = int(self.ids[i][b, page]) if page < self.ids[i].shape[1] else -1
                    w = table[block, slot] if 0 <= block < table.shape[0] else torch.full((H, D), torch.nan).double()
                    w = w.float().to(dtype)  # a code times a power of two is exact in fp32
                    assert torch.equal(row.nan_to_num(7, 8, 9), w.nan_to_num(7, 8, 9)), f"{kind} entry {b} row {s}"


def rows(B, S, H, D, dtype, seed, std=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, S, H, D, generator=g) * std * torch.exp(2 * torch.randn(B, S, 1, 1, generator=g))
    return x.to(dtype).cuda()


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("H,D,layout", [(1, 64, "head"), (3, 128, "head"), (2, 256, "head"), (2, 128, "token"), (2, 64, "apart")])
def test_prompts_and_tokens(H, D, layout, dtype):
    """Prompts from a page's start and from inside one, then tokens one by one across pages."""
    p = Pages(4, 6, H, D, layout, seed=D + H)
    start, lens = [0, 16, 5, 31], [40, 33, 17, 1]
    p.write(rows(4, 40, H, D, dtype, 1), rows(4, 40, H, D, dtype, 2, 0.1), start, lens)
    p.check("prompts")
    at = [a + n for a, n in zip(start, lens)]
    for step in range(20):
        p.write(rows(4, 1, H, D, dtype, 10 + step), rows(4, 1, H, D, dtype, 40 + step, 0.1), at)
        p.check(f"token {step}")
        at = [a + 1 for a in at]
    p.read([0, 3, 16, 40], 37, dtype, [37, 20, 0, 1])
    p.read([0, 0, 0, 0], 60, BF if dtype == HF else HF)


@pytest.mark.parametrize("dtype", [BF, HF])
def test_strided_rows(dtype):
    """k and v as parts of a fused projection."""
    p = Pages(2, 3, 2, 128)
    x = rows(2, 20, 8, 128, dtype, 3)
    p.write(x[:, :, 4:6], x[:, :, 6:8], [0, 9])
    p.check("fused")
    p.write(x[:, :, 0:2].transpose(1, 2).contiguous().transpose(1, 2), x[:, :, 2:4], [20, 1], [3, 20])
    p.check("head by head")


@pytest.mark.parametrize("dtype", [BF, HF])
def test_special_values(dtype):
    """Zeros, the types' ends, NaN and infinities, subnormals, values at the borders between scales, ties."""
    p = Pages(1, 2, 1, 64)
    big = torch.finfo(dtype).max
    x = torch.zeros(1, 16, 1, 64)
    p.write(x.to(dtype).cuda(), x.to(dtype).cuda(), [0])
    p.check("zeros")
    p.write(torch.full((1, 1, 1, 64), 2.0 ** -7).to(dtype).cuda(), torch.full((1, 1, 1, 64), 2.0 ** -13).to(dtype).cuda(), [3])
    p.check("on zeros")
    y = torch.zeros(1, 5, 1, 64)
    y[0, 0, 0, :8] = torch.tensor([big, -big, math.inf, -math.inf, math.nan, 1.0, -0.0, torch.finfo(dtype).smallest_normal])
    y[0, 1, 0, 0], y[0, 2, 0, 0], y[0, 3, 0, 0] = 448.0, 449.0, 1.75 * 2.0 ** 9
    y[0, 4, 0] = torch.arange(64) / 32 + 1 / 64  # ties of the codes
    p.write(y.to(dtype).cuda(), y.flip(1).to(dtype).cuda(), [16])
    p.check("special")
    for r in range(5):
        p.write(y[:, r : r + 1].to(dtype).cuda(), y[:, r : r + 1].flip(3).to(dtype).cuda(), [r])
        p.check(f"special row {r}")
    tiny = torch.finfo(dtype).tiny * torch.rand(1, 16, 1, 64)
    p.write(tiny.to(dtype).cuda(), (tiny / 16).to(dtype).cuda(), [16])
    p.check("subnormal")
    p.read([0], 32, dtype)


def test_idle_and_bad():
    """Entries without tokens or with a negative start, ids that are no blocks, positions past the table."""
    p = Pages(6, 3, 2, 64, seed=5)
    p.ids[0][3, 1], p.ids[1][3, 1], p.ids[0][4, 0] = -1, p.pools[0].shape[0], 2 ** 30
    p.dev = [i.cuda() for i in p.ids]
    start, lens = [0, -1, 40, 8, 0, 2 ** 31 - 3], [0, 20, 20, 25, 20, 20]
    p.write(rows(6, 25, 2, 64, BF, 7), rows(6, 25, 2, 64, BF, 8), start, lens)
    p.check("idle and bad")
    p.read(start[:5] + [47], 25, BF, lens)
    p.write(rows(6, 25, 2, 64, BF, 7), rows(6, 25, 2, 64, BF, 8), [-(2 ** 31)] * 5 + [2 ** 31 - 1], [-5, 99, 1, 25, 3, 25])
    p.check("far off")


def test_scale_of_nan():
    """A scale byte of 255 is NaN for the whole page and stays so until the page begins anew."""
    p = Pages(1, 1, 1, 64)
    for i in range(2):
        p.scales[i].fill_(255)
    one = torch.ones(1, 1, 1, 64, dtype=BF, device="cuda")
    dev = torch.tensor([3], dtype=torch.int32, device="cuda")
    paged.kv_scatter_f8(one, one, *p.pools, *p.scales, *p.dev, dev)
    torch.cuda.synchronize()
    block = int(p.ids[0][0, 0])
    assert int(p.scales[0][block, 0]) == 255
    p.read([0], 16, BF)
    paged.kv_scatter_f8(one, one, *p.pools, *p.scales, *p.dev, dev - 3)
    torch.cuda.synchronize()
    assert int(p.scales[0][block, 0]) == 127 - 8  # 1 <= 448 * 2^-8


def test_far_blocks():
    """Blocks whose offset passes 32 bits."""
    n, H, D = 70000, 8, 256  # 2.3 GB of codes
    pools = [paged.f8_pool(n, H, D) for _ in "kv"]
    ids = torch.tensor([[n - 1, 65537]], dtype=torch.int32, device="cuda")
    k, v = rows(1, 20, H, D, BF, 1), rows(1, 20, H, D, BF, 2)
    zero = torch.zeros(1, dtype=torch.int32, device="cuda")
    paged.kv_scatter_f8(k, v, pools[0][0], pools[1][0], pools[0][1], pools[1][1], ids, ids, zero)
    out = [torch.zeros_like(k) for _ in "kv"]
    paged.kv_gather_f8(pools[0][0], pools[1][0], pools[0][1], pools[1][1], ids, ids, zero, *out)
    torch.cuda.synchronize()
    for x, y, (pool, scales) in zip((k, v), out, pools):
        codes, exps = torch.zeros(2, 16, H, D).double(), torch.zeros(2, H, dtype=torch.int32)
        scatter(x, codes, exps, torch.tensor([[0, 1]]), [0])
        want = codes * torch.ldexp(torch.ones(2, 1, H, 1).double(), exps[:, None, :, None])
        assert torch.equal(y[0].cpu().double(), want.view(32, H, D)[:20].to(BF).double())
        assert int(pool.view(torch.uint8).any((1, 2, 3)).sum()) == 2
