"""Attention of padded batches where fp32's and fp16's ranges end."""
import math

import pytest
import torch

from genllm_amd import paged
from batch import PAGE, assert_attended, attend
from hybrid import half_step

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


class Keys:
    """An entry of n tokens whose pages come from a pool of a few kinds of page, each a row of K and one of V (or
    [16, 64] of them) and V's exponent (8-bit pages); `kinds` gives the kind of each page.  D = 64, H kv heads with the same rows.  Other entries have a token
    each: with enough of them the long one's tiles are not split."""

    D = 64

    def __init__(self, kinds, k, v, S, dtype, f8, H=1, G=1, exps=None, n=None):
        m = k.shape[0]
        self.n, self.S, self.dtype, self.f8, self.H, self.G = n or len(kinds) * PAGE, S, dtype, f8, H, G
        self.kinds = torch.tensor(kinds)
        element = torch.float8_e4m3fn if f8 else dtype
        self.k, self.v = ((x if x.dim() == 3 else x[:, None]).to(element)[:, :, None].expand(m, PAGE, H, self.D) for x in (k, v))
        self.pools = [x.contiguous().cuda() for x in (self.k, self.v)]
        self.scales = [None, None]
        self.two = torch.ones(m).double()
        if f8:
            e = torch.zeros(m, dtype=torch.int32) if exps is None else torch.tensor(exps, dtype=torch.int32)
            self.two = torch.ldexp(torch.ones(m).double(), e)
            self.scales = [torch.full((m, H), 127, dtype=torch.uint8, device="cuda"), (e + 127).to(torch.uint8)[:, None].expand(m, H).contiguous().cuda()]
        self.ids = self.kinds.int()[None].cuda()

    def run(self, q, entries=1, **kw):
        """q [64], the same for every row."""
        out = torch.full((entries, self.S, self.H * self.G, self.D), 2.5, dtype=self.dtype, device="cuda")
        n, ids = torch.ones(entries, dtype=torch.int32), self.ids.expand(entries, -1)
        n[0] = self.n
        paged.paged_attention_batch(q.to(self.dtype).cuda().expand(out.shape).contiguous(), out, *self.pools, ids, ids, n.cuda(), 1.0,
                                    k_scales=self.scales[0], v_scales=self.scales[1], **kw)
        torch.cuda.synchronize()
        return out[0]

    def rows(self):
        v = self.v.double() * self.two[:, None, None, None]
        return [x[self.kinds].reshape(-1, self.H, self.D)[: self.n] for x in (self.k.double(), v)]


def scored(*logs):
    """q, and K rows whose scores with it are these, in log2 units (16 bits of q and K: to 2^-8 or so)."""
    q = torch.zeros(64)
    q[0] = 1.0
    k = torch.zeros(len(logs), 64)
    k[:, 0] = torch.tensor(logs) * math.log(2)
    return q, k


# Few rows; a draft of five; tiles of 64 rows; tiles of 128.
ROWS = [(1, 1), (5, 3), (20, 1), (40, 4)]


@pytest.mark.parametrize("pages", [40, 300])
@pytest.mark.parametrize("S,G", ROWS)
def test_large_values(S, G, pages):
    """Scores that rise by less than the running maximum follows, on values whose weighed sums then leave fp32's range
    though the sum of the values does not."""
    q, k = scored(0.0, 7.75)
    for e in range(104, 118 if pages == 40 else 115):
        kinds = [0] * 8 + [1] * (pages - 8)
        v = torch.full((2, 64), 1.5 * 2.0 ** e)
        v[:, 1::2] *= -1
        c = Keys(kinds, k, v, S, BF, False, G=G)
        assert float(c.rows()[1].abs().sum(0).max()) < 2.0 ** 127
        got = c.run(q)
        kk, vv = c.rows()
        # alike for all queries but for how many of the last keys they see, all of one kind: the first and the last stand for them
        for s in {0, S - 1}:
            want = attend(q.to(BF).expand(1, G, 64), kk, vv, c.n - S + s, 1.0)
            assert_attended(got[s : s + 1], *want, c.n, 2.0 ** -8, f"values of 2^{e}, query {s}")


@pytest.mark.parametrize("S,G,entries", [(1, 1, 1), (1, 1, 1408), (20, 1, 64), (40, 4, 64)])
def test_large_scales(S, G, entries):
    """The same over 8-bit pages, where V's scale rises by less than its reference follows; with many entries the long
    one is not split."""
    pages, H = 4096, 8
    q, k = scored(0.0, 7.5)
    k = k.to(torch.float8_e4m3fn).float()
    for e in (60, 74, 80, 88, 90, 92):
        v = torch.full((2, 64), 448.0)
        v[:, 1::2] *= -1
        c = Keys([0] * 8 + [1] * (pages - 8), k, v, S, BF, True, H, G, exps=[e, e + 6])
        kk, vv = c.rows()
        assert float(vv[:, 0].abs().sum(0).max()) < 2.0 ** 127
        got = c.run(q, entries)
        for s in {0, S - 1}:
            want = attend(q.to(BF).expand(1, G, 64), kk[:, :1], vv[:, :1], c.n - S + s, 1.0)
            for h in (0, H - 1):
                assert_attended(got[s : s + 1, G * h : G * h + G], *want, c.n, 2.0 ** -11, f"scales of 2^{e}, query {s}, head {h}")


def assert_small_weights(got, want, weight, plain, size, n, label):
    """assert_attended's bound with a probability's least step 2^-31 of the largest: they are formed relative to 2^-7 of
    it or less, so that fp16's step of 2^-24, off by up to 2^-25, leaves 2^-32."""
    g, w, a, b, z = (x.detach().cpu().double() for x in (got, want, weight, plain, size))
    part = 2.0 ** -11 + (264 * z + 2 * n) * 2.0 ** -24
    bound = half_step(got.dtype) * (1 + 2.0 ** -6) * w.abs() + part * (a + w.abs()) + torch.finfo(got.dtype).smallest_normal + 2.0 ** -32 * (b + n * w.abs())
    worst = ((g - w).abs() / bound).max().item()
    print(f"[{label}] worst error {worst:.3f} of its bound", flush=True)
    assert worst <= 1.0, f"{label}: {worst} times the bound"


@pytest.mark.parametrize("f8,dtype", [(True, BF), (True, HF), (False, HF)])
@pytest.mark.parametrize("below", [-22.0, -25.0, -28.0, -31.0])
@pytest.mark.parametrize("S,G,entries,pages", [(1, 1, 1, 40), (5, 3, 1, 40), (20, 1, 1, 30), (40, 4, 1, 30), (1, 1, 1408, 4096), (20, 1, 64, 4096), (40, 4, 64, 4096)])
def test_tail_behind_one_key(S, G, entries, pages, below, f8, dtype):
    """A first key that has almost all the weight, on a value of zero, and a long tail of keys that each have less than
    2^-21 of it, on values of one: the result is the tail's weight alone."""
    H = 8 if entries > 1 else 1
    q, k = scored(-below / 2, below / 2)
    k = k[1].expand(2, PAGE, 64).clone()
    k[0, 0] *= -1
    v = torch.ones(2, PAGE, 64)
    v[:, :, 1::2] = -1.0
    v[0, 0] = 0.0
    c = Keys([0] + [1] * (pages - 1), k, v, S, dtype, f8, H, G)
    kk, vv = c.rows()
    got = c.run(q, entries)
    for s in {0, S - 1}:
        want = attend(q.to(dtype).expand(1, G, 64), kk[:, :1], vv[:, :1], c.n - S + s, 1.0)
        for h in {0, H - 1}:
            assert_small_weights(got[s : s + 1, G * h : G * h + G], *want, c.n, f"tail at 2^{below}, query {s}, head {h}")
