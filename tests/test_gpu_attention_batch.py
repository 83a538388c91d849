"""Attention of padded batches over paged caches against the formula in 64 bits."""
import math

import pytest
import torch

from genllm_amd import paged
from batch import PAGE, assert_attended, attend, rows, values

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


class Case:
    def __init__(self, Hq, H, D, dtype, f8, n, S, ql=None, P=None, layout=None, seed=0, std=1.0):
        g = torch.Generator().manual_seed(seed + 1000 * D + S)
        B, self.S, self.n, self.ql = len(n), S, n, ql
        self.Hq, self.H, self.D, self.dtype, self.f8 = Hq, H, D, dtype, f8
        P = P or max(1, -(-max(n) // PAGE))
        blocks = B * P + 2
        self.ids = [torch.randperm(blocks, generator=g)[: B * P].view(B, P).int() for _ in "kv"]
        self.pools, self.scales = [], []
        for kind in "kv":
            if f8:
                codes = torch.randint(0, 256, (blocks, 16, H, D), generator=g, dtype=torch.uint8)
                # codes of a normal distribution; scales that differ from page to page
                codes = (torch.randn(codes.shape, generator=g) * 60).to(torch.float8_e4m3fn)
                e = torch.randint(-3, 4, (blocks, H), generator=g) - 6 + (0 if kind == "k" else -3)
                pool, scale = paged.f8_pool(blocks, H, D)
                if layout == "token":
                    pool = pool.view(torch.uint8).contiguous().view(torch.float8_e4m3fn)
                pool.view(torch.uint8).copy_(codes.view(torch.uint8))
                scale.copy_((e + 127).to(torch.uint8))
            else:
                x = torch.randn(blocks, 16, H, D, generator=g).to(dtype)
                pool, scale = x.cuda(), None
                if layout == "head":
                    pool = x.transpose(1, 2).contiguous().cuda().transpose(1, 2)
            self.pools.append(pool), self.scales.append(scale)
        self.q = (torch.randn(B, S, Hq, D, generator=g) * std).to(dtype).cuda()
        self.out = torch.full((B, S, Hq, D), 2.5, dtype=dtype, device="cuda")
        self.scale = 1 / math.sqrt(D)

    def run(self, out=None, q=None, **kw):
        dev = lambda x: None if x is None else torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
        out = self.out if out is None else out
        paged.paged_attention_batch(self.q if q is None else q, out, *self.pools, *(i.cuda() for i in self.ids), dev(self.n), self.scale,
                                    q_lens=dev(self.ql), k_scales=self.scales[0], v_scales=self.scales[1], **kw)
        torch.cuda.synchronize()
        return out

    def tables(self):
        return [values(p, s) if self.f8 else p.cpu().double() for p, s in zip(self.pools, self.scales)]

    def check(self, label, out=None, window=None, sinks=0, causal=True, q=None):
        out = self.out if out is None else out
        tables = self.tables()
        few = self.S * (self.Hq // self.H) <= 16
        p_step = 2.0 ** -11 if self.f8 or self.dtype == HF else 2.0 ** -16 if few else 2.0 ** -8
        for b, n in enumerate(self.n):
            ql = self.S if self.ql is None else min(max(self.ql[b], 0), self.S)
            n = min(max(n, 0), self.ids[0].shape[1] * PAGE)
            k, v = (rows(t, i[b], n, self.H, self.D) for t, i in zip(tables, self.ids))
            want = attend((self.q if q is None else q)[b, :ql], k, v, n - ql, self.scale, causal, window, sinks)
            assert_attended(out[b, :ql], *want, max(n, 1), p_step, f"{label} entry {b} n={n} ql={ql}")
            assert bool((out[b, ql:] == 2.5).all()), f"{label}: rows behind entry {b}"


HEADS = [(4, 1, 64), (8, 2, 128), (4, 2, 256), (6, 2, 128), (16, 1, 128), (5, 5, 64)]


@pytest.mark.parametrize("f8", [True, False])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("Hq,H,D", HEADS)
def test_tokens(Hq, H, D, dtype, f8):
    """One token each of unlike contexts, from none to several splits."""
    c = Case(Hq, H, D, dtype, f8, [1, 0, 15, 16, 17, 33, 1500, 257], 1)
    c.run()
    c.check("tokens")


@pytest.mark.parametrize("f8", [True, False])
@pytest.mark.parametrize("Hq,H,D,S", [(4, 1, 64, 4), (8, 2, 128, 3), (4, 2, 256, 7), (16, 16, 64, 16), (20, 1, 64, 1), (8, 2, 128, 16), (4, 2, 256, 9)])
def test_drafts(Hq, H, D, S, f8):
    """A few queries each, up to a tile of 64 rows; q_lens from none to all; more queries than tokens."""
    c = Case(Hq, H, D, BF, f8, [S, 40, 16, 700, 2, 0, 90], S, [S, S, 0, max(1, S - 1), S, S, 1])
    c.q[2] = c.q[6, 1:] = math.nan
    c.run()
    c.check("drafts")


@pytest.mark.parametrize("f8", [True, False])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("Hq,H,D,S", [(4, 2, 64, 150), (8, 2, 128, 70), (2, 1, 256, 100), (3, 1, 128, 129)])
def test_prompts(Hq, H, D, S, dtype, f8):
    """Prompts from the first token on, chunks on top of a cache, one shorter than its width."""
    c = Case(Hq, H, D, dtype, f8, [S, S + 333, S - 1, 5], S, [S, S, S - 1, 5])
    c.run()
    c.check("prompts")


@pytest.mark.parametrize("f8,window", [(True, None), (False, 300)])
@pytest.mark.parametrize("Hq,H,D", [(6, 3, 64), (8, 8, 128), (6, 3, 256)])
def test_whole_prompts(Hq, H, D, f8, window):
    """Prompts of a thousand tokens whose tiles are all there at once, a long tile beside a short one."""
    S = 1030
    B = {64: 4, 128: 3, 256: 2}[D]
    n = [S, S + 900, 700, S - 1][:B]
    c = Case(Hq, H, D, BF, f8, n, S, [S, S, 650, S - 1][:B])
    c.run(window=window)
    c.check("whole prompts", window=window)


def test_many_tiles():
    """More tiles than 16 bits count, most of them of an entry that has few rows."""
    n = [i % 17 for i in range(1100)]
    c = Case(64, 64, 64, BF, True, n, 17, [min(i % 5, x) for i, x in enumerate(n)])
    c.run()
    c.check("many tiles")


@pytest.mark.parametrize("f8", [True, False])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (5, 4), (16, 0), (16, 16), (100, 20), (33, 300), (2 ** 31 - 1, 3)])
@pytest.mark.parametrize("S", [1, 3, 40, 130])
def test_windows(S, window, sinks, f8):
    c = Case(4, 2, 128, BF, f8, [S, 640, 131, 300], S, seed=window)
    c.run(window=window, sinks=sinks)
    c.check(f"window {window} + {sinks}", window=window, sinks=sinks)


@pytest.mark.parametrize("f8", [True, False])
@pytest.mark.parametrize("S", [1, 5, 90])
def test_all_keys(S, f8):
    """Not causal: every query sees every token, also where there are fewer tokens than queries."""
    c = Case(4, 2, 128, BF, f8, [S, 300, 3, 0], S)
    c.run(causal=False)
    c.check("all keys", causal=False)


@pytest.mark.parametrize("f8,layout", [(True, "token"), (False, "head")])
@pytest.mark.parametrize("S", [2, 50])
def test_layouts(S, f8, layout):
    """Pools of the other layout, q head by head, out token by token with room between the rows; longer tables."""
    c = Case(8, 2, 128, HF, f8, [S, 200], S, P=40, layout=layout)
    c.q = c.q.transpose(1, 2).contiguous().transpose(1, 2)
    wide = torch.full((2, S, 10, 160), 2.5, dtype=HF, device="cuda")
    out = wide[:, :, 1:9, 16:144]
    c.run(out)
    c.check(layout, out)
    wide[:, :, 1:9, 16:144] = 2.5
    assert bool((wide == 2.5).all())


@pytest.mark.parametrize("S", [1, 3, 60])
def test_out_is_q(S):
    c = Case(8, 2, 128, BF, True, [S, 900], S)
    q = c.q.clone()
    c.run(out=c.q)
    c.check("in place", c.q, q=q)


@pytest.mark.parametrize("f8", [True, False])
@pytest.mark.parametrize("S", [1, 4, 30, 140])
def test_what_is_not_seen(S, f8):
    """NaN and infinities behind the cache's end, above the diagonal, below the window, in padded rows and behind ids
    that are no blocks reach no row that does not see them; they do reach those that do."""
    c = Case(4, 2, 64, BF, f8, [S + 200, S + 37], S, P=24, seed=7)

    def put(b, t):  # K and V of token t
        for pool, ids in zip(c.pools, c.ids):
            block = int(ids[b, t // PAGE])
            if f8:
                pool.view(torch.uint8)[block, t % PAGE] = 0x7F
            else:
                pool[block, t % PAGE, :, ::2] = math.nan
                pool[block, t % PAGE, :, 1::2] = math.inf

    for t in range(S + 200, 24 * PAGE):
        put(0, t)
    put(0, 30), put(0, 100)  # under the window of 64 + 20 sinks, until S + 200 - 64
    for t in range(S + 37, S + 37 + PAGE):
        put(1, t)
    if S > 2:
        put(1, S + 36), put(1, 37 + S // 2)  # only the last queries see these
    c.ids[0][1, -1], c.ids[1][0, -2] = -5, 10 ** 6
    c.ids[0][0, 3] = -1  # tokens 48 to 63, under the window
    c.run(window=64, sinks=20)
    c.check("not seen", window=64, sinks=20)


@pytest.mark.parametrize("S", [1, 40])
def test_bad_pages(S):
    """An id that is no block, or a scale that is NaN, gives NaN to the rows that see it and to no other."""
    c = Case(4, 2, 128, BF, True, [S + 100, S + 60, S], S, seed=3)
    c.ids[1][0, 2] = c.pools[0].shape[0]
    c.scales[0][int(c.ids[0][1, 1]), 1] = 255  # kv head 1 alone
    c.run()
    tables = c.tables()
    tables[0][int(c.ids[0][1, 1]), :, 1] = math.nan
    c.tables = lambda: tables
    c.check("bad pages")
    assert bool(torch.isnan(c.out[0]).all()) and bool(torch.isnan(c.out[1, :, 2:]).all())
    assert not bool(torch.isnan(c.out[1, :, :2]).any()) and not bool(torch.isnan(c.out[2]).any())


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("S", [1, 20, 70])
def test_wide_scores(S, dtype):
    """Scores far apart, so that one key has all the weight, and a scale of zero, where all have the same."""
    c = Case(4, 2, 128, dtype, False, [S + 400], S, std=30.0)
    c.run()
    c.check("far apart")
    c.scale = 0.0
    c.run()
    c.check("all alike")


@pytest.mark.parametrize("S", [1, 33])
def test_scales_far_apart(S):
    """Pages of V whose scales differ by up to 120 binades, in rising and falling order."""
    c = Case(4, 2, 64, BF, True, [S + 300, S + 300], S, seed=11)
    for b in range(2):
        at = c.ids[1][b].long()
        e = torch.linspace(-60, 60, len(at)).int()
        c.scales[1][at.cuda()] = ((e if b else e.flip(0)) + 127).to(torch.uint8)[:, None].expand(-1, 2).cuda()
    c.run()
    c.check("scales")


def scaled(c, exponents):
    """V's pages, in the order of each entry's table, with these exponents in turn."""
    for ids in c.ids[1]:
        e = torch.tensor([exponents[i % len(exponents)] for i in range(len(ids))], dtype=torch.int32)
        c.scales[1][ids.long().cuda()] = (e + 127).to(torch.uint8)[:, None].expand(-1, c.H).cuda()


@pytest.mark.parametrize("e", [-90, -40, 25, 100])
@pytest.mark.parametrize("S", [1, 7, 40, 130])
def test_one_scale(S, e):
    """Values of any one size, also where a step has fewer pages than it takes."""
    c = Case(8, 2, 128, BF, True, [S, S + 17, 900, S + 40], S)
    scaled(c, [e])
    c.run()
    c.check("one scale")


@pytest.mark.parametrize("exponents", [(-60, -20, 20, 60), (60, 20, -20, -60), (-30, -30, 0), (0, -14, -30), (-9, 6)])
@pytest.mark.parametrize("S", [1, 3, 33, 150])
def test_scales_of_unseen_pages(S, exponents):
    """A query's result has its own keys' precision, whatever the pages behind it hold (bf16: 2^60 is no fp16 value)."""
    c = Case(4, 2, 128, BF, True, [S, S + 20, 400], S)
    scaled(c, exponents)
    c.run()
    c.check("unseen scales")


@pytest.mark.parametrize("S", [1, 3, 33, 150])
def test_pages_of_zeros(S):
    """Pages of zeros, which have the least scale, among others."""
    c = Case(4, 2, 128, BF, True, [S, S + 20, 400], S)
    for ids in c.ids[1]:
        at = ids.long().cuda()[::2]
        c.pools[1].view(torch.uint8)[at] = 0
        c.scales[1][at] = 27
    c.run()
    c.check("zeros")


@pytest.mark.parametrize("size", [2.0 ** -20, 2.0 ** -12])
@pytest.mark.parametrize("S", [1, 3, 33, 150])
def test_small_elements(S, size):
    """fp16's subnormal values, as keys, values and queries."""
    c = Case(4, 2, 128, HF, False, [S, S + 20, 400], S)
    for pool in c.pools:
        pool.mul_(size)
    c.run()
    c.check("small")
    c.q.mul_(size)
    c.run()
    c.check("small q")


@pytest.mark.parametrize("f8", [True, False])
def test_many_entries(f8):
    """More entries than a wave has lanes, most of them empty, one long."""
    n = [(7 * i) % 40 if i % 3 else 0 for i in range(150)]
    n[97] = 3000
    c = Case(4, 2, 64, BF, f8, n, 1, [1 if i % 5 else 0 for i in range(150)])
    c.run()
    c.check("many")


@pytest.mark.parametrize("pages", [12, 400])
def test_more_entries_than_workgroups(pages):
    """Enough entries for several turns of the workgroups there are, with short tables and with long ones."""
    n = [(i * 37) % 90 for i in range(1100)]
    n[3], n[1050] = 16 * pages, 16 * pages - 5
    c = Case(4, 2, 128, BF, True, [1] * 1100, 1, P=1)
    blocks = c.scales[0].shape[0]
    g = torch.Generator().manual_seed(pages)
    c.n, c.ids = n, [torch.randint(0, blocks, (1100, pages), generator=g).int() for _ in "kv"]
    c.run()
    c.check("more entries")


@pytest.mark.parametrize("S", [1, 30])
def test_more_tokens_than_the_table(S):
    """n_cached past the table: the table's tokens alone, the last query at their end."""
    c = Case(4, 2, 64, BF, True, [10 ** 6, 2 ** 31 - 1, -7], S, P=5)
    c.run()
    c.check("past the table")


@pytest.mark.parametrize("S,f8", [(1, True), (1, False), (20, True), (150, False)])
def test_same_twice(S, f8):
    """No result depends on the order in which workgroups run."""
    c = Case(8, 2, 128, BF, f8, [S + 1000, S + 50, S], S)
    first = c.run().clone()
    for _ in range(3):
        c.out.fill_(2.5)
        assert torch.equal(c.run(), first)


@pytest.mark.parametrize("f8", [True, False])
def test_far_blocks(f8):
    """Blocks whose offset passes 32 bits."""
    near, far = (Case(4, 2, 256, BF, f8, [30], 1) for _ in range(2))
    blocks = 140000 if f8 else 140000 // 2
    for i in range(2):
        at = blocks - 1 - 3 * torch.arange(2, device="cuda")
        src = near.ids[i][0].long().cuda()
        pool = torch.zeros(blocks, 16, 2, 256, dtype=torch.uint8 if f8 else BF, device="cuda")
        pool[at] = (near.pools[i].view(torch.uint8) if f8 else near.pools[i])[src]
        far.pools[i], far.ids[i] = pool, at.int().cpu().view(1, 2)
        if f8:
            far.scales[i] = torch.zeros(blocks, 2, dtype=torch.uint8, device="cuda")
            far.scales[i][at] = near.scales[i][src]
    near.check("far blocks", far.run())
