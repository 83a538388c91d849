"""The batch operators as a server uses them: prompts, then tokens, in 8-bit pages; captured, and on other streams."""
import math

import pytest
import torch

from genllm_amd import paged
from batch import PAGE, assert_attended, attend, scatter

pytestmark = pytest.mark.gpu

BF = torch.bfloat16
B, HQ, H, D, P = 3, 8, 2, 128, 12
SCALE = 1 / math.sqrt(D)


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class Server:
    """Pools of one layer on the GPU, and what the definitions make of them on the CPU."""

    def __init__(self, seed=0):
        self.g = torch.Generator().manual_seed(seed)
        n = B * P + 1
        self.ids = torch.randperm(n, generator=self.g)[: B * P].view(B, P).int()
        self.dev_ids = self.ids.cuda()
        self.pools = [paged.f8_pool(n, H, D) for _ in "kv"]
        self.want = [(torch.zeros(n, PAGE, H, D).double(), torch.zeros(n, H, dtype=torch.int32)) for _ in "kv"]

    def rows(self, S, heads, std=1.0):
        return (torch.randn(B, S, heads, D, generator=self.g) * std).to(BF)

    def write(self, k, v, start, lens, **kw):
        (kp, ks), (vp, vs) = self.pools
        paged.kv_scatter_f8(k, v, kp, vp, ks, vs, self.dev_ids, self.dev_ids, start, seq_lens=lens, **kw)

    def attend(self, q, out, n, lens, **kw):
        (kp, ks), (vp, vs) = self.pools
        paged.paged_attention_batch(q, out, kp, vp, self.dev_ids, self.dev_ids, n, SCALE, q_lens=lens, k_scales=ks, v_scales=vs, **kw)

    def expect(self, k, v, start, lens):
        for x, (codes, e) in zip((k, v), self.want):
            scatter(x, codes, e, self.ids, start, lens)

    def check(self, q, out, n, lens, label, **kw):
        for b in range(B):
            kv = [(codes * torch.ldexp(torch.ones(1).double(), e)[:, None, :, None])[self.ids[b].long()].reshape(-1, H, D)[: n[b]]
                  for codes, e in self.want]
            assert_attended(out[b, : lens[b]], *attend(q[b, : lens[b]], *kv, n[b] - lens[b], SCALE, **kw), max(1, n[b]), 2.0 ** -11, f"{label} entry {b}")


@pytest.mark.parametrize("window", [None, 20])
def test_conversation(window):
    """Prompts of unlike length, tokens one by one, a turn of several; then the rows read back and attended plainly."""
    s, n = Server(), [0] * B
    for S, lens in ((70, [70, 33, 1]), (1, [1, 1, 1]), (1, [1, 1, 0]), (1, [1, 1, 1]), (20, [4, 20, 17]), (1, [1, 1, 1])):
        k, v, q = s.rows(S, H), s.rows(S, H, 0.2), s.rows(S, HQ)
        out = torch.zeros(B, S, HQ, D, dtype=BF, device="cuda")
        s.write(k.cuda(), v.cuda(), ints(n), ints(lens))
        s.expect(k, v, n, lens)
        n = [a + m for a, m in zip(n, lens)]
        s.attend(q.cuda(), out, ints(n), ints(lens), window=window, sinks=3)
        torch.cuda.synchronize()
        s.check(q, out, n, lens, f"{S} tokens", window=window, sinks=3)
    (kp, ks), (vp, vs) = s.pools
    back = [torch.zeros(B, max(n), H, D, dtype=BF, device="cuda") for _ in "kv"]
    paged.kv_gather_f8(kp, vp, ks, vs, s.dev_ids, s.dev_ids, ints([0] * B), *back, seq_lens=ints(n))
    torch.cuda.synchronize()
    for b in range(B):
        assert_attended(out[b, :1], *attend(q[b], *(x[b, : n[b]].cpu().double() for x in back), n[b] - 1, SCALE, window=window, sinks=3), n[b],
                        2.0 ** -11, f"read back, entry {b}")


@pytest.mark.parametrize("S", [1, 20])
def test_captured(S):
    """A step captured once and replayed for positions, lengths and rows that change, with eager work between; two graphs
    with a workspace in common, replayed in order."""
    s = Server(S)
    k, v, q = (torch.zeros(B, S, h, D, dtype=BF, device="cuda") for h in (H, H, HQ))
    out, other = (torch.zeros(B, S, HQ, D, dtype=BF, device="cuda") for _ in range(2))
    at = [1, 5, 17]
    x = [s.rows(17, H) for _ in "kv"]
    s.write(*(t.cuda() for t in x), ints([0] * B), ints(at))
    s.expect(*x, [0] * B, at)
    start, n, lens = ints(at), ints(at), ints([0] * B)
    room = torch.empty(paged.paged_attention_batch_workspace_bytes(B, S, HQ, H, D, P), dtype=torch.uint8, device="cuda")
    room = room if room.numel() else None
    s.write(k, v, start, lens), s.attend(q, out, n, lens, workspace=room)  # the first calls
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    with torch.cuda.graph(graphs[0]):
        s.write(k, v, start, lens)
        s.attend(q, out, n, lens, workspace=room)
    with torch.cuda.graph(graphs[1]):
        s.attend(q, other, n, lens, workspace=room, window=9, sinks=1)
    for turn in range(4):
        m = [S, max(1, S - 3 * turn), 1 if turn % 2 else S]
        x = [s.rows(S, h) for h in (H, H, HQ)]
        for t, y in zip((k, v, q), x):
            t.copy_(y)
        now = [a + b for a, b in zip(at, m)]
        start.copy_(ints(at)), lens.copy_(ints(m)), n.copy_(ints(now))
        s.expect(x[0], x[1], at, m)
        graphs[0].replay(), graphs[1].replay()
        torch.cuda.synchronize()
        s.check(x[2], out, now, m, f"replay {turn}"), s.check(x[2], other, now, m, f"window, replay {turn}", window=9, sinks=1)
        eager = torch.zeros_like(out)
        s.attend(q, eager, n, lens)
        torch.cuda.synchronize()
        for b in range(B):
            assert torch.equal(eager[b, : m[b]], out[b, : m[b]])
        at = now if turn < 2 else [a - 3 for a in now]  # drafts taken back


@pytest.mark.parametrize("S", [1, 40])
def test_captured_splits(S):
    """Contexts that are split over workgroups: two graphs with a workspace in common, replayed in order while lengths
    change, eager calls in that workspace between them."""
    g = torch.Generator().manual_seed(S)
    pages, n = 120, [1900, 300]
    pools = [torch.randn(2 * pages, PAGE, H, D, generator=g).to(BF) for _ in "kv"]
    ids = torch.randperm(2 * pages, generator=g).view(2, pages).int()
    dev, dev_ids = [x.cuda() for x in pools], ids.cuda()
    q = torch.randn(2, S, HQ, D, generator=g).to(BF)
    dev_q = q.cuda()
    need = paged.paged_attention_batch_workspace_bytes(2, S, HQ, H, D, pages)
    assert need > 0
    room = torch.full((need,), 255, dtype=torch.uint8, device="cuda")
    lens, outs = ints(n), [torch.zeros_like(dev_q) for _ in range(3)]
    how = [dict(), dict(window=700, sinks=5)]

    def run(out, **kw):
        paged.paged_attention_batch(dev_q, out, *dev, dev_ids, dev_ids, lens, SCALE, workspace=room, **kw)

    run(outs[0])
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in how]
    for graph, out, kw in zip(graphs, outs, how):
        with torch.cuda.graph(graph):
            run(out, **kw)
    for turn, n in enumerate([n, [S, 1920], [1000, 0], [1920, 1919]]):
        lens.copy_(ints(n))
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for out, kw in zip(outs, how):
            outs[2].zero_()
            run(outs[2], **kw)
            torch.cuda.synchronize()
            assert torch.equal(out, outs[2]), f"replay {turn}"
            for b in range(2):
                k, v = (x[ids[b].long()].reshape(-1, H, D)[: n[b]].double() for x in pools)
                assert_attended(out[b], *attend(q[b], k, v, n[b] - S, SCALE, **kw), max(1, n[b]), 2.0 ** -8, f"replay {turn} entry {b}")


def test_streams():
    """Two streams at once, each with workspaces of its own; streams given as objects and as handles."""
    s = Server(9)
    k, v = s.rows(150, H), s.rows(150, H)
    lens = [150, 150, 150]
    s.write(k.cuda(), v.cuda(), ints([0] * B), ints(lens))
    s.expect(k, v, [0] * B, lens)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    qs = [s.rows(S, HQ) for S in (1, 1, 30, 30)]
    dev = [q.cuda() for q in qs]
    outs = [torch.zeros_like(q) for q in dev]
    n, m = ints(lens), [ints([q.shape[1]] * B) for q in qs]
    torch.cuda.synchronize()
    for i, (q, out) in enumerate(zip(dev, outs)):
        s.attend(q, out, n, m[i], stream=streams[i % 2] if i < 2 else streams[i % 2].cuda_stream)
    torch.cuda.synchronize()
    for i, q in enumerate(qs):
        s.check(q, outs[i], lens, [q.shape[1]] * B, f"call {i}")


def test_streams_that_split():
    """Split contexts on two streams at once, the workspaces taken for each call: a stream as an object, as a handle, and
    the current one."""
    g = torch.Generator().manual_seed(5)
    pages, n = 100, [1600, 900]
    pools = [torch.randn(2 * pages, PAGE, H, D, generator=g).to(BF) for _ in "kv"]
    ids = torch.randperm(2 * pages, generator=g).view(2, pages).int()
    dev, dev_ids, lens = [x.cuda() for x in pools], ids.cuda(), ints(n)
    streams = [torch.cuda.Stream() for _ in range(2)]
    qs = [torch.randn(2, S, HQ, D, generator=g).to(BF) for S in (1, 30, 1, 30, 1, 30)]
    dev_q = [q.cuda() for q in qs]
    outs = [torch.zeros_like(q) for q in dev_q]
    for q in qs:
        assert paged.paged_attention_batch_workspace_bytes(2, q.shape[1], HQ, H, D, pages) > 0
    torch.cuda.synchronize()
    for i, (q, out) in enumerate(zip(dev_q, outs)):
        on = [streams[i % 2], streams[i % 2].cuda_stream, None][i // 2]
        with torch.cuda.stream(streams[i % 2] if on is None else torch.cuda.current_stream()):
            paged.paged_attention_batch(q, out, *dev, dev_ids, dev_ids, lens, SCALE, stream=on)
    torch.cuda.synchronize()
    for i, q in enumerate(qs):
        for b in range(2):
            k, v = (x[ids[b].long()].reshape(-1, H, D)[: n[b]].double() for x in pools)
            step = 2.0 ** -16 if q.shape[1] == 1 else 2.0 ** -8
            assert_attended(outs[i][b], *attend(q[b], k, v, n[b] - q.shape[1], SCALE), n[b], step, f"call {i} entry {b}")


def test_managed_pools():
    """The pages of a PagedAttentionManager's layer, attended as a batch of one: the op's own result but for its rounding."""
    mgr = paged.PagedAttentionManager(8 << 20)
    mgr.init_layer(0, H, D)
    mgr.reserve_layer(0, P)
    g = torch.Generator().manual_seed(4)
    k, v, q = (torch.randn(1, h, S, D, generator=g).to(BF).cuda() for h, S in ((H, 90), (H, 90), (HQ, 90)))
    out = torch.zeros_like(q)
    paged.paged_attention(mgr, 0, q, k, v, out, HQ // H, SCALE)
    mine = torch.zeros(1, 90, HQ, D, dtype=BF, device="cuda")
    paged.paged_attention_batch(q.transpose(1, 2), mine, mgr.pool(0, 0), mgr.pool(0, 1), mgr.device_table(0, 0)[None], mgr.device_table(0, 1)[None],
                                ints([90]), SCALE)
    torch.cuda.synchronize()
    want = attend(q[0].transpose(0, 1), k[0].transpose(0, 1).cpu().double(), v[0].transpose(0, 1).cpu().double(), 0, SCALE)
    assert_attended(mine[0], *want, 90, 2.0 ** -8, "batch")
    assert_attended(out[0].transpose(0, 1), *want, 90, 2.0 ** -8, "op")
    mgr.close()
