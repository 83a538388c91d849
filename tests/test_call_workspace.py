"""Workspaces that a call takes for itself come from the pool of the stream that it runs on.

A block of the current stream's pool may still be read or written by what that stream has queued; a call on another stream
does not wait for it."""
import contextlib

import pytest
import torch

from genllm_amd import paged


@pytest.fixture
def pools(monkeypatch):
    """torch's stream context and allocations, recorded: a list of (function, bytes, stream it was under)."""
    seen, under = [], [None]

    class Stream:
        def __init__(self, handle, device=None):
            self.cuda_stream = handle

    class External(Stream):
        pass

    @contextlib.contextmanager
    def on(s):
        under.append(s)
        yield
        under.pop()

    monkeypatch.setattr(torch.cuda, "Stream", Stream)
    monkeypatch.setattr(torch.cuda, "ExternalStream", External)
    monkeypatch.setattr(torch.cuda, "stream", on)
    for name in ("empty", "zeros"):
        monkeypatch.setattr(torch, name, lambda n, dtype, device, f=name: seen.append((f, n, under[-1])))
    return seen


def test_stream_objects_and_handles(pools):
    s = torch.cuda.Stream(77)
    paged._workspace(100, "cuda", s)
    paged._workspace(200, "cuda", 88)
    paged._workspace(300, "cuda", 0)
    paged._workspace(400, "cuda", None)
    assert [(f, n, u and u.cuda_stream) for f, n, u in pools[:2]] == [("empty", 100, 77), ("empty", 200, 88)]
    assert pools[0][2] is s and pools[2][2].cuda_stream == 0 and pools[3][2] is None


def gpu_inputs(S=300):
    g = torch.Generator().manual_seed(S)
    x = [torch.randn(1, S, h, 128, generator=g).bfloat16().cuda() for h in (2, 2, 4)]
    gates = [(-torch.rand(1, S, 4, generator=g)).cuda(), torch.rand(1, S, 4, generator=g).cuda()]
    return x, gates, torch.zeros(1, 4, 128, 128, device="cuda"), torch.zeros_like(x[2])


def pool_bytes(stream):
    return sum(seg["total_size"] for seg in torch.cuda.memory_snapshot() if seg["stream"] == stream.cuda_stream)


@pytest.mark.gpu
@pytest.mark.parametrize("handle", [False, True])
def test_delta_rule_beside_pending_work(handle):
    """A block that the current stream has given back, but not yet written, is not what a call on another stream uses."""
    x, gates, state, out = gpu_inputs()
    paged.gated_delta_rule(*x, *gates, state, out, 0.1, l2_eps=1e-6)
    want, left = out.clone(), state.clone()
    need = paged.gated_delta_workspace_bytes(1, 300, 2, 4, 128, 128)
    s = torch.cuda.Stream()
    state.zero_()
    out.zero_()
    torch.cuda.synchronize()
    block = torch.empty(need, dtype=torch.uint8, device="cuda")
    torch.cuda._sleep(20_000_000)
    block.fill_(3)
    kept = block.clone()
    del block
    paged.gated_delta_rule(*x, *gates, state, out, 0.1, l2_eps=1e-6, stream=s.cuda_stream if handle else s)
    torch.cuda.synchronize()
    assert pool_bytes(s) >= need
    assert bool((kept == 3).all()) and torch.equal(out, want) and torch.equal(state, left)


def test_decode_takes_its_workspace_on_the_stream(pools, monkeypatch):
    """Allocated and cleared under the call's stream: the clearing has to come before the kernels."""

    class Row:
        shape, device = (8, 1, 128), "cuda"

        def stride(self, i):
            return 128

    class Block:
        def numel(self):
            return 64

        def element_size(self):
            return 1

    calls = []
    monkeypatch.setattr(paged, "call", lambda *a: calls.append(a))
    monkeypatch.setattr(paged, "_ptr", lambda t: t)
    monkeypatch.setattr(torch, "zeros", lambda n, dtype, device, was=torch.zeros: (was(n, dtype, device), Block())[1])
    s = torch.cuda.Stream(77)
    paged.paged_decode(Row(), Row(), 0, 0, 0, 0, 4, 60, 2, 0.1, stream=s)
    assert [(f, u) for f, _, u in pools] == [("zeros", s)] and calls[0][-1] == 77
    paged.paged_decode(Row(), Row(), 0, 0, 0, 0, 4, 60, 2, 0.1, stream=88)
    assert pools[1][2].cuda_stream == 88 and calls[1][-1] == 88


@pytest.mark.gpu
def test_decode_beside_pending_work():
    g = torch.Generator().manual_seed(5)
    pages, H, D, n = 64, 2, 128, 1000
    k, v = (torch.randn(pages, 16, H, D, generator=g).bfloat16().cuda() for _ in "kv")
    ids = torch.randperm(pages, generator=g).int().cuda()
    q = torch.randn(8, 1, D, generator=g).bfloat16().cuda()
    want, out = torch.zeros_like(q), torch.zeros_like(q)
    args = (k, v, ids, ids, -(-n // 16), n, H, D ** -0.5)
    paged.paged_decode(q, want, *args)
    need = paged.decode_workspace_bytes(8, H, 1, D, -(-n // 16))
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    block = torch.empty(need, dtype=torch.uint8, device="cuda")
    torch.cuda._sleep(20_000_000)
    block.fill_(3)
    kept = block.clone()
    del block
    paged.paged_decode(q, out, *args, stream=s)
    torch.cuda.synchronize()
    assert pool_bytes(s) >= need
    assert bool((kept == 3).all()) and torch.equal(out, want)
