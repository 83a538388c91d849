"""The batch operators' entry points refuse bad arguments with their code and message before any device work: the
addresses below are placeholders far apart that no check lets through to a launch."""
import pytest
import torch

from genllm_amd import _lib, paged

INV, UNS = _lib.ERR_INVALID, _lib.ERR_UNSUPPORTED
NAN, INF = float("nan"), float("inf")
GB = 1 << 30


def pages(gather=False, **kw):
    """Four heads of 128, three entries of five tokens; blocks of [head][token] rows."""
    rows = dict(k=1 * GB, kb=2560, kt=512, kh=128, v=2 * GB, vb=2560, vt=512, vh=128)
    pool = dict(kp=3 * GB, kpb=8192, kpt=128, kph=2048, vp=4 * GB, vpb=8192, vpt=128, vph=2048, ks=5 * GB, vs=6 * GB, n=10,
                ki=7 * GB, kis=4, vi=8 * GB, vis=4, P=4, start=9 * GB, lens=None)
    rest = dict(B=3, S=5, H=4, D=128, dtype=30, stream=None)
    a = {**pool, **rows, **rest} if gather else {**rows, **pool, **rest}
    assert not set(kw) - set(a)
    f = _lib.lib().genllm_kv_gather_f8 if gather else _lib.lib().genllm_kv_scatter_f8
    return f(*dict(a, **kw).values())


def attend(**kw):
    """Eight q heads on two kv heads of 128, three entries of two queries; 16-bit blocks of [token][head] rows."""
    a = dict(q=1 * GB, qb=2048, qt=1024, qh=128, out=2 * GB, ob=2048, ot=1024, oh=128, kp=3 * GB, kpb=4096, kpt=256, kph=128,
             vp=4 * GB, vpb=4096, vpt=256, vph=128, ks=None, vs=None, n=10, ki=7 * GB, kis=4, vi=8 * GB, vis=4, P=4, nc=9 * GB,
             ql=None, B=3, S=2, Hq=8, H=2, D=128, dtype=30, scale=0.1, causal=1, window=0, sinks=0, ws=None, wsb=0, stream=None)
    assert not set(kw) - set(a)
    return _lib.lib().genllm_paged_attention_batch(*dict(a, **kw).values())


def refused(rc, code, msg):
    assert rc == code
    assert msg in _lib.lib().genllm_last_error(), _lib.lib().genllm_last_error()


@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("kw,code,msg", [
    *[({x: None}, INV, b"null pointer") for x in ("k", "v", "kp", "vp", "ks", "vs", "ki", "vi", "start")],
    *[({x: -1}, INV, b"negative") for x in ("B", "S", "H", "n", "P")],
    (dict(D=96), UNS, b"64, 128 or 256"), (dict(dtype=0), UNS, b"bf16 or fp16"), (dict(P=(1 << 26) + 1), INV, b"2^26"),
    (dict(S=(1 << 30) + 1), INV, b"2^30"), (dict(k=GB + 8), INV, b"16-byte aligned"), (dict(kt=516), INV, b"16-byte aligned"),
    (dict(vh=132), INV, b"16-byte aligned"), (dict(kpt=136), INV, b"16-byte aligned"), (dict(vpb=8200), INV, b"16-byte aligned"),
    (dict(start=9 * GB + 2), INV, b"aligned to its type"), (dict(lens=9 * GB + 1), INV, b"aligned to its type"),
    (dict(ki=7 * GB + 3), INV, b"aligned to its type"), (dict(B=1 << 30, kis=0, vis=0, kb=0, vb=0, S=1), INV, b"one launch" )])
def test_pages(gather, kw, code, msg):
    if gather and msg == b"one launch":
        kw, msg = dict(kw, kb=2560, vb=2560), b"k_out overlaps"  # 5 TB of rows lie over everything
    refused(pages(gather, **kw), code, msg)


@pytest.mark.parametrize("kw,msg", [
    (dict(kp=GB + 64), b"k_pool overlaps k"), (dict(vp=3 * GB + 8192 * 9), b"v_pool overlaps k_pool"), (dict(ks=4 * GB + 16), b"k_scales overlaps v_pool"),
    (dict(vs=5 * GB + 39), b"v_scales overlaps k_scales"), (dict(vs=7 * GB), b"v_scales overlaps k_ids"), (dict(lens=5 * GB), b"k_scales overlaps seq_lens"),
    (dict(vp=9 * GB), b"v_pool overlaps start_pos"), (dict(kpt=64), b"rows of k_pool share memory"), (dict(vph=0), b"rows of v_pool share memory"),
    (dict(vpb=4096), b"rows of v_pool share memory")])
def test_scatter_refuses_what_it_would_write_over(kw, msg):
    refused(pages(**kw), INV, msg)


@pytest.mark.parametrize("kw,msg", [
    (dict(k=3 * GB), b"k_out overlaps k_pool"), (dict(v=GB + 512), b"v_out overlaps k_out"), (dict(v=5 * GB), b"v_out overlaps k_scales"),
    (dict(k=8 * GB), b"k_out overlaps v_ids"), (dict(k=9 * GB), b"k_out overlaps start_pos"), (dict(kt=256), b"rows of k_out share memory"),
    (dict(vb=0), b"rows of v_out share memory")])
def test_gather_refuses_what_it_would_write_over(kw, msg):
    refused(pages(True, **kw), INV, msg)


@pytest.mark.parametrize("kw,code,msg", [
    *[({x: None}, INV, b"null pointer") for x in ("q", "out", "kp", "vp", "ki", "vi", "nc")],
    *[({x: -1}, INV, b"negative") for x in ("B", "S", "n", "P", "window", "sinks")], (dict(H=-2), INV, b"negative"),
    (dict(D=192), UNS, b"64, 128 or 256"), (dict(dtype=2), UNS, b"bf16 or fp16"), (dict(Hq=7), INV, b"multiple of n_kv_heads"),
    (dict(H=0), INV, b"multiple of n_kv_heads"), (dict(scale=NAN), INV, b"finite"), (dict(scale=INF), INV, b"finite"), (dict(scale=3e38), INV, b"finite"),
    (dict(scale=-0.1), INV, b"not negative"), (dict(window=4, causal=0), INV, b"causal"), (dict(ks=5 * GB), INV, b"go together"),
    (dict(vs=5 * GB), INV, b"go together"), (dict(P=(1 << 26) + 1), INV, b"2^26"), (dict(S=1 << 29), INV, b"2^30"),
    (dict(q=GB + 8), INV, b"16-byte aligned"), (dict(out=2 * GB + 4), INV, b"16-byte aligned"), (dict(qt=1028), INV, b"16-byte aligned"),
    (dict(kpt=260), INV, b"16-byte aligned"), (dict(vp=4 * GB + 8), INV, b"16-byte aligned"), (dict(nc=9 * GB + 2), INV, b"aligned to its type"),
    (dict(ql=9 * GB + 1), INV, b"aligned to its type"), (dict(kpt=64), INV, b"follow each other"), (dict(kpt=-256), INV, b"follow each other"),
    (dict(vph=-128), INV, b"follow each other"), (dict(vpt=1 << 27), INV, b"follow each other"), (dict(kph=1 << 31), INV, b"follow each other"),
    (dict(P=400), INV, b"workspace"), (dict(P=400, ws=16 * GB, wsb=1000), INV, b"workspace"), (dict(P=400, ws=16 * GB + 8, wsb=GB), INV, b"workspace"),
    (dict(B=1 << 22, qb=0, ob=2048, kis=0, vis=0), INV, b"one launch")])
def test_attention(kw, code, msg):
    refused(attend(**kw), code, msg)


@pytest.mark.parametrize("kw,msg", [
    (dict(out=GB + 2048), b"out overlaps q"), (dict(out=GB, ot=2048, ob=4096), b"out overlaps q"), (dict(out=3 * GB + 8192), b"out overlaps k_pool"),
    (dict(out=4 * GB), b"out overlaps v_pool"), (dict(out=7 * GB), b"out overlaps k_ids"), (dict(out=8 * GB), b"out overlaps v_ids"),
    (dict(out=9 * GB), b"out overlaps n_cached"), (dict(out=10 * GB, ql=10 * GB), b"out overlaps q_lens"),
    (dict(out=5 * GB, ks=5 * GB, vs=6 * GB, kpt=256, vpt=256), b"out overlaps k_scales"), (dict(ob=0), b"rows of out share memory"), (dict(oh=64), b"rows of out share memory"),
    (dict(P=400, ws=GB, wsb=GB), b"the workspace overlaps q"), (dict(P=400, ws=2 * GB, wsb=GB), b"the workspace overlaps out"),
    (dict(P=400, ws=9 * GB, wsb=GB), b"the workspace overlaps n_cached")])
def test_attention_refuses_what_it_would_write_over(kw, msg):
    refused(attend(**kw), INV, msg)


def test_nothing_to_do():
    for kw in (dict(B=0), dict(S=0), dict(H=0)):
        assert pages(**kw) == _lib.OK and pages(True, **kw) == _lib.OK
    for kw in (dict(B=0), dict(S=0), dict(Hq=0), dict(Hq=0, H=0)):
        assert attend(**kw) == _lib.OK


@pytest.mark.parametrize("shape", [(0, 1, 8, 2, 128, 100), (1, 0, 8, 2, 128, 100), (1, 1, 7, 2, 128, 100), (1, 1, 8, 0, 128, 100), (1, 1, 8, 2, 96, 100),
                                   (-1, 1, 8, 2, 128, 100), (1, 1, 8, 2, 128, -1), (1, 1, 8, 2, 128, 1 << 27), (2 ** 31 - 1, 1, 8, 8, 128, 100),
                                   (2 ** 31 - 1,) * 6, (1, 2 ** 31 - 1, 8, 2, 128, 100)])
def test_workspace_of_sizes_that_are_not_served(shape):
    assert _lib.lib().genllm_paged_attention_batch_workspace_bytes(*shape) == 0


def test_workspace():
    f = _lib.lib().genllm_paged_attention_batch_workspace_bytes
    assert f(64, 1, 32, 8, 128, 4) == 0  # one workgroup for each kv head
    assert 0 < f(1, 1, 32, 8, 128, 8192) < 1 << 26 and 0 < f(64, 1, 32, 8, 128, 256) < 1 << 26
    assert 0 < f(1, 64, 32, 8, 128, 8192) < 1 << 28 and f(1, 4096, 32, 8, 128, 8192) == 0


def _bf16(*shape):
    return torch.zeros(shape, dtype=torch.bfloat16)


@pytest.mark.parametrize("call", [
    lambda t: paged.kv_scatter_f8(t, t, t, t, t, t, t, t, t),
    lambda t: paged.kv_gather_f8(t, t, t, t, t, t, t, t, t),
    lambda t: paged.paged_attention_batch(t, t, t, t, t, t, t, 1.0),
    lambda t: paged.paged_attention_batch(t, t, t, t, t, t, t, 1.0, stream=0),
])
def test_calls_on_tensors(call):
    for bad, msg in ((3, "must be a tensor"), (None, "must be a tensor"), (torch.zeros(2, 2, 2, 2), "bf16 or float16"),
                     (_bf16(2, 2, 2, 2), "GPU tensor"), (_bf16(2, 2, 2, 2).to_sparse(), "strided")):
        with pytest.raises(ValueError, match=msg):
            call(bad)


def test_calls_argument_count():
    m = _lib.calls()
    for f in (m.kv_scatter_f8, m.kv_gather_f8, m.paged_attention_batch):
        with pytest.raises(TypeError):
            f(1)
    with pytest.raises(TypeError):
        m.bind_batch(0)
    with pytest.raises(ValueError):
        m.bind_batch(0, 0, 0, 0)


def test_f8_pool():
    pool, scales = paged.f8_pool(5, 3, 64, device="cpu")
    assert pool.shape == (5, 16, 3, 64) and pool.dtype == torch.float8_e4m3fn and pool.stride() == (3072, 64, 1024, 1)
    assert scales.shape == (5, 3) and scales.dtype == torch.uint8
