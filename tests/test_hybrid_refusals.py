"""The hybrid layers' entry points refuse bad arguments with their code and message before any device work: the
addresses below are aligned placeholders that no check lets through to a launch."""
import ctypes as C

import pytest
import torch

from genllm_amd import _lib, paged

INV, UNS = _lib.ERR_INVALID, _lib.ERR_UNSUPPORTED
NAN, INF = float("nan"), float("inf")


def delta(**kw):
    a = dict(q=0x10000, qb=4096, qt=1024, qh=128, k=0x20000, kb=4096, kt=1024, kh=128, v=0x30000, vb=8192, vt=2048, vh=128,
             a=0x40000, ab=64, at=16, b=0x50000, bb=64, bt=16, a_log=0x60000, dt=0x70000, state=0x80000, n=4, ids=None,
             lens=None, out=0x90000, ob=8192, ot=2048, oh=128, B=2, S=4, Hk=8, Hv=16, Dk=128, Dv=128, dtype=30, scale=0.1,
             l2=1e-6, ws=None, wsb=0, stream=None)
    assert not set(kw) - set(a)
    return _lib.lib().genllm_gated_delta_rule(*dict(a, **kw).values())


def conv(**kw):
    a = dict(x=0x100000, xb=4096, xt=64, w=0x20000, bias=None, out=0x900000, ob=4096, ot=64, state=0x80000, n=4, ids=None,
             lens=None, B=2, S=64, C=64, W=4, dtype=30, silu=1, stream=None)
    assert not set(kw) - set(a)
    return _lib.lib().genllm_causal_conv(*dict(a, **kw).values())


def axes(sections=(11, 11, 10), **kw):
    sec = (C.c_int32 * 8)(*sections) if sections is not None else None
    a = dict(q=0x10000, qt=2560, qh=256, qo=0x20000, qot=256, qoh=1024, gq=0x30000, Hq=8, k=0x40000, kt=2560, kh=256,
             ko=0x50000, kot=256, koh=1024, gk=0x60000, Hk=2, eps=1e-6, cos=0x70000, sin=0x80000, rows=100, rope=64,
             pos=0x90000, ps=4, n=3, sec=sec, inter=1, S=4, D=256, dtype=30, stream=None)
    assert not set(kw) - set(a)
    return _lib.lib().genllm_qk_norm_rope_axes(*dict(a, **kw).values())


@pytest.mark.parametrize("kw,code,msg", [
    *[({p: None}, INV, b"null pointer") for p in ("q", "k", "v", "a", "b", "state", "out")],
    (dict(Dk=96), UNS, b"64 or 128"), (dict(Dv=256), UNS, b"64 or 128"), (dict(dtype=0), UNS, b"bf16 or fp16"),
    (dict(Hv=12), INV, b"multiple of n_k_heads"), (dict(Hk=0), INV, b"zero size"), (dict(B=-1), INV, b"negative"),
    (dict(S=-1), INV, b"negative"), (dict(n=1), INV, b"fewer states"), (dict(a_log=None), INV, b"go together"),
    (dict(dt=None), INV, b"go together"), (dict(scale=NAN), INV, b"finite"), (dict(scale=INF), INV, b"finite"),
    (dict(l2=NAN), INV, b"finite"), (dict(l2=INF), INV, b"finite"), (dict(q=0x10008), INV, b"16-byte aligned"),
    (dict(kt=1020), INV, b"16-byte aligned"), (dict(vh=100), INV, b"16-byte aligned"), (dict(ob=4), INV, b"16-byte aligned"),
    (dict(state=0x80004), INV, b"16-byte aligned"), (dict(a=0x40001), INV, b"aligned to its type"),
    (dict(a=0x40002, a_log=None, dt=None), INV, b"aligned to its type"), (dict(ids=0x1002), INV, b"aligned to its type"),
    (dict(ot=0), INV, b"share memory"), (dict(oh=0), INV, b"share memory"),
    (dict(out=0x10000), INV, b"overlaps"), (dict(out=0x20000), INV, b"overlaps"), (dict(out=0x80000), INV, b"overlaps"),
    (dict(out=0x30000, ot=4096), INV, b"overlaps"),
    (dict(B=1 << 16, Hv=16, n=1 << 16), INV, b"2^19"), (dict(S=100), INV, b"workspace"), (dict(S=(1 << 30) + 1), INV, b"2^30"),
    (dict(S=100, ws=0xA00000, wsb=100), INV, b"workspace"), (dict(S=100, ws=0xA00004, wsb=1 << 40), INV, b"workspace"),
])
def test_gated_delta_rule(kw, code, msg):
    assert delta(**kw) == code
    assert msg in _lib.lib().genllm_last_error()


def test_gated_delta_rule_nothing_to_do():
    for kw in (dict(B=0), dict(S=0), dict(B=0, q=None, state=None)):
        assert delta(**kw) == _lib.OK


@pytest.mark.parametrize("kw,code,msg", [
    *[({p: None}, INV, b"null pointer") for p in ("x", "w", "out")],
    (dict(W=1), UNS, b"widths"), (dict(W=5), UNS, b"widths"), (dict(dtype=7), UNS, b"bf16 or fp16"),
    (dict(C=-1), INV, b"negative"), (dict(n=1), INV, b"fewer states"), (dict(state=None, ids=0x1000), INV, b"without a state"),
    (dict(state=0x100000), INV, b"state overlaps"), (dict(state=0x900000), INV, b"state overlaps"),
    (dict(x=0x100001), INV, b"aligned"), (dict(ot=0), INV, b"share memory"), (dict(out=0x100000), INV, b"overlaps"),
    (dict(out=0x100000 + 2 * 64 * 3), INV, b"overlaps"), (dict(out=0x100000 - 64), INV, b"overlaps"),
    (dict(out=0x100000 + 2 * 64, xt=96, ot=96, xb=96 * 64, ob=96 * 64), INV, b"overlaps"),
    (dict(out=0x100000 + 2 * 64, xt=128, ot=192, xb=128 * 64, ob=192 * 64), INV, b"overlaps"),
])
def test_causal_conv(kw, code, msg):
    assert conv(**kw) == code
    assert msg in _lib.lib().genllm_last_error()


def test_causal_conv_nothing_to_do():
    for kw in (dict(B=0), dict(S=0), dict(C=0, x=None)):
        assert conv(**kw) == _lib.OK


@pytest.mark.parametrize("kw,code,msg", [
    *[({p: None}, INV, b"null pointer") for p in ("q", "qo", "k", "ko", "cos", "sin", "pos")],
    (dict(D=96), UNS, b"head_dim"), (dict(dtype=2), UNS, b"bf16 or fp16"), (dict(rope=24), INV, b"rope_dim"),
    (dict(rope=512), INV, b"rope_dim"), (dict(rope=0), INV, b"rope_dim"), (dict(n=0), INV, b"axes"), (dict(n=5), INV, b"axes"),
    (dict(sections=None), INV, b"axes"), (dict(sections=(11, 11, 11)), INV, b"sum to"),
    (dict(sections=(20, 20, -8)), INV, b"negative section"), (dict(sections=(2, 15, 15)), INV, b"interleaved"),
    (dict(eps=-1.0), INV, b"eps"), (dict(eps=NAN), INV, b"eps"), (dict(S=-1), INV, b"negative"), (dict(Hk=-1), INV, b"negative"),
    (dict(q=0x10008), INV, b"16-byte"), (dict(kot=4), INV, b"16-byte"), (dict(gk=0x60002), INV, b"16-byte"),
    (dict(qo=0x10000), INV, b"same strides"), (dict(ko=0x40000), INV, b"same strides"), (dict(qo=0x40000), INV, b"overlaps"),
    (dict(ko=0x10000), INV, b"overlaps"), (dict(ko=0x20000), INV, b"overlaps"),
    (dict(cos=0x70001), INV, b"aligned to its type"), (dict(qot=0), INV, b"share memory"), (dict(koh=0), INV, b"share memory"),
])
def test_qk_norm_rope_axes(kw, code, msg):
    assert axes(**kw) == code
    assert msg in _lib.lib().genllm_last_error()


def test_qk_norm_rope_axes_nothing_to_do():
    for kw in (dict(S=0), dict(Hq=0, Hk=0, q=None, k=None)):
        assert axes(**kw) == _lib.OK


def _bf16(*shape):
    return torch.zeros(shape, dtype=torch.bfloat16)


@pytest.mark.parametrize("call", [
    lambda t: paged.gated_delta_rule(t, t, t, t, t, t, t, 1.0),
    lambda t: paged.gated_delta_rule(t, t, t, t, t, t, t, 1.0, stream=0),
    lambda t: paged.causal_conv(t, t, t),
    lambda t: paged.qk_norm_rope_axes(t, None, t, None, None, None, 1e-6, t, t, t, (1,)),
])
def test_calls_on_tensors(call):
    """What is no tensor, has another type or is not on a GPU is refused before anything else is looked at."""
    for bad, msg in ((3, "must be a tensor"), (None, "must be a tensor"), (torch.zeros(2, 2, 2), "bf16 or float16"),
                     (_bf16(2, 2, 2), "GPU tensor"), (_bf16(2, 2, 2).to_sparse(), "strided")):
        with pytest.raises(ValueError, match=msg):
            call(bad)


def test_calls_argument_count():
    m = _lib.calls()
    for f in (m.gated_delta_rule, m.causal_conv, m.qk_norm_rope_axes):
        with pytest.raises(TypeError):
            f(1)
    with pytest.raises(TypeError):
        m.bind(0)
    with pytest.raises(ValueError):
        m.bind(0, 0, 0, 0)
