"""Sizes and addresses that the hybrid layers' entry points have to refuse or answer without any device work."""
import ctypes as C

import pytest

from genllm_amd import _lib

INT_MAX = 2 ** 31 - 1


@pytest.mark.parametrize("shape", [
    (1, 100, 1, 1, 64, 8), (1, 100, 1, 1, 64, 15), (1, 100, 1, 1, 8, 64), (1, 100, 1, 1, 96, 128), (1, 100, 1, 1, 128, 256),
    (INT_MAX, INT_MAX, 1, INT_MAX, INT_MAX, INT_MAX), (INT_MAX, 100, 1, INT_MAX, 128, 128), (1 << 16, 100, 8, 16, 64, 64),
    (1, (1 << 30) + 1, 1, 1, 64, 64), (0, 100, 1, 1, 64, 64), (1, 0, 1, 1, 64, 64), (1, 100, 0, 1, 64, 64), (1, 100, 1, -1, 64, 64)])
def test_workspace_of_sizes_that_are_not_served(shape):
    """None, for any sizes at all: a caller asks before the call itself refuses them."""
    assert _lib.lib().genllm_gated_delta_workspace_bytes(*shape) == 0


def test_workspace_at_the_limits():
    f = _lib.lib().genllm_gated_delta_workspace_bytes
    assert f(1, 12, 16, 32, 128, 128) == 0 and f(1, 1 << 30, 16, 32, 128, 128) > 0
    assert 0 < f(1 << 15, 64, 16, 16, 64, 64) < 1 << 30 and f(1, 64, 1, 1 << 19, 64, 64) > 0


def delta(**kw):
    """A call on placeholder addresses far apart from each other; only ones that are refused are made."""
    a = dict(q=0x1000000, qb=4096, qt=1024, qh=128, k=0x2000000, kb=4096, kt=1024, kh=128, v=0x3000000, vb=8192, vt=2048, vh=128,
             a=0x4000000, ab=64, at=16, b=0x5000000, bb=64, bt=16, a_log=0x6000000, dt=0x7000000, state=0x10000000, n=4,
             ids=None, lens=None, out=0x9000000, ob=8192, ot=2048, oh=128, B=2, S=4, Hk=8, Hv=16, Dk=128, Dv=128, dtype=30,
             scale=0.1, l2=1e-6, ws=None, wsb=0, stream=None)
    assert not set(kw) - set(a)
    return _lib.lib().genllm_gated_delta_rule(*dict(a, **kw).values())


@pytest.mark.parametrize("kw,msg", [
    (dict(out=0x1000000 + 2 * 1024), b"out overlaps q"),  # a token further on
    (dict(out=0x1000000 - 0x8000 + 16), b"out overlaps q"),  # the last row's last elements
    (dict(out=0x2000000 + 16), b"out overlaps k"), (dict(out=0x3000000 + 2 * 128), b"out overlaps v"),
    (dict(out=0x3000000 - 2 * 2048), b"out overlaps v"), (dict(out=0x3000000, ob=8192 * 2), b"out overlaps v"),
    (dict(out=0x4000000), b"out overlaps a"), (dict(out=0x5000000), b"out overlaps b"),
    (dict(out=0x5000000 - 0x8000 + 16), b"out overlaps b"), (dict(out=0x6000020), b"out overlaps a_log"),
    (dict(out=0x10000000 + 0x100000), b"the state overlaps out"), (dict(state=0x3000000), b"the state overlaps v"),
    (dict(state=0x4000000 - 0x100000), b"the state overlaps a"),
    # states that only ids reach
    (dict(ids=0x8000000, out=0x10000000 + 3 * 0x100000), b"the state overlaps out"), (dict(ids=0x9000100), b"out overlaps state_ids"),
    (dict(lens=0x10000010), b"the state overlaps seq_lens"), (dict(ot=1024), b"rows of out share memory"),
    (dict(oh=64), b"rows of out share memory"),
    (dict(S=100, qb=1 << 17, kb=1 << 17, vb=1 << 18, ob=1 << 18, ws=0x3000000, wsb=1 << 30), b"the workspace overlaps v"),
    (dict(S=100, qb=1 << 17, kb=1 << 17, vb=1 << 18, ob=1 << 18, ws=0xFFFF000, wsb=1 << 30), b"the workspace overlaps the state"),
    (dict(S=100, qb=1 << 17, kb=1 << 17, vb=1 << 18, ob=1 << 18, ws=0x9000000, wsb=1 << 30), b"the workspace overlaps out")])
def test_delta_rule_refuses_what_it_would_write_over(kw, msg):
    assert delta(**kw) == _lib.ERR_INVALID
    assert msg in _lib.lib().genllm_last_error(), _lib.lib().genllm_last_error()


def axes(sections=(11, 11, 10), **kw):
    """Eight heads of q and two of k beside each other in rows of 2560; outputs head by head."""
    a = dict(q=0x1000000, qt=2560, qh=256, qo=0x2000000, qot=256, qoh=1024, gq=0x3000000, Hq=8, k=0x1000000 + 2 * 2048, kt=2560,
             kh=256, ko=0x5000000, kot=256, koh=1024, gk=0x6000000, Hk=2, eps=1e-6, cos=0x7000000, sin=0x8000000, rows=100,
             rope=64, pos=0x9000000, ps=4, n=3, sec=(C.c_int32 * 8)(*sections), inter=1, S=4, D=256, dtype=30, stream=None)
    assert not set(kw) - set(a)
    return _lib.lib().genllm_qk_norm_rope_axes(*dict(a, **kw).values())


@pytest.mark.parametrize("kw,msg", [
    (dict(qo=0x1000000 + 2 * 2560, qot=2560, qoh=256), b"q_out overlaps q"),  # a token further on
    (dict(qo=0x1000000 + 2 * 256, qot=2560, qoh=256), b"q_out overlaps q"),  # a head further on
    (dict(qo=0x1000000 + 2 * 512, qot=2560, qoh=256), b"q_out overlaps q"),
    (dict(ko=0x1000000 + 2 * 2048 + 16, kot=2560, koh=256), b"k_out overlaps"), (dict(ko=0x1000000, kot=2560, koh=256), b"k_out overlaps q"),
    (dict(ko=0x2000000 + 2 * 7 * 1024), b"k_out overlaps q_out"), (dict(ko=0x2000000 - 2 * 2048 + 16), b"k_out overlaps q_out"),
    (dict(qo=0x3000000), b"q_out overlaps gamma_q"), (dict(ko=0x3000000), b"k_out overlaps gamma_q"),
    (dict(qo=0x6000000 - 512), b"q_out overlaps gamma_k"), (dict(qo=0x7000000 + 99 * 256), b"q_out overlaps cos"),
    (dict(ko=0x8000000 - 16), b"k_out overlaps sin"), (dict(ko=0x9000000), b"k_out overlaps positions"),
    (dict(qot=128), b"rows of q_out share memory"), (dict(koh=256), b"rows of k_out share memory")])
def test_rotation_refuses_what_it_would_write_over(kw, msg):
    assert axes(**kw) == _lib.ERR_INVALID
    assert msg in _lib.lib().genllm_last_error(), _lib.lib().genllm_last_error()


def conv(**kw):
    a = dict(x=0x1000000, xb=4096, xt=64, w=0x2000000, bias=0x3000000, out=0x9000000, ob=4096, ot=64, state=0x8000000, n=4, ids=None,
             lens=None, B=2, S=64, C=64, W=4, dtype=30, silu=1, stream=None)
    assert not set(kw) - set(a)
    return _lib.lib().genllm_causal_conv(*dict(a, **kw).values())


@pytest.mark.parametrize("kw,msg", [
    (dict(state=0x1000000 + 64), b"the state overlaps x"), (dict(state=0x1000000 - 2 * 3 * 64 * 2 + 2), b"the state overlaps x"),
    (dict(state=0x9000000 + 2 * 4096 * 2 - 2), b"the state overlaps out"), (dict(state=0x2000000), b"the state overlaps the weight"),
    (dict(state=0x3000000 - 2), b"the state overlaps the bias"), (dict(out=0x2000000 + 510), b"out overlaps the weight"),
    # a state that only ids reach
    (dict(ids=0x7000000, out=0x8000000 + 3 * 3 * 64 * 2), b"the state overlaps out"), (dict(lens=0x9000000), b"out overlaps seq_lens"),
    (dict(out=0x1000000 + 2 * 64, xt=128, ot=128, ob=8192 + 64, xb=8192), b"out overlaps x"),  # beside x in the first entry only
    (dict(ot=32, ob=4096), b"rows of out share memory"), (dict(ob=128, ot=128), b"rows of out share memory")])
def test_convolution_refuses_what_it_would_write_over(kw, msg):
    assert conv(**kw) == _lib.ERR_INVALID
    assert msg in _lib.lib().genllm_last_error(), _lib.lib().genllm_last_error()
