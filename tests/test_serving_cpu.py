"""The serving entries' argument checks, on a machine without a device: what cannot be meant is INVALID or UNSUPPORTED
before anything is launched, and empty work is fine."""

import ctypes

import pytest

from intent_ir_b200 import _lib

torch = pytest.importorskip("torch")

P = ctypes.c_void_p(0x7F0000000000)  # stands for a device address; nothing on the host dereferences it
ODD = ctypes.c_void_p(0x7F0000000008)
BIG = 1 << 62


def _norm(**k):
    a = dict(x=P, xs=64, res=P, rs=64, w=P, y=P, h=P, hs=64, scale=P, dtype=_lib.BF16, wt=_lib.BF16, out=_lib.E4M3, rows=4, cols=64, group=32, eps=1e-6)
    a.update(k)
    return _lib.load().ib200_rmsnorm(*a.values(), None)


def _w4(**k):
    a = dict(x=P, xs=64, xsc=None, xg=0, q=P, s=P, z=P, bias=P, y=P, xt=_lib.BF16, st=_lib.BF16, out=_lib.BF16, m=4, n=8, k=64, group=32, scratch=None,
             bytes=0, status=None)
    a.update(k)
    return _lib.load().ib200_w4_matmul(*a.values(), None)


def _append(**k):
    a = dict(k=P, kt=128, kh=64, v=P, vt=128, vh=64, kc=P, vc=P, ks=P, vs=P, table=P, lens=P, cu=None, dtype=_lib.BF16, held=_lib.I8, tokens=4, batch=2, heads=2,
             dim=64, pages=9, block=16, blocks=4)
    a.update(k)
    return _lib.load().ib200_kv8_append(*a.values(), None)


def _attention(**k):
    a = dict(q=P, qt=256, qh=64, kc=P, vc=P, ks=P, vs=P, table=P, lens=P, cu=None, o=P, lse=P, dtype=_lib.BF16, held=_lib.I8, tokens=4, batch=2, qheads=4, heads=2,
             dim=64, pages=9, block=16, blocks=4, window=0, scale=0.1, scratch=P, bytes=1 << 40)
    a.update(k)
    return _lib.load().ib200_attention_kv8(*a.values(), None)


@pytest.mark.parametrize("call,bad", [
    (_norm, dict(rows=-1)), (_norm, dict(cols=-1)), (_norm, dict(rows=BIG)), (_norm, dict(rows=1 << 30, cols=1 << 30)), (_norm, dict(x=None)), (_norm, dict(y=None)),
    (_norm, dict(scale=None)), (_norm, dict(res=None)), (_norm, dict(xs=63)), (_norm, dict(rs=1)), (_norm, dict(hs=-64)), (_norm, dict(xs=BIG)),
    (_w4, dict(m=-1)), (_w4, dict(n=-1)), (_w4, dict(k=-32)), (_w4, dict(n=1 << 30, k=1 << 30)), (_w4, dict(x=None)), (_w4, dict(q=None)), (_w4, dict(s=None)), (_w4, dict(y=None)),
    (_w4, dict(q=ODD)), (_w4, dict(xs=63)), (_w4, dict(xg=1)), (_w4, dict(xt=_lib.I8)), (_w4, dict(xt=_lib.I8, xg=3, xsc=P)), (_w4, dict(xt=_lib.I8, xg=1)),
    (_w4, dict(scratch=ODD)),
    (_append, dict(tokens=-1)), (_append, dict(batch=-1)), (_append, dict(pages=-1)), (_append, dict(tokens=3)), (_append, dict(k=None)), (_append, dict(vs=None)),
    (_append, dict(table=None)), (_append, dict(lens=None)), (_append, dict(kc=ODD)), (_append, dict(pages=1 << 31 - 1, heads=1 << 15, block=1024)), (_append, dict(blocks=1 << 40)),
    (_attention, dict(tokens=-1)), (_attention, dict(blocks=-1)), (_attention, dict(tokens=3)), (_attention, dict(qheads=3)), (_attention, dict(qheads=-2)), (_attention, dict(heads=0)),
    (_attention, dict(window=-1)), (_attention, dict(q=None)), (_attention, dict(o=None)), (_attention, dict(ks=None)), (_attention, dict(table=None)),
    (_attention, dict(vc=ODD)), (_attention, dict(scratch=ODD)),
])
def test_arguments_that_cannot_be_meant_are_invalid(call, bad):
    assert call(**bad) == _lib.ERR_INVALID, (bad, _lib.last_error())


@pytest.mark.parametrize("call,bad", [
    (_norm, dict(dtype=_lib.F64)), (_norm, dict(dtype=_lib.E4M3)), (_norm, dict(wt=_lib.F16)), (_norm, dict(out=_lib.U8)), (_norm, dict(out=_lib.F32)), (_norm, dict(group=48)),
    (_norm, dict(group=-32)), (_norm, dict(out=_lib.BF16)),
    (_w4, dict(xt=_lib.F32)), (_w4, dict(xt=99)), (_w4, dict(st=_lib.F64)), (_w4, dict(out=_lib.I8)), (_w4, dict(group=16)), (_w4, dict(group=0)), (_w4, dict(k=72)),
    (_append, dict(held=_lib.U8)), (_append, dict(dtype=_lib.F32)), (_append, dict(dim=80)), (_append, dict(block=8)), (_append, dict(block=0)), (_append, dict(block=2048)),
    (_append, dict(heads=1 << 17)), (_append, dict(tokens=1 << 31)),
    (_attention, dict(held=_lib.BF16)), (_attention, dict(dtype=_lib.F32)), (_attention, dict(dim=96)), (_attention, dict(block=24)), (_attention, dict(qheads=1 << 17)),
])
def test_what_the_kernels_do_not_cover_is_unsupported(call, bad):
    assert call(**bad) == _lib.ERR_UNSUPPORTED, (bad, _lib.last_error())


def test_empty_work_launches_nothing():
    for rows, cols in ((0, 64), (4, 0)):
        assert _norm(rows=rows, cols=cols, x=None, y=None) == _lib.OK
    assert _w4(m=0, x=None) == _lib.OK and _w4(n=0, q=None) == _lib.OK
    for empty in (dict(tokens=0), dict(heads=0), dict(batch=0, tokens=0)):
        assert _append(**empty) == _lib.OK
    for empty in (dict(tokens=0), dict(qheads=0, heads=0), dict(batch=0, tokens=0)):
        assert _attention(**empty) == _lib.OK


def test_serving_ops_have_no_cpu_path():
    from intent_ir_b200 import ops
    from intent_ir_b200.errors import B200RuntimeError

    x = torch.zeros(2, 64, dtype=torch.bfloat16)
    with pytest.raises(B200RuntimeError):
        ops.rmsnorm(x)
    with pytest.raises(B200RuntimeError):
        ops.w4_matmul(x, torch.zeros(4, 32, dtype=torch.uint8), torch.ones(4, 1))
    with pytest.raises(B200RuntimeError):
        ops.kv8_append(x, x, x, x, x, x, x, x)
    with pytest.raises(B200RuntimeError):
        ops.attention_kv8(x, x, x, x, x, x, x)
