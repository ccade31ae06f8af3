"""The serving entries' argument checks, on a machine without a device: what cannot be meant is INVALID or UNSUPPORTED
before anything is launched, and empty work is fine."""

import ctypes

import pytest

from intent_ir_b200 import _lib

torch = pytest.importorskip("torch")

P = ctypes.c_void_p(0x7F0000000000)  # stands for a device address; nothing on the host dereferences it
ODD = ctypes.c_void_p(0x7F0000000008)
BIG = 1 << 62


def _call(entry, layout, pointers, fields, changes):
    """The entry with these arguments, `changes` made."""
    a = {**{p: P for p in pointers.split()}, **fields}
    assert set(changes) <= set(a)
    a.update(changes)
    return getattr(_lib.load(), entry)(layout.pack(*(v or 0 if v is None or isinstance(v, (int, float)) else v.value for v in a.values())), None)


def _norm(**k):
    return _call("ib200_rmsnorm", _lib.RMSNORM_ARGS, "x res w y h scale",
                 dict(xs=64, rs=64, hs=64, dtype=_lib.BF16, wt=_lib.BF16, out=_lib.E4M3, rows=4, cols=64, group=32, eps=1e-6), k)


def _w4(**k):
    return _call("ib200_w4_matmul", _lib.W4_ARGS, "x xsc q s z bias y scratch status",
                 dict(xs=64, xg=0, xt=_lib.BF16, st=_lib.BF16, out=_lib.BF16, m=4, n=8, k=64, group=32, bytes=1 << 40), k)


def _append(**k):
    return _call("ib200_kv8_append", _lib.KV8_APPEND_ARGS, "k v kc vc ks vs table lens cu",
                 dict(kt=128, kh=64, vt=128, vh=64, dtype=_lib.BF16, held=_lib.I8, tokens=4, batch=2, heads=2, dim=64, pages=9, block=16, blocks=4),
                 {"cu": None, **k})


def _attention(**k):
    return _call("ib200_attention_kv8", _lib.ATTENTION_KV8_ARGS, "q kc vc ks vs table lens cu o lse scratch",
                 dict(qt=256, qh=64, dtype=_lib.BF16, held=_lib.I8, tokens=4, batch=2, qheads=4, heads=2, dim=64, pages=9, block=16, blocks=4, window=0,
                      bytes=1 << 40, scale=0.1), {"cu": None, **k})


@pytest.mark.parametrize("call,bad", [
    (_norm, dict(rows=-1)), (_norm, dict(cols=-1)), (_norm, dict(rows=BIG)), (_norm, dict(rows=1 << 30, cols=1 << 30)), (_norm, dict(x=None)), (_norm, dict(y=None)),
    (_norm, dict(scale=None)), (_norm, dict(res=None)), (_norm, dict(xs=63)), (_norm, dict(rs=1)), (_norm, dict(hs=-64)), (_norm, dict(xs=BIG)),
    (_w4, dict(m=-1)), (_w4, dict(n=-1)), (_w4, dict(k=-32)), (_w4, dict(n=1 << 30, k=1 << 30)), (_w4, dict(x=None)), (_w4, dict(q=None)), (_w4, dict(s=None)), (_w4, dict(y=None)),
    (_w4, dict(q=ODD)), (_w4, dict(xs=63)), (_w4, dict(xg=1)), (_w4, dict(xt=_lib.I8)), (_w4, dict(xt=_lib.I8, xg=3, xsc=P)), (_w4, dict(xt=_lib.I8, xg=1, xsc=None)),
    (_w4, dict(scratch=ODD)),
    (_append, dict(tokens=-1)), (_append, dict(batch=-1)), (_append, dict(pages=-1)), (_append, dict(tokens=3)), (_append, dict(k=None)), (_append, dict(vs=None)),
    (_append, dict(table=None)), (_append, dict(lens=None)), (_append, dict(kc=ODD)), (_append, dict(pages=1 << 31 - 1, heads=1 << 15, block=1024)), (_append, dict(blocks=1 << 40)),
    (_attention, dict(tokens=-1)), (_attention, dict(blocks=-1)), (_attention, dict(tokens=3)), (_attention, dict(qheads=3)), (_attention, dict(qheads=-2)), (_attention, dict(heads=0)),
    (_attention, dict(window=-1)), (_attention, dict(q=None)), (_attention, dict(o=None)), (_attention, dict(ks=None)), (_attention, dict(table=None)),
    (_attention, dict(vc=ODD)), (_attention, dict(scratch=ODD)), (_attention, dict(o=ctypes.c_void_p(0x7F0000000004))),
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


def test_scratch_that_is_too_small_is_refused_and_no_arguments_are_invalid():
    size = _lib.load().ib200_attention_kv8_scratch_bytes
    need = size(4, 2, 4, 2, 64, 16, 4, 0)
    assert need > 0 and _attention(cu=P, bytes=need - 1) == _lib.ERR_BUFFER and _attention(cu=P, scratch=None) == _lib.ERR_BUFFER
    assert size(4, 2, 4, 2, 64, 16, 4, 1) == 0 and size(4, 2, 4, 2, 64, 16, 4000, 1) > 0  # short tables: a cluster to a unit, no scratch
    assert _attention(blocks=4000, bytes=8) == _lib.ERR_BUFFER
    w4 = _lib.load().ib200_w4_scratch_bytes
    assert w4(_lib.BF16, 4, 64, 64, 32) == 0 and w4(_lib.BF16, 20, 64, 64, 32) == 32 * 256 * 2 and _w4(m=20, bytes=8) == _lib.ERR_BUFFER
    for entry in ("ib200_rmsnorm", "ib200_w4_matmul", "ib200_kv8_append", "ib200_attention_kv8"):
        assert getattr(_lib.load(), entry)(None, None) == _lib.ERR_INVALID


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
