"""The C entry points of sorted and combined tokens refuse bad arguments before any launch (no GPU)."""
import pytest

from eva_amd import _lib

FAKE = 0x10000


def _order(**kw):
    a = dict(sel=FAKE, rows=8, k=4, first=0, n=16, starts=FAKE, pos=FAKE, ws=FAKE, nb=1 << 20)
    a.update(kw)
    return _lib.lib().evamx_expert_order(a["sel"], a["rows"], a["k"], a["first"], a["n"], a["starts"], a["pos"], a["ws"], a["nb"], None)


def _sort(**kw):
    a = dict(x=FAKE, dt=1, st=64, rows=8, h=64, k=4, pos=FAKE, starts=FAKE, n=16, out=FAKE, ost=64, orows=32)
    a.update(kw)
    return _lib.lib().evamx_sort_tokens(a["x"], a["dt"], a["st"], a["rows"], a["h"], a["k"], a["pos"], a["starts"], a["n"], a["out"], a["ost"],
                                        a["orows"], None)


def _combine(**kw):
    a = dict(y=FAKE, dt=1, st=64, yrows=32, rows=8, h=64, k=4, pos=FAKE, w=FAKE, res=None, rst=0, out=FAKE, ost=64)
    a.update(kw)
    return _lib.lib().evamx_combine_tokens(a["y"], a["dt"], a["st"], a["yrows"], a["rows"], a["h"], a["k"], a["pos"], a["w"], a["res"], a["rst"],
                                           a["out"], a["ost"], None)


def _grad(**kw):
    a = dict(g=FAKE, dt=1, gst=64, y=FAKE, yst=64, yrows=32, rows=8, h=64, k=4, pos=FAKE, starts=FAKE, n=16, w=FAKE, dy=FAKE, dyst=64, dw=FAKE)
    a.update(kw)
    return _lib.lib().evamx_combine_tokens_grad(a["g"], a["dt"], a["gst"], a["y"], a["yst"], a["yrows"], a["rows"], a["h"], a["k"], a["pos"],
                                                a["starts"], a["n"], a["w"], a["dy"], a["dyst"], a["dw"], None)


SIZES = [dict(rows=-1), dict(k=0), dict(k=33), dict(rows=(1 << 26) // 4 + 1)]
ROWS = SIZES + [dict(dt=3), dict(dt=-1), dict(h=0), dict(h=(1 << 18) + 1)]
EXPERTS = [dict(n=0), dict(n=1025)]


@pytest.mark.parametrize("call,bad", [
    *((_order, b) for b in SIZES + EXPERTS + [dict(sel=0), dict(starts=0), dict(pos=0), dict(rows=1000, ws=0), dict(rows=1000, ws=FAKE + 2)]),
    *((_sort, b) for b in ROWS + EXPERTS + [dict(x=0), dict(pos=0), dict(starts=0), dict(out=0), dict(st=63), dict(ost=63), dict(orows=-1)]),
    *((_combine, b) for b in ROWS + [dict(y=0), dict(pos=0), dict(out=0), dict(st=63), dict(ost=63), dict(yrows=-1), dict(res=FAKE, rst=63)]),
    *((_grad, b) for b in ROWS + EXPERTS + [dict(g=0), dict(y=0), dict(pos=0), dict(starts=0), dict(w=0), dict(dy=0), dict(dw=0),
                                            dict(gst=63), dict(yst=63), dict(dyst=63), dict(yrows=-1)])])
def test_refused(call, bad):
    assert call(**bad) == _lib.EVAMX_EINVAL
    assert _lib.lib().evamx_last_error()


def test_sizes():
    L = _lib.lib()
    assert L.evamx_expert_order_workspace_bytes(256, 8, 256) == 0                                      # one workgroup's work
    assert 0 < L.evamx_expert_order_workspace_bytes(1 << 23, 8, 1024) <= 256 * 1024 * 4
    assert L.evamx_expert_order_workspace_bytes(8, 8, 1025) == 0
    assert _order(rows=1000, nb=0) == _lib.EVAMX_ENOSPACE
    assert _combine(rows=0, pos=None, out=None) == _lib.EVAMX_OK             # nothing to do, nothing launched
    assert _sort(orows=0, out=None) == _lib.EVAMX_OK
