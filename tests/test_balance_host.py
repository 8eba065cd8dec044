"""The balance loss's C entry points refuse bad arguments before any launch (no GPU)."""
import pytest

from eva_amd import _lib

FAKE = 0x10000


def _loss(**kw):
    a = dict(z=FAKE, dt=2, st=64, rows=8, e=64, sel=FAKE, k=4, score=0, starts=None, n=1, mask=None, loss=FAKE, counts=FAKE, tokens=FAKE,
             ws=FAKE, nb=1 << 30)
    a.update(kw)
    return _lib.lib().evamx_balance_loss(a["z"], a["dt"], a["st"], a["rows"], a["e"], a["sel"], a["k"], a["score"], a["starts"], a["n"],
                                         a["mask"], a["loss"], a["counts"], a["tokens"], a["ws"], a["nb"], None)


def _grad(**kw):
    a = dict(gl=FAKE, z=FAKE, dt=2, st=64, rows=8, e=64, k=4, score=0, starts=None, n=1, mask=None, counts=FAKE, tokens=FAKE, grad=FAKE)
    a.update(kw)
    return _lib.lib().evamx_balance_grad(a["gl"], a["z"], a["dt"], a["st"], a["rows"], a["e"], a["k"], a["score"], a["starts"], a["n"],
                                         a["mask"], a["counts"], a["tokens"], a["grad"], None)


COMMON = [dict(z=0), dict(dt=3), dict(dt=-1), dict(st=63), dict(st=-1), dict(rows=-1), dict(rows=(1 << 24) + 1), dict(e=0), dict(e=513),
          dict(k=0), dict(k=33), dict(score=2), dict(n=0), dict(n=2), dict(n=(1 << 16) + 1, starts=FAKE), dict(counts=0), dict(tokens=0)]


@pytest.mark.parametrize("bad", COMMON + [dict(sel=0), dict(loss=0), dict(ws=0)])
def test_loss_refuses(bad):
    assert _loss(**bad) == _lib.EVAMX_EINVAL
    assert _lib.lib().evamx_last_error()


@pytest.mark.parametrize("bad", COMMON + [dict(gl=0), dict(grad=0)])
def test_grad_refuses(bad):
    assert _grad(**bad) == _lib.EVAMX_EINVAL
    assert _lib.lib().evamx_last_error()


def test_workspace_is_checked():
    assert _loss(nb=0) == _lib.EVAMX_ENOSPACE
    assert _lib.lib().evamx_balance_workspace_bytes(1000, 64, 4) > 0
    assert _grad(rows=0, z=None, grad=None) == _lib.EVAMX_OK          # nothing to do, nothing launched
