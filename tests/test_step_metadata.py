"""Host checks of the calls that take a step's metadata. Nothing is launched."""
from serving import _native

INVALID = -1


def test_write_accepted_step_refusals():
    L = _native.lib()
    commit = lambda **kw: L.pkv_write_accepted_step(*{**dict(  # noqa: E731
        kp=16, vp=16, pl=64, layers=1, nb=4, bs=16, k=16, v=16, rl=64, table=16, max_blk=2,
        start=16, step=16, qsl=16, path=16, lens=16, n=2, T=8, depth=2, row=64, dtype=2),
        **kw}.values(), None, None)
    assert commit(dtype=7) == INVALID and commit(bs=10) == INVALID
    assert commit(row=0) == INVALID and commit(layers=-1) == INVALID
    assert commit(path=None) == INVALID and commit(table=None) == INVALID
    assert commit(layers=0, k=None) == 0 and commit(n=0, step=None) == 0 and commit(depth=0) == 0
