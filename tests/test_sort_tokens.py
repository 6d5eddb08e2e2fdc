"""What the moves of tokens to their experts and back refuse (no GPU needed: an error before anything is launched)."""
import pytest

X, Y, D, P = 1 << 20, 1 << 21, 1 << 22, 4096


def sort(x=X, ldx=8, y=Y, ldy=8, pos=P, total=P, T=4, k=2, H=8, dtype=0):
    from promoe_amd import _lib as L
    return L.lib.moe_sort_rows(x, ldx, y, ldy, pos, total, T, k, H, dtype, None)


def unsort(x=X, ldx=8, y=Y, ldy=8, pos=P, total=P, T=4, k=2, H=8, dtype=0):
    from promoe_amd import _lib as L
    return L.lib.moe_unsort_rows(x, ldx, y, ldy, pos, None, T, k, H, dtype, None)


def grad(x=X, ldx=8, y=Y, ldy=8, pos=P, total=P, T=4, k=2, H=8, dtype=0, dy=D, lddy=8, w=P, dw=P + 2048):
    from promoe_amd import _lib as L
    return L.lib.moe_unsort_rows_grad(dy, lddy, x, ldx, pos, w, total, y, ldy, dw, T, k, H, dtype, None)


@pytest.mark.parametrize("call", [sort, unsort, grad], ids=lambda c: c.__name__)
@pytest.mark.parametrize("kw", [dict(T=-1), dict(k=0), dict(H=-1), dict(dtype=3), dict(dtype=-1), dict(ldx=7), dict(ldy=7), dict(x=None), dict(pos=None),
                                dict(T=1 << 26), dict(T=1 << 25, k=64), dict(H=1 << 24, ldx=1 << 24, ldy=1 << 24), dict(ldx=1 << 31),
                                dict(ldy=1 << 31)], ids=str)
def test_refused(call, kw):
    from promoe_amd import _lib as L
    assert call(**kw) == L.MOE_EINVAL and b"sort_rows" in L.lib.moe_last_error()


def test_refused_each_by_itself():
    from promoe_amd import _lib as L
    for rc in (sort(total=None), sort(y=None), unsort(y=None), grad(dy=None), grad(w=None), grad(total=None), grad(y=None, dw=None), grad(lddy=7)):
        assert rc == L.MOE_EINVAL
    for rc in (sort(y=X + 16), sort(y=X - 7 * 16), unsort(y=X + 7 * 16), unsort(y=X - 4 * 16 + 8), grad(y=D + 48), grad(y=X + 7 * 16)):
        assert rc == L.MOE_EINVAL and b"overlap" in L.lib.moe_last_error()
    odd = (1 << 23) - 1                                   # single elements, more than a grid has room for
    for call in (sort, unsort):
        assert call(H=odd, ldx=odd, ldy=odd, T=1, k=1, x=1 << 40, y=1 << 41) == L.MOE_EINVAL and b"boundaries" in L.lib.moe_last_error()


def test_nothing_to_do():
    for call in (sort, unsort, grad):
        assert call(T=0, x=None, y=None) == 0 or call is grad
    assert sort(H=0, ldx=0, ldy=0, x=None, y=None) == 0 and unsort(H=0, ldx=0, ldy=0, x=None, y=None) == 0


def test_gradient_of_rows_without_columns():
    """dw is written (zeros) whatever the columns, so places and weights have to be there; without dw nothing is left to do."""
    from promoe_amd import _lib as L
    none = dict(H=0, ldx=0, ldy=0, lddy=0)
    for kw in (dict(pos=None), dict(w=None)):
        assert grad(**none, **kw) == L.MOE_EINVAL and b"missing" in L.lib.moe_last_error()
    assert grad(**none, dw=None, pos=None, w=None, total=None, x=None, y=None, dy=None) == 0
