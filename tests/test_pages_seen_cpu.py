"""The bound over seen positions by hand: what a row does not see leaves its
result and its bound as they are."""
import math

import pytest

torch = pytest.importorskip("torch")

import pages_ref as R  # noqa: E402
import pages_seen as V  # noqa: E402


def pool(hidden):
    """Six positions of one sequence in pages of two; positions 0 and 1 hold ``hidden``."""
    class Pages:
        head_dim, n_head_kv, page_size = 4, 2, 2
        k_scale = v_scale = None
    g = torch.Generator().manual_seed(3)
    Pages.k = torch.randn((3, 2, 2, 4), generator=g).double()
    Pages.v = torch.randn((3, 2, 2, 4), generator=g).double()
    if hidden is not None:
        Pages.k[0] = hidden
        Pages.v[0] = hidden
    return Pages


TABLE = torch.tensor([[0, 1, 2]], dtype=torch.int32)


@pytest.mark.parametrize("hidden", [1e3, 1e30, math.inf, math.nan])
def test_hidden_positions_leave_the_bound(hidden):
    q = torch.randn((2, 16), generator=torch.Generator().manual_seed(5))
    a = V.attention(q, 4, pool(None), TABLE, [0, 2], [6], window=3)
    b = V.attention(q, 4, pool(hidden), TABLE, [0, 2], [6], window=3)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    assert (a[1] > 0).all()


@pytest.mark.parametrize("window,sink", [(0, 0), (2, 0), (2, 1)])
def test_the_two_forms_agree(window, sink):
    q = torch.randn((4, 16), generator=torch.Generator().manual_seed(7))
    a, bound_a = R.attention(q, 4, pool(None), TABLE, [0, 4], [6], window, sink)
    b, bound_b = V.attention(q, 4, pool(None), TABLE, [0, 4], [6], window, sink)
    assert torch.allclose(a, b, rtol=1e-12, atol=1e-12)
    assert (bound_b <= bound_a * (1 + 1e-12)).all()


def test_rows_that_see_a_value_that_is_not_finite():
    p = pool(None)
    p.v[1, 1, 0, 3] = math.inf  # position 2, KV head 1
    q = torch.randn((6, 16), generator=torch.Generator().manual_seed(9))
    a, _ = V.attention(q, 4, p, TABLE, [0, 6], [6])
    b, _ = R.attention(q, 4, p, TABLE, [0, 6], [6])
    hit = torch.isinf(a)
    assert torch.equal(hit, torch.isinf(b)) and not torch.isnan(a).any()
    assert hit.nonzero()[:, 0].unique().tolist() == [2, 3, 4, 5]
    assert hit.nonzero()[:, 1].unique().tolist() == [11, 15]


def test_nothing_seen():
    q = torch.randn((3, 16))
    out, _ = V.attention(q, 4, pool(None), torch.full((1, 3), -1, dtype=torch.int32), [0, 3], [6])
    assert (out == 0).all()
    out, _ = V.attention(q, 4, pool(None), TABLE, [0, 3], [1])
    assert (out[:2] == 0).all() and (out[2] != 0).any()
