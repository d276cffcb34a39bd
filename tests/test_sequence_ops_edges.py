"""attention, relative_attention and linear_cross_entropy where values are not finite, where masks leave nothing of a tile, and
where scales meet the ends of fp32's range. References and bounds are those of test_sequence_ops."""
import numpy as np
import pytest

from test_sequence_ops import U, attend, attention_reference, loss_of, loss_reference, within

NAMES = ("o", "dq", "dk", "dv")


# ---- attention: NaN that takes part ---------------------------------------------------------------------------
# 1 to 16 rows per key head are streamed, 17 and more go through the tiles; 300 keys make several parts in both.
QUERIES, KEYS = [1, 4, 16, 17, 130], [10, 77, 300]


def _two_heads(Q, K, seed=0):
    rng = np.random.default_rng(seed)
    return [rng.standard_normal((1, n, 2, 64)).astype(np.float32) for n in (Q, K, K, Q)]


@pytest.mark.gpu
@pytest.mark.parametrize("K", KEYS)
@pytest.mark.parametrize("Q", QUERIES)
def test_attention_nan_in_a_query_reaches_its_row(Q, K):
    """A NaN in a query of head 0: its row of o and dq is NaN, as is all that its head's keys and values get. Nothing else is."""
    import endia_amd as nd
    for i in {0, Q - 1}:
        q, k, v, go = _two_heads(Q, K)
        want = attention_reference(q, k, v, go)
        q[0, i, 0, 3] = np.nan
        got = attend(nd, q, k, v, go)
        for n in ("o", "dq"):
            assert np.isnan(got[n][0, i, 0]).all(), n
            got[n][0, i, 0] = want[n][0][0, i, 0]
            within(got[n], want[n], n)
        for n in ("dk", "dv"):
            assert np.isnan(got[n][0, :, 0]).all(), n
            within(got[n][:, :, 1], [a[:, :, 1] for a in want[n]], n)


@pytest.mark.gpu
@pytest.mark.parametrize("K", KEYS)
@pytest.mark.parametrize("Q", QUERIES)
def test_attention_nan_in_a_key_or_value_reaches_every_row(Q, K):
    """A NaN in a key: every query of its head. In one element of a value: that element of every query of its head."""
    import endia_amd as nd
    for j in (0, K // 2, K - 1):
        q, k, v, _ = _two_heads(Q, K)
        want = attention_reference(q, k, v)["o"]
        bad = k.copy()
        bad[0, j, 0, 3] = np.nan
        o = attend(nd, q, bad, v)["o"]
        assert np.isnan(o[:, :, 0]).all(), j
        within(o[:, :, 1], [a[:, :, 1] for a in want], "o")
        for value in (np.nan, np.inf):
            bad = v.copy()
            bad[0, j, 0, 5] = value
            o = attend(nd, q, k, bad)["o"]
            assert not np.isfinite(o[:, :, 0, 5]).any(), j
            o[:, :, 0, 5] = want[0][:, :, 0, 5]
            within(o, want, "o")
