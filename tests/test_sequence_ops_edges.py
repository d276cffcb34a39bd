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


# ---- attention: keys and queries that the causal mask leaves without a partner -----------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("buckets", [None, 16])
@pytest.mark.parametrize("Q", [1, 4, 17, 130])
def test_attention_keys_behind_the_last_query(Q, buckets):
    """A chunk of queries in a cache with room: what the slots behind the last query hold (NaN, infinities, values that would take a
    common scale) is never looked at, and their gradients are zeros."""
    import endia_amd as nd
    rng = np.random.default_rng(0)
    for offset, K in ((40, Q + 90), (0, Q + 5), (300, Q + 333)):
        q, k, v, go = (rng.standard_normal((2, n, 2, 64)).astype(np.float32) for n in (Q, K, K, Q))
        table = rng.standard_normal((buckets, 2)).astype(np.float32) if buckets else None
        kw = dict(table=table, causal=True, offset=offset, max_distance=32)
        want = attention_reference(q, k, v, go, **kw)
        seen = Q + offset
        for ends in ((np.nan, np.inf), (1e30, -1e30), (-np.inf, np.nan)):
            k[:, seen:], v[:, seen:] = ends
            got = attend(nd, q, k, v, go, **kw)
            for n in want:
                within(got[n], want[n], "%s at offset %d" % (n, offset))
            assert not got["dk"][:, seen:].any() and not got["dv"][:, seen:].any()


@pytest.mark.gpu
def test_attention_causal_before_the_first_key():
    """All queries stand before the first key."""
    import endia_amd as nd
    rng = np.random.default_rng(0)
    for Q, offset in ((3, -3), (3, -1000), (70, -70), (70, -100000)):
        q, k, v, go = (rng.standard_normal((1, n, 2, 32)).astype(np.float32) for n in (Q, 40, 40, Q))
        k[:], v[:] = np.nan, np.inf
        got = attend(nd, q, k, v, go, causal=True, offset=offset)
        assert not any(got[n].any() for n in NAMES), (Q, offset)


@pytest.mark.gpu
@pytest.mark.parametrize("Q, K", [(20, 40), (100, 90), (200, 40)])
def test_attention_queries_without_a_key_pass_nothing_on(Q, K):
    """What stands in a query, or comes as the cotangent of one, that sees no key reaches no gradient."""
    import endia_amd as nd
    rng = np.random.default_rng(0)
    for none in (1, Q // 2 + 3):
        q, k, v, go = (rng.standard_normal((1, n, 2, 64)).astype(np.float32) for n in (Q, K, K, Q))
        table = rng.standard_normal((16, 2)).astype(np.float32)
        kw = dict(table=table, causal=True, offset=-none, max_distance=32)
        want = attention_reference(q, k, v, go, **kw)
        for values in ((np.nan, np.nan), (np.inf, 1e30), (1e30, -np.inf)):
            q[:, :none], go[:, :none] = values
            got = attend(nd, q, k, v, go, **kw)
            for n in want:
                within(got[n], want[n], n)
            assert not got["dq"][:, :none].any()


# ---- attention: a value that some queries of a tile see and others do not ------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("buckets", [None, 16])
@pytest.mark.parametrize("T", [12, 40, 300])
def test_attention_causal_nan_stays_behind_its_place(T, buckets):
    """A NaN at place j reaches the queries from j on and the gradients of what they see; the queries before keep their values."""
    import endia_amd as nd
    rng = np.random.default_rng(0)
    for j in {0, 5, T // 2, T - 1}:
        q, k, v, go = (rng.standard_normal((1, T, 2, 64)).astype(np.float32) for _ in range(4))
        table = rng.standard_normal((buckets, 2)).astype(np.float32) if buckets else None
        kw = dict(table=table, causal=True, max_distance=32)
        want = attention_reference(q, k, v, go, **kw)

        def check(got, name, nan, rest):
            assert np.isnan(got[nan]).all(), (name, j)
            within(got[rest], [a[rest] for a in want[name]], "%s, NaN at %d" % (name, j))

        late, early, head1 = np.s_[:, j:, 0], np.s_[:, :j, 0], np.s_[:, :, 1]
        bad = v.copy()
        bad[0, j, 0, 5] = np.nan
        o = attend(nd, q, k, bad, **kw)["o"]
        check(o, "o", np.s_[:, j:, 0, 5], early)
        within(np.delete(o, 5, 3), [np.delete(a, 5, 3) for a in want["o"]], "the other elements")
        bad = k.copy()
        bad[0, j, 0, 5] = np.nan
        got = attend(nd, q, bad, v, go, **kw)
        for n in ("o", "dq"):
            check(got[n], n, late, early)
            within(got[n][head1], [a[head1] for a in want[n]], n)
        bad = q.copy()
        bad[0, j, 0, 5] = np.nan
        got = attend(nd, bad, k, v, go, **kw)
        for n in ("dk", "dv"):
            check(got[n], n, np.s_[:, :j + 1, 0], np.s_[:, j + 1:, 0])
        bad = go.copy()
        bad[0, j, 0, 5] = np.nan
        got = attend(nd, q, k, v, bad, **kw)
        check(got["dk"], "dk", np.s_[:, :j + 1, 0], np.s_[:, j + 1:, 0])
        check(got["dv"], "dv", np.s_[:, :j + 1, 0, 5], np.s_[:, j + 1:, 0])
        within(np.delete(got["dv"], 5, 3), [np.delete(a, 5, 3) for a in want["dv"]], "the other elements")


# ---- attention: memory ----------------------------------------------------------------------------------------
@pytest.mark.gpu
def test_attention_holds_the_cotangent_through_the_call(monkeypatch):
    """A cotangent that is spread out (a mean's) is copied for the call; the copy lives until the call has been made."""
    import endia_amd as nd
    from endia_amd import _array, _lib
    call, held = _lib.call, []

    def watch(name, *args):
        if name == "endia_hip_attention_bwd":
            held.append(not any(args[8] in free for free in _array._FREE.values()))
        return call(name, *args)

    monkeypatch.setattr(_lib, "call", watch)
    x = nd.ones([2, 20, 2, 32], requires_grad=True)
    nd.mean(nd.attention(x, x, x)).backward()
    assert held == [True]


# ---- linear_cross_entropy: scales at the ends of the range ------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("tied", [False, True])
@pytest.mark.parametrize("N", [513, 768, 8392, 9000])
def test_linear_cross_entropy_left_out_tail(N, tied):
    """Padding at the end of the batch: the last rows are left out, whole tiles of 256 among them, alone in their part of the walk or
    behind other tiles; small cotangents, small rows."""
    import endia_amd as nd
    rng = np.random.default_rng(0)
    for left in (N % 256 or 256, 300):
        for size in (1.0, 1e-3):
            x, w = (size * rng.standard_normal((N, 40))).astype(np.float32), (rng.standard_normal((40, 333)) / 6).astype(np.float32)
            t = rng.integers(0, 333, N).astype(np.float32)
            t[N - left:] = -1
            for g in (1.0, 1e-4, 1e-8):
                want, got = loss_reference(x, w, t, g), loss_of(nd, x, w, t, tied, g=g)
                for n in got:
                    within(got[n], want[n], "%s with %d of %d left out, size %g, cotangent %g" % (n, left, N, size, g))


@pytest.mark.gpu
@pytest.mark.parametrize("tied", [False, True])
def test_linear_cross_entropy_long_sums_before_left_out_rows(tied):
    """A million rows that are all wrong about one class, in a column of x that never changes its sign: sums of 2^16 such rows, and
    then 256 rows that are left out."""
    import endia_amd as nd
    N = (1 << 20) + 256
    x = np.full((N, 2), 1.99, np.float32)
    x[:, 1] = np.random.default_rng(0).standard_normal(N)
    w = np.array([[-8, 8, 0], [0.1, 0.2, 0.3]], np.float32)
    t = np.zeros(N, np.float32)
    t[1 << 20:] = -1
    want, got = loss_reference(x, w, t), loss_of(nd, x, w, t, tied)
    for n in got:
        within(got[n], want[n], n)


@pytest.mark.gpu
@pytest.mark.parametrize("tied", [False, True])
@pytest.mark.parametrize("N", [9, 90, 600])
def test_linear_cross_entropy_of_a_tiny_cotangent(N, tied):
    import endia_amd as nd
    rng = np.random.default_rng(0)
    x, w = rng.standard_normal((N, 40)).astype(np.float32), (rng.standard_normal((40, 333)) / 6).astype(np.float32)
    t = rng.integers(0, 333, N).astype(np.float32)
    for g in (1e-20, -1e-30, 1e20):
        want, got = loss_reference(x, w, t, g), loss_of(nd, x, w, t, tied, g=g)
        for n in got:
            within(got[n], want[n], "%s with a cotangent of %g" % (n, g))


@pytest.mark.gpu
@pytest.mark.parametrize("tied", [False, True])
@pytest.mark.parametrize("N", [9, 90, 600])
def test_linear_cross_entropy_left_out_rows_get_no_gradient_from_a_broken_weight(N, tied):
    """An infinity or NaN in the weight: the rows that count become NaN, those that are left out keep their zeros."""
    import endia_amd as nd
    rng = np.random.default_rng(0)
    x, w = rng.standard_normal((N, 40)).astype(np.float32), rng.standard_normal((40, 333)).astype(np.float32)
    for value in (np.nan, np.inf):
        bad = w.copy()
        bad[3, 7] = value
        for left in (np.arange(N) % 3 == 1, np.ones(N, bool)):
            t = np.where(left, -1, 5).astype(np.float32)
            got = loss_of(nd, x, bad, t, tied)
            assert not got["dx"][left].any() and np.isnan(got["dx"][~left]).any(axis=1).all(), value
            assert got["loss"][0] == 0 if left.all() else np.isnan(got["loss"][0])
            assert np.isnan(got["dw"]).any() != left.all()
