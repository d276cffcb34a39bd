"""linear_cross_entropy, attention and relative_attention against their definitions in float64.

Tolerances are bounds on rounding, evaluated in float64 beside the reference. u = 2^-24 is half a step of fp32. A product of
length n that is accumulated in fp32 is off by at most (n + 16) u times the sum of the absolute products (16: a factor held as
two fp16 halves is off by 2^-22 = 4 u, twice, the product of the two lower halves, left out, by 4 u, and the rest are single
roundings of scales and stores). exp and log are good to 2 u here; exp turns an absolute error of its argument into a relative
one. First-order bounds; factor 2 over the whole covers the second order.
"""
import ctypes

import numpy as np
import pytest

from endia_amd import _lib as L

U = 2.0 ** -24


# ---- definitions in float64 -----------------------------------------------------------------------------------
def bucket_of(rel, buckets, max_distance, both_sides):
    """In whole numbers: the logarithm's steps by comparing integer powers."""
    base, n = 0, -rel
    if both_sides:
        buckets //= 2
        base = buckets if rel > 0 else 0
        n = abs(n)
    n = max(n, 0)
    e = buckets // 2
    if n < e:
        return base + n
    steps, far = buckets - e, 0
    while far + 1 < steps and n ** steps * e ** (far + 1) >= max_distance ** (far + 1) * e ** steps:
        far += 1
    return base + e + far


def attention_reference(q, k, v, go=None, table=None, lengths=None, causal=False, scale=None, offset=0, max_distance=128):
    """{name: (value, bound)} of the output and, with go, of the gradients."""
    q, k, v = (a.astype(np.float64) for a in (q, k, v))
    B, Q, H, D = q.shape
    K, Hk = k.shape[1:3]
    G = H // Hk
    scale = D ** -0.5 if scale is None else scale
    out = {"o": (np.zeros_like(q), np.zeros_like(q))}
    if go is not None:
        go = go.astype(np.float64)
        for n, a in (("dq", q), ("dk", k), ("dv", v)):
            out[n] = (np.zeros_like(a), np.zeros_like(a))
        if table is not None:
            out["dtable"] = (np.zeros(table.shape), np.zeros(table.shape))
    rel = np.arange(K)[None, :] - (np.arange(Q)[:, None] + offset)
    if table is not None:
        lut = {r: bucket_of(int(r), table.shape[0], max_distance, not causal) for r in np.unique(rel)}
        bucket = np.vectorize(lut.get)(rel)
    for b in range(B):
        n = K if lengths is None else int(min(max(lengths[b], 0), K))
        left = np.broadcast_to(np.arange(K)[None, :] < n, (Q, K))
        if causal:
            left = left & (rel <= 0)
        for h in range(H):
            ks, vs = np.where(np.arange(K)[:, None] < n, k[b, :, h // G], 0), np.where(np.arange(K)[:, None] < n, v[b, :, h // G], 0)
            qs = q[b, :, h]
            s = qs @ ks.T * scale
            off_s = (D + 16) * U * abs(scale) * (np.abs(qs) @ np.abs(ks).T)
            if table is not None:
                s = s + table.astype(np.float64)[bucket, h]
                off_s = off_s + 2 * U * np.abs(s) + 2 * U * np.abs(table[bucket, h])
            s = np.where(left, s, -np.inf)
            top = s.max(axis=1, keepdims=True)
            top = np.where(np.isfinite(top), top, 0)
            p = np.exp(s - top)
            total = p.sum(axis=1, keepdims=True)
            p = p / np.where(total > 0, total, 1)
            # relative error of p: twice the largest error of the row's scores (its own and the normaliser's), the sum, exp
            # of an argument that is itself rounded (relative to its size) and the division
            arg = np.where(left, np.abs(s - top) + np.abs(top), 0).max(axis=1, keepdims=True)
            rel_p = 2 * np.where(left, off_s, 0).max(axis=1, keepdims=True) + (K + 16 + 4 * arg) * U
            o = p @ vs
            o_abs = p @ np.abs(vs)
            out["o"][0][b, :, h], out["o"][1][b, :, h] = o, 2 * (rel_p + (K + 16) * U) * o_abs
            if go is None:
                continue
            gs = go[b, :, h]
            dp, dp_abs = gs @ vs.T, np.abs(gs) @ np.abs(vs).T
            delta, delta_abs = (gs * o).sum(1, keepdims=True), (np.abs(gs) * o_abs).sum(1, keepdims=True)
            ds, ds_abs = p * (dp - delta), p * (dp_abs + delta_abs)
            off_ds = (2 * rel_p + (K + 2 * D + 48) * U) * ds_abs
            c = h // G
            for name, value, bound, at in (
                    ("dv", p.T @ gs, (p * (rel_p + (Q * G + 16) * U)).T @ np.abs(gs), np.s_[b, :, c]),
                    ("dq", ds @ ks * scale, (off_ds + (K + 16) * U * ds_abs) @ np.abs(ks) * abs(scale), np.s_[b, :, h]),
                    ("dk", ds.T @ qs * scale, (off_ds + (Q * G + 16) * U * ds_abs).T @ np.abs(qs) * abs(scale), np.s_[b, :, c])):
                out[name][0][at] += value
                out[name][1][at] += 2 * bound
            if table is not None:
                np.add.at(out["dtable"][0][:, h], bucket.ravel(), ds.ravel())
                np.add.at(out["dtable"][1][:, h], bucket.ravel(), 2 * (off_ds + (Q + K + B + 16) * U * ds_abs).ravel())
    return out


def loss_reference(x, w, t, g=1.0):
    x, w, t = x.astype(np.float64), w.astype(np.float64), t.astype(np.float64)
    N, D = x.shape
    V = w.shape[1]
    kept = ~(t < 0)
    xs = x[kept]
    n = max(int(kept.sum()), 1)
    z = xs @ w
    off_z = (D + 16) * U * (np.abs(xs) @ np.abs(w))
    top = z.max(axis=1, keepdims=True) if len(xs) else z[:, :1]
    e = np.exp(z - top)
    lse = top + np.log(e.sum(axis=1, keepdims=True))
    at = (np.arange(len(xs)), t[kept].astype(int))
    arg = np.abs(z - top).max(axis=1, keepdims=True) + np.abs(top) if len(xs) else z[:, :1]
    off_row = off_z.max(axis=1, keepdims=True)
    each, off_each = lse[:, 0] - z[at], 2 * off_row[:, 0] + (V + 16) * U + 8 * U * arg[:, 0]
    p = np.exp(z - lse)
    dz = p.copy()
    dz[at] -= 1
    rel_p = 2 * off_row + (V + 16 + 8 * arg) * U
    hot = np.zeros_like(p)
    hot[at] = 1
    off_dz = rel_p * p + 2 * U * hot
    dx, off_dx = np.zeros_like(x), np.zeros_like(x)
    dx[kept] = dz @ w.T * (g / n)
    off_dx[kept] = 2 * (off_dz + (V + 24) * U * np.abs(dz)) @ np.abs(w).T * (abs(g) / n)
    return {"loss": (np.array([each.sum() / n]), np.array([2 * off_each.sum() / n + 4 * U * abs(each.sum()) / n])),
            "dx": (dx, off_dx),
            "dw": (xs.T @ dz * (g / n), 2 * np.abs(xs).T @ (off_dz + (N + 24) * U * np.abs(dz)) * (abs(g) / n))}


def within(got, want, name=""):
    value, bound = want
    got = np.asarray(got, np.float64).reshape(value.shape)
    off = np.abs(got - value)
    floor = 1e-37  # values that fp32 cannot hold in full precision
    bad = ~(off <= bound + floor)
    assert not bad.any(), "%s: %d of %d values off by more than their bound; worst %.3g of it, at %s" % (
        name, bad.sum(), bad.size, np.nanmax(np.where(bad, off / (bound + floor), 0)), np.argwhere(bad)[0])


# ---- refusals: checked before any device is touched -----------------------------------------------------------
P = 1 << 20  # stands for a device address; a refused call reads nothing


def _desc(**change):
    d = L.AttentionDesc()
    d.B, d.Q, d.K, d.H, d.Hk, d.D = 2, 3, 5, 4, 2, 8
    d.q_strides[:], d.k_strides[:], d.v_strides[:] = (96, 32, 8), (80, 16, 8), (80, 16, 8)
    d.scale, d.buckets, d.max_distance, d.both_sides = 1.0, 8, 16, 1
    for n, v in change.items():
        setattr(d, n, v)
    return d


@pytest.mark.parametrize("change, table, code", [
    ({"B": 0}, None, L.ERR_INVALID), ({"Q": 0}, None, L.ERR_INVALID), ({"K": -1}, None, L.ERR_INVALID), ({"D": 0}, None, L.ERR_INVALID),
    ({"Hk": 3}, None, L.ERR_INVALID), ({"Hk": 0}, None, L.ERR_INVALID), ({"D": 129}, None, L.ERR_UNSUPPORTED),
    ({"K": 1 << 25}, None, L.ERR_INVALID), ({"query_offset": 1 << 40}, None, L.ERR_INVALID),
    ({"scale": float("nan")}, None, L.ERR_INVALID), ({"scale": float("inf")}, None, L.ERR_INVALID),
    ({"buckets": 7}, P, L.ERR_INVALID), ({"buckets": 2}, P, L.ERR_INVALID), ({"buckets": 0}, P, L.ERR_INVALID),
    ({"max_distance": 2}, P, L.ERR_INVALID), ({"max_distance": 4096}, P, L.ERR_UNSUPPORTED), ({"buckets": 1024, "max_distance": 1024}, P, L.ERR_UNSUPPORTED),
    ({"B": 1 << 40}, None, L.ERR_UNSUPPORTED),
])
def test_attention_refuses(change, table, code):
    d = _desc(**change)
    assert L.lib().endia_hip_attention_fwd(ctypes.byref(d), P, P, P, None, table, P, P) == code
    assert L.lib().endia_hip_attention_bwd(ctypes.byref(d), P, P, P, None, table, P, P, P, P, P, P, None) == code
    assert b"endia_hip_attention" in L.lib().endia_hip_last_error()


def test_attention_refuses_null_pointers():
    d = ctypes.byref(_desc())
    fwd, bwd = L.lib().endia_hip_attention_fwd, L.lib().endia_hip_attention_bwd
    for args in ((None, P, P, P, None, None, P, P), (d, None, P, P, None, None, P, P), (d, P, None, P, None, None, P, P),
                 (d, P, P, None, None, None, P, P), (d, P, P, P, None, None, None, P)):
        assert fwd(*args) == L.ERR_INVALID
    for args in ((d, P, P, P, None, None, None, P, P, P, P, P, None), (d, P, P, P, None, None, P, None, P, P, P, P, None),
                 (d, P, P, P, None, None, P, P, None, P, P, P, None), (d, P, P, P, None, None, P, P, P, None, None, None, None),
                 (d, P, P, P, None, None, P, P, P, P, P, P, P)):
        assert bwd(*args) == L.ERR_INVALID


def test_linear_cross_entropy_refuses():
    fwd, bwd = L.lib().endia_hip_linear_cross_entropy_fwd, L.lib().endia_hip_linear_cross_entropy_bwd
    good = [4, 8, 16, P, 8, 0, P, 16, P, P, P]
    for i, v in ((0, 0), (1, -1), (2, 0), (3, None), (4, 7), (5, 2), (6, None), (7, 15), (8, None), (9, None), (10, None), (0, 1 << 24),
                 (2, (1 << 24) + 1)):
        args = list(good)
        args[i] = v
        if i == 2 and v:
            args[7] = v
        assert fwd(*args) == L.ERR_INVALID, (i, v)
    assert fwd(4, 8, 16, P, 8, 1, P, 7, P, P, P) == L.ERR_INVALID
    back = [4, 8, 16, P, 8, 0, P, 16, P, P, P, P, P]
    for i in (3, 6, 8, 9, 10):
        args = list(back)
        args[i] = None
        assert bwd(*args) == L.ERR_INVALID, i
    assert bwd(*(back[:11] + [None, None])) == L.ERR_INVALID


def test_refused_without_a_device():
    import torch
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    d = _desc()
    assert L.lib().endia_hip_attention_fwd(ctypes.byref(d), P, P, P, None, None, P, P) == L.ERR_NOT_INIT
    assert L.lib().endia_hip_linear_cross_entropy_fwd(4, 8, 16, P, 8, 0, P, 16, P, P, P) == L.ERR_NOT_INIT


def test_reference_against_differences():
    """The float64 gradients used below against central differences of the float64 values (h = 1e-5: the difference is off by
    h^2 times a third derivative of order one, and by 1e-16 / h, both far below 1e-6)."""
    rng = np.random.default_rng(0)
    q, k, v, go = rng.standard_normal((1, 3, 2, 4)), rng.standard_normal((1, 5, 1, 4)), rng.standard_normal((1, 5, 1, 4)), rng.standard_normal((1, 3, 2, 4))
    table = rng.standard_normal((4, 2))
    arrays = {"dq": q, "dk": k, "dv": v, "dtable": table}
    f = lambda: (attention_reference(q, k, v, table=table, offset=1, max_distance=3)["o"][0] * go).sum()
    want = attention_reference(q, k, v, go, table=table, offset=1, max_distance=3)
    for name, a in arrays.items():
        for i in np.ndindex(a.shape):
            old = a[i]
            a[i] = old + 1e-5
            up = f()
            a[i] = old - 1e-5
            down = f()
            a[i] = old
            assert abs((up - down) / 2e-5 - want[name][0][i]) < 1e-6
    x, w, t = rng.standard_normal((4, 3)), rng.standard_normal((3, 6)), np.array([0, 5, -1, 2.0])
    want = loss_reference(x, w, t)
    for name, a in (("dx", x), ("dw", w)):
        for i in np.ndindex(a.shape):
            old = a[i]
            a[i] = old + 1e-5
            up = loss_reference(x, w, t)["loss"][0][0]
            a[i] = old - 1e-5
            down = loss_reference(x, w, t)["loss"][0][0]
            a[i] = old
            assert abs((up - down) / 2e-5 - want[name][0][i]) < 1e-6


# ---- attention on the device ----------------------------------------------------------------------------------
def attend(nd, q, k, v, go=None, table=None, lengths=None, offset=0, max_distance=128, **kw):
    arrays = [nd.array(np.asarray(a, np.float32), requires_grad=go is not None) for a in (q, k, v)]
    lens = nd.array(np.asarray(lengths, np.float32)) if lengths is not None else None
    if table is None:
        o = nd.attention(*arrays, key_lengths=lens, query_offset=offset, **kw)
        names = ("dq", "dk", "dv")
    else:
        arrays.append(nd.array(np.asarray(table, np.float32), requires_grad=go is not None))
        o = nd.relative_attention(*arrays, key_lengths=lens, query_offset=offset, max_distance=max_distance, **kw)
        names = ("dq", "dk", "dv", "dtable")
    out = {"o": o.to_numpy()}
    if go is not None:
        grads = nd.grad(outs=[o], inputs=arrays, grad_outs=[nd.array(np.asarray(go, np.float32))])
        out.update((n, g.to_numpy()) for n, g in zip(names, grads))
    return out


def check_attention(B, Q, K, H, Hk, D, seed=0, buckets=None, step=True, size=1.0, poison=False, **kw):
    import endia_amd as nd
    rng = np.random.default_rng(seed)
    q, k, v, go = ((size * rng.standard_normal(s)).astype(np.float32) for s in ((B, Q, H, D), (B, K, Hk, D), (B, K, Hk, D), (B, Q, H, D)))
    table = rng.standard_normal((buckets, H)).astype(np.float32) if buckets else None
    want = attention_reference(q, k, v, go if step else None, table=table, **kw)
    if poison:  # what stands behind the lengths is never looked at
        for b in range(B):
            n = int(kw["lengths"][b])
            k[b, n:], v[b, n:] = np.nan, np.inf
    got = attend(nd, q, k, v, go if step else None, table=table, **kw)
    assert set(got) == set(want)
    for name in want:
        within(got[name], want[name], "%s of %s" % (name, (B, Q, K, H, Hk, D)))
    return got


SHAPES = [
    (1, 1, 1, 1, 1, 1), (1, 1, 1, 1, 1, 64), (2, 1, 77, 3, 3, 64), (1, 1, 1000, 8, 2, 128), (3, 2, 5, 2, 1, 3), (2, 7, 33, 4, 4, 40),
    (1, 31, 32, 2, 2, 32), (1, 33, 65, 2, 1, 64), (2, 64, 64, 2, 2, 64), (1, 127, 129, 2, 1, 80), (1, 128, 200, 4, 2, 96),
    (1, 130, 257, 3, 1, 128), (2, 300, 17, 2, 2, 127), (1, 513, 300, 1, 1, 64), (1, 40, 1500, 2, 2, 64), (5, 16, 1, 2, 2, 64),
    (1, 5, 700, 12, 3, 65),
]


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES)
def test_attention_values_and_gradients(shape):
    check_attention(*shape)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES[::3])
def test_attention_without_gradient(shape):
    check_attention(*shape, step=False)


@pytest.mark.gpu
@pytest.mark.parametrize("Q, lengths", [(1, [0, 40, 13, 1]), (1, [41, 50, 0, 0]), (70, [0, 40, 13, 1]), (70, [50, 33, 32, 31]), (70, [0, 0, 0, 0])])
def test_attention_lengths(Q, lengths):
    """Lengths of zero (rows without a key), of one, at the borders of a tile; NaN and infinities behind them."""
    check_attention(4, Q, 50, 4, 2, 64, lengths=lengths, poison=True)
    check_attention(4, Q, 50, 2, 2, 64, lengths=lengths, poison=True, buckets=16, max_distance=32)


@pytest.mark.gpu
def test_attention_lengths_are_clamped():
    import endia_amd as nd
    rng = np.random.default_rng(1)
    q, k, v = (rng.standard_normal((3, 9, 2, 32)).astype(np.float32) for _ in range(3))
    a = attend(nd, q, k, v, lengths=[-5, 100, np.nan])
    b = attend(nd, q, k, v, lengths=[0, 9, 0])
    assert np.array_equal(a["o"], b["o"]) and not b["o"][[0, 2]].any()


@pytest.mark.gpu
@pytest.mark.parametrize("Q, K, offset", [(1, 1, 0), (1, 60, 59), (1, 60, 10), (1, 60, -1), (50, 50, 0), (200, 200, 0), (65, 300, 235), (65, 300, 100),
                                          (100, 40, 0), (100, 40, -30), (40, 100, -200), (33, 70, 1000)])
def test_attention_causal(Q, K, offset):
    """Aligned at the start, at the end and in between; offsets that leave the first rows, or all, without a key."""
    check_attention(2, Q, K, 2, 1, 64, causal=True, offset=offset, lengths=[K, max(K - 7, 0)])


@pytest.mark.gpu
@pytest.mark.parametrize("Q, K, offset, buckets, max_distance, causal", [
    (1, 1, 0, 4, 2, False), (1, 300, 299, 32, 128, True), (1, 300, 100, 32, 128, False), (50, 50, 0, 32, 128, False), (200, 200, 0, 32, 128, True),
    (300, 290, 0, 32, 128, False), (300, 300, 0, 8, 9, False), (130, 700, 500, 16, 20, False), (90, 130, -20, 32, 1000, False), (300, 130, 5, 2, 3, True),
    (70, 2500, 0, 64, 2048, False), (260, 260, 0, 256, 2048, False), (64, 64, 0, 64, 2048, True),
])
def test_relative_attention(Q, K, offset, buckets, max_distance, causal):
    check_attention(2, Q, K, 2, 1 if Q % 2 else 2, 64, offset=offset, buckets=buckets, max_distance=max_distance, causal=causal)


@pytest.mark.gpu
def test_relative_attention_buckets_are_exact():
    """One query and one-hot values: the output is the softmax of the table's rows by bucket, so a wrong bucket shows. Every
    difference up to the largest distance, both sides."""
    import endia_amd as nd
    for buckets, far, causal in ((32, 128, False), (32, 128, True), (16, 32, False), (64, 2048, True), (32, 1000, False)):
        K = 2 * far + 9
        place = far + 4
        table = (np.arange(buckets, dtype=np.float32) / buckets)[:, None]
        q, k = np.zeros((1, 1, 1, 1), np.float32), np.zeros((1, K, 1, 1), np.float32)
        s = np.array([table[bucket_of(j - place, buckets, far, not causal), 0] for j in range(K)], np.float64)
        if causal:
            s[place + 1:] = -np.inf
        p = np.exp(s) / np.exp(s).sum()
        for first in range(0, K, 128):  # 128 one-hot columns at a time
            cols = min(128, K - first)
            v = np.zeros((1, K, 1, cols), np.float32)
            v[0, first + np.arange(cols), 0, np.arange(cols)] = 1
            q, k = np.zeros((1, 1, 1, cols), np.float32), np.zeros((1, K, 1, cols), np.float32)
            o = attend(nd, q, k, v, table=table, offset=place, max_distance=far, causal=causal)["o"].ravel()
            # neighbouring buckets differ by 1 / buckets >= 1.5 percent; rounding by (K + 20) u < 3e-4
            assert np.all(np.abs(o - p[first:first + cols]) <= (K + 20) * U * p[first:first + cols] + 1e-12), (buckets, far, causal, first)


@pytest.mark.gpu
@pytest.mark.parametrize("size", [1e-6, 30.0, 300.0])
def test_attention_of_small_and_large_values(size):
    check_attention(1, 70, 90, 2, 2, 64, size=size, scale=1.0 / min(size, 30.0) ** 2 if size < 1 else 0.125, step=size < 100)
    check_attention(1, 1, 90, 2, 2, 64, size=size, scale=1.0 / min(size, 30.0) ** 2 if size < 1 else 0.125, step=False)


@pytest.mark.gpu
def test_attention_rows_of_very_different_size():
    """One key, one value row and one query 2^20 times the others: the others keep their precision."""
    import endia_amd as nd
    rng = np.random.default_rng(3)
    q, k, v, go = (rng.standard_normal((1, n, 1, 64)).astype(np.float32) for n in (100, 150, 150, 100))
    q[0, 50] *= 2.0 ** 20
    k[0, 149] *= 2.0 ** -20
    v[0, 20] *= 2.0 ** 20
    go[0, 7] *= 2.0 ** -20
    want = attention_reference(q, k, v, go)
    got = attend(nd, q, k, v, go)
    for name in want:
        within(got[name], want[name], name)


@pytest.mark.gpu
def test_attention_reads_views_in_place():
    """Slices of one fused projection, heads before positions, an offset that is not a multiple of 16 bytes, a broadcast batch."""
    import endia_amd as nd
    rng = np.random.default_rng(4)
    B, T, H, D = 2, 45, 3, 40
    fused = rng.standard_normal((B, T, H, 3 * D + 1)).astype(np.float32)
    go = rng.standard_normal((B, T, H, D)).astype(np.float32)
    f = nd.array(fused, requires_grad=True)
    cut = [f[:, :, :, 1 + i * D:1 + (i + 1) * D] for i in range(3)]
    o = nd.attention(*cut)
    want = attention_reference(*(fused[..., 1 + i * D:1 + (i + 1) * D] for i in range(3)), go)
    within(o.to_numpy(), want["o"], "o")
    g = nd.grad(outs=[o], inputs=[f], grad_outs=[nd.array(go)])[0].to_numpy()
    assert not g[..., 0].any()
    for i, n in enumerate(("dq", "dk", "dv")):
        within(g[..., 1 + i * D:1 + (i + 1) * D], want[n], n)
    heads_first = rng.standard_normal((B, H, T, D)).astype(np.float32)
    q = nd.array(heads_first, requires_grad=True)
    kv = rng.standard_normal((1, 70, H, D)).astype(np.float32)
    k = nd.array(kv, requires_grad=True)
    o = nd.attention(nd.permute(q, [0, 2, 1, 3]), nd.functional.expand(k, [B, 70, H, D]), nd.functional.expand(k, [B, 70, H, D]))
    qs, ks = heads_first.transpose(0, 2, 1, 3), np.broadcast_to(kv, (B, 70, H, D))
    want = attention_reference(qs, ks, ks, go)
    within(o.to_numpy(), want["o"], "o")
    gq, gk = nd.grad(outs=[o], inputs=[q, k], grad_outs=[nd.array(go)])
    within(gq.to_numpy().transpose(0, 2, 1, 3), want["dq"], "dq")
    both = [(want["dk"][i] + want["dv"][i]).sum(0, keepdims=True) for i in (0, 1)]
    both[1] = both[1] + 8 * U * sum(np.abs(want[n][0]).sum(0, keepdims=True) for n in ("dk", "dv"))
    within(gk.to_numpy(), tuple(both), "dk + dv over the batch")


@pytest.mark.gpu
def test_attention_one_token_over_a_long_cache():
    """A cache of over 2^31 bytes of k; the last keys carry the answer."""
    import endia_amd as nd
    B, K, H, D = 1, 70000, 64, 128
    k = nd.zeros([B, K, H, D])
    assert 4 * k.size() > 2 ** 31
    v = nd.zeros([B, K, H, D])
    rng = np.random.default_rng(5)
    last = rng.standard_normal((B, 3, H, D)).astype(np.float32)
    k[:, K - 3:] = nd.array(last)
    v[:, K - 3:] = nd.array(last + 1)
    q = (4 * last[:, 1:2]).astype(np.float32)
    o = nd.attention(nd.array(q), k, v, key_lengths=nd.array(np.array([K - 1], np.float32))).to_numpy()
    s = np.einsum("bqhd,bkhd->bhk", q.astype(np.float64), last.astype(np.float64))[0] * D ** -0.5
    s = np.concatenate([np.full((H, 1), np.log(K - 3.0)), s[:, :2]], axis=1)
    p = np.exp(s - s.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    want = np.einsum("hk,khd->hd", p[:, 1:], last[0, :2].astype(np.float64) + 1)
    # scores of up to 64, products of 128: rel. error of p at most 2 (128 + 16) u 64 * 2 + the sum over 70000 equal terms
    assert np.abs(o[0, 0] - want).max() <= (2 * 144 * 128 + 70016) * U * np.abs(want).max()


@pytest.mark.gpu
def test_attention_repeats_itself_bit_for_bit():
    a = check_attention(2, 200, 300, 4, 2, 64, buckets=32, max_distance=64)
    b = check_attention(2, 200, 300, 4, 2, 64, buckets=32, max_distance=64)
    for n in a:
        assert np.array_equal(a[n], b[n]), n


@pytest.mark.gpu
def test_attention_selected_gradients():
    """Only what requires a gradient gets one."""
    import endia_amd as nd
    rng = np.random.default_rng(6)
    q, k, v = (rng.standard_normal((1, n, 2, 32)).astype(np.float32) for n in (40, 50, 50))
    table = rng.standard_normal((8, 2)).astype(np.float32)
    go = rng.standard_normal((1, 40, 2, 32)).astype(np.float32)
    want = attention_reference(q, k, v, go, table=table, max_distance=16)
    for i, n in enumerate(("dq", "dk", "dv", "dtable")):
        arrays = [nd.array(a, requires_grad=j == i) for j, a in enumerate((q, k, v, table))]
        o = nd.relative_attention(*arrays, max_distance=16)
        within(nd.grad(outs=[o], inputs=[arrays[i]], grad_outs=[nd.array(go)])[0].to_numpy(), want[n], n)


@pytest.mark.gpu
def test_attention_python_refusals():
    import endia_amd as nd
    q, k = nd.ones([2, 3, 4, 8]), nd.ones([2, 5, 2, 8])
    for bad in ((q, k, nd.ones([2, 6, 2, 8])), (q, nd.ones([1, 5, 2, 8]), nd.ones([1, 5, 2, 8])), (q, nd.ones([2, 5, 3, 8]), nd.ones([2, 5, 3, 8])),
                (q, nd.ones([2, 5, 2, 4]), nd.ones([2, 5, 2, 4])), (nd.ones([3, 4, 8]), k, k)):
        with pytest.raises(ValueError):
            nd.attention(*bad)
    with pytest.raises(ValueError):
        nd.attention(q, k, k, key_lengths=nd.ones([3]))
    with pytest.raises(ValueError):
        nd.relative_attention(q, k, k, nd.ones([8, 3]))
    with pytest.raises(ValueError):
        nd.attention(nd.randn_complex([2, 3, 4, 8]), k, k)
    with pytest.raises(L.EndiaHipError):
        nd.relative_attention(q, k, k, nd.ones([7, 4]))
    x = nd.ones([2, 3, 4, 8], requires_grad=True)
    o = nd.attention(x, k, k)
    with pytest.raises(NotImplementedError):
        nd.sum(o).backward(create_graph=True)


# ---- linear_cross_entropy on the device -----------------------------------------------------------------------
def loss_of(nd, x, w, t, tied=False, step=True, g=None):
    xa = nd.array(np.asarray(x, np.float32), requires_grad=step)
    wa = nd.array(np.ascontiguousarray(np.asarray(w, np.float32).T if tied else np.asarray(w, np.float32)), requires_grad=step)
    loss = nd.linear_cross_entropy(xa, wa.T() if tied else wa, nd.array(np.asarray(t, np.float32)))
    out = {"loss": loss.to_numpy()}
    if step:
        dx, dw = nd.grad(outs=[loss], inputs=[xa, wa], grad_outs=None if g is None else [nd.array(np.array([g], np.float32))])
        out["dx"], out["dw"] = dx.to_numpy(), dw.to_numpy().T if tied else dw.to_numpy()
    return out


def check_loss(N, D, V, tied=False, size=1.0, left_out=0.2, seed=0, poison=False, g=None, step=True):
    import endia_amd as nd
    rng = np.random.default_rng(seed)
    x, w = (size * rng.standard_normal((N, D))).astype(np.float32), (rng.standard_normal((D, V)) / np.sqrt(D)).astype(np.float32)
    t = rng.integers(0, V, N).astype(np.float32)
    t[rng.random(N) < left_out] = -1
    want = loss_reference(x, w, t, 1.0 if g is None else g)
    if poison:
        x[t < 0] = np.nan
        x[np.nonzero(t < 0)[0][::2]] = np.inf
    got = loss_of(nd, x, w, t, tied, step, g)
    for name in got:
        within(got[name], want[name], "%s of %s" % (name, (N, D, V, tied)))
    return got


LOSSES = [(1, 1, 1), (1, 1, 2), (1, 7, 5), (2, 64, 100), (3, 5, 1000), (16, 96, 777), (17, 33, 4099), (64, 64, 256), (65, 128, 300), (100, 200, 1001),
          (257, 100, 513), (300, 65, 2000), (513, 40, 257), (700, 256, 1030)]


@pytest.mark.gpu
@pytest.mark.parametrize("tied", [False, True])
@pytest.mark.parametrize("shape", LOSSES)
def test_linear_cross_entropy(shape, tied):
    check_loss(*shape, tied=tied)


@pytest.mark.gpu
@pytest.mark.parametrize("N", [5, 70, 600])
def test_linear_cross_entropy_left_out_rows(N):
    """NaN and infinities in the rows that are left out; all rows left out."""
    for tied in (False, True):
        check_loss(N, 48, 333, tied=tied, left_out=0.6, poison=True)
    got = check_loss(N, 48, 333, left_out=1.1, poison=True)
    assert got["loss"][0] == 0 and not got["dx"].any() and not got["dw"].any()


@pytest.mark.gpu
@pytest.mark.parametrize("N", [5, 600])
@pytest.mark.parametrize("size", [1e-6, 30.0, 1000.0])
def test_linear_cross_entropy_of_small_and_large_logits(N, size):
    check_loss(N, 64, 500, size=size)


@pytest.mark.gpu
def test_linear_cross_entropy_in_several_pieces():
    """More rows than one piece of the vocabulary has room for, last piece ragged."""
    check_loss(20000, 8, 8003)
    check_loss(20000, 8, 8003, tied=True, step=False)


@pytest.mark.gpu
@pytest.mark.parametrize("N", [7, 90, 600])
def test_linear_cross_entropy_cotangent(N):
    check_loss(N, 40, 300, g=-2.5)


@pytest.mark.gpu
@pytest.mark.parametrize("N", [6, 90, 600])
def test_linear_cross_entropy_targets_that_are_no_class(N):
    import endia_amd as nd
    rng = np.random.default_rng(0)
    x, w = rng.standard_normal((N, 32)).astype(np.float32), rng.standard_normal((32, 50)).astype(np.float32)
    for bad in (50.0, np.nan, 1e30, np.inf):
        t = np.full(N, 3, np.float32)
        t[N // 2] = bad
        got = loss_of(nd, x, w, t)
        assert np.isnan(got["loss"][0]) and np.isnan(got["dx"][N // 2]).all() and np.isnan(got["dw"]).all(), bad
        assert np.isfinite(np.delete(got["dx"], N // 2, 0)).all(), bad


@pytest.mark.gpu
@pytest.mark.parametrize("N", [6, 600])
def test_linear_cross_entropy_views(N):
    """A weight that is a slice of columns, or of an embedding's rows; x of three axes; an unaligned start."""
    import endia_amd as nd
    rng = np.random.default_rng(0)
    D, V = 36, 130
    x = rng.standard_normal((2, N // 2, D)).astype(np.float32)
    big = rng.standard_normal((D + 1, V + 21)).astype(np.float32)
    t = rng.integers(0, V, N).astype(np.float32)
    for tied in (False, True):
        xa, wa = nd.array(x, requires_grad=True), nd.array(np.ascontiguousarray(big.T) if tied else big, requires_grad=True)
        w = wa[7:7 + V, 1:].T() if tied else wa[1:, 7:7 + V]
        loss = nd.linear_cross_entropy(xa, w, nd.array(t.reshape(2, N // 2)))
        dx, dw = nd.grad(outs=[loss], inputs=[xa, wa])
        want = loss_reference(x.reshape(N, D), big[1:, 7:7 + V], t)
        within(loss.to_numpy(), want["loss"], "loss")
        within(dx.to_numpy().reshape(N, D), want["dx"], "dx")
        dw = dw.to_numpy().T if tied else dw.to_numpy()
        within(dw[1:, 7:7 + V], want["dw"], "dw")
        dw[1:, 7:7 + V] = 0
        assert not dw.any()


@pytest.mark.gpu
def test_linear_cross_entropy_rows_of_very_different_size():
    """One row of x and one class 2^20 times smaller or larger: the others keep their precision."""
    import endia_amd as nd
    rng = np.random.default_rng(2)
    for N in (9, 600):
        x, w = rng.standard_normal((N, 64)).astype(np.float32), (rng.standard_normal((64, 400)) / 8).astype(np.float32)
        x[3] *= 2.0 ** 10
        w[:, 100] *= 2.0 ** -20
        t = rng.integers(0, 400, N).astype(np.float32)
        want = loss_reference(x, w, t)
        got = loss_of(nd, x, w, t)
        for name in got:
            within(got[name], want[name], name)


@pytest.mark.gpu
def test_linear_cross_entropy_repeats_itself_bit_for_bit():
    for N in (8, 100, 700):
        a, b = check_loss(N, 72, 900), check_loss(N, 72, 900)
        for n in a:
            assert np.array_equal(a[n], b[n]), (N, n)


@pytest.mark.gpu
def test_linear_cross_entropy_python_refusals():
    import endia_amd as nd
    x, w, t = nd.ones([4, 8]), nd.ones([8, 16]), nd.zeros([4])
    for bad in ((x, nd.ones([9, 16]), t), (x, w, nd.zeros([5])), (x, nd.ones([2, 8, 16]), t), (nd.randn_complex([4, 8]), w, t),
                (x, w, nd.zeros([4], requires_grad=True))):
        with pytest.raises(ValueError):
            nd.linear_cross_entropy(*bad)
    x = nd.ones([4, 8], requires_grad=True)
    with pytest.raises(NotImplementedError):
        nd.linear_cross_entropy(x, w, t).backward(create_graph=True)


@pytest.mark.gpu
@pytest.mark.parametrize("shape, tied", [((129, 300, 1001), False), ((200, 513, 700), True), ((511, 260, 1500), False), ((390, 33, 5001), True),
                                         ((33, 1030, 640), False), ((20, 70, 40000), True), ((1100, 300, 3001), False), ((1030, 520, 700), True),
                                         ((2600, 20, 900), False), ((600, 1400, 300), True)])
def test_linear_cross_entropy_between_the_kernels(shape, tied):
    """Either side of the changes of kernel by rows, classes and width: several column tiles, cut reductions, ragged everything."""
    check_loss(*shape, tied=tied)


@pytest.mark.gpu
def test_linear_cross_entropy_selected_gradients():
    import endia_amd as nd
    rng = np.random.default_rng(0)
    for N in (9, 100, 600):
        x, w = rng.standard_normal((N, 40)).astype(np.float32), rng.standard_normal((40, 300)).astype(np.float32)
        t = rng.integers(0, 300, N).astype(np.float32)
        want = loss_reference(x, w, t)
        for i, n in enumerate(("dx", "dw")):
            arrays = [nd.array(a, requires_grad=j == i) for j, a in enumerate((x, w))]
            loss = nd.linear_cross_entropy(*arrays, nd.array(t))
            within(nd.grad(outs=[loss], inputs=[arrays[i]])[0].to_numpy(), want[n], n)


@pytest.mark.gpu
def test_linear_cross_entropy_of_one_vector_and_of_a_shared_array():
    """x without a rows axis; the rows and the classes' weights one and the same array."""
    import endia_amd as nd
    rng = np.random.default_rng(0)
    x, w = rng.standard_normal(24).astype(np.float32), rng.standard_normal((24, 50)).astype(np.float32)
    want = loss_reference(x[None], w, np.array([7.0]))
    xa = nd.array(x, requires_grad=True)
    loss = nd.linear_cross_entropy(xa, nd.array(w), nd.array(np.array([7.0], np.float32)))
    within(loss.to_numpy(), want["loss"])
    within(nd.grad(outs=[loss], inputs=[xa])[0].to_numpy(), want["dx"])
    e = rng.standard_normal((70, 24)).astype(np.float32)
    t = np.arange(70, dtype=np.float32)[::-1].copy()
    want = loss_reference(e, e.T, t)
    ea = nd.array(e, requires_grad=True)
    loss = nd.linear_cross_entropy(ea, ea.T(), nd.array(t))
    got = nd.grad(outs=[loss], inputs=[ea])[0].to_numpy()
    both = want["dx"][0] + want["dw"][0].T, want["dx"][1] + want["dw"][1].T + 4 * U * (np.abs(want["dx"][0]) + np.abs(want["dw"][0].T))
    within(got, both, "dx + dw")


@pytest.mark.gpu
@pytest.mark.parametrize("T", [3, 65])
def test_attention_of_one_array_to_itself(T):
    import endia_amd as nd
    rng = np.random.default_rng(0)
    x, go = (rng.standard_normal((2, T, 3, 32)).astype(np.float32) for _ in range(2))
    xa = nd.array(x, requires_grad=True)
    o = nd.attention(xa, xa, xa, causal=True)
    want = attention_reference(x, x, x, go, causal=True)
    within(o.to_numpy(), want["o"], "o")
    got = nd.grad(outs=[o], inputs=[xa], grad_outs=[nd.array(go)])[0].to_numpy()
    value = sum(want[n][0] for n in ("dq", "dk", "dv"))
    within(got, (value, sum(want[n][1] + 4 * U * np.abs(want[n][0]) for n in ("dq", "dk", "dv"))), "dq + dk + dv")


@pytest.mark.gpu
@pytest.mark.parametrize("T", [4, 50])
def test_attention_under_a_mean_and_behind_a_product(T):
    """The cotangent of a mean is one number spread out; the output also meets an elementwise product first."""
    import endia_amd as nd
    rng = np.random.default_rng(0)
    q, k, v, w = (rng.standard_normal((2, n, 2, 32)).astype(np.float32) for n in (T, 40, 40, T))
    n = q.size
    for weights in (None, w):
        arrays = [nd.array(a, requires_grad=True) for a in (q, k, v)]
        o = nd.attention(*arrays)
        nd.mean(o if weights is None else o * nd.array(weights)).backward()
        go = (np.ones_like(q) if weights is None else weights) / np.float32(n)
        want = attention_reference(q, k, v, go)
        for a, name in zip(arrays, ("dq", "dk", "dv")):
            value, bound = want[name]  # the cotangent itself is rounded once more on the way
            within(a.grad().to_numpy(), (value, bound + 4 * U * np.abs(bound).max() + 8 * U * np.abs(value)), name)


@pytest.mark.gpu
def test_two_captured_steps_share_nothing():
    """Two captured steps of different sizes, replayed in turn, and eager calls between them."""
    import endia_amd as nd
    rng = np.random.default_rng(0)
    steps = []
    for N, V, T in ((40, 300, 20), (700, 900, 150)):
        x = nd.array(rng.standard_normal((N, 48)).astype(np.float32), requires_grad=True)
        w = nd.array(rng.standard_normal((48, V)).astype(np.float32), requires_grad=True)
        t = nd.array(rng.integers(0, V, N).astype(np.float32))
        q = nd.array(rng.standard_normal((1, T, 4, 64)).astype(np.float32), requires_grad=True)
        table = nd.array(rng.standard_normal((16, 4)).astype(np.float32), requires_grad=True)
        go = nd.array(rng.standard_normal((1, T, 4, 64)).astype(np.float32))

        def step(x=x, w=w, t=t, q=q, table=table, go=go):
            loss = nd.linear_cross_entropy(x, w, t)
            o = nd.relative_attention(q, q, q, table, max_distance=30)
            return [loss, o] + nd.grad(outs=[loss], inputs=[x, w]) + nd.grad(outs=[o], inputs=[q, table], grad_outs=[go])

        eager = [a.to_numpy() for a in step()]
        steps.append((nd.capture(step), eager))
    for turn in (0, 1, 1, 0, 1, 0, 0, 1):
        captured, eager = steps[turn]
        captured.replay()
        check_attention(1, 40, 60, 2, 2, 64)
        for a, b in zip(captured.outputs, eager):
            assert np.array_equal(a.to_numpy(), b), turn
    for captured, _ in steps:
        captured.close()


# ---- together -------------------------------------------------------------------------------------------------
def _little_model(nd, rng, B, T, S, H, D, V):
    """One decoder layer: causal self attention with position buckets, cross attention to encoder states, tied loss."""
    C = H * D
    p = {n: nd.array((rng.standard_normal(s) / np.sqrt(s[0])).astype(np.float32), requires_grad=True)
         for n, s in (("qkv", (C, 3 * C)), ("q2", (C, C)), ("kv", (C, 2 * C)), ("table", (16, H)))}
    p["emb"] = nd.array((0.3 * rng.standard_normal((V, C))).astype(np.float32), requires_grad=True)

    def loss(x, enc, lengths, target):
        zero = lambda n: nd.zeros([n])
        f = nd.reshape(nd.linear(nd.reshape(x, [B * T, C]), p["qkv"], zero(3 * C)), [B, T, 3 * H, D])
        a = nd.relative_attention(f[:, :, :H], f[:, :, H:2 * H], f[:, :, 2 * H:], p["table"], causal=True, max_distance=20)
        h = nd.reshape(a, [B * T, C]) + nd.reshape(x, [B * T, C])
        q = nd.reshape(nd.linear(h, p["q2"], zero(C)), [B, T, H, D])
        e = nd.reshape(nd.linear(nd.reshape(enc, [B * S, C]), p["kv"], zero(2 * C)), [B, S, 2 * H, D])
        h = h + nd.reshape(nd.attention(q, e[:, :, :H], e[:, :, H:], key_lengths=lengths), [B * T, C])
        return nd.linear_cross_entropy(h, p["emb"].T(), target)

    return p, loss


@pytest.mark.gpu
@pytest.mark.parametrize("T", [9, 70])
def test_operators_together_against_float64(T):
    import torch

    import endia_amd as nd
    rng = np.random.default_rng(0)
    B, S, H, D, V = 2, 33, 2, 32, 211
    C = H * D
    p, loss = _little_model(nd, rng, B, T, S, H, D, V)
    x, enc = rng.standard_normal((B, T, C)).astype(np.float32), rng.standard_normal((B, S, C)).astype(np.float32)
    lengths, target = np.array([33, 20], np.float32), rng.integers(0, V, B * T).astype(np.float32)
    target[::5] = -1
    value = loss(nd.array(x), nd.array(enc), nd.array(lengths), nd.array(target))
    got = nd.grad(outs=[value], inputs=list(p.values()))
    w = {n: torch.tensor(a.to_numpy(), dtype=torch.float64, requires_grad=True) for n, a in p.items()}
    tx, te = torch.tensor(x, dtype=torch.float64), torch.tensor(enc, dtype=torch.float64)
    heads = lambda a, n: a.reshape(B, n, -1, D).transpose(1, 2)
    f = tx @ w["qkv"]
    q, k, v = (heads(f[..., i * C:(i + 1) * C], T) for i in range(3))
    rel = [[bucket_of(j - i, 16, 20, False) for j in range(T)] for i in range(T)]
    s = q @ k.transpose(2, 3) * D ** -0.5 + w["table"][torch.tensor(rel)].permute(2, 0, 1)
    s = s.masked_fill(torch.triu(torch.ones(T, T, dtype=torch.bool), 1), -torch.inf)
    h = tx + (torch.softmax(s, 3) @ v).transpose(1, 2).reshape(B, T, C)
    e = te @ w["kv"]
    k, v = (heads(e[..., i * C:(i + 1) * C], S) for i in range(2))
    s = heads(h @ w["q2"], T) @ k.transpose(2, 3) * D ** -0.5
    s = s.masked_fill(torch.arange(S)[None, None, None, :] >= torch.tensor(lengths)[:, None, None, None], -torch.inf)
    h = h + (torch.softmax(s, 3) @ v).transpose(1, 2).reshape(B, T, C)
    kept = torch.tensor(target) >= 0
    want = torch.nn.functional.cross_entropy((h.reshape(B * T, C) @ w["emb"].T)[kept], torch.tensor(target)[kept].long())
    want.backward()
    # Five products of lengths up to 70, 3 C and 211 in a row, each good to (n + 16) u relative to its absolute sum, whose
    # size is at most sqrt(n) times the sum's: 1e-4 relative to the gradient's norm, as everywhere in these tests.
    assert abs(value.item() - want.item()) <= 1e-5 * abs(want.item())
    for g, (n, a) in zip(got, w.items()):
        ref = a.grad.numpy()
        assert np.linalg.norm(g.to_numpy() - ref) <= 1e-4 * np.linalg.norm(ref), n


@pytest.mark.gpu
@pytest.mark.parametrize("T", [5, 70])
def test_operators_in_a_captured_step(T):
    """A training step of the operators together, captured and replayed several times with eager work between the replays."""
    import endia_amd as nd
    rng = np.random.default_rng(0)
    B, S, H, D, V = 2, 33, 2, 32, 211
    p, loss = _little_model(nd, rng, B, T, S, H, D, V)
    lengths, target = nd.array(np.array([33, 20], np.float32)), nd.array(rng.integers(0, V, B * T).astype(np.float32))
    x, enc = nd.zeros([B, T, H * D]), nd.zeros([B, S, H * D])

    def step():
        value = loss(x, enc, lengths, target)
        return [value] + nd.grad(outs=[value], inputs=list(p.values()))

    batches = [(rng.standard_normal((B, T, H * D)), rng.standard_normal((B, S, H * D))) for _ in range(4)]
    eager = []
    for bx, be in batches:
        x.copy_from_numpy(bx)
        enc.copy_from_numpy(be)
        eager.append([a.to_numpy() for a in step()])
    captured = nd.capture(step)
    for turn in (0, 1, 2, 3, 1, 0):
        x.copy_from_numpy(batches[turn][0])
        enc.copy_from_numpy(batches[turn][1])
        captured.replay()
        got = [a.to_numpy() for a in captured.outputs]
        for a, b in zip(got, eager[turn]):
            assert np.array_equal(a, b), turn
        check_loss(600, 48, 333)  # eager work of other sizes on the same scratch memory
        nd.synchronize()
    captured.close()
