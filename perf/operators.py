"""Timing cases of the sequence-model operators: linear_cross_entropy, attention and relative_attention.

Every case has a plain form in elementary torch operations (float32 throughout, float64 for the bucket sums of the
position table) and, with `own = True`, the calls a program makes of endia_amd. `exact` evaluates the definitions once
more in float64.

Shapes: x [rows, width], weight [width, vocab] (a tied embedding is held [vocab, width] and used through its transposed
view); q [batch, queries, heads, dim], k and v [batch, keys, kv_heads, dim], position table [buckets, heads].
"""
import math

import torch

own = False  # True: run() calls endia_amd instead of the plain forms

LEFT_OUT = -1  # target of a row that has no class: it takes no part in the loss

_LOSS_LARGEST = 8192 * 4096 * 131072
_PAIRS_LARGEST = 16 * 4096 * 16384 * 128


def _loss(name, rows, width, vocab, step, tied):
    return {"name": name, "op": "loss", "rows": rows, "width": width, "vocab": vocab, "step": step, "tied": tied}


def _attend(name, batch, queries, keys, heads, kv_heads, dim, step, padded):
    return {"name": name, "op": "attend", "batch": batch, "queries": queries, "keys": keys, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "step": step, "padded": padded}


def _relative(name, batch, queries, keys, heads, kv_heads, dim, step, padded, causal, offset, buckets, distance):
    return dict(_attend(name, batch, queries, keys, heads, kv_heads, dim, step, padded), op="relative", causal=causal,
                offset=offset, buckets=buckets, distance=distance)


def listed():
    return [
        # a fine-tuning step on a handful of tokens: the weight matrix and its gradient are all there is to move
        _loss("loss_few_rows", 16, 768, 32001, True, True),
        # one ordinary training batch, no size a multiple of anything
        _loss("loss_odd", 2043, 1000, 50021, True, False),
        # the loss of a held-out batch: no gradient
        _loss("loss_evaluation", 4096, 2048, 65536, False, True),
        # a large model's training step
        _loss("loss_large", 8192, 4096, 131072, True, False),
        # one generated token of one sentence looks at a short encoded text
        _attend("cross_token", 1, 1, 77, 12, 12, 64, False, False),
        # one generated token for each of a batch of sentences, encoder states of many lengths
        _attend("cross_tokens_batch", 64, 1, 4000, 16, 16, 64, False, True),
        # a decoder's training step over padded encoder states
        _attend("cross_step", 8, 448, 1500, 16, 16, 64, True, True),
        # image positions looking at a short text, without a gradient
        _attend("cross_wide", 2, 4096, 77, 10, 10, 64, False, False),
        # long documents on both sides, query heads that share key heads
        _attend("cross_long", 1, 4096, 16384, 16, 4, 128, True, False),
        # one generated token with position buckets over what was generated before
        _relative("relative_token", 16, 1, 2049, 12, 12, 64, False, True, True, 2048, 32, 128),
        # an encoder's training step with buckets on both sides
        _relative("relative_step", 8, 512, 512, 12, 12, 64, True, True, False, 0, 32, 128),
        # a decoder's training step over a long text
        _relative("relative_long", 1, 5001, 5001, 16, 16, 128, True, False, True, 0, 32, 128),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("loss", "loss", "attend", "attend", "relative", "relative"))
    while True:
        if op == "loss":
            c = _loss("", _log_int(rng, 1, 8192), _log_int(rng, 64, 4096), _log_int(rng, 1000, 131072), rng.random() < 0.7,
                      rng.random() < 0.5)
            if c["rows"] * c["width"] * c["vocab"] > _LOSS_LARGEST // 2:
                continue
        else:
            step = rng.random() < 0.6
            kv_heads = rng.choice((1, 2, 3, 4, 8, 12, 16))
            heads = kv_heads * rng.choice((1, 1, 2, 4))
            one = not step and rng.random() < 0.4
            queries = 1 if one else _log_int(rng, 2, 4096)
            keys = _log_int(rng, 1, 16384)
            causal = op == "relative" and (one or rng.random() < 0.5)
            if op == "relative" and not one:
                keys = queries
            c = _attend("", _log_int(rng, 1, 64), queries, keys, heads, kv_heads, rng.choice((32, 40, 64, 64, 80, 96, 128, 128)),
                        step, rng.random() < 0.5)
            if op == "relative":
                c = _relative("", c["batch"], queries, keys, heads, kv_heads, c["dim"], step, c["padded"], causal,
                              keys - 1 if one else 0, rng.choice((16, 32, 32, 64)), rng.choice((64, 128, 128, 256)))
            if c["batch"] * heads * queries * keys * c["dim"] > _PAIRS_LARGEST // 4:
                continue
        del c["name"]
        return c


def _lengths(case):
    """Keys that belong to each sequence of the batch: all of them, or from all of them down to half as many."""
    B, K = case["batch"], case["keys"]
    return [max(1, K - (b * K) // (2 * B)) if case["padded"] else K for b in range(B)]


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)

    if case["op"] == "loss":
        N, D, V = case["rows"], case["width"], case["vocab"]
        x = normal(N, D)
        w = (normal(V, D) if case["tied"] else normal(D, V)).mul_(2.0 / math.sqrt(D))  # logits of a spread of 2
        t = torch.randint(0, V, (N,), generator=g, device="cuda").float()
        if N > 8:  # padding positions of the batch
            t[torch.rand(N, generator=g, device="cuda") < 0.1] = LEFT_OUT
        return {"x": x, "w": w, "t": t}
    B, Q, K, H, Hk, D = (case[n] for n in ("batch", "queries", "keys", "heads", "kv_heads", "dim"))
    s = {"q": normal(B, Q, H, D), "k": normal(B, K, Hk, D), "v": normal(B, K, Hk, D)}
    if case["padded"]:
        s["lengths"] = torch.tensor(_lengths(case), device="cuda", dtype=torch.float32)
    if case["step"]:
        s["g"] = normal(B, Q, H, D)
    if case["op"] == "relative":
        s["table"] = normal(case["buckets"], H)
    return s


# ---- the calls of endia_amd -----------------------------------------------------------------------------------
def _arrays(case, tensors):
    """The tensors as arrays of the framework."""
    import endia_amd as nd
    from endia_amd import _lib as L

    held = {}
    for name, t in tensors.items():
        a = nd.Array.empty(t.shape)
        torch.cuda.synchronize()
        L.call("endia_hip_memcpy_d2d", a.data_ptr(), t.data_ptr(), 4 * t.numel())
        if case["step"] and name in ("x", "w", "q", "k", "v", "table"):
            a.requires_grad_(True)
        held[name] = a
    nd.synchronize()
    return held


class _Device:
    """An array's memory as torch sees it; keeps the array alive."""

    def __init__(self, array):
        array = array if array.is_contiguous() else _contiguous(array)
        self.array = array
        self.__cuda_array_interface__ = {"shape": tuple(array.shape()), "typestr": "<f4", "data": (array.data_ptr(), False),
                                         "version": 2, "strides": None}


def _contiguous(array):
    import endia_amd as nd
    return nd.contiguous(array)


def _tensor(array):
    return torch.as_tensor(_Device(array), device="cuda")


def _run_own(case, s):
    import endia_amd as nd

    if case["op"] == "loss":
        w = s["w"].T() if case["tied"] else s["w"]
        loss = nd.linear_cross_entropy(s["x"], w, s["t"])
        wanted = [s["x"], s["w"]]
        out, names = {"loss": _tensor(loss)}, ("dx", "dw")
        if case["step"]:
            out.update(zip(names, map(_tensor, nd.grad(outs=[loss], inputs=wanted))))
        return out
    if case["op"] == "attend":
        o = nd.attention(s["q"], s["k"], s["v"], key_lengths=s.get("lengths"))
        wanted, names = [s["q"], s["k"], s["v"]], ("dq", "dk", "dv")
    else:
        o = nd.relative_attention(s["q"], s["k"], s["v"], s["table"], key_lengths=s.get("lengths"), causal=case["causal"],
                                  query_offset=case["offset"], max_distance=case["distance"])
        wanted, names = [s["q"], s["k"], s["v"], s["table"]], ("dq", "dk", "dv", "dtable")
    out = {"o": _tensor(o)}
    if case["step"]:
        out.update(zip(names, map(_tensor, nd.grad(outs=[o], inputs=wanted, grad_outs=[s["g"]]))))
    return out


# ---- the plain forms ------------------------------------------------------------------------------------------
def _plain_loss(case, s):
    x, t = s["x"], s["t"]
    w = s["w"].t() if case["tied"] else s["w"]
    logits = x @ w
    top = logits.amax(dim=1, keepdim=True)
    rows = torch.arange(x.shape[0], device=x.device)
    valid = t >= 0
    at = torch.where(valid, t, torch.zeros_like(t)).long()
    picked = logits[rows, at]
    p = logits.sub_(top).exp_()
    total = p.sum(dim=1, keepdim=True)
    count = valid.sum().clamp(min=1)
    each = torch.where(valid, (total.log() + top)[:, 0] - picked, torch.zeros_like(picked))
    out = {"loss": (each.sum(dtype=torch.float64) / count).float().reshape(1)}
    if case["step"]:
        p.div_(total)
        p[rows, at] -= 1.0
        p.mul_((valid.float() / count)[:, None])
        out["dx"] = p @ w.t()
        out["dw"] = p.t() @ x if case["tied"] else x.t() @ p
    return out


def _bucket(rel, buckets, distance, both_sides):
    """The bucket of each position difference key - query: one bucket a step at first, then logarithmically wider ones."""
    first = torch.zeros_like(rel)
    if both_sides:
        buckets //= 2
        first = (rel > 0).long() * buckets
        n = rel.abs()
    else:
        n = (-rel).clamp(min=0)
    exact_ones = buckets // 2
    far = torch.log(n.clamp(min=1).double() / exact_ones) / math.log(distance / exact_ones) * (buckets - exact_ones)
    far = (exact_ones + torch.floor(far + 1e-9).long()).clamp(max=buckets - 1)  # 1e-9: whole steps land on their own bucket
    return first + torch.where(n < exact_ones, n, far)


def _plain_attention(case, s):
    q, k, v = (s[n].transpose(1, 2) for n in ("q", "k", "v"))  # [batch, heads, length, dim]
    B, H, Q, D = q.shape
    Hk, K = k.shape[1], k.shape[2]
    G, scale = H // Hk, 1.0 / math.sqrt(D)
    q = q.reshape(B, Hk, G * Q, D)
    scores = (q @ k.transpose(2, 3)).mul_(scale).view(B, H, Q, K)
    if case["op"] == "relative":
        rel = torch.arange(K, device=q.device)[None, :] - (torch.arange(Q, device=q.device)[:, None] + case["offset"])
        bucket = _bucket(rel, case["buckets"], case["distance"], not case["causal"])
        scores += s["table"].t()[:, bucket]
        if case["causal"]:
            scores.masked_fill_(rel > 0, -math.inf)
    if case["padded"]:
        beyond = torch.arange(K, device=q.device)[None, :] >= s["lengths"][:, None]
        scores.masked_fill_(beyond[:, None, None, :], -math.inf)
    top = scores.amax(dim=3, keepdim=True)
    p = scores.sub_(top).exp_()
    p = p.div_(p.sum(dim=3, keepdim=True))
    pg = p.view(B, Hk, G * Q, K)
    o = pg @ v
    out = {"o": o.view(B, H, Q, D).transpose(1, 2).contiguous()}
    if case["step"]:
        g = s["g"].transpose(1, 2).reshape(B, Hk, G * Q, D)
        out["dv"] = (pg.transpose(2, 3) @ g).transpose(1, 2).contiguous()
        ds = (g @ v.transpose(2, 3)).sub_((g * o).sum(dim=3, keepdim=True)).mul_(pg)
        out["dq"] = (ds @ k).mul_(scale).view(B, H, Q, D).transpose(1, 2).contiguous()
        out["dk"] = (ds.transpose(2, 3) @ q).mul_(scale).transpose(1, 2).contiguous()
        if case["op"] == "relative":
            # each query's row set one place further than the row below it: a column is then one difference key - query
            rows = torch.zeros(H, Q, Q + K, device=q.device)
            rows[:, :, :K] = ds.view(B, H, Q, K).sum(dim=0).flip(1)
            each = rows.view(H, -1)[:, : Q * (Q + K - 1)].view(H, Q, Q + K - 1).sum(dim=1, dtype=torch.float64)
            rel = torch.arange(1 - Q, K, device=q.device) - case["offset"]
            bucket = _bucket(rel, case["buckets"], case["distance"], not case["causal"])
            table = torch.zeros(H, case["buckets"], device=q.device, dtype=torch.float64)
            out["dtable"] = table.index_add_(1, bucket, each).t().float().contiguous()
    return out


# ---- the interface of the timing tool -------------------------------------------------------------------------
def prepare(case, seed):
    s = _inputs(case, seed)
    if own:  # a program of the framework holds its data in arrays
        s = _arrays(case, s)
    return {"case": case, "data": s}


def run(state):
    case, s = state["case"], state["data"]
    if own:
        return _run_own(case, s)
    return _plain_loss(case, s) if case["op"] == "loss" else _plain_attention(case, s)


def work(case):
    if case["op"] == "loss":
        N, D, V = case["rows"], case["width"], case["vocab"]
        once = N * D + D * V
        return {"bytes": 4.0 * (once * (2 if case["step"] else 1) + N + 1), "flops": (6.0 if case["step"] else 2.0) * N * D * V}
    B, Q, K, H, Hk, D = (case[n] for n in ("batch", "queries", "keys", "heads", "kv_heads", "dim"))
    lengths = _lengths(case)
    pairs = 0
    for n in lengths:
        if case["op"] == "relative" and case["causal"]:
            first = min(n, case["offset"] + 1)  # keys that the first query sees; each later one sees one more, up to n
            more = min(Q - 1, n - first)
            pairs += first * Q + more * (more + 1) // 2 + (Q - 1 - more) * more
        else:
            pairs += Q * n
    moved = 2 * B * Q * H * D + 2 * sum(lengths) * Hk * D
    if case["step"]:
        moved += 2 * B * Q * H * D + 2 * B * K * Hk * D
    if case["op"] == "relative":
        moved += case["buckets"] * H * (2 if case["step"] else 1)
    return {"bytes": 4.0 * moved, "flops": (12.0 if case["step"] else 4.0) * pairs * H * D}


# ---- the definitions in float64 -------------------------------------------------------------------------------
def _exact_loss(case, s):
    x, t = s["x"].double(), s["t"].double()
    w = s["w"].double()
    if case["tied"]:
        w = w.t()
    kept = torch.nonzero(t >= 0)[:, 0]
    n = max(1, kept.numel())
    loss = torch.zeros((), dtype=torch.float64, device=x.device)
    dx, dw = torch.zeros_like(x), torch.zeros(w.shape, dtype=torch.float64, device=x.device)
    for part in kept.split(2048):
        xs = x[part]
        z = xs @ w
        lse = torch.logsumexp(z, dim=1)
        at = t[part].long()[:, None]
        loss += (lse - z.gather(1, at)[:, 0]).sum()
        if case["step"]:
            d = torch.exp(z - lse[:, None])
            d.scatter_add_(1, at, torch.full(at.shape, -1.0, dtype=torch.float64, device=x.device))
            d /= n
            dx[part] = d @ w.t()
            dw += xs.t() @ d
    out = {"loss": (loss / n).reshape(1)}
    if case["step"]:
        out.update(dx=dx, dw=dw.t().contiguous() if case["tied"] else dw)
    return out


def _exact_bucket(case, distance_to_key):
    """Bucket of key - query = distance_to_key in whole numbers: the logarithm's steps by comparing integer powers."""
    buckets, base, n = case["buckets"], 0, -distance_to_key
    if not case["causal"]:
        buckets //= 2
        base = buckets if distance_to_key > 0 else 0
        n = abs(n)
    n = max(n, 0)
    e = buckets // 2
    if n < e:
        return base + n
    steps, far = buckets - e, 0
    while far + 1 < steps and n ** steps * e ** (far + 1) >= case["distance"] ** (far + 1) * e ** steps:
        far += 1
    return base + e + far


def _exact_attention(case, s):
    B, Q, K, H, Hk, D = (case[n] for n in ("batch", "queries", "keys", "heads", "kv_heads", "dim"))
    G, dev = H // Hk, s["q"].device
    q, k, v = (s[n].double() for n in ("q", "k", "v"))
    g = s["g"].double() if case["step"] else None
    lengths = _lengths(case)
    out = {"o": torch.zeros_like(q)}
    if case["step"]:
        out.update(dq=torch.zeros_like(q), dk=torch.zeros_like(k), dv=torch.zeros_like(v))
    relative = case["op"] == "relative"
    if relative:
        table = s["table"].double()
        span = torch.tensor([_exact_bucket(case, d) for d in range(-(Q + case["offset"] - 1), K)], device=dev)
        out["dtable"] = torch.zeros_like(table)
    for b in range(B):
        n = lengths[b]
        for h in range(H):
            c = h // G
            ks, vs = k[b, :n, c], v[b, :n, c]
            for first in range(0, Q, 4096):
                last = min(Q, first + 4096)
                qs = q[b, first:last, h]
                z = qs @ ks.t() / math.sqrt(D)
                if relative:
                    place = torch.arange(first, last, device=dev)[:, None] + case["offset"]
                    to_key = torch.arange(n, device=dev)[None, :] - place
                    where = span[to_key + Q + case["offset"] - 1]
                    z = z + table[where, h]
                    if case["causal"]:
                        z = torch.where(to_key <= 0, z, torch.full_like(z, -math.inf))
                p = torch.softmax(z, dim=1)
                out["o"][b, first:last, h] = p @ vs
                if case["step"]:
                    gs = g[b, first:last, h]
                    out["dv"][b, :n, c] += p.t() @ gs
                    dp = gs @ vs.t()
                    dz = p * (dp - (p * dp).sum(dim=1, keepdim=True))
                    out["dq"][b, first:last, h] = dz @ ks / math.sqrt(D)
                    out["dk"][b, :n, c] += dz.t() @ qs / math.sqrt(D)
                    if relative:
                        out["dtable"][:, h] += torch.zeros(case["buckets"], dtype=torch.float64, device=dev).index_add_(
                            0, where.reshape(-1), dz.reshape(-1))
    if relative and not case["step"]:
        del out["dtable"]
    return out


def exact(case, seed):
    s = _inputs(case, seed)
    return _exact_loss(case, s) if case["op"] == "loss" else _exact_attention(case, s)
