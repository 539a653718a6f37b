"""The scoring operators in 64 bits, one row at a time, with the bounds that
the kernels' arithmetic has to keep.

Bounds, with u = 2^-24 (half a step of fp32, relative).  A term
2^((x - m) a) with a = fp32(log2(e) / T) is off by
  - at most a subtraction or a reference's rounding, a product, and the rounding
    of a: 3 u |x - m| / T in the exponent (nats),
  - the exponential: ex2.approx, 2^-22 relative = 4 u,
and a thread adds at most `n` such terms in fp32 (n u relative, all terms being
positive; fewer where it adds steps), with one rescaling (a term of its own, and
a product) each time its maximum moves: at most 6 u for each of at most 16 moves
counted here as 96 u, in which a warp's five fp32 additions are too.  Sums over
warps are in fp64.
"""
import math

import numpy as np

U = 2.0 ** -24
NO_TAIL = 2.0 ** -20
THREADS = 128  # the fewest threads that share a row
# half a step of each type, relative, and half its smallest step
HALF = {"float32": (2.0 ** -24, 2.0 ** -150), "bfloat16": (2.0 ** -8, 2.0 ** -134), "float16": (2.0 ** -11, 2.0 ** -25)}


def terms(V):
    """fp32 roundings, in units of u, of a sum over a row of V: terms and rescalings."""
    return 4 + (V / THREADS + 17) + 96


def rounded(v, dtype):
    """Bound of one rounding of v to the type."""
    rel, least = HALF[dtype]
    return np.abs(v) * rel + least


class RowDist:
    """softmax(x / T) of one row, with the bounds of the kernels' sums over it."""

    def __init__(self, x, T):
        x = np.asarray(x, np.float64)
        self.x, self.T = x, T
        self.nan = bool(np.isnan(x).any() or (x == np.inf).any())
        self.empty = not self.nan and bool((x == -np.inf).all())
        if self.nan or self.empty:
            return
        self.m = x.max()
        with np.errstate(over="ignore"):
            self.d = (x - self.m) / T  # -inf where masked
        e = np.exp(self.d)
        self.s = math.fsum(e)
        self.p = e / self.s
        self.logp = self.d - math.log(self.s)
        dd = np.where(self.p > 0, self.d, 0.0)
        E, E2 = float((self.p * -dd).sum()), float((self.p * dd * dd).sum())
        self.H = math.log(self.s) + E
        n = terms(len(x))
        self.eps_s = (3 * E + n) * U  # relative, of s
        self.eps_H = self.eps_s + (3 * E2 + n * E) * U + E * self.eps_s


def score(x, T, tokens, top_n):
    """{logprobs, entropy, top_ids, top_logprobs, row_max, row_sum} and the bounds of each."""
    V = len(x)
    tokens = None if tokens is None else [int(t) for t in tokens]
    valid = None if tokens is None else [0 <= t < V for t in tokens]
    n = 0 if tokens is None else len(tokens)
    ids, tops = np.full(top_n, -1, np.int64), np.full(top_n, -np.inf)
    if tokens is not None and not any(valid):
        o = dict(logprobs=np.zeros(n), entropy=0.0, top_ids=ids, top_logprobs=tops, row_max=0.0, row_sum=0.0)
        return o, {k: 0.0 for k in o}
    R = RowDist(x, T)
    if R.nan:
        o = dict(logprobs=np.array([np.nan if v else 0.0 for v in valid or []]), entropy=np.nan, top_ids=ids,
                 top_logprobs=np.full(top_n, np.nan), row_sum=np.nan)
        return o, {k: 0.0 for k in o}
    if R.empty:
        o = dict(logprobs=np.array([-np.inf if v else 0.0 for v in valid or []]), entropy=0.0, top_ids=ids,
                 top_logprobs=tops, row_max=-np.inf, row_sum=0.0)
        return o, {k: 0.0 for k in o}
    order = np.lexsort((np.arange(V), -np.asarray(x, np.float64)))[:top_n]
    order = order[np.asarray(x, np.float64)[order] > -np.inf]
    ids[: len(order)], tops[: len(order)] = order, R.logp[order]
    lp = np.array([R.logp[t] if v else 0.0 for t, v in zip(tokens or [], valid or [])])

    def b(v):  # log s, then one rounding
        with np.errstate(invalid="ignore"):
            return np.where(np.isfinite(v), R.eps_s + np.abs(v) * U, 0.0)

    o = dict(logprobs=lp, entropy=R.H, top_ids=ids, top_logprobs=tops, row_max=R.m / T, row_sum=R.s)
    return o, dict(logprobs=b(lp), entropy=R.eps_H + abs(R.H) * U, top_ids=0, top_logprobs=b(tops),
                   row_max=abs(R.m / T) * 2.0 ** -50, row_sum=R.s * R.eps_s)


def score_grad(x, T, tokens, g_lp, g_H, dtype):
    """The gradient of sum(g_lp * logprobs) + g_H * entropy, and its bound.  The
    kernel takes row_max, row_sum and the entropy as the forward kernel gave
    them, with their errors."""
    V = len(x)
    zero = np.zeros(V)
    if tokens is not None and not any(0 <= int(t) < V for t in tokens):
        return zero, zero
    gs = np.zeros(V)
    G = 0.0
    for t, g in zip(tokens if tokens is not None else [], g_lp if g_lp is not None else []):
        if 0 <= int(t) < V:
            gs[int(t)] += float(g)
            G += float(g)
    g_H = 0.0 if g_H is None else float(g_H)
    R = RowDist(x, T)
    if R.empty or (not gs.any() and g_H == 0.0 and G == 0.0):
        return zero, zero
    if R.nan:
        if G == 0.0 and g_H == 0.0:
            return gs / T, None
        return np.full(V, np.nan), zero
    lp = np.where(R.p > 0, R.logp, 0.0)
    dx = (gs - R.p * (G + g_H * np.where(R.p > 0, lp + R.H, 0.0))) / T
    dd = np.where(R.p > 0, -R.d, 0.0)
    # one term (3 u |d| + 4 u), its two roundings with c0 + c1 d, and c0, c1's own
    rel = (3 * dd + 4 + 6) * U + R.eps_s
    size = abs(G) + abs(g_H) * (np.abs(lp) + R.H + math.log(R.s) + dd)
    b = R.p / T * (size * rel + abs(g_H) * (R.eps_s + R.eps_H))
    return dx, b + rounded(np.abs(dx) + b, dtype) + 2.0 ** -126 * (1 + size / T)


def distill(x, T, ids, values, kind, weight, dtype):
    """(loss, its bound, gradient, its bound) of one row."""
    V = len(x)
    there = [(int(i), float(v)) for i, v in zip(ids, values) if 0 <= int(i) < V
             and not (kind == "logits" and v == -np.inf)]
    zero = np.zeros(V)
    if not there:
        return 0.0, 0.0, zero, zero
    v = np.array([t[1] for t in there])
    if kind == "logits":
        z = v / T
        logq = z - z.max() - math.log(math.fsum(np.exp(z - z.max())))
    else:
        logq = v
    q = np.exp(logq)
    Q = math.fsum(q)
    rest = 0.0 if kind == "logits" else 1.0 - Q
    rest = 0.0 if rest < NO_TAIL else rest
    R = RowDist(x, T)
    if R.nan:
        g = zero if weight == 0 else np.full(V, np.nan)
        return np.nan, 0.0, g, zero
    if R.empty:
        return np.inf, 0.0, zero, zero
    listed = np.zeros(V, bool)
    mass = np.zeros(V)
    for (i, _), qi in zip(there, q):
        listed[i] = True
        mass[i] += qi
    others = np.asarray(x, np.float64)[~listed]
    tail_empty = len(others) == 0 or bool((others == -np.inf).all())
    loss = 0.0
    for (i, _), qi, lq in zip(there, q, logq):
        if qi > 0:
            loss += qi * (lq - R.logp[i])
    n = terms(V)
    eps_t = 0.0
    if not tail_empty:
        mo = others.max()
        do = (others - mo) / T
        eo = np.exp(do)
        so = math.fsum(eo)
        po = eo / so
        E = float((po * np.where(po > 0, -do, 0.0)).sum())
        eps_t = (3 * E + n) * U
        log_R = math.log(so) + (mo - R.m) / T - math.log(R.s)
        tail = math.exp(log_R)
    else:
        log_R, tail = -np.inf, 0.0
    if rest > 0:
        loss += rest * (math.log(rest) - log_R)
    eps_s = eps_t * tail  # the listed ids' terms are in fp64
    b_loss = 0.0
    if np.isfinite(loss):
        b_loss = (Q + rest) * eps_s + rest * eps_t + abs(loss) * U + 1e-12
    if weight == 0:
        return loss, b_loss, zero, zero
    all_ = Q + rest
    dx = np.where(listed, R.p * all_ - mass, 0.0)
    b = np.where(listed, R.p * all_ * eps_s + 1e-13, 0.0)
    if not tail_empty:
        share = np.zeros(V)
        share[~listed] = po
        dx = np.where(listed, dx, share * (tail * all_ - rest))
        dist = np.zeros(V)
        dist[~listed] = np.where(po > 0, -do, 0.0)
        rel = (3 * dist + 4 + 4) * U + eps_t
        b = np.where(listed, b, share * (tail * all_ * (rel + eps_s) + rest * rel))
    w = abs(weight) / T
    dx = dx * (weight / T)
    b = b * w
    return loss, b_loss, dx, b + rounded(np.abs(dx) + b, dtype) + 2.0 ** -126 * (1 + w)
