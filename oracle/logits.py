"""float64 restatement of the operators over wide rows of logits (log-probabilities of given tokens; top-k distillation), for the tests:
values, gradients, and first-order bounds on what fp32 arithmetic may add to either."""
import numpy as np

U = 2.0 ** -24        # half a step of fp32, relative


def chain(v):
    """additions one after another in a lane's sums over v logits: a row of more than 2048 16-byte pieces (of 4 logits at least) belongs to 256 threads
    or more and a lane adds a piece's own sum; fewer pieces are at most 32 for each of 64 lanes (of which the shortest rows have v / 64 logits)"""
    return min(v / 64, max(32, v / 1024))


def order_key(z):
    """descending order of a row: NaN first, then by value (-0 = +0)"""
    return np.where(np.isnan(z), np.inf, z), np.isnan(z)


def top_ids(z, k):
    """z [N, V] -> [N, k] int64: the k largest, ties by the lower index, NaN above +inf"""
    out = np.empty((z.shape[0], k), dtype=np.int64)
    idx = np.arange(z.shape[1])
    for n in range(z.shape[0]):
        v, nan = order_key(z[n])
        out[n] = np.lexsort((idx, -v, ~nan))[:k]
    return out


def log_softmax(z, tau):
    """-> (log-probabilities, lse, the rows' largest finite x); a row of nothing but -inf has log-probabilities -inf"""
    x = z.astype(np.float64) / tau
    m = x.max(axis=1, keepdims=True)
    m0 = np.where(np.isfinite(m), m, 0.0)
    with np.errstate(divide="ignore", invalid="ignore"):
        s = np.exp(x - m0).sum(axis=1, keepdims=True)
        lse = m0 + np.log(s)
        lp = np.where(np.isneginf(lse), -np.inf, (x - m0) - np.log(s))     # (not x - lse: at the type's lowest value ln s is lost in lse)
    return lp, lse[:, 0], m0[:, 0]


def _xlogy(p, lp):
    return np.where(p > 0, p * np.where(p > 0, lp, 0.0), 0.0)


def token_logprobs(z, tokens, k, tau):
    """-> dict of logp, entropy, lse, top_ids, top_logp and the bounds err_* of an fp32 evaluation"""
    lp, lse, m = log_softmax(z, tau)
    p = np.exp(lp)
    ent = -_xlogy(p, lp).sum(axis=1)
    n, v = z.shape
    # a sum of v positive terms in chains and a tree, terms of relative error (4 + 3 |d|) U each, |d| e^-|d| <= 0.37
    sum_u = (chain(v) + 48) * U
    out = {"lse": lse, "entropy": ent, "err_lse": sum_u + 4 * U * (np.abs(lse) + np.abs(m)), "err_entropy": sum_u * (4 + 3 * np.log(max(v, 2)))}

    def bound(values):
        spread = np.where(np.isfinite(values), np.abs(values), 0.0)
        return sum_u + 6 * U * (1 + spread + np.log(max(v, 2)))

    if tokens is not None:
        t = np.clip(tokens, 0, v - 1)
        got = lp[np.arange(n), t]
        out["logp"] = np.where(tokens < 0, 0.0, np.where(tokens >= v, np.nan, got))
        out["err_logp"] = bound(got)
    if k:
        out["top_ids"] = top_ids(z, k)
        out["top_logp"] = np.take_along_axis(lp, out["top_ids"], 1)
        out["err_top_logp"] = bound(out["top_logp"])
    return out


def token_logprobs_grad(z, tokens, ids, tau, g_logp=None, g_entropy=None, g_lse=None, g_top=None):
    """-> (gradient [N, V], bound of an fp32 evaluation per element)"""
    n, v = z.shape
    lp, lse, _ = log_softmax(z, tau)
    live = ~np.isneginf(lse)
    p = np.where(live[:, None], np.exp(lp), 0.0)
    lp0 = np.where(p > 0, lp, 0.0)
    ent = -(p * lp0).sum(axis=1)
    zero = np.zeros(n)
    ge = zero if g_entropy is None else g_entropy.astype(np.float64)
    gl = zero if g_lse is None else g_lse.astype(np.float64)
    sparse = np.zeros((n, v))
    mass = zero.copy()
    size = np.abs(gl) + np.abs(ge) * (1 + ent)
    if g_logp is not None:
        g = np.where(tokens < 0, 0.0, g_logp.astype(np.float64))
        np.add.at(sparse, (np.arange(n), np.clip(tokens, 0, v - 1)), g)
        mass, size = mass + g, size + np.abs(g)
    if g_top is not None:
        g = g_top.astype(np.float64)
        np.add.at(sparse, (np.arange(n)[:, None], ids), g)
        mass, size = mass + g.sum(axis=1), size + np.abs(g).sum(axis=1)
    grad = p * ((gl - mass)[:, None] - ge[:, None] * (lp0 + ent[:, None])) + sparse
    k = 0 if ids is None else ids.shape[1]
    rel = U * (chain(v) + 64 + 2 * k + 8 * np.abs(lp0))
    bound = p * (size[:, None] + np.abs(ge)[:, None] * np.abs(lp0)) * rel + 8 * U * np.abs(sparse)
    live = live[:, None]
    return np.where(live, grad / tau, 0.0), np.where(live, bound / tau, 0.0)


def distill(z, ids, t_logp, tau, tail, w):
    """-> (row losses, d sum(w L) / dz, bounds of both in fp32)"""
    n, v = z.shape
    k = ids.shape[1]
    z = np.where((w == 0)[:, None], 0.0, z.astype(np.float64))       # a row of weight 0 takes no part
    lp, lse, _ = log_softmax(z, tau)
    live = ~np.isneginf(lse)
    p = np.where(live[:, None], np.exp(lp), 0.0)
    there = ids >= 0
    t = np.where(there, t_logp.astype(np.float64), -np.inf)
    with np.errstate(invalid="ignore", divide="ignore"):
        if not tail:
            tm = t.max(axis=1, keepdims=True)
            tm = np.where(np.isfinite(tm), tm, 0.0)
            t = t - (tm + np.log(np.exp(t - tm).sum(axis=1, keepdims=True)))
            t = np.where(there & ~np.isnan(t), t, -np.inf)
        q = np.exp(t)
        lq = np.where(q > 0, t, 0.0)
        at = np.clip(ids, 0, v - 1)
        ls = np.take_along_axis(lp, at, 1)
        row = np.where(q > 0, q * (lq - ls), 0.0).sum(axis=1)
        on_list = np.zeros((n, v), dtype=bool)
        r, c = np.nonzero(there)
        on_list[r, ids[r, c]] = True
        qi = np.zeros((n, v))
        np.add.at(qi, (r, ids[r, c]), q[r, c])
        Q = q.sum(axis=1)
        rest = np.where(on_list.all(axis=1), 0.0, np.maximum(1.0 - Q, 0.0)) if tail else np.zeros(n)
        off = np.where(on_list, -np.inf, lp)
        om = off.max(axis=1)
        om0 = np.where(np.isfinite(om), om, 0.0)
        lp_off = om0 + np.log(np.exp(off - om0[:, None]).sum(axis=1))
        row = row + np.where(rest > 0, rest * (np.log(np.where(rest > 0, rest, 1.0)) - lp_off), 0.0)
        share = np.where(np.isfinite(lp_off)[:, None], np.exp(off - np.where(np.isfinite(lp_off), lp_off, 0.0)[:, None]), 0.0)
    grad = p * (Q + rest)[:, None] - qi - rest[:, None] * share
    # bounds: sums as above; 1 - sum q to (k + 8) U of what is left beside its largest term
    d_rest = (k + 8) * U * (1.0 - np.minimum(q.max(axis=1), 1.0) + 4 * U) * (1 if tail else 0)
    sum_u = (chain(v) + 64 + 2 * k) * U
    fin = lambda a: np.where(np.isfinite(a), np.abs(a), 0.0)   # noqa: E731
    e_row = sum_u * (np.where(q > 0, q * (1 + np.abs(lq) + fin(ls)) * (1 + 4 * U * fin(ls)), 0.0).sum(axis=1) + np.log(max(v, 2)))
    e_row = e_row + (d_rest + sum_u * rest) * (2 + fin(np.log(np.where(rest > 0, rest, 1.0))) + fin(lp_off))
    lp0 = np.where(p > 0, np.abs(lp), 0.0)
    e_grad = (p * (Q + rest)[:, None] + rest[:, None] * share) * (sum_u + 8 * U * lp0) + d_rest[:, None] * (share + p) \
        + qi * U * (2 * k + 32 + 4 * np.abs(np.where(qi > 0, np.log(np.where(qi > 0, qi, 1.0)), 0.0)))
    part = (w != 0) & live
    row = np.where(w != 0, tau ** 2 * row, 0.0)
    scale = (tau * w)[:, None]
    return row, np.where(part[:, None], grad * scale, 0.0), np.where(w != 0, tau ** 2 * e_row, 0.0), np.where(part[:, None], e_grad * np.abs(scale), 0.0)
