"""The token-model operators in float64, straight from their definitions, with a bound on the rounding error of a
float32 evaluation beside each value.

The bounds count roundings.  U = 2^-24 is half a step of float32 relative to the value.  A softmax exponent
z = (x - max) / T takes at most three roundings (difference, reciprocal or quotient, product), and the exponential
itself is good to 8 U, so every term of a sum is good to EXP(z) = 8 U + 4 U |z| of itself.  A sum of n terms in chains
of at most n / 128 + 64 additions (128 threads or more walk a row; their partial sums meet in short trees) adds
CHAIN(n) = (n / 128 + 64) U of the sum of absolute values."""
import numpy as np

U = 2.0 ** -24


def exp_err(z):
    return 8 * U + 4 * U * np.abs(z)


def chain(n):
    return (n / 128 + 64) * U


def _softmax(x, t):
    """z, p, log-sum, and the error bound of the log-sum, for rows without NaN / +inf that are not all -inf."""
    x = np.asarray(x, np.float64)
    m = x.max(1, keepdims=True)
    z = (x - m) / t
    e = np.exp(z)
    s = e.sum(1, keepdims=True)
    p, ls = e / s, np.log(s)
    zf = np.where(p > 0, z, 0.0)
    ls_err = (p * exp_err(zf)).sum(1, keepdims=True) + chain(x.shape[1]) + 2 * U * np.abs(ls) + U
    return z, zf, p, ls, ls_err


def embedding_forward(table, tokens, scale):
    table = np.asarray(table, np.float32)
    ok = (tokens >= 0) & (tokens < table.shape[0])
    return np.where(ok[:, None], np.float32(scale) * table[np.where(ok, tokens, 0)], np.float32(0))   # one rounding: exact


def embedding_backward(grad_out, tokens, vocab, scale, old=None):
    g, scale = np.asarray(grad_out, np.float64), float(np.float32(scale))
    out = np.zeros((vocab, g.shape[1])) if old is None else np.asarray(old, np.float64).copy()
    size = np.abs(out)
    count = np.zeros(vocab)
    ok = (tokens >= 0) & (tokens < vocab)
    np.add.at(out, tokens[ok], scale * g[ok])
    np.add.at(size, tokens[ok], abs(scale) * np.abs(g[ok]))
    np.add.at(count, tokens[ok], 1.0)
    # a sum of m terms in any order: (m - 1) roundings on a path at most, then the scale and the old value
    return out, (count[:, None] + 2) * U * size


def token_logprobs(x, tokens, t, top_k):
    """logprob, entropy, stats, top tokens, top logprobs; each but the tokens with its bound."""
    t = float(np.float32(t))
    z, zf, p, ls, ls_err = _softmax(x, t)
    v, rows = x.shape[1], np.arange(x.shape[0])
    lp_all = z - ls
    ids = np.where((tokens >= 0) & (tokens < v), tokens, 0)
    zt = z[rows, ids]
    has = tokens >= 0
    lp = np.where(has, lp_all[rows, ids], 0.0)
    lp_err = np.where(has & np.isfinite(lp), ls_err[:, 0] + 4 * U * np.abs(np.where(np.isfinite(zt), zt, 0)) + 2 * U * np.abs(np.where(np.isfinite(lp), lp, 0)), 0.0)
    h = (ls - (p * zf).sum(1, keepdims=True))[:, 0]
    h_err = ls_err[:, 0] + (p * np.abs(zf) * (2 * exp_err(zf) + 2 * chain(v) + 8 * U)).sum(1) + 2 * U * np.abs(h) + ls_err[:, 0] * (p * np.abs(zf)).sum(1)
    stats = np.stack([np.asarray(x, np.float64).max(1), ls[:, 0]], 1)
    stats_err = np.stack([np.zeros(len(rows)), ls_err[:, 0]], 1)
    x32 = np.asarray(x, np.float32) + np.float32(0)
    order = np.argsort(-x32.astype(np.float64), axis=1, kind="stable")[:, :top_k]
    vals = np.take_along_axis(x32, order, 1)
    top = np.where(np.isneginf(vals), -1, order).astype(np.int32)
    tl = np.take_along_axis(lp_all, order, 1)
    tl_err = np.where(np.isfinite(tl), ls_err + 4 * U * np.abs(np.where(np.isfinite(tl), np.take_along_axis(z, order, 1), 0)) + 2 * U * np.abs(np.where(np.isfinite(tl), tl, 0)), 0)
    if top_k > v:
        pad = ((0, 0), (0, top_k - v))
        top = np.pad(top, pad, constant_values=-1)
        tl, tl_err = np.pad(tl, pad, constant_values=-np.inf), np.pad(tl_err, pad)
    return (lp, lp_err), (h, h_err), (stats, stats_err), top, (tl, tl_err)


def token_logprobs_backward(x, tokens, t, grad_logprob, grad_entropy):
    """The gradient from the definition, statistics included; the call under test gets them in float32, so their own
    rounding (one each, on the log-sum and the entropy) is part of the bound."""
    t = float(np.float32(t))
    z, zf, p, ls, ls_err = _softmax(x, t)
    v, rows = x.shape[1], np.arange(x.shape[0])
    logp = np.where(p > 0, zf - ls, 0.0)
    h = -(p * logp).sum(1, keepdims=True)
    gl = np.zeros((len(rows), 1)) if grad_logprob is None else np.where((tokens >= 0) & (tokens < v), grad_logprob, 0.0)[:, None].astype(np.float64)
    gh = np.zeros((len(rows), 1)) if grad_entropy is None else np.asarray(grad_entropy, np.float64)[:, None]
    grad = -p * gl - gh * p * (logp + h)
    hit = np.zeros_like(p)
    ok = (tokens >= 0) & (tokens < v)
    hit[rows[ok], tokens[ok]] = 1
    grad = (grad + hit * gl) / t
    rel = exp_err(zf) + 4 * U * np.abs(logp) + 2 * U * np.abs(ls) + 8 * U
    _, (he, h_err), _, _, _ = token_logprobs(x, np.full(len(rows), -1), t, 0)
    err = (p * rel * np.abs(gl) + np.abs(gh) * p * ((rel + 4 * U) * np.abs(logp + h) + 4 * U * (np.abs(zf) + np.abs(ls) + np.abs(h)))
           + hit * np.abs(gl) * 4 * U) / t + 4 * U * np.abs(grad) + 1e-37
    return grad, err


def distill_loss(x, ids, u, t, w):
    """Loss and gradient with bounds; rows whose logits are finite or -inf, entries in range or negative."""
    t = float(np.float32(t))
    z, zf, p, ls, ls_err = _softmax(x, t)
    n, v = x.shape
    u = np.asarray(u, np.float64)
    there = (ids >= 0) & ~np.isneginf(u)
    um = np.where(there, u, -np.inf).max(1, keepdims=True)
    any_ = there.any(1)
    uz = np.where(there, (u - np.where(any_[:, None], um, 0)) / t, -np.inf)
    qe = np.exp(uz)
    mass = np.where(any_[:, None], qe.sum(1, keepdims=True), 1.0)
    q = qe / mass
    uzf = np.where(there, uz, 0.0)
    lq = np.where(there, uzf - np.log(mass), 0.0)
    lq_err = (q * exp_err(uzf)).sum(1, keepdims=True) + chain(u.shape[1]) + 8 * U * (1 + np.abs(uzf) + np.abs(np.log(mass)))
    at = np.where(there, ids, 0)
    zt = np.take_along_axis(z, at, 1)
    lp = np.where(there, zt - ls, 0.0)
    fin = np.where(np.isfinite(lp), lp, 0.0)
    lp_err = ls_err + 4 * U * np.abs(np.where(np.isfinite(zt), zt, 0)) + 2 * U * np.abs(fin)
    w = np.asarray(w, np.float64)
    live = (w != 0) & any_
    terms = np.where(q > 0, q * (lq - lp), 0.0)
    loss = np.where(live, terms.sum(1) * t * t * w, 0.0)
    size = np.where(q > 0, q * np.abs(lq - fin), 0.0)
    loss_err = (q * (lq_err + lp_err) + size * (lq_err + exp_err(0) + chain(u.shape[1]) + 8 * U)).sum(1) * t * t * np.abs(w)
    qt = np.zeros_like(p)
    qt_err = np.zeros_like(p)
    for j in range(u.shape[1]):
        r = np.nonzero(there[:, j])[0]
        qt[r, ids[r, j]] += q[r, j]
        qt_err[r, ids[r, j]] += q[r, j] * (lq_err[r, j] + exp_err(0) + (u.shape[1] + 8) * U)
    grad = np.where(live[:, None], (p - qt) * t * w[:, None], 0.0)
    err = (p * (exp_err(zf) + ls_err + 8 * U) + qt_err) * t * np.abs(w[:, None]) + 4 * U * np.abs(grad) + 1e-37
    return (loss, loss_err), (grad, np.where(live[:, None], err, 0.0))


def quantize4(w, group):
    """Codes [n, k padded to 128] and scales [n, groups] with the roundings the definition names, in float32."""
    w = np.asarray(w, np.float32)
    k, n = w.shape
    kp, groups = -(-k // 128) * 128, -(-k // group)
    codes, scales = np.full((n, kp), 8, np.int64), np.zeros((n, groups), np.float32)
    for g in range(groups):
        block = w[g * group:(g + 1) * group]
        top = np.abs(block).max(0)
        s = (top / np.float32(7)).astype(np.float32)
        bad = ~np.isfinite(block).all(0)
        scales[:, g] = np.where(bad, np.float32(np.nan), s)
        with np.errstate(all="ignore"):
            c = np.clip(np.rint(block / np.where(s > 0, s, np.float32(1))), -7, 7)
        c = np.where((s > 0) & ~bad, c, 0)
        codes[:, g * group:g * group + block.shape[0]] = 8 + c.T.astype(np.int64)
    return codes, scales


def pack4(codes):
    n, kp = codes.shape
    c = codes.reshape(n, kp // 8, 8).astype(np.uint64)
    words = sum(c[:, :, b] << np.uint64(4 * b) for b in range(8)).astype(np.uint32)
    return np.ascontiguousarray(words.reshape(n, kp // 128, 4, 4).transpose(0, 1, 3, 2).reshape(n, kp // 8))


def dequantize4(codes, scales, k, group):
    return ((codes[:, :k] - 8) * np.repeat(scales.astype(np.float64), group, 1)[:, :k]).T


def matmul4(x, codes, scales, k, group, bias):
    """x . w + bias with its bound.  The products of a 24-bit x (in parts) and a code are exact.  At most k / 4 + 64
    additions follow each other on the way to an output; the tensor cores may drop a whole step (2 U) at each."""
    w = dequantize4(codes, scales, k, group)
    x = np.asarray(x, np.float64)
    y = x @ w + (0 if bias is None else bias)
    size = np.abs(x) @ np.abs(w) + (0 if bias is None else np.abs(bias))
    return y, (k / 4 + 64) * 2 * U * size


def check(got, want, err, what=""):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    odd = ~np.isfinite(want)
    assert np.array_equal(np.where(odd, got, 0), np.where(odd, want, 0), equal_nan=True), f"{what}: infinities or NaN differ"
    off = np.where(odd, 0.0, np.abs(got - np.where(odd, 0, want)))
    over = ~(off <= np.broadcast_to(err, off.shape))
    at = tuple(np.argwhere(over)[0]) if over.any() else None
    assert at is None, f"{what}: {over.sum()} of {over.size} off, first at {at}: got {got[at]!r}, want {want[at]!r}, allowed {np.broadcast_to(err, off.shape)[at]:.3e}"
