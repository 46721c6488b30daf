"""The sequence-layer and scoring operators in 64 bits, one definition after the other, with the error an fp32 evaluation may have.

Every function returns (values, bounds): float64 arrays, and for each how far an evaluation in 32 bits may be from it, before the one
rounding to the output's type.  U = 2^-24 is half an fp32 step; an exp(-|x|) by a rounded x log2(e) and a one-ulp exp2 is
off by (2 |x| + 2) U, with the reciprocal and products of a gate (2 |x| + 8) U; a bound follows its operator's recursion or sums
with absolute values in place of the values, so cancellation is paid for."""
from __future__ import annotations

import numpy as np

U = 2.0 ** -24
# a gate weight p = exp(-|f|) / (1 + exp(-|f|)) below the smallest normal fp32 number is taken as 0: p is off by less than 2^-126,
# which moves a state by less than 2^-126 (|x| + |h|) a step and a gradient by less than 2^-126 |g|
FLUSH = 2.0 ** -126


def sigmoid(x):
    with np.errstate(over="ignore"):
        return 1.0 / (1.0 + np.exp(-x))


def gated_scan(x, f, ranges, h0=None, reverse=False, grad_y=None, grad_h_last=None):
    """x, f [n_tokens, C]; ranges [(begin, end)].  Values / bounds: y, h_last, and with grad_y grad_x, grad_f, grad_h0.
    Tokens of no sequence are NaN in y and the gradients."""
    x, f = x.astype(np.float64), f.astype(np.float64)
    n, c = x.shape
    k = len(ranges)
    v = {"y": np.full((n, c), np.nan), "h_last": np.zeros((k, c))}
    w = {"y": np.zeros((n, c)), "h_last": np.zeros((k, c))}
    if grad_y is not None:
        grad_y = grad_y.astype(np.float64)
        for name, shape in (("grad_x", (n, c)), ("grad_f", (n, c)), ("grad_h0", (k, c))):
            v[name], w[name] = np.full(shape, np.nan), np.zeros(shape)
    for s, (b, e) in enumerate(ranges):
        order = range(e - 1, b - 1, -1) if reverse else range(b, e)
        h = np.zeros(c) if h0 is None else h0[s].astype(np.float64)
        m, err = np.abs(h), np.zeros(c)  # |h| without cancellation; bound of the state's error
        trace = []
        for t in order:
            a, g = sigmoid(f[t]), sigmoid(-f[t])
            p = np.minimum(a, g)
            xt = np.where(g == 0.0, 0.0, x[t])  # a gate of +inf does not look at x
            trace.append((t, a, g, p, h, m, err, xt))
            prev = np.where(a == 0.0, 0.0, h)
            fin = np.where(np.isfinite(f[t]), np.abs(f[t]), 0.0)
            step = ((2 * fin + 8) * U * p + FLUSH) * (np.abs(xt) + m)
            h, m = a * prev + g * xt, a * m + g * np.abs(xt)
            err = a * err + step + 6 * U * m
            v["y"][t], w["y"][t] = h, err
        v["h_last"][s], w["h_last"][s] = h, err
        if grad_y is None:
            continue
        q = np.zeros(c) if grad_h_last is None else grad_h_last[s].astype(np.float64)  # what comes back from t + 1
        mq, eq = np.abs(q), np.zeros(c)
        for t, a, g, p, h, m, err, xt in reversed(trace):
            fin = np.where(np.isfinite(f[t]), np.abs(f[t]), 0.0)
            rel = (2 * fin + 8) * U
            total = q + grad_y[t]
            mt, et = mq + np.abs(grad_y[t]), eq + 2 * U * (mq + np.abs(grad_y[t]))
            v["grad_x"][t] = g * total
            w["grad_x"][t] = g * et + mt * (p * rel + FLUSH) + 3 * U * g * mt
            v["grad_f"][t] = total * (h - xt) * a * g
            w["grad_f"][t] = a * g * (et * (m + np.abs(xt)) + mt * (err + U * (m + np.abs(xt))) + mt * (m + np.abs(xt)) * (2 * rel + 6 * U)) + FLUSH * mt * (m + np.abs(xt))
            q, mq, eq = a * total, a * mt, a * et + (rel * p + FLUSH) * mt + 4 * U * a * mt
        v["grad_h0"][s], w["grad_h0"][s] = q, eq
    return v, w


def _adds(d):
    """Additions in a row behind each other: up to 16 terms a lane, a tree over the lanes and waves, and what little code adds."""
    return min(d / 64, 64.0) + 14.0


def _norm(x, ein, kind, eps):
    """Normalised row, its error for an error `ein` of the row, 1 / deviation and that factor's relative error."""
    d = x.shape[-1]
    mean = x.mean(-1, keepdims=True) if kind == "layer" else np.zeros_like(x[..., :1])
    rho = 1.0 / np.sqrt(((x - mean) ** 2).mean(-1, keepdims=True) + eps)
    hat = (x - mean) * rho
    off = _adds(d) * U * np.abs(x).mean(-1, keepdims=True) + ein.mean(-1, keepdims=True) if kind == "layer" else 0.0 * rho  # of the mean
    rel = (_adds(d) / 2 + 8) * U + rho * (np.abs(hat) * ein).mean(-1, keepdims=True) + (rho * off) ** 2
    return hat, rho * (ein + off + 2 * U * np.abs(x - mean)) + np.abs(hat) * rel, rho, rel


def _norm_back(g, eg, hat, ehat, rho, rel, kind):
    """Gradient of the row for the gradient g of the normalised row, and its error."""
    d = g.shape[-1]
    m = lambda t: t.mean(-1, keepdims=True)  # noqa: E731
    s, es = (m(g), m(eg) + _adds(d) * U * m(np.abs(g))) if kind == "layer" else (0.0, 0.0)
    q, eq = m(g * hat), m(eg * np.abs(hat) + np.abs(g) * ehat) + (_adds(d) + 1) * U * m(np.abs(g * hat))
    size = np.abs(g) + np.abs(s) + np.abs(hat * q)
    return rho * (g - s - hat * q), rho * (eg + es + np.abs(hat) * eq + ehat * np.abs(q) + size * (rel + 4 * U))


def block_norm(y, residual, gate, *, kind, act, scale=None, post=True, post_weight=None, post_bias=None, pre=True, pre_weight=None, pre_bias=None,
               eps=1e-5, grad_residual=None, grad_normed=None):
    """Values / bounds: residual, normed, and with either gradient grad_y, grad_gate, grad_residual and the vectors' sums."""
    f64 = lambda a: None if a is None else a.astype(np.float64)  # noqa: E731
    y, residual, gate, gr, gn = map(f64, (y, residual, gate, grad_residual, grad_normed))
    shape = (y if y is not None else residual).shape
    d = shape[-1]
    one, zero, none = np.ones(d), np.zeros(d), np.zeros(shape)
    vec = lambda t, other: other if t is None else t.astype(np.float64)  # noqa: E731
    sc, pw, pb, qw, qb = vec(scale, one), vec(post_weight, one), vec(post_bias, zero), vec(pre_weight, one), vec(pre_bias, zero)
    r2, e2 = (none if residual is None else residual), none
    ab = np.abs
    if y is not None:
        if post:
            hat, eh, rho, rel = _norm(y, none, kind, eps)
            u, eu = hat * pw + pb, eh * ab(pw) + 2 * U * (ab(hat * pw) + ab(pb))
        else:
            u, eu = y, none
        a, slope, ea, esl = np.ones(shape), none, none, none
        if gate is not None and act == "identity":
            a, slope = gate, np.ones(shape)
        elif gate is not None:
            s = sigmoid(gate)
            es = s * (1 - s) * (2 * ab(gate) + 4) * U + 4 * U * s
            if act == "sigmoid":
                a, ea, slope, esl = s, es, s * (1 - s), es * (1 - s) + s * (es + U) + 2 * U * s * (1 - s)
            else:
                a, ea, slope = gate * s, ab(gate) * es + 2 * U * ab(gate * s), s * (1 + gate * (1 - s))
                esl = es * (1 + ab(gate) * (1 - s)) + s * ab(gate) * (es + U) + 4 * U * (s + ab(gate) * s * (1 - s))
        v, ev = a * u, ab(a) * eu + ea * ab(u) + 2 * U * ab(a * u)
        e2 = ab(sc) * ev + 2 * U * (ab(r2) + ab(sc * v))
        r2 = r2 + sc * v
    out, err = {"residual": r2}, {"residual": e2}
    if pre:
        hat2, eh2, rho2, rel2 = _norm(r2, e2, kind, eps)
        out["normed"], err["normed"] = hat2 * qw + qb, eh2 * ab(qw) + 2 * U * (ab(hat2 * qw) + ab(qb))
    if gr is None and gn is None:
        return out, err
    add = (int(np.prod(shape[:-1])) + 8) * U  # a column's sum, term after term at worst
    col = lambda t: t.reshape(-1, d).sum(0)  # noqa: E731
    total, et = none if gr is None else gr, none
    if pre and gn is not None:
        back, eb = _norm_back(gn * qw, U * ab(gn * qw), hat2, eh2, rho2, rel2, kind)
        total, et = total + back, eb + U * (ab(total) + ab(back))
        out["grad_pre_weight"], err["grad_pre_weight"] = col(gn * hat2), col(ab(gn) * (eh2 + add * ab(hat2)))
        out["grad_pre_bias"], err["grad_pre_bias"] = col(gn), col(ab(gn)) * add
    out["grad_residual"], err["grad_residual"] = total, et
    if y is None:
        return out, err
    out["grad_scale"], err["grad_scale"] = col(total * v), col(et * ab(v) + ab(total) * (ev + add * ab(v) + 2 * U * ab(v)))
    gv, egv = total * sc, et * ab(sc) + U * ab(total * sc)
    out["grad_gate"], err["grad_gate"] = gv * u * slope, egv * ab(u * slope) + ab(gv) * (eu * ab(slope) + esl * ab(u) + 4 * U * ab(u * slope))
    gu, egu = gv * a, egv * ab(a) + ab(gv) * (ea + 2 * U * ab(a))
    if not post:
        out["grad_y"], err["grad_y"] = gu, egu
        return out, err
    out["grad_post_weight"], err["grad_post_weight"] = col(gu * hat), col(egu * ab(hat) + ab(gu) * (eh + add * ab(hat)))
    out["grad_post_bias"], err["grad_post_bias"] = col(gu), col(egu + add * ab(gu))
    out["grad_y"], err["grad_y"] = _norm_back(gu * pw, egu * ab(pw) + U * ab(gu * pw), hat, eh, rho, rel, kind)
    return out, err


def token_logprobs(z, tokens=None, ignore=-100, n_top=0, grad_logprob=None, grad_entropy=None):
    """z [n, V].  Values / bounds: logprob, entropy, lse parts, top_ids, top_logprob, and with a gradient grad_logits.
    A sum over V classes is at most V / 64 terms after each other and a tree."""
    z = z.astype(np.float64)
    n, classes = z.shape
    live = np.ones(n, bool) if tokens is None else tokens != ignore
    bad = np.isnan(z).any(1) | (z == np.inf).any(1)
    m = np.where(bad, 0.0, np.nan_to_num(z, nan=0.0, posinf=0.0, neginf=-np.inf).max(1))
    empty = (z == -np.inf).all(1)
    m0 = np.where(empty, 0.0, m)[:, None]
    with np.errstate(all="ignore"):
        dd = np.where(bad[:, None], 0.0, z - m0)
        e = np.exp(dd)
        s = np.where(empty, 1.0, e.sum(1))[:, None]
        logp = np.where(empty[:, None], -np.inf, dd - np.log(s))
        p = np.where(empty[:, None], 0.0, e / s)
        plogp = np.where(p > 0, p * np.where(p > 0, logp, 0.0), 0.0)
    entropy = -plogp.sum(1)
    sums = (classes / 64 + 24) * U
    elp = np.where(np.isfinite(logp), sums + 4 * U * np.abs(np.where(np.isfinite(dd), dd, 0.0)) + 4 * U * np.log(s), 0.0)
    eent = sums * (2 + 2 * entropy + np.log(s)[:, 0])
    logp, entropy = np.where(bad[:, None], np.nan, logp), np.where(bad, np.nan, entropy)
    out, err = {"entropy": np.where(live, entropy, 0.0)}, {"entropy": np.where(live, eent, 0.0)}
    at = np.zeros(n, int) if tokens is None else np.where(live, tokens, 0).astype(np.int64)
    wrong = (at < 0) | (at >= classes)
    at, rows = np.where(wrong, 0, at), np.arange(n)
    if tokens is not None:
        out["logprob"] = np.where(live, np.where(wrong, np.nan, logp[rows, at]), 0.0)
        err["logprob"] = elp[rows, at]
    if n_top:
        key = np.where(np.isnan(z), np.inf, z)
        ids = np.stack([np.lexsort((np.arange(classes), ~np.isnan(z[i]), -key[i]))[:n_top] for i in range(n)]) if n else np.zeros((0, n_top), int)
        out["top_ids"] = np.where(live[:, None], ids, -1)
        out["top_logprob"] = np.where(live[:, None], np.take_along_axis(logp, ids, 1), 0.0)
        err["top_logprob"] = np.take_along_axis(elp, ids, 1)
    if grad_logprob is not None or grad_entropy is not None:
        gl = np.zeros(n) if grad_logprob is None else grad_logprob.astype(np.float64)
        gh = np.zeros(n) if grad_entropy is None else grad_entropy.astype(np.float64)
        lp0, ent0 = np.where(p > 0, logp, 0.0), entropy[:, None]
        g = -p * (gl[:, None] + gh[:, None] * (lp0 + ent0))
        size = p * (np.abs(gl)[:, None] + np.abs(gh)[:, None] * (np.abs(lp0) + ent0))
        w = size * (elp + (2 * np.abs(lp0) + 8) * U) + p * np.abs(gh)[:, None] * (elp + eent[:, None]) + 2 * U * size
        if grad_logprob is not None:
            g[rows, at] += np.where(wrong, 0.0, gl)
            w[rows, at] += 2 * U * np.abs(gl)
        gone = ~live | empty
        out["grad_logits"] = np.where(gone[:, None], 0.0, np.where((bad | (wrong & (grad_logprob is not None)))[:, None], np.nan, g))
        err["grad_logits"] = np.where(gone[:, None], 0.0, w)
    return out, err
