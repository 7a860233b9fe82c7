"""The training-block operators in 64 bits, plainly, for the tests: dropout, block norms and bucketed-bias softmax
with their gradients, each returning the values and how far 32-bit arithmetic may be from them.

The bounds count roundings.  With u = 2^-24 a sum of n terms in any order is within (n - 1) u of the sum of the
terms' magnitudes; the kernels add at most 16 terms a thread and fold them in trees of depth 12, so a row sum is
within C u of its magnitudes with C = 64, which leaves room for the few products around it.  A result stored in 16
bits adds half a unit in its last place."""
import math

import numpy as np

U = 2.0 ** -24
C = 64.0
HALF_ULP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"f32": 0.0, "f16": 2.0 ** -25, "bf16": 0.0}


def philox_words(seed, offset, stream, n, domain=1):
    """The first n words from block `offset` on: Philox4x32-10 of (lo b, hi b, stream, domain)."""
    m = np.uint64(0xFFFFFFFF)
    b = (np.arange((n + 3) // 4, dtype=np.uint64) + np.uint64(offset % 2 ** 64))
    c = [b & m, b >> np.uint64(32), np.full_like(b, stream), np.full_like(b, domain)]
    k0, k1 = seed % 2 ** 32, (seed % 2 ** 64) >> 32
    for _ in range(10):
        p0, p1 = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(p1 >> np.uint64(32)) ^ c[1] ^ np.uint64(k0), p1 & m, (p0 >> np.uint64(32)) ^ c[3] ^ np.uint64(k1), p0 & m]
        k0, k1 = (k0 + 0x9E3779B9) % 2 ** 32, (k1 + 0xBB67AE85) % 2 ** 32
    return np.stack(c, 1).reshape(-1)[:n]


def keep_mask(p, seed, offset, stream, shape):
    n = int(np.prod(shape))
    return (philox_words(seed, offset, stream, n) >= np.uint64(math.floor(p * 2 ** 32))).reshape(shape)


def drop_factor(drop, shape):
    """drop: None or (p, seed, offset, stream)."""
    if drop is None:
        return np.ones(shape)
    return keep_mask(drop[0], *drop[1:], shape) / (1.0 - drop[0])


def stored(value, mag, dtype):
    """Tolerance of a value of 32-bit error C u mag, stored as `dtype`."""
    err = C * U * mag
    return err + (HALF_ULP[dtype] * (np.abs(value) + err) + TINY[dtype])


# ---- block norms ------------------------------------------------------------------------
def stats(v, layer, eps):
    mean = v.mean(1) if layer else np.zeros(v.shape[0])
    rstd = 1.0 / np.sqrt(((v - mean[:, None]) ** 2).mean(1) + eps)
    return mean, rstd


def block_norm(x, y, w_post, b_post, gate, w_pre, b_pre, layer, eps, alpha, drop, post, pre):
    """{name: (value, magnitude)}; a magnitude bounds the terms that a value is the sum of."""
    out = {}

    def normed(v, vmag, w, b, name):
        mean, rstd = stats(v, layer, eps)
        hat = (v - mean[:, None]) * rstd[:, None]
        # v's own error, the mean's, and rstd's relative one (of its mean square, which v's error moves too)
        spread = (vmag + np.abs(v).mean(1)[:, None] + vmag.mean(1)[:, None]) * rstd[:, None] + np.abs(hat) * (
            1 + (vmag * np.abs(hat)).mean(1)[:, None] * rstd[:, None])
        out["stats_" + name] = (np.stack([mean, rstd], 1) if layer else rstd[:, None],
                                np.stack([vmag.mean(1) + np.abs(v).mean(1),
                                          rstd * (1 + (vmag * np.abs(hat)).mean(1) * rstd)], 1)[:, 0 if layer else 1:])
        n = hat * w
        return (n + b if b is not None else n), spread * np.abs(w) + (np.abs(b) if b is not None else 0)

    h, hmag = x, np.abs(x)
    if y is not None:
        n, nmag = y, np.abs(y)
        if post:
            n, nmag = normed(y, np.abs(y) * 0, w_post, b_post, "post")
        if gate is not None:
            g = np.repeat(gate, x.shape[0] // gate.shape[0], 0)
            n, nmag = n * g, nmag * np.abs(g)
        f = drop_factor(drop, x.shape)
        h, hmag = alpha * x + n * f, np.abs(alpha * x) + (np.abs(n) + nmag) * f
        out["h"] = (h, hmag)
    if pre:
        out["u"] = normed(h, hmag if y is not None else hmag * 0, w_pre, b_pre, "pre")
        out["u"] = (out["u"][0], out["u"][1] + np.abs(out["u"][0]))
    return out


def block_norm_grad(dh, du, h, y, w_post, b_post, gate, w_pre, stats_post, stats_pre, layer, alpha, drop, bias):
    """As block_norm; statistics are given (the kernel reads them)."""
    out = {}

    def hat(v, s):
        return (v - (s[:, :1] if layer else 0.0)) * s[:, -1:]

    def hat_mag(v, s):
        return (np.abs(v) + (np.abs(s[:, :1]) if layer else 0.0)) * s[:, -1:]

    def back(a, amag, z, zmag, s):
        k, kmag = (a * z).mean(1)[:, None], (amag * zmag).mean(1)[:, None]
        m, mmag = (a.mean(1)[:, None], amag.mean(1)[:, None]) if layer else (0.0, 0.0)
        return s[:, -1:] * (a - m - z * k), s[:, -1:] * (amag + mmag + zmag * kmag)

    def column(v, mag, groups=1):
        v, mag = v.reshape(groups, -1, v.shape[1]), mag.reshape(groups, -1, v.shape[1])
        # a column's terms are added one row after the other
        return v.sum(1), mag.sum(1) * (1 + v.shape[1] / C)

    g, gmag = (dh, np.abs(dh)) if dh is not None else (0.0, 0.0)
    if du is not None:
        z, zmag = hat(h, stats_pre), hat_mag(h, stats_pre)
        out["dw_pre"] = tuple(a[0] for a in column(du * z, np.abs(du) * zmag))
        if bias:
            out["db_pre"] = tuple(a[0] for a in column(du, np.abs(du)))
        t, tmag = back(du * w_pre, np.abs(du * w_pre), z, zmag, stats_pre)
        g, gmag = g + t, gmag + tmag
    a = alpha if dh is not None else 1.0
    out["dx"] = (a * g, np.abs(a) * gmag)
    if dh is not None:
        f = drop_factor(drop, g.shape)
        d, dmag = g * f, gmag * f
        post = stats_post is not None
        if post:
            z, zmag = hat(y, stats_post), hat_mag(y, stats_post)
        if gate is not None:
            n, nmag = (z * w_post, zmag * np.abs(w_post)) if post else (y, np.abs(y))
            if b_post is not None:
                n, nmag = n + b_post, nmag + np.abs(b_post)
            out["dgate"] = column(d * n, dmag * nmag, gate.shape[0])
            gr = np.repeat(gate, d.shape[0] // gate.shape[0], 0)
            d, dmag = d * gr, dmag * np.abs(gr)
        if post:
            out["dw_post"] = tuple(v[0] for v in column(d * z, dmag * zmag))
            if bias:
                out["db_post"] = tuple(v[0] for v in column(d, dmag))
            d, dmag = back(d * w_post, dmag * np.abs(w_post), z, zmag, stats_post)
        out["dy"] = (d, dmag)
    return out


# ---- bucketed-bias softmax -------------------------------------------------------------------
def bucket(rel, thresholds, both):
    n = abs(rel) if both else max(-rel, 0)
    b = sum(t <= n for t in thresholds)
    return b + len(thresholds) + 1 if both and rel > 0 else b


def masks_and_bias(shape, table, thresholds, both, causal, lengths, offsets):
    """visible [b, 1, q, k] and the bias [b, h, q, k] with its buckets."""
    nb, _, nq, nk = shape
    off = np.zeros(nb, np.int64) if offsets is None else np.asarray(offsets, np.int64)
    rel = np.arange(nk)[None, None] - np.arange(nq)[None, :, None] - off[:, None, None]
    lo, hi = (int(rel.min()), int(rel.max())) if rel.size else (0, 0)
    far = max(thresholds) + 1
    lut = {r: bucket(r, thresholds, both) for r in range(max(lo, -far), min(hi, far) + 1)}
    ids = np.vectorize(lambda r: lut[max(-far, min(far, r))] if max(-far, min(far, r)) in lut
                       else bucket(r, thresholds, both), otypes=[np.int64])(rel)
    seen = np.ones(rel.shape, bool)
    if lengths is not None:
        seen &= np.arange(nk)[None, None] < np.asarray(lengths)[:, None, None]
    if causal:
        seen &= rel <= 0
    return seen[:, None], np.moveaxis(table[ids], 3, 1), ids


def _logits(s, table, thresholds, both, scale, causal, lengths, offsets):
    seen, bias, ids = masks_and_bias(s.shape, table, thresholds, both, causal, lengths, offsets)
    with np.errstate(invalid="ignore", over="ignore"):
        l = np.where(seen, s * scale + bias, -np.inf)
    lmag = np.where(seen & np.isfinite(l), np.abs(np.where(seen, s, 0) * scale) + np.abs(bias), 0)
    return seen, l, lmag, ids


def bias_softmax(s, table, thresholds, both, scale, causal, lengths, offsets, drop):
    """p, its error bound; lse, its error bound.  exp's argument errs by 4 u of the logit's terms (and of the row's
    largest, through the maximum), exp itself by 4 u, the sum as a row sum."""
    seen, l, lmag, _ = _logits(s, table, thresholds, both, scale, causal, lengths, offsets)
    top = l.max(3, keepdims=True, initial=-np.inf)
    top = np.where(np.isfinite(top), top, 0.0)
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        e = np.exp(l - top)
        total = e.sum(3, keepdims=True)
        p = np.where(seen & (total != 0), e / total, 0.0)
        lse = (np.log(total) + top)[..., 0]
    rowmag = lmag.max(3, keepdims=True, initial=0)
    f = drop_factor(drop, s.shape)
    rel = (8 * (lmag + rowmag) + C) * U
    return p * f, p * f * rel + 2.0 ** -120, lse, (8 * rowmag[..., 0] + C) * U


def bias_softmax_grad(s, dp, lse, table, thresholds, both, scale, causal, lengths, offsets, drop):
    seen, l, lmag, ids = _logits(s, table, thresholds, both, scale, causal, lengths, offsets)
    with np.errstate(invalid="ignore", over="ignore"):
        p = np.where(seen & (l > -np.inf), np.exp(l - np.where(np.isfinite(lse), lse, 0)[..., None]), 0.0)
    d = np.where(seen, dp, 0) * drop_factor(drop, s.shape)
    dl = p * (d - (p * d).sum(3, keepdims=True))
    # P errs by `rel` of itself, so does the sum of P d of its magnitudes
    rel = (8 * (lmag + np.abs(np.where(np.isfinite(lse), lse, 0))[..., None]) + C) * U
    mag = p * (np.abs(d) + (p * np.abs(d)).sum(3, keepdims=True))
    err = mag * (2 * rel.max(3, keepdims=True, initial=0)) + 2.0 ** -120
    n_buckets = (len(thresholds) + 1) * (2 if both else 1)
    dtable, terr = np.zeros((n_buckets, s.shape[1])), np.zeros((n_buckets, s.shape[1]))
    rows = s.shape[0] * s.shape[2]
    for h in range(s.shape[1]):
        np.add.at(dtable[:, h], ids, dl[:, h])
        np.add.at(terr[:, h], ids, err[:, h] + mag[:, h] * (C + rows) * U)
    return dl * scale, err * abs(scale), dtable, terr
