"""64-bit definitions of the token-policy operators with bounds on what the fp32 kernels may be off.

Every function returns values and error bounds of the same shape.  U = 2^-24 is half a step of fp32; a
result stored in type t is off by another finfo(t).eps / 2 of its value (and by half the smallest
subnormal of fp16 near zero).  The bounds count the roundings on the way to each value, they are not
fitted: an exponential of argument y through exp2 is off by (|y| + 3) U relative (the argument's own
rounding, the constant's, the instruction's), a reciprocal by 2 U, products and sums by U each."""
import numpy as np
import torch

U = 2.0 ** -24


def stored(value, bound, dtype):
    """The bound after one rounding of the result to `dtype`."""
    half = torch.finfo(dtype).eps / 2
    tiny = 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -126
    return bound * (1 + half) + np.abs(value) * half + tiny


def check(got, value, bound, dtype, what):
    g = got.detach().double().cpu().numpy()
    assert g.shape == value.shape, (what, g.shape, value.shape)
    nan = np.isnan(value)
    assert np.array_equal(np.isnan(g), nan), f"{what}: NaN in other places"
    inf = np.isinf(value)
    assert np.array_equal(g[inf], value[inf]), f"{what}: infinities"
    ok = ~(nan | inf)
    far = np.abs(g[ok] - value[ok]) - stored(value[ok], bound[ok] if np.ndim(bound) else bound, dtype)
    if far.size and far.max() > 0:
        at = np.argmax(far)
        raise AssertionError(f"{what}: got {g[ok][at]!r}, want {value[ok][at]!r}, "
                             f"off by {far[at]:.3g} more than the bound ({int((far > 0).sum())} values)")


# ------------------------------------------------------------------------------------------ embedding
def embed(weight, tokens, scale):
    w, t = np.asarray(weight, np.float64), np.asarray(tokens)
    out = np.full(t.shape + (w.shape[1],), np.nan)
    out[t == -1] = 0.0
    ok = (t >= 0) & (t < w.shape[0])
    out[ok] = np.float64(np.float32(scale)) * w[t[ok]]
    return out, 2 * U * np.abs(np.nan_to_num(out))


def embed_grad(d_out, tokens, vocab, scale):
    d, t = np.asarray(d_out, np.float64).reshape(-1, np.shape(d_out)[-1]), np.asarray(tokens).reshape(-1)
    out, mag, count = (np.zeros((vocab, d.shape[1])) for _ in range(3))
    for i, v in enumerate(t):
        if 0 <= v < vocab:
            out[v] += d[i]
            mag[v] += np.abs(d[i])
            count[v] += 1
    s = np.float64(np.float32(scale))
    return s * out, np.abs(s) * mag * (count + 2) * U


# ------------------------------------------------------------------------------------------ recurrence
def _sigmoid(z):
    e = np.exp(-np.abs(z))
    r = 1.0 / (1.0 + e)
    return np.where(z >= 0, r, e * r), np.where(z >= 0, e * r, r)


def recurrence(x, g, h0, resets, lengths, logits, reverse, d_h=None, d_last=None):
    """{name: (value, bound)} for h, last and, with d_h / d_last, d_x, d_g, d_h0."""
    x, g = np.asarray(x, np.float64), np.asarray(g, np.float64)
    b, t, d = x.shape
    h0 = np.zeros((b, d)) if h0 is None else np.asarray(h0, np.float64)
    out = {k: (np.zeros_like(x), np.zeros_like(x)) for k in ("h", "d_x", "d_g")}
    out.update({k: (np.zeros((b, d)), np.zeros((b, d))) for k in ("last", "d_h0")})
    for i in range(b):
        n = t if lengths is None else min(max(int(lengths[i]), 0), t)
        order = range(n - 1, -1, -1) if reverse else range(n)
        h, mag, err = h0[i], np.abs(h0[i]), np.zeros(d)
        before, e_before, forgot = [], [], []
        for s in order:
            r = bool(resets is not None and resets[i][s])
            if r:
                h, mag, err = np.zeros(d), np.zeros(d), np.zeros(d)
            before.append(h)
            e_before.append(err)
            forgot.append(r)
            if logits:
                a, keep = _sigmoid(g[i, s])
                step = (np.abs(g[i, s]) + 8) * U       # the gate, and the products and sums of one step
                into, e_into = keep * x[i, s], (np.abs(g[i, s]) + 8) * U * np.abs(keep * x[i, s])
            else:
                a, keep, step = g[i, s], np.ones(d), 4 * U
                into, e_into = x[i, s], 0.0
            h_new = into if r else a * h + into
            mag_new = np.abs(into) + np.abs(a) * mag
            # joining lanes, waves and tiles adds up to 32 roundings to a path once per tile of at least 32 steps
            err = np.abs(a) * (err + (step + 2 * U) * mag) + e_into + 40 * U * np.abs(into)
            h, mag = h_new, mag_new
            out["h"][0][i, s], out["h"][1][i, s] = h, err
        out["last"][0][i], out["last"][1][i] = h, err
        if d_h is None and d_last is None:
            continue
        c = np.zeros(d) if d_last is None else np.asarray(d_last, np.float64)[i]
        c_mag, c_err = np.abs(c), np.zeros(d)
        for k in range(n - 1, -1, -1):
            s = list(order)[k] if n < 64 else (n - 1 - k if reverse else k)
            dh = np.zeros(d) if d_h is None else np.asarray(d_h[i, s], np.float64)
            z = np.abs(g[i, s])
            grad, g_mag = c + dh, c_mag + np.abs(dh)
            g_err = c_err + 2 * U * g_mag + 40 * U * np.abs(dh)
            if logits:
                a, keep = _sigmoid(g[i, s])
                gate = (z + 8) * U
                diff = before[k] - x[i, s]
                e_diff = e_before[k] + 2 * U * (np.abs(before[k]) + np.abs(x[i, s]))
                out["d_x"][0][i, s] = keep * grad
                out["d_x"][1][i, s] = keep * (g_err + (gate + U) * np.abs(grad))
                out["d_g"][0][i, s] = a * keep * grad * diff
                out["d_g"][1][i, s] = a * keep * (g_err * np.abs(diff) + np.abs(grad) * e_diff
                                                  + (2 * gate + 4 * U) * np.abs(grad * diff))
            else:
                a, gate = g[i, s], 0.0
                out["d_x"][0][i, s], out["d_x"][1][i, s] = grad, g_err
                out["d_g"][0][i, s] = grad * before[k]
                out["d_g"][1][i, s] = g_err * np.abs(before[k]) + np.abs(grad) * e_before[k] + 2 * U * np.abs(grad * before[k])
            if forgot[k]:
                c, c_mag, c_err = np.zeros(d), np.zeros(d), np.zeros(d)
            else:
                c_err = np.abs(a) * (g_err + (gate + 4 * U) * g_mag)
                c, c_mag = a * grad, np.abs(a) * g_mag
        out["d_h0"][0][i], out["d_h0"][1][i] = c, c_err
    return out


# ------------------------------------------------------------------------------------------ log probabilities
def log_probs(logits, actions, mask, temperature, top, g_lp=None, g_h=None):
    """Dict of (value, bound); "top" holds the exact indices."""
    l = np.asarray(logits, np.float64)
    rows, width = l.shape
    t32 = np.float64(np.float32(temperature))
    res = {"log_prob": (np.zeros(rows), np.zeros(rows)), "entropy": (np.zeros(rows), np.zeros(rows)),
           "top": np.full((rows, top), -1, np.int64),
           "top_log_prob": (np.full((rows, top), -np.inf), np.zeros((rows, top))),
           "d_logits": (np.zeros((rows, width)), np.zeros((rows, width)))}
    for r in range(rows):
        on = np.ones(width, bool) if mask is None else ~np.asarray(mask, bool)[r]
        on = on & ~np.isneginf(l[r])
        a = int(actions[r])
        outside = a != -1 and not 0 <= a < width
        idx = np.nonzero(on)[0]
        z = l[r][idx] / t32
        key = np.where(np.isnan(l[r][idx]), np.inf, l[r][idx])
        nan_first = np.isnan(l[r][idx])
        order = idx[np.lexsort((idx, -key, ~nan_first))][:top]
        res["top"][r, :len(order)] = order
        bad = bool(np.isnan(z).any() or np.isposinf(z).any())
        if bad:
            res["entropy"][0][r] = np.nan
            res["log_prob"][0][r] = 0.0 if a == -1 else np.nan
            res["top_log_prob"][0][r, :len(order)] = np.nan
            res["d_logits"][0][r, idx] = np.nan
            continue
        if len(idx) == 0:
            res["log_prob"][0][r] = 0.0 if a == -1 else np.nan if outside else -np.inf
            continue
        m = z.max()
        e = np.exp(z - m)
        s = e.sum()
        log_s, p = np.log(s), e / s
        dist = np.abs(z - m)
        mean_dist = (p * dist).sum()
        # running sums: as many roundings as a lane adds values, and those of the joins; an exponential is
        # off by its distance from the maximum, which its own size makes up for (y exp(-y) < 1)
        sums = (width / 16 + 24) * U
        e_log_s = sums + (mean_dist + 6) * U + 2 * U * log_s
        lp = z - m - log_s
        e_lp = e_log_s + 4 * U * (dist + log_s)
        ent = log_s + (p * (m - z)).sum()
        e_ent = e_log_s + sums * (mean_dist + 1) + (p * dist * (dist + 8)).sum() * U + 4 * U * (log_s + mean_dist)
        res["entropy"][0][r], res["entropy"][1][r] = ent, e_ent
        where = {j: k for k, j in enumerate(idx)}
        if a != -1:
            res["log_prob"][0][r] = np.nan if outside else lp[where[a]] if a in where else -np.inf
            if a in where:
                res["log_prob"][1][r] = e_lp[where[a]]
        for k, j in enumerate(order):
            res["top_log_prob"][0][r, k] = lp[where[j]]
            res["top_log_prob"][1][r, k] = e_lp[where[j]]
        if g_lp is None and g_h is None:
            continue
        ga = 0.0 if g_lp is None or a == -1 else float(g_lp[r])
        gh = 0.0 if g_h is None else float(g_h[r])
        if outside:
            res["d_logits"][0][r, idx] = np.nan
            continue
        if a not in where:
            ga = 0.0        # -inf whatever the logits are
        inner = ga + gh * (lp + ent)
        d = -p * inner
        e_in = np.abs(gh) * (e_lp + e_ent) + 4 * U * (np.abs(ga) + np.abs(gh) * (np.abs(lp) + ent))
        bound = p * (e_in + (e_lp + 4 * U) * np.abs(inner))
        if a in where:
            d[where[a]] += ga
            bound[where[a]] += 2 * U * (np.abs(ga) + np.abs(d[where[a]]))
        res["d_logits"][0][r, idx] = d / t32
        res["d_logits"][1][r, idx] = (bound + 4 * U * np.abs(d)) / t32
    return res
