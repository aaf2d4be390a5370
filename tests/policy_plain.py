"""Plain forms in 64 bits of the learned policy's operators, for the tests: straight from the formulas, in numpy."""
import numpy as np

HALF_STEP = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}          # of a rounding to nearest, relative to the value
FLT_MAX = float(np.finfo(np.float32).max)
TINY = {"f32": 2.0 ** -126, "bf16": 2.0 ** -126, "f16": 2.0 ** -24}             # below the normal numbers: one step


def logprobs(x, taken=None, legal=None, scale=1.0, top=0):
    """x (rows, actions) float64 -> logprob, entropy, top actions, top logprobs, log p (rows, actions)."""
    x = np.array(x, np.float64)
    n, v = x.shape
    if legal is not None:
        x = np.where(np.broadcast_to(legal, x.shape) != 0, x, -np.inf)
    logp, h = np.full((n, v), -np.inf), np.zeros(n)
    lp, ta, tl = np.zeros(n), np.full((n, top), -1, np.int32), np.full((n, top), -np.inf)
    for r in range(n):
        row = x[r]
        if np.isnan(row).any() or (row == np.inf).any():
            logp[r], h[r], tl[r], lp[r] = np.nan, np.nan, np.nan, np.nan
            continue
        there = row > -np.inf
        if there.any():
            d = row - row.max()
            d = np.where(d < -FLT_MAX, -np.inf, d) * scale                   # results are floats: what passes their range is infinite
            d = np.where(d < -FLT_MAX, -np.inf, d)
            s = np.exp(d).sum()
            logp[r] = d - np.log(s)
            p = np.exp(logp[r])
            h[r] = -(p[p > 0] * logp[r][p > 0]).sum()
            order = np.lexsort((np.arange(v), -row))[:top]
            order = order[there[order]]
            ta[r, :len(order)], tl[r, :len(order)] = order, logp[r][order]
        if taken is not None:
            lp[r] = logp[r][taken[r]] if 0 <= taken[r] < v else 0.0
    return lp, h, ta, tl, logp


def gradient(x, taken, gl, gh, legal=None, scale=1.0):
    _lp, h, _a, _t, logp = logprobs(x, taken, legal, scale)
    n, v = logp.shape
    p = np.exp(logp)
    g = np.zeros((n, v))
    for r in range(n):
        a = taken[r] if taken is not None and 0 <= taken[r] < v else -1
        l = gl[r] if gl is not None and a >= 0 else 0.0
        e = gh[r] if gh is not None else 0.0
        if np.isnan(h[r]):
            g[r] = np.nan
        elif (logp[r] > -np.inf).any():
            lq = np.where(p[r] > 0, logp[r], 0.0)
            g[r] = -p[r] * (l + e * (lq + h[r]))
            if a >= 0:
                g[r, a] += l
            g[r] *= scale
    return np.where(np.broadcast_to(legal, g.shape) != 0, g, 0.0) if legal is not None else g


def philox(quads, step, seed, tag):
    """Philox4x32-10 of the counters (quad, step) under the key of the seed: (quads, 4) words."""
    u = np.uint64
    low = u(0xFFFFFFFF)
    q = np.asarray(quads, np.uint64)
    c = [q & low, q >> u(32), np.full_like(q, step & 0xFFFFFFFF), np.full_like(q, step >> 32)]
    k = [seed & 0xFFFFFFFF, (seed >> 32) ^ tag]
    for _ in range(10):
        m0, m1 = c[0] * u(0xD2511F53), c[2] * u(0xCD9E8D57)
        c = [(m1 >> u(32)) ^ c[1] ^ u(k[0]), m1 & low, (m0 >> u(32)) ^ c[3] ^ u(k[1]), m0 & low]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return np.stack(c, 1)


E4M3 = np.array([0.0] + [(i % 8) * 2.0 ** -9 if i < 8 else (1 + (i % 8) / 8) * 2.0 ** (i // 8 - 7) for i in range(1, 127)])      # what the codes 0 .. 126 stand for


def adamw(w, g, m, v, step, lr, decay, clip=1.0, beta1=0.9, beta2=0.999, eps=1e-8, lr_scale=1.0):
    """One step in 64 bits: w, m, v as they are after it; `step`: of this one, from 1."""
    g = g * clip
    m = beta1 * m + (1 - beta1) * g
    v = beta2 * v + (1 - beta2) * g * g
    return w - lr * lr_scale * (decay * w + m / (1 - beta1 ** step) / (np.sqrt(v / (1 - beta2 ** step)) + eps)), m, v
