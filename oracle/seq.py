"""float64 restatements of the sequence operators (engine/seq_ops.py), from their formulas alone.

Every function takes and returns float64 numpy arrays.  ``keep_mask`` is Philox4x32-10 of Salmon, Moraes,
Dror and Shaw (SC 2011), checked against that paper's published known answers in tests/test_seq_ops_cpu.py.
"""
import numpy as np

_M0, _M1, _W0, _W1, _LOW = 0xD2511F53, 0xCD9E8D57, 0x9E3779B9, 0xBB67AE85, 0xFFFFFFFF


def philox(counter, key, rounds=10):
    """One block: four 32-bit words from a 4-word counter and a 2-word key (Python integers)."""
    c, k = list(counter), list(key)
    for _ in range(rounds):
        a, b = _M0 * c[0], _M1 * c[2]
        c = [(b >> 32) ^ c[1] ^ k[0], b & _LOW, (a >> 32) ^ c[3] ^ k[1], a & _LOW]
        k = [(k[0] + _W0) & _LOW, (k[1] + _W1) & _LOW]
    return c


def threshold(p):
    return int(np.floor(65536.0 * p + 0.5))


def keep_mask(n, p, seed, step, first=0):
    """For elements first .. first + n, first a multiple of 8."""
    out = np.empty((n + 7) // 8 * 8, bool)
    key = (seed & _LOW, seed >> 32 & _LOW)
    step &= 2 ** 64 - 1
    for b in range(len(out) // 8):
        at = first // 8 + b
        words = philox((at & _LOW, at >> 32, step & _LOW, step >> 32), key)
        for e in range(8):
            out[8 * b + e] = (words[e // 2] >> 16 * (e & 1) & 0xFFFF) >= threshold(p)
    return out[:n]


def dropout(x, residual, p, seed, step):
    t = threshold(p)
    keep = keep_mask(x.size, p, seed, step).reshape(x.shape)
    y = np.where(keep, x, 0.0) * (65536.0 / (65536 - t) if t < 65536 else 0.0)
    return y if residual is None else y + residual


def embedding(idx, w, scale):
    ok = (idx >= 0) & (idx < len(w))
    return np.where(ok[..., None], w[np.where(ok, idx, 0)] * scale, 0.0)


def embedding_grad(idx, g, rows, scale, pad=-1):
    dw = np.zeros((rows, g.shape[-1]))
    idx = idx.reshape(-1)
    ok = (idx >= 0) & (idx < rows) & (idx != pad)
    np.add.at(dw, idx[ok], g.reshape(-1, g.shape[-1])[ok] * scale)
    return dw


def rms_norm(x, residual, w, eps):
    h = x if residual is None else x + residual
    rstd = 1.0 / np.sqrt((h * h).mean(-1, keepdims=True) + eps)
    return h * rstd * w, h, rstd


def rms_norm_grad(h, w, eps, dy, dh):
    _, _, rstd = rms_norm(h, None, w, eps)
    xh, g = h * rstd, dy * w
    dx = rstd * (g - xh * (g * xh).mean(-1, keepdims=True)) + (0.0 if dh is None else dh)
    return dx, (dy * xh).reshape(-1, h.shape[-1]).sum(0)


def item_log_probs(h, w, ids, scale):
    z = h @ w.T * scale
    top = z.max(1, keepdims=True)
    lse = top[:, 0] + np.log(np.exp(z - top).sum(1))
    ok = (ids >= 0) & (ids < len(w))
    return np.where(ok, z[np.arange(len(ids)), np.where(ok, ids, 0)] - lse, 0.0), z, lse


def item_log_probs_grad(h, w, ids, scale, up):
    ok = (ids >= 0) & (ids < len(w))
    h = np.where(ok[:, None], h, 0.0)
    _, z, lse = item_log_probs(h, w, ids, scale)
    g = -np.exp(z - lse[:, None])
    g[np.arange(len(ids))[ok], ids[ok]] += 1.0
    g *= np.where(ok, up * scale, 0.0)[:, None]
    return g @ w, g.T @ h, g


def preference_loss(logp, ref, offsets, beta, smoothing):
    """With a reference, a position whose logp is +0 has no target: it takes no part, whatever ref holds there."""
    pairs = (len(offsets) - 1) // 2
    lost = (logp == 0) & ~np.signbit(logp) & (ref is not None)
    v = np.where(lost, 0.0, logp - (0.0 if ref is None else ref))
    s = np.array([v[a:b].sum() for a, b in zip(offsets[:-1], offsets[1:])])
    m = beta * (s[:pairs] - s[pairs:])
    loss = ((1 - smoothing) * np.logaddexp(0, -m) + smoothing * np.logaddexp(0, m)).mean()
    slope = beta / pairs * (smoothing * np.exp(-np.logaddexp(0, -m)) - (1 - smoothing) * np.exp(-np.logaddexp(0, m)))
    grad = np.zeros(len(logp))
    for p in range(pairs):
        grad[offsets[p]:offsets[p + 1]] = slope[p]
        grad[offsets[pairs + p]:offsets[pairs + p + 1]] = -slope[p]
    grad[lost] = 0.0
    return loss, grad
