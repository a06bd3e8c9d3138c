"""One Adam / AdamW step with 8-bit moments in 64 bits with numpy, from its definition."""
import numpy as np


def blocks(x):
    return np.concatenate([x, np.zeros(-x.size % 256)]).reshape(-1, 256)


def encode(x, second):
    """fp64 [n] -> (integer codes [n], fp32 scales)"""
    levels, power = (255, 4) if second else (127, 2)
    b = blocks(x)
    s = np.abs(b).max(1).astype(np.float32)
    s = np.where(s < np.finfo(np.float32).tiny, np.float32(0), s)
    s = np.where(np.isfinite(s), s, np.float32(np.nan))
    q = np.zeros(b.shape)
    for i in range(len(b)):
        if s[i] > 0:
            q[i] = np.sign(b[i]) * np.minimum(levels, np.rint(levels * (np.abs(b[i]) / np.float64(s[i])) ** (1 / power)))
            if second:
                q[i] = np.where((b[i] > 0) & (q[i] < 1), 1, q[i])
    return q.reshape(-1)[:x.size], s


def decode(q, s, second):
    levels, power = (255, 4) if second else (127, 2)
    b = blocks(np.asarray(q, np.float64))
    return (np.sign(b) * (np.abs(b) / levels) ** power * np.asarray(s, np.float64)[:, None]).reshape(-1)[:np.size(q)]


def step(w, g, m, v, t, lr, b1, b2, eps, wd, adamw, inv_scale=1.0):
    """(new w, m', v') in fp64; m and v are values, m' and v' not yet coded."""
    w, g = w.astype(np.float64), (g.astype(np.float32) * np.float32(inv_scale)).astype(np.float64)
    if adamw:
        w = w * (1 - lr * wd)
    elif wd:
        g = g + wd * w
    m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    return w - lr / (1 - b1**t) * m / (np.sqrt(v / (1 - b2**t)) + eps), m, v
