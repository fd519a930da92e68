"""Plain 64-bit forms of the operators around a decode step's attention and of
sampling, for the tests that hold the HIP kernels against them."""
import numpy as np

INV127 = np.float32(1.0) / np.float32(127.0)


def norm_rope(x, w, eps, pos, theta):
    """x [t, heads, hd]: per-head RMS norm (w None: none), then NeoX rotation at
    positions pos [t].  Returns (rotated, the size of what each value sums)."""
    x = np.asarray(x, np.float64)
    hd = x.shape[-1]
    if w is not None:
        x = x / np.sqrt(np.mean(x * x, axis=-1, keepdims=True) + eps) * np.asarray(w, np.float64)
    half = hd // 2
    ang = np.asarray(pos, np.float64)[:, None] * float(theta) ** (-2.0 * np.arange(half) / hd)
    c, s = np.cos(ang)[:, None, :], np.sin(ang)[:, None, :]
    a, b = x[..., :half], x[..., half:]
    size = np.abs(a) + np.abs(b)
    return (np.concatenate([a * c - b * s, a * s + b * c], -1),
            np.concatenate([size, size], -1))


def q8_rows(x):
    """The Q8 of f32 rows [t, n]: int8 [t, n], f32 [t, n/32]."""
    x = np.asarray(x, np.float32)
    y = x.reshape(x.shape[0], -1, 32)
    d = np.abs(y).max(-1) * INV127
    safe = np.where(d > 0, d, np.float32(1))
    return np.rint(y / safe[..., None]).astype(np.int8).reshape(x.shape), d


def q8_values(q, d):
    y = q.reshape(q.shape[0], -1, 32).astype(np.float64) * d.astype(np.float64)[..., None]
    return y.reshape(q.shape)


def attention(q, k, v, n_kv, scale):
    """q [heads, hd], k/v [seq, n_kv*hd]: (out [heads, hd], its tolerance in f32).

    Tolerance: a score sums head_dim products in f32, each within 2^-23 of the
    largest |q| (q in two 11-bit parts) and some eight roundings of the partial
    sums: 16 * 2^-24 * scale * sum |q k|.  A weight inherits twice that (its own
    score and the normalisation), plus the exponential's 2^-22 (1 + |x|) with x
    no larger than the span at which a weight still counts (16): 2^-17 of it;
    sums of weights and products round a further 2^-20."""
    heads, hd = q.shape
    out, tol = np.zeros((heads, hd)), np.zeros((heads, hd))
    if k.shape[0] == 0:
        return out, tol
    q, k, v = (np.asarray(a, np.float64) for a in (q, k, v))
    for h in range(heads):
        j = h // (heads // n_kv)
        kh, vh = k[:, j * hd:(j + 1) * hd], v[:, j * hd:(j + 1) * hd]
        x = scale * (kh @ q[h])
        size = abs(scale) * (np.abs(kh).sum(1) * np.abs(q[h]).max())
        p = np.exp(x - x.max())
        p /= p.sum()
        out[h] = p @ vh
        spread = p @ np.abs(vh)
        # weights that matter: those above 2^-24 of the sum
        err = 2 * 16 * 2.0**-24 * size[p > 2.0**-24].max() + 2.0**-17
        tol[h] = err * spread + 1e-30
    return out, tol


def sample(logits, t, k, p, m, u):
    """One row: the token that the filters and u draw (see tf_sample)."""
    x = np.asarray(logits, np.float64) + 0.0  # -0 is +0
    n = x.size
    x = np.where(np.isnan(x), -np.inf, x)
    if x.max() == -np.inf:
        return 0
    if not t > 0:
        return int(np.argmax(x))
    if x.max() == np.inf:
        w = (x == np.inf).astype(np.float64)
    else:
        with np.errstate(invalid="ignore"):
            z = np.where(x == -np.inf, -np.inf, x / np.float64(np.float32(t)))
        w = np.exp(z - z.max())
    order = np.argsort(-x, kind="stable")
    keep = n
    if 0 < k < n:
        keep = k
    s = w[order][:keep]
    if p < 1:
        goal = float(np.float32(p)) * s.sum()
        keep = min(keep, int((np.cumsum(s) < goal).sum()) + 1)
    if m > 0:
        keep = min(keep, int((s >= min(float(np.float32(m)), 1.0)).sum()))
    kept = np.sort(order[:max(1, keep)])
    c = np.cumsum(w[kept])
    u = float(np.float32(u))
    at = int((c <= (u if u > 0 else 0.0) * c[-1]).sum())
    if at >= len(kept):
        at = int(np.nonzero(w[kept] > 0)[0][-1])
    return int(kept[at])
