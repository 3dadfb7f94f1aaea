"""Plain 64-bit numpy forms of the pre-norm block's operators (dropout, layer norm, their fusion, scaled embedding), and bounds on
what fp32 arithmetic with one final rounding may be off by.

Bounds. Every fp32 operation is off by at most half a step, U = 2^-24 relative to its result; a sum of n terms taken one after
the other by at most (n - 1) U times the sum of magnitudes, whatever the order of partial sums of at most n terms. The kernels
add at most ``hidden / 32`` terms per thread, five levels of a warp and 32 warps, so ``chain(hidden)`` below bounds the number of
additions behind any row sum, with room for the few operations around it. The final rounding is off by half a step of the storage type."""
import numpy as np
import torch

U = 2.0 ** -24


def chain(terms, lanes=32):
    return terms / lanes + 5 + 32 + 16


def rounding(want, dtype):
    """Half a step of the storage type at each value (half a subnormal step near zero)."""
    f = torch.finfo(dtype)
    return f.eps / 2 * np.abs(want) + f.smallest_normal * f.eps / 2


# ------------------------------------------------------------------------------------------------------------ dropout
def philox4x32_10(counter, key):
    """One block: counter of four words (arrays or ints), key of two. Salmon et al., SC 2011."""
    m = np.uint64(0xffffffff)
    c = [np.asarray(v, dtype=np.uint64) for v in counter]
    k = [int(v) for v in key]
    for _ in range(10):
        a, b = np.uint64(0xD2511F53) * c[0], np.uint64(0xCD9E8D57) * c[2]
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), b & m, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), a & m]
        k = [(k[0] + 0x9E3779B9) & 0xffffffff, (k[1] + 0xBB67AE85) & 0xffffffff]
    return c


def threshold(p):
    return min(65535, int(np.rint(float(np.float32(p)) * 65536)))


def keep(count, p, seed, step, site, first=0):
    """Decisions of elements first .. first + count."""
    if threshold(p) == 0:
        return np.ones(count, bool)
    blocks = np.arange(first // 8, (first + count + 7) // 8, dtype=np.uint64)
    words = philox4x32_10([blocks, site, step & 0xffffffff, step >> 32], [seed & 0xffffffff, seed >> 32])
    halves = np.stack([h for w in words for h in (np.broadcast_to(w, blocks.shape) & np.uint64(0xffff), np.broadcast_to(w, blocks.shape) >> np.uint64(16))], 1)
    return (halves.reshape(-1) >= threshold(p))[first % 8:first % 8 + count]


def drop(x, p, seed, step, site):
    x = np.asarray(x, np.float64)
    mask = keep(x.size, p, seed, step, site).reshape(x.shape)
    return np.where(mask, x * (65536.0 / (65536 - threshold(p))), 0.0)


# --------------------------------------------------------------------------------------------------------- layer norm
def layernorm(x, w, b, eps):
    x = np.asarray(x, np.float64)
    d = x - x.mean(1, keepdims=True)
    rstd = 1 / np.sqrt((d * d).mean(1, keepdims=True) + eps)
    return d * rstd * w + (0 if b is None else b)


def _parts(x, eps):
    x = np.asarray(x, np.float64)
    d = x - x.mean(1, keepdims=True)
    rstd = 1 / np.sqrt((d * d).mean(1, keepdims=True) + eps)
    xh = d * rstd
    # error of xh in units of U: the mean's, carried through, and the relative error of rstd
    return xh, rstd, np.abs(x).mean(1, keepdims=True) * rstd + np.abs(xh)


def layernorm_error(x, w, b, eps):
    xh, _, dxh = _parts(x, eps)
    return U * (chain(x.shape[1]) * dxh * np.abs(w) + 4 * (np.abs(xh * w) + (0 if b is None else np.abs(b))))


def layernorm_backward(dy, x, w, eps):
    xh, rstd, _ = _parts(x, eps)
    g = dy * w
    dx = rstd * (g - g.mean(1, keepdims=True) - xh * (g * xh).mean(1, keepdims=True))
    return dx, (dy * xh).sum(0), dy.sum(0)


def layernorm_backward_error(dy, x, w, eps):
    """Bounds of dx, dw and db. A column's sum has at most rows / 8 terms one after the other, then 8 and 32 + 32 parts."""
    rows, hidden = x.shape
    xh, rstd, dxh = _parts(x, eps)
    g = np.abs(dy * w)
    mean = lambda v: v.mean(1, keepdims=True)
    c2 = np.abs(mean(dy * w * xh))
    dx = U * chain(hidden) * rstd * (2 * g + 2 * mean(g) + 2 * np.abs(xh) * mean(g * np.abs(xh)) + c2 * dxh + np.abs(xh) * mean(g * dxh))
    n = rows / 8 + 8 + 64 + 8
    dw = U * (n * np.abs(dy * xh).sum(0) + chain(hidden) * (np.abs(dy) * dxh).sum(0))
    return dx, dw, U * n * np.abs(dy).sum(0)


# ---------------------------------------------------------------------------------------------------------- embedding
def embedding(ids, weight, scale):
    out = np.zeros((len(ids), weight.shape[1]))
    inside = ids < len(weight)
    out[inside] = scale * np.asarray(weight, np.float64)[ids[inside]]
    return out


def embedding_backward(ids, grad, vocab, scale, padding=None):
    """Gradient table and the sum of magnitudes and the token count behind each row, for the bound."""
    table, size, count = np.zeros((vocab, grad.shape[1])), np.zeros((vocab, grad.shape[1])), np.zeros(vocab)
    use = (ids < vocab) & (ids != (vocab if padding is None else padding))
    np.add.at(table, ids[use], scale * grad[use])
    np.add.at(size, ids[use], np.abs(scale * grad[use]))
    np.add.at(count, ids[use], 1)
    return table, size, count
