"""Normed, weighted and turned heads and their gradients in 64 bits (numpy), with the sums of magnitudes that error
bounds count in."""
import numpy as np

import serve_ref as R

U = 2.0 ** -24                                    # a rounding of fp32


def _heads(x, heads):
    return np.asarray(x, np.float64).reshape(len(x), heads, -1)


def _turned(x, heads, table, positions, rot, interleaved, transpose=False):
    n = len(x)
    y = R.rope(x.reshape(n, -1), heads, table, positions, rot, interleaved, transpose)
    # |a c| + |b s|: the rotation of magnitudes with all signs positive
    t = np.abs(np.asarray(table, np.float64))
    m = np.abs(x).reshape(n, heads, -1).copy()
    src = m.copy()
    for i in range(rot // 2):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
        c, s = t[positions, i, 0][:, None], t[positions, i, 1][:, None]
        m[:, :, a] = src[:, :, a] * c + src[:, :, b] * s
        m[:, :, b] = src[:, :, b] * c + src[:, :, a] * s
    return y, m.reshape(n, -1)


def forward(x, heads, weight, eps, table, positions, rot, interleaved):
    """(n, heads * d) -> result, and |a c| + |b s| of each element."""
    v = _heads(x, heads)
    r = 1.0 / np.sqrt((v * v).mean(-1, keepdims=True) + eps)
    return _turned(v * r * weight, heads, table, positions, rot, interleaved)


def backward(x, grad, heads, weight, eps, table, positions, rot, interleaved):
    """dx, dw and, for their bounds, r (G |w| + |x| r^2 mean(G |w x|)) and sum G |x| r, G the magnitudes of the gradient
    turned back."""
    n = len(x)
    v = _heads(x, heads)
    g, G = (a.reshape(v.shape) for a in _turned(np.asarray(grad, np.float64), heads, table, positions, rot, interleaved, transpose=True))
    r = 1.0 / np.sqrt((v * v).mean(-1, keepdims=True) + eps)
    dw = (g * v * r).sum((0, 1))
    gw = g * weight
    dx = r * (gw - v * r * r * (gw * v).mean(-1, keepdims=True))
    most = r * (G * np.abs(weight) + np.abs(v) * r * r * (G * np.abs(weight * v)).mean(-1, keepdims=True))
    return dx.reshape(n, -1), dw, most.reshape(n, -1), (G * np.abs(v) * r).sum((0, 1))
