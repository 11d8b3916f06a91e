"""The paged key-value cache's operators in float64: write of new tokens, attention of one row over the
keys it may see, for packed sequences of different lengths. Each attention result comes with the bound
that a 16-bit kernel with fp32 arithmetic is held to."""
import numpy as np


def rotate(x, weight, cos, sin, eps):
    """Head RMSNorm and rotate-half rotary position of ``x`` ``[..., D]``."""
    x, weight, cos, sin = (np.asarray(a, np.float64) for a in (x, weight, cos, sin))
    half = x.shape[-1] // 2
    y = x / np.sqrt((x ** 2).mean(-1, keepdims=True) + eps) * weight
    return y * cos + np.concatenate((-y[..., half:], y[..., :half]), -1) * sin


def sequence_rows(cu, tokens, lens):
    """(row, sequence, position) of each packed new token."""
    for b in range(len(lens)):
        n = cu[b + 1] - cu[b]
        for i in range(n):
            if cu[b] + i < tokens:
                yield cu[b] + i, b, lens[b] - n + i


def gather(pages, table_row, length):
    """The first ``length`` rows of a sequence, ``[length, heads, D]``; a page that is not there is zeros."""
    count, heads, size, d = pages.shape
    out = np.zeros((length, heads, d))
    for first in range(0, length, size):
        page, rows = int(table_row[first // size]), min(size, length - first)
        if 0 <= page < count:
            out[first:first + rows] = pages[page, :, :rows].transpose(1, 0, 2)
    return out


def attention(q, k, v, scale, causal, unit, weight_unit):
    """(out, bound) of queries ``[n, nq, D]`` over keys ``[m, nkv, D]``, the last query at the last key.

    ``unit`` is half a step of the output's type and ``weight_unit`` of the type that softmax weights round
    to. With w the weights and A = sum w |v|: the output's rounding is unit |o|; weights off by a relative
    r move o by r A. r adds up the weights' rounding, the sum's and the scores' errors: a score is a sum of
    D exact products in fp32 (truncating accumulation: 2^-23 an addition of at most scale sum |q k|) and
    enters the numerator and the sum; n additions of weights, and of weighted values, 2^-23 each; exp2 to 2^-20.
    """
    q, k, v = (np.asarray(a, np.float64) for a in (q, k, v))
    n, nq, d = q.shape
    m, nkv = k.shape[:2]
    rep = nq // nkv
    out, bound = np.zeros((n, nq, d)), np.zeros((n, nq, d))
    for i in range(n):
        seen = min(max(m - n + i + 1, 0), m) if causal else m
        if not seen:
            continue
        for h in range(nkv):
            qs = q[i, h * rep:(h + 1) * rep]
            kk, vv = k[:seen, h], v[:seen, h]
            s = scale * qs @ kk.T
            w = np.exp(s - s.max(-1, keepdims=True))
            w /= w.sum(-1, keepdims=True)
            o = w @ vv
            size = (abs(scale) * np.abs(qs) @ np.abs(kk).T).max(-1, keepdims=True)
            r = weight_unit + 2.0 * (d + 2) * 2.0 ** -23 * size + 2.0 * (seen + 2) * 2.0 ** -23 + 2.0 ** -20
            out[i, h * rep:(h + 1) * rep] = o
            # fp16 weights under 2^-14 and outputs round by an absolute 2^-25 (the largest weight is 1)
            tiny = 2.0 ** -25 * (1 + np.abs(vv).sum(0)) if unit < 2.0 ** -9 else 2.0 ** -120
            bound[i, h * rep:(h + 1) * rep] = unit * np.abs(o) + (1 + unit) * r * (w @ np.abs(vv)) + tiny
    return out, bound
