"""64-bit numpy forms of the operators of mi355x-layer.h."""
import numpy as np

from paged_ref import HALF_STEP, decode, encode, storage  # noqa: F401  (what the tests use)


def codes_of(t, loose=0.0):
    """(codes, scales in 64 bits, whether either neighbour may stand) of rows of 64-bit values, ties to even.
    A quotient within `loose` of a border may go either way."""
    t = np.asarray(t, np.float64)
    bad = ~np.isfinite(t).all(1)
    t = np.where(bad[:, None], 0.0, t)
    most = np.abs(t).max(1)
    y = t * 127 / np.where(most > 0, most, 1)[:, None]
    c = np.rint(y)
    off = np.abs(np.abs(y - np.trunc(y)) - 0.5)
    scale = most / 127
    scale[bad] = np.nan
    return c.astype(np.int8), scale, off < loose


def norm_rows(x, residual, residual_type, norm, eps):
    """(h as residual_type holds it, t before the root's factor, that factor)."""
    h = x
    if residual is not None:
        with np.errstate(over="ignore", invalid="ignore"):
            h = decode(encode(x.astype(np.float32) + residual.astype(np.float32), residual_type), residual_type)
    if norm is None:
        return h, h, np.ones(len(x))
    with np.errstate(over="ignore", invalid="ignore"):
        return h, h * norm.astype(np.float64), 1 / np.sqrt((h * h).mean(1) + np.float64(np.float32(eps)))


def swiglu(g, u):
    with np.errstate(over="ignore", invalid="ignore"):
        return g / (1 + np.exp(-g)) * u


def matmul(x, w, x_scales, w_scales, bias, t):
    """The bits of out: the sum in whole numbers, then f32 roundings in the stated order."""
    s = x.astype(np.int64) @ w.astype(np.int64).T if x.shape[1] < 64 else \
        np.rint(x.astype(np.float64) @ w.astype(np.float64).T)  # sums below 2^31: exact in 64-bit floats
    with np.errstate(over="ignore", invalid="ignore"):
        y = s.astype(np.float32) * w_scales[None, :] * x_scales[:, None]
        if bias is not None:
            y = y + bias[None, :]
    return encode(y, t)


def logprobs(x, scale):
    """(log p, entropy) of rows of logits in 64 bits."""
    z = np.asarray(x, np.float64) * np.float64(np.float32(scale))
    with np.errstate(invalid="ignore", divide="ignore"):
        top = z.max(1, keepdims=True)
        empty = np.isneginf(top)
        d = z - np.where(empty, 0, top)
        p = np.exp(d)
        total = p.sum(1, keepdims=True)
        lp = d - np.where(empty, 0, np.log(total))
        ent = -(np.where(p > 0, p * lp, 0)).sum(1) / total[:, 0]
    bad = ~(x < np.inf).all(1)
    lp[bad], ent[bad] = np.nan, np.nan
    ent[empty[:, 0]] = 0
    return lp, ent


def top_tokens(x, n):
    """The n largest logits' tokens of each row, equal ones in ascending order; -1 where fewer are above -inf."""
    out = np.full((len(x), n), -1, np.int32)
    for r, row in enumerate(x):
        if not (row < np.inf).all():
            continue
        order = np.argsort(-row, kind="stable")[:n]
        order = order[row[order] > -np.inf]
        out[r, :len(order)] = order
    return out
