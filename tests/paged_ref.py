"""64-bit numpy forms of the operators over a paged KV cache, and the device
buffers of a test's call (16-bit values are rounded to nearest even here)."""
import numpy as np

import mi355x
from mi355x import BF16, F16, F32

# half a step relative to the value: f32, f16, bf16
HALF_STEP = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}


def encode(x, t):
    """float64 values as the type's bits (an array of the type's size)."""
    x = np.asarray(x, np.float32)
    if t == F32:
        return x
    if t == F16:
        with np.errstate(over="ignore"):
            return x.astype(np.float16)
    b = x.view(np.uint32)
    r = ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def decode(a, t):
    if t == BF16:
        return (a.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return a.astype(np.float64)


def storage(t):
    return {F32: np.float32, F16: np.float16, BF16: np.uint16}[t]


class Pool:
    """Pages of keys and values: float64 values as the type holds them
    (k, v: [page][token][head][value]) and the same on the device, with `gap`
    values between tokens, heads and pages that no one may touch."""

    def __init__(self, ctx, rng, t, n_pages, page, heads, hd, hnd=False, gap=0, fill=None):
        self.ctx, self.t, self.n_pages, self.page, self.heads, self.hd = ctx, t, n_pages, page, heads, hd
        # strides in values: [page][token][head][hd] or [page][head][token][hd]
        inner = hd + gap
        if hnd:
            self.token, self.head = inner, inner * page + gap
            self.stride = self.head * heads + gap
        else:
            self.head, self.token = inner, inner * heads + gap
            self.stride = self.token * page + gap
        self.size = self.stride * max(n_pages, 1)
        shape = (n_pages, page, heads, hd)
        if fill is None:
            self.k, self.v = (decode(encode(rng.standard_normal(shape), t), t) for _ in range(2))
        else:
            self.k, self.v = np.full(shape, fill), np.full(shape, fill)
        p, tok, h, d = np.ogrid[:n_pages, :page, :heads, :hd]
        self.at = p * self.stride + tok * self.token + h * self.head + d
        self.gaps = np.ones(self.size, bool)
        self.gaps[self.at] = False
        self.bufs = []
        self.upload()

    def upload(self):
        for b in self.bufs:
            b.free()
        self.bufs = []
        for a in (self.k, self.v):
            flat = encode(np.full(self.size, 7.0), self.t)
            flat[self.at] = encode(a, self.t)
            self.bufs.append(self.ctx.to_device(flat))

    def download(self):
        """(k, v) as float64, the gaps checked to be as they were."""
        out = []
        for b in self.bufs:
            flat = decode(b.download(storage(self.t), self.size), self.t)
            assert np.all(flat[self.gaps] == 7.0), "values between the tokens were written"
            out.append(flat[self.at])
        return out

    def struct(self, **over):
        f = dict(type=self.t, n_kv_heads=self.heads, head_dim=self.hd, page_tokens=self.page, n_pages=self.n_pages,
                 k=self.bufs[0].ptr, v=self.bufs[1].ptr, page_stride=self.stride, token_stride=self.token,
                 head_stride=self.head)
        f.update(over)
        return mi355x.KvPool(**f)

    def free(self):
        for b in self.bufs:
            b.free()


def plan(cached, added, page, table, free, head, n_rows):
    """The plan's outputs (the lengths and pages suffice)."""
    table = table.copy()
    offsets = np.concatenate([[0], np.cumsum(added)]).astype(np.int32)
    positions, slots = np.zeros(n_rows, np.int32), np.full(n_rows, -1, np.int64)
    for s, (c, a) in enumerate(zip(cached, added)):
        for col in range(-(-c // page), -(-(c + a) // page)):
            table[s, col] = free[head]
            head += 1
        for i in range(a):
            r, p = offsets[s] + i, c + i
            positions[r] = p
            slots[r] = int(table[s, p // page]) * page + p % page
    return dict(row_offsets=offsets, kv_lens=np.asarray(cached, np.int32) + np.asarray(added, np.int32), table=table,
                head=head, positions=positions, slots=slots)


def rope(x, bias, norm, eps, positions, inv_freq, rot, pairs):
    """x: [rows, heads, hd] in float64; (result, error scale): |turned| <= scale."""
    x = np.asarray(x, np.float64)
    if bias is not None:
        x = x + np.asarray(bias, np.float64).reshape(x.shape[1:])
    if norm is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * np.asarray(norm, np.float64)
    y = x.copy()
    size = np.abs(x)
    if rot:
        i = np.arange(0, rot, 2) if pairs else np.arange(rot // 2)
        j = i + (1 if pairs else rot // 2)
        f = np.asarray(positions, np.float64)[:, None, None] * np.asarray(inv_freq, np.float64)
        y[..., i] = x[..., i] * np.cos(f) - x[..., j] * np.sin(f)
        y[..., j] = x[..., j] * np.cos(f) + x[..., i] * np.sin(f)
        size[..., i] = size[..., j] = np.abs(x[..., i]) + np.abs(x[..., j])
    return y, size


def attention(q, pool, offsets, kv_lens, table, scale, softcap=0.0, window=0, causal=True):
    """q: [rows, heads, hd] as the type holds it.  (out, weighted |v|, score
    scale): out[row, head], sum_j w_j |v_j|, and max_j scale sum_d |q_d k_jd|."""
    T, H, hd = q.shape
    G = H // pool.heads
    out, mag, size = np.zeros((T, H, hd)), np.zeros((T, H, hd)), np.zeros((T, H))
    reach = table.shape[1] * pool.page
    for s in range(len(kv_lens)):
        kv, n = int(kv_lens[s]), int(offsets[s + 1]) - int(offsets[s])
        j = np.arange(max(0, min(kv, reach)))
        pg = table[s][j // pool.page]
        good = (pg >= 0) & (pg < pool.n_pages)
        r0, i = int(offsets[s]), np.arange(n)
        i = i[r0 + i < T]
        if not j.size or not i.size:
            continue
        p = (kv - n + i)[:, None]
        see = np.broadcast_to(good, (i.size, j.size)) & ((j <= p) if causal else True)
        if window:
            see = see & (j > p - window)
        pp = np.where(good, pg, 0)
        k, v = pool.k[pp, j % pool.page], pool.v[pp, j % pool.page]  # [keys, kv heads, hd]
        some = see.any(0)
        k, v = np.where(some[:, None, None], k, 0.0), np.where(some[:, None, None], v, 0.0)
        for h in range(H):
            kh, vh, qh = k[:, h // G], v[:, h // G], q[r0 + i, h]
            sc = scale * (qh @ kh.T)
            size[r0 + i, h] = np.where(see, np.abs(scale) * (np.abs(qh) @ np.abs(kh).T), 0.0).max(1)
            if softcap:
                sc = softcap * np.tanh(sc / softcap)
            sc = np.where(see, sc, -np.inf)
            w = np.exp(sc - np.where(see.any(1), sc.max(1), 0.0)[:, None])
            w /= np.maximum(w.sum(1, keepdims=True), 1e-300)
            out[r0 + i, h], mag[r0 + i, h] = w @ vh, w @ np.abs(vh)
    return out, mag, size
