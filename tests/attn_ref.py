"""The quantised cache and its attention in numpy, from their definitions (include/hako_attn.h)."""
import numpy as np

from hako_amd.gpu import KV_F16, KV_Q8, Kv

FLT_MIN = np.float32(1.17549435e-38)


def rows(x, kind):
    """Codes and scales of float32 rows [..., head_dim]."""
    x = np.asarray(x, np.float32)
    bad = ~np.isfinite(x).all(-1)
    x = np.where(bad[..., None], np.float32(0), x)
    a = np.abs(x)
    amax = np.where(a < FLT_MIN, np.float32(0), a).max(-1)
    if kind == KV_Q8:
        with np.errstate(divide="ignore", invalid="ignore", over="ignore"):
            scale = amax * np.float32(1 / 127)
            scale = np.where(scale < FLT_MIN, np.float32(0), scale)
            inv = np.where(scale > 0, np.float32(127) / amax, np.float32(0)).astype(np.float32)
        c = np.clip(np.rint(np.where(a < FLT_MIN, np.float32(0), x) * inv[..., None]), -127, 127).astype(np.int8)
    else:
        e = np.where(bad, 0, np.maximum(np.where(a.max(-1) > 0, np.frexp(a.max(-1))[1] - 1, -126), -126))
        scale = np.ldexp(np.float32(1), e).astype(np.float32)
        c = np.ldexp(x.astype(np.float64), -e[..., None]).astype(np.float16)
    return c, np.where(bad, np.float32(np.nan), scale).astype(np.float32)


def rotate(x, table, rot, interleaved):
    """x [tokens][heads][head_dim] float32, table [tokens][rot/2][2]: every product and sum rounded to float32."""
    y = x.copy()
    i = np.arange(rot // 2)
    lo, hi = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
    a, b, c, s = x[..., lo], x[..., hi], table[:, None, :, 0], table[:, None, :, 1]
    y[..., lo], y[..., hi] = a * c - b * s, a * s + b * c
    return y


def table(n_pos, rot, theta=1e6, stretch=1.0):
    f = theta ** (-np.arange(0, rot, 2) / rot) / stretch
    a = np.arange(n_pos)[:, None] * f
    return np.stack([np.cos(a), np.sin(a)], 2).astype(np.float32)


class Cache:
    """Host arrays of a cache and their copies on the device."""

    def __init__(self, gpu, kind, slots, max_seq, kvh, hd, rng=None, fill=None):
        self.gpu, self.kind, self.slots, self.max_seq, self.kvh, self.hd = gpu, kind, slots, max_seq, kvh, hd
        shape = (slots, kvh, max_seq)
        if rng is not None:
            self.k, self.ks = rows(rng.standard_normal((*shape, hd)), kind)
            self.v, self.vs = rows(rng.standard_normal((*shape, hd)), kind)
        else:
            dt = np.int8 if kind == KV_Q8 else np.float16
            self.k, self.v = (np.full((*shape, hd), fill, dt) for _ in range(2))
            self.ks, self.vs = (np.full(shape, fill, np.float32) for _ in range(2))
        self.bufs = [gpu.upload(a) for a in (self.k, self.v, self.ks, self.vs)]
        self.kv = Kv(kind, slots, max_seq, kvh, hd, *(b.ptr for b in self.bufs))

    def push(self):
        for b, a in zip(self.bufs, (self.k, self.v, self.ks, self.vs)):
            self.gpu.h2d(b, a)

    def pull(self):
        """(k, v, k scales, v scales) as the device holds them."""
        return [self.gpu.download(b, a.dtype, a.shape) for b, a in zip(self.bufs, (self.k, self.v, self.ks, self.vs))]

    def free(self):
        for b in self.bufs:
            b.free()

    def values(self):
        return (self.k.astype(np.float64) * self.ks.astype(np.float64)[..., None],
                self.v.astype(np.float64) * self.vs.astype(np.float64)[..., None])


def attend(q, K, V, slot, end, scale, prefix_slot=0, prefix_len=0):
    """One token in float64: q [heads][head_dim] over positions [0, end) of values K, V [slot][kv head][position][dim]."""
    H, hd = q.shape
    G = H // K.shape[1]
    out = np.zeros((H, hd))
    if end <= 0:
        return out
    p = min(prefix_len, end)
    for g in range(K.shape[1]):
        k, v = (np.concatenate([x[prefix_slot, g, :p], x[slot, g, p:end]]) for x in (K, V))
        s = q[g * G:(g + 1) * G].astype(np.float64) @ k.T * scale
        w = np.exp(s - s.max(1, keepdims=True))
        out[g * G:(g + 1) * G] = w @ v / w.sum(1, keepdims=True)
    return out
