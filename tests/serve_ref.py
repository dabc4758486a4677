"""Float64 references of the serving operators (include/hq_serve.h) and what their tests share: pools whose unused places
hold NaN, page tables in no order, error bounds of each output element."""
import numpy as np

U16, U32 = 2.0 ** -11, 2.0 ** -24  # roundings to fp16 and fp32


class Pool:
    """A paged cache on the host in float16 (Q8: int8 codes and fp16 scales), every place of it not a number (Q8: scales)
    until written."""

    def __init__(self, rng, n_pos, page, kv_heads, hd, q8=False, layout="pos", spare=3):
        self.page, self.kv, self.hd, self.q8, self.layout = page, kv_heads, hd, q8, layout
        need = [(n + page - 1) // page for n in n_pos]
        self.n_pages = max(1, sum(need) + spare)
        order = rng.permutation(self.n_pages)[:sum(need)]
        self.table = np.full((len(need), max(need + [1])), 0, np.uint32)
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = order[at:at + n]
            at += n
        shape = (self.n_pages, page, kv_heads, hd) if layout == "pos" else (self.n_pages, kv_heads, page, hd)
        self.c = {n: (rng.integers(-128, 128, shape).astype(np.int8) if q8 else np.full(shape, np.nan, np.float16)) for n in "kv"}
        self.d = {n: np.full((self.n_pages, kv_heads, page), np.nan, np.float16) for n in "kv"} if q8 else None
        self.strides = (page * kv_heads * hd, kv_heads * hd, hd) if layout == "pos" else (page * kv_heads * hd, hd, page * hd)

    def _at(self, s, p):
        return self.table[s, p // self.page], p % self.page

    def put(self, s, p, k, v):
        """Positions p (array) of sequence s take k and v [len(p), kv, hd] (Q8: quantised)."""
        pg, sl = self._at(s, np.asarray(p))
        for n, x in (("k", k), ("v", v)):
            if self.q8:
                d = (np.abs(x.astype(np.float32)).max(-1) / np.float32(127)).astype(np.float16)
                c = np.rint(x / np.where(d > 0, d, 1)[..., None].astype(np.float32)).clip(-127, 127).astype(np.int8)
                self.d[n][pg, :, sl] = d
                x = c
            if self.layout == "pos":
                self.c[n][pg, sl] = x
            else:
                self.c[n][pg, :, sl] = x

    def get(self, name, s, n):
        """Positions 0 .. n - 1 of sequence s [n, kv, hd] in float64."""
        pg, sl = self._at(s, np.arange(n))
        x = (self.c[name][pg, sl] if self.layout == "pos" else self.c[name][pg, :, sl]).astype(np.float64)
        return x * self.d[name][pg, :, sl].astype(np.float64)[..., None] if self.q8 else x

    def device(self, hq):
        b = [hq.DevBuf.from_array(self.c[n]) for n in "kv"] + ([hq.DevBuf.from_array(self.d[n]) for n in "kv"] if self.q8 else [None, None])
        return hq.KvCache(hq.KV_Q8 if self.q8 else hq.KV_F16, self.n_pages, self.page, self.kv, self.hd, b[0], b[1], self.strides, b[2], b[3])

    def read(self, hq, kv):
        """The device's contents back into c and d."""
        for i, n in enumerate("kv"):
            self.c[n] = kv.keep[i].download(self.c[n].shape, self.c[n].dtype)
            if self.q8:
                self.d[n] = kv.keep[2 + i].download(self.d[n].shape, np.float16)


def fill(pool, rng, n_pos, std=1.0):
    for s, n in enumerate(n_pos):
        if n:
            pool.put(s, np.arange(n), *(rng.normal(0, std, (2, n, pool.kv, pool.hd)).astype(np.float16)))


def attention(pool, q, n_new, n_pos, scale, gate=None):
    """Outputs in float64 and a bound of the error of an fp16 kernel, [tokens, heads, hd]. The bound: the output's rounding;
    the weights' to fp16 and, of a Q8 cache, the decoded values', each 2^-11 of sum p |v|; and the scores' error e (fp32
    sums over hd products, a Q8 key's rounding to fp16, the exponential's 2^-20), which moves a weight by 2 e."""
    T, nh, hd = q.shape
    rep = nh // pool.kv
    y, bound = np.zeros((T, nh, hd)), np.zeros((T, nh, hd))
    q = q.astype(np.float64)
    t = 0
    for s, (new, tot) in enumerate(zip(n_new, n_pos)):
        k, v = pool.get("k", s, tot), pool.get("v", s, tot)
        for j in range(new):
            n = tot - new + j + 1
            if n > 0:
                for h in range(nh):
                    kk, vv = k[:n, h // rep], v[:n, h // rep]
                    with np.errstate(invalid="ignore", over="ignore"):
                        x = kk @ q[t, h] * scale
                        p = np.exp(x - x.max())
                        p /= p.sum()
                        y[t, h] = p @ vv
                        e = ((hd + 8) * U32 + (U16 if pool.q8 else 0)) * (np.abs(kk) @ np.abs(q[t, h])).max() * abs(scale) + 2.0 ** -20
                        bound[t, h] = U16 * np.abs(y[t, h]) + (U16 * (2 if pool.q8 else 1) + 2 * e) * (p @ np.abs(vv)) + 2.0 ** -24
            if gate is not None:
                g = 1 / (1 + np.exp(-gate[t].astype(np.float64)))
                y[t] *= g
                bound[t] = bound[t] * g + U16 * np.abs(y[t]) + 2.0 ** -24
            t += 1
    return y, bound


def rope(x, w, cs, rot, off, eps):
    """x [tokens, heads, hd] in float64 normalised by w (or None) and rotated by cs [tokens, rot / 2, 2]; and the sum of the
    magnitudes that an output element is made of."""
    x = x.astype(np.float64)
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * (off + w.astype(np.float64))
    half = rot // 2
    c, s = (cs[:, None, :, i].astype(np.float64) for i in (0, 1))
    y, mag = x.copy(), np.abs(x)
    a, b = x[..., :half], x[..., half:rot]
    y[..., :half], y[..., half:rot] = a * c - b * s, b * c + a * s
    mag[..., :half], mag[..., half:rot] = np.abs(a * c) + np.abs(b * s), np.abs(b * c) + np.abs(a * s)
    return y, mag
