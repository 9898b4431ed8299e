"""The 8-bit paged cache's operators as their definitions say, in 64 bits on the CPU, position by position."""
import numpy as np
import torch

D, BLOCK = 128, 16


class Cache:
    """Host copy of a cache; codes and scales as the GPU holds them."""

    def __init__(self, cache, table):
        self.k, self.v, self.ks, self.vs = (t.detach().cpu().clone().numpy() for t in cache)
        self.table = table.detach().cpu().numpy()
        self.rows = self.k.shape[2]
        self.capacity = self.table.shape[1] * self.rows

    def place(self, s, p):
        return int(self.table[s, p // self.rows]), p % self.rows

    def values(self, s, n):
        """K, V of the positions 0 .. n - 1, float64 [n, H, 128]."""
        out = []
        for codes, scales in ((self.k, self.ks), (self.v, self.vs)):
            rows = np.zeros((n,) + codes.shape[1::2])
            for p in range(n):
                page, i = self.place(s, p)
                rows[p] = codes[page, :, i].astype(np.float64) * scales[page, :, i // BLOCK].astype(np.float64)[:, None]
            out.append(rows)
        return out


def rotate(x, pos, inv_freq):
    """x [n, H, 128] float64 at the positions pos [n]; angles are float32 products."""
    ang = (np.asarray(pos, np.float32)[:, None] * inv_freq[None, :64].astype(np.float32)).astype(np.float64)[:, None]
    a, b = x[..., :64], x[..., 64:]
    return np.concatenate([a * np.cos(ang) - b * np.sin(ang), b * np.cos(ang) + a * np.sin(ang)], -1)


def code(x, s):
    """x and s float32 values in float64: the quotient has more digits than two codes' middle needs."""
    if s == 0:
        return np.zeros(x.shape, np.int8)
    with np.errstate(invalid="ignore"):
        q = np.clip(np.rint(x / s), -127, 127)
    return np.where(np.isnan(q), 0, q).astype(np.int8)


def rows_of(S, T, cu):
    return [(s * (T // S), T // S) for s in range(S)] if cu is None else [(int(cu[s]), int(cu[s + 1] - cu[s])) for s in range(S)]


def append(c, k, v, pos0, cu=None, inv_freq=None):
    """Writes float32 values k, v [T, H, 128] (numpy) into c; rotates k first."""
    for s, (row0, n) in enumerate(rows_of(len(c.table), len(k), cu)):
        p0 = int(pos0[s])
        pos = [p for p in range(p0, p0 + n) if 0 <= p < c.capacity]
        for at in sorted({p // BLOCK * BLOCK for p in pos}):
            new = [p for p in pos if at <= p < at + BLOCK]
            page, i0 = c.place(s, at)
            for codes, scales, x, turn in ((c.k, c.ks, k, True), (c.v, c.vs, v, False)):
                rows = x[[row0 + p - p0 for p in new]].astype(np.float64)
                if turn and inv_freq is not None:
                    rows = rotate(rows, new, inv_freq)
                rows = rows.astype(np.float32).astype(np.float64)
                for h in range(codes.shape[1]):
                    finite = np.abs(rows[:, h][np.isfinite(rows[:, h])])
                    most = np.float32(finite.max() if finite.size else 0) * (np.float32(1) / np.float32(127))
                    most = np.float32(0) if most < 2.0 ** -100 else most
                    was = scales[page, h, i0 // BLOCK] if p0 > at else np.float32(0)
                    now = max(was, most)
                    if now > was:
                        for p in range(at, min(max(p0, at), at + BLOCK)):
                            i = p % c.rows
                            codes[page, h, i] = code((codes[page, h, i].astype(np.float32) * was).astype(np.float64), np.float64(now))
                    for j, p in enumerate(new):
                        codes[page, h, p % c.rows] = code(rows[j, h], np.float64(now))
                    scales[page, h, i0 // BLOCK] = now


def attention(c, q, pos0, cu=None, scale=None, inv_freq=None):
    """(result, sum of p |v|, largest error of a score, what a p too small for its pair moves) float64 for q [T, Hq, 128] (numpy)."""
    T, Hq, _ = q.shape
    H = c.k.shape[1]
    scale = D ** -0.5 if scale is None else scale
    out, spread, score, tiny = np.zeros(q.shape), np.zeros(q.shape), np.zeros((T, Hq, 1)), np.zeros((T, Hq, 1))
    for s, (row0, n) in enumerate(rows_of(len(c.table), T, cu)):
        limits = [int(min(max(int(pos0[s]) + r + 1, 0), c.capacity)) for r in range(n)]
        if not n or not max(limits):
            continue
        k, v = (torch.from_numpy(x) for x in c.values(s, max(limits)))
        x = q[row0:row0 + n].astype(np.float64)
        if inv_freq is not None:
            x = rotate(x, [int(pos0[s]) + r for r in range(n)], inv_freq)
        x = torch.from_numpy(x).view(n, H, Hq // H, D)
        sc = torch.einsum("nhgd,lhd->nhgl", x, k) * scale
        for r in range(n):
            L = limits[r]
            if not L:
                continue
            p = torch.softmax(sc[r, ..., :L], -1)
            out[row0 + r] = torch.einsum("hgl,lhd->hgd", p, v[:L]).reshape(Hq, D).numpy()
            spread[row0 + r] = torch.einsum("hgl,lhd->hgd", p, v[:L].abs()).reshape(Hq, D).numpy()
            # p vs is held as a pair of fp16 numbers, scaled so that the largest is 2^6 or more: the pair's last step is 2^-24, half
            # of it 2^-31 of the largest p vs, for every key, times a code of at most 127
            steps = torch.tensor(np.array([c.vs[c.place(s, i)[0], :, c.place(s, i)[1] // BLOCK] for i in range(L)]), dtype=torch.float64)
            tiny[row0 + r] = (L * 2.0 ** -31 * 127 * torch.einsum("hgl,lh->hgl", p, steps).amax(-1)).reshape(Hq, 1).numpy()
            mag = torch.einsum("hgd,lhd->hgl", x[r].abs(), k[:L].abs()).amax(-1)
            tall = torch.einsum("hg,lh->hgl", x[r].abs().amax(-1), k[:L].abs().sum(-1)).amax(-1)
            score[row0 + r] = (abs(scale) * (2.0 ** -19 * mag + 2.0 ** -21 * tall)).reshape(Hq, 1).numpy()
    return out, spread, score, tiny


def bound(want, spread, score, tiny, keys, dtype, p_single=False):
    """How far a result may be off `want`.  Half a step of its type.  A score is a sum of 128 exact products in eight steps
    of sixteen, each cut to 24 bits: 2^-19 of its magnitude holds twice that, and 2^-21 of the largest |q| times sum |k| a
    query kept as two 11-bit halves; e^error moves every p by twice the largest one's error.  p as two halves and its
    exponential: 2^-20, and `tiny` where the pair runs out of exponents.  p_single: p as one fp16 number, half a step of which is
    2^-11 of it (prompts with fp16 queries).  The sums over the keys, sixteen at a time: 2^-23 a step of sum p |v|."""
    half = torch.finfo(dtype).eps / 2
    return np.abs(want) * half * 1.01 + spread * (2 * score + 2.0 ** -20 + (2.0 ** -11 if p_single else 0) + (keys / 16 + 8) * 2.0 ** -23) + tiny + (2.0 ** -25 if dtype == torch.float16 else 1e-30)
