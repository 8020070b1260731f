"""The paged 4-bit cache in numpy and 64 bits: the tile by byte positions, the quantizer, the
attention and the importance, and bounds on what rounding may do to the kernels' results."""
import numpy as np

TOP = 61440.0


def tile_bytes(D, G):
    return 16 * D + 128 * (D // G)


def places(D, G):
    """Of K and V: byte and shift of code (token, channel), byte of scale (token, group), of zero."""
    NG = D // G
    out = []
    t, c = np.meshgrid(np.arange(16), np.arange(D), indexing="ij")
    g, i, n = c // 32, c % 32 // 8, c % 8
    out.append([t * (D // 2) + (i * (D // 32) + g) * 4 + n // 2, 4 * (n % 2)])
    a, p, e = t // 4, t // 2 % 2, t % 2
    h, l, r, b = c // 64, c // 32 % 2, c % 32 // 2, c % 2
    out.append([8 * D + (((a * 16 + r) * 2 + p) * (D // 64) + h) * 4 + e * 2 + l, 4 * b])
    t, q = np.meshgrid(np.arange(16), np.arange(NG), indexing="ij")
    k = 16 * D + (t * NG + q) * 4
    out[0] += [k, k + 2]
    v = 16 * D + 64 * NG + ((t // 4 * NG + q) * 4 + t % 4) * 2
    out[1] += [v, v + 32 * NG]
    return out


def quantize(x, G):
    """(..., D) float64 -> codes (..., D) uint8, scale and zero (..., NG) float16."""
    xg = x.reshape(*x.shape[:-1], x.shape[-1] // G, G)
    bad = ~np.isfinite(xg).all(-1)
    xg = np.clip(np.where(np.isfinite(xg), xg, 0.0), -TOP, TOP)
    lo, hi = xg.min(-1), xg.max(-1)
    s, z = ((hi - lo) / 15.0).astype(np.float16), lo.astype(np.float16)
    s1 = np.where(s == 0, 1.0, s.astype(np.float64))[..., None]
    c = np.clip(np.rint((xg - z.astype(np.float64)[..., None]) / s1), 0, 15)
    c = np.where((s == 0)[..., None] | bad[..., None], 0, c)
    nan = np.float16(np.nan)
    return c.astype(np.uint8).reshape(x.shape), np.where(bad, nan, s), np.where(bad, nan, z)


class Pool:
    """A numpy pool (layers, pages, H, P / 16, tile) with the tokens of page tables in it."""

    def __init__(self, data, D, G):
        self.data, self.D, self.G = data, D, G
        self.P = 16 * data.shape[3]
        self.places = places(D, G)

    def rows(self, layer, table, pos):
        pos = np.asarray(pos, dtype=np.int64)
        return layer, np.asarray(table)[pos // self.P], pos % self.P // 16, pos % 16

    def write(self, layer, table, pos, k, v):
        """k, v (n, H, D) float64 at positions pos."""
        _, page, tile, tok = self.rows(layer, table, pos)
        H = k.shape[1]
        for j in range(len(page)):
            for h in range(H):
                t = self.data[layer, page[j], h, tile[j]]
                for (at, sh, sa, za), x in zip(self.places, (k, v)):
                    c, s, z = quantize(x[j, h], self.G)
                    np.bitwise_and.at(t, at[tok[j]], (0xF0 >> sh[tok[j]]).astype(np.uint8))
                    np.bitwise_or.at(t, at[tok[j]], (c << sh[tok[j]]).astype(np.uint8))
                    for q in range(len(s)):
                        t[sa[tok[j], q]:sa[tok[j], q] + 2] = np.frombuffer(s[q:q + 1].tobytes(), np.uint8)
                        t[za[tok[j], q]:za[tok[j], q] + 2] = np.frombuffer(z[q:q + 1].tobytes(), np.uint8)

    def parts(self, layer, table, pos):
        """Of K and V: code * scale and zero, (n, H, D) float64."""
        _, page, tile, tok = self.rows(layer, table, pos)
        t = self.data[layer, page, :, tile]  # (n, H, tile bytes)
        out = []
        for at, sh, sa, za in self.places:
            pick = lambda a: np.take_along_axis(t, np.broadcast_to(a[tok][:, None], (len(tok), t.shape[1], a.shape[1])), 2)  # noqa: E731
            half = lambda a: (pick(a).astype(np.uint16) | (pick(a + 1).astype(np.uint16) << 8)).view(np.float16)  # noqa: E731
            code = (pick(at) >> sh[tok][:, None]) & 15
            s, z = (np.repeat(half(a).astype(np.float64), self.G, axis=-1) for a in (sa, za))
            with np.errstate(invalid="ignore"):
                out.append((code * s, z))
        return out

    def read(self, layer, table, pos):
        return [a + b for a, b in self.parts(layer, table, pos)]


def attention(q, kp, vp, scale, seen, half, rounded=False):
    """One sequence: q (m, Hq, D), parts of its cached keys and values (n, H, D), row i sees the
    first seen[i] tokens.  Returns out, lse and how far each may be off: `half` is half a step
    of the output's type.

    The scores are exact but for float32 sums (at most 64 roundings of terms that add up to
    `mass`); p and p * scale are rounded to float16 (2^-11 each, or 2^-25 absolute below its
    normal range, p times 4 and codes up to 15).  `rounded`: the keys are rounded to float16 too,
    half a step (2^-11) of each, which moves a score by 2^-11 of the terms |q||k| that it sums."""
    m, Hq, D = q.shape
    n, H = kp[0].shape[:2]
    out, lse = np.zeros((m, Hq, D)), np.full((m, Hq), -np.inf)
    eo, el = np.zeros((m, Hq, D)), np.zeros((m, Hq))
    for i in range(m):
        N = int(seen[i])
        if N <= 0:
            continue
        for h in range(Hq):
            kc, kz, vc, vz = (a[:N, h // (Hq // H)] for a in (*kp, *vp))
            x = scale * ((kc + kz) @ q[i, h])
            mass = scale * ((np.abs(kc) + np.abs(kz)) @ np.abs(q[i, h])).max()
            d = 64 * 2.0 ** -24 * mass
            if rounded:
                d += 2.0 ** -11 * scale * (np.abs(kc + kz) @ np.abs(q[i, h])).max()
            e = np.exp(x - x.max())
            l = e.sum()
            p = e / l
            out[i, h] = p @ (vc + vz)
            lse[i, h] = x.max() + np.log(l)
            A, Z = p @ np.abs(vc), p @ np.abs(vz)
            eo[i, h] = (2.0 ** -11 * (2 * A + Z) + (2 * d + 2.0 ** -18) * (A + Z) + half * np.abs(out[i, h])
                        + N * 2.0 ** -25 * (15 + np.abs(vz).max()) / (4 * l) + 2.0 ** -25)
            el[i, h] = d + 2.0 ** -23 * (4 + abs(lse[i, h])) + N * 2.0 ** -26
    return out, lse, eo, el


def importance(q, kp, scale, seen, lse):
    """sum over rows of the mean over heads of exp(scale q.k - lse), and its bound."""
    m, Hq, D = q.shape
    n, H = kp[0].shape[:2]
    total, err = np.zeros(n), np.zeros(n)
    for i in range(m):
        N = int(seen[i])
        for h in range(Hq if N > 0 else 0):
            kc, kz = (a[:N, h // (Hq // H)] for a in kp)
            mass = scale * ((np.abs(kc) + np.abs(kz)) @ np.abs(q[i, h])).max()
            p = np.exp(scale * ((kc + kz) @ q[i, h]) - lse[i, h])
            total[:N] += p / Hq
            err[:N] += p / Hq * (64 * 2.0 ** -24 * mass + 2.0 ** -22 * (4 + abs(lse[i, h])) + m * Hq * 2.0 ** -24)
    return total, err
