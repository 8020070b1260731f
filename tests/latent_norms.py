"""How far the latent attention's outputs may be off by their norms: the output's own rounding, and
little beside it.  `expanded` is the expanded form with chosen roundings on the host, which shows
what such a limit tells apart."""
import torch


def weights(w):
    """(H, C, Dc) as float16 over a power of two for each channel, and those powers."""
    top = w.abs().amax(-1, keepdim=True)
    e = torch.where(top > 0, torch.frexp(top)[1] + 4, torch.zeros_like(top, dtype=torch.int32))
    return torch.ldexp(w, -e).half().double(), torch.ldexp(torch.ones_like(top), e)


def halves(x, n):
    """x as a sum of n float16, the largest first."""
    out = []
    for _ in range(n):
        out.append(x.half().double())
        x = x - out[-1]
    return out


def expanded(q, rows, w_k, w_v, scale, dtype, keys=2, values=2, p=2, rest=lambda x: x, skip=None):
    """One sequence's causal rows: q (m, H, 128 + Dr), rows (kv, Dc + Dr), float64.  keys, values, p: how many
    float16 they are; rest: what becomes of the values' second ones (H, kv, 128); skip: a token left out."""
    m, kv, Dc = q.shape[0], rows.shape[0], w_k.shape[2]
    c, r = rows[:, :Dc], rows[:, Dc:]
    (wk, sk), (wv, sv) = weights(w_k), weights(w_v)
    k = sum(halves(torch.matmul(c, wk.transpose(1, 2)), keys))
    v = halves(torch.matmul(c, wv.transpose(1, 2)), values)
    x = q.transpose(0, 1)
    s = scale * (torch.matmul(x[..., :128] * sk.transpose(1, 2), k.transpose(1, 2)) + torch.matmul(x[..., 128:], r.T))
    s = s.masked_fill(torch.arange(kv) > torch.arange(kv - m, kv)[:, None], float("-inf"))
    if skip is not None:
        s[..., skip] = float("-inf")
    e = torch.exp(s - s.amax(-1, keepdim=True)) * 2.0 ** 13
    ps = halves(e, p)
    o = torch.matmul(sum(ps), v[0])
    if values > 1:
        o = o + torch.matmul(ps[0], rest(v[1]))
    return (o / e.sum(-1, keepdim=True) * sv.transpose(1, 2)).transpose(0, 1).to(dtype).double()


def off(got, want):
    """The error's norm over the whole output's, and the largest of those over a row of a head."""
    d = got - want
    return float(d.norm() / want.norm()), float((d.norm(dim=-1) / want.norm(dim=-1).clamp_min(1e-30)).max())


def limits(want, dtype):
    """Rounding the outputs leaves `own` of their norm, and at most half a step of any row's.  What comes before it
    may add a quarter of that in quadrature (1.03 in all): for float16 5.1e-5, where 300 tokens and one float16 for keys,
    values or p add 1.2e-4 and more, and float32 sums some 1e-5; for bfloat16 4.1e-4, where one float16 for all three and scores of
    standard deviation 1 add 2.3e-4.  In quadrature means over many outputs: with errors r of the rounding and d before it,
    |r + d|^2 has a cross term 2 r.d that differs from 0 by 2 |r| |d| / sqrt(N), for 256 outputs and d = 0.15 r 2% of |r|^2 at one
    standard deviation, for 25600 0.2%; so the norm is a whole call's.  A row's part of what comes before may be larger than the whole's: a quarter of a
    half step is granted."""
    own = off(want.to(dtype).double(), want)[0]
    return 1.03 * own, 1.25 * torch.finfo(dtype).eps / 2
