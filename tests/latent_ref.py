"""The paged latent cache in torch and 64 bits on the host: what it holds, both forms of the
attention, the importance and the eviction, and bounds on what rounding may do to the kernels'
results."""
import torch

TOP = 61440.0


def held(x):
    """Rows (n, Dc + Dr) float64 as the cache holds them, float16 rounded once; and as they read back."""
    bad = ~torch.isfinite(x).all(dim=-1, keepdim=True)
    y = x.clamp(-TOP, TOP).half()
    return y, torch.where(bad, torch.full_like(y, float("nan")), y)


def _sees(m, n, kv, causal):
    """Tokens that each of m rows of a sequence of n tokens, kv of them there, sees."""
    i = torch.arange(m)
    return (n - m + i + 1).clamp(0, kv) if causal else torch.full((m,), kv)


def attention(q, qr, rows, scale, half, causal=True, n=None):
    """One sequence, absorbed form: q (m, H, Dc), qr (m, H, Dr) and its rows (kv, Dc + Dr), float64.
    Returns out, lse and how far each may be off; `half` is half a step of the output's type.

    The query times a power of two is exact in float16 but for values below 2^-28 of its row's
    largest (2^-38 of that).  Scores are float32 sums: at most 64 roundings of terms that add up to `mass`.
    p is rounded to float16, half a step of 2^-11, or 2^-25 of it where the weight is below 2^-27 of the row's."""
    m, H, Dc = q.shape
    kv = rows.shape[0]
    x = torch.cat([q, qr], dim=-1)
    c = rows[:, :Dc]
    see = _sees(m, kv if n is None else n, kv, causal)
    s = scale * torch.matmul(x.reshape(m * H, -1), rows.T).reshape(m, H, kv)
    mass = scale * torch.matmul(x.abs().reshape(m * H, -1), rows.abs().T).reshape(m, H, kv)
    mass = mass + scale * 2.0 ** -14 * x.abs().amax(-1, keepdim=True) * rows.abs().sum(-1)
    hidden = torch.arange(kv) >= see[:, None]
    return _softmax_out(s, mass, hidden[:, None], c, half, 64 * 2.0 ** -24, 0.0)


def _softmax_out(s, mass, hidden, v, half, per_mass, v_err):
    """v (kv, D), or (H, kv, D) one for each head."""
    s = s.masked_fill(hidden, float("-inf"))
    d = (per_mass * mass.masked_fill(hidden, 0.0)).amax(-1, keepdim=True) if s.shape[-1] else torch.zeros(*s.shape[:-1], 1)
    top = s.amax(-1, keepdim=True) if s.shape[-1] else torch.full((*s.shape[:-1], 1), float("-inf"), dtype=s.dtype)
    none = torch.isneginf(top)
    e = torch.exp(s - top.masked_fill(none, 0.0))
    l = e.sum(-1, keepdim=True)
    p = torch.where(l > 0, e / l, torch.zeros_like(e))
    mul = lambda a, b: (torch.matmul(a, b) if b.dim() == 2 else torch.matmul(a.transpose(0, 1), b).transpose(0, 1))  # noqa: E731
    out, A = mul(p, v), mul(p, v.abs())
    big = v.abs().amax(dim=tuple(range(v.dim())), keepdim=False) if v.numel() else torch.zeros((), dtype=s.dtype)
    lse = (top + torch.log(l)).squeeze(-1)
    light = s.shape[-1] * 2.0 ** -36 * big / l.clamp_min(1.0)
    eo = (2.0 ** -11 + v_err + 2 * d + 2.0 ** -18) * A + half * out.abs() + light + 2.0 ** -25 + v_err * 2.0 ** -13 * big
    el = d.squeeze(-1) + 2.0 ** -23 * (4 + lse.abs().masked_fill(none.squeeze(-1), 0.0)) + s.shape[-1] * 2.0 ** -26
    return out, lse, eo, el


def prefill(q, rows, w_k, w_v, scale, half, causal=True, n=None):
    """One sequence, expanded form: q (m, H, 128 + Dr), w_k and w_v (H, 128, Dc), float64.

    Beyond attention()'s: weights, keys and values are rounded to float16 (2^-11 each; weights that are
    float16 or bfloat16 but for those far below their channel's largest are not), which moves a score by that of the
    terms that it sums."""
    m, H = q.shape[:2]
    kv, Dc = rows.shape[0], w_k.shape[2]
    c, r = rows[:, :Dc], rows[:, Dc:]
    k = torch.cat([torch.matmul(c, w_k.transpose(1, 2)), r.expand(H, *r.shape)], dim=-1)
    v = torch.matmul(c, w_v.transpose(1, 2))
    # a product's own rounding: float32 sums over what their terms add up to
    k_mass = torch.cat([torch.matmul(c.abs(), w_k.abs().transpose(1, 2)) * (64 * 2.0 ** -24 + 2.0 ** -18), torch.zeros_like(r).expand(H, *r.shape)], dim=-1)
    v_mass = torch.matmul(c.abs(), w_v.abs().transpose(1, 2)) * (64 * 2.0 ** -24 + 2.0 ** -18)
    s = scale * torch.matmul(q.transpose(0, 1), k.transpose(1, 2)).transpose(0, 1)
    mass = scale * torch.matmul(q.abs().transpose(0, 1), k.abs().transpose(1, 2)).transpose(0, 1)
    mass = mass + 2.0 ** 11 * scale * torch.matmul(q.abs().transpose(0, 1), k_mass.transpose(1, 2)).transpose(0, 1)
    mass = mass + scale * 2.0 ** -14 * q.abs().amax(-1, keepdim=True) * k.abs().sum(-1).amax(0)
    see = _sees(m, kv if n is None else n, kv, causal)
    hidden = torch.arange(kv) >= see[:, None]
    out, lse, eo, el = _softmax_out(s, mass, hidden[:, None], v, half, 2.0 ** -11 + 64 * 2.0 ** -24, 2.0 ** -11)
    if v_mass.numel():
        eo = eo + v_mass.amax()
    return out, eo


def importance(q, qr, rows, scale, lse, causal=True, n=None, window=0):
    """sum over rows of the mean over heads of exp(score - lse), and its bound."""
    m, H = q.shape[:2]
    kv = rows.shape[0]
    x = torch.cat([q, qr], dim=-1)
    s = scale * torch.matmul(x.reshape(m * H, -1), rows.T).reshape(m, H, kv)
    mass = scale * torch.matmul(x.abs().reshape(m * H, -1), rows.abs().T).reshape(m, H, kv)
    hidden = (torch.arange(kv) >= _sees(m, kv if n is None else n, kv, causal)[:, None])[:, None].expand(m, H, kv)
    if window:
        hidden = hidden | (torch.arange(m) < m - window)[:, None, None]
    p = torch.exp(s - lse[..., None]).masked_fill(hidden, 0.0)
    err = p * (64 * 2.0 ** -24 * mass + 2.0 ** -22 * (4 + lse.abs().masked_fill(torch.isinf(lse), 0.0))[..., None] + m * H * 2.0 ** -24)
    return p.sum((0, 1)) / H, err.sum((0, 1)) / H


def evict(scores, n, budget, first, last):
    """Positions that stay of a sequence of n tokens with scores (N,), by a plain sort."""
    n = max(0, min(n, len(scores)))
    k = min(n, max(budget, 0))

    def rank(j):
        if j < first or j >= n - last:
            return (2, 0.0, j)
        x = float(scores[j])
        return (1, 0.0, j) if x != x else (0, x, j)
    return sorted(sorted(range(n), key=rank)[n - k:])
