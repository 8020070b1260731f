"""The paged 4-bit cache's attention where a row's weight is concentrated: one token of nearly all of
it and a small value (an attention sink), the rest spread over thousands, over values of several
sizes.  What the many light tokens add up to must survive beside the heavy one."""
import math

import pytest
import torch

from gpu_util import announce

pytestmark = pytest.mark.gpu

WEIGHTS = [0.5, 0.9, 0.99, 0.999, 0.9999]
SIZES = [(0.3, 1 / 64), (0.05, 1 / 64), (0.3, 0.0), (3e-3, 0.0), (1e-4, 1 / 64)]  # of the values; the sink's share of it
LIFT = 8.0  # channel 0 of the queries; of the keys, the sink's alone has one


def _pool(kv, H, D, G, gen):
    import akv
    pages = -(-kv // 16)
    pool = akv.PagedPool.empty(1, pages, H, D, 16, G)
    table = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32).view(1, -1)
    one = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    return pool, table, akv.PagedBatch(table, one(kv), one(0, kv), kv, kv)


def _fill(pool, whole, kv, weight, size, share, gen):
    """Keys and values as the cache holds them, float64; the sink's place."""
    import akv
    H, D = pool.heads, pool.head_dim
    at = kv // 3
    k, v = torch.randn(2, kv, H, D, generator=gen, device="cuda")
    v *= size
    v[at] *= share
    k[..., 0] = 0.0
    k[at] = 0.0
    # the others' scores are normal, so the log of the sum of their exponentials is near log(kv) + 1 / 2
    k[at, :, 0] = (math.log(weight / (1 - weight)) + math.log(kv) + 0.5) * D ** 0.5 / LIFT
    akv.paged_append(pool, whole, k, v)
    return (*(x.double() for x in akv.paged_read(pool, whole, 0, torch.float32)), at)


def _exact(q, k, v, g, see):
    """q (n, Hq, D), keys and values (kv, H, D) float64: out (n, Hq, D), lse (n, Hq), all weights' sum but the heaviest."""
    out, lse, rest = [], [], []
    for h in range(q.shape[1]):
        x = (q[:, h].double() @ k[:, h // g].T) * q.shape[2] ** -0.5
        x = x.masked_fill(~see, -torch.inf)
        l = torch.logsumexp(x, -1)
        p = torch.exp(x - l[:, None])
        out.append(p @ v[:, h // g])
        lse.append(l)
        rest.append(1 - p.amax(-1))
    return torch.stack(out, 1), torch.stack(lse, 1), torch.stack(rest, 1)


def _check(got, exact, what):
    """Rounding to the output's type alone leaves 0.58 of half a step (of float16 below its normal
    range: of half its smallest, 2^-25), and the kernel's own part stays below 0.47 of it for float16
    and 0.15 for bfloat16: 0.75 and 0.6 together."""
    half, share = (2.0 ** -11, 0.75) if got.dtype == torch.float16 else (2.0 ** -8, 0.6)
    err = got.double() - exact
    limit = share * half * float(exact.norm())
    if got.dtype == torch.float16:
        limit += share * 2.0 ** -25 * float((exact.abs() < 2.0 ** -14).sum()) ** 0.5
    assert float(err.norm()) <= limit, f"{what}: error {float(err.norm() / exact.norm()):.2e} of the norm, {float(err.norm()) / limit:.2f} of the limit"


@pytest.mark.parametrize("kv,n,H,g,D,G", [(8192, 1, 2, 4, 128, 32), (65536, 1, 1, 2, 128, 64), (16384, 3, 2, 1, 64, 32), (500, 2, 2, 3, 128, 128),
                                          (8192, 40, 1, 2, 128, 32), (16384, 80, 1, 1, 64, 64), (65536, 70, 1, 1, 128, 128)])
def test_one_sequence(kv, n, H, g, D, G):
    """Alone; of more than 64 rows a cached head (the tile kernel's) too."""
    import akv
    gen = torch.Generator(device="cuda").manual_seed(kv + n)
    pool, table, whole = _pool(kv, H, D, G, gen)
    one = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    batch = akv.PagedBatch(table, one(kv), one(0, n), n, n)
    see = torch.ones(n, kv, dtype=torch.bool, device="cuda").tril(kv - n)
    for size, share in SIZES:
        for weight in WEIGHTS:
            announce(f"paged attention kv={kv} rows={n} H={H} g={g} D={D} G={G}, a sink of {weight}, values of {size}, its own {share} of it")
            k, v, _ = _fill(pool, whole, kv, weight, size, share, gen)
            for dt in (torch.float16, torch.bfloat16):
                q = torch.randn(n, H * g, D, generator=gen, device="cuda")
                q[..., 0] = LIFT
                q = q.to(dt)
                eo, el, rest = _exact(q, k, v, g, see)
                assert bool((rest > (1 - weight) / 2).all()) and bool((rest < (1 - weight) * 2).all())
                out, lse = akv.paged_attention(q, pool, batch, return_lse=True)
                _check(out, eo, f"{dt}, sink {weight}, values {size}, {share}")
                assert float((lse.double() - el).norm() / el.norm()) < 2.0 ** -20
                assert torch.equal(out, akv.paged_attention(q, pool, batch))


@pytest.mark.parametrize("D,G", [(128, 32), (64, 64)])
def test_long_runs(D, G):
    """A batch so large that one wave takes the sink and thousands of tokens with it: 64 sequences that
    share the pages of 16384 tokens, 16 heads."""
    import akv
    kv, H, S = 16384, 16, 64
    gen = torch.Generator(device="cuda").manual_seed(D)
    pool, table, whole = _pool(kv, H, D, G, gen)
    batch = akv.PagedBatch(table.expand(S, -1).contiguous(), torch.full((S,), kv, dtype=torch.int32, device="cuda"),
                           torch.arange(S + 1, dtype=torch.int32, device="cuda"), S, 1)
    see = torch.ones(1, kv, dtype=torch.bool, device="cuda")
    for size, share in SIZES:
        for weight in WEIGHTS:
            announce(f"paged attention, runs of 8192 tokens, D={D} G={G}, a sink of {weight}, values of {size}, its own {share} of it")
            k, v, _ = _fill(pool, whole, kv, weight, size, share, gen)
            for dt in (torch.float16, torch.bfloat16):
                q = torch.randn(S, H, D, generator=gen, device="cuda")
                q[..., 0] = LIFT
                q = q.to(dt)
                out = akv.paged_attention(q, pool, batch)
                for s in (0, 31, 63):
                    _check(out[s:s + 1], _exact(q[s:s + 1], k, v, 1, see)[0], f"sequence {s}, {dt}, sink {weight}, values {size}, {share}")


@pytest.mark.parametrize("D,G", [(128, 32), (128, 128), (64, 32)])
def test_scales_that_grow_and_shrink(D, G):
    """Values whose size changes a thousandfold along the context, both ways, and groups that are flat or zero."""
    import akv
    kv, H, g = 6000, 2, 4
    gen = torch.Generator(device="cuda").manual_seed(D + G)
    pool, table, whole = _pool(kv, H, D, G, gen)
    one = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    sizes = torch.logspace(-3, 0, kv, device="cuda")
    for turn, size in enumerate((sizes, sizes.flip(0), sizes[torch.randperm(kv, generator=gen, device="cuda")])):
        announce(f"paged attention D={D} G={G}, sizes in order {turn}")
        k, v = torch.randn(2, kv, H, D, generator=gen, device="cuda")
        v *= size[:, None, None]
        v[5::97, 0, :G] = 0.0
        v[7::89, 1, D - G:] = 0.25
        akv.paged_append(pool, whole, k, v)
        k, v = (x.double() for x in akv.paged_read(pool, whole, 0, torch.float32))
        for n in (1, 3, 20):
            batch = akv.PagedBatch(table, one(kv), one(0, n), n, n)
            see = torch.ones(n, kv, dtype=torch.bool, device="cuda").tril(kv - n)
            for dt in (torch.float16, torch.bfloat16):
                q = torch.randn(n, H * g, D, generator=gen, device="cuda").to(dt)
                _check(akv.paged_attention(q, pool, batch), _exact(q, k, v, g, see)[0], f"{dt}, {n} rows, order {turn}")


@pytest.mark.parametrize("n,size", [(n, s) for n in (1, 5) for s in (1e3, -1e3, 2e4, 6e4, -6e4, 2e5, -2e5)] +
                         [(30, s) for s in (1e3, -1e3, 2e4, -2e4, 6e4)])
def test_scores_of_any_size(n, size):
    """Scores up to 5e8, where float32 holds every 32nd unit (chunks of more than 64 rows: 1.6e8): one token
    far above the others gives its value, one far below them nothing."""
    import akv
    kv, H, g, D, G = 1000, 2, 3, 128, 32
    gen = torch.Generator(device="cuda").manual_seed(n)
    announce(f"paged attention, {n} rows, a score of {size * 3e4 / 11.3:.0e}")
    pool, table, whole = _pool(kv, H, D, G, gen)
    one = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    k, v = torch.randn(2, kv, H, D, generator=gen, device="cuda")
    k.zero_()  # beside other values a zero would be read back as up to half a step: scores of some hundreds
    k[kv // 2, :, 0] = size
    v[..., 1] = 1.0
    akv.paged_append(pool, whole, k, v)
    v = akv.paged_read(pool, whole, 0, torch.float32)[1].repeat_interleave(g, 1)
    batch = akv.PagedBatch(table, one(kv), one(0, n), n, n)
    for dt in (torch.float16, torch.bfloat16):
        q = torch.zeros(n, H * g, D, device="cuda", dtype=dt)
        q[..., 0] = 3e4
        out, lse = akv.paged_attention(q, pool, batch, causal=False, return_lse=True)
        if size > 0:
            # the one value, rounded to the output's type; beside it what the matrix cores round of two parts below |v| + 7 s
            worst = float(((out.float() - v[kv // 2]).abs() - torch.finfo(dt).eps * v[kv // 2].abs()).max())
            assert worst <= 2.0 ** -11
            score = float(q[0, 0, 0]) * akv.paged_read(pool, whole, 0, torch.float32)[0][kv // 2, :, 0].repeat_interleave(g) * D ** -0.5
            assert bool(((lse - score).abs() <= score.abs() * 2.0 ** -20).all())
        else:
            # the other 999 tokens have one score: their values' mean
            mean = (v.double().sum(0) - v[kv // 2].double()) / (kv - 1)
            worst = float(((out.double() - mean).abs() - torch.finfo(dt).eps * mean.abs()).max())
            assert worst <= 2.0 ** -11
            assert bool(((lse - math.log(kv - 1)).abs() < 1e-4).all())


@pytest.mark.parametrize("D,G", [(128, 32), (64, 64)])
@pytest.mark.parametrize("size", [1e-2, 1e-3, 1e-4, 1e-6])
def test_small_values(size, D, G):
    """Flat weights over small values, few rows and chunks: the limits follow the outputs' size (and
    float16's smallest step), so that zeros in their place would not pass."""
    import akv
    H, g = 2, 4
    gen = torch.Generator(device="cuda").manual_seed(D)
    one = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    for kv, n in ((90, 1), (2000, 3), (300, 90)):
        announce(f"paged attention D={D} G={G} kv={kv} rows={n}, values of {size}")
        pool, table, whole = _pool(kv, H, D, G, gen)
        k, v = torch.randn(2, kv, H, D, generator=gen, device="cuda")
        akv.paged_append(pool, whole, k, v * size)
        k, v = (x.double() for x in akv.paged_read(pool, whole, 0, torch.float32))
        batch = akv.PagedBatch(table, one(kv), one(0, n), n, n)
        see = torch.ones(n, kv, dtype=torch.bool, device="cuda").tril(kv - n)
        for dt in (torch.float16, torch.bfloat16):
            q = torch.randn(n, H * g, D, generator=gen, device="cuda").to(dt)
            eo = _exact(q, k, v, g, see)[0]
            for lse in (True, False):
                out = akv.paged_attention(q, pool, batch, return_lse=lse)
                _check(out[0] if lse else out, eo, f"{dt}, kv {kv}, log-sums {lse}")
            if dt == torch.bfloat16 or size > 1e-6:
                with pytest.raises(AssertionError):
                    _check(torch.zeros_like(q), eo, "zeros")


@pytest.mark.parametrize("kv,n,H,g,D,G", [(8192, 65, 1, 8, 128, 32), (20000, 300, 1, 1, 128, 64), (4000, 90, 2, 2, 64, 32), (3000, 100, 1, 1, 128, 128)])
def test_chunks_with_channels_that_stand_out(kv, n, H, g, D, G):
    """Chunks over keys with a channel ten times the others: outputs are the same with and without log-sums,
    and for bfloat16 no more than 3% farther from 64 bits than rounding alone leaves them."""
    import akv
    announce(f"paged attention of a chunk, kv={kv} rows={n} D={D} G={G}, a channel ten times the others")
    gen = torch.Generator(device="cuda").manual_seed(kv)
    pool, table, whole = _pool(kv, H, D, G, gen)
    k, v = torch.randn(2, kv, H, D, generator=gen, device="cuda")
    k[..., 3] *= 10.0
    akv.paged_append(pool, whole, k, v)
    k, v = (x.double() for x in akv.paged_read(pool, whole, 0, torch.float32))
    one = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    batch = akv.PagedBatch(table, one(kv), one(0, n), n, n)
    see = torch.ones(n, kv, dtype=torch.bool, device="cuda").tril(kv - n)
    for dt in (torch.float16, torch.bfloat16):
        q = torch.randn(n, H * g, D, generator=gen, device="cuda").to(dt)
        eo = _exact(q, k, v, g, see)[0]
        out = akv.paged_attention(q, pool, batch)
        assert torch.equal(out, akv.paged_attention(q, pool, batch, return_lse=True)[0])
        _check(out, eo, str(dt))
        if dt == torch.bfloat16:
            # p and the values in float16 leave 2^-12 / sqrt(3) = 1.4e-4 each, 2.0e-4 together: beside
            # bfloat16's 1.65e-3 and more, the root of both squares is 0.8% above it
            assert float((out.double() - eo).norm()) <= 1.03 * float((eo.to(dt).double() - eo).norm())
