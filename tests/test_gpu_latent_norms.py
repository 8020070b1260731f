"""The latent attention's precision by norms: the output's own rounding and little beside it, whole and
row by row."""
import pytest
import torch

import latent_norms as ln
import latent_ref as ref
from gpu_util import announce
from test_gpu_latent import DT, World, _queries, _randn, _scale

pytestmark = pytest.mark.gpu


def _check(w, H, dt, size, heads):
    """Heads `heads` of H against 64 bits, in norms."""
    import akv
    wk, wv = (_randn(H, 128, w.Dc, seed=s, dt=dt, scale=w.Dc ** -0.5) for s in (21, 22))
    q = _randn(w.T, H, 192, seed=23, dt=dt, scale=size)
    out = akv.latent_prefill(q.cuda(), w.pool, w.batch, akv.LatentWeights(wk.cuda(), wv.cuda())).double().cpu()
    gots, wants = [], []
    for s in range(len(w.kv)):
        r = w.mine(s)
        if w.q[s] == 0:
            continue
        want, _ = ref.prefill(q[r][:, heads].double(), w.rows(s), wk[heads].double(), wv[heads].double(), _scale(), 0.0, n=w.kv[s])
        none = (torch.arange(w.q[s]) + w.kv[s] - w.q[s] + 1) <= 0
        assert not bool(out[r][none].any())
        gots.append(out[r][~none][:, heads]), wants.append(want[~none])
    got, want = torch.cat(gots), torch.cat(wants)
    got, most = ln.off(got, want), ln.limits(want, DT[dt])
    print(f"{dt} size {size}: off by {got[0]:.3e} (limit {most[0]:.3e}), rows {got[1]:.3e} ({most[1]:.3e})", flush=True)
    assert got[0] <= most[0] and got[1] <= most[1], (got, most)


# workgroups of 128 query tokens, and of 256 (many heads of more than 128 tokens); short and long contexts
CASES = [(4, 300, 50, 512, 16), (2, 3000, 20, 256, 64), (1, 6000, 130, 512, 16), (128, 400, 300, 512, 64), (128, 2100, 257, 256, 32)]


@pytest.mark.parametrize("size", [1.0, 4.0])
@pytest.mark.parametrize("H,kv,m,Dc,P", CASES)
def test_float16(H, kv, m, Dc, P, size):
    announce(f"latent prefill precision, float16: H={H} kv={kv} m={m} Dc={Dc} size={size}")
    w = World(Dc, P, [kv], [m])
    w.fill()
    _check(w, H, "fp16", size, torch.arange(H)[:: max(1, H // 5)])


@pytest.mark.parametrize("H,kv,m,Dc,P", CASES)
def test_bfloat16(H, kv, m, Dc, P):
    announce(f"latent prefill precision, bfloat16: H={H} kv={kv} m={m} Dc={Dc}")
    w = World(Dc, P, [kv], [m])
    w.fill()
    _check(w, H, "bf16", 1.0, torch.arange(H)[:: max(1, H // 5)])


@pytest.mark.parametrize("H,kv,m,Dc,P", [(16, 300, 1, 512, 64), (8, 300, 2, 256, 16), (16, 4000, 1, 512, 16), (1, 700, 16, 512, 64),
                                         (40, 300, 1, 512, 64), (64, 4000, 1, 512, 16), (32, 900, 2, 256, 32), (128, 300, 1, 512, 32),
                                         (128, 3000, 1, 256, 16), (16, 500, 40, 512, 64)])
def test_absorbed_float16(H, kv, m, Dc, P):
    """p as two float16: the output's own rounding alone, as the plain formula has it."""
    import akv
    announce(f"latent attention precision, float16: H={H} kv={kv} m={m} Dc={Dc}")
    S = 12
    w = World(Dc, P, [kv + i for i in range(S)], [m] * S)
    w.fill()
    q, qr, x = _queries(w, H, "fp16")
    out = akv.latent_attention(q, qr, w.pool, w.batch, _scale()).double().cpu()
    want = torch.cat([ref.attention(x[w.mine(s), :, :Dc], x[w.mine(s), :, Dc:], w.rows(s), _scale(), 0.0)[0] for s in range(S)])
    got, most = ln.off(out, want), ln.limits(want, torch.float16)
    print(f"off by {got[0]:.3e} (limit {most[0]:.3e}), rows {got[1]:.3e} ({most[1]:.3e})", flush=True)
    assert got[0] <= most[0] and got[1] <= most[1]


def _ragged(n, most, seed):
    """Tokens and query tokens of n sequences, idle ones and ones without tokens among them."""
    g = torch.Generator().manual_seed(seed)
    q = torch.randint(1, most, (n,), generator=g).tolist()
    q = [0 if i % 7 == 3 else m for i, m in enumerate(q)]
    past = torch.randint(0, 60, (n,), generator=g).tolist()
    return [0 if i % 11 == 5 and m == 0 else m + p for i, (m, p) in enumerate(zip(q, past))], q


@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("n,H,most", [(257, 3, 20), (700, 2, 9), (513, 1, 40)])
def test_expanded_form_of_many_sequences(n, H, most, dt):
    """Several sequences a thread of the scans, items that workgroups share between them; one long one among the short."""
    announce(f"latent prefill of {n} sequences, H={H} {dt}")
    kv, q = _ragged(n, most, n)
    kv[n // 2], q[n // 2] = 1500, 300
    w = World(256, 16, kv, q)
    w.fill()
    _check(w, H, dt, 1.0, torch.arange(H))
    w.same_pool()


def test_tiles_of_many_sequences():
    """Workgroups of 256 query tokens over more sequences than the scans have threads."""
    announce("latent prefill of 300 sequences, 128 heads")
    kv, q = _ragged(300, 12, 4)
    kv[7], q[7] = 350, 290
    w = World(256, 32, kv, q)
    w.fill()
    for dt in ("fp16", "bf16"):
        _check(w, 128, dt, 1.0, torch.arange(3, 128, 31))


@pytest.mark.parametrize("Dc,P", [(512, 16), (256, 64)])
def test_an_appended_row_is_all_that_changes(Dc, P):
    """A token that holds NaN and its neighbours: every other slot of the pool keeps its bits."""
    import akv
    announce(f"latent append of a NaN token, Dc={Dc} P={P}")
    kv, m = 70, 6
    w = World(Dc, P, [kv, 33], [m, 0], layers=2)
    x = _randn(m, w.W, seed=4)
    x[m // 2, 100] = float("nan")
    akv.latent_append(w.pool, w.batch, x[:, :Dc].cuda(), x[:, Dc:].cuda(), layer=1)
    page, row = w.slots(0, torch.arange(kv - m, kv))
    got = w.pool.data.cpu()[1, page, row]
    bad = torch.arange(m) == m // 2
    assert torch.equal(got[~bad], x[~bad])
    assert not bool(got[bad, :Dc].any()) and bool(torch.isnan(got[bad, Dc:]).all())
    w.data[1, page, row] = got
    w.same_pool()
