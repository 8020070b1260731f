"""The expanded form's precision by norms: the output's own rounding and little beside it, whole and
row by row."""
import pytest
import torch

import latent_norms as ln
import latent_ref as ref
from gpu_util import announce
from test_gpu_latent import DT, World, _randn, _scale

pytestmark = pytest.mark.gpu


def _check(w, H, dt, size, heads):
    """Heads `heads` of H against 64 bits, in norms."""
    import akv
    wk, wv = (_randn(H, 128, w.Dc, seed=s, dt=dt, scale=w.Dc ** -0.5) for s in (21, 22))
    q = _randn(w.T, H, 192, seed=23, dt=dt, scale=size)
    out = akv.latent_prefill(q.cuda(), w.pool, w.batch, akv.LatentWeights(wk.cuda(), wv.cuda())).double().cpu()
    for s in range(len(w.kv)):
        r = w.mine(s)
        if w.q[s] == 0:
            continue
        want, _ = ref.prefill(q[r][:, heads].double(), w.rows(s), wk[heads].double(), wv[heads].double(), _scale(), 0.0)
        got, most = ln.off(out[r][:, heads], want), ln.limits(want, DT[dt])
        print(f"{dt} size {size}: off by {got[0]:.3e} (limit {most[0]:.3e}), rows {got[1]:.3e} ({most[1]:.3e})", flush=True)
        assert got[0] <= most[0] and got[1] <= most[1], (s, got, most)


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
