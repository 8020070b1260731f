"""The latent importance where rows see every token, where pages are missing and beside rows of no sequence."""
import pytest
import torch

import latent_ref as ref
from gpu_util import announce
from test_gpu_latent import World, _queries, _scale

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("H,kv,q,win,holes", [(4, [200, 0, 33], [4, 0, 1], 0, ()), (4, [200, 40], [4, 1], 2, ((0, 3), (1, 0))),
                                              (40, [200, 70], [9, 1], 0, ()), (40, [300, 64, 17], [20, 3, 17], 5, ((0, 2), (0, 18), (1, 1), (2, 0))),
                                              (128, [90], [30], 0, ((0, 0),))])
def test_importance(H, kv, q, win, holes, causal, dt):
    import akv
    announce(f"latent importance H={H} kv={kv} q={q} win={win} causal={causal} holes={holes} {dt}")
    Dc, P = 512, 16
    w = World(Dc, P, kv, q)
    w.fill()
    stay = [torch.ones(n, dtype=torch.bool) for n in kv]
    for s, page in holes:
        w.batch.page_table[s, page] = 2 ** 30
        stay[s][page * P:(page + 1) * P] = False
    q_, qr, x = _queries(w, H, dt)
    _, lse = akv.latent_attention(q_, qr, w.pool, w.batch, _scale(), causal=causal, return_lse=True)
    old = torch.rand(len(kv), max(kv), generator=torch.Generator().manual_seed(1))
    scores = old.cuda()
    akv.latent_importance(q_, qr, lse, w.pool, w.batch, scores, _scale(), decay=0.5, q_window=win, causal=causal)
    scores, old = scores.double().cpu(), old.double()
    for s, n in enumerate(kv):
        assert torch.equal(scores[s, n:], old[s, n:])
        if not w.q[s]:
            assert torch.equal(scores[s], old[s])
            continue
        r, rows, l = w.mine(s), w.rows(s), lse[w.mine(s)].double().cpu()
        want, bound = torch.zeros(n, dtype=torch.float64), torch.zeros(n, dtype=torch.float64)
        for i in range(w.q[s] - min(win or w.q[s], w.q[s]), w.q[s]):  # row by row: what it sees of what is there
            see = min(n, n - w.q[s] + 1 + i) if causal else n
            some = torch.nonzero(stay[s][:see])[:, 0]
            at = slice(r.start + i, r.start + i + 1)
            _, el, _, bl = ref.attention(x[at, :, :Dc], x[at, :, Dc:], rows[some], _scale(), 0.0)
            none = torch.isneginf(el)
            assert torch.equal(torch.isneginf(l[i:i + 1]), none) and bool(((l[i:i + 1] - el).abs()[~none] <= bl[~none]).all())
            if len(some):
                e, b = ref.importance(x[at, :, :Dc], x[at, :, Dc:], rows[some], _scale(), l[i:i + 1], causal=False)
                want[some] += e
                bound[some] += b
        full = old[s, :n] * 0.5 + want
        assert bool(((scores[s, :n] - full).abs() <= bound + 2.0 ** -22 * full).all()), s
