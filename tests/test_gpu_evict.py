"""The eviction by accumulated attention weight against a plain sort."""
import pytest
import torch

import latent_ref as ref
from gpu_util import announce

pytestmark = pytest.mark.gpu


def _check(scores, lens, budget, first, last, max_keep=None):
    import akv
    b = budget if isinstance(budget, int) else torch.tensor(budget, dtype=torch.int32, device="cuda")
    keep, n_keep, kept = akv.evict_select(scores.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), b, first, last, max_keep)
    keep, n_keep, kept = keep.cpu(), n_keep.cpu(), kept.cpu()
    S, N = scores.shape
    assert kept.shape == (S, N)
    for s in range(S):
        want = ref.evict(scores[s], lens[s], min(budget if isinstance(budget, int) else budget[s], keep.shape[1]), first, last)
        assert int(n_keep[s]) == len(want), s
        assert keep[s, :len(want)].tolist() == want, s
        assert not bool(keep[s, len(want):].any())
        got, w = kept[s, :len(want)], scores[s][torch.tensor(want, dtype=torch.long)]
        assert torch.equal(torch.isnan(got), torch.isnan(w)) and torch.equal(got.nan_to_num(), w.nan_to_num())
        assert not bool(kept[s, len(want):].any())


def _scores(S, N, seed, kind="heavy"):
    g = torch.Generator().manual_seed(seed)
    x = torch.rand(S, N, generator=g)
    if kind == "heavy":
        x = x.pow(8) * 3
        x[x < 1e-6] = 0
    elif kind == "few values":
        x = (x * 4).floor()
    elif kind == "signed":
        x = torch.randn(S, N, generator=g) * 1e3
    elif kind == "equal":
        x = torch.full((S, N), 0.25)
    elif kind == "narrow":  # values that share their upper bits
        x = 1.0 + x * 2.0 ** -12
    return x


@pytest.mark.parametrize("kind", ["heavy", "few values", "signed", "equal", "narrow"])
@pytest.mark.parametrize("N", [1, 63, 1024, 2047, 2049, 8192, 8193, 33000])
def test_positions_and_scores(N, kind):
    announce(f"evict N={N} {kind}")
    x = _scores(6, N, N, kind)
    lens = [N, max(0, N - 1), N // 2, 1, 0, N]
    for budget, first, last in ((N // 2, 4, 16), (1, 0, 0), (0, 4, 4), (N, 4, 4), (N + 7, 0, 9), (max(1, N // 10), 0, 40)):
        _check(x, lens, budget, first, last)


def test_longer_than_a_workgroup_holds():
    announce("evict, long sequences")
    for kind in ("heavy", "few values", "narrow"):
        x = _scores(2, 100001, 7, kind)
        _check(x, [100001, 70000], 20000, 4, 64)
        _check(x, [100001, 40000], 99999, 0, 0)


def test_budgets_on_the_device():
    announce("evict, a budget each")
    x = _scores(5, 3000, 2)
    _check(x, [3000, 2000, 17, 0, 2999], [100, 2000, 40, 5, -3], 4, 8)
    _check(x, [3000, 2000, 17, 0, 2999], [100, 2000, 40, 5, 2 ** 31 - 1], 4, 8, max_keep=500)


def test_values_that_are_not_numbers():
    announce("evict, NaN and infinities")
    x = _scores(3, 400, 4, "signed")
    x[0, 5::9] = float("nan")
    x[1, ::3], x[1, 1::3] = float("inf"), float("-inf")
    x[2] = -x[2].abs()
    x[2, 7], x[2, 8], x[2, 9] = -0.0, 0.0, -0.0
    nan = torch.tensor([-1], dtype=torch.int32).view(torch.float32)  # a NaN of the other sign
    x[0, 50] = nan[0]
    for budget in (1, 2, 3, 30, 133, 134, 267, 399):
        _check(x, [400, 400, 400], budget, 0, 0)
        _check(x, [400, 390, 11], budget, 3, 5)


def test_protected_tokens_past_the_budget():
    announce("evict, more protected than the budget holds")
    x = _scores(4, 200, 5)
    _check(x, [200, 100, 30, 5], 10, 20, 0)
    _check(x, [200, 100, 30, 5], 10, 4, 50)
    _check(x, [200, 100, 30, 5], 10, 300, 300)


def test_rows_apart_and_replays():
    """Scores as columns of a larger buffer; captured, and replayed with other lengths and scores."""
    import akv
    announce("evict, strided and captured")
    S, N = 4, 5000
    buf = torch.zeros(S, 3 * N, device="cuda")
    view, lens, budget = buf[:, N:2 * N], torch.zeros(S, dtype=torch.int32, device="cuda"), torch.zeros(S, dtype=torch.int32, device="cuda")

    def run():
        return akv.evict_select(view, lens, 1500, 4, 32) + akv.evict_select(view, lens, budget, 0, 0, max_keep=999)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = run()
    for i in range(4):
        view.copy_(_scores(S, N, 20 + i, ["heavy", "few values", "signed", "narrow"][i]))
        lens.copy_(torch.tensor([N, 1499, 1501, 10 * i]))
        budget.copy_(torch.tensor([i, 900, 2000, 7]))
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, run()):
            assert torch.equal(a, b), i
        for k, (j, n) in enumerate(((0, 1500), (3, 999))):
            for s in range(S):
                want = ref.evict(view[s].cpu(), int(lens[s]), n if k == 0 else min(999, int(budget[s])), 4 if k == 0 else 0, 32 if k == 0 else 0)
                assert out[j][s, :len(want)].tolist() == want and int(out[j + 1][s]) == len(want)


def test_refusals():
    import akv
    announce("evict refusals")
    x, n = torch.zeros(3, 10, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    for err, call in (
        (RuntimeError, lambda: akv.evict_select(x.cpu(), n, 4)),
        (RuntimeError, lambda: akv.evict_select(x, n.cpu(), 4)),
        (RuntimeError, lambda: akv.evict_select(x, n, n.cpu())),
        (ValueError, lambda: akv.evict_select(x.half(), n, 4)),
        (ValueError, lambda: akv.evict_select(x[0], n, 4)),
        (ValueError, lambda: akv.evict_select(x, n[:2], 4)),
        (ValueError, lambda: akv.evict_select(x, n, n[:2])),
        (ValueError, lambda: akv.evict_select(x, n.float(), 4)),
        (ValueError, lambda: akv.evict_select(x, n, -1)),
        (ValueError, lambda: akv.evict_select(x, n, n, max_keep=-1)),
        (ValueError, lambda: akv.evict_select(x, n, 4, -1, 0)),
        (ValueError, lambda: akv.evict_select(x, n, 4, 0, -1)),
        (TypeError, lambda: akv.evict_select(x, n, 4.5)),
    ):
        with pytest.raises(err):
            call()
    for S, N in ((0, 5), (3, 0), (0, 0)):
        keep, k, kept = akv.evict_select(torch.zeros(S, N, device="cuda"), torch.zeros(S, dtype=torch.int32, device="cuda"), 4)
        assert keep.shape == (S, min(4, N)) and not bool(k.any()) and kept.shape == (S, N)
