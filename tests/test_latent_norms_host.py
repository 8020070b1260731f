"""What the norms of latent_norms tell apart, on the host."""
import pytest
import torch

import latent_norms as ln
import latent_ref as ref

SCALE = 192 ** -0.5


def _inputs(m, kv, H, size, dtype, Dc=256):
    g = torch.Generator().manual_seed(8)
    r = lambda *n: torch.randn(*n, generator=g)  # noqa: E731
    rows = r(kv, Dc + 64)
    rows[:, 3] *= 6.0
    rows[:, Dc + 5] *= 3.0
    q = (r(m, H, 192) * size).to(dtype).double()
    return q, rows.half().double(), *((r(H, 128, Dc) * Dc ** -0.5).to(dtype).double() for _ in range(2))


def _within(x, dtype, **kw):
    want, _ = ref.prefill(*x, SCALE, 0.0)
    a, b = ln.off(ln.expanded(*x, SCALE, dtype, **kw), want)
    la, lb = ln.limits(want, dtype)
    return a <= la and b <= lb


@pytest.mark.parametrize("m,kv,H,size", [(50, 300, 4, 1.0), (50, 300, 4, 4.0), (20, 3000, 2, 4.0)])
def test_float16(m, kv, H, size):
    x = _inputs(m, kv, H, size, torch.float16)
    assert _within(x, torch.float16)
    for wrong in (dict(keys=1), dict(values=1), dict(p=1), dict(rest=lambda v: -v), dict(rest=lambda v: v.roll(16, 1)),
                  dict(rest=lambda v: v.roll(1, 2)), dict(skip=0), dict(skip=kv // 2), dict(skip=kv - m)):
        assert not _within(x, torch.float16, **wrong), wrong


@pytest.mark.parametrize("m,kv,H", [(50, 300, 4), (20, 6000, 1)])
def test_bfloat16(m, kv, H):
    x = _inputs(m, kv, H, 1.0, torch.bfloat16)
    assert _within(x, torch.bfloat16, keys=1, values=1, p=1)
    for token in (0, kv // 2, kv - m):
        assert not _within(x, torch.bfloat16, keys=1, values=1, p=1, skip=token), token
