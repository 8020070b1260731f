"""The latent attention where a call's sizes are large."""
import pytest
import torch

import latent_ref as ref
from gpu_util import announce

pytestmark = pytest.mark.gpu

SCALE = 192 ** -0.5


def test_attention_of_2_to_the_24_rows_and_more():
    """A prompt of 131077 tokens and 128 heads, an item a token: a join launched for every row that the call may have
    would be more than 2^32 work items, and wrap.  Workgroups share some 250 items, at the runs' borders; those
    are looked at, and 500 others."""
    import akv
    announce("latent attention, 131077 query tokens of 128 heads")
    T, H, Dc, kv = 131077, 128, 512, 100
    g = torch.Generator(device="cuda").manual_seed(1)
    pool = akv.PagedLatentPool.empty(1, 7, Dc, 64, 16)
    pool.data.copy_(torch.randn(pool.data.shape, generator=g, device="cuda"))
    i = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    batch = akv.PagedBatch(torch.arange(7, dtype=torch.int32, device="cuda").view(1, 7), i(kv), i(0, T), T, T)
    x = torch.randn(T, H, Dc + 64, generator=g, device="cuda", dtype=torch.bfloat16)
    out, lse = akv.latent_attention(x[..., :Dc], x[..., Dc:], pool, batch, SCALE, causal=False, return_lse=True)
    # an item costs its two units of 64 tokens and five more
    total, groups = T * 7, 256
    share = -(-total // groups)
    shared = [r * share // 7 for r in range(1, groups) if r * share % 7]
    assert len(shared) > 200
    tokens = torch.tensor(sorted(set(shared + list(range(0, T, 263)) + [T - 1])), device="cuda")
    heads = torch.arange(len(tokens), device="cuda") * 37 % H
    q = x[tokens, heads].double().cpu()[:, None]
    rows = pool.data[0].flatten(0, 1)[:kv].double().cpu()
    e, el, b, bl = ref.attention(q[..., :Dc], q[..., Dc:], rows, SCALE, 2.0 ** -8, causal=False)
    assert bool(((out[tokens, heads].double().cpu() - e[:, 0]).abs() <= b[:, 0]).all())
    assert bool(((lse[tokens, heads].double().cpu() - el[:, 0]).abs() <= bl[:, 0]).all())
