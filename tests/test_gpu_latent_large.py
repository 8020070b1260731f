"""The latent attention where a call's sizes are large."""
import pytest
import torch

import latent_norms as ln
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


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_expanded_form_of_131077_tokens(dt):
    """The same prompt in the expanded form: 513 tiles of each of 128 heads."""
    import akv
    announce(f"latent prefill, 131077 query tokens of 128 heads, {dt}")
    T, H, Dc, kv = 131077, 128, 256, 100
    g = torch.Generator(device="cuda").manual_seed(2)
    pool = akv.PagedLatentPool.empty(1, 7, Dc, 64, 16)
    pool.data.copy_(torch.randn(pool.data.shape, generator=g, device="cuda"))
    i = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    batch = akv.PagedBatch(torch.arange(7, dtype=torch.int32, device="cuda").view(1, 7), i(kv), i(0, T), T, T)
    q = torch.randn(T, H, 192, generator=g, device="cuda", dtype=dt)
    wk, wv = ((torch.randn(H, 128, Dc, generator=g, device="cuda") * Dc ** -0.5).to(dt) for _ in range(2))
    out = akv.latent_prefill(q, pool, batch, akv.LatentWeights(wk, wv), causal=False)
    # both sides of every tile's border, and what lies between now and then
    tokens = torch.tensor(sorted(set([t + d for t in range(0, T, 256) for d in (0, 255) if t + d < T] + list(range(0, T, 331)) + [T - 1])), device="cuda")
    heads = torch.tensor([0, 1, 63, 126, 127])
    rows = pool.data[0].flatten(0, 1)[:kv].double().cpu()
    got = out[tokens][:, heads.cuda()].double().cpu()
    want, _ = ref.prefill(q[tokens][:, heads.cuda()].double().cpu(), rows, wk.cpu()[heads].double(), wv.cpu()[heads].double(), SCALE, 0.0,
                          causal=False)
    off, most = ln.off(got, want), ln.limits(want, dt)
    assert off[0] <= most[0] and off[1] <= most[1], (off, most)
