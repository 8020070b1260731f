"""The paged 4-bit cache's operators together, as a serving loop runs them: prompts, decode
steps, forks that write on, importance, compaction, crops and the end of sequences, against
lists of quantized tokens in 64 bits; captured and replayed; on other streams."""
import numpy as np
import pytest
import torch

import paged_ref as ref
from gpu_util import announce

pytestmark = pytest.mark.gpu


def _parts(x, G):
    """What the cache holds of rows (n, H, D): code * scale and zero."""
    c, s, z = ref.quantize(x.double().cpu().numpy(), G)
    s, z = (np.repeat(a.astype(np.float64), G, axis=-1) for a in (s, z))
    return [c * s, z]


class Twin:
    """Every sequence's tokens of every layer as the reference holds them."""

    def __init__(self, cache, layers, G):
        self.cache, self.layers, self.G, self.kv = cache, layers, G, {}

    def add(self, s, like=None):
        self.kv[s] = [[a.copy() for a in self.kv[like][l]] if like is not None else None for l in range(self.layers)]

    def step(self, seqs, counts, Hq, seed, dtype):
        """One step of all layers; the last layer's queries, log-sums and batch."""
        H, D = self.cache.pool.heads, self.cache.pool.head_dim
        batch = self.cache.extend(seqs, counts)
        g = torch.Generator(device="cuda").manual_seed(seed)
        x = lambda h: torch.randn(sum(counts), h, D, generator=g, device="cuda").to(dtype)  # noqa: E731
        at = np.concatenate([[0], np.cumsum(counts)])
        for l in range(self.layers):
            k, v, q = x(H), x(H), x(Hq)
            self.cache.append(l, k, v, batch)
            out, lse = self.cache.attention(l, q, batch, return_lse=True)
            for i, (s, m) in enumerate(zip(seqs, counts)):
                r = slice(at[i], at[i + 1])
                new = _parts(k[r], self.G) + _parts(v[r], self.G)
                old = self.kv[s][l]
                self.kv[s][l] = new if old is None else [np.concatenate([a, b]) for a, b in zip(old, new)]
                kv = self.kv[s][l]
                if m == 0:
                    continue
                n = len(kv[0])
                e, el, b, bl = ref.attention(q[r].double().cpu().numpy(), kv[:2], kv[2:], D ** -0.5,
                                             np.arange(n - m, n) + 1, torch.finfo(dtype).eps / 2)
                assert (np.abs(out[r].double().cpu().numpy() - e) <= b).all(), (s, l)
                assert (np.abs(lse[r].double().cpu().numpy() - el) <= bl).all(), (s, l)
        return q, lse, batch

    def same(self, s):
        for l in range(self.layers):
            kv = self.kv[s][l]
            assert self.cache.get_seq_length(s) == (0 if kv is None else len(kv[0]))
            if kv is None:
                continue
            for got, c, z in zip(self.cache.get_kv(l, s, torch.float32), kv[::2], kv[1::2]):
                assert np.allclose(got.transpose(0, 1).double().cpu().numpy(), c + z, rtol=2.0 ** -24, atol=0)


@pytest.mark.parametrize("dtype,D,G,P,H,Hq", [(torch.float16, 128, 32, 16, 2, 12), (torch.bfloat16, 64, 64, 32, 4, 4)])
def test_a_serving_loop(dtype, D, G, P, H, Hq):
    import akv
    announce(f"serving loop {dtype} D={D} G={G} P={P}")
    L = 2
    cache = akv.PackedPagedCache(L, H, D, page_size=P, max_pages=40, group_size=G)
    t = Twin(cache, L, G)
    a, b, c = (cache.add_sequence() for _ in range(3))
    for s in (a, b, c):
        t.add(s)
    t.step([a, b, c], [70, 1, 33], Hq, 1, dtype)          # prompts
    t.step([a, b, c], [1, 1, 0], Hq, 2, dtype)            # a decode step, one sequence idle
    d, e = cache.fork(a, 2)
    free = cache.num_free_pages
    for s in (d, e):
        t.add(s, like=a)
    t.step([d, b, a, e], [1, 1, 1, 3], Hq, 3, dtype)      # forks write on: two of the three copy the last page
    assert free - cache.num_free_pages == 2
    for s in (a, b, c, d, e):
        t.same(s)
    # the importance of a step says what stays: the first four tokens and the best others
    q, lse, batch = t.step([a, d], [1, 1], Hq, 4, dtype)
    n = [cache.get_seq_length(s) for s in (a, d)]
    scores = torch.zeros(2, max(n), device="cuda")
    cache.importance(L - 1, q, lse, batch, scores, decay=0.9)
    assert torch.allclose(scores.sum(dim=1), torch.ones(2, device="cuda"), atol=1e-4)
    scores[:, :4] = 10.0
    keep = [scores[i, :n[i]].topk(40).indices.sort().values for i in range(2)]
    cache.compact([a, d], keep)
    for s, k in zip((a, d), keep):
        t.kv[s] = [[x[k.cpu().numpy()] for x in kv] for kv in t.kv[s]]
    for s in (a, b, c, d, e):                               # e still reads the pages it shared
        t.same(s)
    cache.crop(e, 50)
    t.kv[e] = [[x[:50] for x in kv] for kv in t.kv[e]]
    t.step([a, b, d, e], [2, 1, 1, 1], Hq, 5, dtype)
    for s in (a, b, c, d, e):
        t.same(s)
        cache.remove(s)
    assert cache.num_free_pages == 40


def test_compaction_in_turns_and_refusals_leave_the_cache_whole():
    import akv
    announce("compaction with few free pages")
    cache = akv.PackedPagedCache(1, 1, 64, page_size=16, max_pages=12, group_size=32)
    t = Twin(cache, 1, 32)
    s = [cache.add_sequence() for _ in range(3)]
    for x in s:
        t.add(x)
    t.step(s, [48, 64, 50], 2, 1, torch.float16)            # 3 + 4 + 4 of 12 pages
    keep = [torch.arange(0, 48, 3, device="cuda"), torch.arange(1, 49, device="cuda"), torch.arange(0, device="cuda")]
    with pytest.raises(RuntimeError, match="exhausted"):
        cache.compact(s[:1], [torch.arange(48, device="cuda")])
    with pytest.raises(RuntimeError, match="exhausted"):
        cache.extend(s, [40, 0, 0])
    with pytest.raises(ValueError):
        cache.compact(s[:1], [torch.arange(49, device="cuda")])
    with pytest.raises(RuntimeError):
        cache.compact(s[:1], [torch.arange(5)])
    with pytest.raises(ValueError):
        cache.compact(s[:1], [torch.zeros(2, 2, dtype=torch.int64, device="cuda")])
    for x in s:
        t.same(x)
    cache.compact(s, keep)                                  # one page, then three of the four freed, then none
    for x, k in zip(s, keep):
        t.kv[x] = [[y[k.cpu().numpy()] for y in t.kv[x][0]]]
        t.same(x)
    assert cache.num_free_pages == 12 - 1 - 3
    t.step(s, [1, 1, 1], 2, 2, torch.float16)


def _world(seed=0, layers=2, S=3, D=128, H=2, P=16):
    """A pool, tables for up to 160 tokens a sequence, and tokens already there."""
    import akv
    g = torch.Generator(device="cuda").manual_seed(seed)
    pool = akv.PagedPool.empty(layers, 10 * S, H, D, P)
    table = torch.randperm(10 * S, generator=g, device="cuda").to(torch.int32).view(S, 10)
    lens = torch.tensor([30, 1, 97][:S], dtype=torch.int32, device="cuda")
    starts = torch.cat([lens.new_zeros(1), lens.cumsum(0).to(torch.int32)])
    T = int(starts[-1])
    first = akv.PagedBatch(table, lens, starts, T, int(lens.max()))
    for l in range(layers):
        akv.paged_append(pool, first, *(torch.randn(T, H, D, generator=g, device="cuda").half() for _ in range(2)), layer=l)
    batch = akv.PagedBatch(table, lens.clone(), torch.arange(S + 1, dtype=torch.int32, device="cuda"), S, 1)
    return pool, batch, torch.zeros(layers, S, 160, device="cuda")


def _step(pool, batch, scores, x, Hq=8):
    """One decode step of all layers on the rows x (layers, S, Hq + 2 H, D); lengths grow on the device."""
    import akv
    batch.kv_lens.add_(1)
    outs = []
    H = pool.heads
    for l in range(pool.num_layers):
        akv.paged_append(pool, batch, x[l, :, Hq:Hq + H], x[l, :, Hq + H:], layer=l)
        out, lse = akv.paged_attention(x[l, :, :Hq], pool, batch, l, return_lse=True)
        akv.paged_importance(x[l, :, :Hq], lse, pool, batch, scores[l], l)
        outs.append(out)
    return torch.stack(outs)


def test_captured_steps_follow_the_lengths():
    """Two graphs on one pool, each with buffers of its own, replayed in turn with eager work
    between them, against eager steps."""
    announce("captured decode steps")
    S, Hq, H, D, L = 3, 8, 2, 128, 2
    eager, cap = _world(), _world()
    xs = [torch.randn(L, S, Hq + 2 * H, D, device="cuda").half() for _ in range(2)]
    warm = _world(1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _step(*warm, xs[0])
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for x in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_step(*cap, x))
        graphs.append(g)
    assert torch.equal(cap[1].kv_lens, eager[1].kv_lens) and torch.equal(cap[0].data, eager[0].data)
    for i in range(8):
        x = torch.randn(L, S, Hq + 2 * H, D, device="cuda").half()
        xs[i % 2].copy_(x)
        graphs[i % 2].replay()
        want = _step(*eager, x)
        assert torch.equal(outs[i % 2], want), i
        assert torch.equal(cap[0].data, eager[0].data) and torch.equal(cap[2], eager[2]), i
        assert torch.equal(cap[1].kv_lens, eager[1].kv_lens)


def test_other_streams():
    announce("steps on other streams")
    x = torch.randn(2, 3, 12, 128, device="cuda").half()
    a, b = _world(), _world()
    want = _step(*a, x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(2_000_000)
        got = _step(*b, x)
    assert not side.query()      # the work went to the side stream, behind the wait
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want) and torch.equal(a[0].data, b[0].data) and torch.equal(a[2], b[2])


def test_python_refusals():
    import akv
    announce("paged refusals")
    pool, batch, scores = _world()
    q, kv = torch.zeros(3, 8, 128, device="cuda").half(), torch.zeros(3, 2, 128, device="cuda").half()
    lse = torch.zeros(3, 8, device="cuda")
    for err, call in (
        (RuntimeError, lambda: akv.paged_attention(q.cpu(), pool, batch)),
        (TypeError, lambda: akv.paged_attention(q.float(), pool, batch)),
        (ValueError, lambda: akv.paged_attention(q[:2], pool, batch)),
        (ValueError, lambda: akv.paged_attention(q[0], pool, batch)),
        (ValueError, lambda: akv.paged_attention(q[:, :3], pool, batch)),
        (ValueError, lambda: akv.paged_attention(q, pool, batch, layer=2)),
        (ValueError, lambda: akv.paged_attention(q, pool, batch, sm_scale=0.0)),
        (ValueError, lambda: akv.paged_append(pool, batch, kv[:, :1], kv)),
        (TypeError, lambda: akv.paged_append(pool, batch, kv, kv.float())),
        (TypeError, lambda: akv.paged_append(pool, batch, kv.double(), kv.double())),
        (RuntimeError, lambda: akv.paged_append(pool, batch, kv.cpu(), kv)),
        (TypeError, lambda: akv.paged_read(pool, batch, dtype=torch.int32)),
        (ValueError, lambda: akv.paged_importance(q, lse[:, :2], pool, batch, scores[0])),
        (ValueError, lambda: akv.paged_importance(q, lse.half(), pool, batch, scores[0])),
        (ValueError, lambda: akv.paged_importance(q, lse, pool, batch, scores[0, :2])),
        (ValueError, lambda: akv.paged_importance(q, lse, pool, batch, scores[0].double())),
        (ValueError, lambda: akv.paged_importance(q, lse, pool, batch, scores[0], out=scores[0, :, :5])),
        (ValueError, lambda: akv.paged_importance(q, lse, pool, batch, scores[0], q_window=-1)),
        (ValueError, lambda: akv.copy_pages(pool, torch.zeros(2, device="cuda"), torch.zeros(2, device="cuda"))),
        (ValueError, lambda: akv.copy_pages(pool, batch.kv_lens[:2], batch.kv_lens[:1])),
        (RuntimeError, lambda: akv.copy_pages(pool, torch.zeros(1, dtype=torch.int32), batch.kv_lens[:1])),
        (ValueError, lambda: akv.compact_pages(pool, batch.page_table[:2], batch.page_table, batch.page_table, batch.kv_lens)),
        (ValueError, lambda: akv.PagedBatch(batch.page_table, batch.kv_lens, batch.kv_lens, 3, 1)),
        (ValueError, lambda: akv.PagedBatch(batch.page_table, batch.kv_lens, batch.q_starts, 3, 4)),
        (ValueError, lambda: akv.PagedBatch(batch.page_table.float(), batch.kv_lens, batch.q_starts, 3, 1)),
        (ValueError, lambda: akv.PagedPool(pool.data.transpose(0, 1), 128)),
        (ValueError, lambda: akv.PagedPool(pool.data, 128, 64)),
    ):
        with pytest.raises(err):
            call()


def test_empty_calls():
    import akv
    announce("paged calls without sequences, rows or pages")
    z = lambda *n: torch.zeros(*n, dtype=torch.int32, device="cuda")  # noqa: E731
    pool = akv.PagedPool.empty(1, 0, 2, 128)
    for S in (0, 2):
        none = akv.PagedBatch(z(S, 0), z(S), z(S + 1), 0, 0)
        q, kv = torch.empty(0, 4, 128, device="cuda").half(), torch.empty(0, 2, 128, device="cuda").half()
        assert akv.paged_attention(q, pool, none).shape == (0, 4, 128)
        akv.paged_append(pool, none, kv, kv)
        assert akv.paged_read(pool, none)[0].shape == (0, 2, 128)
        scores = torch.rand(S, 5, device="cuda")
        out = akv.paged_importance(q, torch.empty(0, 4, device="cuda"), pool, none, scores, out=torch.zeros_like(scores))
        assert torch.equal(out, scores)
    one = akv.PagedBatch(z(1, 0), z(1), torch.tensor([0, 2], dtype=torch.int32, device="cuda"), 2, 2)
    out, lse = akv.paged_attention(torch.ones(2, 4, 128, device="cuda").half(), pool, one, return_lse=True)
    assert not bool(out.any()) and bool(lse.isneginf().all())
    akv.copy_pages(pool, z(0), z(0))
    akv.compact_pages(pool, z(0, 1), z(0, 1), z(0, 4), z(0))
    akv.compact_pages(pool, z(2, 1), z(2, 1), z(2, 0), z(2))


def test_compaction_refuses_positions_that_are_no_tokens():
    """A position at or behind a sequence's length would move a stale slot into it, a negative one none at
    all: refused before anything moves, whatever the lists' types, and however the turns fall."""
    import akv
    announce("compaction, positions out of range")
    cache = akv.PackedPagedCache(2, 1, 64, page_size=16, max_pages=10, group_size=32)
    t = Twin(cache, 2, 32)
    s = [cache.add_sequence() for _ in range(3)]
    for x in s:
        t.add(x)
    t.step(s, [40, 20, 0], 2, 1, torch.float16)
    free = cache.num_free_pages
    one = lambda *x, dtype=torch.int64: torch.tensor(x, dtype=dtype, device="cuda")  # noqa: E731
    good = one(0, 5, 39), one(19, dtype=torch.int32), one()
    for i, bad in ((0, one(1, 40)), (0, one(-1, 3, dtype=torch.int32)), (1, one(20, dtype=torch.int32)), (1, one(2 ** 32 + 1)),
                   (0, one(47)), (1, one(0, 10 ** 9, dtype=torch.int32))):
        keep = list(good)
        keep[i] = bad
        with pytest.raises(ValueError, match="position"):
            cache.compact(s, keep)
        assert cache.num_free_pages == free
        for x in s:
            t.same(x)
    cache.compact(s, good)
    for x, k in zip(s, good):
        if t.kv[x][0] is not None:
            t.kv[x] = [[y[k.cpu().numpy()] for y in kv] for kv in t.kv[x]]
        t.same(x)
    cache.compact([], [])
