"""The paged latent cache's operators together, as a serving loop runs them: prompts in both forms of
the attention, decode steps, forks that write on, importance, evictions, crops and the end of
sequences, against lists of rows in 64 bits; the 4-bit cache's eviction; captured and replayed; on
other streams and from several at once."""
import pytest
import torch

import latent_ref as ref
from gpu_util import announce

pytestmark = pytest.mark.gpu

DR = 64
SCALE = 192 ** -0.5


class Twin:
    """Every sequence's rows of every layer as the reference holds them."""

    def __init__(self, cache, H, dtype):
        self.cache, self.H, self.dtype, self.kv = cache, H, dtype, {}
        self.layers, self.Dc = cache.pool.num_layers, cache.pool.latent_dim
        g = torch.Generator().manual_seed(77)
        r = lambda: (torch.randn(H, 128, self.Dc, generator=g) * self.Dc ** -0.5).to(dtype)  # noqa: E731
        import akv
        self.w = [(r(), r()) for _ in range(self.layers)]
        self.weights = [akv.LatentWeights(a.cuda(), b.cuda()) for a, b in self.w]

    def add(self, s, like=None):
        self.kv[s] = [self.kv[like][l].clone() if like is not None else torch.zeros(0, self.Dc + DR, dtype=torch.float64)
                      for l in range(self.layers)]

    def step(self, seqs, counts, seed, prefill=False):
        """One step of all layers; the last layer's queries, log-sums and batch.  Both forms compute the same."""
        batch = self.cache.extend(seqs, counts)
        g = torch.Generator().manual_seed(seed)
        T, half = sum(counts), torch.finfo(self.dtype).eps / 2
        at = [0]
        for c in counts:
            at.append(at[-1] + c)
        for l in range(self.layers):
            x = torch.randn(T, self.Dc + DR, generator=g).to(self.dtype)
            q = torch.randn(T, self.H, 128 + DR, generator=g).to(self.dtype)
            wk, wv = self.w[l]
            ql = torch.matmul(q[..., :128].float().transpose(0, 1), wk.float()).transpose(0, 1).to(self.dtype)
            self.cache.append(l, x[:, :self.Dc].cuda(), x[:, self.Dc:].cuda(), batch)
            out, lse = self.cache.attention(l, ql.cuda(), q[..., 128:].cuda(), batch, SCALE, return_lse=True)
            pre = self.cache.prefill(l, q.cuda(), batch, self.weights[l]) if prefill else None
            for i, (s, m) in enumerate(zip(seqs, counts)):
                r = slice(at[i], at[i + 1])
                self.kv[s][l] = torch.cat([self.kv[s][l], ref.held(x[r].double())[0].double()])
                if m == 0:
                    continue
                rows = self.kv[s][l]
                e, el, b, bl = ref.attention(ql[r].double(), q[r, :, 128:].double(), rows, SCALE, half)
                assert bool(((out[r].double().cpu() - e).abs() <= b).all()), (s, l)
                assert bool(((lse[r].double().cpu() - el).abs() <= bl).all()), (s, l)
                if prefill:
                    e, b = ref.prefill(q[r].double(), rows, wk.double(), wv.double(), SCALE, half)
                    assert bool(((pre[r].double().cpu() - e).abs() <= b).all()), (s, l)
        return ql.cuda(), q[..., 128:].cuda(), lse, batch

    def same(self, s):
        for l in range(self.layers):
            want = self.kv[s][l]
            assert self.cache.get_seq_length(s) == len(want)
            if len(want):
                assert torch.equal(torch.cat(self.cache.get_rows(l, s), -1).double().cpu(), want), (s, l)


@pytest.mark.parametrize("dtype,Dc,P,H", [(torch.float16, 512, 16, 16), (torch.bfloat16, 256, 32, 5), (torch.bfloat16, 512, 64, 40)])
def test_a_serving_loop(dtype, Dc, P, H):
    import akv
    announce(f"latent serving loop {dtype} Dc={Dc} P={P} H={H}")
    L = 2
    pages = 60 * 16 // P
    cache = akv.PagedLatentCache(L, Dc, DR, page_size=P, max_pages=pages)
    t = Twin(cache, H, dtype)
    a, b, c = (cache.add_sequence() for _ in range(3))
    for s in (a, b, c):
        t.add(s)
    t.step([a, b, c], [130, 1, 33], 1, prefill=True)      # prompts
    t.step([a, b, c], [1, 1, 0], 2)                       # a decode step, one sequence idle
    d, e = cache.fork(a, 2)
    for s in (d, e):
        t.add(s, like=a)
    t.step([d, b, a, e], [1, 1, 1, 3], 3)                 # forks write on
    for s in (a, b, c, d, e):
        t.same(s)
    # the importance of some steps says what stays
    seqs = [a, d, b]
    scores = torch.zeros(3, 160, device="cuda")
    for i in range(3):
        q, qr, lse, batch = t.step(seqs, [1, 2, 1], 4 + i, prefill=i == 1)
        akv_scores = cache.importance(L - 1, q, qr, lse, batch, scores, SCALE, decay=1.0)
        assert akv_scores is scores
    want = torch.tensor([3.0, 6.0, 3.0])                  # a row's weights add up to one
    assert torch.allclose(scores.sum(dim=1).cpu(), want, atol=1e-3)
    n = [cache.get_seq_length(s) for s in seqs]
    keep = [ref.evict(scores[i].cpu(), n[i], 50, 4, 8) for i in range(3)]
    kept = cache.evict(seqs, scores, 50, protect_initial=4, protect_recent=8)
    for i, (s, k) in enumerate(zip(seqs, keep)):
        k = torch.tensor(k, dtype=torch.long)
        t.kv[s] = [x[k] for x in t.kv[s]]
        assert torch.equal(kept[i, :len(k)].cpu(), scores[i].cpu()[k]) and not bool(kept[i, len(k):].any())
    assert [cache.get_seq_length(s) for s in seqs] == [50, 50, n[2]]
    for s in (a, b, c, d, e):                             # e still reads the pages it shared
        t.same(s)
    cache.compact([e], [torch.arange(0, 131, 3, device="cuda")])
    t.kv[e] = [x[torch.arange(0, 131, 3)] for x in t.kv[e]]
    cache.crop(e, 30)
    t.kv[e] = [x[:30] for x in t.kv[e]]
    t.step([a, b, d, e], [2, 1, 40, 1], 9, prefill=True)
    for s in (a, b, c, d, e):
        t.same(s)
        cache.remove(s)
    assert cache.num_free_pages == pages


def test_eviction_of_the_4_bit_cache():
    import akv
    announce("4-bit cache, eviction")
    cache = akv.PackedPagedCache(2, 2, 64, page_size=16, max_pages=24, group_size=32)
    s = [cache.add_sequence() for _ in range(3)]
    batch = cache.extend(s, [100, 20, 70])
    g = torch.Generator(device="cuda").manual_seed(1)
    for l in range(2):
        cache.append(l, *(torch.randn(190, 2, 64, generator=g, device="cuda").half() for _ in range(2)), batch)
    q = torch.randn(190, 8, 64, generator=g, device="cuda").half()
    _, lse = cache.attention(1, q, batch, return_lse=True)
    scores = cache.importance(1, q, lse, batch, torch.zeros(3, 100, device="cuda"), decay=1.0)
    before = [[[x.clone() for x in cache.get_kv(l, i)] for l in range(2)] for i in s]
    keep = [ref.evict(scores[i].cpu(), n, 33, 4, 16) for i, n in enumerate((100, 20, 70))]
    kept = cache.evict(s, scores, 33)
    assert [cache.get_seq_length(i) for i in s] == [33, 20, 33] and cache.num_free_pages == 24 - 3 - 2 - 3
    for i in range(3):
        k = torch.tensor(keep[i], device="cuda")
        assert torch.equal(kept[i, :len(k)], scores[i, k])
        for l in range(2):
            for x, y in zip(cache.get_kv(l, s[i]), before[i][l]):
                assert torch.equal(x, y[:, k])


def _world(seed=0, layers=2, S=3, Dc=512, P=16):
    """A pool, tables for up to 160 tokens a sequence, and tokens already there."""
    import akv
    g = torch.Generator(device="cuda").manual_seed(seed)
    pool = akv.PagedLatentPool.empty(layers, 10 * S, Dc, DR, P)
    table = torch.randperm(10 * S, generator=g, device="cuda").to(torch.int32).view(S, 10)
    lens = torch.tensor([30, 1, 97][:S], dtype=torch.int32, device="cuda")
    starts = torch.cat([lens.new_zeros(1), lens.cumsum(0).to(torch.int32)])
    T = int(starts[-1])
    first = akv.PagedBatch(table, lens, starts, T, int(lens.max()))
    for l in range(layers):
        x = torch.randn(T, Dc + DR, generator=g, device="cuda").half()
        akv.latent_append(pool, first, x[:, :Dc], x[:, Dc:], layer=l)
    batch = akv.PagedBatch(table, lens.clone(), torch.arange(S + 1, dtype=torch.int32, device="cuda"), S, 1)
    w = akv.LatentWeights(*(torch.randn(16, 128, Dc, generator=g, device="cuda") * Dc ** -0.5 for _ in range(2)))
    return pool, batch, torch.zeros(layers, S, 160, device="cuda"), w


def _step(pool, batch, scores, w, x, H=16):
    """One decode step of all layers on the rows x (layers, S, 2 H + 1, Dc + Dr); lengths grow on the device."""
    import akv
    batch.kv_lens.add_(1)
    outs, D = [], pool.latent_dim
    for l in range(pool.num_layers):
        akv.latent_append(pool, batch, x[l, :, -1, :D], x[l, :, -1, D:], layer=l)
        out, lse = akv.latent_attention(x[l, :, :H, :D], x[l, :, :H, D:], pool, batch, SCALE, l, return_lse=True)
        akv.latent_importance(x[l, :, :H, :D], x[l, :, :H, D:], lse, pool, batch, scores[l], SCALE, l)
        outs.append(torch.cat([out, akv.latent_prefill(x[l, :, H:2 * H, :192], pool, batch, w, l)], -1))
    keep, n, kept = akv.evict_select(scores[0], batch.kv_lens, 40, 2, 4)
    return torch.stack(outs), keep, n, kept


def test_captured_steps_follow_the_lengths():
    """Two graphs on one pool, each with buffers of its own, replayed in turn with eager work
    between them, against eager steps."""
    announce("captured latent steps")
    S, H, L = 3, 16, 2
    rows = lambda: torch.randn(L, S, 2 * H + 1, 576, device="cuda").half()  # noqa: E731
    eager, cap = _world(), _world()
    xs = [rows() for _ in range(2)]
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
        xs[i % 2].copy_(rows())
        graphs[i % 2].replay()
        want = _step(*eager, xs[i % 2])
        torch.cuda.synchronize()
        for a, b in zip(outs[i % 2], want):
            assert torch.equal(a, b), i
        assert torch.equal(cap[0].data, eager[0].data) and torch.equal(cap[2], eager[2]), i
        assert torch.equal(cap[1].kv_lens, eager[1].kv_lens)


def test_other_streams():
    announce("latent steps on other streams")
    x = torch.randn(2, 3, 33, 576, device="cuda").half()
    a, b = _world(), _world()
    want = _step(*a, x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(2_000_000)
        got = _step(*b, x)
    assert not side.query()      # the work went to the side stream, behind the wait
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(got, want)) and torch.equal(a[0].data, b[0].data) and torch.equal(a[2], b[2])


def test_one_batch_on_two_streams_at_once():
    """Calls of one batch object on two streams have workspaces of their own."""
    import akv
    announce("latent calls on two streams at once")
    pool = akv.PagedLatentPool.empty(1, 300)
    n = 18000
    table = torch.randperm(300, device="cuda").to(torch.int32).view(1, 300)
    i = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    x = torch.randn(n, 576, device="cuda").half()
    akv.latent_append(pool, akv.PagedBatch(table, i(n), i(0, n), n, n), x[:, :512], x[:, 512:])
    batch = akv.PagedBatch(table, i(n), i(0, 1), 1, 1)
    w = akv.LatentWeights(*(torch.randn(64, 128, 512, device="cuda") * 512 ** -0.5 for _ in range(2)))
    qs = [torch.randn(1, 64, 576, device="cuda").half() for _ in range(2)]
    run = lambda q: (akv.latent_attention(q[..., :512], q[..., 512:], pool, batch, SCALE), akv.latent_prefill(q[..., :192], pool, batch, w))  # noqa: E731
    want = [run(q) for q in qs]
    sides = [torch.cuda.Stream() for _ in qs]
    for _ in range(5):
        got = []
        for s, q in zip(sides, qs):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(run(q))
        for s in sides:
            torch.cuda.current_stream().wait_stream(s)
        for a, b in zip(got, want):
            assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_python_refusals():
    import akv
    announce("latent refusals")
    pool, batch, scores, w = _world()
    q, qr = torch.zeros(3, 16, 512, device="cuda").half(), torch.zeros(3, 16, 64, device="cuda").half()
    c, r = torch.zeros(3, 512, device="cuda").half(), torch.zeros(3, 64, device="cuda").half()
    qe, lse = torch.zeros(3, 16, 192, device="cuda").half(), torch.zeros(3, 16, device="cuda")
    w256 = akv.LatentWeights(*(torch.zeros(16, 128, 256, device="cuda") for _ in range(2)))
    attend = lambda q=q, qr=qr, **k: akv.latent_attention(q, qr, pool, batch, k.pop("scale", SCALE), **k)  # noqa: E731
    imp = lambda lse=lse, s=scores[0], **k: akv.latent_importance(q, qr, lse, pool, batch, s, SCALE, **k)  # noqa: E731
    for err, call in (
        (RuntimeError, lambda: attend(q=q.cpu())), (RuntimeError, lambda: attend(qr=qr.cpu())), (TypeError, lambda: attend(q=q.float())),
        (TypeError, lambda: attend(qr=qr.bfloat16())), (ValueError, lambda: attend(q=q[:2])), (ValueError, lambda: attend(qr=qr[:, :5])),
        (ValueError, lambda: attend(q=q[0])), (ValueError, lambda: attend(q=q[..., :256])), (ValueError, lambda: attend(layer=2)),
        (ValueError, lambda: attend(scale=0.0)), (ValueError, lambda: attend(scale=float("nan"))),
        (ValueError, lambda: akv.latent_append(pool, batch, c[:2], r)), (ValueError, lambda: akv.latent_append(pool, batch, c, r[:, :32])),
        (TypeError, lambda: akv.latent_append(pool, batch, c, r.float())), (TypeError, lambda: akv.latent_append(pool, batch, c.double(), r.double())),
        (RuntimeError, lambda: akv.latent_append(pool, batch, c.cpu(), r)), (TypeError, lambda: akv.latent_read(pool, batch, dtype=torch.int32)),
        (ValueError, lambda: akv.latent_read(pool, batch, layer=-1)),
        (ValueError, lambda: akv.latent_prefill(qe[:, :8], pool, batch, w)), (ValueError, lambda: akv.latent_prefill(qe[..., :128], pool, batch, w)),
        (TypeError, lambda: akv.latent_prefill(qe.float(), pool, batch, w)), (ValueError, lambda: akv.latent_prefill(qe, pool, batch, w256)),
        (ValueError, lambda: akv.latent_prefill(qe, pool, batch, w, sm_scale=-1.0)), (RuntimeError, lambda: akv.latent_prefill(qe.cpu(), pool, batch, w)),
        (ValueError, lambda: imp(lse=lse[:, :2])), (ValueError, lambda: imp(lse=lse.half())), (ValueError, lambda: imp(s=scores[0, :2])),
        (ValueError, lambda: imp(s=scores[0].double())), (ValueError, lambda: imp(out=scores[0, :, :5])), (ValueError, lambda: imp(q_window=-1)),
        (ValueError, lambda: imp(s=scores[0, :, :100], out=scores[0, :, 1:101])),
        (NotImplementedError, lambda: akv.LatentWeights(torch.zeros(2, 64, 512, device="cuda"), torch.zeros(2, 64, 512, device="cuda"))),
        (NotImplementedError, lambda: akv.LatentWeights(torch.zeros(2, 128, 384, device="cuda"), torch.zeros(2, 128, 384, device="cuda"))),
        (NotImplementedError, lambda: akv.LatentWeights(torch.zeros(2, 128, 512, device="cuda"), torch.zeros(3, 128, 512, device="cuda"))),
        (ValueError, lambda: akv.PagedLatentPool(pool.data.transpose(0, 1), 512)), (NotImplementedError, lambda: akv.PagedLatentPool(pool.data, 448)),
        (NotImplementedError, lambda: akv.PagedLatentPool.empty(1, 2, page_size=40)), (NotImplementedError, lambda: akv.PagedLatentPool.empty(1, 2, rope_dim=32)),
        (ValueError, lambda: akv.copy_pages(pool, batch.kv_lens[:2], batch.kv_lens[:1])),
        (ValueError, lambda: akv.compact_pages(pool, batch.page_table[:2], batch.page_table, batch.page_table, batch.kv_lens)),
    ):
        with pytest.raises(err):
            call()


def test_empty_calls():
    import akv
    announce("latent calls without sequences, rows or pages")
    z = lambda *n: torch.zeros(*n, dtype=torch.int32, device="cuda")  # noqa: E731
    pool = akv.PagedLatentPool.empty(1, 0)
    w = akv.LatentWeights(*(torch.ones(4, 128, 512, device="cuda") for _ in range(2)))
    for S in (0, 2):
        none = akv.PagedBatch(z(S, 0), z(S), z(S + 1), 0, 0)
        q, qr = torch.empty(0, 4, 512, device="cuda").half(), torch.empty(0, 4, 64, device="cuda").half()
        assert akv.latent_attention(q, qr, pool, none, SCALE).shape == (0, 4, 512)
        assert akv.latent_prefill(torch.empty(0, 4, 192, device="cuda").half(), pool, none, w).shape == (0, 4, 128)
        akv.latent_append(pool, none, torch.empty(0, 512, device="cuda"), torch.empty(0, 64, device="cuda"))
        assert akv.latent_read(pool, none)[0].shape == (0, 512)
        scores = torch.rand(S, 5, device="cuda")
        out = akv.latent_importance(q, qr, torch.empty(0, 4, device="cuda"), pool, none, scores, SCALE, out=torch.zeros_like(scores))
        assert torch.equal(out, scores)
    for H in (4, 40):
        w = akv.LatentWeights(*(torch.ones(H, 128, 512, device="cuda") for _ in range(2)))
        for some in (pool, akv.PagedLatentPool.empty(1, 3)):
            one = akv.PagedBatch(z(1, 0) if some is pool else z(1, 2), z(1), torch.tensor([0, 2], dtype=torch.int32, device="cuda"), 2, 2)
            ones = torch.ones(2, H, 576, device="cuda").half()
            out, lse = akv.latent_attention(ones[..., :512], ones[..., 512:], some, one, SCALE, return_lse=True)
            assert not bool(out.any()) and bool(lse.isneginf().all())
            assert not bool(akv.latent_prefill(ones[..., :192], some, one, w).any())
            x = torch.ones(2, 576, device="cuda")
            akv.latent_append(some, one, x[:, :512], x[:, 512:])
            assert not bool(akv.latent_read(some, one)[0].any())
    akv.copy_pages(pool, z(0), z(0))
    akv.compact_pages(pool, z(0, 1), z(0, 1), z(0, 4), z(0))
    akv.compact_pages(pool, z(2, 1), z(2, 1), z(2, 0), z(2))
