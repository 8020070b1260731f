"""Calls of the paged 4-bit cache that a program makes seldom: values that are not finite next
to rows that do not see them, batches on both sides of a choice of kernel, calls that overlap,
calls that are replayed, tables of other orders, lists that name a token twice."""
import numpy as np
import pytest
import torch

import paged_ref as ref
from gpu_util import announce
from test_gpu_paged import DT, FORMS, World, _check_attention, _x

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D,G,P", FORMS)
@pytest.mark.parametrize("Hq,kv,m", [(8, 70, 6), (8, 500, 16), (8, 300, 90), (2, 3001, 200), (2, 150, 150)])
def test_rows_do_not_feel_what_they_do_not_see(Hq, kv, m, D, G, P):
    """Tokens with NaN values or keys among a chunk's own: the rows before them come out bit for
    bit as if they were finite, the rows behind them NaN where the token's group reaches."""
    import akv
    announce(f"paged attention Hq={Hq} D={D} G={G} kv={kv} rows={m}, NaN in tokens that some rows see")
    w = World(D, G, P, 2, [kv, 40], [m, 1])
    w.fill()
    g = Hq // 2
    first, second, last = m // 3, m // 2, m - 1  # rows of the sequence: their own tokens
    for dt in ("fp16", "bf16"):
        k, v, q = (_x((w.T, h, D), i, dt) for i, h in ((1, 2), (2, 2), (3, Hq)))
        akv.paged_append(w.pool, w.batch, k, v)
        plain = [akv.paged_attention(q, w.pool, w.batch), *akv.paged_attention(q, w.pool, w.batch, return_lse=True)]
        v[first, 1, D - 1] = float("nan")   # the last group of head 1
        v[second, 0, 3] = float("inf")      # the first of head 0
        k[last, 0, 0] = float("nan")
        akv.paged_append(w.pool, w.batch, k, v)
        got = [akv.paged_attention(q, w.pool, w.batch), *akv.paged_attention(q, w.pool, w.batch, return_lse=True)]
        for a, b in zip(plain, got):
            nan = torch.zeros_like(a, dtype=torch.bool)
            nan[last:m, :g] = True          # a key that is NaN: everything of the rows that see it
            if a.dim() == 3:
                nan[first:m, g:, D - G:] = True
                nan[second:m, :g, :G] = True
            assert bool(b[nan].isnan().all())
            assert torch.equal(a[~nan], b[~nan])


def _check_importance(w, x, lse, N, win, causal):
    import akv
    kv, q = w.kv, w.q
    scores = torch.rand(len(kv), N + 3, device="cuda")[:, 1:N + 1]
    old = scores.double().cpu().numpy()
    out = torch.full((len(kv), N), -5.0, device="cuda")
    akv.paged_importance(x, lse, w.pool, w.batch, scores, decay=0.75, q_window=win, causal=causal, out=out)
    for s, (n, m) in enumerate(zip(kv, q)):
        got = out[s].double().cpu().numpy()
        at = min(n, N) if m else 0
        assert np.array_equal(got[at:], old[s, at:])
        if not at:
            continue
        first = max(0, m - win) if win else 0
        r = slice(w.starts[s] + first, w.starts[s + 1])
        seen = np.arange(n - m + first, n) + 1 if causal else np.full(m - first, n)
        kp, _ = w.ref.parts(0, w.table[s], np.arange(n))
        e, d = ref.importance(x[r].double().cpu().numpy(), kp, w.D ** -0.5, seen, lse[r].double().cpu().numpy())
        # keys as two float16 add up to them to 2^-22, which the bound's 64 roundings of 2^-24 hold
        exp = 0.75 * old[s, :at] + e[:at]
        assert (np.abs(got[:at] - exp) <= d[:at] + 2.0 ** -22 * (np.abs(exp) + old[s, :at])).all()
    again = torch.full((len(kv), N), 3.0, device="cuda")
    akv.paged_importance(x, lse, w.pool, w.batch, scores, decay=0.75, q_window=win, causal=causal, out=again)
    assert torch.equal(out, again)
    akv.paged_importance(x, lse, w.pool, w.batch, scores, decay=0.75, q_window=win, causal=causal)
    assert torch.equal(out, scores)


@pytest.mark.parametrize("D,G,P", FORMS)
@pytest.mark.parametrize("Hq,H,kv,q,win", [
    (8, 2, [200, 70, 5], [40, 1, 5], 0), (3, 3, [1, 300, 0, 131], [1, 260, 0, 129], 0), (16, 2, [500, 65], [30, 17], 20),
    (64, 1, [100, 64, 63], [3, 2, 1], 0),
])
def test_importance_of_chunks(Hq, H, kv, q, win, D, G, P):
    """More rows than the wave kernel takes, ragged beside sequences of few and of none."""
    import akv
    announce(f"paged importance of chunks Hq={Hq} H={H} D={D} G={G} P={P} kv={kv} q={q} window={win}")
    w = World(D, G, P, H, kv, q)
    w.fill()
    for dt, causal in (("fp16", True), ("bf16", False), ("bf16", True)):
        x, lse = _check_attention(w, Hq, dt, causal)
        for N in (max(kv) + 7, max(kv) // 2):
            _check_importance(w, x, lse, N, win, causal)


@pytest.mark.parametrize("D,G,P", [FORMS[0], FORMS[1], FORMS[2], FORMS[4]])
@pytest.mark.parametrize("Hq,H", [(4, 1), (6, 2), (9, 3), (8, 4), (10, 5), (16, 8), (24, 12)])
def test_importance_of_a_large_step(Hq, H, D, G, P):
    """Few rows of calls large enough for several runs a wave: scores far wider than the sequences,
    all splits of the heads over waves, two to four runs."""
    announce(f"paged importance of a large step Hq={Hq} H={H} D={D} G={G} P={P}")
    w = World(D, G, P, H, [1100, 0, 65, 257], [2, 0, 5, 1])
    w.fill()
    tokens = 64 * (4 if H == 1 else 2 if H < 4 else 1)
    for runs, dt, win, causal in ((2, "fp16", 0, True), (3, "bf16", 1, True), (4, "fp16", 3, False)):
        x, lse = _check_attention(w, Hq, dt, causal)
        _check_importance(w, x, lse, 768 * runs // 4 * tokens - 5, win, causal)


def test_importance_of_many_short_sequences():
    """700 sequences of up to 200 tokens, idle and empty ones among them; pages outside the pool."""
    import akv
    announce("paged importance, 700 sequences")
    rng = np.random.default_rng(2)
    kv = rng.integers(0, 200, 700).tolist()
    q = [0 if i % 7 == 3 else min(n, 1 + i % 3) for i, n in enumerate(kv)]
    w = World(64, 32, 16, 5, kv, q)
    w.fill()
    x, lse = _check_attention(w, 5, "fp16", True)
    _check_importance(w, x, lse, 203, 0, True)
    before = akv.paged_importance(x, lse, w.pool, w.batch, torch.zeros(700, 203, device="cuda"))
    w.batch.page_table[:, 1] = 10 ** 6
    got = akv.paged_importance(x, lse, w.pool, w.batch, torch.zeros(700, 203, device="cuda"))
    assert not bool(got[:, 16:32].any()) and torch.equal(got[:, :16], before[:, :16]) and torch.equal(got[:, 32:], before[:, 32:])


def test_importance_of_chunks_over_odd_pages():
    """Table entries outside the pool and keys that are not finite count for no row that does not see them."""
    import akv
    announce("paged importance of chunks, pages outside the pool, NaN keys")
    w = World(128, 32, 16, 2, [300], [150])
    w.fill()
    q = _x((150, 4, 128), 1)
    k, v = _x((150, 2, 128), 2), _x((150, 2, 128), 3)
    k[140, 0, 7] = float("nan")  # token 290: the last ten rows of heads 0 and 1 see it
    akv.paged_append(w.pool, w.batch, k, v)
    w.batch.page_table[0, 2] = 10 ** 6
    w.batch.page_table[0, 7] = -1
    zero = torch.zeros(1, 300, device="cuda")
    _, lse = akv.paged_attention(q, w.pool, w.batch, return_lse=True)
    assert bool(lse[140:, :2].isnan().all()) and bool(lse[:140].isfinite().all()) and bool(lse[:, 2:].isfinite().all())
    got = akv.paged_importance(q[:140].contiguous(), lse[:140].contiguous(), w.pool, akv.PagedBatch(
        w.batch.page_table, torch.tensor([290], device="cuda"), torch.tensor([0, 140], device="cuda"), 140, 140), zero, out=torch.empty_like(zero))
    assert bool(got.isfinite().all()) and not bool(got[0, 32:48].any()) and not bool(got[0, 112:128].any())
    assert bool((got[0, :32] > 0).all()) and not bool(got[0, 290:].any())
    # every row's weights add up to 1: the two calls' scores are off by at most 64 roundings of 2^-24 of
    # the terms they sum each, which are below 30
    assert abs(float(got.double().sum()) - 140.0) < 140 * 2.0 ** -12
    got = akv.paged_importance(q, lse, w.pool, w.batch, zero, out=torch.empty_like(zero))
    assert bool(got[0, :32].isnan().all()) and not bool(got[0, 32:48].any()) and not bool(got[0, 112:128].any())


@pytest.mark.parametrize("Hq,H,q", [(1, 1, [64, 65, 1, 66]), (8, 1, [8, 9, 0, 10]), (7, 1, [9, 10, 9]), (6, 2, [21, 22, 40])])
def test_rows_on_both_sides_of_the_kernels(Hq, H, q):
    """Sequences just below and above the rows from which on the tile kernel takes them, in one batch."""
    announce(f"paged attention Hq={Hq} H={H} rows {q}")
    w = World(128, 32, 16, H, [m + 130 for m in q], q)
    w.fill()
    for dt in ("fp16", "bf16"):
        _check_attention(w, Hq, dt, True)


def test_many_chunks():
    """More chunks than the tile kernel's scan has threads, and runs of sequences without any."""
    announce("paged attention, 700 sequences, every third a chunk of 70 rows")
    q = [70 if i % 3 == 0 else (1 if i < 400 else 0) for i in range(700)]
    kv = [m + i % 17 for i, m in enumerate(q)]
    w = World(64, 32, 16, 1, kv, q)
    w.fill()
    _check_attention(w, 1, "fp16", True)


def test_a_long_chunk_over_many_pages():
    """Page tables longer than the entries a wave holds at a time, and runs that start inside."""
    announce("paged attention, one chunk after 5000 tokens on 16-token pages")
    w = World(64, 64, 16, 1, [5077], [77])
    w.fill()
    for dt in ("fp16", "bf16"):
        _check_attention(w, 1, dt, True)
        _check_attention(w, 1, dt, False)


def test_one_batch_on_two_streams_at_once():
    import akv
    announce("paged attention, one batch on two streams")
    w = World(128, 32, 16, 2, [700, 900, 80], [40, 1, 5])
    w.fill()
    qs = [_x((w.T, 8, 128), i, "bf16") for i in range(2)]
    scores = torch.rand(3, 900, device="cuda")
    alone = [akv.paged_attention(q, w.pool, w.batch, return_lse=True) for q in qs]
    imps = [akv.paged_importance(q, a[1], w.pool, w.batch, scores, out=torch.empty_like(scores)) for q, a in zip(qs, alone)]
    streams = [torch.cuda.Stream() for _ in qs]
    torch.cuda.synchronize()
    both = [[], []]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                o, l = akv.paged_attention(qs[i], w.pool, w.batch, return_lse=True)
                both[i].append((o, l, akv.paged_importance(qs[i], l, w.pool, w.batch, scores, out=torch.empty_like(scores))))
    torch.cuda.synchronize()
    for i in range(2):
        for o, l, imp in both[i]:
            assert torch.equal(o, alone[i][0]) and torch.equal(l, alone[i][1]) and torch.equal(imp, imps[i])


def test_replayed_chunks_follow_lengths_tables_and_rows():
    """Two captured chunk calls, replayed in turns with eager work between, after the lengths, the
    rows and the tables on the device have changed."""
    import akv
    announce("paged attention and importance of chunks, captured and replayed")
    w = World(128, 32, 16, 2, [400, 900, 70], [30, 60, 2])
    w.fill()
    q = _x((w.T, 8, 128), 4)
    scores = torch.rand(3, 900, device="cuda")

    def work():
        o, l = akv.paged_attention(q, w.pool, w.batch, return_lse=True)
        return o, l, akv.paged_importance(q, l, w.pool, w.batch, scores, out=torch.empty_like(scores))
    work()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = work()
        graphs.append((graph, out))
    for turn, (kv, starts) in enumerate([([400, 900, 70], [0, 30, 90, 92]), ([31, 64, 0], [0, 30, 90, 92]),
                                         ([300, 899, 60], [0, 60, 61, 92]), ([300, 899, 60], [0, 0, 60, 60]),
                                         ([400, 900, 70], [0, 30, 90, 92])]):
        w.batch.kv_lens.copy_(torch.tensor(kv, dtype=torch.int32))
        w.batch.q_starts.copy_(torch.tensor(starts, dtype=torch.int32))
        if turn == 2:
            w.batch.page_table[[0, 1]] = w.batch.page_table[[1, 0]]
        want = work()
        for graph, out in graphs:
            for t in out:
                t.fill_(7.0)
            graph.replay()
            torch.cuda.synchronize()
            n = starts[-1]
            assert torch.equal(out[0][:n], want[0][:n]) and torch.equal(out[1][:n], want[1][:n]) and torch.equal(out[2], want[2])
            assert bool((out[0][n:] == 7.0).all()) and bool((out[1][n:] == 7.0).all())  # rows behind the last sequence's


def test_tables_and_lists_of_other_kinds():
    """int64, transposed, sliced and broadcast tables, and rows of other strides, say the same."""
    import akv
    announce("paged calls with tables and rows of other strides")
    w = World(128, 64, 32, 2, [200, 200, 200], [3, 3, 3])
    w.fill()
    b = w.batch
    b.page_table[:] = b.page_table[0]  # the three share their pages (read only)
    q = _x((w.T, 8, 128), 1)
    want = akv.paged_attention(q, w.pool, b)
    wide = torch.full((3, 20), -1, dtype=torch.int32, device="cuda")
    wide[:, 3:3 + b.page_table.shape[1]] = b.page_table
    lens = torch.stack([b.kv_lens, b.kv_lens * 0], 1)[:, 0]
    for table in (b.page_table.long(), b.page_table.t().contiguous().t(), wide[:, 3:3 + b.page_table.shape[1]],
                  b.page_table[:1].expand(3, -1)):
        other = akv.PagedBatch(table, lens, b.q_starts.long(), w.T, 3)
        assert torch.equal(akv.paged_attention(q, w.pool, other), want)
    for x in (_x((8, w.T, 128), 1).transpose(0, 1), _x((w.T, 8, 256), 1)[..., 100:228], _x((128, w.T, 8), 1).permute(1, 2, 0),
              _x((1, 8, 128), 1).expand(w.T, 8, 128), _x((w.T, 1, 128), 1).expand(w.T, 8, 128)):
        assert torch.equal(akv.paged_attention(x, w.pool, b), akv.paged_attention(x.contiguous(), w.pool, b))


def test_compact_lists_that_name_a_token_often():
    """keep may name a token twice, out of order, or none: what it says is moved."""
    import akv
    announce("paged compact, tokens named twice, lists of other kinds")
    w = World(128, 32, 16, 2, [50, 33], [1, 1], spare=12, layers=2)
    for layer in range(2):
        w.fill(seed=layer, layer=layer)
    dst = torch.from_numpy(w.spare[:8].reshape(2, 4).copy()).cuda()
    keep = [[7] * 5 + [49, 0, 49, 3] * 6 + [2], [32, 31, 30] * 7]
    rows = torch.full((2, 40), -1, dtype=torch.int64, device="cuda")
    for s, k in enumerate(keep):
        rows[s, :len(k)] = torch.tensor(k)
    akv.compact_pages(w.pool, w.batch.page_table, dst, rows, torch.tensor([len(k) for k in keep], device="cuda"))
    full = akv.PagedBatch(dst, torch.tensor([len(k) for k in keep], dtype=torch.int32, device="cuda"),
                          torch.tensor([0, len(keep[0]), len(keep[0]) + len(keep[1])], dtype=torch.int32, device="cuda"),
                          sum(map(len, keep)), max(map(len, keep)))
    for layer in range(2):
        k, v = akv.paged_read(w.pool, full, layer, torch.float32)
        at = 0
        for s, idx in enumerate(keep):
            ek, ev = w.ref.read(layer, w.table[s], np.array(idx))
            # c s + z in float32: one rounding of the sum, 2^-24 of it and of its parts
            for x, e in ((k, ek), (v, ev)):
                x = x[at:at + len(idx)].double().cpu().numpy()
                assert (np.abs(x - e) <= np.abs(e) * 2.0 ** -23 + 2.0 ** -30).all()
            at += len(idx)


def test_a_prompt_of_more_rows_than_a_decode_call_may_count():
    """131072 tokens' rows in one call are no decode work: only their own sequence's size counts.
    (A few cached tokens and one head of them: the rows are padding past the sequence.)"""
    import akv
    announce("paged attention, a batch that allows 131072 rows a sequence")
    w = World(64, 64, 256, 1, [300], [5])
    w.fill()
    T = 131072
    table = torch.full((1, 512), -1, dtype=torch.int32, device="cuda")
    table[:, :w.batch.page_table.shape[1]] = w.batch.page_table
    big = akv.PagedBatch(table, w.batch.kv_lens, w.batch.q_starts, T, T)
    q = torch.zeros(T, 64, 64, dtype=torch.float16, device="cuda")
    q[:5] = _x((5, 64, 64), 2)
    out = akv.paged_attention(q, w.pool, big)
    # 5 rows x 64 heads are a chunk's rows in both calls
    assert torch.equal(out[:5], akv.paged_attention(q[:5].contiguous(), w.pool, w.batch))


def test_a_cache_whose_work_fails_is_as_it_was(monkeypatch):
    """Uploads and launches that fail inside extend and compact: pages, lengths and contents stay."""
    import akv
    from akv import paged_packed
    announce("paged cache, work that fails inside a call")
    cache = akv.PackedPagedCache(2, 2, 64, max_pages=12)
    a = cache.add_sequence()
    batch = cache.extend([a], 40)
    for layer in range(2):
        cache.append(layer, _x((40, 2, 64), layer), _x((40, 2, 64), layer + 2), batch)
    b, = cache.fork(a)

    def state():
        return ([cache.get_seq_length(s) for s in (a, b)], cache.num_free_pages,
                [t for s in (a, b) for layer in range(2) for t in cache.get_kv(layer, s)])

    def same(x, y):
        return x[:2] == y[:2] and all(torch.equal(s, t) for s, t in zip(x[2], y[2]))
    before = state()
    keep = [torch.arange(0, 40, 3, device="cuda"), torch.arange(5, device="cuda")]

    def fail(*args, **kw):
        raise torch.OutOfMemoryError("no room")
    for name in ("copy_pages", "compact_pages"):
        monkeypatch.setattr(paged_packed, name, fail)
    for _ in range(20):  # more often than there are pages
        with pytest.raises(torch.OutOfMemoryError):
            cache.extend([a, b], [1, 30])
        with pytest.raises(torch.OutOfMemoryError):
            cache.compact([a, b], keep)
    monkeypatch.undo()
    monkeypatch.setattr(cache, "_upload", fail)
    for _ in range(20):
        with pytest.raises(torch.OutOfMemoryError):
            cache.extend([b], [30])
        with pytest.raises(torch.OutOfMemoryError):
            cache.compact([b], keep[1:])
    monkeypatch.undo()
    assert same(state(), before)
    cache.compact([a, b], keep)
    got = state()
    for i in range(4):  # keys and values of both layers of a
        assert torch.equal(got[2][i], before[2][i][:, ::3]) and torch.equal(got[2][4 + i], before[2][i][:, :5])


def test_pages_past_32_bits_of_bytes():
    """A pool of 5 GiB: sequences on its last pages answer as those on a small pool's."""
    import akv
    announce("paged cache, pages 4 GiB into a pool")
    H, D, n = 8, 128, 262144
    if torch.cuda.mem_get_info()[0] < 8 << 30:
        pytest.skip("needs 8 GiB")
    w = World(D, 32, 16, H, [100, 333], [100, 60], spare=30)
    big = akv.PagedPool.empty(1, n, H, D, 16, 32)
    assert big.nbytes() == 5 << 30
    shift = n - w.ref.data.shape[1]
    far = akv.PagedBatch(torch.where(w.batch.page_table < 0, w.batch.page_table, w.batch.page_table + shift), w.batch.kv_lens,
                         w.batch.q_starts, w.T, 100)
    w.fill()
    big.data[:, shift:].copy_(w.pool.data)
    k, v, q = _x((w.T, H, D), 1), _x((w.T, H, D), 2), _x((w.T, 16, D), 3, "bf16")
    one = q[[0, 100]].contiguous()
    spare = torch.from_numpy(w.spare[:20].copy()).cuda()
    dst = spare[:14].view(2, 7)
    keep = torch.arange(100, device="cuda", dtype=torch.int32).repeat(2, 1).flip(1)
    res = []
    for pool, batch, off in ((w.pool, w.batch, 0), (big, far, shift)):
        akv.paged_append(pool, batch, k, v)
        o, l = akv.paged_attention(q, pool, batch, return_lse=True)
        ones = akv.PagedBatch(batch.page_table, batch.kv_lens, torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda"), 2, 1)
        o1, l1 = akv.paged_attention(one, pool, ones, return_lse=True)
        imp = akv.paged_importance(one, l1, pool, ones, torch.zeros(2, 333, device="cuda"))
        akv.copy_pages(pool, batch.page_table[1, :6], spare[14:20] + off)
        akv.compact_pages(pool, batch.page_table, dst + off, keep, torch.tensor([100, 90], device="cuda"))
        res.append([o, l, o1, l1, imp, *akv.paged_read(pool, batch)])
    assert all(torch.equal(a, b) for a, b in zip(*res))
    assert torch.equal(big.data[:, shift:], w.pool.data) and not bool(big.data[:, :shift:997].any())


@pytest.mark.parametrize("kv,n,H,g,D,G", [(60000, 1, 2, 2, 128, 64), (30000, 4, 1, 7, 128, 128), (20000, 2, 2, 1, 64, 32), (120, 2, 4, 4, 128, 128),
                                          (50, 1, 1, 2, 128, 128), (85, 1, 1, 1, 128, 32), (20000, 80, 1, 1, 128, 32), (400, 100, 2, 3, 64, 64), (700001, 1, 1, 4, 128, 32)])
def test_precision(kv, n, H, g, D, G):
    """How far outputs and log-sums are off, by the norm.  Rounding to float16 alone leaves at most
    2^-10 / sqrt(12) = 0.58 2^-11 of it, and the kernel's own part must stay below 0.47 2^-11 (then both
    are below 0.75 2^-11 together); bfloat16 likewise with 2^-8, its own part below 0.15 2^-8 (0.6
    together).  Log-sums are float32: sums and scores of up to 64 in steps of 2^-19 of log2 leave
    2^-20 of theirs."""
    import akv
    announce(f"paged attention, precision at kv={kv} rows={n} H={H} g={g} D={D} G={G}")
    gen = torch.Generator(device="cuda")
    gen.manual_seed(kv)
    pages = -(-kv // 16)
    pool = akv.PagedPool.empty(1, pages, H, D, 16, G)
    table = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32).view(1, -1)
    one = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    whole = akv.PagedBatch(table, one(kv), one(0, kv), kv, kv)
    k, v = torch.randn(2, kv, H, D, generator=gen, device="cuda")
    k[..., 3] *= 10.0
    akv.paged_append(pool, whole, k, v)
    k, v = (x.double().repeat_interleave(g, 1) for x in akv.paged_read(pool, whole, 0, torch.float32))
    batch = akv.PagedBatch(table, one(kv), one(0, n), n, n)
    see = torch.ones(n, kv, dtype=torch.bool, device="cuda").tril(kv - n)
    for dt, half in ((torch.float16, 2.0 ** -11), (torch.bfloat16, 2.0 ** -8)):
        q = torch.randn(n, H * g, D, generator=gen, device="cuda").to(dt)
        x = torch.stack([(q[:, h].double() @ k[:, h].T) * D ** -0.5 for h in range(H * g)])
        x = x.masked_fill(~see, -torch.inf)
        el = torch.logsumexp(x, -1)
        eo = torch.stack([torch.exp(x[h] - el[h, :, None]) @ v[:, h] for h in range(H * g)], 1)
        for want_lse in (True, False):
            o = akv.paged_attention(q, pool, batch, return_lse=want_lse)
            if want_lse:
                o, lse = o
                assert float((lse.double() - el.T).norm() / el.norm()) < 2.0 ** -20
            assert float((o.double() - eo).norm() / eo.norm()) < (0.75 if dt == torch.float16 else 0.6) * half


@pytest.mark.parametrize("D,G,P", FORMS)
@pytest.mark.parametrize("size", [1e-6, 3e-3, 3e4])
def test_attention_over_values_of_any_size(size, D, G, P):
    """Caches of values at the clamp, of float16's smallest, and of groups of one value (scale 0)."""
    import akv
    announce(f"paged attention D={D} G={G} over values of {size}")
    w = World(D, G, P, 2, [200, 90, 300], [3, 1, 90])
    rng = np.random.default_rng(7)
    for s, n in enumerate(w.kv):
        k, v = rng.standard_normal((2, n, 2, D)) * size
        k[:, 0, :G] = k[:, 0, :1]           # one value: scale 0
        v[5::7, 1, D - G:] = 0.0
        if size > 1:
            v[3::5, 0, 1], v[4::5, 0, 2] = 1e9, -1e9    # clamped: a range of 122880
            k[2::3, 1, 7] = 61440.0
        w.ref.write(0, w.table[s], np.arange(n), k, v)
    w.pool.data.copy_(torch.from_numpy(w.ref.data))
    scale = D ** -0.5 / size
    for dt in ("fp16", "bf16"):
        q = _x((w.T, 8, D), 3, dt)
        half = torch.finfo(q.dtype).eps / 2
        for want in (True, False):
            out = akv.paged_attention(q, w.pool, w.batch, sm_scale=scale, return_lse=want)
            out, lse = out if want else (out, None)
            for s, (n, m) in enumerate(zip(w.kv, w.q)):
                kp, vp = w.ref.parts(0, w.table[s], np.arange(n))
                r = w.rows(s)
                eo, el, bo, bl = ref.attention(q[r].double().cpu().numpy(), kp, vp, scale, np.arange(n - m, n) + 1, half,
                                               rounded=not want and m * 4 > 64)
                # float16's smallest step, for values and outputs below its normal range
                assert (np.abs(out[r].double().cpu().numpy() - eo) <= bo + 2.0 ** -24).all()
                if want:
                    assert (np.abs(lse[r].double().cpu().numpy() - el) <= bl).all()


@pytest.mark.parametrize("Hq,H,kv,q", [(4, 2, [256, 1, 0, 130], [1, 1, 0, 1]), (8, 1, [64, 33], [8, 5]), (2, 1, [1], [1]), (12, 4, [17, 240, 90], [16, 3, 1]),
                                       (4, 4, [1000] + [37 * i % 1024 for i in range(69)], [2] + [i % 2 for i in range(69)])])
def test_attention_of_short_contexts(Hq, H, kv, q):
    """An item a workgroup: fewer units than waves, sequences far shorter than the longest, idle ones,
    chunks of 16 rows beside single ones, and many sequences of up to a thousand tokens."""
    announce(f"paged attention of short contexts Hq={Hq} H={H} kv={kv[:4]} rows={q[:4]}")
    for D, G in ((128, 32), (64, 64)):
        q = [min(m, n) for m, n in zip(q, kv)]
        w = World(D, G, 16, H, kv, q, spare=1)
        w.fill()
        for dt in ("fp16", "bf16"):
            _check_attention(w, Hq, dt, True)
            _check_attention(w, Hq, dt, False)


@pytest.mark.parametrize("T,H", [(1, 2), (1, 1), (3, 1), (3, 2)])
def test_rows_of_a_padded_projection(T, H):
    """Keys, values and queries sliced from rows whose stride is no multiple of 16 bytes: one token too."""
    import akv
    announce(f"paged calls on {T} rows of {H} heads, 8 bytes beside the alignment")
    w = World(128, 32, 16, H, [40], [T])
    w.fill()
    D, g = 128, 2
    wide = _x((T + 1, (2 + g) * H * D + 4), 3)[1:]
    k, v, q = (t.unflatten(1, (-1, D)) for t in (wide[:, :H * D], wide[:, H * D:2 * H * D], wide[:, 2 * H * D:(2 + g) * H * D]))
    akv.paged_append(w.pool, w.batch, k, v)
    w.ref.write(0, w.table[0], np.arange(40 - T, 40), k.double().cpu().numpy(), v.double().cpu().numpy())
    w.same_pool()
    plain = torch.empty(T, g * H, D, dtype=q.dtype, device="cuda").copy_(q)
    out, lse = akv.paged_attention(q, w.pool, w.batch, return_lse=True)
    want, wl = akv.paged_attention(plain, w.pool, w.batch, return_lse=True)
    assert torch.equal(out, want) and torch.equal(lse, wl)
    zero = torch.zeros(1, 40, device="cuda")
    assert torch.equal(akv.paged_importance(q, lse, w.pool, w.batch, zero.clone()), akv.paged_importance(plain, lse, w.pool, w.batch, zero.clone()))


@pytest.mark.parametrize("D,n", [(128, 5), (64, 3001)])
def test_read_of_padded_batches(D, n):
    """Rows of a read that are no sequence's, or that no sequence has a slot for, are 0: behind the last
    sequence, and where there is none."""
    import akv
    announce(f"paged read of {n} rows, D={D}, padded")
    w = World(D, 32, 16, 3, [40, 9], [2, 1])
    w.fill()
    b = w.batch
    want = akv.paged_read(w.pool, b)
    junk = [torch.full((n, 3, D), 7.0, dtype=torch.float16, device="cuda") for _ in range(2)]  # what the allocator may hand out
    del junk
    got = akv.paged_read(w.pool, akv.PagedBatch(b.page_table, b.kv_lens, b.q_starts, n, 2))
    for x, y in zip(got, want):
        assert torch.equal(x[:3], y) and not bool(x[3:].any())
    junk = [torch.full((n, 3, D), 7.0, dtype=torch.float16, device="cuda") for _ in range(2)]
    del junk
    none = akv.PagedBatch(b.page_table[:0], b.kv_lens[:0], b.q_starts[:1], n, 2)
    assert not any(bool(x.any()) for x in akv.paged_read(w.pool, none))
    akv.paged_append(w.pool, none, *want_rows(n, D))
    w.same_pool()


def want_rows(n, D):
    return _x((n, 3, D), 1), _x((n, 3, D), 2)


def test_rows_past_the_table_have_no_slot():
    """A sequence that outgrew its table: the rows whose place lies past its end are not written over the
    tokens that are there, and are read as 0; those before it keep theirs."""
    import akv
    announce("paged append and read past the table's end")
    w = World(128, 32, 16, 2, [32, 32, 32], [4, 4, 4], spare=0)
    w.fill()
    table = w.batch.page_table[:, :2].contiguous()
    lens = torch.tensor([36, 34, 10 ** 9], dtype=torch.int32, device="cuda")  # places 32.., 30.., far away
    batch = akv.PagedBatch(table, lens, w.batch.q_starts, 12, 4)
    k, v = _x((12, 2, 128), 1), _x((12, 2, 128), 2)
    akv.paged_append(w.pool, batch, k, v)
    w.ref.write(0, w.table[1], [30, 31], *(x[4:6].double().cpu().numpy() for x in (k, v)))
    w.same_pool()
    for got, e in zip(akv.paged_read(w.pool, batch, dtype=torch.float32), w.ref.read(0, w.table[1], [30, 31])):
        assert not bool(got[:4].any()) and not bool(got[6:].any())
        assert (np.abs(got[4:6].double().cpu().numpy() - e) <= np.abs(e) * 2.0 ** -24 + 2.0 ** -25).all()


@pytest.mark.parametrize("D,G", [(128, 32), (64, 64)])
@pytest.mark.parametrize("Hq,n,lens", [(4, 4, [66, 64, 63, 70]), (4, 40, [66, 100, 64, 80]), (2, 200, [90, 200, 264, 300])])
def test_rows_past_the_table_see_what_is_there(Hq, n, lens, D, G):
    """The rows of a sequence that outgrew its table count from its length: each sees the tokens up to its
    own, of those that have a slot; the importance likewise."""
    import akv
    announce(f"paged attention past the table's end, {n} rows, D={D}")
    cap, H = 64, 2
    w = World(D, G, 16, H, [cap] * 4, [n] * 4)
    w.fill()
    batch = akv.PagedBatch(w.batch.page_table[:, :cap // 16].contiguous(), torch.tensor(lens, dtype=torch.int32, device="cuda"),
                           w.batch.q_starts, 4 * n, n)
    for dt in ("fp16", "bf16"):
        q = _x((4 * n, Hq, D), 5, dt)
        out, lse = akv.paged_attention(q, w.pool, batch, return_lse=True)
        scores = torch.zeros(4, cap, device="cuda")
        akv.paged_importance(q, lse, w.pool, batch, scores)
        for s, m in enumerate(lens):
            seen = np.clip(np.arange(m - n, m) + 1, 0, cap)
            r = slice(s * n, s * n + n)
            kp, vp = w.ref.parts(0, w.table[s], np.arange(cap))
            x = q[r].double().cpu().numpy()
            eo, el, bo, bl = ref.attention(x, kp, vp, D ** -0.5, seen, torch.finfo(q.dtype).eps / 2)
            ok = seen > 0
            go, gl = out[r].double().cpu().numpy(), lse[r].double().cpu().numpy()
            assert (np.abs(go - eo) <= bo).all() and (np.abs(gl[ok] - el[ok]) <= bl[ok]).all() and np.isneginf(gl[~ok]).all()
            e, d = ref.importance(x, kp, D ** -0.5, seen, gl)
            assert (np.abs(scores[s].double().cpu().numpy() - e) <= d + 2.0 ** -22 * e).all()


@pytest.mark.parametrize("dt", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("D,G,P,H,T", [(128, 32, 16, 8, 1700), (128, 64, 32, 3, 7001), (64, 32, 64, 8, 5003), (128, 128, 16, 1, 60001), (64, 64, 16, 16, 2500)])
def test_large_prompts_like_their_parts(D, G, P, H, T, dt):
    """Calls whose waves take several sets of rows each write and read the bytes that small calls do."""
    import akv
    announce(f"paged append and read of {T} tokens at once and in parts, D={D} G={G} P={P} H={H} {dt}")
    q = [T // 2 + 3, 0, T - T // 2 - 8, 5]
    past = [0, 7, 21, 3]
    kv = [a + b for a, b in zip(q, past)]
    pages = [-(-n // P) for n in kv]
    up = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    ids = torch.randperm(sum(pages) + 2, device="cuda").to(torch.int32)
    table = torch.full((4, max(pages)), -1, dtype=torch.int32, device="cuda")
    for s, c in enumerate(pages):
        table[s, :c] = ids[sum(pages[:s]):sum(pages[:s]) + c]
    starts = np.concatenate([[0], np.cumsum(q)]).tolist()
    k, v = _x((T, H, D), 1, dt), _x((T, H, D), 2, dt)
    k[T // 3, 0, 5] = float("nan")
    one, parts = (akv.PagedPool.empty(1, sum(pages) + 2, H, D, P, G) for _ in range(2))
    whole = akv.PagedBatch(table, up(kv), up(starts), T, max(q))
    akv.paged_append(one, whole, k, v)
    got = akv.paged_read(one, whole, dtype=DT[dt])
    step = max(1, 4000 // H)
    for s in range(4):
        for a in range(0, q[s], step):
            n = min(step, q[s] - a)
            r = slice(starts[s] + a, starts[s] + a + n)
            some = akv.PagedBatch(table[s:s + 1], up([past[s] + a + n]), up([0, n]), n, n)
            akv.paged_append(parts, some, k[r], v[r])
            for x, y in zip(got, akv.paged_read(parts, some, dtype=DT[dt])):
                assert torch.equal(x[r].view(torch.uint8), y.view(torch.uint8))
    assert torch.equal(one.data, parts.data)
