"""The paged 4-bit cache's kernels against numpy in 64 bits: bytes where bytes are moved or
quantized, the bounds of paged_ref elsewhere.  Free slots hold random bytes throughout, NaN
scales among them: they must neither count nor change."""
import numpy as np
import pytest
import torch

import paged_ref as ref
from gpu_util import announce

pytestmark = pytest.mark.gpu

DT = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
FORMS = [(128, 32, 16), (128, 64, 32), (128, 128, 256), (64, 32, 16), (64, 64, 64)]


def _x(shape, seed, dt="fp16", outliers=False):
    x = np.random.default_rng(seed).standard_normal(shape)
    if outliers:
        x[..., 3] *= 10.0
    return torch.from_numpy(x).to(DT[dt]).cuda()


class World:
    """A pool of random bytes and sequences of given lengths on shuffled pages of it."""

    def __init__(self, D, G, P, H, kv, q, layers=1, spare=3, seed=0):
        import akv
        rng = np.random.default_rng(seed)
        self.kv, self.q, self.H, self.D, self.P = list(kv), list(q), H, D, P
        pages = [-(-n // P) for n in kv]
        n = sum(pages) + spare
        data = rng.integers(0, 256, (layers, n, H, P // 16, ref.tile_bytes(D, G)), dtype=np.uint8)
        self.ref = ref.Pool(data, D, G)
        ids = rng.permutation(n).astype(np.int32)
        width = max(pages, default=0) + 1
        self.table = np.full((len(kv), width), -1, np.int32)  # entries behind the last page: no page
        at = 0
        for s, c in enumerate(pages):
            self.table[s, :c] = ids[at:at + c]
            at += c
        self.spare = ids[at:]
        self.starts = np.concatenate([[0], np.cumsum(q)]).astype(np.int32)
        self.T = int(self.starts[-1])
        self.pool = akv.PagedPool(torch.from_numpy(data.copy()).cuda(), D, G)
        up = lambda a: torch.from_numpy(np.asarray(a, np.int32)).cuda()  # noqa: E731
        self.batch = akv.PagedBatch(up(self.table), up(kv), up(self.starts), self.T, max(q, default=0))

    def fill(self, seed=5, layer=0):
        """Every sequence's tokens, quantized by the reference."""
        rng = np.random.default_rng(seed)
        for s, n in enumerate(self.kv):
            k, v = rng.standard_normal((2, n, self.H, self.D))
            k[..., 3] *= 10.0
            self.ref.write(layer, self.table[s], np.arange(n), k, v)
        self.pool.data.copy_(torch.from_numpy(self.ref.data))

    def rows(self, s):
        return slice(self.starts[s], self.starts[s + 1])

    def same_pool(self):
        got = self.pool.data.cpu().numpy()
        bad = np.argwhere(got != self.ref.data)
        assert len(bad) == 0, f"{len(bad)} bytes differ, first at {bad[:4].tolist()}"


LENS = [([1], [1]), ([5, 0, 64], [5, 0, 1]), ([33, 16, 300, 17], [33, 1, 0, 17]), ([257], [200])]


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("D,G,P", FORMS)
@pytest.mark.parametrize("kv,q", LENS)
def test_append_and_read(D, G, P, kv, q, dt):
    import akv
    H = 3
    announce(f"paged append D={D} G={G} P={P} kv={kv} q={q} {dt}")
    w = World(D, G, P, H, kv, q, layers=2)
    qkv = _x((w.T, 2 * H + 1, D), 3, dt, outliers=True)  # keys and values as a model's projection gives them
    k, v = qkv[:, 1:H + 1], qkv[:, H + 1:]
    akv.paged_append(w.pool, w.batch, k, v, layer=1)
    for s in range(len(kv)):
        r = w.rows(s)
        w.ref.write(1, w.table[s], np.arange(kv[s] - q[s], kv[s]), *(x[r].double().cpu().numpy() for x in (k, v)))
    w.same_pool()
    for out in DT.values():
        got = akv.paged_read(w.pool, w.batch, layer=1, dtype=out)
        for s in range(len(kv)):
            for g, e in zip(got, w.ref.read(1, w.table[s], np.arange(kv[s] - q[s], kv[s]))):
                d = np.abs(g[w.rows(s)].double().cpu().numpy() - e)
                assert (d <= np.abs(e) * (torch.finfo(out).eps / 2 + 2.0 ** -24) + 2.0 ** -25).all()


@pytest.mark.parametrize("dt", ["fp16", "fp32"])
@pytest.mark.parametrize("D,G,P,H", [(128, 32, 16, 3), (64, 32, 64, 8), (128, 64, 32, 1)])
def test_append_and_read_of_many_rows(D, G, P, H, dt):
    """Prompts: waves take several sets of rows, of one token or of several."""
    import akv
    T = 9001 // H
    announce(f"paged append of {T} tokens, D={D} G={G} P={P} H={H} {dt}")
    q = [T // 3, 0, T - T // 3 - 5, 5]
    kv = [q[0], 9, q[2] + 21, 5]
    w = World(D, G, P, H, kv, q)
    k, v = _x((w.T, H, D), 3, dt, outliers=True), _x((w.T, H, D), 4, dt)
    akv.paged_append(w.pool, w.batch, k, v)
    for s in range(len(kv)):
        r = w.rows(s)
        w.ref.write(0, w.table[s], np.arange(kv[s] - q[s], kv[s]), *(x[r].double().cpu().numpy() for x in (k, v)))
    w.same_pool()
    got = akv.paged_read(w.pool, w.batch, dtype=torch.float32)
    for s in range(len(kv)):
        for g, e in zip(got, w.ref.read(0, w.table[s], np.arange(kv[s] - q[s], kv[s]))):
            assert (np.abs(g[w.rows(s)].double().cpu().numpy() - e) <= np.abs(e) * 2.0 ** -24 + 2.0 ** -25).all()


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("D,G,P", FORMS[:4:3])
def test_append_odd_values(D, G, P, dt):
    """Flat groups, ties, tiny and huge values, values that are not finite."""
    import akv
    announce(f"paged append odd values D={D} {dt}")
    w = World(D, G, P, 1, [12], [12])
    k = torch.zeros(12, 1, D)
    k[1] = 3.25
    k[2] = torch.arange(D) % 16 * 0.5                     # exact codes
    k[3] = torch.arange(D) % 31 * 0.5                     # every second one between two codes
    k[4] = torch.arange(D) * 1e-6
    k[5] = torch.linspace(-65504, 65504, D)
    k[6] = torch.linspace(-65504, 65504, D) * (1e33 if dt != "fp16" else 1)
    k[7, 0, 1] = float("nan")
    k[8, 0, 0] = float("inf")
    k[9, 0, D - 1] = float("-inf")
    k[10] = torch.linspace(-1, 1, D) * 2.0 ** -22
    k[11] = 1000 + torch.arange(D) % 2 * 0.25
    v = k.flip(0).contiguous()
    k, v = k.to(DT[dt]).cuda(), v.to(DT[dt]).cuda()
    akv.paged_append(w.pool, w.batch, k, v)
    w.ref.write(0, w.table[0], np.arange(12), k.double().cpu().numpy(), v.double().cpu().numpy())
    got = ref.Pool(w.pool.data.cpu().numpy(), D, G).read(0, w.table[0], np.arange(12))
    for a, b in zip(got, w.ref.read(0, w.table[0], np.arange(12))):
        assert np.array_equal(a, b, equal_nan=True)
        assert (np.isfinite(a) | np.isnan(a)).all() and np.nanmax(np.abs(a)) < 65504
    back = akv.paged_read(w.pool, w.batch)[0]
    assert torch.equal(back[1], k[1].half()) and torch.equal(back[2], k[2].half())
    assert bool(back[7, 0, :G].isnan().all()) and (D == G or bool(back[7, 0, G:].eq(0).all()))


def test_append_keeps_what_it_has_no_slot_for():
    """Rows past the table, on pages outside the pool, and of sequences longer than their cache."""
    import akv
    announce("paged append without slots")
    D, G, P = 64, 32, 16
    w = World(D, G, P, 2, [20, 30, 3], [2, 2, 5])
    t = w.batch.page_table
    t[0, 1] = w.pool.num_pages
    t[1, 1] = -7
    k, v = _x((9, 2, D), 1), _x((9, 2, D), 2)
    akv.paged_append(w.pool, w.batch, k, v)
    w.ref.write(0, w.table[2], [0, 1, 2], *(x[6:].double().cpu().numpy() for x in (k, v)))
    w.same_pool()
    got = akv.paged_read(w.pool, w.batch)
    assert all(not bool(x[:6].any()) for x in got)
    t[:] = -1
    w.batch.kv_lens[:] = 10 ** 9
    akv.paged_append(w.pool, w.batch, k, v)
    w.same_pool()


def _check_attention(w, Hq, dt, causal, layer=0, seed=9, big=1.0):
    import akv
    q = (_x((w.T, Hq, w.D), seed).float() * big).to(DT[dt])
    scale = w.D ** -0.5 / big
    out, lse = akv.paged_attention(q, w.pool, w.batch, layer, sm_scale=scale, causal=causal, return_lse=True)
    only = akv.paged_attention(q, w.pool, w.batch, layer, sm_scale=scale, causal=causal)
    # chunks of many rows round the keys where no log-sums are asked for
    many = [m * Hq // w.H > 64 for m in w.q]
    assert out.dtype == only.dtype == q.dtype
    for s in range(len(w.q)):
        assert many[s] or torch.equal(only[w.rows(s)], out[w.rows(s)])
    half = torch.finfo(q.dtype).eps / 2
    worst = 0.0
    for s, (n, m) in enumerate(zip(w.kv, w.q)):
        if m == 0:
            continue
        kp, vp = w.ref.parts(layer, w.table[s], np.arange(n))
        seen = np.maximum(np.arange(n - m, n) + 1, 0) if causal else np.full(m, n)
        r = w.rows(s)
        eo, el, bo, bl = ref.attention(q[r].double().cpu().numpy(), kp, vp, scale, seen, half)
        go, gl = out[r].double().cpu().numpy(), lse[r].double().cpu().numpy()
        none = seen == 0
        assert (go[none] == 0).all() and np.isneginf(gl[none]).all()
        ok = ~none
        assert np.isfinite(go).all()
        assert (np.abs(go - eo) <= bo).all(), f"sequence {s}: {(np.abs(go - eo) / np.maximum(bo, 1e-30)).max():.2f} of the bound"
        assert (np.abs(gl[ok] - el[ok]) <= bl[ok]).all(), f"sequence {s}: lse off by {np.abs(gl[ok] - el[ok]).max():.2e}"
        worst = max(worst, float((np.abs(go - eo) / np.maximum(bo, 1e-30)).max()))
        if many[s]:
            go = only[r].double().cpu().numpy()
            _, _, bo, _ = ref.attention(q[r].double().cpu().numpy(), kp, vp, scale, seen, half, rounded=True)
            assert (np.abs(go - eo) <= bo).all(), f"sequence {s}: {(np.abs(go - eo) / np.maximum(bo, 1e-30)).max():.2f} of the bound"
    print(f"  worst share of the bound {worst:.2f}")
    return q, lse


@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("D,G,P", FORMS)
@pytest.mark.parametrize("Hq,H,kv,q", [
    (1, 1, [1], [1]), (6, 2, [517], [1]), (4, 4, [0, 1, 33, 100, 700, 32], [1, 1, 1, 0, 1, 1]),
    (14, 2, [65, 2, 300], [3, 2, 1]), (32, 2, [47, 64], [1, 1]), (10, 2, [70, 5, 129], [4, 9, 3]),
])
def test_attention(Hq, H, kv, q, D, G, P, dt):
    announce(f"paged attention Hq={Hq} H={H} D={D} G={G} P={P} kv={kv} q={q} {dt}")
    w = World(D, G, P, H, kv, q)
    w.fill()
    _check_attention(w, Hq, dt, True)
    _check_attention(w, Hq, dt, False)


@pytest.mark.parametrize("D,G,P", [FORMS[0], FORMS[4]])
@pytest.mark.parametrize("Hq,H,kv,q", [
    (8, 1, [300, 20, 65], [33, 20, 1]), (2, 2, [130, 400], [130, 17]), (12, 2, [10, 500, 64], [40, 100, 64]),
])
def test_attention_of_chunks(Hq, H, kv, q, D, G, P):
    announce(f"paged attention of chunks Hq={Hq} H={H} D={D} P={P} kv={kv} q={q}")
    w = World(D, G, P, H, kv, q)
    w.fill()
    for dt in ("fp16", "bf16"):
        _check_attention(w, Hq, dt, True)
        _check_attention(w, Hq, dt, False)


@pytest.mark.parametrize("big", [1e-4, 3e3])
def test_attention_query_scales(big):
    """Queries far from 1: the operand is scaled by row."""
    announce(f"paged attention queries times {big}")
    w = World(128, 32, 16, 2, [200, 40], [1, 2])
    w.fill()
    for dt in ("fp16", "bf16"):
        _check_attention(w, 8, dt, True, big=big)


def test_attention_of_many_short_and_one_long():
    """More sequences than the scan's threads, idle ones among them, one a hundred times as long."""
    announce("paged attention, 300 sequences")
    rng = np.random.default_rng(1)
    kv = rng.integers(0, 50, 300).tolist()
    q = [0 if i % 7 == 3 else 1 for i in range(300)]
    kv[123] = 5000
    w = World(64, 32, 16, 1, kv, q)
    w.fill()
    _check_attention(w, 4, "fp16", True)


def test_attention_reads_no_foreign_page():
    """Table entries outside the pool hold no token: the others alone are attended."""
    import akv
    announce("paged attention, pages outside the pool")
    w = World(128, 32, 16, 1, [64], [1])
    w.fill()
    q = _x((1, 4, 128), 2)
    w.batch.page_table[0, 1] = 10 ** 6
    w.batch.page_table[0, 3] = -1
    out = akv.paged_attention(q, w.pool, w.batch)
    pos = np.r_[0:16, 32:48]
    kp, vp = w.ref.parts(0, w.table[0], pos)
    eo, _, bo, _ = ref.attention(q.double().cpu().numpy(), kp, vp, 128 ** -0.5, [32], 2.0 ** -11)
    assert (np.abs(out.double().cpu().numpy() - eo) <= bo).all()
    w.batch.page_table[:] = -1
    out, lse = akv.paged_attention(q, w.pool, w.batch, return_lse=True)
    assert not bool(out.any()) and bool(lse.isneginf().all())


def test_attention_nan_stays_in_its_sequence():
    import akv
    announce("paged attention, a NaN key and a NaN value")
    w = World(128, 32, 16, 2, [40, 40, 40], [1, 1, 1])
    w.fill()
    k, v = _x((3, 2, 128), 1), _x((3, 2, 128), 2)
    akv.paged_append(w.pool, w.batch, k, v)
    q = _x((3, 4, 128), 3)
    clean = akv.paged_attention(q, w.pool, w.batch)
    k[0, 0, 5] = float("nan")
    v[1, 1, 40] = float("inf")
    akv.paged_append(w.pool, w.batch, k, v)
    out = akv.paged_attention(q, w.pool, w.batch)
    assert bool(out[0, :2].isnan().all()) and bool(out[1, 2:, 32:64].isnan().all())
    assert torch.equal(out[2], clean[2]) and torch.equal(out[0, 2:], clean[0, 2:]) and torch.equal(out[1, :2], clean[1, :2])
    assert torch.equal(out[1, 2:, :32], clean[1, 2:, :32])


@pytest.mark.parametrize("D,G,P", [FORMS[0], FORMS[1], FORMS[4]])
@pytest.mark.parametrize("Hq,H,kv,q,win", [
    (6, 2, [1], [1], 0), (4, 4, [0, 1, 33, 100, 700], [1, 1, 1, 0, 1], 0), (28, 4, [130, 65], [3, 1], 2),
    (8, 8, [300, 64], [40, 20], 32), (6, 1, [90, 5], [7, 9], 0),
])
def test_importance(Hq, H, kv, q, win, D, G, P):
    import akv
    announce(f"paged importance Hq={Hq} H={H} D={D} G={G} P={P} kv={kv} q={q} window={win}")
    w = World(D, G, P, H, kv, q)
    w.fill()
    for dt in ("fp16", "bf16"):
        x, lse = _check_attention(w, Hq, dt, True)
        for N in (max(kv), max(kv) + 7, max(1, max(kv) // 2)):
            scores = torch.rand(len(kv), N + 3, device="cuda")[:, 1:N + 1]
            old = scores.double().cpu().numpy()
            out = torch.full((len(kv), N), -5.0, device="cuda")
            akv.paged_importance(x, lse, w.pool, w.batch, scores, decay=0.75, q_window=win, out=out)
            assert np.array_equal(scores.double().cpu().numpy(), old)
            for s, (n, m) in enumerate(zip(kv, q)):
                exp, err = old[s].copy(), np.zeros(N)
                if m:
                    f = max(0, m - win) if win else 0
                    seen = np.maximum(np.arange(n - m, n) + 1, 0)[f:]
                    kp, _ = w.ref.parts(0, w.table[s], np.arange(n))
                    r = w.rows(s)
                    t, e = ref.importance(x[r][f:].double().cpu().numpy(), kp, D ** -0.5, seen, lse[r][f:].double().cpu().numpy())
                    c = min(n, N)
                    exp[:c] = exp[:c] * 0.75 + t[:c]
                    err[:c] = e[:c] + 2.0 ** -22 * (np.abs(exp[:c]) + old[s, :c])
                got = out[s].double().cpu().numpy()
                assert (np.abs(got - exp) <= err).all(), (s, np.abs(got - exp).max())
            akv.paged_importance(x, lse, w.pool, w.batch, scores, decay=0.75, q_window=win)
            assert torch.equal(scores, out)


@pytest.mark.parametrize("D,G,P,H,L", [(128, 32, 16, 2, 3), (64, 64, 64, 1, 1), (128, 128, 32, 5, 2)])
@pytest.mark.parametrize("n", [0, 1, 7])
def test_copy(D, G, P, H, L, n):
    import akv
    announce(f"copy pages D={D} P={P} H={H} L={L} n={n}")
    w = World(D, G, P, H, [], [], layers=L, spare=19)
    ids = torch.randperm(19)[:2 * n].to(torch.int32)
    akv.copy_pages(w.pool, ids[:n].cuda(), ids[n:].cuda())
    w.ref.data[:, ids[n:].numpy()] = w.ref.data[:, ids[:n].numpy()]
    w.same_pool()
    # pairs outside the pool, a page onto itself
    akv.copy_pages(w.pool, torch.tensor([0, 19, -1, 4]).cuda(), torch.tensor([19, 1, 2, 4]).cuda())
    w.same_pool()


@pytest.mark.parametrize("D,G,P", FORMS)
@pytest.mark.parametrize("kv,keep", [([1], [1]), ([40, 100, 7, 300], [33, 16, 0, 299]), ([600], [77])])
def test_compact(D, G, P, kv, keep):
    import akv
    announce(f"compact pages D={D} G={G} P={P} kv={kv} keep={keep}")
    H, L = 3, 2
    rng = np.random.default_rng(4)
    pages = [-(-k // P) for k in keep]
    w = World(D, G, P, H, kv, [0] * len(kv), layers=L, spare=sum(pages) + 2)
    to = np.full((len(kv), max(pages) + 1), -1, np.int32)
    rows = np.full((len(kv), max(keep) + 1), 2 ** 31 - 1, np.int32)
    at = 0
    for s, (n, k) in enumerate(zip(kv, keep)):
        to[s, :pages[s]] = w.spare[at:at + pages[s]]
        at += pages[s]
        rows[s, :k] = np.sort(rng.permutation(n)[:k])
    up = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
    akv.compact_pages(w.pool, w.batch.page_table, up(to), up(rows), up(np.array(keep, np.int32)))
    old = w.ref.data.copy()
    for s, k in enumerate(keep):
        move_rows(w.ref.data, old, w.table[s], to[s], rows[s, :k], D, G, P)
    w.same_pool()


def move_rows(data, old, src, dst, keep, D, G, P):
    """Token j on dst becomes token keep[j] of `old` on src, byte for byte."""
    for at, sh, sa, za in ref.places(D, G):
        for j, i in enumerate(keep):
            a = old[:, src[i // P], :, i % P // 16]
            b = data[:, dst[j // P], :, j % P // 16]
            for x in (at, sa, sa + 1, za, za + 1):
                b[:, :, x[j % 16]] = a[:, :, x[i % 16]]


def test_compact_in_place_and_past_the_tables():
    """Tokens that stay in their slots may share pages with themselves; positions and pages out
    of range are skipped."""
    import akv
    announce("compact pages, odd tables")
    D, G, P, H = 128, 32, 16, 2
    w = World(D, G, P, H, [64], [0], spare=4)
    up = lambda *a: torch.tensor([list(a)], dtype=torch.int32, device="cuda")  # noqa: E731
    a, b, c, d = w.table[0, :4].tolist()
    n = torch.tensor([40], dtype=torch.int32, device="cuda")
    keep = list(range(16)) + [17, 19, 10 ** 9, -1, 21, 22] + list(range(30, 48))
    f, g = w.spare[:2].tolist()
    akv.compact_pages(w.pool, up(a, b, c, d), up(a, f, g), up(*keep), n)
    old = w.ref.data.copy()
    for j in range(16, 40):
        if 0 <= keep[j] < 64:
            move_rows_at(w.ref.data, old, [a, b, c, d], [a, f, g], j, keep[j], D, G, P)
    w.same_pool()
    akv.compact_pages(w.pool, up(a, b, c, 10 ** 6), up(-1, 99), up(*range(40)), n)
    akv.compact_pages(w.pool, up(a, b)[:, :0], up(f), up(*range(40)), n)
    w.same_pool()


def move_rows_at(data, old, src, dst, j, i, D, G, P):
    for at, sh, sa, za in ref.places(D, G):
        for x in (at, sa, sa + 1, za, za + 1):
            data[:, dst[j // P], :, j % P // 16][:, :, x[j % 16]] = old[:, src[i // P], :, i % P // 16][:, :, x[i % 16]]
