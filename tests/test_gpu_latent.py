"""The paged latent cache's kernels against 64 bits: bits where rows are moved or rounded, the
bounds of latent_ref elsewhere.  Free slots hold random bytes throughout, NaN and infinities
among them: they must neither count nor change."""
import pytest
import torch

import latent_ref as ref
from gpu_util import announce

pytestmark = pytest.mark.gpu

DT = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
FORMS = [(512, 16), (512, 64), (256, 32), (256, 256)]
DR = 64


def _randn(*shape, seed, dt="fp16", scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(DT[dt])


class World:
    """A pool of random bytes and sequences of given lengths on shuffled pages of it."""

    def __init__(self, Dc, P, kv, q, layers=1, spare=3, seed=0, width=None):
        import akv
        g = torch.Generator().manual_seed(seed)
        self.kv, self.q, self.Dc, self.P, self.W = list(kv), list(q), Dc, P, Dc + DR
        pages = [-(-n // P) for n in kv]
        n = sum(pages) + spare
        data = torch.randint(-2 ** 15, 2 ** 15, (layers, n, P, self.W), generator=g, dtype=torch.int16).view(torch.float16)
        ids = torch.randperm(n, generator=g).to(torch.int32)
        width = max(pages, default=0) + 1 if width is None else width
        self.table = torch.full((len(kv), width), -1, dtype=torch.int32)  # entries behind the last page: no page
        at = 0
        for s, c in enumerate(pages):
            c = min(c, width)
            self.table[s, :c] = ids[at:at + c]
            at += c
        self.spare = ids[at:]
        self.starts = torch.tensor([0] + list(q)).cumsum(0)
        self.T = int(self.starts[-1])
        self.data = data
        self.pool = akv.PagedLatentPool(data.cuda(), Dc)
        up = lambda a: torch.as_tensor(a, dtype=torch.int32).cuda()  # noqa: E731
        self.batch = akv.PagedBatch(self.table.cuda(), up(kv), up(self.starts), self.T, max(q, default=0))

    def slots(self, s, pos):
        pos = torch.as_tensor(pos)
        return self.table[s].long()[pos // self.P], pos % self.P

    def fill(self, seed=5, layer=0, scale=1.0):
        """Every sequence's tokens; some channels larger, as a model has them."""
        for s, n in enumerate(self.kv):
            n = min(n, self.table.shape[1] * self.P)
            x = _randn(n, self.W, seed=seed + s, dt="fp32", scale=scale)
            x[:, 3] *= 6.0
            x[:, self.Dc + 5] *= 3.0
            page, row = self.slots(s, torch.arange(n))
            self.data[layer, page, row] = x.half()
        self.pool.data.copy_(self.data)

    def rows(self, s, layer=0):
        page, row = self.slots(s, torch.arange(min(self.kv[s], self.table.shape[1] * self.P)))
        return self.data[layer, page, row].double()

    def mine(self, s):
        return slice(int(self.starts[s]), int(self.starts[s + 1]))

    def same_pool(self):
        got = self.pool.data.cpu().view(torch.int16)
        assert torch.equal(got, self.data.view(torch.int16)), "the pool differs"


def _scale():
    return 192 ** -0.5


def _queries(w, H, dt, seed=11):
    """As slices of one projection: rows of other strides."""
    x = _randn(w.T, H + 1, w.W, seed=seed, dt=dt, scale=0.6)
    return x[:, 1:, :w.Dc].cuda(), x[:, 1:, w.Dc:].cuda(), x[:, 1:].double()


def _check_attention(w, H, dt, causal=True, seed=11):
    import akv
    q, qr, x = _queries(w, H, dt, seed)
    # the padded projection's own strides
    big = torch.empty(w.T, H + 1, w.W, dtype=DT[dt], device="cuda")
    big[:, 1:, :w.Dc], big[:, 1:, w.Dc:] = q, qr
    out, lse = akv.latent_attention(big[:, 1:, :w.Dc], big[:, 1:, w.Dc:], w.pool, w.batch, _scale(), causal=causal, return_lse=True)
    assert torch.equal(out, akv.latent_attention(q.contiguous(), qr.contiguous(), w.pool, w.batch, _scale(), causal=causal))
    half = torch.finfo(DT[dt]).eps / 2
    for s in range(len(w.kv)):
        r = w.mine(s)
        if w.q[s] == 0:
            continue
        e, el, b, bl = ref.attention(x[r, :, :w.Dc], x[r, :, w.Dc:], w.rows(s), _scale(), half, causal, n=w.kv[s])
        d = (out[r].double().cpu() - e).abs()
        assert bool((d <= b).all()), (s, float((d / b).max()))
        got = lse[r].double().cpu()
        none = torch.isneginf(el)
        assert torch.equal(torch.isneginf(got), none), s
        assert bool(((got - el).abs()[~none] <= bl[~none]).all()), s
    return out, lse, q, qr, x


LENS = [([1], [1]), ([5, 0, 64], [5, 0, 1]), ([33, 16, 300, 17], [33, 1, 0, 17]), ([257], [200])]


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("Dc,P", FORMS)
@pytest.mark.parametrize("kv,q", LENS)
def test_append_and_read(Dc, P, kv, q, dt):
    import akv
    announce(f"latent append Dc={Dc} P={P} kv={kv} q={q} {dt}")
    w = World(Dc, P, kv, q, layers=2)
    x = _randn(w.T, w.W + 32, seed=3, dt=dt)
    x[:, 3] *= 1e5                                   # past the clamp, and infinite in float16
    odd = x[::7]
    if dt != "fp16":
        odd[:, 9], odd[:, 70] = 3e9, -3e9            # clamped, not infinite
    if w.T > 3:
        x[2, w.W - 1], x[3, 0] = float("nan"), float("-inf")
    y = x.cuda()
    akv.latent_append(w.pool, w.batch, y[:, :Dc], y[:, Dc:w.W], layer=1)
    rows, back = ref.held(x[:, :w.W].double())
    bad = ~torch.isfinite(x[:, :w.W].double()).all(-1)
    rows[bad, :Dc], rows[bad, Dc:] = 0, float("nan")
    for s in range(len(kv)):
        r = w.mine(s)
        page, row = w.slots(s, torch.arange(kv[s] - q[s], kv[s]))
        mine = rows[r].clone()
        got = w.pool.data[1].cpu()[page, row]
        assert torch.equal(torch.isnan(got), torch.isnan(mine))
        w.data[1, page, row] = got                   # (the NaN's bits are the kernel's)
        assert torch.equal(got.nan_to_num(), mine.nan_to_num())
    w.same_pool()
    for out in DT.values():
        latent, rope = akv.latent_read(w.pool, w.batch, layer=1, dtype=out)
        got, want = torch.cat([latent, rope], -1).cpu(), back.to(out)
        assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got.nan_to_num(), want.nan_to_num())


ROWS = [(16, [517], [1]), (5, [1, 70, 0, 33], [1, 1, 0, 1]), (1, [200, 3], [16, 3]), (20, [90, 64, 65], [1, 1, 1]), (33, [130, 31], [1, 1]),
        (64, [257, 100], [1, 1]), (7, [100, 9], [9, 9]), (128, [300, 1, 64], [1, 1, 1]), (128, [150, 40], [3, 2]), (16, [400, 33, 77], [40, 1, 9]),
        (3, [70], [70])]


@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("Dc,P", FORMS)
@pytest.mark.parametrize("H,kv,q", ROWS)
def test_attention(H, kv, q, Dc, P, dt):
    announce(f"latent attention H={H} kv={kv} q={q} Dc={Dc} P={P} {dt}")
    w = World(Dc, P, kv, q)
    w.fill()
    _check_attention(w, H, dt)
    if max(q) > 1:
        _check_attention(w, H, dt, causal=False)
    w.same_pool()


@pytest.mark.parametrize("H,kv,q,P", [(16, [20011], [1], 64), (16, [9000, 33, 15000], [1, 1, 1], 16), (128, [6001, 17], [1, 1], 64), (40, [5000, 4001], [1, 2], 32),
                                      (64, [4100], [6], 16), (16, [3000, 70], [30, 1], 128)])
@pytest.mark.parametrize("Dc", [512, 256])
def test_attention_split_over_workgroups(H, kv, q, P, Dc):
    announce(f"latent attention, long: H={H} kv={kv} q={q} P={P} Dc={Dc}")
    w = World(Dc, P, kv, q)
    w.fill()
    _check_attention(w, H, "bf16")


@pytest.mark.parametrize("n,H,q", [(300, 16, 1), (700, 8, 2), (257, 48, 1)])
def test_attention_of_many_sequences(n, H, q):
    announce(f"latent attention of {n} sequences, H={H}")
    g = torch.Generator().manual_seed(3)
    kv = torch.randint(0, 90, (n,), generator=g).tolist()
    w = World(256, 16, [max(k, q) if i % 5 else k for i, k in enumerate(kv)], [q if i % 5 else 0 for i in range(n)])
    w.fill()
    _check_attention(w, H, "fp16")


@pytest.mark.parametrize("Dc,P", FORMS[:3])
@pytest.mark.parametrize("H,kv,m", [(8, 70, 6), (16, 500, 4), (2, 300, 90), (128, 90, 3)])
def test_rows_do_not_feel_what_they_do_not_see(H, kv, m, Dc, P):
    """A new token that holds NaN: rows before it are as without it, rows that see it NaN."""
    import akv
    announce(f"latent attention, a NaN token: H={H} kv={kv} m={m} Dc={Dc} P={P}")
    w = World(Dc, P, [kv], [m])
    w.fill()
    at = kv - m + m // 2
    page, row = w.slots(0, torch.tensor([at]))
    q, qr, _ = _queries(w, H, "bf16")
    q, qr = q.contiguous(), qr.contiguous()
    weights = akv.LatentWeights(*(_randn(H, 128, Dc, seed=s, scale=Dc ** -0.5).cuda() for s in (1, 2)))
    qe = _randn(w.T, H, 128 + DR, seed=9, dt="bf16").cuda()
    clean = akv.latent_attention(q, qr, w.pool, w.batch, _scale(), return_lse=True) + (akv.latent_prefill(qe, w.pool, w.batch, weights),)
    bad = _randn(m, w.W, seed=4)
    pos = torch.arange(kv - m, kv)
    keep = w.data[0, page, row].clone()
    bad[:] = w.data[0][w.slots(0, pos)]
    bad[m // 2, 100] = float("nan")
    akv.latent_append(w.pool, w.batch, bad[:, :Dc].cuda(), bad[:, Dc:].cuda())
    got = akv.latent_attention(q, qr, w.pool, w.batch, _scale(), return_lse=True) + (akv.latent_prefill(qe, w.pool, w.batch, weights),)
    for a, b in zip(clean, got):
        assert torch.equal(a[:m // 2], b[:m // 2])
        assert bool(torch.isnan(b[m // 2:]).all())
    scores = torch.zeros(1, kv, device="cuda")
    akv.latent_importance(q, qr, clean[1], w.pool, w.batch, scores, _scale(), q_window=m - m // 2)
    assert bool(torch.isnan(scores[0, at])) and int(torch.isnan(scores).sum()) == 1
    assert keep is not None


def test_rows_past_the_table_and_missing_pages():
    """Tokens without a slot are not seen, the others are; a page outside the pool holds none."""
    import akv
    announce("latent rows past the table, pages outside the pool")
    for H, kv, q in ((16, [70, 40], [1, 1]), (8, [66, 100, 64, 80], [4, 40, 1, 8]), (128, [90, 33], [2, 1])):
        w = World(512, 16, kv, q, width=4)
        w.fill()
        _check_attention(w, H, "fp16")
    for hole in (2 ** 31 - 1, -1, 10 ** 6):
        w = World(512, 16, [200, 60], [1, 3])
        w.fill()
        w.batch.page_table[0, 3] = w.batch.page_table[1, 1] = hole
        gone = {0: slice(48, 64), 1: slice(16, 32)}
        for H in (16, 40):
            q, qr, x = _queries(w, H, "fp16")
            out = akv.latent_attention(q, qr, w.pool, w.batch, _scale())
            weights = [_randn(H, 128, 512, seed=s, scale=512 ** -0.5) for s in (1, 2)]
            qe = _randn(w.T, H, 192, seed=9)
            pre = akv.latent_prefill(qe.cuda(), w.pool, w.batch, akv.LatentWeights(*(a.cuda() for a in weights)))
            for s in (0, 1):
                rows = w.rows(s)
                stay = torch.ones(len(rows), dtype=torch.bool)
                stay[gone[s]] = False
                r = w.mine(s)
                for i in range(w.q[s]):
                    n = w.kv[s] - w.q[s] + 1 + i
                    some = rows[:n][stay[:n]]
                    at = slice(r.start + i, r.start + i + 1)
                    e, _, b, _ = ref.attention(x[at, :, :512], x[at, :, 512:], some, _scale(), 2.0 ** -11)
                    assert bool(((out[at].double().cpu() - e).abs() <= b).all())
                    e, b = ref.prefill(qe[at].double(), some, weights[0].double(), weights[1].double(), _scale(), 2.0 ** -11)
                    assert bool(((pre[at].double().cpu() - e).abs() <= b).all())


def test_rows_of_no_sequence():
    """A padded batch: the C call leaves the rows behind the last sequence alone, a read makes them 0."""
    import akv
    from akv import _native as nat
    from akv import paged_latent as pl
    announce("latent rows of no sequence")
    for H, q in ((16, [1, 1]), (128, [1, 3])):
        w = World(256, 16, [50, 70], q)
        w.fill()
        T = w.T + 5
        batch = akv.PagedBatch(w.batch.page_table, w.batch.kv_lens, w.batch.q_starts, T, max(q))
        qq, qr = _randn(T, H, 256, seed=1).cuda(), _randn(T, H, DR, seed=2).cuda()
        out, lse = torch.full((T, H, 256), 7.0, device="cuda").half(), torch.full((T, H), 7.0, device="cuda")
        head = (nat.ABI_VERSION, 0, H, 0, 1, _scale(), w.pool._c, batch._c, qq.data_ptr(), qr.data_ptr(), H * 512, 512, H * 128, 128,
                out.data_ptr(), lse.data_ptr())
        lib = nat.load()
        need = lib.akv_latent_attn_workspace_bytes(pl._ATTN.pack(*head, 0, 0))
        ws = torch.empty(need, dtype=torch.uint8, device="cuda")
        assert lib.akv_latent_attn(pl._ATTN.pack(*head, ws.data_ptr(), need), torch.cuda.current_stream().cuda_stream) == 0
        assert bool((out[w.T:] == 7).all()) and bool((lse[w.T:] == 7).all()) and not bool((out[:w.T] == 7).all(-1).any())
        latent, rope = akv.latent_read(w.pool, batch)
        assert not bool(latent[w.T:].any()) and not bool(rope[w.T:].any()) and bool(latent[:w.T].any(-1).all())
        x = _randn(T, w.W, seed=8).cuda()
        akv.latent_append(w.pool, batch, x[:, :256], x[:, 256:])
        got = akv.latent_read(w.pool, batch)
        assert torch.equal(got[0][:w.T], x[:w.T, :256]) and not bool(got[0][w.T:].any())


PREFILL = [(4, [1], [1], 0), (3, [5, 0, 64], [5, 0, 1], 0), (2, [200, 130], [200, 65], 0), (5, [300, 16, 90], [129, 16, 0], 1), (1, [700], [300], 0),
           (16, [260, 33], [257, 33], 1)]


@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("Dc,P", FORMS)
@pytest.mark.parametrize("H,kv,q,layer", PREFILL)
def test_prefill(H, kv, q, layer, Dc, P, dt):
    announce(f"latent prefill H={H} kv={kv} q={q} Dc={Dc} P={P} {dt}")
    w = World(Dc, P, kv, q, layers=2)
    w.fill(layer=layer)
    _check_prefill(w, H, dt, layer=layer)
    if max(q) > 1:
        _check_prefill(w, H, dt, layer=layer, causal=False)
    w.same_pool()


def _check_prefill(w, H, dt, layer=0, causal=True, w_scale=1.0):
    import akv
    wk, wv = (_randn(H, 128, w.Dc, seed=s, dt=dt, scale=w_scale * w.Dc ** -0.5) for s in (21, 22))
    x = _randn(w.T, H, 128 + DR + 8, seed=23, dt=dt)
    out = akv.latent_prefill(x.cuda()[..., :128 + DR], w.pool, w.batch, akv.LatentWeights(wk.cuda(), wv.cuda()), layer, causal=causal)
    x = x[..., :128 + DR].double()
    for s in range(len(w.kv)):
        r = w.mine(s)
        if w.q[s] == 0:
            continue
        e, b = ref.prefill(x[r], w.rows(s, layer), wk.double(), wv.double(), _scale(), torch.finfo(DT[dt]).eps / 2, causal, n=w.kv[s])
        d = (out[r].double().cpu() - e).abs()
        assert bool((d <= b).all()), (s, float((d / b).max()))
    return out


@pytest.mark.parametrize("H,kv,q,P", [(2, [3001, 100], [40, 100], 64), (1, [6000], [500], 16), (8, [1500, 1, 700], [300, 1, 600], 32)])
def test_prefill_split_over_workgroups(H, kv, q, P):
    announce(f"latent prefill, long: H={H} kv={kv} q={q} P={P}")
    w = World(512, P, kv, q)
    w.fill()
    _check_prefill(w, H, "bf16")


@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("Dc,P,H,kv,q,causal", [(512, 64, 128, [700, 40, 0], [300, 40, 0], True), (256, 16, 128, [333, 1], [332, 1], False),
                                                (256, 32, 64, [1031], [1000], True)])
def test_prefill_of_many_tiles(Dc, P, H, kv, q, causal, dt):
    """Enough heads and tokens that workgroups take 256 query tokens each."""
    announce(f"latent prefill, many tiles: H={H} kv={kv} q={q} Dc={Dc} P={P} {dt}")
    w = World(Dc, P, kv, q)
    w.fill()
    _check_prefill(w, H, dt, causal=causal)
    w.same_pool()


@pytest.mark.parametrize("dt", ["fp16", "bf16"])
def test_prefill_of_many_tiles_with_missing_pages(dt):
    import akv
    announce(f"latent prefill, many tiles and pages outside the pool: {dt}")
    H = 128
    w = World(512, 16, [500, 40], [300, 40])
    w.fill()
    w.batch.page_table[0, 3] = w.batch.page_table[0, 20] = w.batch.page_table[1, 0] = -1
    stay = [torch.ones(n, dtype=torch.bool) for n in w.kv]
    stay[0][48:64] = stay[0][320:336] = stay[1][:16] = False
    weights = [_randn(H, 128, 512, seed=s, dt=dt, scale=512 ** -0.5) for s in (1, 2)]
    q = _randn(w.T, H, 192, seed=9, dt=dt)
    got = akv.latent_prefill(q.cuda(), w.pool, w.batch, akv.LatentWeights(*(a.cuda() for a in weights))).double().cpu()
    for s, i in ((0, 0), (0, 128), (0, 299), (1, 3), (1, 39)):
        n, at = w.kv[s] - w.q[s] + 1 + i, slice(w.mine(s).start + i, w.mine(s).start + i + 1)
        e, b = ref.prefill(q[at].double(), w.rows(s)[:n][stay[s][:n]], weights[0].double(), weights[1].double(), _scale(),
                           torch.finfo(DT[dt]).eps / 2)
        assert bool(((got[at] - e).abs() <= b).all()), (s, i)
    assert not bool(got[w.mine(1)][:16].any())  # these see no token


def test_prefill_of_many_tiles_captured():
    """A captured call follows lengths and tables that change, as an eager one does."""
    import akv
    announce("latent prefill, many tiles, captured")
    H = 128
    w = World(256, 32, [300, 200], [200, 60])
    w.fill()
    wt = akv.LatentWeights(*(_randn(H, 128, 256, seed=s, scale=256 ** -0.5).cuda() for s in (1, 2)))
    q = _randn(w.T, H, 192, seed=3, dt="bf16").cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        akv.latent_prefill(q, w.pool, w.batch, wt)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = akv.latent_prefill(q, w.pool, w.batch, wt)
    table = w.batch.page_table.clone()
    for lens, hole in (([300, 200], None), ([260, 61], None), ([300, 200], (0, 2)), ([200, 0], None)):
        w.batch.kv_lens.copy_(torch.tensor(lens, dtype=torch.int32))
        w.batch.page_table.copy_(table)
        if hole:
            w.batch.page_table[hole] = -1
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, akv.latent_prefill(q, w.pool, w.batch, wt)), lens


@pytest.mark.parametrize("size", [1e-6, 1e-3, 1e4])
def test_weights_of_any_size(size):
    announce(f"latent prefill, weights times {size}")
    w = World(256, 32, [150], [33])
    w.fill()
    import akv
    H = 3
    wk, wv = (_randn(H, 128, 256, seed=s, dt="bf16", scale=x * 256 ** -0.5) for s, x in ((21, 1.0), (22, size)))
    q = _randn(w.T, H, 192, seed=23, dt="bf16")
    out = akv.latent_prefill(q.cuda(), w.pool, w.batch, akv.LatentWeights(wk.cuda(), wv.cuda()))
    e, b = ref.prefill(q.double(), w.rows(0), wk.double(), wv.double(), _scale(), 2.0 ** -8)
    b = b - 2.0 ** -25  # (bfloat16's smallest step is no limit here)
    d = (out.double().cpu() - e).abs()
    assert bool((d <= b).all()), float((d / b).max())


def test_prefill_types_share_a_batch():
    """Float16 queries take more workspace than bfloat16 ones of the same sizes."""
    import akv
    announce("latent prefill, bfloat16 then float16 on one batch")
    H = 5
    w = World(512, 64, [300, 90], [40, 90])
    w.fill()
    wt = akv.LatentWeights(*(_randn(H, 128, 512, seed=s, scale=512 ** -0.5).cuda() for s in (1, 2)))
    q = _randn(w.T, H, 192, seed=3, dt="bf16")
    first = akv.latent_prefill(q.cuda(), w.pool, w.batch, wt)
    after = akv.latent_prefill(q.half().cuda(), w.pool, w.batch, wt)
    fresh = akv.PagedBatch(w.batch.page_table, w.batch.kv_lens, w.batch.q_starts, w.T, w.batch.max_q)
    assert torch.equal(after, akv.latent_prefill(q.half().cuda(), w.pool, fresh, wt))
    assert torch.equal(first, akv.latent_prefill(q.cuda(), w.pool, w.batch, wt))


@pytest.mark.parametrize("Dc", [256, 512])
def test_prefill_holds_what_float16_cannot(Dc):
    """A value beyond 65504 times its channel's scale is held there: equal weights of 1 have the scale 32."""
    import akv
    announce(f"latent prefill, values beyond float16: Dc={Dc}")
    w = World(Dc, 16, [1], [1])
    page, row = w.slots(0, torch.arange(1))
    w.data[0, page, row] = 61440.0
    w.pool = akv.PagedLatentPool(w.data.cuda(), Dc)
    ones = torch.ones(1, 128, Dc).cuda()
    sign = torch.where(torch.arange(128) % 2 == 0, 1.0, -1.0).cuda()
    out = akv.latent_prefill(torch.zeros(1, 1, 192, dtype=torch.bfloat16).cuda(), w.pool, w.batch,
                             akv.LatentWeights(ones, ones * sign[None, :, None]))
    assert torch.equal(out[0, 0], (65504.0 * 32.0 * sign).bfloat16())


def test_prefill_in_passes_of_heads(monkeypatch):
    """A table so wide that the heads take more than one pass: as one pass with a narrow one."""
    import akv
    announce("latent prefill in passes")
    H = 7
    w = World(256, 256, [500], [60])
    w.fill()
    wt = akv.LatentWeights(*(_randn(H, 128, 256, seed=s, scale=256 ** -0.5).cuda() for s in (1, 2)))
    q = _randn(w.T, H, 192, seed=3).cuda()
    want = akv.latent_prefill(q, w.pool, w.batch, wt)
    wide = torch.full((1, 11000), -1, dtype=torch.int32, device="cuda")  # 2.8 million slots, 1.4 GB a head
    wide[:, :w.batch.page_table.shape[1]] = w.batch.page_table
    got = akv.latent_prefill(q, w.pool, akv.PagedBatch(wide, w.batch.kv_lens, w.batch.q_starts, w.T, 60), wt)
    # heads that share runs with others split elsewhere: the last bits of float32 sums
    assert float((got.float() - want.float()).abs().max()) <= 2.0 ** -10 * float(want.float().abs().max())


def test_importance_of_many_rows_captured():
    """A captured call, with a window and without, follows lengths, rows and tables that change."""
    import akv
    announce("latent importance, many rows, captured")
    H, T = 9, 40
    w = World(512, 16, [260, 90, 300], [20, 8, 12])
    w.fill()
    q, qr, _ = _queries(w, H, "bf16")
    lse = akv.latent_attention(q, qr, w.pool, w.batch, _scale(), return_lse=True)[1]
    table = w.batch.page_table.clone()
    for window in (0, 5):
        scores = torch.rand(3, 290, generator=torch.Generator().manual_seed(2)).cuda()
        out = torch.empty_like(scores)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            akv.latent_importance(q, qr, lse, w.pool, w.batch, scores, _scale(), q_window=window, out=out)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            akv.latent_importance(q, qr, lse, w.pool, w.batch, scores, _scale(), q_window=window, out=out)
        for lens, starts, hole in (([260, 90, 300], [0, 20, 28, 40], None), ([255, 8, 290], [0, 1, 21, 40], None),
                                   ([0, 90, 128], [0, 0, 20, 23], (1, 2)), ([260, 90, 300], [0, 20, 28, 40], None)):
            w.batch.kv_lens.copy_(torch.tensor(lens, dtype=torch.int32))
            w.batch.q_starts.copy_(torch.tensor(starts, dtype=torch.int32))
            w.batch.page_table.copy_(table)
            if hole:
                w.batch.page_table[hole] = -1
            out.fill_(-1.0)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, akv.latent_importance(q, qr, lse, w.pool, w.batch, scores, _scale(), q_window=window, out=torch.empty_like(out)))


@pytest.mark.parametrize("Dc,P", FORMS)
@pytest.mark.parametrize("H,kv,q,win", [(16, [517, 33], [1, 1], 0), (5, [130, 0, 64], [9, 0, 3], 4), (40, [300], [20], 0), (128, [200, 70], [1, 2], 1), (1, [31], [31], 0)])
def test_importance(H, kv, q, win, Dc, P):
    import akv
    announce(f"latent importance H={H} kv={kv} q={q} win={win} Dc={Dc} P={P}")
    w = World(Dc, P, kv, q)
    w.fill()
    for dt in ("fp16", "bf16"):
        _, lse, q_, qr_, x = _check_attention(w, H, dt)
        N = max(kv) - 5 if max(kv) > 50 else max(kv) + 3   # fewer scores than tokens, or more
        both = torch.rand(2 * len(kv), N + 4, generator=torch.Generator().manual_seed(1)).cuda()
        scores, before = both[::2, 2:N + 2], both.clone()
        out = akv.latent_importance(q_, qr_, lse, w.pool, w.batch, scores, _scale(), decay=0.75, q_window=win, out=torch.full_like(scores, -1.0))
        akv.latent_importance(q_, qr_, lse, w.pool, w.batch, scores, _scale(), decay=0.75, q_window=win)
        assert torch.equal(scores, out)
        both[::2, 2:N + 2] = before[::2, 2:N + 2]
        assert torch.equal(both, before)                   # nothing else was written
        old = before[::2, 2:N + 2].double().cpu()
        for s in range(len(kv)):
            n = min(kv[s], N) if w.q[s] else 0
            assert torch.equal(out[s, n:].cpu(), before[2 * s, 2 + n:N + 2].cpu())
            if n == 0:
                continue
            r = w.mine(s)
            e, b = ref.importance(x[r, :, :Dc], x[r, :, Dc:], w.rows(s), _scale(), lse[r].double().cpu(), window=win)
            want = old[s, :n] * 0.75 + e[:n]
            assert bool(((out[s, :n].double().cpu() - want).abs() <= b[:n] + 2.0 ** -22 * want).all()), s


@pytest.mark.parametrize("Dc,P", FORMS)
def test_copies_and_compaction(Dc, P):
    import akv
    announce(f"latent copies and compaction Dc={Dc} P={P}")
    w = World(Dc, P, [300, 1, 0, 95], [0, 0, 0, 0], layers=2, spare=3 + 2 * (300 // P + 3))
    src = torch.tensor([int(w.table[0, 0]), int(w.table[3, 0]), 10 ** 6], dtype=torch.int32)
    dst = torch.tensor([int(w.spare[0]), int(w.spare[1]), int(w.spare[2])], dtype=torch.int32)
    akv.copy_pages(w.pool, src.cuda(), dst.cuda())
    w.data[:, dst[:2].long()] = w.data[:, src[:2].long()]
    w.same_pool()
    keep = [torch.arange(0, 300, 2), torch.tensor([0]), torch.tensor([], dtype=torch.int64), torch.tensor([0, 1, 2, 50, 94, 94])]
    free = w.spare[3:].tolist()
    to = torch.full((4, 150 // P + 1), -1, dtype=torch.int32)
    for s, k in enumerate(keep):
        for j in range(-(-len(k) // P)):
            to[s, j] = free.pop()
    rows = torch.nn.utils.rnn.pad_sequence(keep, batch_first=True, padding_value=-1).to(torch.int32)
    akv.compact_pages(w.pool, w.batch.page_table, to.cuda(), rows.cuda(), torch.tensor([len(k) for k in keep], dtype=torch.int32).cuda())
    for s, k in enumerate(keep):
        j = torch.arange(len(k))
        page, row = w.slots(s, k)
        w.data[:, to[s].long()[j // P], j % P] = w.data[:, page, row]
    w.same_pool()


def test_pages_past_32_bits_of_bytes():
    import akv
    announce("a latent pool of more than 4 GiB")
    P, Dc = 256, 512
    n = 2 ** 32 // (P * 1152) + 40
    pool = akv.PagedLatentPool(torch.empty(1, n, P, 576, dtype=torch.float16, device="cuda"), Dc)
    table = torch.tensor([[n - 1, 3, n - 7]], dtype=torch.int32, device="cuda")
    i = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    x = _randn(700, 576, seed=1).cuda()
    akv.latent_append(pool, akv.PagedBatch(table, i(700), i(0, 700), 700, 700), x[:, :Dc], x[:, Dc:])
    one = akv.PagedBatch(table, i(700), i(0, 1), 1, 1)
    for H in (16, 64):
        q, qr = _randn(1, H, Dc, seed=2, scale=0.6).cuda(), _randn(1, H, DR, seed=3).cuda()
        out = akv.latent_attention(q, qr, pool, one, _scale())
        e, _, b, _ = ref.attention(q.double().cpu(), qr.double().cpu(), x.double().cpu(), _scale(), 2.0 ** -11)
        assert bool(((out.double().cpu() - e).abs() <= b).all())
    wk, wv = (_randn(2, 128, Dc, seed=s, scale=Dc ** -0.5) for s in (5, 6))
    q = _randn(1, 2, 192, seed=7)
    out = akv.latent_prefill(q.cuda(), pool, one, akv.LatentWeights(wk.cuda(), wv.cuda()))
    e, b = ref.prefill(q.double(), x.double().cpu(), wk.double(), wv.double(), _scale(), 2.0 ** -11)
    assert bool(((out.double().cpu() - e).abs() <= b).all())


@pytest.mark.parametrize("dt,limit", [("fp16", 3.1e-4), ("bf16", 2.3e-3)])
@pytest.mark.parametrize("kv,H", [(30000, 2), (9000, 40)])
def test_precision(kv, H, dt, limit):
    """The norm of the outputs' error: rounding the result alone leaves 2.1e-4 (float16) and 1.7e-3
    (bfloat16) of theirs; p in float16 adds up to as much as the former, in quadrature."""
    announce(f"latent precision kv={kv} H={H} {dt}")
    w = World(512, 64, [kv], [1])
    w.fill()
    out, lse, _, _, x = _check_attention(w, H, dt)
    e, el, _, _ = ref.attention(x[..., :512], x[..., 512:], w.rows(0), _scale(), 0.0)
    assert float((out.double().cpu() - e).norm() / e.norm()) < limit
    assert float((lse.double().cpu() - el).norm() / el.norm()) < 1e-6


def test_light_tokens_beside_a_heavy_one():
    """One token has nearly all of the weight and a value of 0, the others share what is left: their
    part keeps its bits, wherever the heavy one stands."""
    import akv
    announce("latent attention, a heavy token")
    n, Dc = 4000, 512
    for H, at in ((16, 0), (16, 3999), (40, 2000), (128, 17)):
        w = World(Dc, 64, [n], [1])
        x = _randn(n, w.W, seed=5, dt="fp32")
        x[:, :Dc] *= 0.5
        x[:, Dc:] = 0
        x[at, :Dc], x[at, Dc] = 0, 64.0
        page, row = w.slots(0, torch.arange(n))
        w.data[0, page, row] = x.half()
        w.pool.data.copy_(w.data)
        q, qr = torch.zeros(1, H, Dc), torch.zeros(1, H, DR)
        qr[..., 0] = 1.0
        scale = float(torch.tensor(n * 1e3).log()) / 64        # the others: 1e-3 of the weight together
        out = akv.latent_attention(q.half().cuda(), qr.half().cuda(), w.pool, w.batch, scale)
        e = ref.attention(q.double(), qr.double(), w.rows(0), scale, 0.0)[0]
        # p in float16 and the output's own rounding, a half step each, and its smallest step
        err = (out.double().cpu() - e).abs()
        A = ref.attention(q.double(), qr.double(), w.rows(0).abs(), scale, 0.0)[0]
        assert bool((err <= 2.0 ** -10 * A + 2.0 ** -25).all()), float((err / A).max())
