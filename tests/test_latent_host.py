"""The paged latent cache's refusals and layouts, on the host."""
import ctypes

import pytest
import torch

from test_paged_host import BATCHES, _batch


def _pool(nat, **kw):
    d = dict(data=4096, n_pages=4, num_layers=2, latent_dim=512, rope_dim=64, page_size=16)
    d.update(kw)
    return nat.LatentPool(**d)


POOLS = [(dict(latent_dim=128), "E_UNSUPPORTED"), (dict(latent_dim=0), "E_UNSUPPORTED"), (dict(rope_dim=32), "E_UNSUPPORTED"),
         (dict(page_size=8), "E_UNSUPPORTED"), (dict(page_size=48), "E_UNSUPPORTED"), (dict(page_size=512), "E_UNSUPPORTED"),
         (dict(num_layers=0), "E_SHAPE"), (dict(n_pages=-1), "E_SHAPE"), (dict(data=0), "E_INVALID"), (dict(data=8), "E_ALIGN")]


@pytest.mark.parametrize("call", ["rows", "attn", "prefill", "importance"])
def test_c_refusals(call):
    from akv import _native as nat
    lib = nat.load()

    def run(pool=None, batch=None, **kw):
        common = dict(abi_version=nat.ABI_VERSION, layer=0, pool=_pool(nat, **(pool or {})), batch=_batch(nat, **(batch or {})))
        if call == "rows":
            a = nat.LatentRowsArgs(**{**common, "dtype": 0, "latent": 4096, "rope": 4096, "latent_t": 1024, "rope_t": 128, **kw})
            return lib.akv_latent_append(ctypes.byref(a), None), lib.akv_latent_read(ctypes.byref(a), None)
        q = dict(H=4, q_dtype=0, causal=1, sm_scale=0.1, q=4096, q_t=4096, q_h=1024, out=4096)
        qr = dict(q_rope=4096, q_rope_t=512, q_rope_h=128, lse=4096)
        ws = dict(workspace=4096, workspace_bytes=64)
        if call == "attn":
            a, fn, ask = nat.LatentAttnArgs(**{**common, **q, **qr, **ws, **kw}), lib.akv_latent_attn, lib.akv_latent_attn_workspace_bytes
        elif call == "prefill":
            a = nat.LatentPrefillArgs(**{**common, **q, **ws, "w": 4096, "w_scale": 4096, **kw})
            fn, ask = lib.akv_latent_prefill, lib.akv_latent_prefill_workspace_bytes
        else:
            a = nat.LatentImportanceArgs(**{**common, **q, **qr, "q_window": 0, "decay": 0.9, "scores": 4096, "n_scores": 10,
                                            "score_stride": 10, "out_stride": 10, **kw})
            return (lib.akv_latent_importance(ctypes.byref(a), None),)
        rc = fn(ctypes.byref(a), None)
        if rc in (nat.AKV_E_SHAPE, nat.AKV_E_DTYPE, nat.AKV_E_UNSUPPORTED, nat.AKV_E_ABI):
            assert ask(ctypes.byref(a)) == -1
        return (rc,)

    code = lambda name: getattr(nat, "AKV_" + name)  # noqa: E731
    for kw, want in POOLS:
        assert set(run(pool=kw)) == {code(want)}, (kw, lib.akv_last_error())
    for kw, want in BATCHES:
        assert set(run(batch=kw)) == {code(want)}, (kw, lib.akv_last_error())
    own = [(dict(abi_version=4), "E_ABI"), (dict(layer=2), "E_SHAPE"), (dict(layer=-1), "E_SHAPE")]
    if call == "rows":
        own += [(dict(dtype=3), "E_DTYPE"), (dict(latent=0), "E_INVALID"), (dict(rope=4100), "E_ALIGN"), (dict(latent_t=1032), "E_ALIGN")]
    else:
        own += [(dict(q_dtype=2), "E_DTYPE"), (dict(H=0), "E_SHAPE"), (dict(H=65536), "E_SHAPE"), (dict(sm_scale=0.0), "E_INVALID"),
                (dict(sm_scale=float("nan")), "E_INVALID"), (dict(sm_scale=float("inf")), "E_INVALID"), (dict(q=0), "E_INVALID"),
                (dict(q=4100), "E_ALIGN"), (dict(q_h=260), "E_ALIGN"), (dict(out=0), "E_INVALID")]
    if call in ("attn", "importance"):
        own += [(dict(q_rope=0), "E_INVALID"), (dict(q_rope_t=8), "E_ALIGN"), (dict(lse=4097), "E_ALIGN")]
    if call in ("attn", "prefill"):
        own += [(dict(workspace=0), "E_WORKSPACE"), (dict(workspace_bytes=63), "E_WORKSPACE"), (dict(out=4100), "E_ALIGN")]
    if call == "prefill":
        own += [(dict(w=0), "E_INVALID"), (dict(w_scale=0), "E_INVALID"), (dict(w=4104), "E_ALIGN")]
    if call == "importance":
        own += [(dict(q_window=-1), "E_SHAPE"), (dict(score_stride=9), "E_SHAPE"), (dict(n_scores=-1), "E_SHAPE"),
                (dict(lse=0), "E_INVALID"), (dict(scores=0), "E_INVALID"), (dict(out=4098), "E_ALIGN"), (dict(out=4100), "E_SHAPE")]
    for kw, want in own:
        assert set(run(**kw)) == {code(want)}, (kw, lib.akv_last_error())
    if call == "attn":  # more units than a call counts
        assert run(batch=dict(max_q=2 ** 20, n_tokens=2 ** 21, table_width=2 ** 16, table_stride=2 ** 16)) == (nat.AKV_E_SHAPE,)


def test_c_attention_counts_units_of_its_tiles():
    """A wide table and a chunk in a batch: refused where the units of the tiles that the call takes pass 2^30, not before."""
    from akv import _native as nat
    lib = nat.load()

    def need(S, q, H, tokens):
        a = nat.LatentAttnArgs(abi_version=nat.ABI_VERSION, layer=0, pool=_pool(nat, page_size=64), H=H, q_dtype=1, causal=1, sm_scale=0.1,
                               batch=_batch(nat, n_seqs=S, n_tokens=S * q, max_q=q, table_width=tokens // 64, table_stride=tokens // 64),
                               q=4096, q_t=4096, q_h=1024, q_rope=4096, q_rope_t=512, q_rope_h=128, out=4096)
        return lib.akv_latent_attn_workspace_bytes(ctypes.byref(a))
    # units (with eight for an item) times tiles of 128, 64 and 16 rows times sequences
    for S, q, H, tokens, tile in ((256, 512, 128, 131072, 128), (4096, 1, 64, 2 ** 22, 64), (8000, 1, 16, 2 ** 22, 16), (1, 2 ** 19, 128, 65536, 128)):
        units = (tokens // 64 + 8) * (q * H // tile + 1) * S
        assert (need(S, q, H, tokens) > 0) == (units < 2 ** 30), (S, q, H, tokens)
        more = 2 * 2 ** 30 // units + 1
        assert need(min(65535, S * more), q, H, tokens) == -1


def test_c_importance_workspace():
    """None for up to 16 rows a sequence, else blocks of 16 rows that hold every sequence's in pairs."""
    from akv import _native as nat
    lib = nat.load()

    def args(H, T, max_q, S=2, window=0, Dc=512, **kw):
        return nat.LatentImportanceArgs(abi_version=nat.ABI_VERSION, layer=0, pool=_pool(nat, latent_dim=Dc),
                                        batch=_batch(nat, n_seqs=S, n_tokens=T, max_q=max_q), H=H, q_dtype=0, causal=1, sm_scale=0.1,
                                        q=4096, q_t=4096, q_h=1024, q_rope=4096, q_rope_t=512, q_rope_h=128, lse=4096, q_window=window,
                                        decay=0.9, scores=4096, out=4096, n_scores=10, score_stride=10, out_stride=10, **kw)

    def need(*a, **kw):
        return lib.akv_latent_importance_workspace_bytes(ctypes.byref(args(*a, **kw)))

    assert need(16, 2, 1) == need(4, 8, 4) == need(4, 50, 30, window=4) == need(1, 16, 16) == 0
    for H, T, q, window, Dc in ((17, 2, 1, 0, 512), (16, 3, 2, 0, 256), (3, 40, 33, 0, 512), (128, 64, 60, 7, 256), (1, 17, 17, 0, 512)):
        block = 1024 * ((Dc + 64) // 32 + 1)
        for lens in ((q, T - q), (T - q, q)):
            at = 0
            for s, n in enumerate(lens):  # a sequence's blocks lie before the next one's, the last one's inside
                rows = min(n, window or n) * H
                first = (s * min(window, q) if window else sum(lens[:s])) * H // 16 + 3 * s
                assert first >= at
                at = first + 2 * -(-rows // 32)
            assert at * block <= need(H, T, q, window=window, Dc=Dc)
    more = need(17, 2, 1)
    for kw, want in ((dict(), nat.AKV_E_WORKSPACE), (dict(workspace=4096, workspace_bytes=more - 1), nat.AKV_E_WORKSPACE),
                     (dict(workspace=4104, workspace_bytes=more), nat.AKV_E_ALIGN)):
        assert lib.akv_latent_importance(ctypes.byref(args(17, 2, 1, **kw)), None) == want


def test_c_refusals_of_moves():
    from akv import _native as nat
    lib = nat.load()
    for kw, want in POOLS:
        p = _pool(nat, **kw)
        assert lib.akv_latent_copy(ctypes.byref(p), 4096, 4096, 1, None) == getattr(nat, "AKV_" + want), kw
    p = _pool(nat)
    assert lib.akv_latent_copy(None, None, None, 0, None) == nat.AKV_E_INVALID
    for n, a, b, want in ((5, 4096, 4096, nat.AKV_E_SHAPE), (-1, 4096, 4096, nat.AKV_E_SHAPE), (1, None, 4096, nat.AKV_E_INVALID),
                          (1, 4096, 4098, nat.AKV_E_ALIGN), (0, None, None, nat.AKV_OK)):
        assert lib.akv_latent_copy(ctypes.byref(p), a, b, n, None) == want
    base = dict(abi_version=nat.ABI_VERSION, n_seqs=2, pool=p, src_table=4096, dst_table=4096, src_stride=4, dst_stride=4,
                src_width=4, dst_width=4, keep=4096, n_keep=4096, keep_stride=9, max_keep=9)
    for kw, want in ((dict(abi_version=3), nat.AKV_E_ABI), (dict(n_seqs=-1), nat.AKV_E_SHAPE), (dict(src_stride=3), nat.AKV_E_SHAPE),
                     (dict(keep_stride=8), nat.AKV_E_SHAPE), (dict(dst_width=2 ** 27, dst_stride=2 ** 27), nat.AKV_E_SHAPE),
                     (dict(keep=0), nat.AKV_E_INVALID), (dict(n_keep=0), nat.AKV_E_INVALID), (dict(src_table=0), nat.AKV_E_INVALID),
                     (dict(dst_table=4097), nat.AKV_E_ALIGN)):
        a = nat.LatentCompactArgs(**{**base, **kw})
        assert lib.akv_latent_compact(ctypes.byref(a), None) == want, kw
    assert lib.akv_latent_compact(None, None) == nat.AKV_E_INVALID


def test_c_refusals_of_launches_that_wrap():
    """2^32 work items are none to the runtime: rows, scores and positions that would take as many are refused."""
    from akv import _native as nat
    lib = nat.load()
    for n in (2 ** 29 - 31, 2 ** 29, 2 ** 30, 2 ** 31 - 1):
        a = nat.LatentRowsArgs(abi_version=nat.ABI_VERSION, layer=0, dtype=0, pool=_pool(nat), batch=_batch(nat, n_tokens=n, max_q=1),
                               latent=4096, rope=4096, latent_t=0, rope_t=0)
        assert lib.akv_latent_append(ctypes.byref(a), None) == lib.akv_latent_read(ctypes.byref(a), None) == nat.AKV_E_SHAPE
        c = nat.LatentCompactArgs(abi_version=nat.ABI_VERSION, n_seqs=1, pool=_pool(nat), src_table=4096, dst_table=4096, src_stride=4,
                                  dst_stride=4, src_width=4, dst_width=4, keep=4096, n_keep=4096, keep_stride=n, max_keep=n)
        assert lib.akv_latent_compact(ctypes.byref(c), None) == nat.AKV_E_SHAPE
        for H in (4, 40):
            i = nat.LatentImportanceArgs(abi_version=nat.ABI_VERSION, layer=0, pool=_pool(nat), batch=_batch(nat, n_seqs=1, n_tokens=1, max_q=1),
                                         H=H, q_dtype=0, causal=1, sm_scale=0.1, q=4096, q_t=4096, q_h=1024, q_rope=4096, q_rope_t=512,
                                         q_rope_h=128, lse=4096, q_window=0, decay=0.9, scores=4096, out=4096, n_scores=n, score_stride=n,
                                         out_stride=n)
            assert lib.akv_latent_importance(ctypes.byref(i), None) == nat.AKV_E_SHAPE


def test_c_refusals_of_evictions():
    from akv import _native as nat
    lib = nat.load()
    at = 1 << 20
    base = dict(abi_version=nat.ABI_VERSION, n_seqs=2, scores=at, n_scores=10, score_stride=10, lens=4096, budgets=0, budget=3,
                protect_initial=0, protect_recent=0, keep=4096, n_keep=4096, kept=at + 80, keep_stride=3, max_keep=3, kept_stride=10)
    for kw, want in ((dict(abi_version=3), nat.AKV_E_ABI), (dict(n_seqs=-1), nat.AKV_E_SHAPE), (dict(n_seqs=65536), nat.AKV_E_SHAPE),
                     (dict(n_scores=-1), nat.AKV_E_SHAPE), (dict(score_stride=9), nat.AKV_E_SHAPE), (dict(keep_stride=2), nat.AKV_E_SHAPE),
                     (dict(kept_stride=9), nat.AKV_E_SHAPE), (dict(max_keep=-1), nat.AKV_E_SHAPE), (dict(budget=-1), nat.AKV_E_SHAPE),
                     (dict(protect_initial=-1), nat.AKV_E_SHAPE), (dict(protect_recent=-1), nat.AKV_E_SHAPE), (dict(lens=0), nat.AKV_E_INVALID),
                     (dict(scores=0), nat.AKV_E_INVALID), (dict(keep=0), nat.AKV_E_INVALID), (dict(n_keep=0), nat.AKV_E_INVALID),
                     (dict(keep=4098), nat.AKV_E_ALIGN), (dict(kept=at + 81), nat.AKV_E_ALIGN), (dict(budgets=4097), nat.AKV_E_ALIGN),
                     (dict(kept=at), nat.AKV_E_SHAPE), (dict(kept=at + 76), nat.AKV_E_SHAPE), (dict(kept=at - 76), nat.AKV_E_SHAPE),
                     (dict(n_seqs=0), nat.AKV_OK)):
        a = nat.EvictArgs(**{**base, **kw})
        assert lib.akv_evict_select(ctypes.byref(a), None) == want, (kw, lib.akv_last_error())
    assert lib.akv_evict_select(None, None) == nat.AKV_E_INVALID


def test_host_tensors_are_refused():
    import akv
    with pytest.raises(RuntimeError, match="CPU"):
        akv.PagedLatentPool.empty(1, 4, device="cpu")
    with pytest.raises(RuntimeError):
        akv.PagedLatentCache(1, device="cpu")
    with pytest.raises(RuntimeError, match="CPU"):
        akv.LatentWeights(torch.zeros(2, 128, 512), torch.zeros(2, 128, 512))
    with pytest.raises(RuntimeError, match="CPU"):
        akv.evict_select(torch.zeros(2, 5), torch.zeros(2, dtype=torch.int32), 3)
    for bad in (torch.zeros(1, 2, 16, 576), torch.zeros(2, 16, 576).half(), torch.zeros(1, 2, 16, 512).half()):
        with pytest.raises(ValueError):
            akv.PagedLatentPool(bad, 512)


@pytest.mark.parametrize("Dc", [512, 256])
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16, torch.float32])
def test_weights_layout(Dc, dt, monkeypatch):
    """Value j of lane l of block 4 a + b of step k is weight (64 a + 16 (l % 16 / 4) + 4 b + l % 4,
    32 k + 8 (l / 16) + j), over a power of two that leaves a channel's largest in [2^-5, 2^-4)."""
    import akv
    from akv import paged_latent as pl
    monkeypatch.setattr(pl.nat, "require_device", lambda *t: None)
    H = 3
    g = torch.Generator().manual_seed(1)
    w = torch.randn(H, 256, Dc, generator=g) * torch.logspace(-6, 4, 256)[:, None]
    w[1, 7] = 0
    w = w.to(dt if dt != torch.float16 else torch.float32)
    if dt == torch.float16:
        w = w.clamp(-6e4, 6e4).half()
    t = akv.LatentWeights(w[:, :128], w[:, 128:])
    assert t.data.is_contiguous() and t.scale.is_contiguous() and t.scale.shape == (H, 256)
    flat = t.data.reshape(H, Dc // 32, 16, 64, 8)
    k, blk, l, j = torch.meshgrid(torch.arange(Dc // 32), torch.arange(16), torch.arange(64), torch.arange(8), indexing="ij")
    ch = 64 * (blk // 4) + 16 * (l % 16 // 4) + 4 * (blk % 4) + l % 4
    back = torch.zeros(H, 256, Dc, dtype=torch.float64)
    back[:, ch, 32 * k + 8 * (l // 16) + j] = flat.double()
    top = back.abs().amax(-1)
    # (rounding up may reach 2^-4 itself)
    assert bool((((top >= 2.0 ** -5) & (top <= 2.0 ** -4)) | (w.double().abs().amax(-1) == 0)).all())
    got = back * t.scale.double()[..., None]
    err = (got - w.double()).abs()
    assert bool((err <= 2.0 ** -11 * w.double().abs() + 2.0 ** -20 * w.double().abs().amax(-1, keepdim=True)).all())
    if dt == torch.bfloat16:  # exact but for what lies below float16's steps
        assert bool((err <= 2.0 ** -20 * w.double().abs().amax(-1, keepdim=True)).all())


def _cache(monkeypatch, lens, pages=12, P=16):
    """A cache's books without a device: what would move is noted."""
    from akv import paged_packed as pp

    class Pool:
        page_size, _index, data = P, -1, torch.zeros(0)
    c = pp._PagedCache(Pool(), pages)
    moved = []
    monkeypatch.setattr(pp, "compact_pages", lambda pool, old, new, rows, n: moved.append((old, new, rows, n)))
    seqs = [c.add_sequence() for _ in lens]
    c._book.extend(seqs, lens)
    return pp, c, seqs, moved


def test_eviction_keeps_the_books(monkeypatch):
    import latent_ref as ref
    lens = [40, 7, 64]
    pp, c, seqs, moved = _cache(monkeypatch, lens)
    scores = torch.rand(3, 70, generator=torch.Generator().manual_seed(2))

    def select(s, n, b, first, last):
        keep = [ref.evict(r, int(k), b, first, last) for r, k in zip(s, n)]
        rows = torch.zeros(len(keep), b, dtype=torch.int32)
        kept = torch.zeros_like(s)
        for i, k in enumerate(keep):
            rows[i, :len(k)] = torch.tensor(k, dtype=torch.int32)
            kept[i, :len(k)] = s[i, torch.tensor(k, dtype=torch.long)]
        return rows, torch.tensor([len(k) for k in keep], dtype=torch.int32), kept
    monkeypatch.setattr(pp, "evict_select", select)
    old = [list(c._book.pages[s]) for s in seqs]
    kept = c.evict(seqs, scores, 20, 2, 3)
    assert [c.get_seq_length(s) for s in seqs] == [20, 7, 20]
    assert c._book.pages[seqs[1]] == old[1]              # within the budget: not moved
    assert [len(c._book.pages[s]) for s in seqs] == [2, 1, 2] and c.num_free_pages == 12 - 5
    rows = torch.cat([m[2] for m in moved]).tolist()
    assert rows == [ref.evict(scores[0], 40, 20, 2, 3), ref.evict(scores[2], 64, 20, 2, 3)]
    assert [n for m in moved for n in m[3].tolist()] == [20, 20] and kept.shape == scores.shape
    assert [p for m in moved for r in m[0].tolist() for p in r][:3] == old[0]


def test_eviction_in_turns_and_refusals(monkeypatch):
    lens = [64, 64, 60]
    pp, c, seqs, moved = _cache(monkeypatch, lens, pages=14)  # 4 + 4 + 4 of 14
    monkeypatch.setattr(pp, "evict_select", lambda s, n, b, f, l: (torch.arange(b, dtype=torch.int32).expand(3, b), None, s))
    scores = torch.zeros(3, 64)
    before = [list(c._book.pages[s]) for s in seqs]
    for err, call in ((ValueError, lambda: c.evict(seqs, scores[:, :63], 20)), (ValueError, lambda: c.evict(seqs[:2], scores, 20)),
                      (ValueError, lambda: c.evict(seqs, scores, -1)), (ValueError, lambda: c.evict([0, 0, 1], scores, 20)),
                      (ValueError, lambda: c.evict([0, 1, 9], scores, 20)), (RuntimeError, lambda: c.evict(seqs, scores, 48))):
        with pytest.raises(err):
            call()
    assert [list(c._book.pages[s]) for s in seqs] == before and c.num_free_pages == 2 and not moved
    c.evict(seqs, scores, 32)                              # two pages each: the first alone, then the others
    assert len(moved) == 2 and [c.get_seq_length(s) for s in seqs] == [32, 32, 32] and c.num_free_pages == 8
    c.evict(seqs, scores, 0)
    assert c.num_free_pages == 14
    fail = lambda *a: (_ for _ in ()).throw(RuntimeError("launch"))  # noqa: E731
    c._book.extend(seqs, lens)
    before, free = [list(c._book.pages[s]) for s in seqs], c.num_free_pages
    monkeypatch.setattr(pp, "compact_pages", fail)
    with pytest.raises(RuntimeError, match="launch"):
        c.evict(seqs, scores, 16)
    assert [list(c._book.pages[s]) for s in seqs] == before and c.num_free_pages == free and [c.get_seq_length(s) for s in seqs] == lens


def test_eviction_needs_a_budget_of_free_pages(monkeypatch):
    """What stays moves to fresh pages: with none, or one too few, it raises and nothing changes; with as many as one
    sequence's budget takes, all sequences move in turns."""
    lens = [64, 48, 64]                                       # 4 + 3 + 4 pages
    for free in range(4):
        pp, c, seqs, moved = _cache(monkeypatch, lens, pages=11 + free)
        monkeypatch.setattr(pp, "evict_select", lambda s, n, b, f, l: (torch.arange(b, dtype=torch.int32).expand(3, b), None, s))
        before = [list(c._book.pages[s]) for s in seqs]
        if free < 3:
            with pytest.raises(RuntimeError, match="exhausted"):
                c.evict(seqs, torch.zeros(3, 64), 40)         # 3 pages
            assert [list(c._book.pages[s]) for s in seqs] == before and c.num_free_pages == free and not moved
        else:
            c.evict(seqs, torch.zeros(3, 64), 40)
            assert len(moved) == 3 and [c.get_seq_length(s) for s in seqs] == [40, 40, 40] and c.num_free_pages == 14 - 9
