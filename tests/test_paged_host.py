"""The paged 4-bit cache's books and refusals, on the host."""
import ctypes
import random

import numpy as np
import pytest
import torch

import paged_ref as ref


@pytest.mark.parametrize("D,G", [(128, 32), (128, 64), (128, 128), (64, 32), (64, 64)])
def test_every_byte_of_a_tile_has_one_use(D, G):
    seen = np.zeros((ref.tile_bytes(D, G), 2), int)
    for at, sh, sa, za in ref.places(D, G):
        np.add.at(seen, (at.ravel(), sh.ravel() // 4), 1)
        for x in (sa, sa + 1, za, za + 1):
            np.add.at(seen, (x.ravel(), 0), 1)
            np.add.at(seen, (x.ravel(), 1), 1)
    assert (seen == 1).all()


def _whole(book):
    """Every page is free once or held by exactly as many sequences as it counts."""
    held = {}
    for pages in book.pages.values():
        for p in pages:
            held[p] = held.get(p, 0) + 1
    assert len(set(book.free)) == len(book.free) and not set(book.free) & set(held)
    assert len(book.free) + len(held) == len(book.refs)
    assert all(book.refs[p] == held.get(p, 0) for p in range(len(book.refs)))
    for s, pages in book.pages.items():
        assert len(pages) == -(-book.lens[s] // book.page_size)


def test_ledger_copy_on_write():
    from akv.paged_packed import PageLedger
    book = PageLedger(10, 16)
    a = book.add()
    assert book.extend([a], [20]) == []
    b, c = book.fork(a), book.fork(a)
    last = book.pages[a][1]
    copies = book.extend([a, b, c], [1, 1, 0])
    # a and b get pages of their own; c, which does not write, keeps the old one
    assert [x for x, _ in copies] == [last, last] and book.pages[c][1] == last
    assert len({book.pages[s][1] for s in (a, b, c)}) == 3 and len({book.pages[s][0] for s in (a, b, c)}) == 1
    assert book.extend([c], [1]) == []       # alone on it now
    _whole(book)
    d = book.fork(a)
    book.crop(d, 16)                          # at a page's end: nothing shared is written
    assert book.extend([d], [1]) == []
    e = book.fork(d)
    assert [x for x, _ in book.extend([d, e], [1, 1])] == [book.pages[e][1]]  # the second one writes in place
    _whole(book)


def test_ledger_refuses_whole():
    from akv.paged_packed import PageLedger
    book = PageLedger(4, 16)
    a, b = book.add(), book.add()
    book.extend([a, b], [17, 1])
    before = (list(book.free), dict(book.lens), [list(p) for p in book.pages.values()])
    for seqs, n, err in (([a, b], [16, 32], RuntimeError), ([a, a], [1, 1], ValueError), ([9], [1], ValueError),
                         ([a], [-1], ValueError), ([a, b], [1], ValueError)):
        with pytest.raises(err):
            book.extend(seqs, n)
    with pytest.raises(ValueError):
        book.plan_compaction([a], [18])
    c = book.fork(a)
    book.extend([b], [15])
    with pytest.raises(RuntimeError):
        book.plan_compaction([a], [17])      # one free page, and the old ones are shared
    book.remove(c)
    book.crop(b, 1)
    assert before == (list(book.free), dict(book.lens), [list(p) for p in book.pages.values()])
    _whole(book)


def test_ledger_undoes_what_was_not_launched():
    """An extend or a replacement that is undone leaves pages, counts and lengths as they were."""
    from akv.paged_packed import PageLedger
    book = PageLedger(20, 16)
    a = book.add()
    book.extend([a], [40])
    b, c = book.fork(a), book.add()
    book.extend([c], [16])
    state = lambda: ({s: list(p) for s, p in book.pages.items()}, dict(book.lens), list(book.refs), sorted(book.free))  # noqa: E731
    before = state()
    for counts in ([1, 1, 1], [30, 0, 5], [0, 9, 0], [0, 0, 0], [8, 8, 100]):
        copies = book.extend([b, a, c], counts)
        assert len(copies) == (1 if counts[0] or counts[1] else 0)
        book.undo_extend([b, a, c], counts, copies)
        assert state() == before
        _whole(book)
    for s, n in ((a, 3), (b, 40), (c, 0)):
        length = book.lens[s]
        old, _ = book.replace(s, n)
        book.undo_replace(s, old, length)
        assert state() == before
        _whole(book)



def test_ledger_at_random():
    from akv.paged_packed import PageLedger
    rng = random.Random(3)
    book = PageLedger(60, 16)
    for _ in range(3000):
        live = list(book.pages)
        op = rng.choice(["add", "fork", "extend", "extend", "crop", "remove", "compact"])
        if op == "add" or not live:
            book.add()
        elif op == "fork":
            book.fork(rng.choice(live))
        elif op == "remove" and len(live) > 6:
            book.remove(rng.choice(live))
        elif op == "crop":
            s = rng.choice(live)
            n = rng.randint(-50, 80)
            want = max(0, min(n if n >= 0 else n + book.lens[s], book.lens[s]))
            book.crop(s, n)
            assert book.lens[s] == want
        else:
            some = rng.sample(live, rng.randint(1, min(4, len(live))))
            try:
                if op == "extend":
                    n = [rng.randint(0, 40) for _ in some]
                    old = [book.lens[s] for s in some]
                    copies = book.extend(some, n)
                    assert len({b for _, b in copies}) == len(copies) and not {a for a, _ in copies} & {b for _, b in copies}
                    assert [book.lens[s] for s in some] == [a + b for a, b in zip(old, n)]
                    for s, o, c in zip(some, old, n):
                        assert all(book.refs[p] == 1 for p in book.pages[s][o // 16:]) or c == 0
                else:
                    n = [rng.randint(0, book.lens[s]) for s in some]
                    groups = book.plan_compaction(some, n)
                    assert sorted(i for g in groups for i in g) == list(range(len(some)))
                    for g in groups:
                        moved = [book.replace(some[i], n[i]) for i in g]
                        assert not {p for a, _ in moved for p in a} & {p for _, b in moved for p in b}
                        for a, _ in moved:
                            book._drop(a)
            except RuntimeError:
                pass
        _whole(book)


# ------------------------------------------------------------------ refusals


def _pool(nat, **kw):
    d = dict(data=4096, n_pages=4, num_layers=2, heads=2, D=128, page_size=16, group_size=32)
    d.update(kw)
    return nat.PagedPool(**d)


def _batch(nat, **kw):
    d = dict(page_table=4096, kv_lens=4096, q_starts=4096, table_stride=4, n_tokens=3, n_seqs=2, table_width=4, max_q=2)
    d.update(kw)
    return nat.PagedBatch(**d)


POOLS = [(dict(D=96), "E_UNSUPPORTED"), (dict(group_size=16), "E_UNSUPPORTED"), (dict(D=64, group_size=128), "E_UNSUPPORTED"),
         (dict(page_size=8), "E_UNSUPPORTED"), (dict(page_size=48), "E_UNSUPPORTED"), (dict(page_size=512), "E_UNSUPPORTED"),
         (dict(heads=0), "E_SHAPE"), (dict(num_layers=0), "E_SHAPE"), (dict(n_pages=-1), "E_SHAPE"),
         (dict(data=0), "E_INVALID"), (dict(data=8), "E_ALIGN")]
BATCHES = [(dict(n_seqs=-1), "E_SHAPE"), (dict(n_seqs=65536), "E_SHAPE"), (dict(table_stride=3), "E_SHAPE"),
           (dict(table_width=-1), "E_SHAPE"), (dict(n_tokens=-1), "E_SHAPE"), (dict(max_q=-1), "E_SHAPE"),
           (dict(table_width=2 ** 27, table_stride=2 ** 27), "E_SHAPE"), (dict(kv_lens=0), "E_INVALID"),
           (dict(q_starts=0), "E_INVALID"), (dict(page_table=0), "E_INVALID"), (dict(kv_lens=4098), "E_ALIGN")]


@pytest.mark.parametrize("call", ["rows", "attn", "importance"])
def test_c_refusals(call):
    from akv import _native as nat
    lib = nat.load()

    def run(pool=None, batch=None, **kw):
        common = dict(abi_version=nat.ABI_VERSION, layer=0, pool=_pool(nat, **(pool or {})), batch=_batch(nat, **(batch or {})))
        if call == "rows":
            a = nat.PagedRowsArgs(**{**common, "dtype": 0, "k": 4096, "v": 4096, "k_t": 512, "k_h": 256, "v_t": 512, "v_h": 256, **kw})
            return lib.akv_paged_append(ctypes.byref(a), None), lib.akv_paged_read(ctypes.byref(a), None)
        q = dict(Hq=4, q_dtype=0, causal=1, sm_scale=0.1, q=4096, q_t=1024, q_h=256, out=4096, lse=4096)
        if call == "attn":
            a = nat.PagedAttnArgs(**{**common, **q, "workspace": 4096, "workspace_bytes": 64, **kw})
            rc = lib.akv_paged_attn(ctypes.byref(a), None)
            if rc in (nat.AKV_E_SHAPE, nat.AKV_E_DTYPE, nat.AKV_E_UNSUPPORTED, nat.AKV_E_ABI):
                assert lib.akv_paged_attn_workspace_bytes(ctypes.byref(a)) == -1
            return (rc,)
        a = nat.PagedImportanceArgs(**{**common, **q, "q_window": 0, "decay": 0.9, "scores": 4096, "n_scores": 10,
                                       "score_stride": 10, "out_stride": 10, **kw})
        return (lib.akv_paged_importance(ctypes.byref(a), None),)

    code = lambda name: getattr(nat, "AKV_" + name)  # noqa: E731
    for kw, want in POOLS:
        assert set(run(pool=kw)) == {code(want)}, (kw, lib.akv_last_error())
    for kw, want in BATCHES:
        assert set(run(batch=kw)) == {code(want)}, (kw, lib.akv_last_error())
    own = [(dict(abi_version=4), "E_ABI"), (dict(layer=2), "E_SHAPE"), (dict(layer=-1), "E_SHAPE")]
    if call == "rows":
        own += [(dict(dtype=3), "E_DTYPE"), (dict(k=0), "E_INVALID"), (dict(v=4100), "E_ALIGN"), (dict(k_t=520), "E_ALIGN")]
    else:
        own += [(dict(q_dtype=2), "E_DTYPE"), (dict(Hq=3), "E_SHAPE"), (dict(Hq=0), "E_SHAPE"), (dict(sm_scale=0.0), "E_INVALID"),
                (dict(sm_scale=float("nan")), "E_INVALID"), (dict(sm_scale=float("inf")), "E_INVALID"), (dict(q=0), "E_INVALID"),
                (dict(q=4100), "E_ALIGN"), (dict(q_h=260), "E_ALIGN"), (dict(out=0), "E_INVALID"), (dict(lse=4097), "E_ALIGN")]
    if call == "attn":
        own += [(dict(workspace=0), "E_WORKSPACE"), (dict(workspace_bytes=63), "E_WORKSPACE"), (dict(out=4100), "E_ALIGN")]
    if call == "importance":
        own += [(dict(q_window=-1), "E_SHAPE"), (dict(score_stride=9), "E_SHAPE"), (dict(n_scores=-1), "E_SHAPE"),
                (dict(lse=0), "E_INVALID"), (dict(scores=0), "E_INVALID"), (dict(out=4098), "E_ALIGN")]
    for kw, want in own:
        assert set(run(**kw)) == {code(want)}, (kw, lib.akv_last_error())


def test_c_refusals_of_moves():
    from akv import _native as nat
    lib = nat.load()
    for kw, want in POOLS:
        p = _pool(nat, **kw)
        assert lib.akv_paged_copy(ctypes.byref(p), 4096, 4096, 1, None) == getattr(nat, "AKV_" + want), kw
    p = _pool(nat)
    assert lib.akv_paged_copy(None, None, None, 0, None) == nat.AKV_E_INVALID
    for n, a, b, want in ((5, 4096, 4096, nat.AKV_E_SHAPE), (-1, 4096, 4096, nat.AKV_E_SHAPE), (1, None, 4096, nat.AKV_E_INVALID),
                          (1, 4096, 4098, nat.AKV_E_ALIGN), (0, None, None, nat.AKV_OK)):
        assert lib.akv_paged_copy(ctypes.byref(p), a, b, n, None) == want
    base = dict(abi_version=nat.ABI_VERSION, n_seqs=2, pool=p, src_table=4096, dst_table=4096, src_stride=4, dst_stride=4,
                src_width=4, dst_width=4, keep=4096, n_keep=4096, keep_stride=9, max_keep=9)
    for kw, want in ((dict(abi_version=3), nat.AKV_E_ABI), (dict(n_seqs=-1), nat.AKV_E_SHAPE), (dict(src_stride=3), nat.AKV_E_SHAPE),
                     (dict(keep_stride=8), nat.AKV_E_SHAPE), (dict(dst_width=2 ** 27, dst_stride=2 ** 27), nat.AKV_E_SHAPE),
                     (dict(keep=0), nat.AKV_E_INVALID), (dict(n_keep=0), nat.AKV_E_INVALID), (dict(src_table=0), nat.AKV_E_INVALID),
                     (dict(dst_table=4097), nat.AKV_E_ALIGN)):
        a = nat.PagedCompactArgs(**{**base, **kw})
        assert lib.akv_paged_compact(ctypes.byref(a), None) == want, kw
    assert lib.akv_paged_compact(None, None) == nat.AKV_E_INVALID


def test_host_tensors_are_refused():
    import akv
    with pytest.raises(RuntimeError, match="CPU"):
        akv.PagedPool.empty(1, 4, 2, 128, device="cpu")
    with pytest.raises(RuntimeError, match="CPU"):
        akv.PagedBatch(torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), 0, 0)
    with pytest.raises(RuntimeError):
        akv.PackedPagedCache(1, 2, 128, device="cpu")
    with pytest.raises(ValueError):
        akv.PagedPool(torch.zeros(1, 2, 3, 4, 5, dtype=torch.uint8), 128)
    with pytest.raises(NotImplementedError):
        akv.PagedPool.empty(1, 4, 2, 128, page_size=40)


def test_strides_of_single_rows_say_nothing():
    """One token, or one head, of a tensor whose rows are padded: what stride its size-1 dimensions
    have does not matter, whether the rows are copied or not."""
    from akv.paged_packed import _rows
    buf = torch.randn(5, 1028)
    for T, H, x in ((1, 8, buf[:, :1024].unflatten(1, (8, 128))[2:3]), (3, 8, buf[:, :1024].unflatten(1, (8, 128))[1:4]),
                    (5, 1, buf[:, :128].unflatten(1, (1, 128))), (1, 1, buf[3:4, 4:132].unflatten(1, (1, 128))),
                    (1, 1, buf[3:4, 1:129].unflatten(1, (1, 128))), (0, 8, buf[:0, :1024].unflatten(1, (8, 128))),
                    (1, 2, buf.t()[:256, 2:3].t().unflatten(1, (2, 128)))):
        for dt in (torch.float16, torch.float32):
            y = torch.empty_strided(x.shape, x.stride(), dtype=dt).copy_(x)
            z, st, sh = _rows(y, "x", T, H, 128)
            e = z.element_size()
            assert st % 16 == 0 and sh % 16 == 0 and z.data_ptr() % 16 == 0
            got = torch.as_strided(z, (T, H, 128), (st // e, sh // e, 1))
            assert torch.equal(got, y)


def test_entries_past_32_bits_stay_out_of_range():
    """64-bit tables and lists: what does not fit 32 bits must not come out as a page or position that is there."""
    from akv.paged_packed import _int32
    t = torch.tensor([3, -1, 2 ** 32 + 1, -2 ** 33, 2 ** 31, 2 ** 62])
    got = _int32("keep", t, 1)
    assert got.dtype == torch.int32 and got.tolist() == [3, -1, 2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1, 2 ** 31 - 1]
    assert _int32("table", t.view(2, 3), 2).tolist() == [[3, -1, 2 ** 31 - 1], [-2 ** 31, 2 ** 31 - 1, 2 ** 31 - 1]]


@pytest.mark.parametrize("scores,out,n,ss,so,S,clash", [
    (0, 0, 10, 10, 10, 3, False), (0, 30, 10, 10, 10, 3, False), (30, 0, 10, 10, 10, 3, False),
    (0, 10, 10, 20, 20, 3, False), (10, 0, 10, 20, 20, 3, False),                                # columns of one buffer
    (0, 1, 10, 20, 20, 3, True), (9, 0, 10, 20, 20, 3, True), (0, 11, 10, 20, 20, 3, True),      # shifted
    (0, 10, 10, 10, 10, 3, True), (0, 20, 10, 20, 20, 3, True), (0, 60, 10, 20, 20, 3, False),   # rows on
    (0, 0, 10, 10, 12, 3, True), (0, 0, 10, 10, 12, 1, False),                                   # one row: strides say nothing
    (0, 5, 10, 10, 10, 1, True), (5, 0, 10, 10, 10, 1, True), (0, 10, 10, 1, 1, 1, False),
])
def test_importance_refuses_scores_that_overlap_its_output(scores, out, n, ss, so, S, clash):
    """out may be scores or lie apart from it, also as columns of one buffer; other views are refused.
    (lse off its alignment is refused behind that: no call here is launched.)"""
    from akv import _native as nat
    lib = nat.load()
    at = 1 << 20
    a = nat.PagedImportanceArgs(abi_version=nat.ABI_VERSION, layer=0, pool=_pool(nat), batch=_batch(nat, n_seqs=S), Hq=4, q_dtype=0,
                                causal=1, sm_scale=0.1, q=4096, q_t=1024, q_h=256, q_window=0, decay=0.9, lse=4097,
                                scores=at + 4 * scores, out=at + 4 * out, n_scores=n, score_stride=ss, out_stride=so)
    assert lib.akv_paged_importance(ctypes.byref(a), None) == (nat.AKV_E_SHAPE if clash else nat.AKV_E_ALIGN), lib.akv_last_error()
