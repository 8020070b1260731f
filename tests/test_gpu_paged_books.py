"""The paged caches' books beside work that is still queued: nothing but `compact` waits for the device."""
import pytest
import torch

from gpu_util import announce

pytestmark = pytest.mark.gpu


def _cache(kind, lens, pages):
    """A cache of random tokens, some of its sequences on pages that another shares."""
    import akv
    g = torch.Generator(device="cuda").manual_seed(3)
    r = lambda *n: torch.randn(*n, generator=g, device="cuda").half()  # noqa: E731
    T = sum(lens)
    if kind == "latent":
        cache = akv.PagedLatentCache(2, 256, 64, page_size=16, max_pages=pages)
        rows = [(r(T, 256), r(T, 64)) for _ in range(2)]
    else:
        cache = akv.PackedPagedCache(2, 2, 64, page_size=16, max_pages=pages)
        rows = [(r(T, 2, 64), r(T, 2, 64)) for _ in range(2)]
    seqs = [cache.add_sequence() for _ in lens]
    batch = cache.extend(seqs, lens)
    for layer in range(2):
        cache.append(layer, *rows[layer], batch)
    return cache, seqs, torch.rand(len(lens), max(lens), generator=g, device="cuda")


def _held(cache, s):
    read = cache.get_rows if hasattr(cache, "get_rows") else cache.get_kv
    return [x.clone() for layer in range(2) for x in read(layer, s)]


@pytest.mark.parametrize("kind", ["latent", "4-bit"])
@pytest.mark.parametrize("lens,pages,budget", [([90, 20, 70], 24, 33), ([64, 64, 60], 14, 32)])  # in one go, and in turns
def test_eviction_and_steps_do_not_wait(kind, lens, pages, budget):
    announce(f"{kind} cache, eviction behind queued work, {pages} pages")
    want, got = _cache(kind, lens, pages), _cache(kind, lens, pages)
    kept = want[0].evict(want[1], want[2], budget)
    want[0].extend(want[1], 1)
    torch.cuda.synchronize()
    torch.cuda._sleep(50_000_000)
    queued = torch.cuda.Event()
    queued.record()
    out = got[0].evict(got[1], got[2], budget)
    batch = got[0].extend(got[1], 1)
    waited = queued.query()
    torch.cuda.synchronize()
    assert not waited, "the host waited for the work queued before"
    assert torch.equal(out, kept) and batch.kv_lens.tolist() == [min(n, budget) + 1 for n in lens]
    for a, b in zip(got[1], want[1]):
        got[0].crop(a, -1), want[0].crop(b, -1)
        assert all(torch.equal(x, y) for x, y in zip(_held(got[0], a), _held(want[0], b)))


def test_many_uploads_behind_queued_work():
    """Lists that are uploaded one after the other before the first copy runs keep their values."""
    announce("uploads behind queued work")
    cache, _, _ = _cache("latent", [5], 8)
    torch.cuda._sleep(50_000_000)
    up = [cache._upload([i] * (1 + i % 7), list(range(i))) for i in range(300)]
    for i, (a, b) in enumerate(up):
        assert a.tolist() == [i] * (1 + i % 7) and b.tolist() == list(range(i))
    assert [x.shape[0] for x in cache._upload([], [])] == [0, 0]


def test_books_are_not_captured():
    """A captured upload would repeat what the books said then; the cache is as it was."""
    announce("books under capture")
    cache, seqs, scores = _cache("latent", [40, 20], 12)
    before = [_held(cache, s) for s in seqs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        keep = scores + 1
        for call in (lambda: cache.extend(seqs, 1), lambda: cache.evict(seqs, scores, 10)):
            with pytest.raises(RuntimeError, match="captured"):
                call()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(keep, scores + 1)
    assert [cache.get_seq_length(s) for s in seqs] == [40, 20] and cache.num_free_pages == 12 - 5
    for s, b in zip(seqs, before):
        assert all(torch.equal(x, y) for x, y in zip(_held(cache, s), b))
