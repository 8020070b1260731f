"""A KV cache of many sequences in 4-bit pages, and the operators that fill, read, score and
rearrange it.

``PagedPool`` is the store: pages of ``page_size`` token slots, each slot the 4-bit codes of a
token's keys and values with one float16 (scale, zero) per ``group_size`` channels.
``PagedBatch`` says which sequences a call is about: their page tables, lengths and the rows
of the call's tensors that are theirs.  Lengths and tables live on the device and are read
when the work runs, so a call captured into a graph follows what is in them at each replay.

  paged_append      new tokens quantized into their slots
  paged_read        the values of those tokens as the cache holds them
  paged_attention   attention of the call's queries over the cached tokens
  paged_importance  the running importance of the cached tokens
  copy_pages        pages duplicated in every layer
  compact_pages     sequences reduced to the tokens that stay, in every layer
  evict_select      which tokens stay, by the attention that they gathered

``PackedPagedCache`` keeps the books: page allocation, forks that share pages and copy them
when one side writes, compaction.  Everything runs in libakv_hip.so; there is no CPU path and
no gradient.  The tile layout is written out in include/akv_hip.h."""
from __future__ import annotations

import ctypes
import struct
from operator import index
from typing import List, Optional, Sequence, Tuple, Union

import torch

from . import _native as nat

_QUERY = (torch.float16, torch.bfloat16)
_stream, _current = torch._C._cuda_getCurrentRawStream, torch.cuda.current_device

# the args structs, packed in one call (a ctypes structure with its nested ones costs five times
# that, which a decode step's calls would feel)
_POOL, _BATCH = ctypes.sizeof(nat.PagedPool), ctypes.sizeof(nat.PagedBatch)
_ROWS = struct.Struct(f"@4i{_POOL}s{_BATCH}s6q")
_ATTN = struct.Struct(f"@5if{_POOL}s{_BATCH}s7q")
_IMPORTANCE = struct.Struct(f"@6i2f{_POOL}s{_BATCH}s9q")
_COMPACT = struct.Struct(f"@2i{_POOL}s4q2i4q")
_EVICT = struct.Struct("@2i6q2i6q")
for _s, _c in ((_ROWS, nat.PagedRowsArgs), (_ATTN, nat.PagedAttnArgs), (_IMPORTANCE, nat.PagedImportanceArgs),
               (_COMPACT, nat.PagedCompactArgs), (_EVICT, nat.EvictArgs)):
    assert _s.size == ctypes.sizeof(_c), _c


def _call(index: int, what: str, fn, *args) -> None:
    """fn(*args, stream): on the current stream of the device, which is made the current one."""
    if index == _current():
        rc = fn(*args, _stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _stream(index))
    if rc:
        nat.check(rc, what)


def _check_device(pool: "PagedPool", *tensors) -> None:
    at = pool._index
    for t in tensors:
        if t.get_device() != at:
            nat.require_device(t)
            raise ValueError(f"a tensor on {t.device} beside a pool on {pool.data.device}")


def _int32(name: str, t: torch.Tensor, dims: int) -> torch.Tensor:
    """An int32 tensor of ``dims`` dimensions, its last one consecutive and its rows apart."""
    if t.dim() != dims or t.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{name} must be an int32 tensor of {dims} dimension{'s' if dims > 1 else ''}")
    if t.dtype != torch.int32:
        t = t.clamp(-2 ** 31, 2 ** 31 - 1).to(torch.int32)  # what is out of range stays so
    plain = t.numel() == 0 or (t.stride(-1) == 1 and (dims == 1 or t.shape[0] == 1 or t.stride(0) >= t.shape[1]))
    return t if plain else t.contiguous()


class PagedPool:
    """The pages: ``data`` (layers, pages, heads, page_size / 16, tile bytes) uint8.

    head_dim 64 or 128, group_size 32, 64 or 128 (at most head_dim), page_size a power of two
    from 16 to 256.  What free slots hold does not matter."""

    def __init__(self, data: torch.Tensor, head_dim: int, group_size: int = 32):
        tile = 16 * head_dim + 128 * (head_dim // group_size if group_size > 0 else 0)
        if data.dim() != 5 or data.dtype != torch.uint8 or data.shape[4] != tile:
            raise ValueError(f"a pool is a (layers, pages, heads, page_size / 16, {tile}) uint8 tensor, got "
                             f"{tuple(data.shape)} {data.dtype}")
        nat.require_device(data)
        if not data.is_contiguous() or data.data_ptr() % 16:
            raise ValueError("a pool must be contiguous and 16-byte aligned")
        self.data, self.head_dim, self.group_size = data, head_dim, group_size
        self.num_layers, self.num_pages, self.heads = data.shape[:3]
        self.page_size = 16 * data.shape[3]
        self._index = data.get_device()
        self._c = bytes(nat.PagedPool(data.data_ptr(), self.num_pages, self.num_layers, self.heads, head_dim,
                                      self.page_size, group_size, 0))
        lib = nat.load()
        self._copy, self._compact, self._compact_args = lib.akv_paged_copy, lib.akv_paged_compact, _COMPACT
        # every refusal of a pool's shape is the library's
        nat.check(self._copy(self._c, None, None, 0, None), "PagedPool")

    @classmethod
    def empty(cls, num_layers: int, num_pages: int, heads: int, head_dim: int, page_size: int = 16,
              group_size: int = 32, device="cuda") -> "PagedPool":
        if page_size < 16 or page_size % 16 or group_size < 1:
            raise NotImplementedError(f"page_size a power of two from 16 to 256, group_size 32, 64 or 128; got "
                                      f"{page_size}, {group_size}")
        tile = 16 * head_dim + 128 * (head_dim // group_size)
        data = torch.zeros(num_layers, num_pages, heads, page_size // 16, tile, dtype=torch.uint8, device=device)
        return cls(data, head_dim, group_size)

    def nbytes(self) -> int:
        return self.data.numel()


class PagedBatch:
    """The sequences of a call.

    page_table (S, W) int32: token j of sequence s lies in slot j % page_size of page
    ``page_table[s, j // page_size]``.  kv_lens (S,) int32: cached tokens, those of this call
    among them.  q_starts (S + 1,) int32: sequence s owns rows ``q_starts[s]`` to
    ``q_starts[s + 1]`` of the call's (n_tokens, heads, head_dim) tensors; they are its newest
    tokens.  n_tokens: the rows; max_q: no sequence has more of them.  Rows that are no sequence's
    (those of a padded batch) are read as 0; what the attention returns for them is not defined.

    The tensors are kept, not copied (other integer types and orders are): what they hold when
    the work runs counts.  n_tokens and max_q are fixed."""

    def __init__(self, page_table: torch.Tensor, kv_lens: torch.Tensor, q_starts: torch.Tensor, n_tokens: int, max_q: int):
        nat.require_device(page_table, kv_lens, q_starts)
        self.page_table = _int32("page_table", page_table, 2)
        self.kv_lens, self.q_starts = _int32("kv_lens", kv_lens, 1), _int32("q_starts", q_starts, 1)
        S, W = self.page_table.shape
        if self.kv_lens.shape[0] != S or self.q_starts.shape[0] != S + 1:
            raise ValueError(f"{S} sequences take {S} kv_lens and {S + 1} q_starts")
        if not 0 <= max_q <= n_tokens:
            raise ValueError("max_q lies between 0 and n_tokens")
        self.n_seqs, self.n_tokens, self.max_q = S, int(n_tokens), int(max_q)
        self._index = self.page_table.get_device()
        if self.kv_lens.get_device() != self._index or self.q_starts.get_device() != self._index:
            raise ValueError("a batch's tensors live on one device")
        self._c = bytes(nat.PagedBatch(self.page_table.data_ptr(), self.kv_lens.data_ptr(), self.q_starts.data_ptr(),
                                       self.page_table.stride(0), self.n_tokens, S, W, self.max_q, 0))
        self._workspace: dict = {}  # bytes an attention call needs, by the sizes they depend on


def _rows(x: torch.Tensor, name: str, T: int, H: int, D: int) -> Tuple[torch.Tensor, int, int]:
    """(T, H, D) with consecutive channels and rows on 16 bytes, copied if it is not, and the byte
    strides of tokens and heads (those of a dimension of size 1 say nothing, to contiguous() either)."""
    if x.shape != (T, H, D):
        raise ValueError(f"{name} must be ({T}, {H}, {D}), got {tuple(x.shape)}")
    e = x.element_size()
    st, sh, sc = x.stride()
    if T <= 1:
        st = H * D
    if H <= 1:
        sh = D
    if sc != 1 or (st * e | sh * e | x.data_ptr()) & 15:
        x, st, sh = nat.dev_contig(x), H * D, D
    return x, st * e, sh * e


def _rows_args(pool: PagedPool, batch: PagedBatch, k: tuple, v: tuple, layer: int) -> bytes:
    (k, kt, kh), (v, vt, vh) = k, v
    return _ROWS.pack(nat.ABI_VERSION, layer, nat.dtype_code(k.dtype), 0, pool._c, batch._c, k.data_ptr(), v.data_ptr(),
                      kt, kh, vt, vh)


def paged_append(pool: PagedPool, batch: PagedBatch, k: torch.Tensor, v: torch.Tensor, layer: int = 0) -> None:
    """Quantize k and v (n_tokens, heads, head_dim), float16, bfloat16 or float32 and strided
    as they come, into the slots of the batch's rows.

    Per token, head and group of channels: scale = (max - min) / 15 and zero = min, rounded to
    float16, and codes (x - zero) / scale rounded to the nearest, ties to even, all as in exact
    arithmetic.  Values past +-61440 are clamped; a group with a value that is not finite reads
    back as NaN."""
    T, H, D = batch.n_tokens, pool.heads, pool.head_dim
    _check_device(pool, k, v, batch.page_table)
    if k.dtype != v.dtype:
        raise TypeError(f"k is {k.dtype} and v {v.dtype}")
    k, v = _rows(k, "k", T, H, D), _rows(v, "v", T, H, D)
    _call(pool._index, "paged_append", nat.load().akv_paged_append, _rows_args(pool, batch, k, v, layer))


def paged_read(pool: PagedPool, batch: PagedBatch, layer: int = 0,
               dtype: torch.dtype = torch.float16) -> Tuple[torch.Tensor, torch.Tensor]:
    """Keys and values (n_tokens, heads, head_dim) of the batch's rows as the cache holds them."""
    _check_device(pool, batch.page_table)
    nat.dtype_code(dtype)
    k, v = torch.empty(2, batch.n_tokens, pool.heads, pool.head_dim, dtype=dtype, device=pool.data.device).unbind(0)
    sh = pool.head_dim * k.element_size()
    st = pool.heads * sh
    _call(pool._index, "paged_read", nat.load().akv_paged_read, _rows_args(pool, batch, (k, st, sh), (v, st, sh), layer))
    return k, v


def _queries(q: torch.Tensor, pool: PagedPool, batch: PagedBatch) -> Tuple[torch.Tensor, int, int]:
    _check_device(pool, q, batch.page_table)
    if q.dtype not in _QUERY:
        raise TypeError("paged attention takes float16 or bfloat16 queries")
    if q.dim() != 3:
        raise ValueError("q must be (n_tokens, heads, head_dim)")
    return _rows(q, "q", batch.n_tokens, q.shape[1], pool.head_dim)


def paged_attention(q: torch.Tensor, pool: PagedPool, batch: PagedBatch, layer: int = 0, sm_scale: Optional[float] = None,
                    causal: bool = True, return_lse: bool = False):
    """Attention of q (n_tokens, Hq, head_dim), float16 or bfloat16, over the cached tokens.

    Query head h reads cached head h // (Hq // heads).  With ``causal``, row i of a sequence's
    m rows sees its first kv_len - m + 1 + i tokens, else all of them; a row that sees none is 0.
    ``return_lse`` adds log(sum(exp(sm_scale q.k))) (n_tokens, Hq) float32, -inf for such rows.

    Scores, sums and log-sums are float32.  For bfloat16 outputs the weights are rounded to float16
    (an eighth of the output's own half step), and so are the values in chunks of more than 64 rows a
    cached head, for float16 outputs too."""
    q, qt, qh = _queries(q, pool, batch)
    T, Hq, D = q.shape
    lib = nat.load()
    out = torch.empty(T, Hq, D, dtype=q.dtype, device=q.device)
    lse = torch.empty(T, Hq, dtype=torch.float32, device=q.device) if return_lse else None
    head = (nat.ABI_VERSION, layer, Hq, nat.dtype_code(q.dtype), int(causal),
            nat.default_sm_scale(D) if sm_scale is None else float(sm_scale), pool._c, batch._c, q.data_ptr(), qt, qh,
            out.data_ptr(), 0 if lse is None else lse.data_ptr())
    key = (D, pool.group_size, pool.heads, pool.page_size, Hq)
    need = batch._workspace.get(key)
    if need is None:
        need = lib.akv_paged_attn_workspace_bytes(_ATTN.pack(*head, 0, 0))
        if need >= 0:
            batch._workspace[key] = need
    ws = torch.empty(need, dtype=torch.uint8, device=q.device) if need > 0 else None
    _call(pool._index, "paged_attention", lib.akv_paged_attn,
          _ATTN.pack(*head, 0, 0) if ws is None else _ATTN.pack(*head, ws.data_ptr(), need))
    return out if lse is None else (out, lse)


def paged_importance(q: torch.Tensor, lse: torch.Tensor, pool: PagedPool, batch: PagedBatch, scores: torch.Tensor,
                     layer: int = 0, decay: float = 0.9, q_window: int = 0, sm_scale: Optional[float] = None,
                     causal: bool = True, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The running importance of the cached tokens: scores (S, N) float32 become
    ``scores * decay + sum over rows of the mean over heads of the attention weights`` for the
    tokens of every sequence that has rows in the batch (its first N, where it has more).

    q and lse are those of ``paged_attention``; ``q_window`` > 0 counts a sequence's last rows
    only.  Written in place, or to ``out``, which does not overlap scores; returns what was written."""
    q, qt, qh = _queries(q, pool, batch)
    T, Hq, D = q.shape
    dst = scores if out is None else out
    _check_device(pool, lse, scores, dst)
    if lse.dtype != torch.float32 or lse.shape != (T, Hq):
        raise ValueError(f"lse must be ({T}, {Hq}) float32")
    for t in (scores, dst):
        if t.dtype != torch.float32 or t.dim() != 2 or t.shape[0] != batch.n_seqs or t.shape != scores.shape:
            raise ValueError(f"scores must be ({batch.n_seqs}, tokens) float32")
        if t.shape[1] > 1 and t.stride(1) != 1:
            raise ValueError("a sequence's scores must be consecutive")
    if not lse.is_contiguous():
        lse = lse.contiguous()
    args = _IMPORTANCE.pack(nat.ABI_VERSION, layer, Hq, nat.dtype_code(q.dtype), int(causal), int(q_window),
                            nat.default_sm_scale(D) if sm_scale is None else float(sm_scale), float(decay), pool._c,
                            batch._c, q.data_ptr(), qt, qh, lse.data_ptr(), scores.data_ptr(), dst.data_ptr(),
                            scores.shape[1], scores.stride(0), dst.stride(0))
    _call(pool._index, "paged_importance", nat.load().akv_paged_importance, args)
    return dst


def copy_pages(pool, src: torch.Tensor, dst: torch.Tensor) -> None:
    """Page dst[i] of every layer becomes a copy of page src[i].  ``pool`` is a PagedPool or a
    PagedLatentPool; int32 tensors on its device; no page may be written twice, or both read and written."""
    _check_device(pool, src, dst)
    src, dst = _int32("src", src, 1), _int32("dst", dst, 1)
    if src.shape != dst.shape:
        raise ValueError("src and dst must be of one length")
    _call(pool._index, "copy_pages", pool._copy, pool._c, src.data_ptr(), dst.data_ptr(), src.shape[0])


def compact_pages(pool, src_table: torch.Tensor, dst_table: torch.Tensor, keep: torch.Tensor,
                  n_keep: torch.Tensor) -> None:
    """Token j of sequence s on ``dst_table`` (S, W') becomes token ``keep[s, j]`` on
    ``src_table`` (S, W), j < n_keep[s], in every layer of a PagedPool or a PagedLatentPool.

    keep (S, K) and n_keep (S,) int32.  No slot that is read may be written, except tokens that
    stay where they are.  Slots behind the last token keep what they hold."""
    _check_device(pool, src_table, dst_table, keep, n_keep)
    src_table, dst_table = _int32("src_table", src_table, 2), _int32("dst_table", dst_table, 2)
    keep, n_keep = _int32("keep", keep, 2), _int32("n_keep", n_keep, 1)
    S = n_keep.shape[0]
    if src_table.shape[0] != S or dst_table.shape[0] != S or keep.shape[0] != S:
        raise ValueError(f"{S} sequences take {S} rows of src_table, dst_table and keep")
    args = pool._compact_args.pack(nat.ABI_VERSION, S, pool._c, src_table.data_ptr(), dst_table.data_ptr(), src_table.stride(0),
                         dst_table.stride(0), src_table.shape[1], dst_table.shape[1], keep.data_ptr(), n_keep.data_ptr(),
                         keep.stride(0), keep.shape[1])
    _call(pool._index, "compact_pages", pool._compact, args)


def evict_select(scores: torch.Tensor, lens: torch.Tensor, budget: Union[int, torch.Tensor], protect_initial: int = 4,
                 protect_recent: int = 16, max_keep: Optional[int] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Which tokens stay where each sequence is held to a budget, by the attention they gathered.

    scores (S, N) float32, a sequence's consecutive: accumulated weights, as ``paged_importance`` and
    ``latent_importance`` keep them; lens (S,) int32, at most N.  ``budget`` is a number of tokens, or (S,) int32 on the
    device with ``max_keep`` the most it may say (N where that is not given).  The first ``protect_initial`` and
    last ``protect_recent`` tokens stay before all others (where the budget does not hold those, the later ones), then those of the
    highest score, NaN above all; of equal ones the lowest position leaves first.

    Returns keep (S, K) int32, ascending positions, n_keep (S,) int32, as ``compact_pages`` takes them, and
    the scores of the tokens that stay at their new positions, (S, N) float32; all three are 0 behind the last."""
    nat.require_device(scores, lens)
    if scores.dtype != torch.float32 or scores.dim() != 2:
        raise ValueError("scores must be a (sequences, tokens) float32 tensor")
    S, N = scores.shape
    dev = scores.get_device()
    lens = _int32("lens", lens, 1)
    each = isinstance(budget, torch.Tensor)
    if each:
        nat.require_device(budget)
        budget = _int32("budget", budget, 1)
    K = min(N, N if max_keep is None else index(max_keep)) if each else min(N, index(budget), N if max_keep is None else index(max_keep))
    for name, t in (("lens", lens),) + ((("budget", budget),) if each else ()):
        if t.shape[0] != S:
            raise ValueError(f"{S} sequences take {S} entries of {name}")
        if t.get_device() != dev:
            raise ValueError(f"{name} on {t.device} beside scores on {scores.device}")
    if K < 0:
        raise ValueError("a budget must be at least 0")
    if N > 1 and scores.stride(1) != 1 or (S > 1 and scores.stride(0) < N):
        scores = scores.contiguous()
    out = torch.empty(S * (K + 1 + N), dtype=torch.int32, device=scores.device)
    keep, n_keep, kept = out.split([S * K, S, S * N])
    kept = kept.view(torch.float32)
    args = _EVICT.pack(nat.ABI_VERSION, S, scores.data_ptr(), N, scores.stride(0), lens.data_ptr(),
                       budget.data_ptr() if each else 0, 0 if each else min(index(budget), N), index(protect_initial), index(protect_recent),
                       keep.data_ptr(), n_keep.data_ptr(), kept.data_ptr(), K, K, N)
    _call(dev, "evict_select", nat.load().akv_evict_select, args)
    return keep.view(S, K), n_keep, kept.view(S, N)


class PageLedger:
    """Which sequence holds which pages (host only).  A page may belong to several sequences
    after a fork; it is written only while it belongs to one."""

    def __init__(self, num_pages: int, page_size: int):
        self.page_size = page_size
        self.free: List[int] = list(range(num_pages))  # taken from the end
        self.refs = [0] * num_pages
        self.pages: dict = {}
        self.lens: dict = {}
        self._next = 0

    def _take(self) -> int:
        page = self.free.pop()
        self.refs[page] = 1
        return page

    def _drop(self, pages) -> None:
        for page in pages:
            self.refs[page] -= 1
            if self.refs[page] == 0:
                self.free.append(page)

    def _count(self, n: int) -> int:
        return -(-n // self.page_size)

    def _known(self, seqs) -> None:
        for s in seqs:
            if s not in self.pages:
                raise ValueError(f"no sequence {s}")
        if len(set(seqs)) != len(seqs):
            raise ValueError("a sequence is listed twice")

    def add(self) -> int:
        s, self._next = self._next, self._next + 1
        self.pages[s], self.lens[s] = [], 0
        return s

    def fork(self, seq: int) -> int:
        self._known([seq])
        s = self.add()
        self.pages[s], self.lens[s] = list(self.pages[seq]), self.lens[seq]
        for page in self.pages[s]:
            self.refs[page] += 1
        return s

    def remove(self, seq: int) -> None:
        self._known([seq])
        self._drop(self.pages.pop(seq))
        del self.lens[seq]

    def crop(self, seq: int, length: int) -> None:
        self._known([seq])
        if length < 0:
            length += self.lens[seq]
        length = max(0, min(length, self.lens[seq]))
        n = self._count(length)
        self._drop(self.pages[seq][n:])
        del self.pages[seq][n:]
        self.lens[seq] = length

    def extend(self, seqs: Sequence[int], counts: Sequence[int]) -> List[Tuple[int, int]]:
        """Slots for ``counts`` more tokens; (from, to) of the shared pages that get written and
        have to be copied first.  Raises, and changes nothing, when the pages do not suffice."""
        self._known(seqs)
        counts = [index(c) for c in counts]
        if len(counts) != len(seqs) or any(c < 0 for c in counts):
            raise ValueError("one count of new tokens, at least 0, for each sequence")
        need, left = 0, {}
        for s, c in zip(seqs, counts):
            n = self.lens[s]
            need += self._count(n + c) - len(self.pages[s])
            if c and n % self.page_size:
                last = self.pages[s][-1]
                left.setdefault(last, self.refs[last])
                if left[last] > 1:
                    left[last] -= 1
                    need += 1
        if need > len(self.free):
            raise RuntimeError("Page pool exhausted")
        copies = []
        for s, c in zip(seqs, counts):
            n, pages = self.lens[s], self.pages[s]
            if c and n % self.page_size and self.refs[pages[-1]] > 1:
                old, pages[-1] = pages[-1], self._take()
                self.refs[old] -= 1
                copies.append((old, pages[-1]))
            while len(pages) < self._count(n + c):
                pages.append(self._take())
            self.lens[s] = n + c
        return copies

    def undo_extend(self, seqs: Sequence[int], counts: Sequence[int], copies: Sequence[Tuple[int, int]]) -> None:
        """Back to before an ``extend`` whose work could not be launched."""
        for s, c in zip(seqs, counts):
            self.crop(s, self.lens[s] - c)
        back = {new: old for old, new in copies}
        for s in seqs:
            pages = self.pages[s]
            if pages and pages[-1] in back:
                new, pages[-1] = pages[-1], back[pages[-1]]
                self.refs[pages[-1]] += 1
                self._drop([new])

    def plan_compaction(self, seqs: Sequence[int], counts: Sequence[int]) -> List[List[int]]:
        """Indices of ``seqs`` in groups whose new pages are free at their turn (each group's
        old pages are given back before the next).  Raises when one does not fit."""
        self._known(seqs)
        if len(counts) != len(seqs) or any(not 0 <= c <= self.lens[s] for s, c in zip(seqs, counts)):
            raise ValueError("one count of tokens that stay, at most its length, for each sequence")
        free, refs, groups, at, back = len(self.free), {}, [], [], []
        for i, (s, c) in enumerate(zip(seqs, counts)):
            need = self._count(c)
            if need > free and at:
                for page in back:
                    refs[page] = refs.get(page, self.refs[page]) - 1
                    free += refs[page] == 0
                groups.append(at)
                at, back = [], []
            if need > free:
                raise RuntimeError("Page pool exhausted")
            free -= need
            at.append(i)
            back += self.pages[s]
        return groups + [at] if at else groups

    def replace(self, seq: int, count: int) -> Tuple[List[int], List[int]]:
        """New pages for ``count`` tokens of a sequence; (old, new).  The old ones are still
        held: ``_drop`` them when what reads them has been launched."""
        old, new = self.pages[seq], [self._take() for _ in range(self._count(count))]
        self.pages[seq], self.lens[seq] = new, count
        return old, new

    def undo_replace(self, seq: int, old: List[int], length: int) -> None:
        self._drop(self.pages[seq])
        self.pages[seq], self.lens[seq] = old, length


class _PagedCache:
    """The books of sequences in a pool's pages: what ``PackedPagedCache`` and
    ``PagedLatentCache`` share."""

    def __init__(self, pool, max_pages: int):
        self.pool = pool
        self._book = PageLedger(max_pages, pool.page_size)

    # ---- sequences
    def add_sequence(self) -> int:
        return self._book.add()

    def fork(self, seq: int, n: int = 1) -> List[int]:
        """n sequences that share the tokens of ``seq``."""
        return [self._book.fork(seq) for _ in range(n)]

    def remove(self, seq: int) -> None:
        self._book.remove(seq)

    def crop(self, seq: int, length: int) -> None:
        """Drop the tokens at or past ``length``; a negative one counts back."""
        self._book.crop(seq, length)

    def get_seq_length(self, seq: int) -> int:
        self._book._known([seq])
        return self._book.lens[seq]

    @property
    def num_free_pages(self) -> int:
        return len(self._book.free)

    # ---- batches
    def _upload(self, *rows: List[int]) -> List[torch.Tensor]:
        """Lists of integers as int32 tensors on the device, with one copy that the host does not wait for: pinned
        memory, which torch's allocator holds until the copy has ended."""
        device = self.pool.data.device
        pinned = device.type == "cuda"
        if pinned and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("a cache's books cannot be captured: each replay would upload what they said at the capture")
        flat = torch.tensor([x for r in rows for x in r], dtype=torch.int32, pin_memory=pinned).to(device, non_blocking=True)
        return list(flat.split([len(r) for r in rows]))

    def _table(self, page_lists) -> Tuple[List[int], int]:
        width = max((len(p) for p in page_lists), default=0)
        return [x for p in page_lists for x in (*p, *([0] * (width - len(p))))], width

    def _batch(self, seqs: Sequence[int], counts: Sequence[int]) -> PagedBatch:
        table, width = self._table([self._book.pages[s] for s in seqs])
        starts = [0]
        for c in counts:
            starts.append(starts[-1] + c)
        t, lens, q = self._upload(table, [self._book.lens[s] for s in seqs], starts)
        return PagedBatch(t.view(len(seqs), width), lens, q, starts[-1], max(counts, default=0))

    def extend(self, seqs: Sequence[int], counts: Union[int, Sequence[int]] = 1) -> PagedBatch:
        """Room for ``counts`` new tokens of each sequence: the batch whose rows they are."""
        counts = [counts] * len(seqs) if isinstance(counts, int) else [index(c) for c in counts]
        copies = self._book.extend(seqs, counts)
        try:
            batch = self._batch(seqs, counts)
            if copies:
                copy_pages(self.pool, *self._upload([a for a, _ in copies], [b for _, b in copies]))
        except BaseException:
            self._book.undo_extend(seqs, counts, copies)
            raise
        return batch

    # ---- compaction
    def compact(self, seqs: Sequence[int], keep: Sequence[torch.Tensor]) -> None:
        """Sequence ``seqs[i]`` keeps the tokens at positions ``keep[i]`` (ascending integers on
        the device, below its length), in every layer, and gives the rest of its pages back.

        The tokens move to fresh pages: a shared page stays as it is for those who share it.
        Where the free pages do not hold all sequences at once, they move in turns.  The positions are
        looked at before anything moves, which waits for the device."""
        counts = [int(t.shape[0]) for t in keep]
        nat.require_device(*keep)
        for t in keep:
            if t.dim() != 1 or t.dtype not in (torch.int32, torch.int64):
                raise ValueError("keep holds a one-dimensional integer tensor for each sequence")
        _check_device(self.pool, *keep)
        book = self._book
        groups = book.plan_compaction(seqs, counts)
        if any(counts):
            n, c = self._upload([book.lens[s] for s in seqs], counts)
            at, end = torch.cat(list(keep)), n.repeat_interleave(c, output_size=sum(counts))
            if bool(((at < 0) | (at >= end)).any()):
                raise ValueError("keep names a position that is not one of its sequence's tokens")
        self._move(seqs, counts, groups, lambda group: torch.nn.utils.rnn.pad_sequence(
            [keep[i].to(torch.int32) for i in group], batch_first=True))

    def _move(self, seqs: Sequence[int], counts: Sequence[int], groups, rows) -> None:
        """The compaction of the groups of ``plan_compaction``; rows(group): the positions that stay."""
        book = self._book
        for group in groups:
            lens = [book.lens[seqs[i]] for i in group]
            moved = [book.replace(seqs[i], counts[i]) for i in group]
            try:
                old, wo = self._table([a for a, _ in moved])
                new, wn = self._table([b for _, b in moved])
                t_old, t_new, n = self._upload(old, new, [counts[i] for i in group])
                compact_pages(self.pool, t_old.view(len(group), wo), t_new.view(len(group), wn), rows(group), n)
            except BaseException:
                for i, (a, _), n in zip(group, moved, lens):
                    book.undo_replace(seqs[i], a, n)
                raise
            for a, _ in moved:
                book._drop(a)

    def evict(self, seqs: Sequence[int], scores: torch.Tensor, budget: int, protect_initial: int = 4,
              protect_recent: int = 16) -> torch.Tensor:
        """Hold each sequence to ``budget`` tokens: those past it that gathered the least attention leave,
        in every layer, by ``evict_select``'s rule.  scores (len(seqs), N) float32, N at least the longest
        sequence's length: the running importance of their tokens.  Returns it for the tokens that stay, at
        their new positions and 0 behind them.

        Nothing waits for the device.  Tokens move as in ``compact``, to fresh pages, in turns where need be; sequences
        within the budget stay as they are.  So a full pool is not relieved: it raises, and changes nothing, where the
        free pages do not hold one sequence's budget (``ceil(budget / page_size)``) at a time.  Keep as many free, or evict
        before ``extend`` finds none."""
        book = self._book
        book._known(seqs)
        budget, lens = index(budget), [book.lens[s] for s in seqs]
        if budget < 0:
            raise ValueError("a budget must be at least 0")
        if scores.dim() != 2 or scores.shape[0] != len(seqs) or scores.shape[1] < max(lens, default=0):
            raise ValueError(f"scores must be ({len(seqs)}, {max(lens, default=0)} or more)")
        _check_device(self.pool, scores)
        over = [i for i, n in enumerate(lens) if n > budget]
        groups = book.plan_compaction([seqs[i] for i in over], [budget] * len(over))
        keep, _, kept = evict_select(scores, self._upload(lens)[0], budget, protect_initial, protect_recent)
        self._move([seqs[i] for i in over], [budget] * len(over), groups,
                   lambda group: keep[self._upload([over[i] for i in group])[0].long()])
        return kept


class PackedPagedCache(_PagedCache):
    """Sequences of one model in a pool of 4-bit pages, shared by all its layers.

    A step: ``batch = cache.extend(seqs, counts)`` makes room (and copies the shared pages that
    will be written), then per layer ``append`` and ``attention``.  ``fork`` shares a sequence's
    pages; ``compact`` keeps chosen tokens, ``evict`` those that gathered the most attention;
    ``crop`` drops the last ones; ``remove`` frees.
    Calls that raise leave the cache as it was (a compaction in turns, the turns that are done).
    Work goes to the current stream."""

    def __init__(self, num_layers: int, num_heads: int, head_dim: int, page_size: int = 16, max_pages: int = 4096,
                 group_size: int = 32, device="cuda"):
        if torch.device(device).type != "cuda":
            raise RuntimeError("PackedPagedCache lives on the GPU (device 'cuda')")
        super().__init__(PagedPool.empty(num_layers, max_pages, num_heads, head_dim, page_size, group_size, device), max_pages)

    # ---- a layer's work
    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, batch: PagedBatch) -> None:
        paged_append(self.pool, batch, k, v, layer)

    def attention(self, layer: int, q: torch.Tensor, batch: PagedBatch, sm_scale: Optional[float] = None,
                  causal: bool = True, return_lse: bool = False):
        return paged_attention(q, self.pool, batch, layer, sm_scale, causal, return_lse)

    def importance(self, layer: int, q: torch.Tensor, lse: torch.Tensor, batch: PagedBatch, scores: torch.Tensor,
                   decay: float = 0.9, q_window: int = 0, sm_scale: Optional[float] = None, causal: bool = True) -> torch.Tensor:
        return paged_importance(q, lse, self.pool, batch, scores, layer, decay, q_window, sm_scale, causal)

    def get_kv(self, layer: int, seq: int, dtype: torch.dtype = torch.float16) -> Tuple[torch.Tensor, torch.Tensor]:
        """A sequence's keys and values (heads, length, head_dim) as the cache holds them."""
        k, v = paged_read(self.pool, self._batch([seq], [self.get_seq_length(seq)]), layer, dtype)
        return k.transpose(0, 1), v.transpose(0, 1)
