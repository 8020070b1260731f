"""A paged KV cache for models whose heads share one latent vector a token, and its operators.

Such a model keeps, for each token, a latent of ``latent_dim`` channels and a rotated key of
``rope_dim``; head h's keys are ``[W_k,h latent | rope]`` and its values ``W_v,h latent``.
``PagedLatentPool`` holds those rows of many sequences in pages; the batches are ``PagedBatch``.

  latent_append      new tokens into their slots
  latent_read        those tokens as the cache holds them
  latent_attention   the absorbed form: the key matrices are in the queries, outputs are sums of
                     latents, which the caller's value matrices follow.  For decode steps and drafts
  latent_prefill     the expanded form: keys and values of every head are made from the latents.
                     For chunks of some 170 query tokens and more it is the cheaper one
  latent_importance  the running importance of the cached tokens

``copy_pages``, ``compact_pages`` and ``evict_select`` serve this cache as they do the 4-bit one, and
``PagedLatentCache`` keeps the books.  Everything runs in libakv_hip.so; there is no CPU path and no
gradient."""
from __future__ import annotations

import ctypes
import struct
from typing import Optional, Tuple

import torch

from . import _native as nat
from .paged_packed import PagedBatch, _call, _check_device, _PagedCache, _rows

_QUERY = (torch.float16, torch.bfloat16)
_POOL, _BATCH = ctypes.sizeof(nat.LatentPool), ctypes.sizeof(nat.PagedBatch)
_ROWS = struct.Struct(f"@4i{_POOL}s{_BATCH}s4q")
_ATTN = struct.Struct(f"@5if{_POOL}s{_BATCH}s10q")
_PREFILL = struct.Struct(f"@5if{_POOL}s{_BATCH}s8q")
_IMPORTANCE = struct.Struct(f"@6i2f{_POOL}s{_BATCH}s14q")
_COMPACT = struct.Struct(f"@2i{_POOL}s4q2i4q")
for _s, _c in ((_ROWS, nat.LatentRowsArgs), (_ATTN, nat.LatentAttnArgs), (_PREFILL, nat.LatentPrefillArgs),
               (_IMPORTANCE, nat.LatentImportanceArgs), (_COMPACT, nat.LatentCompactArgs)):
    assert _s.size == ctypes.sizeof(_c), _c

HEAD_DIM = 128  # channels of a head's own keys, and of its values, in the expanded form


class PagedLatentPool:
    """The pages: ``data`` (layers, pages, page_size, latent_dim + rope_dim) float16.

    latent_dim 256 or 512, rope_dim 64, page_size a power of two from 16 to 256.  Rows are written by
    ``latent_append``; what free slots hold does not matter."""

    def __init__(self, data: torch.Tensor, latent_dim: int = 512):
        if data.dim() != 4 or data.dtype != torch.float16 or data.shape[3] <= latent_dim:
            raise ValueError(f"a pool is a (layers, pages, page_size, latent_dim + rope_dim) float16 tensor, got "
                             f"{tuple(data.shape)} {data.dtype}")
        nat.require_device(data)
        if not data.is_contiguous() or data.data_ptr() % 16:
            raise ValueError("a pool must be contiguous and 16-byte aligned")
        self.data, self.latent_dim, self.rope_dim = data, latent_dim, data.shape[3] - latent_dim
        self.num_layers, self.num_pages, self.page_size = data.shape[:3]
        self._index = data.get_device()
        self._c = bytes(nat.LatentPool(data.data_ptr(), self.num_pages, self.num_layers, latent_dim, self.rope_dim,
                                       self.page_size))
        lib = nat.load()
        self._copy, self._compact, self._compact_args = lib.akv_latent_copy, lib.akv_latent_compact, _COMPACT
        # every refusal of a pool's shape is the library's
        nat.check(self._copy(self._c, None, None, 0, None), "PagedLatentPool")

    @classmethod
    def empty(cls, num_layers: int, num_pages: int, latent_dim: int = 512, rope_dim: int = 64, page_size: int = 64,
              device="cuda") -> "PagedLatentPool":
        data = torch.zeros(num_layers, num_pages, page_size, latent_dim + rope_dim, dtype=torch.float16, device=device)
        return cls(data, latent_dim)

    def nbytes(self) -> int:
        return self.data.numel() * 2


def _tokens(x: torch.Tensor, name: str, T: int, D: int) -> Tuple[torch.Tensor, int]:
    """(T, D) with consecutive channels and rows on 16 bytes, copied if it is not, and the rows' byte stride."""
    if x.shape != (T, D):
        raise ValueError(f"{name} must be ({T}, {D}), got {tuple(x.shape)}")
    x, st, _ = _rows(x.unsqueeze(1), name, T, 1, D)
    return x, st


def _rows_args(pool: PagedLatentPool, batch: PagedBatch, latent: tuple, rope: tuple, layer: int) -> bytes:
    (latent, lt), (rope, rt) = latent, rope
    return _ROWS.pack(nat.ABI_VERSION, layer, nat.dtype_code(latent.dtype), 0, pool._c, batch._c, latent.data_ptr(),
                      rope.data_ptr(), lt, rt)


def latent_append(pool: PagedLatentPool, batch: PagedBatch, latent: torch.Tensor, rope: torch.Tensor, layer: int = 0) -> None:
    """latent (n_tokens, latent_dim) and rope (n_tokens, rope_dim), float16, bfloat16 or float32 and strided as
    they come, into the slots of the batch's rows, clamped to +-61440 and rounded to float16.

    A token with a value that is not finite reads back as NaN, and is NaN to every row that sees it."""
    _check_device(pool, latent, rope, batch.page_table)
    if latent.dtype != rope.dtype:
        raise TypeError(f"latent is {latent.dtype} and rope {rope.dtype}")
    latent = _tokens(latent, "latent", batch.n_tokens, pool.latent_dim)
    rope = _tokens(rope, "rope", batch.n_tokens, pool.rope_dim)
    _call(pool._index, "latent_append", nat.load().akv_latent_append, _rows_args(pool, batch, latent, rope, layer))


def latent_read(pool: PagedLatentPool, batch: PagedBatch, layer: int = 0,
                dtype: torch.dtype = torch.float16) -> Tuple[torch.Tensor, torch.Tensor]:
    """Latents (n_tokens, latent_dim) and rotated keys (n_tokens, rope_dim) of the batch's rows as the
    cache holds them; rows without a slot, and those that are no sequence's, are 0."""
    _check_device(pool, batch.page_table)
    nat.dtype_code(dtype)
    T, dev = batch.n_tokens, pool.data.device
    latent = torch.empty(T, pool.latent_dim, dtype=dtype, device=dev)
    rope = torch.empty(T, pool.rope_dim, dtype=dtype, device=dev)
    e = latent.element_size()
    _call(pool._index, "latent_read", nat.load().akv_latent_read,
          _rows_args(pool, batch, (latent, pool.latent_dim * e), (rope, pool.rope_dim * e), layer))
    return latent, rope


def _queries(q: torch.Tensor, q_rope: torch.Tensor, pool: PagedLatentPool, batch: PagedBatch) -> tuple:
    _check_device(pool, q, q_rope, batch.page_table)
    if q.dtype not in _QUERY or q_rope.dtype != q.dtype:
        raise TypeError("latent attention takes float16 or bfloat16 queries, q and q_rope alike")
    if q.dim() != 3:
        raise ValueError("q must be (n_tokens, heads, latent_dim)")
    T, H = batch.n_tokens, q.shape[1]
    return _rows(q, "q", T, H, pool.latent_dim) + _rows(q_rope, "q_rope", T, H, pool.rope_dim)


def _workspace(batch: PagedBatch, key: tuple, ask, args: struct.Struct, head: tuple) -> int:
    """Bytes that a call needs, remembered with the batch's sizes."""
    need = batch._workspace.get(key)
    if need is None:
        need = ask(args.pack(*head, 0, 0))
        if need >= 0:
            batch._workspace[key] = need
    return need


def latent_attention(q: torch.Tensor, q_rope: torch.Tensor, pool: PagedLatentPool, batch: PagedBatch, sm_scale: float,
                     layer: int = 0, causal: bool = True, return_lse: bool = False):
    """Attention in its absorbed form: q (n_tokens, H, latent_dim) holds ``W_k,h^T q_h``, q_rope (n_tokens, H,
    rope_dim) the rotated parts, float16 or bfloat16.  Returns the weighted sums of latents (n_tokens, H, latent_dim).

    ``sm_scale`` is that of the heads' own keys (their channels are not the latent's).  With ``causal``, row i of a
    sequence's m rows sees its first kv_len - m + 1 + i tokens, else all of them; a row that sees none is 0.
    ``return_lse`` adds the log-sums of exp(scores) (n_tokens, H) float32, -inf for such rows.  Scores, sums and
    log-sums are float32; the weights are rounded to float16, for float16 queries to 14 bits or more."""
    q, qt, qh, qr, qrt, qrh = _queries(q, q_rope, pool, batch)
    T, H, D = q.shape
    lib = nat.load()
    out = torch.empty(T, H, D, dtype=q.dtype, device=q.device)
    lse = torch.empty(T, H, dtype=torch.float32, device=q.device) if return_lse else None
    head = (nat.ABI_VERSION, layer, H, nat.dtype_code(q.dtype), int(causal), float(sm_scale), pool._c, batch._c, q.data_ptr(),
            qr.data_ptr(), qt, qh, qrt, qrh, out.data_ptr(), 0 if lse is None else lse.data_ptr())
    need = _workspace(batch, ("latent", D, pool.page_size, H), lib.akv_latent_attn_workspace_bytes, _ATTN, head)
    ws = torch.empty(need, dtype=torch.uint8, device=q.device) if need > 0 else None
    _call(pool._index, "latent_attention", lib.akv_latent_attn,
          _ATTN.pack(*head, 0, 0) if ws is None else _ATTN.pack(*head, ws.data_ptr(), need))
    return out if lse is None else (out, lse)


class LatentWeights:
    """The heads' matrices for ``latent_prefill``, laid out once: w_k (H, 128, latent_dim) from latents to a
    head's own keys, w_v (H, 128, latent_dim) to its values; float16, bfloat16 or float32, held as float16 over a
    power of two for each channel."""

    def __init__(self, w_k: torch.Tensor, w_v: torch.Tensor):
        nat.require_device(w_k, w_v)
        if w_k.dim() != 3 or w_k.shape != w_v.shape or w_k.shape[1] != HEAD_DIM:
            raise NotImplementedError(f"w_k and w_v must be (heads, {HEAD_DIM}, latent_dim), got {tuple(w_k.shape)} and "
                                      f"{tuple(w_v.shape)}")
        if w_k.shape[2] not in (256, 512):
            raise NotImplementedError(f"latent_dim 256 or 512, got {w_k.shape[2]}")
        if w_k.device != w_v.device:
            raise ValueError(f"w_k on {w_k.device} and w_v on {w_v.device}")
        nat.dtype_code(w_k.dtype), nat.dtype_code(w_v.dtype)
        self.heads, _, self.latent_dim = w_k.shape
        w = torch.cat([w_k.detach().float(), w_v.detach().float()], dim=1)
        top = w.abs().amax(dim=-1, keepdim=True)
        # a channel's largest weight in [2^-5, 2^-4): then sums over latents of the cache's size fit float16
        exponent = torch.where(top > 0, torch.frexp(top)[1] + 4, torch.zeros_like(top, dtype=torch.int32)).clamp(-100, 100)
        w = torch.ldexp(w, -exponent).half()
        # (head, wave, quarter, block, channel) x (step, part, 8): the operand's order
        w = w.view(self.heads, 4, 4, 4, 4, self.latent_dim // 32, 4, 8).permute(0, 5, 1, 3, 6, 2, 4, 7)
        self.data = w.contiguous()
        self.scale = torch.ldexp(torch.ones_like(top), exponent).view(self.heads, 2 * HEAD_DIM).contiguous()


def latent_prefill(q: torch.Tensor, pool: PagedLatentPool, batch: PagedBatch, weights: LatentWeights, layer: int = 0,
                   sm_scale: Optional[float] = None, causal: bool = True) -> torch.Tensor:
    """Attention in its expanded form: q (n_tokens, H, 128 + rope_dim), float16 or bfloat16, over the keys
    ``[W_k,h latent | rope]`` and values ``W_v,h latent`` of the cached tokens.  Returns (n_tokens, H, 128).

    ``sm_scale`` is by default one over the root of q's channels.  Rows see what they do in ``latent_attention``.
    Keys and values are float16, by channel over 16 times the power of two above its largest weight and clamped to +-65504
    there; the attention weights are float16 too.  For float16 queries all of them are two float16 each (and the clamp is twice
    as wide).  Keys and values are made for as many heads at a time as 4 GiB of workspace hold, and for as many tokens of a
    sequence as its row of the page table has slots."""
    _check_device(pool, q, batch.page_table, weights.data)
    if q.dtype not in _QUERY:
        raise TypeError("latent attention takes float16 or bfloat16 queries")
    if weights.latent_dim != pool.latent_dim:
        raise ValueError(f"weights for latents of {weights.latent_dim} beside a pool of {pool.latent_dim}")
    T, H, D = batch.n_tokens, weights.heads, HEAD_DIM + pool.rope_dim
    q, qt, qh = _rows(q, "q", T, H, D)
    lib = nat.load()
    out = torch.empty(T, H, HEAD_DIM, dtype=q.dtype, device=q.device)
    head = (nat.ABI_VERSION, layer, H, nat.dtype_code(q.dtype), int(causal),
            nat.default_sm_scale(D) if sm_scale is None else float(sm_scale), pool._c, batch._c, weights.data.data_ptr(),
            weights.scale.data_ptr(), q.data_ptr(), qt, qh, out.data_ptr())
    need = _workspace(batch, ("prefill", q.dtype, pool.latent_dim, pool.page_size, H), lib.akv_latent_prefill_workspace_bytes,
                      _PREFILL, head)
    ws = torch.empty(need, dtype=torch.uint8, device=q.device) if need > 0 else None
    _call(pool._index, "latent_prefill", lib.akv_latent_prefill,
          _PREFILL.pack(*head, 0, 0) if ws is None else _PREFILL.pack(*head, ws.data_ptr(), need))
    return out


def latent_importance(q: torch.Tensor, q_rope: torch.Tensor, lse: torch.Tensor, pool: PagedLatentPool, batch: PagedBatch,
                      scores: torch.Tensor, sm_scale: float, layer: int = 0, decay: float = 0.9, q_window: int = 0,
                      causal: bool = True, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The running importance of the cached tokens, by the rule of ``paged_importance``: scores (S, N) float32
    become ``scores * decay + sum over rows of the mean over heads of the attention weights``.

    q, q_rope and lse are those of ``latent_attention``.  Written in place, or to ``out``, which does not
    overlap scores; returns what was written."""
    q, qt, qh, qr, qrt, qrh = _queries(q, q_rope, pool, batch)
    T, H, D = q.shape
    dst = scores if out is None else out
    _check_device(pool, lse, scores, dst)
    if lse.dtype != torch.float32 or lse.shape != (T, H):
        raise ValueError(f"lse must be ({T}, {H}) float32")
    for t in (scores, dst):
        if t.dtype != torch.float32 or t.dim() != 2 or t.shape[0] != batch.n_seqs or t.shape != scores.shape:
            raise ValueError(f"scores must be ({batch.n_seqs}, tokens) float32")
        if t.shape[1] > 1 and t.stride(1) != 1:
            raise ValueError("a sequence's scores must be consecutive")
    if not lse.is_contiguous():
        lse = lse.contiguous()
    lib = nat.load()
    head = (nat.ABI_VERSION, layer, H, nat.dtype_code(q.dtype), int(causal), int(q_window), float(sm_scale), float(decay), pool._c,
            batch._c, q.data_ptr(), qr.data_ptr(), qt, qh, qrt, qrh, lse.data_ptr(), scores.data_ptr(), dst.data_ptr(),
            scores.shape[1], scores.stride(0), dst.stride(0))
    need = _workspace(batch, ("importance", D, H, int(q_window)), lib.akv_latent_importance_workspace_bytes, _IMPORTANCE, head)
    ws = torch.empty(need, dtype=torch.uint8, device=q.device) if need > 0 else None
    _call(pool._index, "latent_importance", lib.akv_latent_importance,
          _IMPORTANCE.pack(*head, 0, 0) if ws is None else _IMPORTANCE.pack(*head, ws.data_ptr(), need))
    return dst


class PagedLatentCache(_PagedCache):
    """Sequences of one model with latent attention in a pool of pages, shared by all its layers.

    A step is ``PackedPagedCache``'s: ``extend``, then per layer ``append`` and ``attention`` (``prefill`` for
    chunks of a prompt); ``fork``, ``compact``, ``evict``, ``crop`` and ``remove`` are the same."""

    def __init__(self, num_layers: int, latent_dim: int = 512, rope_dim: int = 64, page_size: int = 64, max_pages: int = 4096,
                 device="cuda"):
        if torch.device(device).type != "cuda":
            raise RuntimeError("PagedLatentCache lives on the GPU (device 'cuda')")
        super().__init__(PagedLatentPool.empty(num_layers, max_pages, latent_dim, rope_dim, page_size, device), max_pages)

    # ---- a layer's work
    def append(self, layer: int, latent: torch.Tensor, rope: torch.Tensor, batch: PagedBatch) -> None:
        latent_append(self.pool, batch, latent, rope, layer)

    def attention(self, layer: int, q: torch.Tensor, q_rope: torch.Tensor, batch: PagedBatch, sm_scale: float,
                  causal: bool = True, return_lse: bool = False):
        return latent_attention(q, q_rope, self.pool, batch, sm_scale, layer, causal, return_lse)

    def prefill(self, layer: int, q: torch.Tensor, batch: PagedBatch, weights: LatentWeights, sm_scale: Optional[float] = None,
                causal: bool = True) -> torch.Tensor:
        return latent_prefill(q, self.pool, batch, weights, layer, sm_scale, causal)

    def importance(self, layer: int, q: torch.Tensor, q_rope: torch.Tensor, lse: torch.Tensor, batch: PagedBatch,
                   scores: torch.Tensor, sm_scale: float, decay: float = 0.9, q_window: int = 0,
                   causal: bool = True) -> torch.Tensor:
        return latent_importance(q, q_rope, lse, self.pool, batch, scores, sm_scale, layer, decay, q_window, causal)

    def get_rows(self, layer: int, seq: int, dtype: torch.dtype = torch.float16) -> Tuple[torch.Tensor, torch.Tensor]:
        """A sequence's latents (length, latent_dim) and rotated keys (length, rope_dim) as the cache holds them."""
        return latent_read(self.pool, self._batch([seq], [self.get_seq_length(seq)]), layer, dtype)
