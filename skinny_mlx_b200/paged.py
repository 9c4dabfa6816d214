"""Paged key-value caches for batches of sequences on B200: append with rotation, attention.

A pool of pages per layer serves sequences of any length: `k_pages`, `v_pages` are
[n_pages, n_kv_heads, page, head_dim] (bf16, or float8_e4m3fn with one f32 scale per kv head) and row b
of the int32 `block_table` [B, width] names sequence b's pages in order.  One step of a batch is

    q = paged.append(q, k, v, k_pages, v_pages, block_table, lengths, inv_freq)   # per layer
    o = paged.attention(q, k_pages, v_pages, block_table, lengths)
    lengths += counts                                                             # once, after the last layer

with `lengths` (int32 [B]) the tokens cached BEFORE the step.  `counts` (int32 [B], default T each) are
the new tokens of every sequence: rows t >= counts[b] of the [B, T, ...] inputs are padding, so a batch
may have idle slots and drafts of different lengths.  All arguments stay on the device; a call makes no
host synchronisation and may be captured in a CUDA graph.

The contiguous, single-sequence counterpart is the attention of the fused verify step
(skinny_mlx_b200.fused); the reference's own cache is mlx_lm's contiguous KVCache
(skinny_mlx/rollback.py:72-73).
"""

from __future__ import annotations

import ctypes
import math

import torch

from . import _lib

_KV_TYPES = {torch.bfloat16: 0, torch.float8_e4m3fn: 1}
HEAD_DIMS = (64, 128, 256)
MAX_TOKENS = 16     # new tokens per sequence of one attention call
MAX_BATCH = 8192
MAX_POSITIONS = 2**31 - 4096  # of one sequence
_Strides = ctypes.c_longlong * 3


def _rows(x: torch.Tensor, name: str, b: int, t: int, d: int, dev: torch.device) -> tuple[torch.Tensor, ctypes.Array]:
    """A bf16 [B, T, heads, D] input whose dims are dense and whose rows are 16-byte aligned (copied if
    they are not), and its strides."""
    shape = x.shape
    if x.dtype != torch.bfloat16 or len(shape) != 4 or shape[0] != b or shape[1] != t or shape[3] != d:
        raise ValueError(f"{name} must be bf16 [{b}, {t}, heads, {d}], got {x.dtype} {tuple(shape)}")
    if x.device != dev:
        raise ValueError(f"{name} is on {x.device}, the pages on {dev}")
    sb, st, sh, sd = x.stride()
    # the stride of an axis of one element says nothing
    sb, st, sh = 0 if b == 1 else sb, 0 if t == 1 else st, 0 if shape[2] == 1 else sh
    if sd != 1 or (sb | st | sh) & 7 or x.data_ptr() & 15:
        x = x.clone(memory_format=torch.contiguous_format)
        sb, st, sh, _ = x.stride()
    return x, _Strides(sb, st, sh)


def _pool(k_pages: torch.Tensor, v_pages: torch.Tensor, k_scale, v_scale) -> int:
    """Checks a pool; returns its kv_type."""
    if not k_pages.is_cuda:
        raise ValueError("k_pages must be a CUDA tensor (no CPU fallback)")
    kv = _KV_TYPES.get(k_pages.dtype)
    if kv is None or v_pages.dtype != k_pages.dtype:
        raise ValueError("k_pages and v_pages must both be bfloat16 or float8_e4m3fn")
    if k_pages.dim() != 4 or k_pages.shape != v_pages.shape or v_pages.device != k_pages.device:
        raise ValueError("k_pages and v_pages must be [n_pages, n_kv_heads, page, head_dim] of one shape and device")
    _, h, page, d = k_pages.shape
    if d not in HEAD_DIMS:
        raise ValueError(f"head_dim must be one of {HEAD_DIMS}, got {d}")
    for name, x in (("k_pages", k_pages), ("v_pages", v_pages)):
        s = x.stride()
        if s[3] != 1 or (page > 1 and s[2] != d) or (h > 1 and s[1] != page * d) or x.data_ptr() % 16:
            raise ValueError(f"{name} must be dense inside a page ([n_kv_heads, page, head_dim]) and 16-byte aligned")
        if x.shape[0] > 1 and (s[0] < h * page * d or s[0] % d):
            raise ValueError(f"{name}: the page stride must be a multiple of head_dim and hold a page")
    for name, x in (("k_scale", k_scale), ("v_scale", v_scale)):
        if kv == 0:
            if x is not None:
                raise ValueError(f"{name} is for float8_e4m3fn pages")
        elif x is None or x.dtype != torch.float32 or x.shape != (h,) or not x.is_contiguous() or x.device != k_pages.device:
            raise ValueError(f"{name} must be a contiguous f32 [{h}] tensor on the pages' device")
    return kv


def _page_stride(x: torch.Tensor) -> int:
    if x.numel() == 0:
        raise ValueError("a pool holds at least one page of one kv head and one position")
    return x.stride(0) if x.shape[0] > 1 else x[0].numel()


def _seqs(block_table: torch.Tensor, lengths: torch.Tensor, counts, b: int, t: int, page: int, dev) -> None:
    if block_table.dtype != torch.int32 or block_table.dim() != 2 or block_table.shape[0] != b \
            or (block_table.shape[1] > 1 and block_table.stride(1) != 1) or block_table.device != dev:
        raise ValueError(f"block_table must be int32 [{b}, width] with dense rows on the pages' device")
    if block_table.shape[1] < 1 or (b > 1 and block_table.stride(0) < block_table.shape[1]):
        raise ValueError("block_table needs at least one entry per sequence and rows that do not overlap")
    if block_table.shape[1] * page > MAX_POSITIONS:
        raise ValueError(f"a sequence's pages must hold at most {MAX_POSITIONS} positions")
    for name, x in (("lengths", lengths), ("counts", counts)):
        if x is None and name == "counts":
            continue
        if x.dtype != torch.int32 or x.shape != (b,) or not x.is_contiguous() or x.device != dev:
            raise ValueError(f"{name} must be a contiguous int32 [{b}] tensor on the pages' device")
    if b > MAX_BATCH:
        raise ValueError(f"at most {MAX_BATCH} sequences per call")
    if b * t > 2**31 - 1:
        raise ValueError("too many tokens in one call")


def append(q: torch.Tensor | None, k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
           block_table: torch.Tensor, lengths: torch.Tensor, inv_freq: torch.Tensor | None = None, *,
           counts: torch.Tensor | None = None, k_scale: torch.Tensor | None = None,
           v_scale: torch.Tensor | None = None) -> torch.Tensor | None:
    """Write k, v (bf16 [B, T, n_kv_heads, D]) of the step's tokens into their pages, the keys rotated;
    returns the rotated queries (bf16 [B, T, n_heads, D]; None for q=None).

    Token t < counts[b] of sequence b sits at position lengths[b] + t; the first 2 * len(inv_freq) dims of
    its queries and keys are rotated (rotate-half) by position * inv_freq (f32; None: no rotation; the
    width a multiple of 16).  The angle is formed in f64, so far positions lose nothing.  Rows of padding
    write nothing and return zero queries.  float8_e4m3fn pages take x / scale[head], rounded to nearest and
    saturated.  T is not limited (a prompt is appended at once).  The inputs may be slices of a fused
    projection.  A page that is written must belong to one sequence of the batch only; pages that are only
    read may be shared.  A sequence that does not fit its row of the table, or a page id outside the pool,
    writes nothing and is reported by device_errors()."""
    kv = _pool(k_pages, v_pages, k_scale, v_scale)
    dev = k_pages.device
    n_pages, hkv, page, d = k_pages.shape
    if k.dim() != 4:
        raise ValueError("k must be [B, T, n_kv_heads, head_dim]")
    b, t = k.shape[:2]
    k, ks = _rows(k, "k", b, t, d, dev)
    v, vs = _rows(v, "v", b, t, d, dev)
    if k.shape[2] != hkv or v.shape[2] != hkv:
        raise ValueError(f"k and v must have the pages' {hkv} heads")
    out = qs = None
    hq = 0
    if q is not None:
        q, qs = _rows(q, "q", b, t, d, dev)
        hq = q.shape[2]
        out = torch.empty(b, t, hq, d, dtype=torch.bfloat16, device=dev)
    rot = 0
    if inv_freq is not None:
        if inv_freq.dtype != torch.float32 or inv_freq.dim() != 1 or not inv_freq.is_contiguous() or inv_freq.device != dev:
            raise ValueError("inv_freq must be a contiguous f32 vector on the pages' device")
        rot = 2 * inv_freq.numel()
        if rot % 16 or rot > d:
            raise ValueError("2 * len(inv_freq) must be a multiple of 16, at most head_dim")
    _seqs(block_table, lengths, counts, b, t, page, dev)
    if b == 0 or t == 0:
        return out
    _lib.launch("skinny_paged_append", dev.index, q.data_ptr() if hq else None, qs, k.data_ptr(), ks, v.data_ptr(), vs,
                out.data_ptr() if hq else None, k_pages.data_ptr(), v_pages.data_ptr(), _page_stride(k_pages),
                _page_stride(v_pages), kv, None if k_scale is None else k_scale.data_ptr(),
                None if v_scale is None else v_scale.data_ptr(), block_table.data_ptr(), block_table.stride(0),
                block_table.shape[1], n_pages, page, lengths.data_ptr(), None if counts is None else counts.data_ptr(),
                inv_freq.data_ptr() if rot else None, rot, b, t, hq, hkv, d)
    return out


_ws_bytes: dict[tuple, int] = {}


def attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor,
              lengths: torch.Tensor, *, counts: torch.Tensor | None = None, scale: float | None = None,
              window: int | None = None, k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None,
              return_lse: bool = False):
    """Attention of the step's new tokens (q bf16 [B, T, n_heads, D], T <= 16, already appended) over the
    pages of their sequences: bf16 [B, T, n_heads, D], and with return_lse the f32 [B, T, n_heads]
    ln sum exp of every row's scores.

    Token t sees the positions up to its own, lengths[b] + t, and with `window` only the last `window` of
    them.  scale defaults to head_dim ** -0.5.  Rows of padding (t >= counts[b]) are zero with lse -inf, and
    so is a row none of whose pages is in the pool (device_errors() reports those).  What a row does not see
    has no influence on it, whatever it holds."""
    kv = _pool(k_pages, v_pages, k_scale, v_scale)
    dev = k_pages.device
    n_pages, hkv, page, d = k_pages.shape
    if q.dim() != 4:
        raise ValueError("q must be [B, T, n_heads, head_dim]")
    b, t = q.shape[:2]
    q, qs = _rows(q, "q", b, t, d, dev)
    hq = q.shape[2]
    if t > MAX_TOKENS:
        raise ValueError(f"at most {MAX_TOKENS} new tokens per sequence")
    if hq < 1 or hkv < 1 or hq % hkv or hq > 1024 * hkv:
        raise ValueError(f"{hq} query heads do not divide over {hkv} kv heads, at most 1024 each")
    if window is not None and not 1 <= window < 2**31:
        raise ValueError("window must be at least 1")
    if scale is None:
        scale = 1.0 / math.sqrt(d)
    _seqs(block_table, lengths, counts, b, t, page, dev)
    out = torch.empty(b, t, hq, d, dtype=torch.bfloat16, device=dev)
    lse = torch.empty(b, t, hq, dtype=torch.float32, device=dev) if return_lse else None
    if b and t:
        key = (dev.index, b, t, hq, hkv, d)
        n = _ws_bytes.get(key)
        if n is None:
            with torch.cuda.device(dev):
                n = _ws_bytes[key] = int(_lib.lib().skinny_paged_attn_workspace_bytes(b, t, hq, hkv, d))
        # scratch of this call alone: calls on other streams and captured graphs have their own
        ws = torch.empty(n, dtype=torch.uint8, device=dev)
        _lib.launch("skinny_paged_attn", dev.index, q.data_ptr(), qs, k_pages.data_ptr(), v_pages.data_ptr(),
                    _page_stride(k_pages), _page_stride(v_pages), kv, None if k_scale is None else k_scale.data_ptr(),
                    None if v_scale is None else v_scale.data_ptr(), block_table.data_ptr(), block_table.stride(0),
                    block_table.shape[1], n_pages, page, lengths.data_ptr(),
                    None if counts is None else counts.data_ptr(), scale, window or 0, out.data_ptr(),
                    None if lse is None else lse.data_ptr(), b, t, hq, hkv, d, ws.data_ptr(), n)
    return (out, lse) if return_lse else out


class PagePool:
    """Pages for the attention layers of a model, handed out to sequences: per layer k, v
    [n_pages, n_kv_heads, page, head_dim] in bf16 or float8_e4m3fn.  A page id means the same page in every
    layer, so a sequence has one table for all of them.  k_scale, v_scale (f32 [layers, n_kv_heads],
    float8_e4m3fn only): what a stored value is multiplied by; ones by default."""

    def __init__(self, layers: int, n_pages: int, n_kv_heads: int, head_dim: int, page: int = 64, *,
                 dtype: torch.dtype = torch.bfloat16, k_scale: torch.Tensor | None = None,
                 v_scale: torch.Tensor | None = None, device="cuda"):
        if dtype not in _KV_TYPES:
            raise ValueError("pages are bfloat16 or float8_e4m3fn")
        if head_dim not in HEAD_DIMS:
            raise ValueError(f"head_dim must be one of {HEAD_DIMS}, got {head_dim}")
        if min(layers, n_pages, n_kv_heads, page) < 1:
            raise ValueError("layers, n_pages, n_kv_heads and page must be at least 1")
        if dtype == torch.bfloat16 and (k_scale is not None or v_scale is not None):
            raise ValueError("scales are for float8_e4m3fn pages")
        for name, x in (("k_scale", k_scale), ("v_scale", v_scale)):
            if x is not None and tuple(x.shape) != (layers, n_kv_heads):
                raise ValueError(f"{name} must be [{layers}, {n_kv_heads}], got {tuple(x.shape)}")
        self.page, self.n_pages, self.dtype = page, n_pages, dtype
        shape = (layers, n_pages, n_kv_heads, page, head_dim)
        self.k, self.v = (torch.zeros(shape, dtype=dtype, device=device) for _ in range(2))
        self.k_scale = self.v_scale = [None] * layers
        if dtype == torch.float8_e4m3fn:
            one = lambda s: torch.ones(layers, n_kv_heads, device=device) if s is None else s
            self.k_scale, self.v_scale = (list(one(s).to(device, torch.float32).contiguous()) for s in (k_scale, v_scale))
        self._free = list(range(n_pages - 1, -1, -1))
        self._taken: set[int] = set()

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def take(self, n: int) -> list[int]:
        """n pages of nobody; raises when there are not as many."""
        if n > len(self._free):
            raise RuntimeError(f"the page pool is exhausted: {n} pages wanted, {len(self._free)} of {self.n_pages} free")
        pages = [self._free.pop() for _ in range(n)]
        self._taken.update(pages)
        return pages

    def give(self, pages: list[int]) -> None:
        """Pages that were taken, back to nobody; a page that nobody has would later be two sequences'."""
        if len(set(pages)) != len(pages) or not self._taken.issuperset(pages):
            raise ValueError("only pages that are taken can be given back, each once")
        self._taken.difference_update(pages)
        self._free.extend(pages)


class PageTable:
    """One sequence's pages of a pool: the host list, and the row of the device table that the kernels read."""

    def __init__(self, pool: PagePool, max_len: int):
        self.pool, self.pages = pool, []
        self.width = -(-max_len // pool.page)
        self.device = torch.full((1, max(self.width, 1)), -1, dtype=torch.int32, device=pool.k.device)

    def reserve(self, length: int, cached: int = 0) -> None:
        """Pages for the first `length` positions (those that are there stay).  Of `cached` of them something is
        already stored: without their pages, released meanwhile, nothing is reserved."""
        need = -(-length // self.pool.page)
        if cached > len(self.pages) * self.pool.page:
            raise ValueError(f"the pages of {cached} cached positions have been released: empty the cache first")
        if need > self.width:
            raise ValueError(f"{length} positions do not fit a cache of {self.width * self.pool.page}")
        n = len(self.pages)
        if need > n:
            self.pages += self.pool.take(need - n)
            self.device[0, n:need] = torch.tensor(self.pages[n:], dtype=torch.int32).to(self.device.device, non_blocking=True)

    def release(self) -> None:
        """Every page back to the pool (also when the table is dropped)."""
        self.pool.give(self.pages)
        self.pages = []

    def __del__(self):
        if getattr(self, "pages", None):
            self.release()


def device_errors(device: torch.device | None = None, clear: bool = False) -> int:
    """The error bits of the paged calls made on `device` so far (synchronises with the current stream; calls on
    other streams are to be waited for first): 0; bit 9: a sequence or page id out of range; bit 0: a bounded
    wait ran out, the outputs of that call are void (skinny_b200.h).  clear: reset them afterwards."""
    word = ctypes.c_uint32()
    with torch.cuda.device(device):
        stream = torch.cuda.current_stream()
        _lib.call("skinny_paged_errors", ctypes.addressof(word), int(clear), stream.cuda_stream)
        stream.synchronize()
    return word.value


__all__ = ["append", "attention", "device_errors", "PagePool", "PageTable", "HEAD_DIMS", "MAX_BATCH", "MAX_POSITIONS", "MAX_TOKENS"]
