"""Latent attention over a paged latent cache: the attention half of a DeepSeek-V3 decoder layer.

A token is cached as 512 latent values, which are keys and values of every head, and a rotary
key of 64 that all heads share:

    cache = latent_cache(num_pages, page_size, dtype)
    latent_cache_write(cache, latent, k_rope, slots)                  # a step's new tokens
    out = latent_attention_decode(q, cache, block_table, lens, scale)    # absorbed form
    latent, k_rope = latent_cache_read(cache, block_table, cu_lens, total)
    out = latent_attention_prefill(q, kv, k_rope, cu_q, cu_k, scale)     # expanded form

The absorbed form multiplies the key up-projection into the query (q [.., 576] attends to the
cached rows themselves); the expanded form takes the up-projected keys and values of a prompt.
The kernels are inference only, like the rest of the library. As everywhere here there is no CPU
path: CPU tensors, a missing library or a non-sm_100 device raise.
"""

from __future__ import annotations

import torch

from . import _lib
from .ops import _DTYPES, _ptr, _require_cuda, _stream, _workspace, status_word

LATENT_DIM = 512
ROPE_DIM = 64
NOPE_DIM = 128
PAGE_SIZES = (16, 32, 64, 128)
_ROW8 = LATENT_DIM + 2 * ROPE_DIM + LATENT_DIM // 128


def latent_cache(num_pages: int, page_size: int = 64, dtype: torch.dtype = torch.bfloat16, device=None):
    """A zeroed paged latent cache: [num_pages, page_size, 576] in bf16 or fp16, or for
    ``torch.float8_e4m3fn`` uint8 [num_pages, page_size, 644] whose pages hold the codes
    [page_size, 512], then the rotary keys in bf16 [page_size, 64], then the exponent bytes of
    the power-of-two block scales [page_size, 4]."""
    if page_size not in PAGE_SIZES:
        raise ValueError(f"latent_cache: page_size must be one of {PAGE_SIZES}, got {page_size}")
    device = torch.device("cuda") if device is None else device
    if dtype == torch.float8_e4m3fn:
        return torch.zeros(num_pages, page_size, _ROW8, dtype=torch.uint8, device=device)
    if dtype not in _DTYPES:
        raise TypeError(f"latent_cache: dtype {dtype} not supported (bf16, fp16 or float8_e4m3fn)")
    return torch.zeros(num_pages, page_size, LATENT_DIM + ROPE_DIM, dtype=dtype, device=device)


def _cache_fmt(name: str, cache: torch.Tensor) -> int:
    if cache.dim() == 3 and cache.shape[1] in PAGE_SIZES and cache.is_contiguous():
        if cache.dtype == torch.uint8 and cache.shape[2] == _ROW8:
            return _lib.MOE_CACHE_E4M3
        if cache.dtype in _DTYPES and cache.shape[2] == LATENT_DIM + ROPE_DIM:
            return _DTYPES[cache.dtype]
    raise ValueError(f"{name}: cache must be a contiguous tensor made by latent_cache, got {cache.dtype} "
                     f"{tuple(cache.shape)}")


def _rows(name: str, what: str, t: torch.Tensor, cols: int) -> torch.Tensor:
    if t.dim() != 2 or t.shape[1] != cols:
        raise ValueError(f"{name}: {what} must be [tokens, {cols}], got {tuple(t.shape)}")
    return t if t.stride(1) == 1 else t.contiguous()


def _table(name: str, block_table: torch.Tensor, num_seqs: int) -> torch.Tensor:
    if block_table.dim() != 2 or block_table.shape[0] != num_seqs:
        raise ValueError(f"{name}: block_table must be [{num_seqs}, pages], got {tuple(block_table.shape)}")
    t = block_table if block_table.dtype == torch.int32 else block_table.to(torch.int32)
    return t if t.stride(1) == 1 or t.shape[1] <= 1 else t.contiguous()


def _ints(name: str, what: str, t: torch.Tensor) -> torch.Tensor:
    if t.dim() != 1 or t.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{name}: {what} must be a 1-D int32 or int64 tensor")
    return t if t.dtype == torch.int32 and t.is_contiguous() else t.to(torch.int32).contiguous()


def latent_cache_write(cache: torch.Tensor, latent: torch.Tensor, k_rope: torch.Tensor, slots: torch.Tensor) -> None:
    """Writes latent [n, 512] and k_rope [n, 64] (rows of any pitch) to the cache slots
    ``slots`` [n] = page * page_size + offset, each at most once; negative slots are skipped. 16-bit caches take their
    own dtype; an e4m3 cache takes bf16 and quantises each 128 latent values with the power-of-two
    scale of ``quantize_rows_fp8`` (non-finite values are kept as NaN and leave their block's scale
    alone; finite ones read back finite: those that would round to 2^128 take 15/16 of it). Slots past the cache are skipped and reported by ``check_device_status``."""
    name = "latent_cache_write"
    dev = _require_cuda(name, cache, latent, k_rope, slots)
    fmt = _cache_fmt(name, cache)
    want = torch.bfloat16 if fmt == _lib.MOE_CACHE_E4M3 else cache.dtype
    if latent.dtype != want or k_rope.dtype != want:
        raise TypeError(f"{name}: latent and k_rope must be {want} for this cache")
    latent, k_rope = _rows(name, "latent", latent, LATENT_DIM), _rows(name, "k_rope", k_rope, ROPE_DIM)
    n = latent.shape[0]
    if k_rope.shape[0] != n or slots.dim() != 1 or slots.shape[0] != n:
        raise ValueError(f"{name}: latent, k_rope and slots must have the same number of rows")
    if slots.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{name}: slots must be int32 or int64")
    if slots.dtype != torch.int64 or slots.stride(0) != 1:
        slots = slots.to(torch.int64).contiguous()
    _lib.check(
        _lib.load().moe_latent_cache_write(_DTYPES[want], _ptr(latent), latent.stride(0), _ptr(k_rope),
                                           k_rope.stride(0), _ptr(slots), n, fmt, _ptr(cache), cache.shape[0],
                                           cache.shape[1], _ptr(status_word(dev)), _stream(dev)),
        "moe_latent_cache_write")


def latent_cache_read(cache: torch.Tensor, block_table: torch.Tensor, cu_lens: torch.Tensor, total: int):
    """The first cu_lens[b + 1] - cu_lens[b] positions of every request as contiguous rows:
    (latent [total, 512], k_rope [total, 64]) in the cache's dtype, bf16 from an e4m3 cache
    (codes times power-of-two scales: exact). block_table [B, pages], cu_lens [B + 1] ascending
    (int32, on the device), total = cu_lens[B] as the caller knows it on the host. Rows before cu_lens[0] and
    past cu_lens[B] are zeros. Positions without a valid page read as NaN and are reported by ``check_device_status``."""
    name = "latent_cache_read"
    dev = _require_cuda(name, cache, block_table, cu_lens)
    fmt = _cache_fmt(name, cache)
    cu = _ints(name, "cu_lens", cu_lens)
    if cu.shape[0] < 1 or total < 0:
        raise ValueError(f"{name}: cu_lens needs at least one value and total must not be negative")
    table = _table(name, block_table, cu.shape[0] - 1)
    dt = torch.bfloat16 if fmt == _lib.MOE_CACHE_E4M3 else cache.dtype
    latent = torch.empty(total, LATENT_DIM, dtype=dt, device=dev)
    k_rope = torch.empty(total, ROPE_DIM, dtype=dt, device=dev)
    _lib.check(
        _lib.load().moe_latent_cache_read(fmt, _ptr(cache), cache.shape[0], cache.shape[1], _ptr(table),
                                          table.stride(0), table.shape[1], _ptr(cu), cu.shape[0] - 1, total,
                                          _ptr(latent), _ptr(k_rope), _ptr(status_word(dev)), _stream(dev)),
        "moe_latent_cache_read")
    return latent, k_rope


def latent_attention_decode(q, cache, block_table, cache_lens, scale, *, out=None, return_lse=False, workspace=None):
    """Latent attention over the paged cache in the absorbed form.

    q [B, n_q, heads, 576] (512 absorbed, 64 rotary; bf16 or fp16 as the cache, bf16 over an
    e4m3 cache), block_table int32 [B, pages], cache_lens int32 [B]: positions held, the n_q query
    tokens among them. Query token i sees positions j <= cache_lens[b] - n_q + i. Returns out
    [B, n_q, heads, 512] and with ``return_lse`` also the natural log-sum-exp fp32
    [B, n_q, heads]; a row that sees nothing gives zeros and -inf. ``workspace``: uint8, at least
    ``latent_attention_decode_workspace_bytes``."""
    name = "latent_attention_decode"
    dev = _require_cuda(name, q, cache, block_table, cache_lens)
    fmt = _cache_fmt(name, cache)
    want = torch.bfloat16 if fmt == _lib.MOE_CACHE_E4M3 else cache.dtype
    if q.dtype != want:
        raise TypeError(f"{name}: q must be {want} for this cache, got {q.dtype}")
    if q.dim() != 4 or q.shape[3] != LATENT_DIM + ROPE_DIM:
        raise ValueError(f"{name}: q must be [requests, n_q, heads, {LATENT_DIM + ROPE_DIM}], got {tuple(q.shape)}")
    B, n_q, heads, _ = q.shape
    lens = _ints(name, "cache_lens", cache_lens)
    if lens.shape[0] != B:
        raise ValueError(f"{name}: cache_lens must have {B} values")
    table = _table(name, block_table, B)
    if not q.is_contiguous() or q.data_ptr() % 16:
        q = q.clone(memory_format=torch.contiguous_format)
    shape = (B, n_q, heads, LATENT_DIM)
    if out is None:
        out = torch.empty(shape, dtype=want, device=dev)
    elif tuple(out.shape) != shape or out.dtype != want or not out.is_contiguous() or out.device != dev:
        raise ValueError(f"{name}: out must be a contiguous {want} {shape} tensor on {dev}")
    lse = torch.empty(B, n_q, heads, dtype=torch.float32, device=dev) if return_lse else None
    lib = _lib.load()
    if B and n_q and heads:
        workspace = _workspace(name, workspace, int(lib.moe_latent_decode_workspace_bytes(B, n_q, heads)), dev)
        _lib.check(
            lib.moe_latent_decode(_DTYPES[want], _ptr(q), B, n_q, heads, fmt, _ptr(cache), cache.shape[0],
                                  cache.shape[1], _ptr(table), table.stride(0), table.shape[1], _ptr(lens),
                                  float(scale), _ptr(out), _ptr(lse), _ptr(workspace),
                                  workspace.numel() * workspace.element_size(), _ptr(status_word(dev)), _stream(dev)),
            "moe_latent_decode")
    return (out, lse) if return_lse else out


def latent_attention_decode_workspace_bytes(num_requests: int, n_q: int, heads: int) -> int:
    return int(_lib.load().moe_latent_decode_workspace_bytes(num_requests, n_q, heads))


def _tma_rows(t: torch.Tensor) -> torch.Tensor:
    """t itself when TMA can read it (16-byte aligned rows, no broadcast), else a contiguous copy.
    The strides of dimensions of one are never used."""
    ok = t.data_ptr() % 16 == 0 and t.stride(-1) == 1
    for n, st in zip(t.shape[:-1], t.stride()[:-1]):
        ok = ok and (n <= 1 or (st > 0 and st % 8 == 0))
    return t if ok else t.clone(memory_format=torch.contiguous_format)


def latent_attention_prefill(q, kv, k_rope, cu_q, cu_k, scale, *, causal=True, out=None, return_lse=False):
    """Latent attention in the expanded form, over requests of different lengths.

    q [Tq, heads, 192] (128 without position, 64 rotary), kv [Tk, heads, 256] (128 key values
    without position, then 128 value values: the up-projection's output), k_rope [Tk, 64] shared by
    all heads; bf16 or fp16, views with strides are read in place. cu_q, cu_k int32 [B + 1], ascending: request
    b's queries and keys. ``causal``: the last query sees all keys, the one before it one less, and
    so on (queries are the last tokens of their context). Returns out [Tq, heads, 128] and with
    ``return_lse`` also the natural log-sum-exp fp32 [Tq, heads], by which pieces of a context can be
    joined; a row that sees nothing, or that belongs to no request, gives zeros and -inf."""
    name = "latent_attention_prefill"
    dev = _require_cuda(name, q, kv, k_rope, cu_q, cu_k)
    dt = q.dtype
    if dt not in _DTYPES:
        raise TypeError(f"{name}: dtype {dt} not supported (bf16 or fp16)")
    if kv.dtype != dt or k_rope.dtype != dt:
        raise TypeError(f"{name}: kv and k_rope must have the dtype of q")
    if q.dim() != 3 or q.shape[2] != NOPE_DIM + ROPE_DIM:
        raise ValueError(f"{name}: q must be [tokens, heads, {NOPE_DIM + ROPE_DIM}], got {tuple(q.shape)}")
    tq, heads, _ = q.shape
    if kv.dim() != 3 or kv.shape[1] != heads or kv.shape[2] != 2 * NOPE_DIM:
        raise ValueError(f"{name}: kv must be [tokens, {heads}, {2 * NOPE_DIM}], got {tuple(kv.shape)}")
    tk = kv.shape[0]
    if tuple(k_rope.shape) != (tk, ROPE_DIM):
        raise ValueError(f"{name}: k_rope must be [{tk}, {ROPE_DIM}], got {tuple(k_rope.shape)}")
    cu_q, cu_k = _ints(name, "cu_q", cu_q), _ints(name, "cu_k", cu_k)
    if cu_q.shape[0] < 1 or cu_q.shape != cu_k.shape:
        raise ValueError(f"{name}: cu_q and cu_k must have the same length, requests + 1")
    q, kv, k_rope = _tma_rows(q), _tma_rows(kv), _tma_rows(k_rope)
    if out is None:
        out = torch.empty(tq, heads, NOPE_DIM, dtype=dt, device=dev)
    elif tuple(out.shape) != (tq, heads, NOPE_DIM) or out.dtype != dt or not out.is_contiguous() or out.device != dev:
        raise ValueError(f"{name}: out must be a contiguous {dt} [{tq}, {heads}, {NOPE_DIM}] tensor on {dev}")
    lse = torch.empty(tq, heads, dtype=torch.float32, device=dev) if return_lse else None
    if tq and heads:
        _lib.check(
            _lib.load().moe_latent_prefill(_DTYPES[dt], _ptr(q), q.stride(0), q.stride(1), _ptr(kv), kv.stride(0),
                                           kv.stride(1), _ptr(k_rope), k_rope.stride(0), _ptr(cu_q), _ptr(cu_k),
                                           cu_q.shape[0] - 1, tq, tk, heads, float(scale), int(bool(causal)),
                                           _ptr(out), _ptr(lse), _ptr(status_word(dev)), _stream(dev)),
            "moe_latent_prefill")
    return (out, lse) if return_lse else out
