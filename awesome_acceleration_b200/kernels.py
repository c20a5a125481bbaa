"""Tensor-level wrappers over the C ABI (one call = one or two kernel launches).

Tensors must be CUDA, contiguous and of the documented dtype; every call
launches on the current PyTorch stream, so it composes with CUDA-graph
capture.  Outputs are allocated here only when the caller passes none.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib

BF16 = torch.bfloat16


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _p(t):
    return None if t is None else t.data_ptr()


def _lib_():
    return _lib.load()


def _req(t: torch.Tensor, dtype, name: str):
    if not t.is_cuda or t.dtype != dtype or not t.is_contiguous():
        raise ValueError(f"{name}: expected a contiguous CUDA {dtype} tensor, got {t.dtype} "
                         f"{'cuda' if t.is_cuda else 'cpu'} contiguous={t.is_contiguous()}")


# ---------------------------------------------------------------- KV cache
def kv_store(k: torch.Tensor, v: torch.Tensor, slot_mapping: torch.Tensor, k_cache: torch.Tensor,
             v_cache: torch.Tensor) -> None:
    """k/v [T, Hkv, 128] (row-strided views allowed); caches [blocks, Hkv, bs, 128]."""
    nb, hkv, bs, _ = k_cache.shape
    _req(slot_mapping, torch.int64, "slot_mapping")
    _lib.check(_lib_().aacc_kv_store(_p(k), _p(v), k.shape[0], k.stride(0), v.stride(0), _p(slot_mapping),
                                     _p(k_cache), _p(v_cache), nb, hkv, bs, _stream()), "kv_store")


def decode_slot_mapping(rows, seqlens, block_tables, block_size: int, num_blocks: int, out) -> None:
    _lib.check(_lib_().aacc_decode_slot_mapping(_p(rows), _p(seqlens), _p(block_tables), block_tables.shape[1],
                                                block_size, num_blocks, _p(out), rows.shape[0], _stream()),
               "decode_slot_mapping")


def advance_seqlens(rows, seqlens, positions=None) -> None:
    _lib.check(_lib_().aacc_advance_seqlens(_p(rows), _p(seqlens), _p(positions), rows.shape[0], _stream()),
               "advance_seqlens")


def gather_rows(src: torch.Tensor, idx: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    if out is None:
        out = torch.empty((idx.shape[0],) + tuple(src.shape[1:]), dtype=src.dtype, device=src.device)
    row_bytes = src[0].numel() * src.element_size()
    _lib.check(_lib_().aacc_gather_rows(_p(src), src.shape[0], row_bytes, _p(idx), idx.shape[0], _p(out),
                                        _stream()), "gather_rows")
    return out


# ---------------------------------------------------------------- attention
def decode_workspace_bytes(batch: int, num_q_heads: int, max_context: int, split_tokens: int = 0) -> int:
    """Workspace of paged_decode_attention (zero-filled before its first use) for calls of up to `batch` rows and
    `max_context` tokens, which may share it in turn."""
    return int(_lib_().aacc_paged_decode_workspace_bytes(batch, num_q_heads, max_context, split_tokens))


def paged_decode_attention(q, k_cache, v_cache, block_tables, rows, seqlens, *, ctx_add: int, scale: float,
                           max_context: int, workspace: torch.Tensor | None, out=None,
                           split_tokens: int = 0) -> torch.Tensor:
    """q [B, Hq, 128] -> out [B, Hq, 128] over seqlens[rows[b]] + ctx_add cached tokens."""
    B, hq, _ = q.shape
    nb, hkv, bs, _ = k_cache.shape
    if out is None:
        out = torch.empty_like(q)
    ws_bytes = 0 if workspace is None else workspace.numel() * workspace.element_size()
    _lib.check(_lib_().aacc_paged_decode_attention(
        _p(q), _p(out), _p(k_cache), _p(v_cache), nb, _p(block_tables), block_tables.shape[1], _p(rows),
        _p(seqlens), ctx_add, B, hq, hkv, bs, scale, split_tokens, max_context, _p(workspace), ws_bytes,
        _stream()), "paged_decode_attention")
    return out


def prefill_attention(q, k_cache, v_cache, block_tables, seq_rows, cu_q, ctx_start, *, max_q_len: int,
                      scale: float, out=None) -> torch.Tensor:
    """q [T, Hq, 128] packed by cu_q -> out [T, Hq, 128] (causal over cached context + chunk)."""
    T, hq, _ = q.shape
    nb, hkv, bs, _ = k_cache.shape
    if out is None:
        out = torch.empty_like(q)
    _lib.check(_lib_().aacc_prefill_attention(
        _p(q), _p(out), T, _p(k_cache), _p(v_cache), nb, _p(block_tables), block_tables.shape[1], _p(seq_rows),
        _p(cu_q), _p(ctx_start), seq_rows.shape[0], max_q_len, hq, hkv, bs, scale, _stream()),
        "prefill_attention")
    return out


# ---------------------------------------------------------------- request maps
# The wrappers below are called once per layer of a decode step, so their checks are one expression each; what
# exactly is wrong is only looked for once something is.
_I32, _I64, _U8 = torch.int32, torch.int64, torch.uint8
_current_device = torch._C._cuda_getDevice
_raw_stream = torch._C._cuda_getCurrentRawStream  # the current stream, without a Stream object around it


def _refuse(what: str, *args) -> None:
    """Raise for the first of (tensor, dtype, ndim, name) that is not a contiguous `ndim`-d `dtype` tensor on the
    current CUDA device, on whose current stream the kernels launch."""
    for t, dtype, ndim, name in args:
        if not isinstance(t, torch.Tensor):
            raise ValueError(f"{what}: {name} is not a tensor")
        if not t.is_cuda or t.get_device() != _current_device():
            raise ValueError(f"{what}: {name} is on {t.device}, expected the current CUDA device")
        if t.dtype is not dtype or t.dim() != ndim or not t.is_contiguous():
            raise ValueError(f"{what}: {name} must be a contiguous {ndim}-d {dtype} tensor, got {tuple(t.shape)} "
                             f"{t.dtype}, contiguous={t.is_contiguous()}")
    raise ValueError(f"{what}: shapes do not fit: " +
                     ", ".join(f"{name} {tuple(t.shape)}" for t, _, _, name in args))


def _ok(t, dtype, ndim: int, dev: int) -> bool:
    return (t is not None and t.dtype is dtype and t.ndim == ndim and t.get_device() == dev and t.is_contiguous())


def _is_current(dev: int) -> bool:
    return dev >= 0 and dev == _current_device()


def build_block_tables(lengths, block_size: int, *, max_blocks: int | None = None, free_blocks=None, out=None,
                       used=None) -> torch.Tensor:
    """Block tables int32 [S, max_blocks] of requests of `lengths` (int32 [S])
    tokens: request i takes ceil(lengths[i] / block_size) blocks of
    `free_blocks` (int32; None: 0, 1, 2, ...) in request order, the rest of
    its row is -1.  `used` (int32 [1]) receives the number of blocks taken."""
    what = "build_block_tables"
    dev = lengths.get_device()
    if not (_ok(lengths, _I32, 1, dev) and _is_current(dev)):
        _refuse(what, (lengths, _I32, 1, "lengths"))
    S = lengths.numel()
    if out is None:
        if max_blocks is None:
            raise ValueError(f"{what}: give max_blocks or out")
        out = torch.empty((S, max_blocks), dtype=_I32, device=lengths.device)
    elif not _ok(out, _I32, 2, dev) or out.shape[0] != S or (max_blocks is not None and out.shape[1] != max_blocks):
        _refuse(what, (out, _I32, 2, "out"), (lengths, _I32, 1, "lengths"))
    num_free = 0x7fffffff
    if free_blocks is not None:
        if not _ok(free_blocks, _I32, 1, dev):
            _refuse(what, (free_blocks, _I32, 1, "free_blocks"))
        num_free = free_blocks.numel()
    if used is not None and not (_ok(used, _I32, 1, dev) and used.numel() == 1):
        _refuse(what, (used, _I32, 1, "used"))
    rc = _lib.load().aacc_build_block_tables(lengths.data_ptr(), S, block_size, _p(free_blocks), num_free,
                                             out.data_ptr(), out.shape[1], _p(used), _raw_stream(dev))
    if rc:
        _lib.check(rc, what)
    return out


def build_slot_maps(lengths, block_tables, *, block_size: int, num_blocks: int, num_tokens: int, starts=None,
                    rows=None, cu=None, positions=None, slots=None):
    """(cu_seqlens int32 [S + 1], positions int64 [num_tokens], slots int64
    [num_tokens]) of tokens [starts[i], starts[i] + lengths[i]) of every
    request, packed.  `lengths`, `starts` int32 [S] (starts None: 0), `rows`
    int64 [S] names each request's row of `block_tables` (None: row i;
    negative: padding).  Entries behind the last request get position 0 and
    slot -1; `num_tokens` may exceed the sum of the lengths."""
    what = "build_slot_maps"
    dev = lengths.get_device()
    if not (_ok(lengths, _I32, 1, dev) and _ok(block_tables, _I32, 2, dev) and _is_current(dev)):
        _refuse(what, (lengths, _I32, 1, "lengths"), (block_tables, _I32, 2, "block_tables"))
    S = lengths.numel()
    if starts is not None and not (_ok(starts, _I32, 1, dev) and starts.numel() == S):
        _refuse(what, (starts, _I32, 1, "starts"), (lengths, _I32, 1, "lengths"))
    if rows is not None and not (_ok(rows, _I64, 1, dev) and rows.numel() == S):
        _refuse(what, (rows, _I64, 1, "rows"), (lengths, _I32, 1, "lengths"))
    if cu is None:
        cu = torch.empty(S + 1, dtype=_I32, device=lengths.device)
    elif not (_ok(cu, _I32, 1, dev) and cu.numel() == S + 1):
        _refuse(what, (cu, _I32, 1, "cu"), (lengths, _I32, 1, "lengths"))
    if positions is None:
        positions = torch.empty(num_tokens, dtype=_I64, device=lengths.device)
    elif not (_ok(positions, _I64, 1, dev) and positions.numel() == num_tokens):
        _refuse(f"{what} (num_tokens {num_tokens})", (positions, _I64, 1, "positions"))
    if slots is None:
        slots = torch.empty(num_tokens, dtype=_I64, device=lengths.device)
    elif not (_ok(slots, _I64, 1, dev) and slots.numel() == num_tokens):
        _refuse(f"{what} (num_tokens {num_tokens})", (slots, _I64, 1, "slots"))
    num_rows, max_blocks = block_tables.shape
    rc = _lib.load().aacc_build_slot_maps(
        lengths.data_ptr(), _p(starts), _p(rows), S, block_tables.data_ptr(), num_rows, max_blocks, block_size,
        num_blocks, cu.data_ptr(), positions.data_ptr(), slots.data_ptr(), num_tokens, _raw_stream(dev))
    if rc:
        _lib.check(rc, what)
    return cu, positions, slots


# ---------------------------------------------------------------- 4-bit KV cache
KV4_TILE = 64            # tokens of one record
KV4_RECORD_BYTES = 4608  # 64 tokens x 128 dims in 4 bits, and their 4 bf16 scales each


def kv4_cache_shape(num_blocks: int, num_kv_heads: int, block_size: int) -> tuple[int, int, int, int]:
    """Shape of one layer's uint8 K (or V) pool of the 4-bit cache."""
    if block_size <= 0 or block_size % KV4_TILE:
        raise ValueError(f"block_size must be a multiple of {KV4_TILE}, got {block_size}")
    return num_blocks, num_kv_heads, block_size // KV4_TILE, KV4_RECORD_BYTES


def _kv_rows(x, hkv: int, T: int, dev: int, what: str, name: str):
    """(row stride, head stride) in elements of bf16 rows [T, hkv, 128] or [T, hkv * 128]."""
    shape, strides = x.shape, x.stride()
    if not (x.dtype is BF16 and x.get_device() == dev and strides[-1] == 1
            and (shape == (T, hkv, 128) or shape == (T, hkv * 128))):
        raise ValueError(f"{what}: {name} must be bf16 rows [{T}, {hkv}, 128] with contiguous dims on cuda:{dev}, got "
                         f"{tuple(shape)} {x.dtype} strides {strides} on {x.device}")
    # a dimension of size 1 may carry any stride: it is never stepped over
    return strides[0] if T > 1 else 0, (strides[1] if len(shape) == 3 else 128) if hkv > 1 else 0


def kv4_store(k: torch.Tensor, v: torch.Tensor, slot_mapping: torch.Tensor, k_cache: torch.Tensor,
              v_cache: torch.Tensor) -> None:
    """Quantise k/v [T, Hkv, 128] bf16 (strided rows and heads allowed) into
    flat slots of the 4-bit pools (see kv4_cache_shape); negative slots skip,
    the others must be distinct."""
    what = "kv4_store"
    dev, pool, T = k_cache.get_device(), k_cache.shape, slot_mapping.numel()
    if not (k_cache.dtype is _U8 and v_cache.dtype is _U8 and v_cache.shape == pool and len(pool) == 4
            and pool[3] == KV4_RECORD_BYTES and slot_mapping.dtype is _I64 and slot_mapping.ndim == 1
            and dev >= 0 and dev == _current_device() and v_cache.get_device() == dev
            and slot_mapping.get_device() == dev and k_cache.is_contiguous() and v_cache.is_contiguous()
            and slot_mapping.is_contiguous()):
        _refuse(what, (k_cache, _U8, 4, "k_cache"), (v_cache, _U8, 4, "v_cache"),
                (slot_mapping, _I64, 1, "slot_mapping"))
    nb, hkv, tiles, _ = pool
    bs = tiles * KV4_TILE
    ks, kh = _kv_rows(k, hkv, T, dev, what, "k")
    vs, vh = _kv_rows(v, hkv, T, dev, what, "v")
    rc = _lib.load().aacc_kv4_store(k.data_ptr(), v.data_ptr(), T, ks, kh, vs, vh, slot_mapping.data_ptr(),
                                    k_cache.data_ptr(), v_cache.data_ptr(), nb, hkv, bs, _raw_stream(dev))
    if rc:
        _lib.check(rc, what)


def kv4_load(k_cache, v_cache, slots, k_out=None, v_out=None, *, out_slots=None):
    """Dequantise flat slots (int64 [T]) of the 4-bit pools into bf16: rows
    k_out/v_out [n, Hkv, 128], or paged caches [blocks, Hkv, bs, 128] of any
    block size; token t goes to row / flat slot out_slots[t] (None: t), and
    these must be distinct.  A negative slot on either side skips the token.
    Returns (k_out, v_out); outputs made here are zero where a token is
    skipped."""
    what = "kv4_load"
    dev, pool, T = k_cache.get_device(), k_cache.shape, slots.numel()
    if not (k_cache.dtype is _U8 and v_cache.dtype is _U8 and v_cache.shape == pool and len(pool) == 4
            and pool[3] == KV4_RECORD_BYTES and slots.dtype is _I64 and slots.ndim == 1
            and dev >= 0 and dev == _current_device() and v_cache.get_device() == dev and slots.get_device() == dev
            and k_cache.is_contiguous() and v_cache.is_contiguous() and slots.is_contiguous()
            and (out_slots is None or (out_slots.dtype is _I64 and out_slots.ndim == 1 and out_slots.numel() == T
                                       and out_slots.get_device() == dev and out_slots.is_contiguous()))):
        _refuse(what, (k_cache, _U8, 4, "k_cache"), (v_cache, _U8, 4, "v_cache"), (slots, _I64, 1, "slots"),
                *(() if out_slots is None else ((out_slots, _I64, 1, "out_slots"),)))
    nb, hkv, tiles, _ = pool
    bs = tiles * KV4_TILE
    if k_out is None or v_out is None:
        if out_slots is not None or k_out is not None or v_out is not None:
            raise ValueError(f"{what}: give both k_out and v_out (or neither and no out_slots)")
        k_out, v_out = torch.zeros((2, T, hkv, 128), dtype=BF16, device=k_cache.device)
    shape = k_out.shape
    ndim = len(shape)
    if not (k_out.dtype is BF16 and v_out.dtype is BF16 and v_out.shape == shape and (ndim == 3 or ndim == 4)
            and shape[1] == hkv and shape[-1] == 128 and k_out.get_device() == dev and v_out.get_device() == dev
            and k_out.is_contiguous() and v_out.is_contiguous()):
        _refuse(f"{what} (outputs [rows, {hkv}, 128] or [blocks, {hkv}, block_size, 128])",
                (k_out, BF16, ndim, "k_out"), (v_out, BF16, ndim, "v_out"))
    rc = _lib.load().aacc_kv4_load(k_cache.data_ptr(), v_cache.data_ptr(), nb, hkv, bs, slots.data_ptr(),
                                   _p(out_slots), T, k_out.data_ptr(), v_out.data_ptr(), shape[0],
                                   1 if ndim == 3 else shape[2], _raw_stream(dev))
    if rc:
        _lib.check(rc, what)
    return k_out, v_out


def kv4_decode_workspace_bytes(num_q_heads: int, num_kv_heads: int) -> int:
    """Workspace of kv4_decode_attention for any batch and context (zero-filled before its first use)."""
    return int(_lib_().aacc_kv4_decode_workspace_bytes(num_q_heads, num_kv_heads))


def kv4_decode_attention(q, k_cache, v_cache, block_tables, rows, seqlens, *, ctx_add: int, scale: float,
                         max_context: int, workspace: torch.Tensor, out=None) -> torch.Tensor:
    """q [B, Hq, 128] -> out [B, Hq, 128] over seqlens[rows[b]] + ctx_add
    tokens of the 4-bit pools (paged_decode_attention over the bf16 cache).
    V scales count in full down to 2^-100 of the largest of a row's context, elements of q down to 2^-100 of the
    largest of their head.
    Calls that share `workspace` (uint8) must be ordered on one stream."""
    what = "kv4_decode_attention"
    if out is None:
        out = torch.empty_like(q)
    dev, shape, pool, bt = q.get_device(), q.shape, k_cache.shape, block_tables.shape
    if not (q.dtype is BF16 and out.dtype is BF16 and out.shape == shape and len(shape) == 3 and shape[2] == 128
            and k_cache.dtype is _U8 and v_cache.dtype is _U8 and v_cache.shape == pool and len(pool) == 4
            and pool[3] == KV4_RECORD_BYTES and block_tables.dtype is _I32 and len(bt) == 2
            and rows.dtype is _I64 and rows.ndim == 1 and rows.numel() == shape[0]
            and seqlens.dtype is _I32 and seqlens.ndim == 1 and seqlens.numel() == bt[0]
            and workspace is not None and workspace.dtype is _U8 and dev >= 0 and dev == _current_device()
            and out.get_device() == dev and k_cache.get_device() == dev and v_cache.get_device() == dev and block_tables.get_device() == dev
            and rows.get_device() == dev and seqlens.get_device() == dev and workspace.get_device() == dev
            and q.is_contiguous() and out.is_contiguous() and k_cache.is_contiguous() and v_cache.is_contiguous()
            and block_tables.is_contiguous() and rows.is_contiguous() and seqlens.is_contiguous()
            and workspace.is_contiguous()):
        _refuse(what, (q, BF16, 3, "q"), (k_cache, _U8, 4, "k_cache"), (v_cache, _U8, 4, "v_cache"),
                (block_tables, _I32, 2, "block_tables"), (rows, _I64, 1, "rows"), (seqlens, _I32, 1, "seqlens"),
                (workspace, _U8, 1, "workspace"), (out, BF16, 3, "out"))
    B, hq, _ = shape
    nb, hkv, tiles, _ = pool
    num_rows, max_blocks = bt
    rc = _lib.load().aacc_kv4_decode_attention(
        q.data_ptr(), out.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), nb, block_tables.data_ptr(), num_rows,
        max_blocks, rows.data_ptr(), seqlens.data_ptr(), ctx_add, B, hq, hkv, tiles * KV4_TILE, scale, max_context,
        workspace.data_ptr(), workspace.numel(), _raw_stream(dev))
    if rc:
        _lib.check(rc, what)
    return out


# ---------------------------------------------------------------- norms
def rmsnorm(x, w, eps: float, out=None):
    H = x.shape[-1]
    rows = x.numel() // H
    if out is None:
        out = torch.empty_like(x)
    _lib.check(_lib_().aacc_rmsnorm(_p(x), _p(w), _p(out), rows, H, eps, _stream()), "rmsnorm")
    return out


def add_rmsnorm(delta, residual, w, eps: float, out=None):
    """residual <- bf16(residual + delta); returns rmsnorm(residual)."""
    H = residual.shape[-1]
    rows = residual.numel() // H
    if out is None:
        out = torch.empty_like(residual)
    _lib.check(_lib_().aacc_add_rmsnorm(_p(delta), _p(residual), _p(w), _p(out), rows, H, eps, _stream()),
               "add_rmsnorm")
    return out


def embed_rmsnorm(ids, table, w, eps: float, residual_out, out):
    rows = ids.numel()
    V, H = table.shape
    _lib.check(_lib_().aacc_embed_rmsnorm(_p(ids), _p(table), V, _p(residual_out), _p(w), _p(out), rows, H, eps,
                                          _stream()), "embed_rmsnorm")
    return out


# ---------------------------------------------------------------- GEMMs
def gemm(x, w, out=None, bias=None):
    """x [M, K] @ w[N, K]^T (+ bias [N], added in fp32 before the bf16 rounding)."""
    M, K = x.shape
    N = w.shape[0]
    if out is None:
        out = torch.empty((M, N), dtype=BF16, device=x.device)
    if bias is None:
        _lib.check(_lib_().aacc_gemm(_p(x), _p(w), _p(out), M, N, K, _stream()), "gemm")
    else:
        _req(bias, BF16, "bias")
        if bias.numel() != N:
            raise ValueError(f"gemm: bias has {bias.numel()} elements, expected {N}")
        _lib.check(_lib_().aacc_gemm_bias(_p(x), _p(w), _p(bias), _p(out), M, N, K, _stream()), "gemm_bias")
    return out


def bias_add(x, bias):
    """x [..., N] <- bf16(x + bias [N]) in place."""
    _req(x, BF16, "x")
    _req(bias, BF16, "bias")
    N = x.shape[-1]
    if bias.numel() != N:
        raise ValueError(f"bias_add: bias has {bias.numel()} elements, expected {N}")
    _lib.check(_lib_().aacc_bias_add(_p(x), _p(bias), x.numel() // N, N, _stream()), "bias_add")
    return x


def pick_splits(M: int, N: int, K: int, sms: int = 148, cap: int = 16, max_elems: int | None = None) -> int:
    """Largest divisor of K/64 (at most `cap`, and with splits*M*N fp32
    partials fitting `max_elems`) that keeps the split-K grid within one wave
    of CTAs (one 128x128 tile per SM) and whose fp32 partials (written, then
    read back) are no more bytes than the weights (splits*M*N*4 <= N*K*2).
    Measured on the cfg2 decode step (M=256): o_proj / down_proj at 4 splits
    beat 8 by 1.0 / 0.6 us per layer; QKV keeps 2."""
    tiles = ((N + 127) // 128) * ((M + 127) // 128)
    nk = K // 64
    best = 1
    for d in range(1, min(nk, cap) + 1):
        if (nk % d == 0 and tiles * d <= sms and (max_elems is None or d * M * N <= max_elems)
                and (d == 1 or 2 * d * M <= K)):
            best = d
    return best


def _check_partial(partial, splits: int, M: int, N: int, what: str):
    """The fp32 partial buffer must hold splits * M * N values (the kernels
    write every one of them; the C ABI cannot see the buffer's size)."""
    _req(partial, torch.float32, f"{what}: partial")
    if partial.numel() < splits * M * N:
        raise ValueError(f"{what}: partial holds {partial.numel()} values, needs {splits} x {M} x {N}")


def gemm_splitk(x, w, partial, splits: int):
    """partial [splits, M, N] fp32 <- split-K partial products of x @ w^T."""
    M, K = x.shape
    N = w.shape[0]
    _check_partial(partial, splits, M, N, "gemm_splitk")
    _lib.check(_lib_().aacc_gemm_splitk(_p(x), _p(w), _p(partial), M, N, K, splits, _stream()), "gemm_splitk")
    return partial


def splitk_add_rmsnorm(partial, splits: int, residual, w, eps: float, out):
    H = residual.shape[-1]
    rows = residual.numel() // H
    _lib.check(_lib_().aacc_splitk_add_rmsnorm(_p(partial), splits, _p(residual), _p(w), _p(out), rows, H, eps,
                                               _stream()), "splitk_add_rmsnorm")
    return out


def splitk_qkv_norm_rope_store(partial, splits: int, q_norm_w, k_norm_w, eps: float, positions, rope_cos_sin,
                               slot_mapping, k_cache, v_cache, num_q_heads: int, q_out):
    M = q_out.shape[0]
    nb, hkv, bs, _ = k_cache.shape
    _lib.check(_lib_().aacc_splitk_qkv_norm_rope_store(
        _p(partial), splits, _p(q_norm_w), _p(k_norm_w), eps, _p(positions), _p(rope_cos_sin),
        rope_cos_sin.shape[0], _p(slot_mapping), _p(q_out), _p(k_cache), _p(v_cache), nb, num_q_heads, hkv, bs, M,
        _stream()), "splitk_qkv_norm_rope_store")
    return q_out


def splitk_silu_mul(partial, splits: int, out):
    M, I = out.shape
    _lib.check(_lib_().aacc_splitk_silu_mul(_p(partial), splits, _p(out), M, I, _stream()), "splitk_silu_mul")
    return out


def splitk_reduce(partial, splits: int, out):
    rows, cols = out.shape
    _lib.check(_lib_().aacc_splitk_reduce(_p(partial), splits, _p(out), rows, cols, _stream()), "splitk_reduce")
    return out


# ---------------------------------------------------------------- small-batch decode projections
SKINNY_MAX_ROWS = 64      # what the kernels take
SKINNY_DEFAULT_ROWS = 32  # batches the engine sends through them
# Batches up to this run the QKV / SiLU epilogues in the GEMM's last split CTAs.  Off: on
# B200 the serial tail of the last CTA cost more than the separate epilogue launch at
# every batch measured (Qwen3-0.6B shapes, B = 1: 30.5 vs 27.4 us per layer).
SKINNY_FUSED_ROWS = 0
SKINNY_TARGET_CTAS = 296      # QKV / gate-up grids: about two CTAs per SM
SKINNY_TARGET_CTAS_ROW = 148  # o / down grids: fewer splits for the norm kernel to sum


def pick_skinny_splits(M: int, N: int, K: int, target: int = 296, max_elems: int | None = None,
                       cap: int = 64) -> int:
    """Split count of the small-batch GEMMs: the largest divisor d <= cap of
    K/64 with (N/128) * d CTAs at most `target` (two per SM by default: a CTA
    takes ~74-98 KB of shared memory), fp32 partials no more than half the
    weight bytes (4 * d * M <= K) and d * M * N fitting `max_elems`; 1 when
    the weight tiles alone reach the target."""
    tiles, nk = N // 128, K // 64
    best = 1
    for d in range(1, min(nk, cap) + 1):
        if (nk % d == 0 and tiles * d <= target and 4 * d * M <= K
                and (max_elems is None or d * M * N <= max_elems)):
            best = d
    return best


def _check_counters(counters, N: int, what: str):
    if counters.dtype != torch.int32 or counters.numel() < N // 128:
        raise ValueError(f"{what}: counters must be int32 with at least {N // 128} entries")


def gemm_skinny_splitk(x, w, partial, splits: int):
    """partial [splits, M, N] fp32 <- split-K partial products of x @ w^T
    (M <= 64 rows; the weights are the MMA's 128-row operand)."""
    M, K = x.shape
    N = w.shape[0]
    _check_partial(partial, splits, M, N, "gemm_skinny_splitk")
    _lib.check(_lib_().aacc_gemm_skinny_splitk(_p(x), _p(w), _p(partial), M, N, K, splits, _stream()),
               "gemm_skinny_splitk")
    return partial


def skinny_qkv_norm_rope_store(x, w_qkv, partial, splits: int, counters, q_norm_w, k_norm_w, eps: float, positions,
                               rope_cos_sin, slot_mapping, k_cache, v_cache, num_q_heads: int, q_out):
    """QKV projection + q/k norm + RoPE + KV store for M <= 64 rows in one
    launch (the epilogue runs in the last split CTA of each head)."""
    M, K = x.shape
    nb, hkv, bs, _ = k_cache.shape
    _check_counters(counters, w_qkv.shape[0], "skinny_qkv_norm_rope_store")
    _check_partial(partial, splits, M, w_qkv.shape[0], "skinny_qkv_norm_rope_store")
    _lib.check(_lib_().aacc_skinny_qkv_norm_rope_store(
        _p(x), _p(w_qkv), _p(partial), splits, _p(counters), _p(q_norm_w), _p(k_norm_w), eps, _p(positions),
        _p(rope_cos_sin), rope_cos_sin.shape[0], _p(slot_mapping), _p(q_out), _p(k_cache), _p(v_cache), nb,
        num_q_heads, hkv, bs, M, K, _stream()), "skinny_qkv_norm_rope_store")
    return q_out


def skinny_silu_mul(x, w_gate_up, partial, splits: int, counters, out):
    """out [M, I] = SiLU(gate) * up for M <= 64 rows in one launch."""
    M, K = x.shape
    I = w_gate_up.shape[0] // 2
    _check_counters(counters, 2 * I, "skinny_silu_mul")
    _check_partial(partial, splits, M, 2 * I, "skinny_silu_mul")
    _lib.check(_lib_().aacc_skinny_silu_mul(_p(x), _p(w_gate_up), _p(partial), splits, _p(counters), _p(out), M, I, K,
                                            _stream()), "skinny_silu_mul")
    return out


def gemm_silu_mul(x, w_gate_up, out=None):
    M, K = x.shape
    I = w_gate_up.shape[0] // 2
    if out is None:
        out = torch.empty((M, I), dtype=BF16, device=x.device)
    _lib.check(_lib_().aacc_gemm_silu_mul(_p(x), _p(w_gate_up), _p(out), M, I, K, _stream()), "gemm_silu_mul")
    return out


def qkv_norm_rope_store(x, w_qkv, q_norm_w, k_norm_w, eps: float, positions, rope_cos_sin, slot_mapping,
                        k_cache, v_cache, num_q_heads: int, q_out=None):
    M, K = x.shape
    nb, hkv, bs, _ = k_cache.shape
    if q_out is None:
        q_out = torch.empty((M, num_q_heads, 128), dtype=BF16, device=x.device)
    _lib.check(_lib_().aacc_qkv_norm_rope_store(
        _p(x), _p(w_qkv), _p(q_norm_w), _p(k_norm_w), eps, _p(positions), _p(rope_cos_sin), rope_cos_sin.shape[0],
        _p(slot_mapping), _p(q_out), _p(k_cache), _p(v_cache), nb, num_q_heads, hkv, bs, M, K, _stream()),
        "qkv_norm_rope_store")
    return q_out


# ---------------------------------------------------------------- decode projections (cluster split-K)
CLUSTER_MAX_ROWS = 256


def gemm_cluster(x, w, out=None, splits: int = 0):
    """bf16 x [M, K] @ w [N, K]^T for a decode batch (M <= 256), K split over a
    thread-block cluster and summed through distributed shared memory."""
    M, K = x.shape
    N = w.shape[0]
    if out is None:
        out = torch.empty((M, N), dtype=BF16, device=x.device)
    _lib.check(_lib_().aacc_gemm_cluster(_p(x), _p(w), _p(out), M, N, K, splits, _stream()), "gemm_cluster")
    return out


def gemm_silu_mul_cluster(x, w_gate_up, out=None, splits: int = 0):
    M, K = x.shape
    I = w_gate_up.shape[0] // 2
    if out is None:
        out = torch.empty((M, I), dtype=BF16, device=x.device)
    _lib.check(_lib_().aacc_gemm_silu_mul_cluster(_p(x), _p(w_gate_up), _p(out), M, I, K, splits, _stream()),
               "gemm_silu_mul_cluster")
    return out


def qkv_norm_rope_store_cluster(x, w_qkv, q_norm_w, k_norm_w, eps: float, positions, rope_cos_sin, slot_mapping,
                                k_cache, v_cache, num_q_heads: int, q_out=None, splits: int = 0):
    M, K = x.shape
    nb, hkv, bs, _ = k_cache.shape
    if q_out is None:
        q_out = torch.empty((M, num_q_heads, 128), dtype=BF16, device=x.device)
    _lib.check(_lib_().aacc_qkv_norm_rope_store_cluster(
        _p(x), _p(w_qkv), _p(q_norm_w), _p(k_norm_w), eps, _p(positions), _p(rope_cos_sin), rope_cos_sin.shape[0],
        _p(slot_mapping), _p(q_out), _p(k_cache), _p(v_cache), nb, num_q_heads, hkv, bs, M, K, splits, _stream()),
        "qkv_norm_rope_store_cluster")
    return q_out


def gemm_cluster_plan(M: int, N: int, K: int) -> tuple[int, int, int]:
    """(tile rows / 128, tiles over M, splits) the cluster GEMMs pick for M x N x K on this GPU."""
    mt, mtiles, splits = ctypes.c_int(), ctypes.c_int(), ctypes.c_int()
    _lib.check(_lib_().aacc_gemm_cluster_plan(M, N, K, ctypes.byref(mt), ctypes.byref(mtiles), ctypes.byref(splits)),
               "gemm_cluster_plan")
    return mt.value, mtiles.value, splits.value


def gemm_cluster_capacity(tile_rows_128: int, splits: int) -> int:
    """CTAs of the cluster GEMM with clusters of `splits` that fit on this GPU at once."""
    return int(_lib_().aacc_gemm_cluster_capacity(tile_rows_128, splits))


def lm_head_workspace_bytes(M: int, vocab: int) -> int:
    return int(_lib_().aacc_lm_head_workspace_bytes(M, vocab))


def lm_head_argmax(x, w, tokens, workspace, *, logits=None, best_val=None, vocab_offset: int = 0,
                   temperature=None, seeds=None, counters=None):
    """Next token of each row of x: greedy, or, for rows whose `temperature`
    (fp32 [M]) is > 0, a sample of softmax(bf16(logits / T)) drawn with
    counter-based Gumbel noise keyed by seeds / counters (int64 [M])."""
    M, K = x.shape
    V = w.shape[0]
    if temperature is not None:
        for t, dt, name in ((temperature, torch.float32, "temperature"), (seeds, torch.int64, "seeds"),
                            (counters, torch.int64, "counters")):
            if t is None or t.dtype != dt or t.numel() < M or not t.is_contiguous():
                raise ValueError(f"lm_head_argmax: {name} must be a contiguous {dt} tensor of >= {M} rows")
    _lib.check(_lib_().aacc_lm_head_sample(
        _p(x), _p(w), M, V, K, vocab_offset, _p(temperature), _p(seeds), _p(counters), _p(tokens), _p(best_val),
        _p(logits), _p(workspace), workspace.numel() * workspace.element_size(), _stream()), "lm_head_argmax")
    return tokens


def argmax_rows(logits, tokens=None):
    M, V = logits.shape
    if tokens is None:
        tokens = torch.empty(M, dtype=torch.int64, device=logits.device)
    _lib.check(_lib_().aacc_argmax_rows(_p(logits), M, V, _p(tokens), _stream()), "argmax_rows")
    return tokens


def sample_rows(logits, temperatures, seeds, counters, tokens=None):
    """Temperature sampling over materialised logits [M, V] (per-row host
    temperatures / seeds / counters); rows with temperature 0 take the argmax."""
    M, V = logits.shape
    dev = logits.device
    t = torch.as_tensor(temperatures, dtype=torch.float32).to(dev)
    sc = torch.as_tensor([list(seeds), list(counters)], dtype=torch.int64).to(dev)
    if tokens is None:
        tokens = torch.empty(M, dtype=torch.int64, device=dev)
    _lib.check(_lib_().aacc_sample_rows(_p(logits), M, V, _p(t), _p(sc[0]), _p(sc[1]), _p(tokens), _stream()),
               "sample_rows")
    return tokens


def argmax_merge(cand_val, cand_idx, tokens=None):
    """cand_val/cand_idx [shards, M] -> tokens [M]."""
    S, M = cand_val.shape
    if tokens is None:
        tokens = torch.empty(M, dtype=torch.int64, device=cand_val.device)
    _lib.check(_lib_().aacc_argmax_merge(_p(cand_val), _p(cand_idx), M, S, _p(tokens), _stream()), "argmax_merge")
    return tokens


def argmax_merge_packed(gathered, M: int, tokens):
    """Merge the vocab shards' candidates all-gathered as one int64 buffer
    [shards, 2 M] per rank: ids in [:M], fp32 values in the first M float32
    of [M:2M] (see Qwen3Runtime._argmax) -> tokens [M]."""
    S, W = gathered.shape
    if W != 2 * M or gathered.dtype != torch.int64 or not gathered.is_contiguous():
        raise ValueError("argmax_merge_packed: expected a contiguous int64 [shards, 2 M] buffer")
    vals = gathered.view(torch.float32)  # [S, 4 M]
    _lib.check(_lib_().aacc_argmax_merge_strided(_p(vals[:, 2 * M:]), _p(gathered), M, S, 4 * M, 2 * M, _p(tokens),
                                                 _stream()), "argmax_merge_packed")
    return tokens


def tp_set_peer_wait_ms(ms: int) -> None:
    """How long an exchange waits for a peer before it reports ERR_PEER_TIMEOUT (default 20 s)."""
    _lib.check(_lib_().aacc_tp_set_peer_wait_ms(int(ms)), "tp_set_peer_wait_ms")


def tp_exchange_bytes(world: int, max_rows: int, hidden: int) -> int:
    return int(_lib_().aacc_tp_exchange_bytes(world, max_rows, hidden))


def peer_buffer_alloc(nbytes: int) -> tuple[int, bytes]:
    """Zero-filled dedicated device buffer + its 64-byte CUDA IPC handle (set-up only)."""
    ptr = ctypes.c_void_p()
    handle = ctypes.create_string_buffer(64)
    _lib.check(_lib_().aacc_peer_buffer_alloc(nbytes, ctypes.byref(ptr), handle), "peer_buffer_alloc")
    return ptr.value, handle.raw


def peer_buffer_open(handle: bytes) -> int:
    ptr = ctypes.c_void_p()
    _lib.check(_lib_().aacc_peer_buffer_open(ctypes.create_string_buffer(handle, 64), ctypes.byref(ptr)),
               "peer_buffer_open")
    return ptr.value


def peer_buffer_close(ptr: int) -> None:
    _lib.check(_lib_().aacc_peer_buffer_close(ptr), "peer_buffer_close")


def peer_buffer_free(ptr: int) -> None:
    _lib.check(_lib_().aacc_peer_buffer_free(ptr), "peer_buffer_free")


def tp_allreduce_add_rmsnorm(src, splits: int, buffers, rank: int, max_rows: int, residual, w, eps: float, out,
                             two_shot: bool = False):
    """All-reduce of a RowParallel output over the group's exchange buffers, fused with the
    split-K sum (src fp32 [splits, M, H], or bf16 [M, H] with splits=0), the residual add
    (residual updated in place) and the RMSNorm into `out`."""
    M, H = residual.shape
    world = len(buffers)
    arr = (ctypes.c_void_p * world)(*buffers)
    _lib.check(_lib_().aacc_tp_allreduce_add_rmsnorm(_p(src), splits, arr, world, rank, int(two_shot), max_rows,
                                                     _p(residual), _p(w), _p(out), M, H, eps, _stream()),
               "tp_allreduce_add_rmsnorm")
    return out
