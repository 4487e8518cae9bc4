"""The steps between the forwards of a bounded cache.

  rope_cache_write        rotary positions on new Q and K, the sign words of both and V's
                          codes, written where the forward reads them
  accumulate_key_weights  a running sum of the attention weight of every cached key
  evict_keys              each cache row cut to a budget by that sum, packed in place

A decode step at the budget is rope_cache_write (slot = the row's context length, then
length + 1), the forward, accumulate_key_weights, evict_keys.  The three keep the
forward's conventions: asynchronous on the current stream of the cache's device, arguments
checked on the host (RuntimeError), bad pages and rows skipped and flagged on the device
(read_device_errors), cache rows numbered sequence * n_kv_heads + head.  They may be
captured into CUDA graphs; scratch is allocated per call, so captured graphs share none.
"""
from __future__ import annotations

from typing import Optional, Union

import torch

from . import _capi, _nbytes, _raw_stream, _workspace

_IN_DTYPES = {torch.float16: _capi.DTYPE_F16, torch.bfloat16: _capi.DTYPE_BF16, torch.float32: _capi.DTYPE_F32}
_LAYOUTS = {"half": _capi.ROPE_HALF, "interleaved": _capi.ROPE_INTERLEAVED}
_WS_BYTES = 1 << 16
_I32, _F32 = torch.int32, torch.float32
_INT_MAX = 0x7FFFFFFF
_F32_MAX = torch.finfo(_F32).max


def _refuse(name: str, msg: str) -> None:
    raise RuntimeError(f"{name}: {msg}")


def _check_tensors(name: str, dev: torch.device, names: str, *tensors: Optional[torch.Tensor]) -> None:
    """Every tensor given is contiguous and on the caches' device."""
    idx = dev.index
    for t in tensors:
        if t is not None and not (t.is_contiguous() and t.get_device() == idx):
            break
    else:
        return
    named = [(n, t) for n, t in zip(names.split(), tensors) if t is not None]
    for n, t in named:
        if not t.is_contiguous():
            _refuse(name, f"{n} must be contiguous")
    if dev.type != "cuda":
        _refuse(name, "the caches must be CUDA tensors")
    for n, t in named:
        if t.device != dev:
            _refuse(name, f"{n} must be on {dev}")


def _tables(name: str, block_tables: Optional[torch.Tensor]):
    """(address, numel) of the block tables; (0, 0) for the contiguous layout."""
    if block_tables is None or block_tables.numel() == 0:
        return 0, 0
    if not (block_tables.dtype is _I32):
        _refuse(name, "block_tables must be int32")
    return block_tables.data_ptr(), block_tables.numel()


def _same_or_apart(name: str, arg: str, a: torch.Tensor, b: torch.Tensor) -> None:
    p, q = a.data_ptr(), b.data_ptr()
    if not (p == q or p + _nbytes(a) <= q or q + _nbytes(b) <= p):
        _refuse(name, f"{arg} overlaps its input")


def _scratch(dev: torch.device, nbytes: int):
    """Fresh scratch of a call and its address (0 where it needs none)."""
    if nbytes == 0:
        return None, 0
    buf = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    return buf, buf.data_ptr()


def _call(name: str, fn, args: bytes, dev: torch.device) -> None:
    """Enqueues `fn` on the current stream of `dev`."""
    if torch.cuda.current_device() != dev.index:
        with torch.cuda.device(dev):
            return _call(name, fn, args, dev)
    ws = _workspace(dev, _WS_BYTES)
    rc = fn(args, ws.data_ptr(), ws.numel(), _raw_stream(dev.index))
    if rc != _capi.HYPERION_OK:
        raise RuntimeError(f"{name} failed (status {rc}): {_capi.last_error()}")


def rope_cache_write(Q_new: torch.Tensor, K_new: torch.Tensor, V_new: torch.Tensor, seq_ids: torch.Tensor,
                     positions: torch.Tensor, rope: Optional[torch.Tensor], block_tables: Optional[torch.Tensor],
                     block_size: int, num_blocks: int, V_scale: torch.Tensor, Q_words: torch.Tensor,
                     K_cache: torch.Tensor, V_cache: torch.Tensor, *, layout: str = "half", seq_q: int = 1,
                     q_idx: Optional[torch.Tensor] = None, slots: Optional[torch.Tensor] = None,
                     slot_positions: Optional[torch.Tensor] = None) -> None:
    """Turns new queries and keys by their positions and writes what the forward reads.

    Q_new [n_tokens, n_heads, head_dim], K_new and V_new [n_tokens, n_kv_heads, head_dim]:
    float16, bfloat16 or float32, any strides between tokens and heads (slices of a fused
    projection), each head's dims contiguous.  Token i belongs to sequence seq_ids[i] and
    stands at positions[i] (int32).

    rope: float32 [n_positions, 2, rotary_dim / 2], the cos and sin row of each position
    (glue.rope_table); the first rotary_dim dims of a head turn, in the pairs
    (j, j + rotary_dim / 2) with layout "half" and (2j, 2j + 1) with "interleaved".  None:
    nothing turns.

    Q_words (int32 storage, head_dim / 32 words a row) gets the sign words of the turned
    queries at row (seq * n_heads + head) * seq_q + q_idx, the forward's Q; q_idx (int32
    [n_tokens]) defaults to 0 when seq_q is 1 and to the positions otherwise.  K_cache and
    V_cache get K's sign words and V's e4m3 codes (as kv_cache_write) at the cache slot
    slots[i] (int32 [n_tokens] or [n_tokens, n_kv_heads]), by default the position.
    slot_positions (int32 [cache rows, num_blocks * block_size]) gets the position there.

    A bit is 1 where the exact x*cos - y*sin (or y*cos + x*sin) is >= 0.  Rows, slots,
    positions and pages out of range are skipped and flagged.  Two tokens of a call must
    not name the same slot or query row."""
    name = "rope_cache_write"
    dtype = Q_new.dtype
    if not (dtype in _IN_DTYPES and K_new.dtype is dtype and V_new.dtype is dtype):
        _refuse(name, "Q_new, K_new and V_new must share a float16, bfloat16 or float32 dtype")
    if not (Q_new.dim() == 3 and K_new.dim() == 3 and V_new.shape == K_new.shape):
        _refuse(name, "Q_new must be [n_tokens, n_heads, head_dim], K_new and V_new [n_tokens, n_kv_heads, head_dim]")
    n_tokens, n_heads, head_dim = Q_new.shape
    k_tokens, n_kv, k_dim = K_new.shape
    if not (k_tokens == n_tokens and k_dim == head_dim):
        _refuse(name, "Q_new and K_new differ in tokens or head_dim")
    if not (head_dim in (128, 256)):
        _refuse(name, "head_dim must be 128 or 256")
    if not (n_heads >= 1 and n_kv >= 1):
        _refuse(name, "n_heads and n_kv_heads must be >= 1")
    if not (n_tokens * (n_heads + n_kv) <= _INT_MAX):
        _refuse(name, "too many (token, head) rows")
    qs, ks, vs = Q_new.stride(), K_new.stride(), V_new.stride()
    if not (n_tokens == 0 or (qs[2] == 1 and ks[2] == 1 and vs[2] == 1)):
        _refuse(name, "the dims of a head must be contiguous")
    if not (seq_ids.dtype is _I32 and positions.dtype is _I32 and seq_ids.numel() == n_tokens
            and positions.numel() == n_tokens):
        _refuse(name, "seq_ids and positions must be int32 [n_tokens]")
    if not (q_idx is None or (q_idx.dtype is _I32 and q_idx.numel() == n_tokens)):
        _refuse(name, "q_idx must be int32 [n_tokens]")
    per_head = 0
    if slots is not None:
        per_head = slots.dim() - 1
        if not (slots.dtype is _I32 and slots.shape == ((n_tokens, n_kv) if per_head else (n_tokens,))):
            _refuse(name, "slots must be int32 [n_tokens] or [n_tokens, n_kv_heads]")
    rot = n_pos = 0
    if rope is not None:
        if not (rope.dtype is _F32 and rope.dim() == 3):
            _refuse(name, "rope must be float32 [n_positions, 2, rotary_dim / 2]")
        n_pos, two, rot = rope.shape
        if not (two == 2 and 1 <= n_pos <= _INT_MAX):
            _refuse(name, "rope must be float32 [n_positions, 2, rotary_dim / 2]")
        rot *= 2
        if not (rot <= head_dim):
            _refuse(name, "rope turns more dims than head_dim")
    if not (layout in _LAYOUTS):
        _refuse(name, "layout must be 'half' or 'interleaved'")
    if not (1 <= seq_q <= _INT_MAX):
        _refuse(name, "seq_q must be >= 1 and fit int32")
    if not (block_size >= 1 and num_blocks >= 1 and block_size * num_blocks <= _INT_MAX):
        _refuse(name, "block_size and num_blocks must be >= 1, their product in int32")
    scales, codes = V_scale.numel(), V_cache.numel()
    if not (V_scale.dtype is _F32 and scales >= 1):
        _refuse(name, "V_scale must be a non-empty float32 tensor")
    if not (V_cache.element_size() == 1 and codes % head_dim == 0 and codes > 0):
        _refuse(name, "V_cache must hold one byte per element, [pool_rows, head_dim]")
    pool_rows = codes // head_dim
    if not (K_cache.numel() * K_cache.element_size() >= codes // 8):
        _refuse(name, "K_cache smaller than pool_rows rows of head_dim/8 bytes")
    q_rows, rest = divmod(Q_words.numel() * Q_words.element_size(), head_dim // 8)
    if rest:
        _refuse(name, "Q_words bytes must be a multiple of head_dim/8")
    slot_rows = 0
    if slot_positions is not None:
        if not (slot_positions.dtype is _I32 and slot_positions.dim() == 2):
            _refuse(name, "slot_positions must be int32 [cache rows, num_blocks * block_size]")
        slot_rows, width = slot_positions.shape
        if width != block_size * num_blocks:
            _refuse(name, "slot_positions must be int32 [cache rows, num_blocks * block_size]")
    bt, bt_numel = _tables(name, block_tables)
    dev = K_cache.device
    _check_tensors(name, dev, "seq_ids positions rope block_tables V_scale Q_words K_cache V_cache q_idx slots slot_positions",
                   seq_ids, positions, rope, block_tables, V_scale, Q_words, K_cache, V_cache, q_idx, slots, slot_positions)
    idx = dev.index
    if not (Q_new.get_device() == idx and K_new.get_device() == idx and V_new.get_device() == idx):
        _refuse(name, f"Q_new, K_new and V_new must be on {dev}")
    args = _capi.pack_rope_write(
        Q_new.data_ptr(), K_new.data_ptr(), V_new.data_ptr(), qs[0], qs[1], ks[0], ks[1], vs[0], vs[1],
        _IN_DTYPES[dtype], n_tokens, n_heads, n_kv, head_dim, rot, _LAYOUTS[layout], n_pos,
        rope.data_ptr() if rot else 0, seq_ids.data_ptr(), positions.data_ptr(),
        0 if q_idx is None else q_idx.data_ptr(), 0 if slots is None else slots.data_ptr(), per_head, seq_q,
        Q_words.data_ptr(), q_rows, bt, bt_numel, block_size, num_blocks,
        V_scale.data_ptr(), scales, K_cache.data_ptr(), V_cache.data_ptr(), pool_rows,
        slot_positions.data_ptr() if slot_rows else 0, slot_rows)
    _call(name, _capi.lib.hyperion_rope_cache_write, args, dev)


def accumulate_key_weights(Q: torch.Tensor, K_cache: torch.Tensor, context_lens: torch.Tensor,
                           block_tables: Optional[torch.Tensor], weights: torch.Tensor, seq_q: int, head_dim: int,
                           block_size: int, num_blocks: int, inv_sqrt_d: float, causal: bool, *, kv_group: int = 1,
                           q_first: Optional[torch.Tensor] = None, n_q: Optional[int] = None, decay: float = 1.0,
                           out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Adds the attention weight of every cached key, summed over a window of query rows.

    out[r, t] = decay * weights[r, t] + sum of softmax(q . k)[t] over the query rows of
    cache row r, for t < context_lens[r]; entries beyond are not written.  The weights are
    the forward's own (clamped softmax, causal: key t is seen by query row i when t <= i).
    Q, K_cache, context_lens, block_tables, seq_q and kv_group are the forward's.

    The window holds the query rows q_first[r] + i, i < n_q, of each of the row's kv_group
    query heads (q_first int32 [cache rows], default 0; n_q default seq_q); those outside
    [0, seq_q) do not count, so q_first = length - 64 with n_q = 64 takes the last 64 rows
    of every prompt, all rows of a shorter one.

    weights: float32 [cache rows, >= num_blocks * block_size]; out: as weights, weights
    itself by default.  Returns out.  The same inputs give the same bits."""
    name = "accumulate_key_weights"
    if not (head_dim in (128, 256)):
        _refuse(name, "head_dim must be 128 or 256")
    if not (context_lens.dtype is _I32):
        _refuse(name, "context_lens must be int32")
    n_kv = context_lens.numel()
    if not (n_kv <= _INT_MAX):
        _refuse(name, "too many cache rows")
    n_q = seq_q if n_q is None else n_q
    if not (1 <= kv_group <= _INT_MAX and 1 <= seq_q <= _INT_MAX and 1 <= n_q <= _INT_MAX):
        _refuse(name, "kv_group, seq_q and n_q must be >= 1 and fit int32")
    if not (block_size >= 1 and num_blocks >= 1 and block_size * num_blocks <= _INT_MAX):
        _refuse(name, "block_size and num_blocks must be >= 1, their product in int32")
    if not (abs(inv_sqrt_d) <= _F32_MAX and abs(decay) <= _F32_MAX):
        _refuse(name, "inv_sqrt_d and decay must be finite in float32")
    row_bytes = head_dim // 8
    if not (Q.numel() * Q.element_size() >= n_kv * kv_group * seq_q * row_bytes):
        _refuse(name, "Q smaller than its rows of head_dim/8 bytes")
    pool_rows, rest = divmod(K_cache.numel() * K_cache.element_size(), row_bytes)
    if rest or pool_rows == 0:
        _refuse(name, "K_cache must be [pool_rows, head_dim/32] words")
    out = weights if out is None else out
    shape = weights.shape
    if not (weights.dtype is _F32 and len(shape) == 2 and shape[0] == n_kv and shape[1] >= block_size * num_blocks):
        _refuse(name, "weights must be float32 [cache rows, >= num_blocks * block_size]")
    if not (out is weights or (out.dtype is _F32 and out.shape == shape)):
        _refuse(name, "out must be float32 of the shape of weights")
    if not (q_first is None or (q_first.dtype is _I32 and q_first.numel() == n_kv)):
        _refuse(name, "q_first must be int32 [cache rows]")
    bt, bt_numel = _tables(name, block_tables)
    if not (bt_numel == 0 or bt_numel >= n_kv * num_blocks):
        _refuse(name, "block_tables numel < cache rows * num_blocks")
    dev = K_cache.device
    if out is not weights:
        _same_or_apart(name, "out", weights, out)
    _check_tensors(name, dev, "Q K_cache context_lens block_tables weights out q_first",
                   Q, K_cache, context_lens, block_tables, weights, out, q_first)
    if n_kv == 0:
        return out
    nbytes = _capi.lib.hyperion_key_weights_scratch_bytes(n_kv, kv_group, n_q, head_dim, block_size, num_blocks)
    buf, scratch = _scratch(dev, nbytes)
    args = _capi.pack_key_weights(
        Q.data_ptr(), K_cache.data_ptr(), pool_rows, context_lens.data_ptr(), bt, bt_numel, n_kv,
        kv_group, seq_q, n_q, 0 if q_first is None else q_first.data_ptr(), head_dim, block_size, num_blocks,
        1 if causal else 0, inv_sqrt_d, decay, weights.data_ptr(), out.data_ptr(), shape[1],
        scratch, nbytes)
    _call(name, _capi.lib.hyperion_accumulate_key_weights, args, dev)
    return out


def evict_keys(K_cache: torch.Tensor, V_cache: torch.Tensor, context_lens: torch.Tensor,
               block_tables: Optional[torch.Tensor], block_size: int, num_blocks: int, weights: torch.Tensor,
               positions: torch.Tensor, keep: Union[int, torch.Tensor], *, sink: int = 0, recent: int = 0,
               V_scale: Optional[torch.Tensor] = None, context_lens_out: Optional[torch.Tensor] = None,
               weights_out: Optional[torch.Tensor] = None,
               positions_out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Cuts every cache row to its budget, in place.

    Of the n = context_lens[r] keys of row r the m = min(n, keep) highest-ranked stay
    (keep: an int, or int32 [cache rows]).  Keys at a position below `sink` or among the
    last `recent` positions up to the row's newest rank above all others; the others rank
    by weights (float32 [cache rows, >= num_blocks * block_size], the sums of
    accumulate_key_weights; NaN lowest); equal ranks go to the lower slot, also among more
    protected keys than the budget holds.

    Slots are not shifted: the i-th slot below m whose key goes takes the i-th kept key at
    or beyond m, so a step that drops one key moves at most one.  K words, V codes, the
    per-slot V_scale where one is given (float32 [pool rows]; other scales do not move),
    weights and positions (int32, as weights: each slot's position, as rope_cache_write's
    slot_positions) move together.  Slots m <= t < n end with weight 0 and position -1,
    ready for the next keys.  Pages beyond ceil(m / block_size) of a row are free to go.

    The new lengths, weights and positions go to the *_out tensors, by default the inputs
    themselves.  Returns the new lengths (context_lens_out).  Rows must not share pages."""
    name = "evict_keys"
    if not (V_cache.element_size() == 1 and V_cache.dim() == 2 and V_cache.shape[1] in (128, 256) and V_cache.shape[0] > 0):
        _refuse(name, "V_cache must hold one byte per element, [pool_rows, head_dim] with head_dim 128 or 256")
    pool_rows, head_dim = V_cache.shape
    if not (K_cache.numel() * K_cache.element_size() >= pool_rows * head_dim // 8):
        _refuse(name, "K_cache smaller than pool_rows rows of head_dim/8 bytes")
    if not (context_lens.dtype is _I32):
        _refuse(name, "context_lens must be int32")
    n_kv = context_lens.numel()
    if not (n_kv <= _INT_MAX):
        _refuse(name, "too many cache rows")
    if not (block_size >= 1 and num_blocks >= 1 and block_size * num_blocks <= _INT_MAX):
        _refuse(name, "block_size and num_blocks must be >= 1, their product in int32")
    ctx_out = context_lens if context_lens_out is None else context_lens_out
    w_out = weights if weights_out is None else weights_out
    p_out = positions if positions_out is None else positions_out
    if not (ctx_out.dtype is _I32 and ctx_out.numel() == n_kv):
        _refuse(name, "context_lens_out must be int32 [cache rows]")
    shape = weights.shape
    if not (weights.dtype is _F32 and w_out.dtype is _F32 and positions.dtype is _I32 and p_out.dtype is _I32
            and len(shape) == 2 and shape[0] == n_kv and shape[1] >= block_size * num_blocks
            and w_out.shape == shape and positions.shape == shape and p_out.shape == shape):
        _refuse(name, "weights and weights_out must be float32, positions and positions_out int32, all [cache rows, >= "
                "num_blocks * block_size] of one shape")
    keep_rows = keep if isinstance(keep, torch.Tensor) else None
    if keep_rows is not None:
        if not (keep.dtype is _I32 and keep.numel() == n_kv):
            _refuse(name, "keep must be an int or int32 [cache rows]")
    else:
        if not (keep >= 0):
            _refuse(name, "keep must be >= 0")
        keep = min(keep, _INT_MAX)
    if not (0 <= sink <= _INT_MAX and 0 <= recent <= _INT_MAX):
        _refuse(name, "sink and recent must be >= 0 and fit int32")
    if not (V_scale is None or (V_scale.dtype is _F32 and V_scale.numel() == pool_rows)):
        _refuse(name, "V_scale must be float32 [pool_rows], one scale per slot; other scales do not move")
    bt, bt_numel = _tables(name, block_tables)
    if not (bt_numel == 0 or bt_numel >= n_kv * num_blocks):
        _refuse(name, "block_tables numel < cache rows * num_blocks")
    if ctx_out is not context_lens:
        _same_or_apart(name, "context_lens_out", context_lens, ctx_out)
    if w_out is not weights:
        _same_or_apart(name, "weights_out", weights, w_out)
    if p_out is not positions:
        _same_or_apart(name, "positions_out", positions, p_out)
    dev = K_cache.device
    _check_tensors(name, dev, "K_cache V_cache context_lens block_tables weights positions keep V_scale context_lens_out "
                   "weights_out positions_out", K_cache, V_cache, context_lens, block_tables, weights, positions, keep_rows,
                   V_scale, ctx_out, w_out, p_out)
    if n_kv == 0:
        return ctx_out
    nbytes = _capi.lib.hyperion_evict_scratch_bytes(n_kv, block_size, num_blocks)
    buf, scratch = _scratch(dev, nbytes)
    args = _capi.pack_evict(
        K_cache.data_ptr(), V_cache.data_ptr(), 0 if V_scale is None else V_scale.data_ptr(), pool_rows, head_dim, n_kv,
        context_lens.data_ptr(), ctx_out.data_ptr(), bt, bt_numel, block_size, num_blocks, weights.data_ptr(),
        w_out.data_ptr(), positions.data_ptr(), p_out.data_ptr(), shape[1],
        0 if keep_rows is None else keep_rows.data_ptr(), 0 if keep_rows is not None else keep, sink, recent, scratch, nbytes)
    _call(name, _capi.lib.hyperion_evict_keys, args, dev)
    return ctx_out
