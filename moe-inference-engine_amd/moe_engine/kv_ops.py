"""Device-side KV append and gather through the HIP library.

These are the tensor operations under PagedKVCache.write / .read on a ROCm
device (reference: src/moe_engine/model.py:167-201).  Pools are the
allocator's [layers, blocks, heads, block_size, head_dim] tensors; the kernels
address one layer through `layer_idx`, the same view the reference takes with
k_pool[layer] (src/moe_engine/paged_attention.py:121-122).

For a serving step over a ragged batch, beyond the reference: reserve / release
(block tables, slots and positions from lengths on the device, blocks from a
device free list) and rope_append (rotary positions, k and v stored by slot).
paged_attention.extend_batched is the attention that goes with them.
"""

import math
from typing import NamedTuple

import torch

from moe_engine import _native


def _check_pools(k_pool: torch.Tensor, v_pool: torch.Tensor) -> None:
    if k_pool.shape != v_pool.shape or k_pool.dtype != v_pool.dtype:
        raise ValueError("K and V pools must share shape and dtype")
    if k_pool.dim() != 5:
        raise ValueError("pools are [layers, blocks, heads, block_size, head_dim]")
    if not (k_pool.is_contiguous() and v_pool.is_contiguous()):
        raise ValueError("pools must be contiguous")
    if not _native.is_rocm_device(k_pool):
        raise RuntimeError("the HIP KV kernels need pools on a ROCm device")


def _layer(pool: torch.Tensor, layer_idx: int) -> torch.Tensor:
    if not 0 <= layer_idx < pool.shape[0]:
        raise IndexError(f"layer {layer_idx} outside [0, {pool.shape[0]})")
    return pool[layer_idx]


def append(
    k_pool: torch.Tensor,
    v_pool: torch.Tensor,
    layer_idx: int,
    k_new: torch.Tensor,
    v_new: torch.Tensor,
    block_tables: torch.Tensor,
    position: int = 0,
    positions: torch.Tensor = None,
) -> None:
    """Scatter new rows k_new/v_new [B, H, S, D] into one layer of the pools.

    Row (b, s) lands at logical position pos_b + s of sequence b, where pos_b is
    positions[b] (device int32 [B]) or `position`.  block_tables is an int32
    device tensor [B, max_blocks] (or the 1-D per-sequence mirror for B == 1).
    One launch writes K and V.
    """
    _check_pools(k_pool, v_pool)
    lib = _native.lib()
    kl, vl = _layer(k_pool, layer_idx), _layer(v_pool, layer_idx)
    nb, heads, block_size, head_dim = kl.shape
    if k_new.dim() != 4 or k_new.shape != v_new.shape:
        raise ValueError("k_new and v_new must both be [batch, heads, seq, head_dim]")
    batch, h2, seq_len, d2 = k_new.shape
    if (h2, d2) != (heads, head_dim):
        raise ValueError(f"new rows have heads/head_dim {h2}/{d2}, pool has {heads}/{head_dim}")
    if k_new.dtype != kl.dtype or v_new.dtype != kl.dtype:
        raise ValueError(f"new rows are {k_new.dtype}, pool is {kl.dtype}")
    if k_new.device != kl.device or v_new.device != kl.device:
        raise ValueError("new rows and pools must be on the same device")
    if k_new.stride() != v_new.stride() or k_new.stride(3) != 1:
        k_new, v_new = k_new.contiguous(), v_new.contiguous()
    if block_tables.dtype != torch.int32 or block_tables.device != kl.device:
        raise ValueError("block tables must be int32 on the pool's device")
    if block_tables.dim() == 1:
        if batch != 1:
            raise ValueError("a 1-D block table serves one sequence")
        if block_tables.numel() < nb or not block_tables.is_contiguous():
            raise ValueError("a 1-D block table must be contiguous with one entry per pool block")
        bt_stride = 0
    else:
        if block_tables.shape[0] != batch or block_tables.stride(1) != 1:
            raise ValueError("block tables must be [batch, max_blocks] with unit inner stride")
        bt_stride = block_tables.stride(0)
    if positions is not None:
        if positions.dtype != torch.int32 or positions.shape != (batch,) or positions.device != kl.device:
            raise ValueError("positions must be an int32 device tensor [batch]")
        positions = positions.contiguous()
    _native.check(
        lib.mie_kv_append(
            kl.data_ptr(), vl.data_ptr(), kl.stride(0), kl.stride(1), nb,
            k_new.data_ptr(), v_new.data_ptr(), k_new.stride(0), k_new.stride(1), k_new.stride(2),
            block_tables.data_ptr(), bt_stride,
            _native.ptr(positions), int(position),
            batch, seq_len, heads, head_dim, block_size,
            _native.dtype_code(kl.dtype), _native.stream_of(kl),
        ),
        "mie_kv_append",
    )


def gather(
    k_pool: torch.Tensor,
    v_pool: torch.Tensor,
    layer_idx: int,
    block_table: torch.Tensor,
    length: int,
    out_k: torch.Tensor = None,
    out_v: torch.Tensor = None,
):
    """Copy tokens [0, length) of one sequence to contiguous K, V [1, H, length, D].

    Same result as the reference's pool[l, bt[:nb]].transpose(0, 1).reshape(...)
    (src/moe_engine/model.py:191-199), produced by one launch for K and V.
    """
    _check_pools(k_pool, v_pool)
    lib = _native.lib()
    kl, vl = _layer(k_pool, layer_idx), _layer(v_pool, layer_idx)
    nb, heads, block_size, head_dim = kl.shape
    if length < 0 or length > nb * block_size:
        raise ValueError(f"length {length} outside [0, {nb * block_size}]")
    if block_table.dtype != torch.int32 or block_table.dim() != 1 or block_table.device != kl.device:
        raise ValueError("block_table must be a 1-D int32 tensor on the pool's device")
    if not block_table.is_contiguous() or block_table.numel() < -(-length // block_size):
        raise ValueError("block_table must be contiguous and cover the gathered length")
    shape = (1, heads, length, head_dim)
    if out_k is None:
        out_k = torch.empty(shape, dtype=kl.dtype, device=kl.device)
    if out_v is None:
        out_v = torch.empty(shape, dtype=kl.dtype, device=kl.device)
    for out in (out_k, out_v):
        if out.shape != shape or out.dtype != kl.dtype or out.stride(3) != 1:
            raise ValueError(f"gather outputs must be {shape} {kl.dtype} with unit inner stride")
    if out_k.stride() != out_v.stride():
        raise ValueError("gather outputs must share strides")
    _native.check(
        lib.mie_kv_gather(
            kl.data_ptr(), vl.data_ptr(), kl.stride(0), kl.stride(1), nb,
            block_table.data_ptr(), length,
            out_k.data_ptr(), out_v.data_ptr(), out_k.stride(1), out_k.stride(2),
            heads, head_dim, block_size,
            _native.dtype_code(kl.dtype), _native.stream_of(kl),
        ),
        "mie_kv_gather",
    )
    return out_k, out_v


def qkv_append_supported(dim: int, dtype: torch.dtype) -> bool:
    """Whether mie_qkv_append is built for this model width and dtype."""
    if not _native.HAS_HIP or dtype not in (torch.float32, torch.bfloat16):
        return False
    return bool(_native.lib().mie_qkv_append_supported(int(dim), _native.dtype_code(dtype)))


def qkv_append(
    x: torch.Tensor,
    in_proj_weight: torch.Tensor,
    in_proj_bias: torch.Tensor,
    k_pool: torch.Tensor,
    v_pool: torch.Tensor,
    layer_idx: int,
    block_table: torch.Tensor,
    *,
    position: int = 0,
    position_dev: torch.Tensor = None,
    norm_weight: torch.Tensor = None,
    norm_bias: torch.Tensor = None,
    norm_eps: float = 1e-5,
    q_out: torch.Tensor = None,
) -> torch.Tensor:
    """QKV projection of one token with K and V stored into their pool slots.

    x holds one token's dim values (any shape of dim elements, contiguous);
    in_proj_weight [3*dim, dim] and in_proj_bias [3*dim] are the attention's
    packed projection (reference model.py:218-224); block_table is the
    sequence's 1-D int32 device table.  The token goes to logical position
    `position`, or to *position_dev (an int32 device [1]) when given.  With
    norm_weight the projection applies to LayerNorm(x) (the block's attn_norm).
    Returns q [1, heads, 1, head_dim] (written into q_out when given); the
    block for the position must already be reserved.
    """
    _check_pools(k_pool, v_pool)
    kl, vl = _layer(k_pool, layer_idx), _layer(v_pool, layer_idx)
    nb, heads, block_size, head_dim = kl.shape
    dim = heads * head_dim
    dtype = kl.dtype
    if x.numel() != dim or not x.is_contiguous():
        raise ValueError(f"x must hold {dim} contiguous values")
    if in_proj_weight.shape != (3 * dim, dim) or not in_proj_weight.is_contiguous():
        raise ValueError(f"in_proj_weight must be a contiguous [{3 * dim}, {dim}] matrix")
    if in_proj_bias is not None and (in_proj_bias.shape != (3 * dim,) or not in_proj_bias.is_contiguous()):
        raise ValueError(f"in_proj_bias must be a contiguous [{3 * dim}] vector")
    norm = [t for t in (norm_weight, norm_bias) if t is not None]
    if norm_bias is not None and norm_weight is None:
        raise ValueError("a norm bias needs a norm weight")
    for t in norm:
        if t.shape != (dim,) or not t.is_contiguous():
            raise ValueError(f"norm parameters must be contiguous [{dim}] vectors")
    params = [x, in_proj_weight, *([in_proj_bias] if in_proj_bias is not None else []), *norm]
    if any(t.dtype != dtype or t.device != kl.device for t in params):
        raise ValueError("x, the projection and norm parameters must match the pools' dtype and device")
    if not qkv_append_supported(dim, dtype):
        raise RuntimeError(f"mie_qkv_append is not built for dim {dim} in {dtype}")
    if block_table.dtype != torch.int32 or block_table.dim() != 1 or block_table.device != kl.device:
        raise ValueError("block_table must be a 1-D int32 tensor on the pool's device")
    if not block_table.is_contiguous():
        raise ValueError("block_table must be contiguous")
    if position_dev is not None:
        if position_dev.dtype != torch.int32 or position_dev.numel() != 1 or position_dev.device != kl.device:
            raise ValueError("position_dev must be an int32 device tensor of one element")
    elif not 0 <= position < block_table.numel() * block_size:
        raise ValueError(f"position {position} outside the block table's {block_table.numel() * block_size} slots")
    if q_out is None:
        q_out = torch.empty((1, heads, 1, head_dim), dtype=dtype, device=kl.device)
    elif q_out.numel() != dim or not q_out.is_contiguous() or q_out.dtype != dtype:
        raise ValueError(f"q_out must hold {dim} contiguous {dtype} values")
    _native.check(
        _native.lib().mie_qkv_append(
            x.data_ptr(), _native.ptr(norm_weight), _native.ptr(norm_bias), float(norm_eps),
            in_proj_weight.data_ptr(), _native.ptr(in_proj_bias), dim,
            kl.data_ptr(), vl.data_ptr(), kl.stride(0), kl.stride(1), nb,
            block_table.data_ptr(), block_table.numel(), _native.ptr(position_dev), int(position),
            q_out.data_ptr(), heads, head_dim, block_size,
            _native.dtype_code(dtype), _native.stream_of(kl),
        ),
        "mie_qkv_append",
    )
    return q_out.view(1, heads, 1, head_dim)


# ---- a serving step over a ragged batch ----------------------------------------


def take_free_blocks(allocator, count: int = None):
    """Hand `count` of a BlockAllocator's free blocks (default: all) to the
    device: (free_ids int32 [count], free_count int32 [1]), a stack whose top
    is the block the allocator would have given next.  The blocks leave the
    host's list, so no PagedKVCache gets them; allocator.free(free_ids[:n]
    .tolist()) with n = int(free_count) takes back those that are free."""
    count = len(allocator.free_blocks) if count is None else int(count)
    if not 1 <= count <= len(allocator.free_blocks):
        raise ValueError(f"count {count} outside [1, {len(allocator.free_blocks)}], the free blocks")
    ids = torch.tensor(allocator.free_blocks[-count:], dtype=torch.int32, device=allocator.k_pool.device)
    del allocator.free_blocks[-count:]
    return ids, torch.full((1,), count, dtype=torch.int32, device=ids.device)


class StepSlots(NamedTuple):
    """What reserve returns, all on the device: the packed tokens' starts
    [B + 1], slots (int64) and positions [max_tokens], the lengths [B] and the
    free blocks [1] after the step, and the status [1] (0, or why nothing was
    reserved: RESERVE_STATUS)."""

    starts: torch.Tensor
    slots: torch.Tensor
    positions: torch.Tensor
    context_lens: torch.Tensor
    free_count: torch.Tensor
    status: torch.Tensor


class StepRelease(NamedTuple):
    """What release returns, all on the device: the free blocks [1] and the
    lengths [B] after it, and the status [1] (0, or why nothing was released)."""

    free_count: torch.Tensor
    context_lens: torch.Tensor
    status: torch.Tensor


# enum of the status words
RESERVE_STATUS = {
    0: "ok",
    1: "not enough free blocks (release: the free list is full)",
    2: "a sequence outgrows its block table",
    3: "more than max_tokens new tokens",
    4: "a negative length, or a free count outside the list",
}


def _check_step(free_ids, free_count, block_tables, context_lens, block_size):
    device = free_ids.device
    if not _native.is_rocm_device(free_ids):
        raise RuntimeError("the HIP step kernels need tensors on a ROCm device")
    if block_tables.dim() != 2 or block_tables.dtype != torch.int32 or block_tables.device != device \
            or block_tables.stride(1) != 1 or (block_tables.shape[0] > 1
                                               and block_tables.stride(0) < block_tables.shape[1]):
        raise ValueError("block tables must be int32 [batch, max_blocks] rows on the free list's device")
    batch = block_tables.shape[0]
    for name, t, n in (("free_ids", free_ids, free_ids.numel()), ("free_count", free_count, 1),
                       ("context_lens", context_lens, batch)):
        if t.dtype != torch.int32 or t.dim() != 1 or t.numel() != n or t.device != device or not t.is_contiguous():
            raise ValueError(f"{name} must be {n} contiguous int32 values on the free list's device")
    if not 1 <= int(block_size) < 1 << 31 or free_ids.numel() > 1 << 30:
        raise ValueError(f"block_size {block_size}, {free_ids.numel()} free ids (at most 2^30)")
    return batch, device


def reserve(
    free_ids: torch.Tensor,
    free_count: torch.Tensor,
    block_tables: torch.Tensor,
    context_lens: torch.Tensor,
    new_lens: torch.Tensor,
    block_size: int,
    max_tokens: int,
) -> StepSlots:
    """Reserve a step's blocks on the device, in one launch and without the
    host reading a length.

    free_ids int32 [capacity] with the top of the stack at free_count[0] - 1;
    block_tables int32 [B, max_blocks] (new blocks are written in place);
    context_lens and new_lens int32 [B] (0 new tokens: the row takes no part).
    The step's tokens are packed sequence after sequence into max_tokens
    places; those past the last get slot -1 and position 0.  Blocks come off
    the stack in the order a host allocator would give them, sequence after
    sequence.

    All or nothing, as PagedKVCache's reservation is; the host is not told
    unless it reads `status`: on a failure no table entry is written, starts
    are all 0 and slots -1, so that the step's other operators do nothing, and
    the lengths and the free count come back unchanged.  The inputs are not
    advanced: carry context_lens and free_count to the next call.
    """
    host = _native.HOST
    if host is not None and free_ids.is_cuda:
        # The usual form in one compiled call; None for any other, which the
        # checks below take (or refuse).
        got = _native.host_result(host.reserve(free_ids, free_count, block_tables, context_lens, new_lens, block_size,
                                               max_tokens, _native.stream_of(free_ids)), "mie_step_reserve")
        if got is not None:
            return StepSlots(*got)
    batch, device = _check_step(free_ids, free_count, block_tables, context_lens, block_size)
    if new_lens.dtype != torch.int32 or new_lens.shape != (batch,) or new_lens.device != device \
            or not new_lens.is_contiguous():
        raise ValueError(f"new_lens must be {batch} contiguous int32 values on the free list's device")
    max_tokens = int(max_tokens)
    if not 0 <= max_tokens <= 1 << 30:
        raise ValueError(f"max_tokens {max_tokens} outside [0, 2^30]")
    word = dict(dtype=torch.int32, device=device)
    starts, positions = torch.empty(batch + 1, **word), torch.empty(max_tokens, **word)
    slots = torch.empty(max_tokens, dtype=torch.int64, device=device)
    lens, count, status = torch.empty(batch, **word), torch.empty(1, **word), torch.empty(1, **word)
    with _native.on_device_of(free_ids):
        _native.check(
            _native.lib().mie_step_reserve(
                free_ids.data_ptr(), free_ids.numel(), free_count.data_ptr(),
                block_tables.data_ptr(), max(block_tables.stride(0), block_tables.shape[1]), block_tables.shape[1],
                context_lens.data_ptr(), new_lens.data_ptr(), batch, int(block_size), max_tokens,
                starts.data_ptr(), slots.data_ptr(), positions.data_ptr(),
                lens.data_ptr(), count.data_ptr(), status.data_ptr(), _native.stream_of(free_ids),
            ),
            "mie_step_reserve",
        )
    return StepSlots(starts, slots, positions, lens, count, status)


def release(
    free_ids: torch.Tensor,
    free_count: torch.Tensor,
    block_tables: torch.Tensor,
    context_lens: torch.Tensor,
    finished: torch.Tensor,
    block_size: int,
) -> StepRelease:
    """Put the blocks of finished sequences (bool [B]) back on the stack, in
    table order, sequence after sequence (PagedKVCache.free's order), in one
    launch: free_ids is written from free_count[0] on, finished sequences'
    lengths become 0.  All or nothing, like reserve.  Each sequence's blocks
    must be its own."""
    host = _native.HOST
    if host is not None and free_ids.is_cuda:
        got = _native.host_result(host.release(free_ids, free_count, block_tables, context_lens, finished, block_size,
                                               _native.stream_of(free_ids)), "mie_step_release")
        if got is not None:
            return StepRelease(*got)
    batch, device = _check_step(free_ids, free_count, block_tables, context_lens, block_size)
    if finished.dtype != torch.bool or finished.shape != (batch,) or finished.device != device \
            or not finished.is_contiguous():
        raise ValueError(f"finished must be {batch} contiguous bool values on the free list's device")
    word = dict(dtype=torch.int32, device=device)
    lens, count, status = torch.empty(batch, **word), torch.empty(1, **word), torch.empty(1, **word)
    with _native.on_device_of(free_ids):
        _native.check(
            _native.lib().mie_step_release(
                free_ids.data_ptr(), free_ids.numel(), free_count.data_ptr(),
                block_tables.data_ptr(), max(block_tables.stride(0), block_tables.shape[1]), block_tables.shape[1],
                context_lens.data_ptr(), finished.data_ptr(), batch, int(block_size),
                lens.data_ptr(), count.data_ptr(), status.data_ptr(), _native.stream_of(free_ids),
            ),
            "mie_step_release",
        )
    return StepRelease(count, lens, status)


ROPE_SCALINGS = (None, "linear", "ntk", "yarn")


def rope_frequencies(rotary_dim: int, base: float = 10000.0, *, scaling: str = None, scale: float = 1.0,
                     original_length: int = None, beta_fast: float = 32.0, beta_slow: float = 1.0, device=None):
    """(frequencies float64 [rotary_dim / 2] in radians per position, factor)
    for rope_append.  Pair i turns by base ** (-2 i / rotary_dim); for contexts
    `scale` times the trained one:

      "linear"  every frequency divided by scale (positions interpolated);
      "ntk"     base times scale ** (rotary_dim / (rotary_dim - 2)): the slowest
                pair is interpolated, the fastest is not;
      "yarn"    pairs that turn more than beta_fast times within
                original_length positions stay, those that turn less than
                beta_slow times are divided by scale, a linear ramp over the
                pairs between; factor = 0.1 log(scale) + 1.
    """
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be even and positive, not {rotary_dim}")
    if scaling not in ROPE_SCALINGS:
        raise ValueError(f"unknown scaling {scaling!r}")
    if not (base > 1 and math.isfinite(base) and scale >= 1 and math.isfinite(scale)):
        raise ValueError(f"base {base} must be above 1 and scale {scale} at least 1")
    if scaling == "ntk":
        if rotary_dim == 2:
            raise ValueError("ntk scaling needs more than one pair")
        base = base * scale ** (rotary_dim / (rotary_dim - 2))
    steps = torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim
    freq, factor = torch.pow(torch.tensor(base, dtype=torch.float64), -steps), 1.0
    if scaling == "linear":
        freq = freq / scale
    elif scaling == "yarn":
        if not original_length or original_length < 1:
            raise ValueError("yarn scaling needs original_length")
        if not beta_fast > beta_slow > 0:
            raise ValueError("yarn scaling needs beta_fast > beta_slow > 0")

        def pair_turning(turns):
            return rotary_dim * math.log(original_length / (turns * 2 * math.pi)) / (2 * math.log(base))

        low = max(math.floor(pair_turning(beta_fast)), 0)
        high = min(math.ceil(pair_turning(beta_slow)), rotary_dim - 1)
        pair = torch.arange(rotary_dim // 2, dtype=torch.float64)
        ramp = ((pair - low) / max(high - low, 1e-3)).clamp(0, 1)
        freq = freq / scale * ramp + freq * (1 - ramp)
        factor = 0.1 * math.log(scale) + 1.0
    return freq.to(device) if device is not None else freq, factor


def rope_append(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    k_pool: torch.Tensor,
    v_pool: torch.Tensor,
    layer_idx: int,
    slots: torch.Tensor,
    positions: torch.Tensor,
    frequencies: torch.Tensor,
    *,
    interleaved: bool = False,
    factor: float = 1.0,
    out: torch.Tensor = None,
) -> torch.Tensor:
    """Rotary positions for a step's packed tokens: q [T, H, D] rotated into a
    new tensor (or `out`, which may be q), k [T, H_kv, D] rotated and v as it
    is stored into one layer of the pools at slots (int64 [T], as reserve gives
    them; outside the pool: not stored).  One launch.

    positions int32 [T]; frequencies float64 [R / 2] on the device, radians per
    position (rope_frequencies); dims from R on are copied.  Pairs are dims
    (i, i + R / 2), or (2 i, 2 i + 1) with `interleaved`; rotated values are
    multiplied by `factor`.  H_kv and D are the pool's; D and R are even.
    Two tokens must not share a slot.
    """
    host = _native.HOST
    if host is not None and out is None and q.is_cuda:
        got = _native.host_result(host.rope_append(q, k, v, k_pool, v_pool, layer_idx, slots, positions, frequencies,
                                                   interleaved, factor, _native.stream_of(q)), "mie_rope_append")
        if got is not None:
            return got
    _check_pools(k_pool, v_pool)
    kl, vl = _layer(k_pool, layer_idx), _layer(v_pool, layer_idx)
    nb, kv_heads, block_size, head_dim = kl.shape
    if q.dim() != 3 or k.dim() != 3 or q.shape[2] != head_dim or k.shape[1:] != (kv_heads, head_dim) \
            or k.shape[0] != q.shape[0] or v.shape != k.shape:
        raise ValueError(f"q must be [tokens, heads, {head_dim}], k and v [tokens, {kv_heads}, {head_dim}]")
    tokens, heads = q.shape[0], q.shape[1]
    dtype, device = kl.dtype, kl.device
    if any(t.dtype != dtype or t.device != device for t in (q, k, v)):
        raise ValueError(f"q, k and v must be {dtype} on the pools' device")
    if slots.dtype != torch.int64 or slots.shape != (tokens,) or slots.device != device or not slots.is_contiguous():
        raise ValueError(f"slots must be {tokens} contiguous int64 values on the pools' device")
    if positions.dtype != torch.int32 or positions.shape != (tokens,) or positions.device != device \
            or not positions.is_contiguous():
        raise ValueError(f"positions must be {tokens} contiguous int32 values on the pools' device")
    if frequencies.dtype != torch.float64 or frequencies.dim() != 1 or frequencies.device != device \
            or not frequencies.is_contiguous():
        raise ValueError("frequencies must be a contiguous float64 vector on the pools' device")
    _native.refuse_gradients("rope_append", q, k, v, frequencies)
    if q.stride(2) != 1:
        q = q.contiguous()
    if k.stride(2) != 1 or k.stride() != v.stride():
        k, v = k.contiguous(), v.contiguous()
    if out is None:
        out = torch.empty((tokens, heads, head_dim), dtype=dtype, device=device)
    elif out.shape != q.shape or out.dtype != dtype or out.device != device or out.stride(2) != 1 \
            or (tokens > 1 and heads > 0 and out.stride(0) < head_dim) or (heads > 1 and out.stride(1) < head_dim):
        raise ValueError(f"out must be {tuple(q.shape)} {dtype} rows on the pools' device")
    with _native.on_device_of(q):
        _native.check(
            _native.lib().mie_rope_append(
                q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), v.data_ptr(), k.stride(0), k.stride(1),
                kl.data_ptr(), vl.data_ptr(), kl.stride(0), kl.stride(1), nb,
                slots.data_ptr(), positions.data_ptr(), frequencies.data_ptr(), 2 * frequencies.numel(),
                bool(interleaved), float(factor), tokens, heads, kv_heads, head_dim, block_size,
                out.data_ptr(), out.stride(0), out.stride(1), _native.dtype_code(dtype), _native.stream_of(q),
            ),
            "mie_rope_append",
        )
    return out
