"""The 4-bit MLA cache on sm_100a: writer, read-back and attention.

``fp4_ds_mla`` is ``fp8_ds_mla`` with 4-bit latents, 416 instead of 656 bytes a
token (no reference counterpart; the entry points stand beside the fp8 ones of
``cache_writer``, ``fp8_dequant`` and ``fp8_ds_mla_sparse_decode``):

    [  0:256)  512 x e2m1    NoPE latent, element 2i in the low nibble of byte i
    [256:288)   32 x e4m3    one scale per 16 latent values
    [288:416)   64 x bf16    RoPE, stored raw

A latent value is ``code * scale``: exact in bf16 (6 significant bits at most).
The writer's rule per group of 16: ``scale = e4m3(amax / 6)`` within
[2^-9, 448], ``code = e2m1(x / scale)``, both to nearest even, the code
saturating at 6 (values beyond +-2688 are held as +-2688); a group with a NaN
reads back as NaN.

* ``concat_and_cache_fp4_ds_mla``     tokens into their slots
* ``dequant_fp4_ds_mla_rows``         rows by slot, as bf16
* ``gather_fp4_ds_mla``               whole sequences through the block table, as
                                      bf16 (prefill over a cached context)
* ``fp4_ds_mla_sparse_decode``        attention over top-k slots
* ``fp4_ds_mla_sparse_decode_paged``  the same over request-local positions
* ``fp4_ds_mla_decode``               attention over whole contexts

The attention takes bf16 q only: the latents enter the tensor cores exactly (as
fp16, beside q in fp16, scaled by a power of two per head), the softmax's weights in fp16 (11 bits;
below 2^-20 of a row's largest with an error of up to 2^-31 of it, so that those
below 2^-31 count as 0), sums in fp32.  All calls
run on the current stream of the tensors' device and never synchronise.
"""

from __future__ import annotations

import torch

from vllm_fp8kv import _native as N

NOPE = 512
ROPE = 64
GROUP = 16             # latent values per scale
ROW_BYTES = 416
SCALE_OFF = 256
ROPE_OFF = 288


def _pool(kv_cache: torch.Tensor) -> int:
    """Checks a pool; its number of slots."""
    assert kv_cache.dtype == torch.uint8, f"an fp4_ds_mla pool is uint8, got {kv_cache.dtype}"
    assert kv_cache.is_contiguous(), "kv_cache must be contiguous"
    assert kv_cache.dim() >= 2 and kv_cache.shape[-1] == ROW_BYTES, "fp4_ds_mla rows are 416 bytes"
    return kv_cache.numel() // ROW_BYTES


def _launch(what: str, fn: str, dev, *args) -> None:
    """Calls C entry `fn` on the tensors' device and its current stream (entering
    the device's context, where it is current already, costs more than the look)."""
    call = getattr(N.lib(), fn)
    if torch.cuda.current_device() == dev.index:
        rc = call(*args, N.raw_stream(dev))
    else:
        with torch.cuda.device(dev):
            rc = call(*args, N.raw_stream(dev))
    if rc:
        N.check(rc, what)


def _int64(t: torch.Tensor) -> torch.Tensor:
    return t if t.dtype == torch.int64 and t.is_contiguous() else t.to(torch.int64).contiguous()


def concat_and_cache_fp4_ds_mla(kv_c: torch.Tensor, k_pe: torch.Tensor, kv_cache: torch.Tensor,
                                slot_mapping: torch.Tensor) -> None:
    """Quantize kv_c [N, 512] and k_pe [N, 64] (bf16) into the kv_cache [..., 416]
    rows that slot_mapping [N] names; slots below 0 or behind the pool are skipped.
    A slot must not be named twice (its row could hold parts of both tokens)."""
    assert kv_c.dtype == torch.bfloat16 and k_pe.dtype == torch.bfloat16, "bf16 latent/rope"
    assert kv_c.dim() == 2 and kv_c.shape[1] == NOPE and kv_c.stride(1) == 1
    assert k_pe.dim() == 2 and k_pe.shape[1] == ROPE and k_pe.stride(1) == 1
    assert slot_mapping.dim() == 1 and kv_c.shape[0] == k_pe.shape[0] == slot_mapping.shape[0]
    num_slots = _pool(kv_cache)
    dev = N.require_cuda(kv_c, k_pe, kv_cache, slot_mapping)
    # one token's stride is never used, but a view's may be anything
    st_c = kv_c.stride(0) if kv_c.shape[0] > 1 else NOPE
    st_pe = k_pe.stride(0) if k_pe.shape[0] > 1 else ROPE
    assert st_c >= NOPE and st_pe >= ROPE, "token rows must not overlap"
    slots = _int64(slot_mapping)
    _launch("concat_and_cache_fp4_ds_mla", "fp8mla_fp4_write", dev, kv_c.data_ptr(), st_c, k_pe.data_ptr(), st_pe,
            slots.data_ptr(), slots.shape[0], kv_cache.data_ptr(), num_slots)


def _check_out(out: torch.Tensor | None, n: int, like: torch.Tensor) -> torch.Tensor:
    if out is None:
        return like.new_empty((n, NOPE + ROPE), dtype=torch.bfloat16)
    assert out.dtype == torch.bfloat16 and out.dim() == 2 and out.shape == (n, NOPE + ROPE) and out.stride(1) == 1, \
        f"out must be bf16 [{n}, {NOPE + ROPE}] with unit last stride"
    return out


def _row_stride(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else NOPE + ROPE


def dequant_fp4_ds_mla_rows(kv_cache: torch.Tensor, slots: torch.Tensor,
                            out: torch.Tensor | None = None) -> torch.Tensor:
    """bf16 [n, 576] rows (latent, rope) of slots [n]; slots outside the pool
    give zero rows.  `out`: a bf16 [n, 576] tensor to fill (16-byte aligned rows)."""
    num_slots = _pool(kv_cache)
    assert slots.dim() == 1 and slots.dtype in (torch.int32, torch.int64), "slots must be int32 or int64 [n]"
    dev = N.require_cuda(kv_cache, slots, out)
    sl = _int64(slots)
    out = _check_out(out, sl.numel(), kv_cache)
    _launch("dequant_fp4_ds_mla_rows", "fp8mla_fp4_dequant_rows", dev, kv_cache.data_ptr(), num_slots,
            sl.data_ptr(), sl.numel(), out.data_ptr(), _row_stride(out))
    return out


def gather_fp4_ds_mla(kv_cache: torch.Tensor, block_table: torch.Tensor, cu_seq_lens: torch.Tensor, num_tokens: int,
                      block_size: int = 64, seq_starts: torch.Tensor | None = None,
                      out: torch.Tensor | None = None) -> torch.Tensor:
    """Whole sequences as bf16 [num_tokens, 576] rows.

    Row r of sequence b (cu_seq_lens[b] <= r < cu_seq_lens[b + 1]) is position
    seq_starts[b] + r - cu_seq_lens[b] of it; block_table [B, max_blocks] int32
    holds its pages.  Positions behind the table, or on pages outside the pool,
    give zero rows.  num_tokens, the rows of `out`, is cu_seq_lens[-1]; where it is
    more, the rows behind the last sequence are left as they were (whatever the
    allocator gave, without `out`)."""
    num_slots = _pool(kv_cache)
    assert block_table.dtype == torch.int32 and block_table.dim() == 2, "block_table [B, max_blocks] int32"
    assert block_table.shape[1] == 0 or block_table.stride(1) == 1, "block_table rows must be unit-strided"
    B = block_table.shape[0]
    assert cu_seq_lens.dtype == torch.int32 and cu_seq_lens.shape == (B + 1,) and cu_seq_lens.is_contiguous(), \
        "cu_seq_lens must be contiguous int32 [B + 1]"
    assert seq_starts is None or (seq_starts.dtype == torch.int32 and seq_starts.shape == (B,)
                                  and seq_starts.is_contiguous()), "seq_starts must be contiguous int32 [B]"
    assert block_size > 0 and num_tokens >= 0
    dev = N.require_cuda(kv_cache, block_table, cu_seq_lens, seq_starts, out)
    out = _check_out(out, num_tokens, kv_cache)
    bt_stride = block_table.stride(0) if B > 1 else block_table.shape[1]
    assert bt_stride >= block_table.shape[1], "block_table rows must not overlap"
    _launch("gather_fp4_ds_mla", "fp8mla_fp4_gather", dev, kv_cache.data_ptr(), num_slots, block_table.data_ptr(),
            bt_stride, block_table.shape[1], int(block_size), cu_seq_lens.data_ptr(), B, seq_starts.data_ptr() if
            seq_starts is not None else None, num_tokens, out.data_ptr(), _row_stride(out))
    return out


def fp4_workspace_bytes(T: int, H: int, G: int = 1, topk: int = -1) -> int:
    """Device workspace one attention call needs (0 where no unit is cut); topk -1:
    the most any call of T tokens needs, whole contexts included."""
    return int(N.lib().fp8mla_fp4_workspace_bytes(T, H, G, topk))


def fp4_kernel_name(H: int, G: int = 1, T: int = 1, topk: int = -1) -> str:
    """The attention kernel that a call with H query heads in G kv groups takes
    (introspection); topk -1: whole contexts."""
    return N.lib().fp8mla_fp4_kernel_name(T, H, G, topk).decode()


def _prepare(q, kv_cache, groups, topk, return_lse, workspace, *others):
    """Checks shared by the attention calls; q in 16-byte rows, the pool's slots,
    out, lse, workspace and the pointers' device."""
    num_slots = _pool(kv_cache)
    assert q.dtype == torch.bfloat16, f"rope is stored bf16; q must be bf16, got {q.dtype}"
    assert q.dim() == 3 and q.shape[2] == NOPE + ROPE, f"q must be [T, H, {NOPE + ROPE}], got {tuple(q.shape)}"
    assert q.stride(-1) == 1, "need unit last-dim strides"
    T, H, _ = q.shape
    assert H % groups == 0, f"h_q={H} not divisible by kv_groups={groups}"
    dev = N.require_cuda(q, kv_cache, workspace, *others)
    # the kernels read q in 16-byte vectors; re-lay a misaligned view once
    # (a dimension of one token or head may have any stride, and contiguous() keeps it)
    st, sh, _ = q.stride()
    if q.data_ptr() % 16 or (st % 8 and T > 1) or (sh % 8 and H > 1):
        q = q.contiguous()
        if q.data_ptr() % 16:
            q = q.clone()
        st, sh, _ = q.stride()
    q_strides = (st if T > 1 else H * (NOPE + ROPE), sh if H > 1 else NOPE + ROPE)
    out = q.new_empty((T, H, NOPE))
    lse = q.new_empty((T, H), dtype=torch.float32) if return_lse else None
    need = N.lib().fp8mla_fp4_workspace_bytes(T, H, groups, topk)
    if workspace is not None:
        assert workspace.is_contiguous(), "workspace must be contiguous"
        if workspace.numel() * workspace.element_size() < need or workspace.data_ptr() % 32:
            workspace = None
    if workspace is None and need:
        workspace = q.new_empty((need,), dtype=torch.uint8)
    ws = (workspace.data_ptr(), workspace.numel() * workspace.element_size()) if workspace is not None else (None, 0)
    return T, H, q, q_strides, num_slots, out, lse, (lse.data_ptr(), H) if return_lse else (None, 0), ws, workspace, dev


def _check_table(req_id, block_table, T, block_size):
    assert req_id.dtype == torch.int32 and block_table.dtype == torch.int32, "int32 tables"
    assert req_id.dim() == 1 and req_id.shape[0] == T and req_id.is_contiguous(), "req_id [T], contiguous"
    assert block_table.dim() == 2 and (block_table.shape[1] == 0 or block_table.stride(1) == 1), \
        "block_table [reqs, max_blocks] with unit-strided rows"
    assert block_size > 0
    stride = block_table.stride(0) if block_table.shape[0] > 1 else block_table.shape[1]
    assert stride >= block_table.shape[1], "block_table rows must not overlap"
    return stride


def _with_groups(indices):
    assert indices.dtype == torch.int32, f"indices must be int32, got {indices.dtype}"
    assert indices.dim() in (2, 3), "indices must be [T, topk] or [T, kv_groups, topk]"
    assert indices.shape[-1] == 0 or indices.stride(-1) == 1, "need unit last-dim strides"
    return indices.unsqueeze(1) if indices.dim() == 2 else indices


def fp4_ds_mla_sparse_decode(
    q: torch.Tensor,            # [T, H, 576] bf16
    kv_cache: torch.Tensor,     # [..., 416] uint8, contiguous
    indices: torch.Tensor,      # [T, kv_groups, topk] or [T, topk] int32 flat slots; -1 = masked
    sm_scale: float,
    return_lse: bool = False,
    *,
    workspace: torch.Tensor | None = None,
):
    """Sparse MLA attention over fp4_ds_mla rows named by flat slot.

    As ``fp8_ds_mla_sparse_decode``: entries < 0 or outside the pool are masked;
    returns ``out`` [T, H, 512] bf16, plus the natural-log ``lse`` [T, H] fp32
    when ``return_lse`` (-inf, and a zero row, where nothing is attended).
    ``workspace``: a uint8 tensor of ``fp4_workspace_bytes``, 32-byte aligned, to
    use (one that does not fit is replaced)."""
    indices = _with_groups(indices)
    G, topk = indices.shape[1], indices.shape[2]
    assert indices.shape[0] == q.shape[0], "one index row per query token"
    T, H, q, q_strides, num_slots, out, lse, lse_at, ws, hold, dev = _prepare(
        q, kv_cache, G, topk, return_lse, workspace, indices)
    _launch("fp4_ds_mla_sparse_decode", "fp8mla_fp4_sparse_decode", dev, q.data_ptr(), T, H, *q_strides,
            kv_cache.data_ptr(), num_slots, indices.data_ptr(), G, topk, indices.stride(0), indices.stride(1),
            float(sm_scale), out.data_ptr(), H * NOPE, NOPE, *lse_at, *ws)
    return (out, lse) if return_lse else out


def fp4_ds_mla_sparse_decode_paged(
    q: torch.Tensor,              # [T, H, 576] bf16
    kv_cache: torch.Tensor,       # [num_blocks, block_size, 416] uint8, contiguous
    req_id: torch.Tensor,         # [T] int32: request of each query token
    block_table: torch.Tensor,    # [num_reqs, max_blocks] int32 page ids
    token_indices: torch.Tensor,  # [T, kv_groups, topk] or [T, topk] int32 positions; -1 = masked
    sm_scale: float,
    block_size: int = 64,
    return_lse: bool = False,
    *,
    workspace: torch.Tensor | None = None,
):
    """``fp4_ds_mla_sparse_decode`` over request-local token positions: the
    block-table conversion runs inside the gather (positions behind the table,
    and all of a token with a negative req_id, are masked)."""
    token_indices = _with_groups(token_indices)
    G, topk = token_indices.shape[1], token_indices.shape[2]
    assert token_indices.shape[0] == q.shape[0], "one index row per query token"
    bt_stride = _check_table(req_id, block_table, q.shape[0], block_size)
    T, H, q, q_strides, num_slots, out, lse, lse_at, ws, hold, dev = _prepare(
        q, kv_cache, G, topk, return_lse, workspace, token_indices, req_id, block_table)
    _launch("fp4_ds_mla_sparse_decode_paged", "fp8mla_fp4_sparse_decode_paged", dev, q.data_ptr(), T, H, *q_strides,
            kv_cache.data_ptr(), num_slots, req_id.data_ptr(), block_table.data_ptr(), bt_stride,
            block_table.shape[1], int(block_size), token_indices.data_ptr(), G, topk, token_indices.stride(0),
            token_indices.stride(1), float(sm_scale), out.data_ptr(), H * NOPE, NOPE, *lse_at, *ws)
    return (out, lse) if return_lse else out


def fp4_ds_mla_decode(
    q: torch.Tensor,             # [T, H, 576] bf16
    kv_cache: torch.Tensor,      # [num_blocks, block_size, 416] uint8, contiguous
    req_id: torch.Tensor,        # [T] int32: request of each query token
    block_table: torch.Tensor,   # [num_reqs, max_blocks] int32 page ids
    context_lens: torch.Tensor,  # [T] int32: positions each query token attends to
    sm_scale: float,
    block_size: int = 64,
    return_lse: bool = False,
    *,
    workspace: torch.Tensor | None = None,
):
    """MLA attention of each query token over the first ``context_lens[t]``
    positions of its request (at most max_blocks * block_size; none where req_id
    is negative, as in a padded batch).

    With several query tokens of one request (drafts, a prefill chunk) each
    token's own length makes the attention causal.  Lengths are read on the
    device: a captured graph serves any lengths.  Returns as
    ``fp4_ds_mla_sparse_decode``."""
    assert context_lens.dtype == torch.int32 and context_lens.dim() == 1 and context_lens.is_contiguous()
    assert context_lens.shape[0] == q.shape[0], "one context length per query token"
    bt_stride = _check_table(req_id, block_table, q.shape[0], block_size)
    T, H, q, q_strides, num_slots, out, lse, lse_at, ws, hold, dev = _prepare(
        q, kv_cache, 1, -1, return_lse, workspace, context_lens, req_id, block_table)
    _launch("fp4_ds_mla_decode", "fp8mla_fp4_decode", dev, q.data_ptr(), T, H, *q_strides, kv_cache.data_ptr(),
            num_slots, req_id.data_ptr(), block_table.data_ptr(), bt_stride, block_table.shape[1], int(block_size),
            context_lens.data_ptr(), float(sm_scale), out.data_ptr(), H * NOPE, NOPE, *lse_at, *ws)
    return (out, lse) if return_lse else out
