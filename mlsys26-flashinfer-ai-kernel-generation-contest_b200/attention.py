"""Causal softmax attention for the layers that stand between Gated DeltaNet layers.

:func:`attn_prefill` is the whole-prompt form beside ``gdn_prefill`` (packed sequences by
``cu_seqlens``); :func:`attn_paged` the form beside ``gdn_decode`` and ``gdn_mtp`` (one
token, draft tokens or a chunk of a prompt per sequence, over a paged cache).  bf16, head
size 128, grouped heads.  The lengths are read on the device only: no host synchronisation,
and a captured graph follows them.  The work is one launch through the C ABI
``gdn_attn_prefill_launch`` / ``gdn_attn_paged_launch``, with scratch from torch's caching
allocator for each call, so that calls on several streams and captured graphs share none.
"""
from __future__ import annotations

import torch

from . import _checks as C
from ._lib import LIB, check

_prefill_plans, _paged_plans = C.Plans(), C.Plans()


def _lengths(name, x, n, dev):
    if not isinstance(x, torch.Tensor) or x.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{name} must be an int32 or int64 tensor")
    if x.dim() != 1 or (n is not None and x.numel() != n) or x.numel() < (n is None):
        raise ValueError(f"{name} must be 1-D with {'num_seqs + 1' if n is None else n} entries")
    if x.device != dev or not x.is_contiguous():
        raise ValueError(f"{name} must be contiguous and on {dev}")
    return x


def _output(output, q, dev):
    if output is None:
        return torch.empty(q.shape, dtype=torch.bfloat16, device=dev)
    C.tensor("output", output, torch.bfloat16, q.dim(), dev, strided=True)
    C.shape("output", output, q.shape)
    return output


def _workspace_bytes(total_q, num_seqs, hq, hk):
    return int(LIB.gdn_attn_workspace_size(total_q, num_seqs, hq, hk))


def _prefill_key(q, k, v, cu, out):
    return (q.shape, q.stride(), q.dtype, q.device, k.shape, k.stride(), k.dtype, k.device,
            v.shape, v.stride(), v.dtype, v.device, cu.shape, cu.stride(), cu.dtype, cu.device,
            out.shape, out.stride(), out.dtype, out.device)


def _launch_prefill(plan, q, k, v, cu, sc, out):
    ws_n, cu64, T, N, HQ, HK, qs, ks, vs, os_, dev = plan
    ws = torch.empty(ws_n, dtype=torch.uint8, device=dev)
    status = LIB.gdn_attn_prefill_launch(q, k, v, cu, cu64, sc, out, T, N, HQ, HK, C.HEAD_SIZE, qs,
                                         ks, vs, os_, ws.data_ptr(), ws_n, C.raw_stream(dev.index))
    if status:
        check("gdn_attn_prefill_launch", status)


def attn_prefill(q, k, v, cu_seqlens, scale=None, output=None):
    """Causal attention over packed whole prompts: q [T, HQ, 128], k, v [T, HK, 128] bf16,
    ``cu_seqlens`` int32 or int64 [num_seqs + 1].  HQ is a multiple of HK; query head h reads
    key/value head h // (HQ // HK).  ``scale`` None or 0 means 1/sqrt(128).  Returns
    ``output`` [T, HQ, 128]; rows behind the last sequence are not written.

    q, k, v and ``output`` may be views whose token rows are strided (slices of a fused
    projection); other layouts go through dense temporaries.

    A token's output does not depend on the values of other sequences, nor, for finite values,
    on those of later tokens (a later value that is infinite or NaN can reach the earlier rows
    of its tile, as 0 * inf).  The lengths in the batch decide how its sums are grouped, so its
    last bits can differ from one batch to another; the same call repeats bit for bit.

    Empty sequences are allowed, but many of them beside a long one cost time: the kernel for
    few rows is chosen by the mean."""
    try:
        out = torch.empty_like(q) if output is None else output
        plan = _prefill_plans.get(_prefill_key(q, k, v, cu_seqlens, out))
    except (AttributeError, TypeError):
        plan = None
    if plan is not None and C.current_device() == plan[-1].index:
        qp, kp, vp, op = q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr()
        cp = cu_seqlens.data_ptr()
        if not (qp | kp | vp | op) & 15 and not cp & 7:
            _launch_prefill(plan, qp, kp, vp, cp, C.scale_arg(scale), op)
            return out
    return _prefill_checked(q, k, v, cu_seqlens, scale, output)


def _prefill_checked(q, k, v, cu_seqlens, scale, output):
    """Every check; layouts that the kernels do not take are copied."""
    dev = C.cuda_device(q)
    C.tensor("q", q, torch.bfloat16, 3, dev, strided=True)
    C.tensor("k", k, torch.bfloat16, 3, dev, strided=True)
    C.tensor("v", v, torch.bfloat16, 3, dev, strided=True)
    T, HQ, D = q.shape
    HK = k.shape[1]
    C.attn_heads(HQ, HK, D)
    C.shape("k", k, (T, HK, D))
    C.shape("v", v, (T, HK, D))
    _lengths("cu_seqlens", cu_seqlens, None, dev)
    sc = C.scale_arg(scale)
    output = _output(output, q, dev)
    N = cu_seqlens.numel() - 1
    if T == 0 or N == 0:
        return output
    with C.on_device(dev):
        cu = C.dense_or_copy(cu_seqlens, 8)
        (x, qs), (y, ks), (z, vs) = C.rows_in(q, 8, 16), C.rows_in(k, 8, 16), C.rows_in(v, 8, 16)
        out, os_, back = C.rows_out(output, 8, 16)
        if back:
            out.copy_(output)  # rows behind the last sequence keep their values
        plan = (_workspace_bytes(T, N, HQ, HK), int(cu.dtype == torch.int64), T, N, HQ, HK, qs, ks,
                vs, os_, torch.device("cuda", q.get_device()))
        _launch_prefill(plan, x.data_ptr(), y.data_ptr(), z.data_ptr(), cu.data_ptr(), sc,
                        out.data_ptr())
        if back:
            output.copy_(out)
        elif x is q and y is k and z is v:
            _prefill_plans.keep(_prefill_key(q, k, v, cu_seqlens, output), plan)
    return output


def _paged_key(q, k, v, table, lens, cu, out):
    return (q.shape, q.stride(), q.dtype, q.device, k.shape, k.stride(), k.dtype, k.device,
            v.shape, v.stride(), v.dtype, v.device, table.shape, table.stride(), table.dtype,
            table.device, lens.shape, lens.stride(), lens.dtype, lens.device, out.shape,
            out.stride(), out.dtype, out.device,
            None if cu is None else (cu.shape, cu.stride(), cu.dtype, cu.device))


def _launch_paged(plan, q, k, v, table, lens, cu, sc, out):
    (ws_n, ts, lens64, cu64, T, N, width, pages, page_size, kps, vps, HQ, HK, qs, os_, dev) = plan
    ws = torch.empty(ws_n, dtype=torch.uint8, device=dev)
    status = LIB.gdn_attn_paged_launch(q, k, v, table, ts, lens, lens64, cu, cu64, sc, out, T, N,
                                       width, pages, page_size, kps, vps, HQ, HK, C.HEAD_SIZE, qs,
                                       os_, ws.data_ptr(), ws_n, C.raw_stream(dev.index))
    if status:
        check("gdn_attn_paged_launch", status)


def attn_paged(q, k_cache, v_cache, block_table, kv_lens, scale=None, output=None, *,
               cu_seqlens=None):
    """Causal attention of each sequence's newest tokens over its paged cache, which holds
    their keys and values already (:func:`attn_append`).

    q bf16 [num_seqs, q_len, HQ, 128], as ``gdn_decode`` and ``gdn_mtp`` have it, or [T, HQ,
    128] packed by ``cu_seqlens`` [num_seqs + 1]; ``k_cache``, ``v_cache`` bf16 [num_pages,
    page_size, HK, 128] (page_size a multiple of 8; pages may be strided); ``block_table``
    int32 [num_seqs, width]: the pages of each sequence in order; ``kv_lens`` int32 or int64
    [num_seqs]: tokens in the cache, the new ones included.  Token i of q_len sees the first
    kv_len - q_len + i + 1 of them; one that sees none, or all of whose scores are -inf (as in
    :func:`attn_prefill`), gets zeros.  Returns ``output`` in q's shape; rows behind the last sequence are not written.

    A page number outside the cache reads as zeros (nothing is read there), a kv_len above
    width * page_size counts as that.  What lies behind kv_len in a page is not used,
    whatever it holds; as in :func:`attn_prefill`, a newer token's infinite or NaN value can
    reach older rows of its tile, the batch's lengths decide how sums are grouped, and a packed
    batch of mostly empty sequences costs time."""
    try:
        out = torch.empty_like(q) if output is None else output
        plan = _paged_plans.get(_paged_key(q, k_cache, v_cache, block_table, kv_lens, cu_seqlens,
                                           out))
    except (AttributeError, TypeError):
        plan = None
    if plan is not None and C.current_device() == plan[-1].index:
        qp, kp, vp, op = q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr()
        tp, lp = block_table.data_ptr(), kv_lens.data_ptr()
        cp = None if cu_seqlens is None else cu_seqlens.data_ptr()
        if not (qp | kp | vp | op) & 15:
            _launch_paged(plan, qp, kp, vp, tp, lp, cp, C.scale_arg(scale), op)
            return out
    return _paged_checked(q, k_cache, v_cache, block_table, kv_lens, scale, output, cu_seqlens)


def _paged_checked(q, k_cache, v_cache, block_table, kv_lens, scale, output, cu_seqlens):
    """Every check; layouts of q and output that the kernels do not take are copied."""
    dev = C.cuda_device(q)
    packed = cu_seqlens is not None
    C.tensor("q", q, torch.bfloat16, 3 if packed else 4, dev, strided=True)
    HQ, D = q.shape[-2:]
    if not isinstance(k_cache, torch.Tensor) or k_cache.dim() != 4:
        raise TypeError("k_cache must be a 4-D torch.Tensor")
    HK = k_cache.shape[2]
    C.attn_heads(HQ, HK, D)
    kps, vps = C.paged_cache(k_cache, v_cache, HK, dev)
    pages, page_size = k_cache.shape[:2]
    if page_size % 8:
        raise ValueError(f"page_size must be a multiple of 8, got {page_size}")
    if not isinstance(block_table, torch.Tensor) or block_table.dtype != torch.int32:
        raise TypeError("block_table must be an int32 tensor")
    if block_table.dim() != 2 or block_table.device != dev:
        raise ValueError(f"block_table must be 2-D and on {dev}")
    if packed:
        _lengths("cu_seqlens", cu_seqlens, None, dev)
        N = cu_seqlens.numel() - 1
    else:
        N = q.shape[0]
    width = block_table.shape[1]
    C.shape("block_table", block_table, (N, width))
    if width > 1 and block_table.stride(1) != 1 or N > 1 and block_table.stride(0) < width:
        raise ValueError("block_table rows must be dense and must not overlap")
    _lengths("kv_lens", kv_lens, N, dev)
    sc = C.scale_arg(scale)
    output = _output(output, q, dev)
    T = q.shape[0] if packed else N * q.shape[1]
    if T == 0 or N == 0:
        return output
    with C.on_device(dev):
        x, out = (q, output) if packed else (C.token_rows(q), C.token_rows(output))
        rows = x  # None: q's tokens are not one stride apart
        x, qs = C.rows_in(q.reshape(T, HQ, D) if x is None else x, 8, 16)
        back = out is None
        if not back:
            out, os_, back = C.rows_out(out, 8, 16)
        else:
            out, os_ = torch.empty((T, HQ, D), dtype=torch.bfloat16, device=dev), HQ * D
        if back:
            out.copy_(output.reshape(T, HQ, D))  # rows behind the last sequence stay
        plan = (_workspace_bytes(T, N, HQ, HK), block_table.stride(0) if N > 1 else width,
                int(kv_lens.dtype == torch.int64),
                int(packed and cu_seqlens.dtype == torch.int64), T, N, width, pages, page_size, kps,
                vps, HQ, HK, qs, os_, torch.device("cuda", q.get_device()))
        _launch_paged(plan, x.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
                      block_table.data_ptr(), kv_lens.data_ptr(),
                      cu_seqlens.data_ptr() if packed else None, sc, out.data_ptr())
        if back:
            output.copy_(out.view(output.shape))
        elif x is rows:
            _paged_plans.keep(_paged_key(q, k_cache, v_cache, block_table, kv_lens, cu_seqlens,
                                         output), plan)
    return output
