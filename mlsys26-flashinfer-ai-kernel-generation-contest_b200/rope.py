"""Per-head norm of queries and keys with the position rotation, for the softmax-attention
layers that stand between Gated DeltaNet layers.

:func:`attn_qk_norm_rope` returns the rotated rows, :func:`attn_append` writes the keys and
values to a paged cache instead (one launch of the kernel in ``csrc/gdn_attn_rope.cu``
through the C ABI ``gdn_attn_qk_norm_rope_launch``).  The cosines and sines come from a
table that :func:`rope_table` computes once, in 64 bits, because a far position times a
frequency loses its angle in 32.
"""
from __future__ import annotations

import math

import torch

from . import _checks as C
from ._lib import LIB, check

SCALINGS = ("none", "linear", "ntk", "yarn")

_plans = C.Plans()


def rope_table(max_position: int, rotary_dim: int, *, base: float = 10000.0,
               scaling: str = "none", factor: float = 1.0, original_max_position: int = 0,
               beta_fast: float = 32.0, beta_slow: float = 1.0, attention_factor=None,
               device="cuda") -> torch.Tensor:
    """fp32 [max_position, rotary_dim]: the cosines, then the sines, of the angles
    ``position * frequency_i``, ``frequency_i = base^(-2i / rotary_dim)``, i < rotary_dim / 2.

    ``scaling`` stretches them to contexts ``factor`` times as long as trained on:
    "linear" divides every position by ``factor``; "ntk" raises the base by
    ``factor^(rotary_dim / (rotary_dim - 2))`` so that the lowest frequency is divided by
    ``factor`` and the highest kept; "yarn" (Peng et al. 2023) divides frequencies that turn
    less than ``beta_slow`` times within ``original_max_position`` tokens, keeps those that
    turn more than ``beta_fast`` times, goes linearly over the index in between, and
    multiplies cosines and sines by ``attention_factor`` (None: 0.1 ln(factor) + 1)."""
    if max_position < 0 or rotary_dim < 2 or rotary_dim > C.HEAD_SIZE or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be even and in 2..{C.HEAD_SIZE}, max_position >= 0; "
                         f"got {rotary_dim}, {max_position}")
    if scaling not in SCALINGS:
        raise ValueError(f"scaling must be one of {SCALINGS}, got {scaling!r}")
    if not base > 1.0 or not factor >= 1.0:
        raise ValueError(f"base must be > 1 and factor >= 1, got {base}, {factor}")
    if attention_factor is not None and scaling != "yarn":
        raise ValueError("attention_factor belongs to the yarn scaling")
    half = rotary_dim // 2
    i = torch.arange(half, dtype=torch.float64, device=device)
    mscale = 1.0
    if scaling == "ntk" and rotary_dim > 2:
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    freq = base ** (-2.0 * i / rotary_dim)
    if scaling == "linear":
        freq = freq / factor
    elif scaling == "yarn":
        if original_max_position <= 0:
            raise ValueError("yarn scaling needs original_max_position")

        def index_of(turns):  # the index whose frequency turns `turns` times
            return (rotary_dim * math.log(original_max_position / (turns * 2 * math.pi))
                    / (2 * math.log(base)))
        lo = max(math.floor(index_of(beta_fast)), 0)
        hi = min(math.ceil(index_of(beta_slow)), rotary_dim - 1)
        slowed = ((i - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        freq = freq * (1 - slowed) + freq / factor * slowed
        mscale = 0.1 * math.log(factor) + 1.0 if attention_factor is None else attention_factor
    angle = torch.arange(max_position, dtype=torch.float64, device=device)[:, None] * freq
    return (torch.cat([angle.cos(), angle.sin()], dim=1) * mscale).float()


def _index(name, x, n, dev):
    if not isinstance(x, torch.Tensor) or x.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{name} must be an int32 or int64 tensor")
    if x.dim() != 1 or x.numel() != n or x.device != dev or not x.is_contiguous():
        raise ValueError(f"{name} must be a contiguous [{n}] tensor on {dev}")
    return x


def _weight(name, w, dev):
    if w is None:
        return None
    C.tensor(name, w, torch.float32, 1, dev, strided=True)
    C.shape(name, w, (C.HEAD_SIZE,))
    return C.dense_or_copy(w, 16)


def _key(q, k, v, positions, table, slots, k_cache, v_cache, q_weight, k_weight, q_out, k_out):
    return (q.shape, q.stride(), q.dtype, q.device, k.shape, k.stride(), k.dtype, k.device,
            positions.shape, positions.stride(), positions.dtype, positions.device, table.shape,
            table.stride(), table.dtype, table.device, q_out.shape, q_out.stride(), q_out.dtype,
            q_out.device,
            None if q_weight is None else (q_weight.shape, q_weight.stride(), q_weight.dtype,
                                           q_weight.device),
            None if k_weight is None else (k_weight.shape, k_weight.stride(), k_weight.dtype,
                                           k_weight.device),
            (k_out.shape, k_out.stride(), k_out.dtype, k_out.device) if k_cache is None else
            (v.shape, v.stride(), v.dtype, v.device, slots.shape, slots.stride(), slots.dtype,
             slots.device, k_cache.shape, k_cache.stride(), k_cache.dtype, k_cache.device,
             v_cache.shape, v_cache.stride(), v_cache.dtype, v_cache.device))


def _launch(plan, ptrs, eps, interleaved):
    (pos64, rows, slots64, pages, page_size, kps, vps, T, HQ, HK, rd, qs, ks, vs, qos, kos,
     dev) = plan
    q, k, v, pos, table, wq, wk, qo, ko, slots, kc, vc = ptrs
    status = LIB.gdn_attn_qk_norm_rope_launch(
        q, k, v, pos, pos64, table, rows, wq, wk, eps, interleaved, qo, ko, slots, slots64, kc, vc,
        pages, page_size, kps, vps, T, HQ, HK, C.HEAD_SIZE, rd, qs, ks, vs, qos, kos,
        C.raw_stream(dev.index))
    if status:
        check("gdn_attn_qk_norm_rope_launch", status)


def _run(q, k, v, positions, table, slots, k_cache, v_cache, q_weight, k_weight, q_out, k_out, eps,
         interleaved):
    try:
        qo = torch.empty_like(q) if q_out is None else q_out
        ko = torch.empty_like(k) if k_out is None and k_cache is None else k_out
        plan = _plans.get(_key(q, k, v, positions, table, slots, k_cache, v_cache, q_weight,
                               k_weight, qo, ko))
    except (AttributeError, TypeError):
        plan = None
    if plan is not None and C.current_device() == plan[-1].index and 0.0 <= eps < math.inf:
        qp, kp, op = q.data_ptr(), k.data_ptr(), qo.data_ptr()
        wq = 0 if q_weight is None else q_weight.data_ptr()
        wk = 0 if k_weight is None else k_weight.data_ptr()
        if k_cache is None:
            vp = sp = kcp = vcp = None
            bits = kop = ko.data_ptr()
        else:
            vp, kcp, vcp = v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr()
            kop, sp, bits = None, slots.data_ptr(), vp | kcp | vcp
        if not (qp | kp | op | wq | wk | bits) & 15:
            _launch(plan, (qp, kp, vp, positions.data_ptr(), table.data_ptr(), wq or None,
                           wk or None, op, kop, sp, kcp, vcp), eps, 1 if interleaved else 0)
            return qo, ko
    return _run_checked(q, k, v, positions, table, slots, k_cache, v_cache, q_weight, k_weight,
                        q_out, k_out, eps, interleaved)


def _run_checked(q, k, v, positions, table, slots, k_cache, v_cache, q_weight, k_weight, q_out,
                 k_out, eps, interleaved):
    """Every check; layouts that the kernel does not take are copied."""
    dev = C.cuda_device(q)
    C.tensor("q", q, torch.bfloat16, 3, dev, strided=True)
    C.tensor("k", k, torch.bfloat16, 3, dev, strided=True)
    T, HQ, D = q.shape
    HK = k.shape[1]
    C.attn_heads(HQ, HK, D)
    C.shape("k", k, (T, HK, D))
    _index("positions", positions, T, dev)
    C.tensor("rope_table", table, torch.float32, 2, dev)
    rd = table.shape[1]
    if rd < 2 or rd > D or rd % 2:
        raise ValueError(f"rope_table must have an even 2..{D} columns, got {rd}")
    eps = float(eps)
    if not (0.0 <= eps < math.inf):
        raise ValueError(f"eps must be >= 0 and finite, got {eps}")
    given = (q, k, v, q_weight, k_weight)
    if q_out is None:
        q_out = torch.empty(T, HQ, D, dtype=torch.bfloat16, device=dev)
    else:
        C.tensor("q_out", q_out, torch.bfloat16, 3, dev, strided=True)
        C.shape("q_out", q_out, (T, HQ, D))
    cached = k_cache is not None
    kps = vps = pages = vs = kos = 0
    page_size = 1
    if cached:
        C.tensor("v", v, torch.bfloat16, 3, dev, strided=True)
        C.shape("v", v, (T, HK, D))
        _index("slots", slots, T, dev)
        kps, vps = C.paged_cache(k_cache, v_cache, HK, dev)
        pages, page_size = k_cache.shape[:2]
    elif k_out is None:
        k_out = torch.empty(T, HK, D, dtype=torch.bfloat16, device=dev)
    else:
        C.tensor("k_out", k_out, torch.bfloat16, 3, dev, strided=True)
        C.shape("k_out", k_out, (T, HK, D))
    with C.on_device(dev):
        wq, wk = _weight("q_weight", q_weight, dev), _weight("k_weight", k_weight, dev)
        if T == 0:
            return q_out, k_out
        x, qs = C.rows_in(q, 8, 16)
        y, ks = C.rows_in(k, 8, 16)
        z, ko, k_back = v, None, False
        if cached:
            z, vs = C.rows_in(v, 8, 16)
        else:
            ko, kos, k_back = C.rows_out(k_out, 8, 16)
        qo, qos, q_back = C.rows_out(q_out, 8, 16)
        plan = (int(positions.dtype == torch.int64), table.shape[0],
                int(cached and slots.dtype == torch.int64), pages, page_size, kps, vps, T, HQ, HK,
                rd, qs, ks, vs, qos, kos, torch.device("cuda", q.get_device()))
        ptr = lambda t: t.data_ptr() if t is not None else None  # noqa: E731
        _launch(plan, (ptr(x), ptr(y), ptr(z) if cached else None, ptr(positions), ptr(table),
                       ptr(wq), ptr(wk), ptr(qo), ptr(ko), ptr(slots) if cached else None,
                       ptr(k_cache), ptr(v_cache)), eps, int(bool(interleaved)))
        if q_back:
            q_out.copy_(qo)
        if k_back:
            k_out.copy_(ko)
    if not q_back and not k_back and all(a is b for a, b in zip((x, y, z, wq, wk), given)):
        _plans.keep(_key(q, k, v, positions, table, slots, k_cache, v_cache, q_weight, k_weight,
                         q_out, k_out), plan)
    return q_out, k_out


def attn_qk_norm_rope(q, k, positions, rope_table, q_weight=None, k_weight=None, q_out=None,
                      k_out=None, *, eps: float = 1e-6, interleaved: bool = False):
    """RMSNorm of every head of q [T, HQ, 128] and k [T, HK, 128] (bf16) with the fp32 [128]
    weights (None: no norm) and the rotation by row ``positions[t]`` of ``rope_table``, fp32
    throughout and rounded once.  Returns ``(q_out, k_out)``, which may be q and k.

    The first ``rope_table.shape[1]`` values of a head turn, in pairs (i, i + half) or, with
    ``interleaved``, (2i, 2i + 1).  A token whose position lies outside the table is padding:
    zeros.  Inputs and outputs may be views whose token rows are strided; other layouts go
    through dense temporaries."""
    return _run(q, k, None, positions, rope_table, None, None, None, q_weight, k_weight, q_out,
                k_out, eps, interleaved)


def attn_append(q, k, v, positions, rope_table, slots, k_cache, v_cache, q_weight=None,
                k_weight=None, q_out=None, *, eps: float = 1e-6, interleaved: bool = False):
    """:func:`attn_qk_norm_rope` whose keys go, with the values v [T, HK, 128], to the paged
    cache: row ``slots[t] % page_size`` of page ``slots[t] // page_size`` of ``k_cache`` and
    ``v_cache`` [num_pages, page_size, HK, 128] (bf16, updated in place; pages may be
    strided).  Returns ``q_out`` (may be q).

    Any page size is written; :func:`attn_paged` reads pages of a multiple of 8 rows.  Slots must
    be distinct.  A slot outside the cache writes nothing there; a token whose
    position lies outside the table is padding: zeros in q_out, nothing in the cache."""
    if k_cache is None:
        raise TypeError("k_cache must be a torch.Tensor, got NoneType")
    return _run(q, k, v, positions, rope_table, slots, k_cache, v_cache, q_weight, k_weight, q_out,
                None, eps, interleaved)[0]
