"""Workloads of the softmax-attention operators that stand beside the Gated DeltaNet ones.

A model that mixes its tokens with Gated DeltaNet layers has softmax-attention layers in
between.  They see the same packed prompts, decode steps and draft-token verifications as
``gdn_prefill``, ``gdn_decode`` and ``gdn_mtp``, and keep a paged cache of keys and values
where those keep a pool of states.  Three operators, head size 128, bf16:

* ``rope``:    per-head RMSNorm of queries and keys and the position rotation in one pass,
               the keys and values either returned or written to the cache's pages;
* ``prefill``: causal attention over packed whole prompts, grouped heads;
* ``paged``:   causal attention of the newest tokens of each sequence (one token, a few
               draft tokens, a chunk of a prompt) over the paged cache.

With ``own`` false, ``run`` computes them in elementary torch operations in 32 bits; with
``own`` true it calls the package.
"""
import importlib
import math
import random

import torch

own = False

D = 128
EPS = 1e-6
BASE = 1e6
HEADS = ((16, 2), (16, 4), (8, 8), (12, 4), (6, 2), (5, 1), (32, 8))
PAGES = (8, 16, 48, 64, 128)


# ----------------------------------------------------------------------------- cases
def listed():
    return [
        # one decode step of 7 sequences: K normalised, rotated and written to its page
        dict(name="rope decode 7", op="rope", tokens=7, hq=16, hkv=2, rd=64, half=True,
             norm=True, cache=True, page=16, table=65536, mix=1),
        # a ragged prompt chunk into the cache, interleaved pairs, no norm
        dict(name="rope chunk 1777", op="rope", tokens=1777, hq=12, hkv=4, rd=96, half=False,
             norm=False, cache=True, page=48, table=32768, mix=2),
        # q and k of one 32768-token prompt, whole-head rotation, returned
        dict(name="rope prompt 32768", op="rope", tokens=32768, hq=16, hkv=4, rd=128, half=True,
             norm=True, cache=False, page=16, table=32768, mix=3),
        # a few short prompts, some empty: launch latency counts
        dict(name="prefill short", op="prefill", seqs=6, tokens=211, hq=16, hkv=2, mix=4),
        # packed prompts of very different lengths, one head per key/value head
        dict(name="prefill packed mha", op="prefill", seqs=11, tokens=8191, hq=8, hkv=8, mix=5),
        # packed prompts, grouped heads
        dict(name="prefill packed", op="prefill", seqs=8, tokens=16384, hq=16, hkv=4, mix=6),
        # one long prompt: the largest case
        dict(name="prefill long", op="prefill", seqs=1, tokens=16384, hq=16, hkv=2, mix=7),
        # one decode step of few sequences with short contexts: latency
        dict(name="paged decode 4", op="paged", seqs=4, q_max=1, ragged_q=False, kv_max=600,
             hq=16, hkv=2, page=16, mix=8),
        # a full decode batch, contexts of different lengths
        dict(name="paged decode 128", op="paged", seqs=128, q_max=1, ragged_q=False,
             kv_max=8192, hq=16, hkv=4, page=16, mix=9),
        # one sequence with a long context: the work is split along it
        dict(name="paged decode long", op="paged", seqs=1, q_max=1, ragged_q=False,
             kv_max=131072, hq=16, hkv=2, page=64, mix=10),
        # verification of 4 draft tokens
        dict(name="paged draft 32x4", op="paged", seqs=32, q_max=4, ragged_q=False, kv_max=6000,
             hq=16, hkv=2, page=48, mix=11),
        # chunks of prompts of different lengths over their earlier tokens
        dict(name="paged chunks", op="paged", seqs=5, q_max=1500, ragged_q=True, kv_max=16000,
             hq=16, hkv=4, page=128, mix=12),
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("rope", "prefill", "paged", "paged"))
    hq, hkv = rng.choice(HEADS)
    mix = rng.randrange(1 << 20)
    if op == "rope":
        return dict(op=op, tokens=_spread(rng, 1, 32768), hq=hq, hkv=hkv,
                    rd=rng.choice((32, 64, 96, 128)), half=rng.random() < 0.5,
                    norm=rng.random() < 0.7, cache=rng.random() < 0.6,
                    page=rng.choice(PAGES), table=32768 + rng.randrange(4096), mix=mix)
    if op == "prefill":
        seqs = _spread(rng, 1, 16)
        tokens = _spread(rng, 16, 8192 if hq > 16 else 12288)
        return dict(op=op, seqs=seqs, tokens=tokens, hq=hq, hkv=hkv, mix=mix)
    kind = rng.choice(("decode", "draft", "chunk"))
    page = rng.choice(PAGES)
    if kind == "decode":
        seqs, q_max, kv_max, ragged = _spread(rng, 1, 128), 1, _spread(rng, 64, 8192), False
    elif kind == "draft":
        seqs, q_max, kv_max, ragged = _spread(rng, 1, 32), rng.randint(2, 8), _spread(rng, 64, 8192), rng.random() < 0.5
    else:
        seqs, q_max, kv_max, ragged = rng.randint(1, 4), _spread(rng, 16, 1500), _spread(rng, 1600, 16000), True
    return dict(op=op, seqs=seqs, q_max=q_max, ragged_q=ragged, kv_max=kv_max, hq=hq, hkv=hkv,
                page=page, mix=mix)


def _lengths(case):
    """(new tokens, cached tokens with the new ones) of each sequence of a case."""
    rng = random.Random(case["mix"])
    n = case["seqs"]
    if case["op"] == "prefill":
        cuts = sorted(rng.randint(0, case["tokens"]) for _ in range(n - 1))
        q = [b - a for a, b in zip([0] + cuts, cuts + [case["tokens"]])]
        return q, list(q)
    q = [rng.randint(1, case["q_max"]) if case["ragged_q"] else case["q_max"] for _ in range(n)]
    kv = [max(x, case["kv_max"] if n == 1 else rng.randint(case["kv_max"] // 4, case["kv_max"]))
          for x in q]
    return q, kv


# ----------------------------------------------------------------------------- inputs
def _randn(shape, g, std=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * std).to(torch.bfloat16)


def _starts(lens):
    cu = [0]
    for x in lens:
        cu.append(cu[-1] + x)
    return torch.tensor(cu, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    hq, hkv = case["hq"], case["hkv"]
    s = {"case": case}
    if case["op"] == "rope":
        t, rd = case["tokens"], case["rd"]
        # slices of one fused projection, as a layer has them
        fused = _randn((t, (hq + 2 * hkv) * D), g, 2.0)
        s["q"] = fused[:, :hq * D].view(t, hq, D)
        s["k"] = fused[:, hq * D:(hq + hkv) * D].view(t, hkv, D)
        s["v"] = fused[:, (hq + hkv) * D:].view(t, hkv, D)
        inv = BASE ** (-torch.arange(0, rd, 2, device="cuda", dtype=torch.float64) / rd)
        angle = torch.arange(case["table"], device="cuda", dtype=torch.float64)[:, None] * inv
        s["table"] = torch.cat([angle.cos(), angle.sin()], dim=1).float()
        first = torch.randint(0, case["table"] - t + 1, (1,), generator=g, device="cuda")
        s["positions"] = first + torch.arange(t, device="cuda")
        s["wq"] = s["wk"] = None
        if case["norm"]:
            s["wq"] = 1 + 0.2 * torch.randn(D, generator=g, device="cuda")
            s["wk"] = 1 + 0.2 * torch.randn(D, generator=g, device="cuda")
        if case["cache"]:
            ps = case["page"]
            pages = (t + ps - 1) // ps + 3
            s["k_cache"] = _randn((pages, ps, hkv, D), g)
            s["v_cache"] = _randn((pages, ps, hkv, D), g)
            order = torch.randperm(pages, generator=g, device="cuda")
            at = torch.arange(t, device="cuda")
            s["slots"] = (order[at // ps] * ps + at % ps).to(torch.int64)
        return s
    q_lens, kv_lens = _lengths(case)
    t = sum(q_lens)
    s["cu"] = _starts(q_lens)
    s["q"] = _randn((t, hq, D), g, 1.5)
    s["q_pad"] = max(q_lens)
    s["kv_pad"] = max(kv_lens)
    if case["op"] == "prefill":
        s["k"] = _randn((t, hkv, D), g, 1.5)
        s["v"] = _randn((t, hkv, D), g)
        return s
    ps = case["page"]
    need = [(x + ps - 1) // ps for x in kv_lens]
    pages = sum(need) + 5
    s["k_cache"] = _randn((pages, ps, hkv, D), g, 1.5)
    s["v_cache"] = _randn((pages, ps, hkv, D), g)
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    width = max(need)
    first = torch.tensor([sum(need[:i]) for i in range(len(need))], device="cuda")
    col = torch.arange(width, device="cuda")
    used = col[None, :] < torch.tensor(need, device="cuda")[:, None]
    at = (first[:, None] + col[None, :]).clamp(max=pages - 1)
    s["block_table"] = torch.where(used, order[at], torch.full_like(order[at], -1)).contiguous()
    s["kv_lens"] = torch.tensor(kv_lens, dtype=torch.int32, device="cuda")
    if not case["ragged_q"]:
        s["q"] = s["q"].view(len(q_lens), case["q_max"], hq, D)
    return s


# ----------------------------------------------------------------------------- plain forms
def _plain_rope(s):
    case = s["case"]
    h = case["rd"] // 2
    cs = s["table"][s["positions"]]
    c, sn = cs[:, None, :h], cs[:, None, h:]

    def turn(x, w):
        x = x.float()
        if w is not None:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w
        part, rest = x[..., :2 * h], x[..., 2 * h:]
        if case["half"]:
            a, b = part[..., :h], part[..., h:]
            part = torch.cat([a * c - b * sn, b * c + a * sn], dim=-1)
        else:
            a, b = part[..., 0::2], part[..., 1::2]
            part = torch.stack([a * c - b * sn, b * c + a * sn], dim=-1).flatten(-2)
        return torch.cat([part, rest], dim=-1).to(torch.bfloat16)

    q, k = turn(s["q"], s["wq"]), turn(s["k"], s["wk"])
    if not case["cache"]:
        return q, k
    s["k_cache"].view(-1, case["hkv"], D)[s["slots"]] = k
    s["v_cache"].view(-1, case["hkv"], D)[s["slots"]] = s["v"]
    return q, s["k_cache"], s["v_cache"]


def _plain_attention(q, cu, k, v, kv_lens, q_pad):
    """q [T, HQ, D] packed by cu; k, v [N, L, HKV, D] padded; the last tokens of each."""
    hq, hkv, n, length = q.shape[1], k.shape[2], k.shape[0], k.shape[1]
    grp = hq // hkv
    start, q_lens = cu[:-1].long(), (cu[1:] - cu[:-1]).long()
    row = torch.arange(q_pad, device=q.device)
    at = (start[:, None] + row).clamp(max=max(q.shape[0] - 1, 0))
    x = q.float()[at].view(n, q_pad, hkv, grp, D).permute(0, 2, 3, 1, 4)
    x = x.reshape(n, hkv, grp * q_pad, D)
    score = (x @ k.float().permute(0, 2, 3, 1)).view(n, hkv, grp, q_pad, length)
    score *= 1 / math.sqrt(D)
    last = (kv_lens.long() - q_lens)[:, None] + row  # the last position that a row sees
    seen = torch.arange(length, device=q.device) <= last[:, :, None]
    score.masked_fill_(~seen[:, None, None], float("-inf"))
    top = score.amax(-1, keepdim=True).clamp(min=-3e38)
    p = score.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = p.view(n, hkv, grp * q_pad, length) @ v.float().permute(0, 2, 1, 3)
    o = o.view(n, hkv, grp, q_pad, D) / total.clamp(min=1e-30)
    o = o.permute(0, 3, 1, 2, 4).reshape(n, q_pad, hq, D)
    return o[row < q_lens[:, None]].to(torch.bfloat16)


def _plain_prefill(s):
    start, q_lens = s["cu"][:-1].long(), (s["cu"][1:] - s["cu"][:-1]).long()
    at = start[:, None] + torch.arange(s["kv_pad"], device="cuda")
    at = at.clamp(max=s["q"].shape[0] - 1)
    return _plain_attention(s["q"], s["cu"], s["k"][at], s["v"][at], q_lens, s["q_pad"])


def _plain_paged(s):
    ps, hkv = s["case"]["page"], s["case"]["hkv"]
    pos = torch.arange(s["kv_pad"], device="cuda")
    at = s["block_table"].long().clamp(min=0)[:, pos // ps] * ps + pos % ps
    q = s["q"].reshape(-1, s["case"]["hq"], D)
    o = _plain_attention(q, s["cu"], s["k_cache"].view(-1, hkv, D)[at],
                         s["v_cache"].view(-1, hkv, D)[at], s["kv_lens"], s["q_pad"])
    return o.view(s["q"].shape)


# ----------------------------------------------------------------------------- the pass
def _run_own(s):
    pkg = importlib.import_module("mlsys26-flashinfer-ai-kernel-generation-contest_b200")
    case = s["case"]
    if case["op"] == "rope":
        if case["cache"]:
            q = pkg.attn_append(s["q"], s["k"], s["v"], s["positions"], s["table"], s["slots"],
                                s["k_cache"], s["v_cache"], s["wq"], s["wk"], eps=EPS,
                                interleaved=not case["half"])
            return q, s["k_cache"], s["v_cache"]
        return pkg.attn_qk_norm_rope(s["q"], s["k"], s["positions"], s["table"], s["wq"],
                                     s["wk"], eps=EPS, interleaved=not case["half"])
    if case["op"] == "prefill":
        return pkg.attn_prefill(s["q"], s["k"], s["v"], s["cu"], None)
    if case["ragged_q"]:
        return pkg.attn_paged(s["q"], s["k_cache"], s["v_cache"], s["block_table"],
                              s["kv_lens"], None, cu_seqlens=s["cu"])
    return pkg.attn_paged(s["q"], s["k_cache"], s["v_cache"], s["block_table"], s["kv_lens"],
                          None)


def run(state):
    if own:
        return _run_own(state)
    op = state["case"]["op"]
    return (_plain_rope if op == "rope" else
            _plain_prefill if op == "prefill" else _plain_paged)(state)


def work(case):
    hq, hkv = case["hq"], case["hkv"]
    if case["op"] == "rope":
        t, rd = case["tokens"], case["rd"]
        heads = hq + hkv + (hkv if case["cache"] else 0)
        # rows in and out, a row of the table, a position and a slot of 8 bytes
        return {"bytes": t * (heads * D * 2 * 2 + rd * 4 + 8 + (8 if case["cache"] else 0)),
                "flops": t * (hq + hkv) * (3 * rd + (4 * D if case["norm"] else 0))}
    q_lens, kv_lens = _lengths(case)
    pairs = sum(q * kv - q * (q - 1) // 2 for q, kv in zip(q_lens, kv_lens))
    return {"bytes": 2 * D * (2 * hq * sum(q_lens) + 2 * hkv * sum(kv_lens)),
            "flops": 4 * D * hq * pairs}


# ----------------------------------------------------------------------------- 64 bits
def _exact_rope(s):
    case, table = s["case"], s["table"].double()
    h = case["rd"] // 2
    out = []
    for x, w in ((s["q"], s["wq"]), (s["k"], s["wk"])):
        y = x.double().clone()
        if w is not None:
            y = y / torch.sqrt(y.pow(2).sum(-1, keepdim=True) / D + EPS) * w.double()
        z = y.clone()
        for i in range(h):
            a, b = (i, i + h) if case["half"] else (2 * i, 2 * i + 1)
            c, sn = table[s["positions"], i, None], table[s["positions"], h + i, None]
            z[:, :, a] = y[:, :, a] * c - y[:, :, b] * sn
            z[:, :, b] = y[:, :, a] * sn + y[:, :, b] * c
        out.append(z)
    if not case["cache"]:
        return tuple(out)
    page, off = s["slots"] // case["page"], s["slots"] % case["page"]
    kc, vc = s["k_cache"].double(), s["v_cache"].double()
    kc[page, off] = out[1]
    vc[page, off] = s["v"].double()
    return out[0], kc, vc


def _exact_rows(q, k, v, first):
    """q [R, D], k, v [L, D] in 64 bits; row i sees positions 0 .. first + i."""
    z = q @ k.T / math.sqrt(D)
    i = torch.arange(q.shape[0], device=q.device)[:, None]
    z[torch.arange(k.shape[0], device=q.device)[None, :] > first + i] = float("-inf")
    return torch.softmax(z, dim=-1) @ v


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rope":
        return _exact_rope(s)
    q_lens, kv_lens = _lengths(case)
    hq, hkv = case["hq"], case["hkv"]
    q = s["q"].reshape(-1, hq, D)
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    at = 0
    for n, (ql, kl) in enumerate(zip(q_lens, kv_lens)):
        if case["op"] == "prefill":
            k, v = s["k"][at:at + kl], s["v"][at:at + kl]
        else:
            used = s["block_table"][n, :-(-kl // case["page"])].long()
            k = s["k_cache"][used].flatten(0, 1)[:kl]
            v = s["v_cache"][used].flatten(0, 1)[:kl]
        for h in range(hkv):
            kh, vh = k[:, h].double(), v[:, h].double()
            for x in range(h * (hq // hkv), (h + 1) * (hq // hkv)):
                for r in range(0, ql, 4096):
                    e = min(ql, r + 4096)
                    end = kl - ql + e
                    out[at + r:at + e, x] = _exact_rows(q[at + r:at + e, x].double(),
                                                        kh[:end], vh[:end], kl - ql + r)
        at += ql
    return out.view(s["q"].shape)
