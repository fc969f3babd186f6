"""GPU: attn_qk_norm_rope and attn_append against the 64-bit oracle, and the layer's run
attn_append -> attn_paged beside attn_prefill."""
import pytest
import torch

from attn_util import D, check, randn, starts
from conftest import load_pkg
from oracle import attn_oracle as A

pytestmark = pytest.mark.gpu

# bf16 output: 2^-8 of the value.  fp32: sum of squares (8 + 4 roundings), rsqrt (2 ulp), two
# products and the rotation's fma: under 16 roundings of |y_a| + |y_b|, 16 * 2^-24 = 2^-20.
BF16 = 2.0 ** -8


def close(out, ref, size):
    off = (out.cpu().double() - ref).abs()
    assert (off <= BF16 * ref.abs() + 2.0 ** -19 * size + 1e-30).all(), (off - BF16 * ref.abs()).max()


def inputs(t, hq, hk, seed, table_rows=4096, rd=64, far=False):
    g = torch.Generator().manual_seed(seed)
    pkg = load_pkg()
    table = pkg.rope_table(table_rows, rd, base=1e4, device="cpu")
    pos = torch.randint(table_rows - t if far else 0, table_rows, (t,), generator=g)
    return dict(q=randn((t, hq, D), g, 2.0), k=randn((t, hk, D), g, 2.0), v=randn((t, hk, D), g),
                pos=pos, table=table, wq=1 + 0.3 * torch.randn(D, generator=g),
                wk=1 + 0.3 * torch.randn(D, generator=g))


def reference(d, x, w, inter):
    ref = A.norm_rope(d[x], d[w] if w else None, d["pos"], d["table"], interleaved=inter)
    size = A.norm_rope(d[x], d[w] if w else None, d["pos"], d["table"][:, :0].new_zeros(
        d["table"].shape[0], 2) + torch.tensor([1.0, 0.0])).abs().amax(-1, keepdim=True) * 2
    return ref, size.expand_as(ref)


@pytest.mark.parametrize("rd", [2, 6, 8, 16, 32, 40, 64, 96, 100, 126, 128])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("norm", [True, False])
def test_norm_rope(cuda, rd, inter, norm):
    pkg = load_pkg()
    for t, hq, hk in ((1, 4, 1), (13, 5, 5), (37, 6, 2)):
        d = inputs(t, hq, hk, seed=rd + t, rd=rd)
        g = {k: v.to(cuda) for k, v in d.items()}
        qo, ko = pkg.attn_qk_norm_rope(g["q"], g["k"], g["pos"], g["table"],
                                       g["wq"] if norm else None, g["wk"] if norm else None,
                                       interleaved=inter)
        close(qo, *reference(d, "q", "wq" if norm else None, inter))
        close(ko, *reference(d, "k", "wk" if norm else None, inter))
        if not norm:  # what does not turn passes through bit for bit
            assert torch.equal(qo[..., rd:], g["q"][..., rd:])


def test_views_in_place_and_padding(cuda):
    pkg = load_pkg()
    t, hq, hk = 29, 6, 3
    d = inputs(t, hq, hk, seed=1, rd=48)
    d["pos"][4], d["pos"][17], d["pos"][28] = -1, d["table"].shape[0], 2 ** 40
    rq, sq = reference(d, "q", "wq", False)
    rk, sk = reference(d, "k", "wk", False)
    g = {k: v.to(cuda) for k, v in d.items()}
    fused = torch.cat([g["q"].flatten(1), g["k"].flatten(1), g["v"].flatten(1)], dim=1)
    q = fused[:, :hq * D].view(t, hq, D)
    k = fused[:, hq * D:(hq + hk) * D].view(t, hk, D)
    qo, ko = pkg.attn_qk_norm_rope(q, k, g["pos"], g["table"], g["wq"], g["wk"], q, k)
    assert qo is q and ko is k
    close(q, rq, sq)
    close(k, rk, sk)
    assert (q[4] == 0).all() and (k[17] == 0).all() and (q[28] == 0).all()
    assert torch.equal(fused[:, (hq + hk) * D:], g["v"].flatten(1))
    # layouts that are copied: a transposed q, an unaligned k, outputs of either kind
    out = torch.empty(t, D, hq, dtype=torch.bfloat16, device=cuda).transpose(1, 2)
    odd = torch.empty(t * hk * D + 1, dtype=torch.bfloat16, device=cuda)[1:].view(t, hk, D)
    odd.copy_(d["k"])
    ko = torch.empty(t * hk * D + 1, dtype=torch.bfloat16, device=cuda)[1:].view(t, hk, D)
    pkg.attn_qk_norm_rope(g["q"].transpose(0, 1).contiguous().transpose(0, 1), odd,
                          g["pos"].where(g["pos"] < 2 ** 31, -1).int(), g["table"],
                          g["wq"].expand(2, D).t().contiguous().t()[0], g["wk"], out, ko)
    close(out, rq, sq)
    close(ko, rk, sk)


@pytest.mark.parametrize("page", [1, 16, 24])
@pytest.mark.parametrize("hq,hk,inter", [(4, 2, False), (5, 1, True), (3, 3, False)])
def test_append(cuda, page, hq, hk, inter):
    pkg = load_pkg()
    t, pages = 53, 100 // page + 4
    d = inputs(t, hq, hk, seed=page, rd=64)
    d["pos"][7] = -3  # padding: nothing in the cache
    slots = torch.randperm(pages * page, generator=torch.Generator().manual_seed(1))[:t]
    slots[3], slots[9] = -1, pages * page  # outside: not written
    rq, sq = reference(d, "q", "wq", inter)
    rk, sk = reference(d, "k", "wk", inter)
    g = {k: v.to(cuda) for k, v in d.items()}
    for dtype in (torch.int32, torch.int64):
        both = torch.full((pages, 2, page, hk, D), 9.0, dtype=torch.bfloat16, device=cuda)
        q = pkg.attn_append(g["q"], g["k"], g["v"], g["pos"].to(dtype), g["table"],
                            slots.to(cuda, dtype), both[:, 0], both[:, 1], g["wq"], g["wk"],
                            interleaved=inter)
        close(q, rq, sq)
        assert (q[7] == 0).all()
        kc, vc = both[:, 0].reshape(-1, hk, D), both[:, 1].reshape(-1, hk, D)
        keep = [i for i in range(t) if i not in (3, 7, 9)]
        close(kc[slots[keep].to(cuda)], rk[keep], sk[keep])
        assert torch.equal(vc[slots[keep].to(cuda)], g["v"][keep])
        rest = torch.ones(pages * page, dtype=torch.bool)
        rest[slots[keep]] = False
        assert (kc[rest.to(cuda)] == 9).all() and (vc[rest.to(cuda)] == 9).all()


def test_many_tokens_and_far_slots(cuda):
    """More tokens than one wave of blocks; slots past 2^32 elements of the cache."""
    pkg = load_pkg()
    t, hq, hk, page = 9001, 4, 2, 64
    pages = 2 ** 32 // (page * hk * D) + 200
    d = inputs(t, hq, hk, seed=2, table_rows=10000, rd=128)
    g = {k: v.to(cuda) for k, v in d.items()}
    kc = torch.empty(pages, page, hk, D, dtype=torch.bfloat16, device=cuda)
    vc = torch.empty_like(kc)
    slots = torch.arange(t, device=cuda) + (pages * page - t)
    q = pkg.attn_append(g["q"], g["k"], g["v"], g["pos"], g["table"], slots, kc, vc, g["wq"],
                        g["wk"])
    sel = torch.arange(0, t, 97)
    small = dict(d, q=d["q"][sel], k=d["k"][sel], pos=d["pos"][sel])
    close(q[sel.to(cuda)], *reference(small, "q", "wq", False))
    close(kc.view(-1, hk, D)[slots[sel.to(cuda)]], *reference(small, "k", "wk", False))
    assert torch.equal(vc.view(-1, hk, D)[-t:], g["v"])


def test_zero_rows_and_extreme_values(cuda):
    """A row of zeros stays zero; rows of the largest and smallest bf16 values: their
    squares leave fp32's range at the top, which is refused by no norm: inf -> 0."""
    pkg = load_pkg()
    d = inputs(3, 2, 1, seed=3)
    d["q"][0] = 0
    d["q"][1] = 2.0 ** -60  # squares underflow to 0: eps rules, y = x / sqrt(eps)
    g = {k: v.to(cuda) for k, v in d.items()}
    qo, _ = pkg.attn_qk_norm_rope(g["q"], g["k"], g["pos"], g["table"], g["wq"], g["wk"])
    assert (qo[0] == 0).all()
    close(qo, *reference(d, "q", "wq", False))


@pytest.mark.parametrize("kw", [dict(), dict(scaling="linear", factor=4.0),
                                dict(scaling="ntk", factor=8.0),
                                dict(scaling="yarn", factor=16.0, original_max_position=4096)])
def test_a_layer_in_chunks_equals_the_whole_prompt(cuda, kw):
    """Prompts appended and attended in chunks, then single tokens and drafts: every row
    agrees with the oracle's whole-prompt attention over the oracle's rotated q and k."""
    pkg = load_pkg()
    hq, hk, page, rd = 6, 2, 16, 64
    lens = [75, 140]
    g0 = torch.Generator().manual_seed(7)
    table = pkg.rope_table(1000, rd, device=cuda, **kw)
    raw = [dict(q=randn((n, hq, D), g0, 2.0), k=randn((n, hk, D), g0, 2.0), v=randn((n, hk, D), g0))
           for n in lens]
    wq, wk = 1 + 0.2 * torch.randn(D, generator=g0), 1 + 0.2 * torch.randn(D, generator=g0)
    pages = [-(-n // page) for n in lens]
    order = torch.randperm(sum(pages) + 2, generator=g0).int()
    bt = torch.full((2, max(pages)), -1, dtype=torch.int32)
    bt[0, :pages[0]], bt[1, :pages[1]] = order[:pages[0]], order[pages[0]:sum(pages)]
    kc = torch.full((sum(pages) + 2, page, hk, D), float("nan"), dtype=torch.bfloat16, device=cuda)
    vc = kc.clone()
    want, size = [], []
    for r, n in zip(raw, lens):
        pos = torch.arange(n)
        q = A.norm_rope(r["q"], wq, pos, table.cpu()).to(torch.bfloat16)
        k = A.norm_rope(r["k"], wk, pos, table.cpu()).to(torch.bfloat16)
        w, s = A.attention_one(q, k, r["v"], None)
        want.append(w)
        size.append(s)
    done = [0, 0]
    for step in ([70, 50], [1, 60], [4, 30], [0, 0]):
        step = [min(x, n - a) for x, n, a in zip(step, lens, done)]
        rows = [slice(a, a + x) for a, x in zip(done, step)]
        cat = lambda x: torch.cat([r[x][i] for r, i in zip(raw, rows)]).to(cuda)  # noqa: E731
        pos = torch.cat([torch.arange(i.start, i.stop) for i in rows])
        slots = torch.cat([bt[n, torch.arange(i.start, i.stop) // page] * page
                           + torch.arange(i.start, i.stop) % page for n, i in enumerate(rows)])
        done = [i.stop for i in rows]
        q = pkg.attn_append(cat("q"), cat("k"), cat("v"), pos.to(cuda), table, slots.to(cuda), kc,
                            vc, wq.to(cuda), wk.to(cuda))
        out = pkg.attn_paged(q, kc, vc, bt.to(cuda), torch.tensor(done, device=cuda),
                             cu_seqlens=starts(step).to(cuda))
        ref = torch.cat([w[i] for w, i in zip(want, rows)])
        sz = torch.cat([w[i] for w, i in zip(size, rows)])
        # q and k are rounded from fp32 here and from fp64 in the oracle: a value next to a
        # border may round the other way, one bf16 step of one of 128 products: 2^-7 * |q k|
        # scale <= 2^-7 * 16 * 0.09 = 2^-6.5 in a score at most, rarely
        off = (out.cpu().double() - ref).abs()
        assert (off <= 2.0 ** -8 * ref.abs() + (2.0 ** -8 + 2.0 ** -6) * sz + 1e-30).all()
        if ref.numel():
            assert off.norm() <= 5e-3 * ref.norm()
    whole = pkg.attn_qk_norm_rope(torch.cat([r["q"] for r in raw]).to(cuda),
                                  torch.cat([r["k"] for r in raw]).to(cuda),
                                  torch.cat([torch.arange(n) for n in lens]).to(cuda), table,
                                  wq.to(cuda), wk.to(cuda))
    out = pkg.attn_prefill(*whole, torch.cat([r["v"] for r in raw]).to(cuda), starts(lens).to(cuda))
    ref = torch.cat(want)
    assert (out.cpu().double() - ref).norm() <= 5e-3 * ref.norm()


def test_refusals(cuda):
    pkg = load_pkg()
    d = inputs(4, 4, 2, seed=1)
    g = {k: v.to(cuda) for k, v in d.items()}
    kc = torch.zeros(2, 16, 2, D, dtype=torch.bfloat16, device=cuda)
    base = dict(q=g["q"], k=g["k"], v=g["v"], pos=g["pos"], table=g["table"],
                slots=torch.arange(4, device=cuda), kc=kc, vc=kc.clone(), wq=g["wq"], wk=g["wk"])

    def call(eps=1e-6, q_out=None, **kw):
        a = {**base, **kw}
        return pkg.attn_append(a["q"], a["k"], a["v"], a["pos"], a["table"], a["slots"], a["kc"],
                               a["vc"], a["wq"], a["wk"], q_out, eps=eps)
    call()
    for kw, err in ((dict(q=g["q"].half()), TypeError), (dict(q=g["q"][:, :3]), ValueError),
                    (dict(k=g["k"][:3]), ValueError), (dict(v=None), TypeError),
                    (dict(pos=g["pos"].float()), TypeError), (dict(pos=g["pos"][:3]), ValueError),
                    (dict(pos=g["pos"].cpu()), ValueError), (dict(table=g["table"].double()), TypeError),
                    (dict(table=g["table"][:, :63]), ValueError),
                    (dict(table=g["table"][:, :7].contiguous()), ValueError),
                    (dict(slots=None), TypeError), (dict(slots=base["slots"].float()), TypeError),
                    (dict(kc=None), TypeError), (dict(kc=kc.transpose(1, 2)), ValueError),
                    (dict(kc=kc.float()), TypeError), (dict(vc=kc[:1]), ValueError),
                    (dict(wq=g["wq"].bfloat16()), TypeError), (dict(wk=g["wk"][:64]), ValueError),
                    (dict(eps=-1.0), ValueError), (dict(eps=float("nan")), ValueError),
                    (dict(q_out=g["q"][:2]), ValueError)):
        with pytest.raises(err):
            call(**kw)
    e = pkg.attn_qk_norm_rope(g["q"][:0], g["k"][:0], g["pos"][:0], g["table"])
    assert e[0].shape == (0, 4, D) and e[1].shape == (0, 2, D)
    # a table without rows: every token is padding
    z = pkg.attn_qk_norm_rope(g["q"], g["k"], g["pos"], g["table"][:0])
    assert (z[0] == 0).all() and (z[1] == 0).all()
