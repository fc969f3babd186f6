"""GPU: attn_qk_norm_rope and attn_append at serving sizes, where a half-warp takes four heads at a
time, of one batch (600 tokens) or of all of a token's heads in turn (4096 and more): every layout
of the pairs, with and without norm, keys returned, cached and in place, last batches that are not
full.  Sampled tokens against the 64-bit oracle, the rest of the outputs for what they must hold."""
import pytest
import torch

from attn_util import D
from conftest import load_pkg
from test_rope_gpu import close, inputs, reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", [600, 4096, 4099])
@pytest.mark.parametrize("hq,hk", [(5, 1), (12, 4), (16, 2)])
@pytest.mark.parametrize("rd", [6, 64, 96, 100, 128])
@pytest.mark.parametrize("inter", [False, True])
def test_forms(cuda, t, hq, hk, rd, inter):
    pkg = load_pkg()
    d = inputs(t, hq, hk, seed=t + hq + rd, table_rows=5000, rd=rd)
    d["pos"][11], d["pos"][t - 2] = -1, 5000  # padding
    g = {k: v.to(cuda) for k, v in d.items()}
    at = torch.tensor([*range(16), *range(16, t, 151), t - 2, t - 1])
    page, pages = 48, (t + 47) // 48 + 2
    slots = torch.randperm(pages * page, generator=torch.Generator().manual_seed(rd))[:t]
    slots[5], slots[9] = -1, pages * page  # nowhere
    held = torch.ones(t, dtype=torch.bool)
    held[[5, 9, 11, t - 2]] = False
    kept = at[held[at]]
    free = torch.ones(pages * page, dtype=torch.bool)
    free[slots[held]] = False

    def ref(x, w, rows):
        return reference(dict(d, **{x: d[x][rows]}, pos=d["pos"][rows]), x, w, inter)

    for norm in (True, False):
        wq, wk = (g["wq"], g["wk"]) if norm else (None, None)
        rq, rk = ref("q", "wq" if norm else None, at), ref("k", "wk" if norm else None, at)
        # returned
        q, k = pkg.attn_qk_norm_rope(g["q"], g["k"], g["pos"], g["table"], wq, wk, interleaved=inter)
        close(q[at.to(cuda)], *rq)
        close(k[at.to(cuda)], *rk)
        # in place, in a fused projection
        fused = torch.cat([g["q"].flatten(1), g["k"].flatten(1), g["v"].flatten(1)], dim=1)
        x = fused[:, :hq * D].view(t, hq, D)
        y = fused[:, hq * D:(hq + hk) * D].view(t, hk, D)
        pkg.attn_qk_norm_rope(x, y, g["pos"], g["table"], wq, wk, x, y, interleaved=inter)
        assert torch.equal(x, q) and torch.equal(y, k)
        assert torch.equal(fused[:, (hq + hk) * D:], g["v"].flatten(1))
        # cached, q in place (the same arithmetic: bit for bit as returned)
        kc = torch.full((pages, page, hk, D), 9.0, dtype=torch.bfloat16, device=cuda)
        vc = kc.clone()
        x = g["q"].clone()
        pkg.attn_append(x, g["k"], g["v"], g["pos"], g["table"], slots.to(cuda), kc, vc, wq, wk, x,
                        interleaved=inter)
        assert torch.equal(x, q) and (x[11] == 0).all() and (x[t - 2] == 0).all()
        kc, vc = kc.view(-1, hk, D), vc.view(-1, hk, D)
        where = slots[held].to(cuda)
        assert torch.equal(kc[where], k[held.to(cuda)])
        assert torch.equal(vc[where], g["v"][held.to(cuda)])
        assert (kc[free.to(cuda)] == 9).all() and (vc[free.to(cuda)] == 9).all()
        close(kc[slots[kept].to(cuda)], *ref("k", "wk" if norm else None, kept))


@pytest.mark.parametrize("t", [37, 600, 4099])
@pytest.mark.parametrize("which", ["q", "k"])
def test_one_weight_only(cuda, t, which):
    """With one of the weights only that side is normalised; the other turns as without any."""
    pkg = load_pkg()
    d = inputs(t, 6, 2, seed=t, rd=64)
    g = {k: v.to(cuda) for k, v in d.items()}
    wq, wk = (g["wq"], None) if which == "q" else (None, g["wk"])
    both = pkg.attn_qk_norm_rope(g["q"], g["k"], g["pos"], g["table"], g["wq"], g["wk"])
    none = pkg.attn_qk_norm_rope(g["q"], g["k"], g["pos"], g["table"])
    one = pkg.attn_qk_norm_rope(g["q"], g["k"], g["pos"], g["table"], wq, wk)
    assert torch.equal(one[0], (both if which == "q" else none)[0])
    assert torch.equal(one[1], (none if which == "q" else both)[1])
