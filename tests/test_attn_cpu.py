"""CPU: the attention entry points' argument checks before any launch, the rope tables, and
the oracle against torch's own operators."""
import math

import pytest
import torch
import torch.nn.functional as F

from attn_util import paged_inputs, paged_ref, prefill_inputs, starts
from conftest import load_pkg
from oracle import attn_oracle as A

FAKE = 0x10000


def prefill_call(**kw):
    a = dict(q=FAKE, k=FAKE, v=FAKE, cu=FAKE, cu64=0, scale=0.0, out=FAKE, t=10, n=1, hq=8, hk=2,
             d=128, qs=1024, ks=256, vs=256, os=1024, ws=None, wsb=0, stream=None)
    a.update(kw)
    return load_pkg().LIB.gdn_attn_prefill_launch(*a.values())


def paged_call(**kw):
    a = dict(q=FAKE, k=FAKE, v=FAKE, table=FAKE, ts=4, lens=FAKE, lens64=0, cu=FAKE, cu64=0,
             scale=0.0, out=FAKE, t=10, n=2, width=4, pages=9, page=16, kps=16 * 256, vps=16 * 256,
             hq=8, hk=2, d=128, qs=1024, os=1024, ws=None, wsb=0, stream=None)
    a.update(kw)
    return load_pkg().LIB.gdn_attn_paged_launch(*a.values())


def rope_call(**kw):
    a = dict(q=FAKE, k=FAKE, v=FAKE, pos=FAKE, pos64=0, table=FAKE, rows=100, wq=None, wk=None,
             eps=1e-6, inter=0, qo=FAKE, ko=None, slots=FAKE, slots64=0, kc=FAKE, vc=FAKE, pages=4,
             page=16, kps=16 * 256, vps=16 * 256, t=3, hq=8, hk=2, d=128, rd=64, qs=1024, ks=256,
             vs=256, qos=1024, kos=0, stream=None)
    a.update(kw)
    return load_pkg().LIB.gdn_attn_qk_norm_rope_launch(*a.values())


@pytest.mark.parametrize("call,bad,unsupported", [
    (prefill_call,
     [dict(q=None), dict(k=None), dict(v=None), dict(cu=None), dict(out=None), dict(t=-1), dict(n=-1),
      dict(q=FAKE + 8), dict(k=FAKE + 2), dict(v=FAKE + 4), dict(out=FAKE + 8), dict(cu=FAKE + 2),
      dict(cu=FAKE + 4, cu64=1), dict(qs=1023), dict(qs=1016), dict(ks=248), dict(vs=260),
      dict(os=1000), dict(hq=0), dict(hk=0)],
     [dict(d=64), dict(d=256), dict(hk=3), dict(hq=65, hk=1, qs=65 * 128)]),
    (paged_call,
     [dict(q=None), dict(k=None), dict(v=None), dict(table=None), dict(lens=None), dict(out=None),
      dict(t=-1), dict(n=-1), dict(width=-1), dict(pages=-1), dict(page=0), dict(q=FAKE + 8),
      dict(k=FAKE + 8), dict(table=FAKE + 2), dict(lens=FAKE + 4, lens64=1), dict(cu=FAKE + 1),
      dict(cu=None, t=11), dict(ts=3), dict(kps=15 * 256), dict(vps=16 * 256 + 4), dict(qs=1020),
      dict(os=512), dict(width=1 << 28, ts=1 << 28)],
     [dict(d=64), dict(hk=3), dict(page=12, kps=4096, vps=4096), dict(page=1)]),
    (rope_call,
     [dict(q=None), dict(k=None), dict(v=None), dict(pos=None), dict(table=None), dict(qo=None),
      dict(slots=None), dict(vc=None), dict(kc=None), dict(t=-1), dict(rows=-1), dict(eps=-1.0),
      dict(eps=float("nan")), dict(q=FAKE + 8), dict(wq=FAKE + 4), dict(pos=FAKE + 4, pos64=1),
      dict(kps=15 * 256), dict(page=0), dict(qs=1016), dict(qos=1028), dict(table=FAKE + 2)],
     [dict(d=64), dict(rd=0), dict(rd=63), dict(rd=130), dict(hk=3)])])
def test_entry_points_refuse_before_launch(call, bad, unsupported):
    for kw in bad:
        assert call(**kw) == -1, kw
    for kw in unsupported:
        assert call(**kw) == -2, kw
    assert call(t=0) == 0  # nothing to do


@pytest.mark.parametrize("t,n,hq,hk", [(1, 1, 1, 1), (10, 1, 8, 2), (10, 2, 8, 2), (64, 64, 8, 2),
                                       (128, 32, 8, 2), (5000, 3, 64, 1), (1500, 1000, 2, 2)])
def test_workspace(t, n, hq, hk):
    """The size is enough for either form of a call: one byte less, none or a misaligned one is
    refused (and with the whole of it the next refusal comes first: alignment)."""
    need = load_pkg().LIB.gdn_attn_workspace_size(t, n, hq, hk)
    assert need > 0
    kw = dict(t=t, n=n, hq=hq, hk=hk, qs=hq * 128, os=hq * 128)
    calls = [(prefill_call, dict(kw, ks=hk * 128, vs=hk * 128)),
             (paged_call, dict(kw, kps=16 * hk * 128, vps=16 * hk * 128))]
    if t % n == 0:
        calls.append((paged_call, dict(calls[1][1], cu=None)))
    for call, a in calls:
        assert call(**a, ws=None, wsb=need) == -4
        assert call(**a, ws=FAKE, wsb=0) == -4
        assert call(**a, ws=FAKE, wsb=need - 1) == -4
        assert call(**a, ws=FAKE + 8, wsb=need) == -1


@pytest.mark.parametrize("bad", [(0, 1, 8, 2), (-3, 1, 8, 2), (10, 0, 8, 2), (10, 1, 8, 0),
                                 (10, 1, 1, 2), (10, 1, 0, 0)])
def test_workspace_of_nothing(bad):
    assert load_pkg().LIB.gdn_attn_workspace_size(*bad) == 0


def test_host_functions_refuse_cpu_tensors():
    pkg = load_pkg()
    d = prefill_inputs([4], 4, 2, seed=0)
    with pytest.raises(ValueError, match="CUDA"):
        pkg.attn_prefill(d["q"], d["k"], d["v"], d["cu"])
    with pytest.raises(TypeError):
        pkg.attn_prefill([1], d["k"], d["v"], d["cu"])
    with pytest.raises(ValueError, match="CUDA"):
        pkg.attn_qk_norm_rope(d["q"], d["k"], torch.arange(4), torch.zeros(8, 64))


@pytest.mark.parametrize("rd", [2, 64, 128])
def test_rope_table(rd):
    pkg = load_pkg()
    n = 50
    pos = torch.arange(n, dtype=torch.float64)[:, None]
    inv = 1e4 ** (-torch.arange(0, rd, 2, dtype=torch.float64) / rd)
    t = pkg.rope_table(n, rd, device="cpu")
    assert t.dtype == torch.float32 and t.shape == (n, rd)
    assert torch.equal(t, torch.cat([(pos * inv).cos(), (pos * inv).sin()], 1).float())
    lin = pkg.rope_table(n, rd, scaling="linear", factor=4.0, device="cpu")
    assert torch.equal(lin, torch.cat([(pos * (inv / 4)).cos(), (pos * (inv / 4)).sin()], 1).float())
    if rd > 2:
        # the ends of the spectrum: the highest frequency kept, the lowest divided
        ntk = pkg.rope_table(n, rd, scaling="ntk", factor=4.0, device="cpu").double()
        half = rd // 2
        assert torch.allclose(ntk[:, half], pos[:, 0].sin(), atol=1e-6)
        assert torch.allclose(ntk[:, -1], (pos[:, 0] * inv[-1] / 4).sin(), atol=1e-6)


def test_yarn_table():
    """Factor 8 from 4096 tokens: fast frequencies kept, slow ones divided by 8, a ramp in
    between, cosines and sines times 0.1 ln 8 + 1."""
    pkg = load_pkg()
    rd, factor, orig = 128, 8.0, 4096
    m = 0.1 * math.log(factor) + 1
    t = pkg.rope_table(2, rd, scaling="yarn", factor=factor, original_max_position=orig, device="cpu")
    got = torch.atan2(t[1, 64:].double(), t[1, :64].double())
    assert torch.allclose(t[0, :64].double(), torch.full((64,), m, dtype=torch.float64), atol=1e-6)
    inv = 1e4 ** (-torch.arange(0, rd, 2, dtype=torch.float64) / rd)
    turns = orig * inv / (2 * math.pi)
    fast, slow = turns > 40, turns < 0.8
    assert fast.sum() > 10 and slow.sum() > 5
    assert torch.allclose(got[fast], inv[fast], rtol=1e-6)
    assert torch.allclose(got[slow], inv[slow] / factor, rtol=1e-5)
    mid = ~fast & ~slow
    assert ((got[mid] <= inv[mid] * (1 + 1e-6)) & (got[mid] >= inv[mid] / factor * (1 - 1e-6))).all()
    one = pkg.rope_table(2, rd, scaling="yarn", factor=8.0, original_max_position=orig,
                         attention_factor=1.0, device="cpu")
    assert torch.allclose(one * m, t, rtol=1e-6)
    far = pkg.rope_table(200001, 2, device="cpu")  # exact at far positions
    assert abs(far[200000, 1].item() - math.sin(200000)) < 1e-7


@pytest.mark.parametrize("kw", [dict(rotary_dim=3), dict(rotary_dim=0), dict(rotary_dim=130),
                                dict(max_position=-1), dict(scaling="cubic"), dict(base=1.0),
                                dict(factor=0.5), dict(scaling="yarn", factor=2.0),
                                dict(attention_factor=1.0)])
def test_rope_table_refusals(kw):
    a = {**dict(max_position=8, rotary_dim=64, device="cpu"), **kw}
    with pytest.raises(ValueError):
        load_pkg().rope_table(a.pop("max_position"), a.pop("rotary_dim"), **a)


def test_oracle_against_torch():
    d = prefill_inputs([6, 0, 9], 4, 2, seed=1)
    out, size = A.prefill(d["q"], d["k"], d["v"], d["cu"])
    for a, b in ((0, 6), (6, 15)):
        q, k, v = (d[x][a:b].double().transpose(0, 1) for x in ("q", "k", "v"))
        k, v = k.repeat_interleave(2, 0), v.repeat_interleave(2, 0)
        want = F.scaled_dot_product_attention(q, k, v, is_causal=True).transpose(0, 1)
        assert torch.allclose(out[a:b], want, atol=1e-12)
    assert (size >= out.abs() - 1e-12).all()
    p = paged_inputs([2, 5, 3], [9, 3, 0], 4, 2, 8, seed=2, stale=float("nan"))
    out, _ = paged_ref(p)
    assert (out[2:4] == 0).all() and (out[7:] == 0).all()  # rows that see nothing
    assert torch.isfinite(out).all() and (out[4:7] != 0).any()
    assert starts([2, 5]).tolist() == [0, 2, 7]


def test_oracle_rotation_is_a_complex_product():
    x = torch.randn(3, 2, 128, dtype=torch.float64)
    pos = torch.tensor([0, 3, 7])
    t = load_pkg().rope_table(8, 128, device="cpu")
    y = A.norm_rope(x, None, pos, t, interleaved=True)
    z = torch.view_as_complex(x.view(3, 2, 64, 2))
    w = torch.complex(t[pos, :64].double(), t[pos, 64:].double())[:, None]
    assert torch.allclose(torch.view_as_real(z * w).flatten(-2), y, atol=1e-12)
    h = A.norm_rope(torch.cat([x[..., 0::2], x[..., 1::2]], -1), None, pos, t)
    assert torch.allclose(h, torch.cat([y[..., 0::2], y[..., 1::2]], -1), atol=1e-12)
