"""Inputs and the comparison shared by the attention tests.

Tolerances, from arithmetic.  The kernels form the scores and sums in fp32 and round the
probabilities to bf16 for their product with v (relative 2^-8 each, so 2^-8 sum_j p_j |v_j|
at most), and the output to bf16 (2^-8 of it).  The fp32 scores are off by at most 128
roundings of sum_d |q_d k_d| * scale <= 64 in these inputs, 128 * 64 * 2^-24 = 2^-11 of each
probability, twice for the normalisation; partial results joined in fp32 add less than that
again: 2^-9 sum_j p_j |v_j| in all.  Over a whole tensor the roundings are independent:
2^-8 / sqrt(3) each in norm, 3.2e-3 for the two of them, held to 4e-3 (with the fp32 part)."""
import torch

from oracle import attn_oracle as A

BF16 = 2.0 ** -8
D = 128


def check(out, ref, size, what=""):
    out = out.detach().cpu().double().reshape(ref.shape)
    assert torch.isfinite(out).all(), f"{what}: not finite"
    off = (out - ref).abs()
    limit = BF16 * ref.abs() + (BF16 + 2.0 ** -9) * size + 1e-30
    worst = (off / limit).max().item() if off.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst:.2f} of the limit at {int((off / limit).argmax())}"
    norm = ref.norm().item()
    if norm > 0 and ref.numel() >= 2048:
        assert off.norm().item() <= 4e-3 * norm, f"{what}: {off.norm().item() / norm:.2e} in norm"


def starts(lens, dtype=torch.int32):
    return torch.tensor([0] + torch.tensor(list(lens), dtype=torch.int64).cumsum(0).tolist(),
                        dtype=dtype)


def randn(shape, g, std=1.0):
    return (torch.randn(shape, generator=g) * std).to(torch.bfloat16)


def prefill_inputs(lens, hq, hk, seed, extra=0, std=1.5):
    g = torch.Generator().manual_seed(seed)
    t = sum(lens) + extra
    return dict(q=randn((t, hq, D), g, std), k=randn((t, hk, D), g, std), v=randn((t, hk, D), g),
                cu=starts(lens))


def paged_inputs(q_lens, kv_lens, hq, hk, page, seed, extra_rows=0, spare=3, stale=None, std=1.5):
    """Pages in random order; table entries that are not used are -1; `stale`: what the rest
    of a sequence's last page and the spare pages hold (None: more random values)."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-max(x, 0) // page) for x in kv_lens]
    pages = sum(need) + spare
    d = dict(q=randn((sum(q_lens) + extra_rows, hq, D), g, std), cu=starts(q_lens),
             k_cache=randn((pages, page, hk, D), g, std), v_cache=randn((pages, page, hk, D), g),
             kv_lens=torch.tensor(kv_lens, dtype=torch.int32))
    order = torch.randperm(pages, generator=g).to(torch.int32)
    table = torch.full((len(kv_lens), max(max(need, default=0), 1)), -1, dtype=torch.int32)
    at = 0
    for n, k in enumerate(need):
        table[n, :k] = order[at:at + k]
        at += k
    if stale is not None:
        used = torch.zeros(pages, page, dtype=torch.bool)
        for n, x in enumerate(kv_lens):
            for j in range(x):
                used[table[n, j // page], j % page] = True
        d["k_cache"][~used] = stale
        d["v_cache"][~used] = stale
    d["table"] = table
    return d


def on(d, dev):
    return {k: v.to(dev) for k, v in d.items()}


def paged_ref(d, scale=None):
    return A.paged(d["q"], d["k_cache"], d["v_cache"], d["table"], d["kv_lens"], d["cu"], scale)
