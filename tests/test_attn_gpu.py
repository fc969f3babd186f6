"""GPU: attn_prefill and attn_paged against the 64-bit oracle."""
import pytest
import torch

from attn_util import D, check, on, paged_inputs, paged_ref, prefill_inputs, starts
from conftest import load_pkg
from oracle import attn_oracle as A

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ whole prompts
@pytest.mark.parametrize("lens", [[1], [1, 0, 2], [127, 128, 129], [0, 5, 300, 0, 33, 256, 1],
                                  [700], [3] * 40, [257, 1, 384]])
@pytest.mark.parametrize("hq,hk", [(4, 1), (3, 3), (6, 2)])
def test_prefill(cuda, lens, hq, hk):
    pkg = load_pkg()
    d = prefill_inputs(lens, hq, hk, seed=len(lens) + hq)
    ref, size = A.prefill(d["q"], d["k"], d["v"], d["cu"])
    g = on(d, cuda)
    out = pkg.attn_prefill(g["q"], g["k"], g["v"], g["cu"])
    torch.cuda.synchronize()
    assert pkg.device_error() == 0
    check(out, ref, size, f"{lens} {hq}/{hk}")


@pytest.mark.parametrize("hq,hk", [(1, 1), (5, 1), (16, 2), (16, 1), (24, 1), (64, 1), (48, 1)])
def test_prefill_head_groups(cuda, hq, hk):
    pkg = load_pkg()
    lens = [70, 129, 12]
    d = prefill_inputs(lens, hq, hk, seed=hq)
    ref, size = A.prefill(d["q"], d["k"], d["v"], d["cu"], 0.05)
    g = on(d, cuda)
    out = pkg.attn_prefill(g["q"], g["k"], g["v"], g["cu"].long(), 0.05)
    torch.cuda.synchronize()
    assert pkg.device_error() == 0
    check(out, ref, size, f"{hq}/{hk}")


def test_prefill_long_matches_blocks_of_the_oracle(cuda):
    """One 2500-token prompt: several tiles of rows and keys, split between CTAs."""
    pkg = load_pkg()
    d = prefill_inputs([2500], 4, 2, seed=9)
    ref, size = A.prefill(d["q"], d["k"], d["v"], d["cu"])
    g = on(d, cuda)
    check(pkg.attn_prefill(g["q"], g["k"], g["v"], g["cu"]), ref, size)


def test_prefill_strided_views_and_rows_behind_the_last(cuda):
    pkg = load_pkg()
    lens, extra, hq, hk = [90, 0, 41], 7, 8, 2
    d = prefill_inputs(lens, hq, hk, seed=3, extra=extra)
    ref, size = A.prefill(d["q"], d["k"], d["v"], d["cu"])
    t = sum(lens) + extra
    for width, dtype in ((hq + 2 * hk, torch.int32), (hq + 2 * hk + 1, torch.int64)):
        fused = torch.full((t, width * D), float("nan"), dtype=torch.bfloat16, device=cuda)
        q = fused[:, :hq * D].view(t, hq, D)
        k = fused[:, hq * D:(hq + hk) * D].view(t, hk, D)
        v = fused[:, (hq + hk) * D:(hq + 2 * hk) * D].view(t, hk, D)
        for x, y in ((q, d["q"]), (k, d["k"]), (v, d["v"])):
            x[:t - extra].copy_(y[:t - extra])  # the rows behind stay NaN
        base = torch.full((t, 2 * hq, D), 7.0, dtype=torch.bfloat16, device=cuda)
        outs = [base[:, :hq], torch.full((t, hq, D + 4), 7.0, dtype=torch.bfloat16,
                                         device=cuda)[..., :D]]  # strided rows; a copied layout
        for out in outs:
            r = pkg.attn_prefill(q, k, v, d["cu"].to(cuda, dtype), None, out)
            assert r is out
            check(out[:t - extra], ref[:t - extra], size[:t - extra])
            assert (out[t - extra:] == 7).all()
        assert (base[:, hq:] == 7).all()
    # heads that are not dense, and rows that are not 16-byte aligned, are copied
    odd = torch.empty(t * hk * D + 1, dtype=torch.bfloat16, device=cuda)[1:].view(t, hk, D)
    odd.copy_(d["k"])
    out = pkg.attn_prefill(d["q"].to(cuda).transpose(0, 1).contiguous().transpose(0, 1), odd,
                           d["v"].to(cuda), d["cu"].to(cuda))
    check(out[:t - extra], ref[:t - extra], size[:t - extra])


def test_prefill_large_scores_and_equal_scores(cuda):
    """Scores of several hundred (one key takes all), and identical keys (the mean)."""
    pkg = load_pkg()
    d = prefill_inputs([300], 2, 1, seed=5)
    g = on(d, cuda)
    out = pkg.attn_prefill(g["q"], g["k"], g["v"], g["cu"], 30.0)
    ref, _ = A.prefill(d["q"], d["k"], d["v"], d["cu"], 30.0)
    # scores up to 30 * 128 * 1.5^2 * ~5: fp32 leaves their probabilities 128 * 2^-24 * 4e4
    # off at most, 0.3 in the exponent: compare where one key has all but 2^-20
    z = torch.einsum("ihd,jd->hij", d["q"].double(), d["k"][:, 0].double()) * 30
    z.masked_fill_(~torch.ones(300, 300, dtype=torch.bool).tril(), -torch.inf)
    top = z.topk(2, dim=-1).values
    sure = ((top[..., 0] - top[..., 1]) > 16).T  # [i, h]
    assert sure.float().mean() > 0.9
    off = (out.cpu().double() - ref)[sure].abs()
    assert (off <= 2.0 ** -7 * ref[sure].abs() + 2.0 ** -12).all()
    k = g["k"][:1].expand(300, 1, D).contiguous()
    out = pkg.attn_prefill(g["q"], k, g["v"], g["cu"])
    ref, size = A.prefill(d["q"], k.cpu(), d["v"], d["cu"])
    check(out, ref, size)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), torch.finfo(torch.bfloat16).min])
def test_prefill_other_sequences_do_not_leak(cuda, bad):
    """A sequence of NaN, infinities or lowest values leaves its neighbours bit for bit."""
    pkg = load_pkg()
    lens = [100, 60, 131]
    g = on(prefill_inputs(lens, 4, 2, seed=6), cuda)
    a = pkg.attn_prefill(g["q"], g["k"], g["v"], g["cu"])
    for x in ("q", "k", "v"):
        g[x][100:160] = bad
    b = pkg.attn_prefill(g["q"], g["k"], g["v"], g["cu"])
    assert torch.equal(a[:100], b[:100]) and torch.equal(a[160:], b[160:])


# ------------------------------------------------------------------ paged cache
PAGED = [  # new tokens, cached tokens, page
    ([1], [1], 16), ([1, 1, 1], [5, 0, 700], 16), ([1] * 9, [1, 63, 64, 65, 127, 128, 129, 300, 17], 8),
    ([4, 4, 4], [4, 130, 999], 48), ([7, 0, 1, 3], [7, 40, 513, 2], 64), ([33, 1, 129], [33, 800, 129], 128),
    ([200], [1500], 24), ([17, 300, 5], [600, 300, 3], 256), ([2, 2], [1, 2000], 32)]


@pytest.mark.parametrize("q_lens,kv_lens,page", PAGED)
@pytest.mark.parametrize("hq,hk", [(4, 1), (3, 3), (16, 2)])
def test_paged(cuda, q_lens, kv_lens, page, hq, hk):
    """Stale rows hold NaN, unused table entries -1; some rows see nothing."""
    pkg = load_pkg()
    d = paged_inputs(q_lens, kv_lens, hq, hk, page, seed=page + hq, stale=float("nan"))
    ref, size = paged_ref(d)
    g = on(d, cuda)
    out = pkg.attn_paged(g["q"], g["k_cache"], g["v_cache"], g["table"], g["kv_lens"],
                         cu_seqlens=g["cu"])
    torch.cuda.synchronize()
    assert pkg.device_error() == 0
    check(out, ref, size, f"{q_lens} {kv_lens} page {page} {hq}/{hk}")
    if len(set(q_lens)) == 1:  # the 4-D form is the same call
        x = g["q"].view(len(q_lens), q_lens[0], hq, D)
        same = pkg.attn_paged(x, g["k_cache"], g["v_cache"], g["table"], g["kv_lens"].long())
        assert same.shape == x.shape and torch.equal(same.view(out.shape), out)


@pytest.mark.parametrize("hq,hk", [(5, 1), (64, 1), (24, 1), (32, 32)])
@pytest.mark.parametrize("q_len", [1, 2, 6])
def test_paged_head_groups(cuda, hq, hk, q_len):
    pkg = load_pkg()
    d = paged_inputs([q_len] * 3, [q_len, 77, 400], hq, hk, 16, seed=hq + q_len, stale=float("inf"))
    ref, size = paged_ref(d, 0.11)
    g = on(d, cuda)
    out = pkg.attn_paged(g["q"], g["k_cache"], g["v_cache"], g["table"], g["kv_lens"], 0.11,
                         cu_seqlens=g["cu"].long())
    check(out, ref, size, f"{hq}/{hk} {q_len}")


@pytest.mark.parametrize("q_len", [1, 3, 50])
def test_paged_long_context_is_split_and_joined(cuda, q_len):
    pkg = load_pkg()
    d = paged_inputs([q_len], [30011], 8, 1, 64, seed=q_len, stale=float("nan"))
    ref, size = paged_ref(d)
    g = on(d, cuda)
    args = (g["q"], g["k_cache"], g["v_cache"], g["table"], g["kv_lens"])
    out = pkg.attn_paged(*args, cu_seqlens=g["cu"])
    check(out, ref, size)
    for _ in range(3):  # the join has a fixed order
        assert torch.equal(out, pkg.attn_paged(*args, cu_seqlens=g["cu"]))


@pytest.mark.parametrize("page", [8, 64])
@pytest.mark.parametrize("q_lens", [[9, 29, 17, 32], [1059, 29, 300, 12]])
def test_paged_last_tile_of_a_block_of_one_row_tile(cuda, page, q_lens):
    """Blocks of one row tile, whose key tiles two warp groups take in turn, over contexts that
    end inside a tile: the values behind the end are zeroed where they arrived, not in the
    stage's tile before (many small pages make those arrive late)."""
    pkg = load_pkg()
    for seed in range(4):
        kv_lens = [2884, 2884 + seed, 1414, 2500 + 31 * seed]
        d = paged_inputs(q_lens, kv_lens, 8, 2, page, seed=seed, stale=float("nan"))
        ref, size = paged_ref(d)
        g = on(d, cuda)
        out = pkg.attn_paged(g["q"], g["k_cache"], g["v_cache"], g["table"], g["kv_lens"],
                             cu_seqlens=g["cu"])
        check(out, ref, size, f"seed {seed}")


@pytest.mark.parametrize("q_len", [1, 40])
def test_paged_bad_pages_read_as_zeros(cuda, q_len):
    """Page numbers outside the cache (checked on the device, nothing is read for them)."""
    pkg = load_pkg()
    d = paged_inputs([q_len, q_len], [200, 90], 4, 2, 16, seed=2)
    pages = d["k_cache"].shape[0]
    d["table"][0, 2] = pages
    d["table"][0, 5] = -7
    d["table"][1, 0] = 2 ** 31 - 1
    d["table"][1, 5] = -2 ** 31
    ref, size = paged_ref(d)
    g = on(d, cuda)
    out = pkg.attn_paged(g["q"], g["k_cache"], g["v_cache"], g["table"], g["kv_lens"],
                         cu_seqlens=g["cu"])
    check(out, ref, size)


@pytest.mark.parametrize("q_len", [1, 30])
def test_paged_views_lengths_beyond_the_table_and_rows_behind(cuda, q_len):
    """K and V in one buffer of pages, a table slice, a kv_len beyond the table (clamped),
    a negative one (nothing seen), padded query rows left as they were."""
    pkg = load_pkg()
    d = paged_inputs([q_len] * 3, [130, 64, 96], 8, 2, 16, seed=8, extra_rows=5)
    both = torch.stack([d["k_cache"], d["v_cache"]], dim=1).to(cuda)
    table = torch.full((6, 20), -1, dtype=torch.int32)
    table[::2, :9] = d["table"]
    view = table.to(cuda)[::2, :8]  # 128 tokens at most
    d["kv_lens"][1] = -5
    d["table"] = d["table"][:, :8]
    ref, size = paged_ref(d)
    t = 3 * q_len
    q = torch.full((t + 5, 12, D), float("nan"), dtype=torch.bfloat16, device=cuda)
    q[:t, 2:10] = d["q"][:t].to(cuda)
    out = torch.full((t + 5, 12, D), 3.0, dtype=torch.bfloat16, device=cuda)
    r = pkg.attn_paged(q[:, 2:10], both[:, 0], both[:, 1], view, d["kv_lens"].to(cuda, torch.int64),
                       None, out[:, 2:10], cu_seqlens=d["cu"].to(cuda))
    check(r[:t], ref[:t], size[:t])
    assert (r[q_len:2 * q_len] == 0).all()
    assert (out[t:] == 3).all() and (out[:, :2] == 3).all() and (out[:, 10:] == 3).all()
    # 4-D views whose tokens are not one stride apart are copied, in and out
    x = torch.zeros(3, q_len + 1, 8, D, dtype=torch.bfloat16, device=cuda)
    x[:, :q_len] = d["q"][:t].view(3, q_len, 8, D).to(cuda)
    o4 = torch.full_like(x, 3.0)
    pkg.attn_paged(x[:, :q_len], both[:, 0], both[:, 1], view, d["kv_lens"].to(cuda), None,
                   o4[:, :q_len])
    # (padded rows count for the kernel's choice: the same values, not the same roundings)
    check(o4[:, :q_len].reshape(t, 8, D), ref[:t], size[:t])
    assert (o4[:, q_len:] == 3).all()


def test_mixed_batch_of_a_chunk_and_single_tokens(cuda):
    pkg = load_pkg()
    q_lens, kv_lens = [1] * 20 + [500] + [1] * 3, list(range(300, 320)) + [900] + [5, 1, 40]
    d = paged_inputs(q_lens, kv_lens, 4, 2, 16, seed=12, stale=float("nan"))
    ref, size = paged_ref(d)
    g = on(d, cuda)
    out = pkg.attn_paged(g["q"], g["k_cache"], g["v_cache"], g["table"], g["kv_lens"],
                         cu_seqlens=g["cu"])
    check(out, ref, size)


def test_many_sequences(cuda):
    """More sequences than any block has threads, most of them short, many empty."""
    pkg = load_pkg()
    q_lens = [(n * 7) % 3 for n in range(1500)]
    kv_lens = [q + (n * 13) % 40 if q else (n % 2) * 9 for n, q in enumerate(q_lens)]
    d = paged_inputs(q_lens, kv_lens, 2, 1, 8, seed=13, stale=float("nan"))
    ref, size = paged_ref(d)
    g = on(d, cuda)
    check(pkg.attn_paged(g["q"], g["k_cache"], g["v_cache"], g["table"], g["kv_lens"],
                         cu_seqlens=g["cu"]), ref, size)
    lens = [(n * 5) % 4 for n in range(1500)]
    d = prefill_inputs(lens, 2, 1, seed=14)
    ref, size = A.prefill(d["q"], d["k"], d["v"], d["cu"])
    g = on(d, cuda)
    check(pkg.attn_prefill(g["q"], g["k"], g["v"], g["cu"]), ref, size)


@pytest.mark.parametrize("hq,hk,q_len", [(8, 8, 1), (16, 8, 1), (16, 2, 2), (16, 2, 4)])
def test_short_contexts_with_long_ones_between(cuda, hq, hk, q_len):
    """Runs of contexts too short for some warps to have a chunk, then longer ones: every warp
    finds its next chunk, however many pieces it had none in."""
    pkg = load_pkg()
    n = 700
    kv_lens = [q_len + ((i * 37) % 90 if i % 11 else 200 + (i * 53) % 500) for i in range(n)]
    d = paged_inputs([q_len] * n, kv_lens, hq, hk, 16, seed=hq + q_len, stale=float("nan"))
    ref, size = paged_ref(d)
    g = on(d, cuda)
    for _ in range(3):
        out = pkg.attn_paged(g["q"], g["k_cache"], g["v_cache"], g["table"], g["kv_lens"],
                             cu_seqlens=g["cu"])
        torch.cuda.synchronize()
        assert pkg.device_error() == 0
        check(out, ref, size)
        x = g["q"].view(n, q_len, hq, D)  # the same number of tokens each: known to the host
        out = pkg.attn_paged(x, g["k_cache"], g["v_cache"], g["table"], g["kv_lens"])
        torch.cuda.synchronize()
        assert pkg.device_error() == 0
        check(out, ref, size)


@pytest.mark.parametrize("hq,hk,chunk", [(2, 2, 200), (2, 2, 300), (16, 2, 30), (16, 2, 140)])
def test_a_chunk_among_many_single_tokens(cuda, hq, hk, chunk):
    """Few tokens a sequence on average, on both sides of the longest chunk for which the
    kernel for few rows is taken."""
    pkg = load_pkg()
    q_lens = [1] * 90 + [chunk] + [1] * 60
    d = paged_inputs(q_lens, [x + (17 * i) % 150 for i, x in enumerate(q_lens)], hq, hk, 16,
                     seed=chunk, stale=float("nan"))
    ref, size = paged_ref(d)
    g = on(d, cuda)
    check(pkg.attn_paged(g["q"], g["k_cache"], g["v_cache"], g["table"], g["kv_lens"],
                         cu_seqlens=g["cu"]), ref, size)
    d = prefill_inputs(q_lens, hq, hk, seed=chunk + 1)
    ref, size = A.prefill(d["q"], d["k"], d["v"], d["cu"])
    g = on(d, cuda)
    check(pkg.attn_prefill(g["q"], g["k"], g["v"], g["cu"]), ref, size)
    torch.cuda.synchronize()
    assert pkg.device_error() == 0


@pytest.mark.parametrize("q_len", [1, 64])
def test_offsets_beyond_32_bits(cuda, q_len):
    """A cache of more than 2^32 elements in each of K and V: the last pages are read."""
    pkg = load_pkg()
    page, hk = 128, 8
    pages = 2 ** 32 // (page * hk * D) + 9
    k = torch.empty(pages, page, hk, D, dtype=torch.bfloat16, device=cuda)
    v = torch.empty_like(k)
    d = paged_inputs([q_len], [700], 8, hk, page, seed=4, spare=0)
    first = pages - d["k_cache"].shape[0]
    k[first:], v[first:] = d["k_cache"].to(cuda), d["v_cache"].to(cuda)
    ref, size = paged_ref(d)
    out = pkg.attn_paged(d["q"].to(cuda), k, v, (d["table"] + first).to(cuda),
                         d["kv_lens"].to(cuda), cu_seqlens=d["cu"].to(cuda))
    check(out, ref, size)


# ------------------------------------------------------------------ streams and graphs
@pytest.mark.parametrize("q_len", [1, 40])
def test_graph_replay_follows_the_lengths(cuda, q_len):
    """A captured call replays with other lengths, tables and values; two captured graphs
    replayed on two streams at once do not disturb one another."""
    pkg = load_pkg()
    made = []
    for seed in (1, 2):
        d = paged_inputs([q_len] * 4, [q_len, 100, 2000, 700], 8, 2, 16, seed=seed, stale=float("nan"))
        g = on(d, cuda)
        run = lambda g=g: pkg.attn_paged(g["q"], g["k_cache"], g["v_cache"], g["table"],  # noqa: E731
                                         g["kv_lens"], cu_seqlens=g["cu"])
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            run()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run()
        made.append((d, g, graph, out))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for lens in ([q_len, 100, 2000, 700], [60, 2, 1203, 0], [48, 112, 16, 650]):
        for d, g, _, out in made:
            d["kv_lens"] = torch.tensor(lens, dtype=torch.int32)
            g["kv_lens"].copy_(d["kv_lens"])
            out.zero_()
        torch.cuda.synchronize()
        for _ in range(5):
            for (_, _, graph, _), st in zip(made, streams):
                with torch.cuda.stream(st):
                    graph.replay()
        torch.cuda.synchronize()
        for d, g, _, out in made:
            # unused entries of the longest setup stay valid pages: only lengths shrink or the
            # stale rows (NaN) must not be needed
            clean = dict(d, k_cache=torch.nan_to_num(d["k_cache"]), v_cache=torch.nan_to_num(d["v_cache"]))
            if any(x > y for x, y in zip(lens, [q_len, 100, 2000, 700])):
                g["k_cache"].copy_(clean["k_cache"])
                g["v_cache"].copy_(clean["v_cache"])
                _ = [graph.replay() for _, _, graph, _ in made]
                torch.cuda.synchronize()
            ref, size = paged_ref(clean)
            check(out, ref, size, str(lens))


def test_graphs_that_share_memory(cuda):
    """Several calls in one graph, and two graphs of one memory pool replayed in turn, use the
    same scratch one after the other: every replay gives the eager calls' results."""
    pkg = load_pkg()
    p = on(prefill_inputs([1500, 3, 700], 8, 2, seed=30), cuda)
    sets = [on(paged_inputs([n] * 3, [5000, 900, 17 + n], 8, 2, 16, seed=31 + n), cuda)
            for n in (1, 3, 50)]

    def paged(g):
        return pkg.attn_paged(g["q"], g["k_cache"], g["v_cache"], g["table"], g["kv_lens"],
                              cu_seqlens=g["cu"])
    first = lambda: [pkg.attn_prefill(p["q"], p["k"], p["v"], p["cu"])] + [paged(g) for g in sets]  # noqa: E731
    second = lambda: [paged(g) for g in reversed(sets)]  # noqa: E731
    want = [[x.clone() for x in f()] for f in (first, second)]
    torch.cuda.synchronize()
    pool, graphs, got = torch.cuda.graph_pool_handle(), [], []
    for f in (first, second):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            got.append(f())
        graphs.append(graph)
    for _ in range(4):
        for i in (0, 1, 1, 0):
            graphs[i].replay()
            torch.cuda.synchronize()
            for x, y in zip(want[i], got[i]):
                assert torch.equal(x, y)
    assert pkg.device_error() == 0


@pytest.mark.parametrize("q_len", [1, 4, 40])
def test_pages_shared_by_sequences(cuda, q_len):
    """A prefix whose pages stand in several tables, and a page twice in one."""
    pkg = load_pkg()
    n, page = 5, 16
    d = paged_inputs([q_len] * n, [700 + 9 * i for i in range(n)], 8, 2, page, seed=40 + q_len)
    d["table"][:, :20] = d["table"][0, :20].clone()
    d["table"][1, 30] = d["table"][1, 29]
    ref, size = paged_ref(d, 0.07)
    g = on(d, cuda)
    check(pkg.attn_paged(g["q"], g["k_cache"], g["v_cache"], g["table"], g["kv_lens"], 0.07,
                         cu_seqlens=g["cu"]), ref, size)


def test_two_streams_at_once(cuda):
    pkg = load_pkg()
    ds = [prefill_inputs([900 + 100 * i, 40], 4, 2, seed=20 + i) for i in range(3)]
    gs = [on(d, cuda) for d in ds]
    want = [pkg.attn_prefill(g["q"], g["k"], g["v"], g["cu"]) for g in gs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in gs]
    for _ in range(10):
        got = []
        for g, s in zip(gs, streams):
            with torch.cuda.stream(s):
                got.append(pkg.attn_prefill(g["q"], g["k"], g["v"], g["cu"]))
        torch.cuda.synchronize()
        for a, b in zip(want, got):
            assert torch.equal(a, b)


# ------------------------------------------------------------------ refusals
def test_refusals(cuda):
    pkg = load_pkg()
    g = on(paged_inputs([1, 1], [20, 30], 4, 2, 16, seed=1), cuda)
    base = dict(q=g["q"], k_cache=g["k_cache"], v_cache=g["v_cache"], block_table=g["table"],
                kv_lens=g["kv_lens"], cu_seqlens=g["cu"])

    def call(**kw):
        a = {**base, **kw}
        return pkg.attn_paged(a["q"], a["k_cache"], a["v_cache"], a["block_table"], a["kv_lens"],
                              a.get("scale"), a.get("output"), cu_seqlens=a["cu_seqlens"])
    for kw, err in ((dict(q=g["q"].float()), TypeError), (dict(q=g["q"][None]), ValueError),
                    (dict(q=g["q"][..., :64]), ValueError), (dict(q=g["q"][:, :3]), ValueError),
                    (dict(q=g["q"].cpu()), ValueError), (dict(cu_seqlens=None), ValueError),
                    (dict(k_cache=g["k_cache"][:, :12], v_cache=g["v_cache"][:, :12]), ValueError),
                    (dict(k_cache=g["k_cache"].transpose(1, 2)), ValueError),
                    (dict(v_cache=g["v_cache"][:-1]), ValueError),
                    (dict(v_cache=None), TypeError),
                    (dict(k_cache=g["k_cache"][:0], v_cache=g["v_cache"][:0]), ValueError),
                    (dict(block_table=g["table"].long()), TypeError),
                    (dict(block_table=g["table"][:1]), ValueError),
                    (dict(block_table=g["table"][:1].expand(2, -1)), ValueError),
                    (dict(block_table=g["table"].cpu()), ValueError),
                    (dict(kv_lens=g["kv_lens"].float()), TypeError),
                    (dict(kv_lens=g["kv_lens"][:1]), ValueError),
                    (dict(cu_seqlens=g["cu"].float()), TypeError),
                    (dict(scale=-1.0), ValueError),
                    (dict(output=g["q"].float()), TypeError),
                    (dict(output=g["q"][:1]), ValueError)):
        with pytest.raises(err):
            call(**kw)
    d = on(prefill_inputs([5, 6], 4, 2, seed=1), cuda)
    for a, err in (((d["q"], d["k"], d["v"], None), TypeError),
                   ((d["q"], d["k"], d["v"][:, :1], d["cu"]), ValueError),
                   ((d["q"], d["k"][:5], d["v"], d["cu"]), ValueError),
                   ((d["q"].half(), d["k"], d["v"], d["cu"]), TypeError),
                   ((d["q"], d["k"], d["v"], d["cu"][:0]), ValueError)):
        with pytest.raises(err):
            pkg.attn_prefill(*a)


def test_empty_calls(cuda):
    pkg = load_pkg()
    e = torch.empty(0, 4, D, dtype=torch.bfloat16, device=cuda)
    z = torch.zeros(1, dtype=torch.int32, device=cuda)
    assert pkg.attn_prefill(e, e[:, :2], e[:, :2], z).shape == (0, 4, D)
    g = on(paged_inputs([1], [20], 4, 2, 16, seed=1), cuda)
    out = torch.full((3, 4, D), 5.0, dtype=torch.bfloat16, device=cuda)
    pkg.attn_prefill(out.clone(), out[:, :2].clone(), out[:, :2].clone(), z, None, out)
    pkg.attn_paged(out.clone(), g["k_cache"], g["v_cache"], g["table"][:0], g["kv_lens"][:0], None,
                   out, cu_seqlens=z)
    assert (out == 5).all()
    assert pkg.attn_paged(g["q"].view(1, 1, 4, D)[:, :0], g["k_cache"], g["v_cache"], g["table"],
                          g["kv_lens"]).shape == (1, 0, 4, D)
    # sequences without a page: rows that see nothing
    none = pkg.attn_paged(g["q"], g["k_cache"], g["v_cache"], g["table"][:, :0], g["kv_lens"],
                          cu_seqlens=g["cu"])
    assert (none == 0).all()
    assert starts([1, 2]).tolist() == [0, 1, 3]
