"""GPU: calls of the softmax-attention operators at the edges of what they allow."""
import ctypes
import threading

import pytest
import torch

from attn_util import D, check, on, paged_inputs, paged_ref, prefill_inputs, randn
from conftest import load_pkg
from oracle import attn_oracle as A

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lens", [[300], [5, 1, 3], [2500]])
def test_rows_whose_scores_are_all_minus_infinity(cuda, lens):
    """They give zeros, as rows that see nothing do, in every kernel, whole and joined.  The
    other rows agree with the oracle as ever (not bit for bit with a call without such rows: the
    32 rows of a warp choose together how their exponentials are taken)."""
    pkg = load_pkg()
    d = prefill_inputs(lens, 4, 2, seed=2)
    d["k"][..., 0] = 1.0
    ref, size = A.prefill(d["q"], d["k"], d["v"], d["cu"])
    g = on(d, cuda)
    rows = [i for i in (0, 5, 8, 200, 299, 2400) if i < sum(lens)]
    g["q"][rows, 1] = 0.0
    g["q"][rows, 1, 0] = float("-inf")  # -inf * 1 + 0 * the rest
    out = pkg.attn_prefill(g["q"], g["k"], g["v"], g["cu"])
    assert (out[rows, 1] == 0).all()
    ref[rows, 1], size[rows, 1] = 0, 0
    check(out, ref, size)


class _NodeParams(ctypes.Structure):  # CUDA_KERNEL_NODE_PARAMS
    _fields_ = [("func", ctypes.c_void_p), ("dims", ctypes.c_uint * 7),
                ("params", ctypes.POINTER(ctypes.c_void_p)), ("extra", ctypes.c_void_p),
                ("kern", ctypes.c_void_p), ("ctx", ctypes.c_void_p)]


def _tag_in(graph, workspace):
    """The 48-bit number that a captured attention launch marks its words of `workspace` with: it
    stands behind the addresses of the words and of the partial results."""
    cu = ctypes.CDLL("libcuda.so.1")
    n = ctypes.c_size_t()
    h = ctypes.c_void_p(graph.raw_cuda_graph())
    assert cu.cuGraphGetNodes(h, None, ctypes.byref(n)) == 0 and n.value == 1
    node, p = ctypes.c_void_p(), _NodeParams()
    assert cu.cuGraphGetNodes(h, ctypes.byref(node), ctypes.byref(n)) == 0
    assert cu.cuGraphKernelNodeGetParams_v2(node, ctypes.byref(p)) == 0
    info = cu.cuFuncGetParamInfo if p.func else cu.cuKernelGetParamInfo
    off, size = ctypes.c_size_t(), ctypes.c_size_t()
    for i in range(8):
        if info(ctypes.c_void_p(p.func or p.kern), ctypes.c_size_t(i), ctypes.byref(off),
                ctypes.byref(size)) != 0:
            break
        words = (ctypes.c_uint64 * (size.value // 8)).from_address(p.params[i])
        for j in range(len(words) - 2):
            if words[j] == workspace.data_ptr():
                return int(words[j + 2])
    raise AssertionError("no launch that was given the workspace")


@pytest.mark.parametrize("q_len", [1, 40])
def test_replay_after_a_failure_was_reported(cuda, q_len):
    """What a replay that gave up left in its scratch, words that count some arrivals under the
    graph's own number, is not taken for arrivals of a replay after gdn_device_error told of the
    failure (which is made here by the wait that nothing ends)."""
    pkg = load_pkg()
    hq, hk, page = 8, 1, 64
    g = on(paged_inputs([q_len], [30011], hq, hk, page, seed=q_len), cuda)
    want = pkg.attn_paged(g["q"], g["k_cache"], g["v_cache"], g["table"], g["kv_lens"],
                          cu_seqlens=g["cu"])
    need = pkg.LIB.gdn_attn_workspace_size(q_len, 1, hq, hk)
    ws = torch.zeros(need // 8 + 1, dtype=torch.int64, device=cuda)
    out = torch.zeros_like(want)

    def launch():
        k = g["k_cache"]
        assert pkg.LIB.gdn_attn_paged_launch(
            g["q"].data_ptr(), k.data_ptr(), g["v_cache"].data_ptr(), g["table"].data_ptr(),
            g["table"].shape[1], g["kv_lens"].data_ptr(), 0, g["cu"].data_ptr(), 0, 0.0,
            out.data_ptr(), q_len, 1, g["table"].shape[1], k.shape[0], page, k.stride(0),
            k.stride(0), hq, hk, D, hq * D, hq * D, ws.data_ptr(), need,
            torch.cuda.current_stream().cuda_stream) == 0
    launch()
    torch.cuda.synchronize()
    assert torch.equal(out, want) and pkg.device_error() == 0
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        launch()
    tag = _tag_in(graph, ws)
    assert 0 < tag < 2 ** 48

    def left(reports):
        """The arrivals of some replays that gave up, after so many reports: more than a join waits
        for (16 pieces a level), so that one which counts on from there never completes."""
        x = (tag + reports) % 2 ** 48 << 16 | 40
        return x - 2 ** 64 if x >= 2 ** 63 else x

    def replay(first_words):
        ws.fill_(-1)  # NaN in the partial results
        ws[:152 * 2 * 2 * 2] = first_words
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        return torch.equal(out, want)
    assert replay(-1)  # anything may stand there
    # not those, before the report (this process may have seen some already)
    words = next(left(r) for r in range(100) if not replay(left(r)))
    assert pkg.LIB.gdn_selftest_bounded_wait(1 << 12, 0, None, None) == 0
    assert pkg.device_error() == 16
    assert replay(words)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want) and pkg.device_error() == 0


@pytest.mark.parametrize("t,rd,inter", [(12, 64, False), (12, 128, True), (12, 6, False),
                                        (4101, 64, False)])
@pytest.mark.parametrize("eps", [1e-6, 0.0, 1e-36])
def test_norm_of_rows_whose_squares_leave_fp32(cuda, t, rd, inter, eps):
    """Rows of the largest bf16 values and, with an eps that does not hide them, of the smallest
    (their squares are beyond or below fp32's range), beside ordinary ones in the same warps; an
    infinite value gives NaN in its own row alone."""
    pkg = load_pkg()
    g0 = torch.Generator().manual_seed(t + rd)
    hq, hk = 5, 1
    q, k = randn((t, hq, D), g0, 2.0), randn((t, hk, D), g0, 2.0)
    top = torch.finfo(torch.bfloat16).max
    q[0, 0], q[1, 1], q[2, 2] = top, -top, q[2, 2] * 2.0 ** 62
    q[3, 0], k[3], q[4, 1] = q[3, 0] * 2.0 ** 120, k[3] * 2.0 ** 63, q[4, 1] * 2.0 ** -60
    q[5, 0], q[6, 1], k[7] = q[5, 0] * 2.0 ** -75, 2.0 ** -133, k[7] * 2.0 ** -130
    q[8, 0] = 0
    q[8, 0, 3] = top  # one large value among zeros
    q[t - 1, hq - 1] = top
    pos = torch.randint(0, 50, (t,), generator=g0)
    table = pkg.rope_table(50, rd, device="cpu")
    w = 1 + 0.3 * torch.randn(D, generator=g0)
    at = torch.tensor([*range(12), *range(12, t, 97), t - 1])
    want = [A.norm_rope(x[at], w, pos[at], table, eps=eps, interleaved=inter) for x in (q, k)]
    # a rotated value is off by at most 16 roundings of |y_a| + |y_b|, of the row's largest twice
    size = [2 * (x[at].double() * w).abs().amax(-1, keepdim=True)
            / torch.sqrt((x[at].double() ** 2).mean(-1, keepdim=True) + eps) for x in (q, k)]
    q[9, 3, 70] = float("inf")
    args = [x.to(cuda) for x in (q, k, pos, table, w, w)]
    got = pkg.attn_qk_norm_rope(*args, eps=eps, interleaved=inter)
    for o, ref, z in zip(got, want, size):
        o = o.cpu()[at].double()
        if o.shape[1] == hq:
            assert not torch.isfinite(o[9, 3]).all()
            o[9, 3], ref[9, 3] = 0, 0
        off = (o - ref).abs()
        assert (off <= 2.0 ** -8 * ref.abs() + 2.0 ** -19 * z + 2.0 ** -133).all()


@pytest.mark.parametrize("page", [200, 208, 256, 1024])
@pytest.mark.parametrize("hq,hk,q_len", [(4, 4, 1), (16, 2, 1), (8, 1, 2), (16, 2, 4)])
def test_few_rows_over_large_pages(cuda, page, hq, hk, q_len):
    """Pages of more rows than all warps take at once."""
    pkg = load_pkg()
    d = paged_inputs([q_len] * 5, [q_len, page, page + 1, 3 * page - 1, 2500], hq, hk, page,
                     seed=page + hq, stale=float("nan"))
    ref, size = paged_ref(d)
    g = on(d, cuda)
    out = pkg.attn_paged(g["q"].view(5, q_len, hq, D), g["k_cache"], g["v_cache"], g["table"],
                         g["kv_lens"])
    torch.cuda.synchronize()
    assert pkg.device_error() == 0
    check(out, ref, size, f"page {page}")


def test_two_threads(cuda):
    """Calls from two host threads, each on a stream of its own, of shapes that are new to both."""
    pkg = load_pkg()
    made = []
    for i in range(2):
        p = on(prefill_inputs([333 + i, 70, 5], 4, 2, seed=50 + i), cuda)
        c = on(paged_inputs([1 + 40 * i] * 3, [900, 77 + i, 41], 4, 2, 16, seed=60 + i), cuda)
        table = pkg.rope_table(500, 64, device=cuda)
        pos = torch.arange(p["q"].shape[0], device=cuda)
        made.append((p, c, table, pos))

    def calls(i):
        p, c, table, pos = made[i]
        q, k = pkg.attn_qk_norm_rope(p["q"], p["k"], pos, table)
        return [q, k, pkg.attn_prefill(q, k, p["v"], p["cu"]),
                pkg.attn_paged(c["q"], c["k_cache"], c["v_cache"], c["table"], c["kv_lens"],
                               cu_seqlens=c["cu"])]
    got, wrong = [[], []], []
    start = threading.Barrier(2)

    def work(i):
        try:
            stream = torch.cuda.Stream()
            start.wait(60)
            with torch.cuda.stream(stream):
                for _ in range(30):
                    got[i].append(calls(i))
            stream.synchronize()
        except Exception as e:  # noqa: BLE001
            wrong.append(e)
    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(120)
    torch.cuda.synchronize()
    assert not wrong and [len(x) for x in got] == [30, 30] and pkg.device_error() == 0
    for i in range(2):
        want = calls(i)
        for run in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(want, run))
