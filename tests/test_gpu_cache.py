"""Paged cache on the GPU -- append, one-token attention, eviction -- against 64-bit restatements
(tests/decode_ref.py), through the package's public calls."""
import numpy as np
import pytest
import torch

import decode_ref
from decode_ref import DTYPES, Paged

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def rt(cuda_lib):
    from spinn_b200 import runtime
    return runtime


# ------------------------------------------------------------------ append
APPENDS = [
    # dtype, past lengths, new tokens per sequence (None: one each, no starts), heads, dim, page, layout
    ("bf16", [0, 5, 16, 31], None, 8, 128, 16, "nhd"),
    ("fp16", [3, 0, 40], [5, 0, 37], 2, 64, 16, "nhd"),
    ("fp16", [7], [1], 1, 256, 1, "nhd"),
    ("fp32", [9, 2, 23], [30, 1, 25], 3, 80, 24, "hnd"),
    ("bf16", [4, 11], [9, 64], 5, 33, 7, "nhd"),         # odd head size: element copies
    ("fp16", [4, 11, 0, 6], [9, 64, 0, 0], 2, 64, 16, "odd"),
    ("fp32", [1, 2], [3, 4], 2, 5, 3, "odd"),
]


@pytest.mark.parametrize("case", APPENDS, ids=lambda c: f"{c[0]}-d{c[4]}-p{c[5]}-{c[6]}")
def test_append_writes_its_rows_and_nothing_else(rt, case):
    dtype, past, new, heads, dim, page, layout = case
    c = Paged(dtype, past, heads, dim, page, seed=1, room=max(new or [1]), layout=layout)
    counts = new or [1] * len(past)
    tokens = sum(counts)
    wide = torch.randn(tokens, heads, dim + 8, device="cuda").to(DTYPES[dtype])  # strided rows
    k, v = wide[..., :dim], torch.randn(tokens, heads, dim, device="cuda").to(DTYPES[dtype])
    starts = torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32, device="cuda") if new else None
    want_k, want_v = c.k.clone(), c.v.clone()
    at = 0
    for s, n in enumerate(past):
        for i in range(counts[s]):
            p, o = int(c.table_host[s, (n + i) // page]), (n + i) % page
            want_k[p, o], want_v[p, o] = k[at], v[at]
            at += 1
    rt.cache_append(k, v, c.k, c.v, c.table, c.lens, starts)
    rt.stream_sync()
    for got, want in ((c.k, want_k), (c.v, want_v)):
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(got.nan_to_num(7.0), want.nan_to_num(7.0))


def test_append_of_nothing_is_a_no_op(rt):
    c = Paged("bf16", [3], 2, 64, 16, room=4)
    empty = torch.empty(0, 2, 64, dtype=torch.bfloat16, device="cuda")
    rt.cache_append(empty, empty, c.k, c.v, c.table, c.lens, torch.zeros(2, dtype=torch.int32, device="cuda"))
    rt.stream_sync()


# ------------------------------------------------------------------ attention
ATTENTIONS = [
    # dtype, lengths, q_heads, kv_heads, dim, page, layout, weights
    ("fp16", [1], 1, 1, 64, 16, "nhd", False),
    ("bf16", [1, 0, 2], 8, 2, 128, 16, "nhd", True),
    ("bf16", [15, 16, 17, 63, 64, 65, 0, 129], 32, 8, 128, 16, "nhd", True),
    ("fp16", [333], 16, 4, 64, 16, "hnd", False),
    ("fp16", [700, 3, 0, 250], 16, 1, 64, 1, "nhd", True),      # group of 16: two column blocks
    ("bf16", [300, 511], 40, 2, 128, 32, "nhd", False),         # group of 20: two head blocks
    ("bf16", [257, 64, 1], 6, 2, 256, 24, "nhd", True),
    ("fp16", [130, 95], 12, 1, 192, 100, "hnd", True),
    ("bf16", [100, 37], 7, 7, 80, 7, "nhd", True),
    ("fp16", [77, 129], 4, 2, 33, 5, "nhd", True),              # odd head size: element loads
    ("bf16", [77, 129, 0], 4, 2, 64, 16, "odd", True),
    ("fp32", [1, 0, 200, 31, 32, 33], 6, 6, 80, 24, "nhd", True),
    ("fp32", [333, 90], 8, 2, 128, 16, "hnd", True),
    ("fp32", [65, 129], 18, 2, 256, 16, "nhd", False),          # group of 9: two head blocks
    ("fp32", [50, 81], 3, 1, 7, 3, "odd", True),
    ("fp16", [4097], 8, 8, 128, 64, "nhd", True),               # one long sequence in many shares
    ("bf16", [5000], 1, 1, 64, 16, "nhd", True),
    ("fp16", [512, 511, 1], 8, 2, 64, 16, "pair", True),        # the longest tables that are not split
    ("bf16", [513, 512, 0, 700], 8, 4, 128, 32, "pair", True),  # and the shortest that are
    ("fp32", [256, 7], 4, 2, 64, 8, "pair", True),
    ("fp32", [257, 300], 2, 2, 128, 16, "pair", False),
]


def _attention_case(rt, case, seed=3, scale=None, inplace=False):
    dtype, lens, q_heads, heads, dim, page, layout, weights = case
    c = Paged(dtype, lens, heads, dim, page, seed=seed, layout=layout)
    g = torch.Generator().manual_seed(seed + 1)
    q = (torch.randn(len(lens), q_heads, dim, generator=g) * 2).to(DTYPES[dtype]).cuda()
    y = torch.full_like(q, float("nan"))
    win = wout = None
    if weights:
        win = torch.rand(len(lens), heads, max(lens) + 9, generator=g).cuda()
        wout = win if inplace else torch.full((len(lens), heads, max(lens) + 5), -3.0, device="cuda")
    before = win.clone() if weights else None
    rt.paged_attention(q, c.k, c.v, c.table, c.lens, y, scale, win, wout)
    rt.stream_sync()
    return c, q, y, before, wout


def _check_attention(case, c, q, y, win, wout, scale=None, inplace=False):
    dtype, lens, q_heads, heads, dim, page, layout, weights = case
    want, mass, absum, ds = decode_ref.attention(c, q, dim ** -0.5 if scale is None else scale)
    n = max(lens)
    half = torch.finfo(DTYPES[dtype]).eps / 2
    # relative error of a probability: its score's, twice 2^-22 for exp2 and the rounding of its
    # argument (at most |score| log2(e) 2^-24, inside ds for these inputs), and, with 16-bit types,
    # 2^-17 for its two-part form (fp16 parts below 2^-14 are off by 2^-25 of the largest
    # probability's term instead: n 2^-25 in all).  The sums of n fp32 terms add n 2^-24.
    rel = 2 * (ds + 2.0 ** -21 + n * 2.0 ** -24)
    if dtype != "fp32":
        rel = rel + 2.0 ** -17
    tiny = n * 2.0 ** -25 * 6 if dtype == "fp16" else 0.0  # |v| <= 6 in these draws
    tol = half * want.abs() + rel * absum * (1 + half) + tiny
    err = (y.cpu().double() - want).abs()
    assert torch.isfinite(y).all()
    assert (err <= tol).all(), float((err / tol.clamp_min(1e-30)).max())
    if weights:
        got, prev = wout.cpu().double(), win.cpu().double()
        group = q_heads // heads
        wrel = rel.view(len(lens), heads, group, 1).amax(2)
        for s, m in enumerate(lens):
            ref = prev[s, :, :m] + mass[s, :, :m]
            t = wrel[s] * mass[s, :, :m] + ref.abs() * 2.0 ** -23
            assert ((got[s, :, :m] - ref).abs() <= t).all()
            rest = got[s, :, m:]
            assert torch.equal(rest, prev[s, :, m:]) if inplace else bool((rest == -3.0).all())


@pytest.mark.parametrize("case", ATTENTIONS, ids=lambda c: f"{c[0]}-h{c[2]}x{c[3]}-d{c[4]}-p{c[5]}-{c[6]}-{max(c[1])}")
def test_attention_matches_its_definition(rt, case):
    _check_attention(case, *_attention_case(rt, case))


def test_attention_scale_and_weights_in_place(rt):
    case = ("bf16", [200, 0, 64], 8, 2, 64, 16, "nhd", True)
    _check_attention(case, *_attention_case(rt, case, scale=0.37, inplace=True), scale=0.37, inplace=True)


def test_attention_scores_far_apart(rt):
    """Scores of hundreds: the running maximum keeps every exponent in range, and a token that
    dominates takes all of the weight."""
    c = Paged("fp16", [150, 70], 2, 64, 16, seed=5)
    q = torch.full((2, 4, 64), 60.0, dtype=torch.float16, device="cuda")
    y = torch.empty_like(q)
    rt.paged_attention(q, c.k, c.v, c.table, c.lens, y, scale=1.0)
    rt.stream_sync()
    want, _, absum, ds = decode_ref.attention(c, q, 1.0)
    tol = 2.0 ** -11 * want.abs() + 2 * (ds + 2.0 ** -16) * absum + 150 * 2.0 ** -25 * 6
    assert ((y.cpu().double() - want).abs() <= tol).all()


def _check_on_gpu(c, q, y, win, wout, dtype):
    """As _check_attention, for many sequences: 64 bits on the GPU, one sequence at a time."""
    half, dim = torch.finfo(DTYPES[dtype]).eps / 2, q.shape[2]
    group = q.shape[1] // c.heads
    for s, n in enumerate(c.lens_host):
        if n == 0:
            assert bool((y[s] == 0).all())
            continue
        t = torch.arange(n, device="cuda")
        pages = c.table[s].long()[t // c.page]
        k = c.k[pages, t % c.page].double().repeat_interleave(group, 1).transpose(0, 1)   # [heads, n, dim]
        v = c.v[pages, t % c.page].double().repeat_interleave(group, 1).transpose(0, 1)
        qs = q[s].double()
        p = torch.softmax(torch.einsum("hd,hnd->hn", qs, k) * dim ** -0.5, -1)
        want, absum = torch.einsum("hn,hnd->hd", p, v), torch.einsum("hn,hnd->hd", p, v.abs())
        ds = torch.einsum("hd,hnd->hn", qs.abs(), k.abs()).amax(-1, keepdim=True) * dim ** -0.5 * dim * 2.0 ** -24
        rel = 2 * (ds + 2.0 ** -21 + n * 2.0 ** -24) + (2.0 ** -17 if dtype != "fp32" else 0.0)
        tiny = n * 2.0 ** -25 * 6 if dtype == "fp16" else 0.0
        assert ((y[s].double() - want).abs() <= half * want.abs() + rel * absum * (1 + half) + tiny).all(), s
        if wout is not None:
            mass = p.view(c.heads, group, n).sum(1)
            ref = win[s, :, :n].double() + mass
            r = rel.view(c.heads, group, 1).amax(1)
            assert ((wout[s, :, :n].double() - ref).abs() <= r * mass + ref.abs() * 2.0 ** -23).all(), s


@pytest.mark.parametrize("dtype,seqs,most,q_heads,heads,dim,page,layout", [
    ("bf16", 300, 700, 16, 4, 64, 16, "nhd"),     # more sequences than threads: scanned in parts
    ("fp16", 129, 90, 8, 8, 128, 24, "nhd"),      # lanes copying, many short ones to a share
    ("bf16", 64, 2300, 16, 8, 64, 32, "hnd"),     # shares of more than 32 tiles
    ("fp32", 200, 400, 6, 3, 80, 8, "nhd"),
    ("fp16", 40, 3000, 14, 2, 128, 7, "nhd"),     # a group of seven, pages that end inside every tile
])
def test_attention_over_large_batches(rt, dtype, seqs, most, q_heads, heads, dim, page, layout):
    rng = np.random.default_rng(seqs)
    lens = [int(x) for x in rng.integers(0, most + 1, seqs)]
    lens[3], lens[7], lens[-1] = 0, most, 0
    c = Paged(dtype, lens, heads, dim, page, seed=seqs, layout=layout)
    q = (torch.randn(seqs, q_heads, dim, device="cuda") * 2).to(DTYPES[dtype])
    y = torch.full_like(q, float("nan"))
    win = torch.rand(seqs, heads, most, device="cuda")
    wout = torch.full((seqs, heads, most), -3.0, device="cuda")
    rt.paged_attention(q, c.k, c.v, c.table, c.lens, y, None, win, wout)
    rt.stream_sync()
    _check_on_gpu(c, q, y, win, wout, dtype)
    y2 = torch.full_like(q, float("nan"))
    rt.paged_attention(q, c.k, c.v, c.table, c.lens, y2)
    rt.stream_sync()
    assert torch.equal(y, y2)
    late = torch.arange(most, device="cuda") >= c.lens[:, None]
    assert bool((wout.transpose(1, 2)[late] == -3.0).all())


def test_calls_at_once_on_two_streams(rt):
    """Eager calls that overlap on the GPU, each on its own stream with its own workspace."""
    runs = []
    for i in range(2):
        c, q, y, win, wout = _attention_case(rt, ("bf16", [4000, 300, 0, 2500], 16, 4, 128, 16, "nhd", True), seed=40 + i)
        runs.append((c, q, y, win, wout, torch.cuda.Stream()))
    x = [torch.randn(200, 1001, device="cuda").half() for _ in range(2)]      # with aligned copies
    w = torch.randn(600, 1001, device="cuda").half()
    want = [torch.empty(200, 600, device="cuda").half() for _ in range(2)]
    for a, b in zip(x, want):
        rt.linear(a, w, b)
    rt.stream_sync()
    for _ in range(10):
        outs = []
        for i, (c, q, y, win, wout, stream) in enumerate(runs):
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                z, y2, w2 = torch.empty_like(want[i]), torch.zeros_like(y), torch.full_like(wout, -3.0)
                rt.paged_attention(q, c.k, c.v, c.table, c.lens, y2, None, win, w2)
                rt.linear(x[i], w, z)
                outs.append((y2, w2, z))
        torch.cuda.synchronize()
        for (c, q, y, win, wout, _s), b, (y2, w2, z) in zip(runs, want, outs):
            assert torch.equal(y, y2) and torch.equal(wout, w2) and torch.equal(b, z)


def test_captured_between_other_nodes(rt):
    """A graph whose calls follow copies, memsets, torch kernels and a join of two streams."""
    c, q, y, win, wout = _attention_case(rt, ("bf16", [700, 33], 8, 2, 64, 16, "nhd", True))
    new = torch.randn(2, 2, 64, device="cuda").to(torch.bfloat16)
    q0, w0 = q.clone(), win.clone()
    y2, w2, src = torch.empty_like(y), torch.zeros_like(wout), torch.zeros_like(q)
    scratch = torch.empty(1 << 20, device="cuda")
    graph, main, side = torch.cuda.CUDAGraph(), torch.cuda.Stream(), torch.cuda.Stream()
    mat, out = torch.randn(64, 64, device="cuda").to(torch.bfloat16), torch.empty(16, 64, device="cuda").to(torch.bfloat16)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=main):
        src.copy_(q0)
        side.wait_stream(main)
        with torch.cuda.stream(side):
            scratch.zero_()
            rt.linear(q0.view(16, 64), mat, out)
        w2.fill_(-3.0)
        main.wait_stream(side)
        rt.paged_attention(src, c.k, c.v, c.table, c.lens, y2, None, w0, w2)
        scratch.add_(1.0)
    for _ in range(3):
        y2.zero_()
        graph.replay()
        rt.stream_sync()
        assert torch.equal(y2, y) and torch.equal(w2[:, :, :700], wout[:, :, :700])
    del new


FIRST_CALLS = """
import torch
from spinn_b200 import runtime as rt
dt = torch.bfloat16
k = torch.randn(800, 16, 2, 64, device="cuda").to(dt); v = k.clone()
table = torch.arange(800, dtype=torch.int32, device="cuda").view(2, 400); lens = torch.tensor([100, 7], dtype=torch.int32, device="cuda")
q = torch.randn(2, 8, 64, device="cuda").to(dt); y = torch.empty_like(q)
w = torch.zeros(2, 2, 6400, device="cuda"); new = torch.empty(2, dtype=torch.int32, device="cuda")
kept = torch.empty(2, 2, 50, dtype=torch.int32, device="cuda")
row = torch.randn(2, 2, 64, device="cuda").to(dt)
x = torch.randn(40, 65, device="cuda").to(dt); m = torch.randn(32, 65, device="cuda").to(dt); z = torch.empty(40, 32, device="cuda").to(dt)
big = torch.randn(64, 2048, device="cuda").to(dt); wide = torch.randn(1000, 2048, device="cuda").to(dt)
split = torch.empty(64, 1000, device="cuda").to(dt)
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    rt.linear(big, wide, split)
    rt.cache_append(row, row, k, v, table, lens)
    rt.paged_attention(q, k, v, table, lens, y, None, w, w)
    rt.linear(x, m, z)
    rt.linear(x[:3], m, z[:3])
    rt.cache_evict(k, v, table, lens, w, w, table, new, kept, 50)
g.replay()
rt.stream_sync()
assert new.tolist() == [50, 7] and abs(float(w[1].sum()) - 8) < 1e-4 and torch.isfinite(z.float()).all()
assert (split.float() - big.float() @ wide.float().T).abs().max() < 1.0
print("replayed")
"""


def test_first_calls_of_a_process_may_be_captured(cuda_lib):
    """Nothing is allocated or asked of the device that a capture forbids, not even the first time."""
    import os
    import subprocess
    import sys

    from conftest import ROOT
    r = subprocess.run([sys.executable, "-c", FIRST_CALLS], cwd=ROOT, capture_output=True, text=True, timeout=300,
                       env=dict(os.environ, PYTHONPATH=ROOT))
    assert r.returncode == 0 and "replayed" in r.stdout, r.stderr[-2000:]


def test_attention_is_deterministic_and_replays(rt):
    """The same call twice gives the same bits; captured into a graph with its workspace it gives
    them again for new inputs, on another stream than the inputs' own."""
    case = ("bf16", [900, 33, 0, 1200], 16, 4, 128, 16, "nhd", True)
    c, q, y, win, wout = _attention_case(rt, case)
    y2, w2 = torch.empty_like(y), torch.zeros_like(wout)
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        rt.paged_attention(q, c.k, c.v, c.table, c.lens, y2, None, win, w2)
    for _ in range(2):
        y2.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y2, y)
    q.mul_(0.5)
    graph.replay()
    torch.cuda.synchronize()
    want, _, absum, _ = decode_ref.attention(c, q, 128 ** -0.5)
    assert ((y2.cpu().double() - want).abs() <= 2.0 ** -8 * want.abs() + 1e-3 * absum).all()


def test_two_graphs_share_nothing(rt):
    """Two captured calls replayed at once on two streams: each has its own workspace."""
    cases = [("bf16", [3000, 100], 8, 2, 128, 16, "nhd", True), ("bf16", [2000, 777], 8, 2, 128, 16, "nhd", True)]
    runs = []
    for i, case in enumerate(cases):
        c, q, y, win, wout = _attention_case(rt, case, seed=20 + i)
        y2, w2 = torch.zeros_like(y), torch.full_like(wout, -3.0)
        graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(graph, stream=stream):
            rt.paged_attention(q, c.k, c.v, c.table, c.lens, y2, None, win, w2)
        runs.append((graph, stream, y, wout, y2, w2, (c, q, win)))  # a graph's inputs stay alive with it
    torch.cuda.synchronize()
    for _ in range(20):
        for graph, stream, *_rest in runs:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for _, _, y, wout, y2, w2, _inputs in runs:
        assert torch.equal(y, y2) and torch.equal(wout, w2)


def test_outputs_that_overlap_are_refused(rt):
    """Results whose rows share memory with one another or with what is read: refused before any work."""
    from spinn_b200.lib import EINVAL, SpinnCudaError
    c = Paged("bf16", [40, 17], 2, 64, 16, seed=3, room=4)
    q = torch.randn(2, 4, 64, device="cuda").bfloat16()
    w = torch.zeros(2, 2, 64, device="cuda")

    def refused(match, fn, *args):
        with pytest.raises(SpinnCudaError, match=match) as e:
            fn(*args)
        assert e.value.code == EINVAL

    attend = lambda q, y, win=None, wout=None: rt.paged_attention(q, c.k, c.v, c.table, c.lens, y, None, win, wout)  # noqa: E731
    refused("y overlap", attend, q, q)
    refused("y overlap", attend, q, torch.empty(2, 1, 64, device="cuda").bfloat16().expand(2, 4, 64))
    refused("weights_out overlap", attend, q, torch.empty_like(q), None, w[:, :1].expand(2, 2, 64))
    wide = torch.zeros(2, 2, 96, device="cuda")
    refused("apart from it", attend, q, torch.empty_like(q), wide[..., :64], wide[..., 32:])
    # query and result side by side in one buffer
    both = torch.randn(2, 8, 64, device="cuda").bfloat16()
    y = torch.empty_like(q)
    attend(both[:, :4], both[:, 4:])
    attend(both[:, :4].contiguous(), y)
    rt.stream_sync()
    assert torch.equal(both[:, 4:], y)
    one = c.k[:, :, :1].expand(-1, -1, 2, -1)
    rows = torch.randn(2, 2, 64, device="cuda").bfloat16()
    refused("pools", rt.cache_append, rows, rows, one, c.v[:, :, :1].expand(-1, -1, 2, -1), c.table, c.lens)
    refused("pools", rt.cache_append, rows, rows, c.k, c.k, c.table, c.lens)
    new_lens, kept = torch.empty(2, dtype=torch.int32, device="cuda"), torch.empty(2, 2, 8, dtype=torch.int32, device="cuda")
    refused("pools", rt.cache_evict, c.k, c.k, c.table, c.lens, w, w, c.table, new_lens, kept, 8)
    refused("weights_out overlap", rt.cache_evict, c.k, c.v, c.table, c.lens, w, w[:1, :1].clone().expand(2, 2, 64), c.table, new_lens,
            kept, 8)


def test_sync_of_a_capturing_stream_is_refused(rt):
    """The refusal leaves the capture whole."""
    from spinn_b200.lib import SpinnCudaError
    c, q, y, _win, _wout = _attention_case(rt, ("fp16", [100, 7], 4, 2, 64, 16, "nhd", False), seed=9)
    y2 = torch.zeros_like(y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rt.paged_attention(q, c.k, c.v, c.table, c.lens, y2)
        with pytest.raises(SpinnCudaError, match="being captured"):
            rt.stream_sync()
    graph.replay()
    rt.stream_sync()
    assert torch.equal(y, y2)


def test_bad_pages_and_lengths_are_reported(rt):
    """A page outside the pool or a length beyond the table is never followed: the operator skips
    it and the next stream_sync raises, once."""
    from spinn_b200.lib import EINVAL, SpinnCudaError
    c = Paged("bf16", [40, 20], 2, 64, 16)
    q = torch.randn(2, 4, 64, device="cuda").to(torch.bfloat16)
    y = torch.empty_like(q)
    for bad in (-1, c.k.shape[0], 2 ** 31 - 1):
        table = c.table.clone()
        table[0, 1] = bad
        rt.paged_attention(q, c.k, c.v, table, c.lens, y)
        with pytest.raises(SpinnCudaError, match="page number") as e:
            rt.stream_sync()
        assert e.value.code == EINVAL
        rt.stream_sync()
    for bad in (-1, c.table.shape[1] * 16 + 1, 2 ** 31 - 1):
        lens = torch.tensor([bad, 20], dtype=torch.int32, device="cuda")
        rt.paged_attention(q, c.k, c.v, c.table, lens, y)
        with pytest.raises(SpinnCudaError, match="length"):
            rt.stream_sync()
        assert bool((y[0] == 0).all())
        new = torch.randn(2, 2, 64, device="cuda").to(torch.bfloat16)
        rt.cache_append(new, new, c.k, c.v, c.table, lens)
        with pytest.raises(SpinnCudaError):
            rt.stream_sync()
    # rows that starts does not cover
    starts = torch.tensor([1, 2, 2], dtype=torch.int32, device="cuda")
    new = torch.randn(3, 2, 64, device="cuda").to(torch.bfloat16)
    rt.cache_append(new, new, c.k, c.v, c.table, torch.zeros(2, dtype=torch.int32, device="cuda"), starts)
    with pytest.raises(SpinnCudaError, match="length"):
        rt.stream_sync()
    rt.stream_sync()


def test_offsets_past_32_bits(rt):
    """Pages whose elements lie past 2^31 in the pool (4.3 GB of bf16 in each)."""
    heads, dim, page = 8, 128, 64
    pages = (2 ** 31) // (heads * dim * page) + 8
    k = torch.zeros(pages, page, heads, dim, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    n = 3 * page + 5
    table = torch.tensor([[pages - 1, 0, pages - 2, pages - 3]], dtype=torch.int32, device="cuda")
    lens = torch.zeros(1, dtype=torch.int32, device="cuda")
    rows_k = torch.randn(n, heads, dim, device="cuda").to(torch.bfloat16)
    rows_v = torch.randn(n, heads, dim, device="cuda").to(torch.bfloat16)
    rt.cache_append(rows_k, rows_v, k, v, table, lens, torch.tensor([0, n], dtype=torch.int32, device="cuda"))
    assert torch.equal(k[pages - 1], rows_k[:page]) and torch.equal(v[pages - 3, :5], rows_v[3 * page:])
    q = torch.randn(1, 16, dim, device="cuda").to(torch.bfloat16)
    y = torch.empty_like(q)
    rt.paged_attention(q, k, v, table, lens + n, y)
    rt.stream_sync()
    kk = rows_k.double().repeat_interleave(2, 1)
    p = torch.softmax(torch.einsum("hd,nhd->hn", q[0].double(), kk) * dim ** -0.5, -1)
    vv = rows_v.double().repeat_interleave(2, 1)
    want, absum = torch.einsum("hn,nhd->hd", p, vv), torch.einsum("hn,nhd->hd", p, vv.abs())
    assert ((y[0].double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -12 * absum).all()


# ------------------------------------------------------------------ eviction
EVICTS = [
    # dtype, lengths, heads, dim, page, budget, recent, layout
    ("bf16", [100, 31, 0, 32, 33], 2, 128, 16, 32, 8, "nhd"),
    ("fp16", [1, 2, 3], 1, 64, 1, 1, 0, "nhd"),
    ("fp16", [257, 300], 3, 64, 16, 40, 40, "hnd"),      # only the recent ones
    ("fp32", [90, 17], 2, 80, 24, 16, 100, "nhd"),       # recent beyond the budget
    ("bf16", [500], 4, 33, 7, 123, 5, "nhd"),            # odd head size
    ("fp16", [200, 64], 2, 64, 16, 50, 3, "odd"),
    ("bf16", [3000, 1025, 7], 2, 64, 16, 1024, 100, "nhd"),
    ("fp32", [2500], 1, 4, 16, 1500, 0, "nhd"),
    ("bf16", [60, 50], 2, 256, 16, 64, 4, "nhd"),        # budget above every length
    ("bf16", [5000, 4097, 33, 4096], 2, 8, 16, 700, 31, "nhd"),   # two CTAs to a head
    ("fp16", [40000, 1, 20000], 1, 8, 64, 9000, 100, "nhd"),      # eight CTAs
    ("fp16", [220000], 1, 8, 64, 5000, 0, "nhd"),                 # past the shared memory of eight
]


def _weights(lens, heads, seed):
    rng = np.random.default_rng(seed)
    w = rng.random((len(lens), heads, max(lens) + 3)).astype(np.float32)
    w = np.where(rng.random(w.shape) < 0.3, np.float32(0.25), w)   # many ties
    w[rng.random(w.shape) < 0.05] = 0.0
    w[rng.random(w.shape) < 0.05] = -0.0
    w[rng.random(w.shape) < 0.02] = np.nan
    w[rng.random(w.shape) < 0.02] = np.inf
    w[rng.random(w.shape) < 0.02] = -np.inf
    return w


@pytest.mark.parametrize("inplace", [False, True], ids=["pages", "inplace"])
@pytest.mark.parametrize("case", EVICTS, ids=lambda c: f"{c[0]}-d{c[3]}-p{c[4]}-b{c[5]}-r{c[6]}-{c[7]}")
def test_evict_keeps_the_heaviest_in_order(rt, case, inplace):
    dtype, lens, heads, dim, page, budget, recent, layout = case
    wide = -(-budget // page)
    c = Paged(dtype, lens, heads, dim, page, seed=7, layout=layout, spare=wide * len(lens) + 1)
    w = _weights(lens, heads, 11)
    weights = torch.from_numpy(w).cuda()
    wout = weights if inplace else torch.full_like(weights, -3.0)
    out = c.table if inplace else torch.tensor(c.free[:wide * len(lens)], dtype=torch.int32).view(len(lens), wide).cuda()
    new_lens = torch.full((len(lens),), -7, dtype=torch.int32, device="cuda")
    kept = torch.full((len(lens), heads, budget), -7, dtype=torch.int32, device="cuda")
    k0, v0 = c.k.cpu().clone(), c.v.cpu().clone()
    rt.cache_evict(c.k, c.v, c.table, c.lens, weights, wout, out, new_lens, kept, budget, recent)
    rt.stream_sync()
    want_kept, want_new = decode_ref.evict(w, lens, budget, recent)
    assert new_lens.tolist() == want_new
    want_k, want_v = k0.clone(), v0.clone()
    out_host = out.cpu().numpy()
    got_w = wout.cpu().numpy()
    for s, n in enumerate(lens):
        for h in range(heads):
            rows = want_kept[s][h]
            assert kept[s, h].tolist() == rows + [-1] * (budget - len(rows))
            ref = (w if inplace else np.full_like(w, -3.0))[s, h].copy()
            ref[:n] = 0.0
            ref[:len(rows)] = w[s, h, rows]
            np.testing.assert_array_equal(got_w[s, h], ref)
            for j, i in enumerate(rows):
                src, so = c.table_host[s, i // page], i % page
                dst, do = out_host[s, j // page], j % page
                want_k[dst, do, h], want_v[dst, do, h] = k0[src, so, h], v0[src, so, h]
    for got, want in ((c.k.cpu(), want_k), (c.v.cpu(), want_v)):
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(got.nan_to_num(7.0), want.nan_to_num(7.0))


def test_evict_reports_a_cloned_table(rt):
    """A copy of the table is not 'in place': its pages are read and written by different CTAs, so
    the call moves nothing and says so."""
    from spinn_b200.lib import SpinnCudaError
    c = Paged("bf16", [100], 2, 64, 16)
    w = torch.rand(1, 2, 100, device="cuda")
    k0 = c.k.clone()
    rt.cache_evict(c.k, c.v, c.table, c.lens, w, torch.zeros_like(w), c.table.clone(),
                   torch.empty(1, dtype=torch.int32, device="cuda"),
                   torch.empty(1, 2, 40, dtype=torch.int32, device="cuda"), 40)
    with pytest.raises(SpinnCudaError, match="in place"):
        rt.stream_sync()
    assert torch.equal(c.k.nan_to_num(7.0), k0.nan_to_num(7.0))


def test_evict_lengths_beyond_the_destination(rt):
    from spinn_b200.lib import SpinnCudaError
    c = Paged("bf16", [100], 1, 64, 16, spare=4)
    w = torch.rand(1, 1, 100, device="cuda")
    out = torch.tensor([c.free[:2]], dtype=torch.int32, device="cuda")  # 32 tokens
    new_lens = torch.empty(1, dtype=torch.int32, device="cuda")
    kept = torch.empty(1, 1, 40, dtype=torch.int32, device="cuda")
    rt.cache_evict(c.k, c.v, c.table, c.lens, w, torch.zeros_like(w), out, new_lens, kept, 40)
    with pytest.raises(SpinnCudaError, match="length"):
        rt.stream_sync()
    assert new_lens.tolist() == [0] and bool((kept == -1).all())
