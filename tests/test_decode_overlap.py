"""What may share memory in the decoder-serving calls: results that overlap what is read, or one another, are
refused before any work; operands that interleave in one buffer are not."""
import itertools

import numpy as np
import pytest

from spinn_b200 import lib
from test_decode import P, attention, cache, elements, evict, append, refused, rows, table


def apart(a, b):
    return bool(lib.lib().spinn_cuda_diag_rows(a, b) & 2)


def test_slices_of_one_buffer_are_told_apart_exactly():
    """Two operands of the same strides: apart if and only if they share no element."""
    rng = np.random.default_rng(9)
    seen = [0, 0]
    for _ in range(3000):
        counts = [rng.integers(1, 4, 3).tolist() for _ in range(2)]
        widths = rng.integers(1, 4, 2).tolist()
        # strides that nest for both, in any order of dimensions
        strides, cover = [], max(widths)
        for i in range(3):
            strides.append(cover + int(rng.integers(0, 6)))
            cover = strides[-1] * max(c[i] for c in counts)
        order = rng.permutation(3)
        a, b = (rows(4096 + 2 * int(at), w, [c[i] for i in order], [strides[i] for i in order])
                for w, c, at in zip(widths, counts, rng.integers(-cover, cover + 1, 2)))
        got, want = apart(a, b), not elements(a)[1] & elements(b)[1]
        assert got == want, (list(a), list(b))
        seen[want] += 1
    assert min(seen) > 300


def test_pools_of_one_buffer():
    """Keys and values of one pool side by side in any dimension; a pool that starts inside the other."""
    pages, page, heads, dim = 5, 4, 3, 8
    for order in itertools.permutations(range(4)):        # where the dimension of (key, value) lies, and the others'
        sizes = {0: pages, 1: 2, 2: page, 3: heads}
        strides, cover = {}, dim
        for d in reversed(order):
            strides[d], cover = cover, cover * sizes[d]
        args = [pages, page, heads], [strides[0], strides[2], strides[3]]
        k, v = rows(4096, dim, *args), rows(4096 + 2 * strides[1], dim, *args)
        assert apart(k, v) and apart(v, k)
        for shift in (1, dim, strides[0], strides[2], strides[3]):
            b = rows(4096 + 2 * shift, dim, *args)
            assert apart(k, b) == (not elements(k)[1] & elements(b)[1])
    # the halves of rows twice as long
    args = [pages, page, heads], [page * heads * 2 * dim, heads * 2 * dim, 2 * dim]
    assert apart(rows(0, dim, *args), rows(2 * dim, dim, *args))
    assert not apart(rows(0, dim, *args), rows(2 * dim - 2, dim, *args))


@pytest.mark.parametrize("shift", [2, 2 * 64, 2 * 128, 2 * 2048, 4 * 2048, 8 * 2048])
def test_pools_that_overlap_are_refused(shift):
    """A value pool some elements, rows, tokens or pages into the key pool (9 pages of 16 tokens, 2 heads of 64)."""
    c = cache(k=P, v=P + shift)
    refused("spinn_cuda_cache_append", c, table(), append(), None, match="pools")
    refused("spinn_cuda_cache_evict", c, table(), evict(), None, match="pools")


FAR = 1 << 40


@pytest.mark.parametrize("kw,match", [
    (dict(kept=P), "lengths or a table"), (dict(kept=P - 16), "lengths or a table"), (dict(new=P + 8), "lengths or a table"),
    (dict(new=P + (1 << 16) + 44), "lengths or a table"), (dict(out=P + 64), "lengths or a table"),
    (dict(wout=P - 64), "lengths or a table"), (dict(kept=P + 64, budget=2), "one another"), (dict(kept=P + (1 << 20)), "one another"),
    (dict(new=P + (1 << 20) + 8), "one another"), (dict(kept=P + (1 << 21)), "one another"),
    (dict(new=P + (1 << 21) + 128), "one another")])
def test_evict_results_that_overlap_are_refused(kw, match):
    """lens at P, the table of 3 rows of 4 pages at P + 2^16, weights in and out at P + 2^20 and P + 2^21."""
    f = dict(win=P + (1 << 20), wout=P + (1 << 21), out=P + 256, new=P + 64, kept=P + (1 << 22))
    f.update(kw)
    refused("spinn_cuda_cache_evict", cache(v=P + FAR), table(pages=P + (1 << 16)), evict(**f), None, match=match)


@pytest.mark.parametrize("kw,match", [(dict(wout=P + 64), "overlap y"), (dict(wout=P + FAR), "weights_out q"),
                                      (dict(wout=P + (1 << 20), win=P + 512), "overlap y")])
def test_attention_weights_that_overlap_are_refused(kw, match):
    """y at P, q far from it."""
    f = dict(q=P + FAR, y=P, cap=64, wis=128, wos=128)
    f.update(kw)
    c = cache(heads=1, ps=16 * 64, ts=64)
    refused("spinn_cuda_paged_attention", c, table(), attention(**f), P, 1 << 15, None, match=match)


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["token", "head", "row", "halves"])
def test_interleaved_pools_work(cuda_lib, layout):
    """Appended, attended and evicted as in two pools of their own."""
    import torch

    from spinn_b200 import runtime as rt
    pages, page, heads, dim, seqs = 40, 16, 2, 64, 3
    shape = {"token": (pages, page, 2, heads, dim), "head": (pages, page, heads, 2, dim), "row": (pages, 2, page, heads, dim),
             "halves": (2, pages, page, heads, dim)}[layout]
    at = {"token": 2, "head": 3, "row": 1, "halves": 0}[layout]
    both = torch.zeros(shape, dtype=torch.bfloat16, device="cuda")
    pools = [(both.select(at, 0), both.select(at, 1)),
             tuple(torch.zeros(pages, page, heads, dim, dtype=torch.bfloat16, device="cuda") for _ in range(2))]
    torch.manual_seed(2)
    table_ = torch.randperm(pages, device="cuda")[:seqs * 12].to(torch.int32).view(seqs, 12)
    starts = torch.tensor([0, 150, 150, 290], dtype=torch.int32, device="cuda")
    new_k, new_v = (torch.randn(290, heads, dim, device="cuda").bfloat16() for _ in range(2))
    q = torch.randn(seqs, 8, dim, device="cuda").bfloat16()
    outs = []
    for k, v in pools:
        lens = torch.zeros(seqs, dtype=torch.int32, device="cuda")
        rt.cache_append(new_k, new_v, k, v, table_, lens, starts)
        lens = torch.tensor([150, 0, 140], dtype=torch.int32, device="cuda")
        # accumulated weights in and out as halves of the same rows
        rows_ = torch.zeros(seqs, heads, 400, device="cuda")
        w0, w1 = rows_[..., :200], rows_[..., 200:]
        y = torch.empty_like(q)
        rt.paged_attention(q, k, v, table_, lens, y, None, w0, w1)
        kept, n = torch.empty(seqs, heads, 60, dtype=torch.int32, device="cuda"), torch.empty_like(lens)
        rt.cache_evict(k, v, table_, lens, w1, w0, table_, n, kept, 60, 7)
        rt.stream_sync()
        outs.append((y, w0.clone(), w1.clone(), kept, n, k.clone(), v.clone()))
    for a, b in zip(*outs):
        assert torch.equal(a, b)
    assert outs[0][4].tolist() == [60, 0, 60]
