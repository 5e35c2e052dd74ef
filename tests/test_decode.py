"""Decoder-serving operators without a GPU: argument checks of the C entry points (which come
before any CUDA call), of the Python calls, and the host arithmetic that the kernels share."""
import ctypes
import struct

import numpy as np
import pytest

from spinn_b200 import lib, runtime

CACHE = struct.Struct("<QQqqqiiiiii")             # SpinnCudaCache
TABLE = struct.Struct("<QQqii")                   # SpinnCudaPageTable
APPEND = struct.Struct("<QQqqqqQii")              # SpinnCudaAppend
ATTENTION = struct.Struct("<QQqqqqQQqqqqiifi")    # SpinnCudaAttention
EVICT = struct.Struct("<QQqqqqQqiiQQii")          # SpinnCudaEvict
LINEAR = struct.Struct("<QQQQQqqqqiiiiii")        # SpinnCudaLinear

BUF = ctypes.create_string_buffer(1 << 16)  # never dereferenced: every call here is refused
P = (ctypes.addressof(BUF) + 255) & ~255


def cache(**kw):
    f = dict(k=P, v=P, ps=16 * 2 * 64, ts=2 * 64, hs=64, dtype=lib.BF16, pages=9, page=16, heads=2, dim=64)
    f.update(kw)
    return CACHE.pack(f["k"], f["v"], f["ps"], f["ts"], f["hs"], f["dtype"], f["pages"], f["page"],
                               f["heads"], f["dim"], 0)


def table(**kw):
    f = dict(pages=P, lens=P, stride=4, seqs=3, wide=4)
    f.update(kw)
    return TABLE.pack(f["pages"], f["lens"], f["stride"], f["seqs"], f["wide"])


def refused(fn, *args, match):
    rc = getattr(lib.lib(), fn)(*args)
    assert rc == lib.EINVAL and match in lib.last_error(), (rc, lib.last_error())


BAD_CACHES = [(dict(k=0), "null"), (dict(v=0), "null"), (dict(dtype=7), "type 7"), (dict(dtype=0), "type 0"),
              (dict(pages=0), "geometry"), (dict(page=0), "geometry"), (dict(page=-16), "geometry"),
              (dict(heads=0), "geometry"), (dict(heads=65536), "geometry"), (dict(dim=0), "head_dim"),
              (dict(dim=257), "head_dim"), (dict(ts=-1), "stride"), (dict(k=P + 1), "misaligned")]
BAD_TABLES = [(dict(pages=0), "null"), (dict(lens=0), "null"), (dict(seqs=0), "page table"), (dict(wide=0), "page table"),
              (dict(stride=-4), "page table"), (dict(lens=P + 2), "misaligned")]


def append(**kw):
    f = dict(k=P, v=P, starts=0, tokens=3, ks=128)
    f.update(kw)
    return APPEND.pack(f["k"], f["v"], f["ks"], 64, 128, 64, f["starts"], f["tokens"], 0)


def attention(**kw):
    f = dict(q=P, y=P, win=0, wout=0, cap=0, q_heads=4, qs=256, wis=0, wos=0)
    f.update(kw)
    return ATTENTION.pack(f["q"], f["y"], f["qs"], 64, 256, 64, f["win"], f["wout"], f["wis"], 0, f["wos"], 0,
                                   f["cap"], f["q_heads"], 0.125, 0)


def evict(**kw):
    f = dict(win=P, wout=P + 8192, out=P + 256, stride=4, wide=4, cap=64, new=P + 64, kept=P + 128, budget=16, recent=0,
             wis=128, wos=128)
    f.update(kw)
    return EVICT.pack(f["win"], f["wout"], f["wis"], 64, f["wos"], 64, f["out"], f["stride"], f["wide"],
                               f["cap"], f["new"], f["kept"], f["budget"], f["recent"])


@pytest.mark.parametrize("kw,match", BAD_CACHES)
def test_bad_caches_are_refused(kw, match):
    refused("spinn_cuda_cache_append", cache(**kw), table(), append(), None, match=match)
    refused("spinn_cuda_paged_attention", cache(**kw), table(), attention(), P, 1 << 15, None, match=match)
    refused("spinn_cuda_cache_evict", cache(**kw), table(), evict(), None, match=match)


@pytest.mark.parametrize("kw,match", BAD_TABLES)
def test_bad_tables_are_refused(kw, match):
    refused("spinn_cuda_cache_append", cache(), table(**kw), append(), None, match=match)
    refused("spinn_cuda_paged_attention", cache(), table(**kw), attention(), P, 1 << 15, None, match=match)
    refused("spinn_cuda_cache_evict", cache(), table(**kw), evict(), None, match=match)


@pytest.mark.parametrize("kw,match", [(dict(k=0), "required"), (dict(tokens=-1), "tokens"), (dict(tokens=5), "without starts"),
                                      (dict(ks=-1), "stride"), (dict(k=P + 1), "misaligned"),
                                      (dict(starts=P + 1), "misaligned")])
def test_append_refusals(kw, match):
    refused("spinn_cuda_cache_append", cache(), table(), append(**kw), None, match=match)


@pytest.mark.parametrize("kw,match", [(dict(q=0), "required"), (dict(y=0), "required"), (dict(q_heads=3), "multiple"),
                                      (dict(q_heads=0), "multiple"), (dict(qs=-1), "stride"), (dict(y=P + 1), "misaligned"),
                                      (dict(win=P), "without weights_out"), (dict(wout=P), "geometry"),
                                      (dict(wout=P, cap=64, q_heads=34), "at most 16"),
                                      (dict(wout=P, win=P, cap=64, wis=64, wos=128), "in place")])
def test_attention_refusals(kw, match):
    refused("spinn_cuda_paged_attention", cache(), table(), attention(**kw), P, 1 << 15, None, match=match)


def test_attention_weights_take_fewer_heads_in_fp32():
    refused("spinn_cuda_paged_attention", cache(dtype=lib.FP32), table(), attention(wout=P, cap=64, q_heads=18), P, 1 << 15,
            None, match="at most 8")


@pytest.mark.parametrize("kw,match", [(dict(win=0), "required"), (dict(kept=0), "required"), (dict(budget=0), "budget"),
                                      (dict(recent=-1), "budget"), (dict(wide=0), "output table"),
                                      (dict(cap=0), "output table"), (dict(new=P), "lengths"), (dict(wis=-1), "stride"),
                                      (dict(out=P, stride=8), "in place"), (dict(wout=P + 16), "apart"),
                                      (dict(wout=P, wos=64), "apart"), (dict(kept=P + 2), "misaligned")])
def test_evict_refusals(kw, match):
    refused("spinn_cuda_cache_evict", cache(), table(), evict(**kw), None, match=match)


def test_evict_refuses_more_pairs_than_a_grid_has():
    refused("spinn_cuda_cache_evict", cache(heads=4096), table(seqs=17), evict(wis=0, wos=0, wout=P + (1 << 20) * 4), None,
            match="65535")


# ------------------------------------------------------------------ Python calls
def test_python_calls_refuse_host_tensors():
    torch = pytest.importorskip("torch")
    k = torch.zeros(4, 16, 2, 64)
    t, n = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    q = torch.zeros(1, 2, 64)
    w = torch.zeros(1, 2, 32)
    with pytest.raises(TypeError, match="CUDA"):
        runtime.cache_append(q, q, k, k, t, n)
    with pytest.raises(TypeError, match="CUDA"):
        runtime.paged_attention(q, k, k, t, n, q)
    with pytest.raises(TypeError, match="CUDA"):
        runtime.cache_evict(k, k, t, n, w, w, t, n, torch.zeros(1, 2, 4, dtype=torch.int32), 4)


def test_python_calls_check_shapes_and_types():
    """Checked before the device, so that host tensors do."""
    torch = pytest.importorskip("torch")
    k = torch.zeros(4, 16, 2, 64)
    t, n = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    q = torch.zeros(1, 2, 64)
    w = torch.zeros(1, 2, 32)
    kept = torch.zeros(1, 2, 4, dtype=torch.int32)

    def attend(kc=k, vc=None, table=t, lens=n, x=q, y=q, win=None, wout=None, scale=None):
        runtime.paged_attention(x, kc, kc if vc is None else vc, table, lens, y, scale, win, wout)

    for bad, err, match in [
            (dict(vc=k[..., :32]), ValueError, "one shape"),
            (dict(vc=torch.zeros(4, 2, 16, 64).transpose(1, 2)), ValueError, "one shape"),
            (dict(vc=k.half()), ValueError, "one shape"), (dict(kc=k.double()), TypeError, "float32"),
            (dict(kc=k[..., ::2]), ValueError, "contiguous"), (dict(kc=k[0]), ValueError, "pages"),
            (dict(table=t.long()), TypeError, "int32"), (dict(lens=n.long()), TypeError, "int32"),
            (dict(table=torch.zeros(2, 2, dtype=torch.int32)), ValueError, "lens"),
            (dict(table=torch.zeros(2, 4, dtype=torch.int32)[:1, ::2]), ValueError, "contiguous"),
            (dict(x=q.half()), TypeError, "type"), (dict(y=q.half()), TypeError, "type"),
            (dict(x=q[0]), ValueError, "q must"), (dict(x=torch.zeros(2, 2, 64)), ValueError, "q must"),
            (dict(y=torch.zeros(1, 3, 64)), ValueError, "y must"), (dict(y=torch.zeros(1, 2, 128)[..., ::2]), ValueError, "y"),
            (dict(win=w), ValueError, "without"), (dict(wout=w.half()), TypeError, "float32"),
            (dict(wout=w[:, :1]), ValueError, "weights_out"), (dict(wout=w, win=w[0]), ValueError, "weights"),
            (dict(scale="x"), TypeError, None)]:
        with pytest.raises(err, match=match):
            attend(**bad)
    with pytest.raises(TypeError, match="torch tensor"):
        attend(x=np.zeros((1, 2, 64), np.float32))
    with pytest.raises(ValueError, match="without starts"):
        runtime.cache_append(torch.zeros(2, 2, 64), torch.zeros(2, 2, 64), k, k, t, n)
    with pytest.raises(ValueError, match="starts"):
        runtime.cache_append(q, q, k, k, t, n, torch.zeros(3, dtype=torch.int32))
    with pytest.raises(TypeError, match="starts"):
        runtime.cache_append(q, q, k, k, t, n, torch.zeros(2))
    with pytest.raises(ValueError, match="v must"):
        runtime.cache_append(q, torch.zeros(1, 2, 63), k, k, t, n)
    for bad, err, match in [
            (dict(kept=kept[..., :3]), ValueError, "kept"), (dict(new=n.long()), TypeError, "int32"),
            (dict(new=torch.zeros(2, dtype=torch.int32)), ValueError, "new_lens"), (dict(out=t[0]), ValueError, "out_table"),
            (dict(budget=2 ** 40), ValueError, "range"), (dict(budget="x"), TypeError, None)]:
        f = dict(out=t, new=n.clone(), kept=kept, budget=4)
        f.update(bad)
        with pytest.raises(err, match=match):
            runtime.cache_evict(k, k, t, n, w, w, f["out"], f["new"], f["kept"], f["budget"])


# ------------------------------------------------------------------ shared host arithmetic
def slot(row, pos, page=16, pages=9, ps=2048, ts=128):
    r = np.asarray(row, np.int32)
    return lib.lib().spinn_cuda_diag_cache_slot(r.ctypes.data_as(ctypes.POINTER(ctypes.c_int32)), len(r), pos, page, pages,
                                                ps, ts)


def test_slots():
    row = [3, 8, 0]
    for pos in range(48):
        assert slot(row, pos) == row[pos // 16] * 2048 + pos % 16 * 128
    assert slot(row, 48) == -2 and slot(row, -1) == -2
    for bad in (-1, 9, 2 ** 31 - 1, -2 ** 31):
        assert slot([3, bad, 0], 16) == -1 and slot([3, bad, 0], 15) == 3 * 2048 + 15 * 128
    # offsets past 32 bits, odd page sizes
    assert slot([2 ** 20], 5, page=7, pages=2 ** 20 + 1, ps=7 * 8 * 128, ts=1024) == 2 ** 20 * 7168 + 5 * 1024
    assert slot([0, 1], 3, page=3, pages=2, ps=30, ts=10) == 30


def test_attention_shares_cover_the_work_once():
    L = lib.lib()
    out = (ctypes.c_int64 * 3)()
    rng = np.random.default_rng(0)
    for units, workers in [(1, 296), (5, 3), (296, 296), (295, 296), (297, 296), (7, 1), (2 ** 31 - 1, 296)] + \
            [(int(rng.integers(1, 5000)), int(rng.integers(1, 300))) for _ in range(40)]:
        starts = []
        for w in range(workers):
            assert L.spinn_cuda_diag_attention_share(units, workers, w, 0, out) == 0
            starts.append((out[0], out[1]))
        assert starts[0][0] == 0 and starts[-1][1] == units
        assert all(a[1] == b[0] for a, b in zip(starts, starts[1:]))
        sizes = [b - a for a, b in starts]
        assert max(sizes) - min(sizes) <= 1
        for u in {0, units - 1, units // 2, *(int(x) for x in rng.integers(0, units, 20))}:
            L.spinn_cuda_diag_attention_share(units, workers, 0, u, out)
            a, b = starts[out[2]]
            assert a <= u < b
    assert L.spinn_cuda_diag_attention_share(0, 1, 0, 0, out) == lib.EINVAL


def rows(at, width, counts, strides, es=2):
    counts, strides = (list(counts) + [1] * 3)[:3], (list(strides) + [0] * 3)[:3]
    return (ctypes.c_int64 * 9)(at, es, width, *counts, *strides)


def elements(r):
    at, es, width, *cs = r
    out = [at + es * (i * cs[3] + j * cs[4] + k * cs[5] + e) + byte for i in range(cs[0]) for j in range(cs[1])
           for k in range(cs[2]) for e in range(width) for byte in range(es)]
    return out, set(out)


def test_overlaps_are_found():
    """No overlap passes, and what decoders do is not refused: slices of one buffer, orders of dimensions."""
    L = lib.lib()
    rng = np.random.default_rng(5)
    seen = [0, 0]
    for _ in range(4000):
        a, b = [rows(4096 + 2 * int(rng.integers(-30, 30)), int(rng.integers(1, 6)), rng.integers(1, 4, 2).tolist(),
                     rng.choice([0, 1, 4, 5, 6, 12, 18, 24], 2).tolist()) for _ in range(2)]
        (la, sa), (lb, sb) = elements(a), elements(b)
        got = L.spinn_cuda_diag_rows(a, b)
        if got & 1:
            assert len(la) == len(sa), list(a)
            seen[0] += 1
        if got & 2:
            assert not sa & sb, (list(a), list(b))
            seen[1] += 1
    assert min(seen) > 400
    far = rows(1 << 20, 8, (2, 2), (0, 0))
    for counts, strides in [((3, 8), (64, 8)), ((3, 8), (8, 24)), ((3, 8), (512, 16)), ((1, 1), (0, 0)), ((1, 4), (5, 8))]:
        assert L.spinn_cuda_diag_rows(rows(0, 8, counts, strides), far) == 3
    # query, key and value slices of one projection's rows, and y beside them
    assert L.spinn_cuda_diag_rows(rows(0, 64, (5, 8), (1024, 64)), rows(2 * 512, 64, (5, 4), (1024, 64))) & 2
    assert not L.spinn_cuda_diag_rows(rows(0, 64, (5, 8), (1024, 64)), rows(2 * 448, 64, (5, 4), (1024, 64))) & 2
    assert not L.spinn_cuda_diag_rows(rows(0, 8, (2,), (0,)), rows(1 << 20, 8, (1,), (0,))) & 1
    assert L.spinn_cuda_diag_rows(rows(0, 8, (1,), (0,)), rows(16, 8, (1,), (0,))) == 3



# ------------------------------------------------------------------ linear
def linear(**kw):
    f = dict(x=P, w=P, b=0, r=0, y=P, ldx=64, ldw=64, ldr=0, ldy=32, m=4, n=32, k=64, dtype=lib.BF16, act=0)
    f.update(kw)
    return LINEAR.pack(f["x"], f["w"], f["b"], f["r"], f["y"], f["ldx"], f["ldw"], f["ldr"], f["ldy"], f["m"],
                                f["n"], f["k"], f["dtype"], f["act"], 0)


@pytest.mark.parametrize("kw,match", [(dict(x=0), "required"), (dict(w=0), "required"), (dict(y=0), "required"),
                                      (dict(dtype=lib.FP32), "type 1"), (dict(m=0), "sizes"), (dict(n=-1), "sizes"),
                                      (dict(k=0), "sizes"), (dict(ldx=63), "stride"), (dict(ldw=0), "stride"),
                                      (dict(ldy=31), "stride"), (dict(r=P, ldr=8), "stride"), (dict(act=4), "activation"),
                                      (dict(act=2), "activation"), (dict(w=P + 1), "misaligned"),
                                      (dict(b=P + 1), "misaligned")])
def test_linear_refusals(kw, match):
    refused("spinn_cuda_linear", linear(**kw), None, 0, None, match=match)
    assert lib.lib().spinn_cuda_linear_workspace(linear(**kw)) == 0


def test_linear_workspace_holds_the_rows_that_are_off_alignment():
    ws = lib.lib().spinn_cuda_linear_workspace
    assert ws(linear(m=17)) == 0                              # aligned rows are read in place
    assert ws(linear(m=16, k=63, ldx=63, ldw=63)) == 0        # few rows: any alignment
    up = lambda b: -(-b // 256) * 256                         # noqa: E731
    assert ws(linear(m=17, k=63, ldx=63)) == up(17 * 128)
    assert ws(linear(m=17, k=63, ldx=64, ldw=63)) == up(32 * 128)
    assert ws(linear(m=17, x=P + 2)) == up(17 * 128)
    assert ws(linear(m=2 ** 20, n=2 ** 20, k=8191, ldx=8191, ldw=8191, ldy=2 ** 20)) == 2 * 2 ** 20 * 16384  # past 32 bits


def test_python_linear_refuses_what_does_not_match():
    torch = pytest.importorskip("torch")
    h = lambda *shape: torch.zeros(*shape, dtype=torch.float16)  # noqa: E731
    with pytest.raises(TypeError, match="CUDA"):
        runtime.linear(h(2, 8), h(4, 8), h(2, 4))
    for args, err, match in [((h(2, 8), h(4, 9), h(2, 4)), ValueError, r"\[m, k\]"),
                             ((h(2, 8), h(4, 8), h(2, 5)), ValueError, r"\[m, k\]"), ((h(8), h(4, 8), h(2, 4)), ValueError, None),
                             ((h(2, 8), h(4, 8).bfloat16(), h(2, 4)), TypeError, "float16"),
                             ((h(2, 8).float(), h(4, 8).float(), h(2, 4).float()), TypeError, "float16"),
                             ((h(2, 8), h(4, 8), h(2, 4), h(5)), ValueError, "bias"),
                             ((h(2, 8), h(4, 8), h(2, 4), h(8)[::2]), ValueError, "bias"),
                             ((h(2, 8), h(4, 8), h(2, 4), None, h(2, 5)), ValueError, "residual"),
                             ((h(2, 16)[:, ::2], h(4, 8), h(2, 4)), ValueError, "contiguous"),
                             ((h(2, 8), h(4, 8), h(4, 2).t()), ValueError, "contiguous"),
                             ((h(2, 8), h(4, 8), h(2, 4), None, None, "tanh"), ValueError, "act")]:
        with pytest.raises(err, match=match):
            runtime.linear(*args)
