"""The decoder-serving operators together, as a serving loop uses them: one layer decodes tokens for
a batch -- projections, append, attention that keeps the accumulated weights, feed-forward -- and
cuts the cache back whenever it passes its budget.  Every operator's result is held against 64
bits on the inputs it got, and a plain mirror of the cache follows all moves."""
import numpy as np
import pytest
import torch

import decode_ref

pytestmark = pytest.mark.gpu

SEQS, HEADS, GROUP, DIM, HIDDEN, PAGE = 3, 2, 4, 64, 512, 16
CAP, BUDGET, RECENT = 64, 40, 8


def lin64(x, w, b=None, r=None):
    z = x.double() @ w.double().T + (0 if b is None else b.double())
    return z, z if r is None else z + r.double()


def close(got, want, mass, k):
    tol = 2.0 ** -8 * want.abs() + 2.0 * k * 2.0 ** -23 * mass + 2.0 ** -18 * (want.abs() + 1)
    assert ((got.double() - want).abs() <= tol).all()


def test_decode_loop(cuda_lib):
    from spinn_b200 import runtime as rt
    torch.manual_seed(0)
    dt, dev = torch.bfloat16, "cuda"
    q_heads = HEADS * GROUP
    width = (q_heads + 2 * HEADS) * DIM
    mk = lambda n, k: (torch.randn(n, k, device=dev) * k ** -0.5).to(dt)  # noqa: E731
    wqkv, wo, w1, w2 = mk(width, HIDDEN), mk(HIDDEN, q_heads * DIM), mk(4 * HIDDEN, HIDDEN), mk(HIDDEN, 4 * HIDDEN)
    bqkv = torch.randn(width, device=dev).to(dt)
    pages = SEQS * (CAP // PAGE) + 1
    k_cache = torch.full((pages, PAGE, HEADS, DIM), float("nan"), dtype=dt, device=dev)
    v_cache = k_cache.clone()
    table = torch.randperm(pages)[:SEQS * (CAP // PAGE)].to(torch.int32).view(SEQS, -1).to(dev)
    lens = torch.tensor([0, 5, 0], dtype=torch.int32, device=dev)
    weights = torch.zeros(SEQS, HEADS, CAP, device=dev)
    # a first prompt for sequence 1
    pk, pv = torch.randn(5, HEADS, DIM, device=dev).to(dt), torch.randn(5, HEADS, DIM, device=dev).to(dt)
    rt.cache_append(pk, pv, k_cache, v_cache, table, torch.zeros_like(lens),
                    torch.tensor([0, 0, 5, 5], dtype=torch.int32, device=dev))
    mirror = {(s, h): [[], []] for s in range(SEQS) for h in range(HEADS)}
    for t in range(5):
        for h in range(HEADS):
            mirror[1, h][0].append(pk[t, h].clone())
            mirror[1, h][1].append(pv[t, h].clone())
    x = torch.randn(SEQS, HIDDEN, device=dev).to(dt)
    qkv = torch.empty(SEQS, width, dtype=dt, device=dev)
    att = torch.empty(SEQS, q_heads, DIM, dtype=dt, device=dev)
    h1, up, nxt = torch.empty_like(x), torch.empty(SEQS, 4 * HIDDEN, dtype=dt, device=dev), torch.empty_like(x)
    kept = torch.empty(SEQS, HEADS, BUDGET, dtype=torch.int32, device=dev)
    cuts = 0
    for step in range(70):
        rt.linear(x, wqkv, qkv, bqkv)
        view = qkv.view(SEQS, q_heads + 2 * HEADS, DIM)
        q, k, v = view[:, :q_heads], view[:, q_heads:q_heads + HEADS], view[:, q_heads + HEADS:]
        rt.cache_append(k, v, k_cache, v_cache, table, lens)
        lens += 1
        before = weights.clone()
        rt.paged_attention(q, k_cache, v_cache, table, lens, att, None, weights, weights)
        rt.linear(att.view(SEQS, -1), wo, h1, None, x)
        rt.linear(h1, w1, up, act="gelu")
        rt.linear(up, w2, nxt, None, h1)
        rt.stream_sync()

        for s in range(SEQS):
            for h in range(HEADS):
                mirror[s, h][0].append(k[s, h].clone())
                mirror[s, h][1].append(v[s, h].clone())
        z, want = lin64(x, wqkv, bqkv)
        close(qkv, want, x.double().abs() @ wqkv.double().abs().T, HIDDEN)
        for s in range(SEQS):
            n = int(lens[s])
            for h in range(HEADS):
                ks, vs = (torch.stack(m).double() for m in mirror[s, h])
                assert ks.shape[0] == n
                g = slice(h * GROUP, (h + 1) * GROUP)
                p = torch.softmax(q[s, g].double() @ ks.T * DIM ** -0.5, -1)
                want, absum = p @ vs, p @ vs.abs()
                ds = (q[s, g].double().abs() @ ks.abs().T).amax() * DIM ** -0.5 * DIM * 2.0 ** -24
                rel = 2 * (float(ds) + 2.0 ** -17 + n * 2.0 ** -24)
                assert ((att[s, g].double() - want).abs() <= 2.0 ** -8 * want.abs() + rel * absum).all()
                got = weights[s, h, :n].double() - before[s, h, :n].double()
                assert ((got - p.sum(0)).abs() <= rel * p.sum(0) + 2.0 ** -22 * weights[s, h, :n]).all()
        _, want = lin64(att.view(SEQS, -1), wo, None, x)
        close(h1, want, att.view(SEQS, -1).double().abs() @ wo.double().abs().T, q_heads * DIM)
        z, _ = lin64(h1, w1)
        close(up, torch.nn.functional.gelu(z), h1.double().abs() @ w1.double().abs().T, HIDDEN)
        _, want = lin64(up, w2, None, h1)
        close(nxt, want, up.double().abs() @ w2.double().abs().T, 4 * HIDDEN)
        x = (nxt / nxt.float().square().mean(-1, keepdim=True).sqrt()).to(dt)

        if int(lens.max()) == CAP:
            cuts += 1
            w = weights.cpu().numpy()
            want_kept, want_new = decode_ref.evict(w, lens.tolist(), BUDGET, RECENT)
            new = torch.empty_like(lens)
            rt.cache_evict(k_cache, v_cache, table, lens, weights, weights, table, new, kept, BUDGET, RECENT)
            rt.stream_sync()
            lens = new
            assert lens.tolist() == want_new
            for s in range(SEQS):
                for h in range(HEADS):
                    slots = want_kept[s][h]
                    assert kept[s, h, :len(slots)].tolist() == slots
                    for m in mirror[s, h]:
                        m[:] = [m[i] for i in slots]
                    np.testing.assert_array_equal(weights[s, h, :len(slots)].cpu().numpy(), w[s, h, slots])
            rows = table.long()[:, torch.arange(CAP, device=dev) // PAGE] * PAGE + torch.arange(CAP, device=dev) % PAGE
            flat_k, flat_v = k_cache.flatten(0, 1), v_cache.flatten(0, 1)
            for (s, h), (ks, vs) in mirror.items():
                at = rows[s, :len(ks)]
                assert torch.equal(flat_k[at, h], torch.stack(ks)) and torch.equal(flat_v[at, h], torch.stack(vs))
    assert cuts >= 1
