"""Workloads of the decoder-serving operators: 16-bit linear layers with a fused epilogue, and a paged
key-value cache with its append, its one-token attention and its eviction by accumulated weight.

``run`` computes a case either in its plain form (elementary torch operations in 32 bits, rounded
once at the end) or, with ``own`` set, through the framework's operators.  ``exact`` gives the same
outputs from the operators' definitions in 64 bits.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"fp32": 4, "fp16": 2, "bf16": 2}


# ------------------------------------------------------------------ cases
def linear_case(name, dtype, m, k, n, act="none", bias=False, residual=False):
    return {"name": name, "op": "linear", "dtype": dtype, "m": m, "k": k, "n": n, "act": act, "bias": bias,
            "residual": residual}


def append_case(name, dtype, seqs, kv_heads, head_dim, page, past, new):
    return {"name": name, "op": "append", "dtype": dtype, "seqs": seqs, "kv_heads": kv_heads, "head_dim": head_dim,
            "page": page, "past": past, "new": new}


def attend_case(name, dtype, seqs, q_heads, kv_heads, head_dim, page, length, weights):
    return {"name": name, "op": "attend", "dtype": dtype, "seqs": seqs, "q_heads": q_heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "page": page, "length": length, "weights": weights}


def evict_case(name, dtype, seqs, kv_heads, head_dim, page, length, budget, recent):
    return {"name": name, "op": "evict", "dtype": dtype, "seqs": seqs, "kv_heads": kv_heads, "head_dim": head_dim,
            "page": page, "length": length, "budget": budget, "recent": recent}


def listed():
    return [
        # the 2048 -> 1000 classifier head for one image, in 16 bits: a call that is all latency
        linear_case("linear token fp16", "fp16", 1, 2048, 1000, bias=True),
        # a decoding batch through a square projection with its residual: reads the weights once
        linear_case("linear decode bf16", "bf16", 48, 4096, 4096, residual=True),
        # a ragged prompt through a layer whose sizes are odd, rows off every alignment
        linear_case("linear odd bf16", "bf16", 777, 1001, 2047, act="gelu", bias=True, residual=True),
        # a long prompt through the first feed-forward projection: bound by the matrix units
        linear_case("linear prompt bf16", "bf16", 4096, 4096, 8192, act="silu", bias=True),
        # one new token for each sequence of a decoding batch
        append_case("append decode bf16", "bf16", 64, 8, 128, 16, 4096, 1),
        # prompts of ragged lengths laid into pages that end inside them
        append_case("append prompt fp16", "fp16", 12, 8, 128, 24, 100, 4001),
        # one short conversation: a call that is all latency
        attend_case("attend short fp16", "fp16", 1, 16, 4, 64, 16, 333, False),
        # a full decoding batch of ragged lengths, one slot of it empty
        attend_case("attend batch bf16", "bf16", 32, 32, 8, 128, 16, 8192, False),
        # the 32-bit cache with an odd head size and pages, every head with its own keys
        attend_case("attend odd fp32", "fp32", 5, 6, 6, 80, 24, 5001, True),
        # few sequences with very long caches, which keep the weights for eviction
        attend_case("attend long bf16", "bf16", 3, 32, 8, 128, 64, 131072, True),
        # a batch cut back to a budget
        evict_case("evict batch bf16", "bf16", 16, 8, 128, 16, 4096, 1024, 64),
        # very long caches cut back
        evict_case("evict long fp16", "fp16", 3, 8, 128, 64, 131072, 16384, 512),
    ]


def spread(rng, low, high):
    """A whole number of [low, high], even over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["linear", "append", "attend", "evict"])
    half = rng.choice(["fp16", "bf16"])
    if op == "linear":
        step = rng.choice([1, 1, 8, 64])
        m, k, n = spread(rng, 1, 4096), spread(rng, 64, 4096), spread(rng, 64, 8192)
        k, n = max(step, k // step * step), max(step, n // step * step)
        c = linear_case("", half, m, k, n, rng.choice(["none", "relu", "silu", "gelu", "gelu_tanh"]),
                        rng.random() < 0.5, rng.random() < 0.5)
    else:
        dtype = rng.choice([half, half, "fp32"])
        kv_heads, head_dim = rng.choice([1, 2, 4, 5, 8]), rng.choice([64, 64, 72, 80, 96, 128, 128, 128, 192, 256])
        page = rng.choice([1, 8, 16, 16, 24, 32, 64, 100, 128])
        row = kv_heads * head_dim * BYTES[dtype]
        seqs = spread(rng, 1, 128)
        if op == "append":
            most = max(1, min(8192, (96 << 20) // (row * seqs)))
            c = append_case("", dtype, seqs, kv_heads, head_dim, page, rng.randrange(0, 2000),
                            rng.choice([1, spread(rng, 1, most)]))
        else:
            most = max(16, min(131072, (768 << 20) // (row * seqs)))
            length = spread(rng, 1, most)
            if op == "attend":
                c = attend_case("", dtype, seqs, kv_heads * rng.choice([1, 2, 4, 7, 8]), kv_heads, head_dim, page,
                                length, rng.random() < 0.4)
            else:
                budget = spread(rng, 1, max(1, min(16384, length)))
                c = evict_case("", dtype, seqs, kv_heads, head_dim, page, length, budget,
                               rng.choice([0, budget // 16, budget // 2]))
    del c["name"]
    return c


# ------------------------------------------------------------------ inputs
def lengths(seqs, most):
    """Lengths of a ragged batch: evenly spread up to `most`, an empty slot among eight and more."""
    return [0 if seqs >= 8 and i == 0 else -(-most * (i + 1) // seqs) for i in range(seqs)]


def randn(gen, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


def pages_for(rng, lens, page, spare=3):
    """A page table for caches of `lens` tokens, with pages in no order, and the number of pages in
    the pool; entries that no token needs are -1."""
    need = [-(-n // page) for n in lens]
    total = sum(need) + spare
    order = rng.permutation(total)
    table, at = np.full((len(lens), max(max(need), 1)), -1, np.int32), 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
    return table, total


def pool(gen, case, pages):
    shape = (pages, case["page"], case["kv_heads"], case["head_dim"])
    dtype = DTYPES[case["dtype"]]
    k = torch.empty(shape, dtype=dtype, device="cuda").normal_(generator=gen)
    v = torch.empty(shape, dtype=dtype, device="cuda").normal_(generator=gen)
    return k, v


def weights_like(gen, seqs, kv_heads, most):
    """Accumulated weights as decoding leaves them: most small, a few tokens with most of the mass."""
    return torch.randn((seqs, kv_heads, most), generator=gen, device="cuda").mul_(2.0).sub_(4.0).exp_()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rng = np.random.default_rng(seed)
    dtype = DTYPES[case["dtype"]]
    st = {"case": dict(case)}
    if case["op"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        st["x"] = randn(gen, (m, k), dtype)
        st["w"] = randn(gen, (n, k), dtype, k ** -0.5)
        st["bias"] = randn(gen, (n,), dtype, 0.5) if case["bias"] else None
        st["residual"] = randn(gen, (m, n), dtype) if case["residual"] else None
        st["y"] = torch.empty((m, n), dtype=dtype, device="cuda")
        return st
    seqs, kv_heads, head_dim, page = case["seqs"], case["kv_heads"], case["head_dim"], case["page"]
    order = rng.permutation(seqs)
    if case["op"] == "append":
        past = np.array(lengths(seqs, case["past"]), np.int64)[order]
        new = np.array(lengths(seqs, case["new"]), np.int64)[order] if case["new"] > 1 else np.ones(seqs, np.int64)
        table, pages = pages_for(rng, list(past + new), page)
        tokens = int(new.sum())
        st["k"] = randn(gen, (tokens, kv_heads, head_dim), dtype)
        st["v"] = randn(gen, (tokens, kv_heads, head_dim), dtype)
        starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        st["starts"] = torch.from_numpy(starts).cuda() if case["new"] > 1 else None
        st["lens"] = torch.from_numpy(past.astype(np.int32)).cuda()
    else:
        lens = np.array(lengths(seqs, case["length"]), np.int64)[order]
        st["lens"] = torch.from_numpy(lens.astype(np.int32)).cuda()
        if case["op"] == "attend":
            table, pages = pages_for(rng, list(lens), page)
            st["q"] = randn(gen, (seqs, case["q_heads"], head_dim), dtype, 2.0)
            st["y"] = torch.empty_like(st["q"])
            st["weights"] = st["weights_out"] = None
            if case["weights"]:
                st["weights"] = weights_like(gen, seqs, kv_heads, case["length"])
                st["weights_out"] = torch.zeros_like(st["weights"])
        else:
            kept = np.minimum(lens, case["budget"])
            both, pages = pages_for(rng, list(lens) + list(kept), page)
            table, wide = both[:seqs], max(1, -(-case["budget"] // page))
            out_table = np.full((seqs, wide), -1, np.int32)
            out_table[:, :min(wide, both.shape[1])] = both[seqs:, :wide]
            st["out_table"] = torch.from_numpy(out_table).cuda()
            st["weights"] = weights_like(gen, seqs, kv_heads, case["length"])
            st["weights_out"] = torch.zeros_like(st["weights"])
            st["new_lens"] = torch.empty(seqs, dtype=torch.int32, device="cuda")
            st["kept"] = torch.empty((seqs, kv_heads, case["budget"]), dtype=torch.int32, device="cuda")
    st["table"] = torch.from_numpy(np.ascontiguousarray(table)).cuda()
    st["k_cache"], st["v_cache"] = pool(gen, case, pages)
    return st


# ------------------------------------------------------------------ one pass
def run(st):
    return {"linear": run_linear, "append": run_append, "attend": run_attend, "evict": run_evict}[st["case"]["op"]](st)


def run_linear(st):
    x, w, y = st["x"], st["w"], st["y"]
    if own:
        from spinn_b200 import runtime
        runtime.linear(x, w, y, st["bias"], st["residual"], st["case"]["act"])
        return y
    z = x.float() @ w.float().t()
    if st["bias"] is not None:
        z = z + st["bias"].float()
    act = st["case"]["act"]
    if act == "relu":
        z = torch.where(z < 0, torch.zeros_like(z), z)
    elif act == "silu":
        z = z / (1 + torch.exp(-z))
    elif act == "gelu":
        z = 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    elif act == "gelu_tanh":
        z = 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    if st["residual"] is not None:
        z = z + st["residual"].float()
    return z.to(y.dtype)


def token_rows(table, positions, page):
    """Row of the pool, counted over its pages' tokens, for positions [seqs, n] of each sequence."""
    blocks = torch.div(positions, page, rounding_mode="floor")
    there = torch.gather(table.long(), 1, blocks.clamp(0, table.shape[1] - 1))
    return there.clamp_min(0) * page + positions % page


def run_append(st):
    k_cache, v_cache, k = st["k_cache"], st["v_cache"], st["k"]
    if own:
        from spinn_b200 import runtime
        runtime.cache_append(k, st["v"], k_cache, v_cache, st["table"], st["lens"], st["starts"])
        return k_cache, v_cache
    seqs, page = st["lens"].shape[0], k_cache.shape[1]
    token = torch.arange(k.shape[0], device=k.device)
    if st["starts"] is None:
        seq, at = token, st["lens"].long()
    else:
        starts = st["starts"].long()
        seq = torch.searchsorted(starts, token, right=True) - 1
        at = st["lens"].long()[seq] + token - starts[seq]
    rows = st["table"].long()[seq, torch.div(at, page, rounding_mode="floor")] * page + at % page
    k_cache.flatten(0, 1)[rows] = k
    v_cache.flatten(0, 1)[rows] = st["v"]
    return k_cache, v_cache


def run_attend(st):
    q, k_cache, v_cache, lens, y = st["q"], st["k_cache"], st["v_cache"], st["lens"], st["y"]
    if own:
        from spinn_b200 import runtime
        runtime.paged_attention(q, k_cache, v_cache, st["table"], lens, y, weights=st["weights"],
                                weights_out=st["weights_out"])
        return (y, st["weights_out"]) if st["weights"] is not None else y
    seqs, q_heads, head_dim = q.shape
    kv_heads, most = k_cache.shape[2], st["case"]["length"]
    at = torch.arange(most, device=q.device)
    rows = token_rows(st["table"], at.expand(seqs, most), k_cache.shape[1])
    there = at < lens[:, None]                                              # [seqs, most]
    k = k_cache.flatten(0, 1)[rows].permute(0, 2, 3, 1).float()             # [seqs, kv_heads, head_dim, most]
    scores = (q.float().view(seqs, kv_heads, -1, head_dim) @ k) / math.sqrt(head_dim)
    del k
    scores = torch.where(there[:, None, None], scores, torch.full_like(scores, -math.inf))
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(total == 0, torch.ones_like(total), total)
    v = v_cache.flatten(0, 1)[rows].float()
    v = torch.where(there[:, :, None, None], v, torch.zeros_like(v)).transpose(1, 2)
    out = (p @ v).reshape(seqs, q_heads, head_dim).to(y.dtype)
    if st["weights"] is None:
        return out
    w = torch.where(there[:, None], st["weights"] + p.sum(2), st["weights_out"])
    return out, w


def run_evict(st):
    k_cache, v_cache, lens, weights = st["k_cache"], st["v_cache"], st["lens"], st["weights"]
    budget, recent = st["case"]["budget"], st["case"]["recent"]
    if own:
        from spinn_b200 import runtime
        runtime.cache_evict(k_cache, v_cache, st["table"], lens, weights, st["weights_out"], st["out_table"],
                            st["new_lens"], st["kept"], budget, recent)
        return st["kept"], st["new_lens"], st["weights_out"], k_cache, v_cache
    seqs, kv_heads, most = weights.shape
    page = k_cache.shape[1]
    at = torch.arange(most, device=weights.device)
    n = lens.clamp_max(budget)
    there = at < lens[:, None]
    late = there & (at >= (lens - n.clamp_max(recent))[:, None])
    # NaN counts as the lowest; what is not there sorts behind everything that is
    key = torch.where(torch.isnan(weights), torch.full_like(weights, -math.inf), weights)
    key = torch.where(late[:, None], torch.full_like(key, math.inf), key)
    group = torch.where(late, 0, torch.where(there, 1, 2))[:, None].expand(seqs, kv_heads, most)
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices
    order = torch.gather(order, -1, torch.sort(torch.gather(group, -1, order), dim=-1, stable=True).indices)
    rank = torch.empty_like(order).scatter_(-1, order, at.expand_as(order).contiguous())
    keep = rank < n[:, None, None]
    wide = min(budget, most)
    slots = torch.sort((~keep).to(torch.int8), dim=-1, stable=True).indices[..., :wide]   # [seqs, kv_heads, wide]
    filled = (at[:wide] < n[:, None])[:, None].expand_as(slots)
    kept = torch.full((seqs, kv_heads, budget), -1, dtype=torch.int32, device=weights.device)
    kept[..., :wide] = torch.where(filled, slots, torch.full_like(slots, -1)).to(torch.int32)
    w = st["weights_out"].clone()
    w[..., :wide] = torch.where(filled, torch.gather(weights, -1, slots), w[..., :wide])
    w = torch.where((there & (at >= n[:, None]))[:, None], torch.zeros_like(w), w)
    src = torch.gather(st["table"].long()[:, None].expand(seqs, kv_heads, -1), -1,
                       torch.div(slots, page, rounding_mode="floor"))
    src = src * page + slots % page
    dst = token_rows(st["out_table"], at[:wide].expand(seqs, wide), page)[:, None].expand_as(src)
    head = torch.arange(kv_heads, device=weights.device)[None, :, None].expand_as(src)
    src, dst, head = src[filled], dst[filled], head[filled]
    k_rows, v_rows = k_cache.flatten(0, 1), v_cache.flatten(0, 1)
    k_rows[dst, head] = k_rows[src, head]
    v_rows[dst, head] = v_rows[src, head]
    return kept, n.to(torch.int32), w, k_cache, v_cache


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    size = BYTES[case["dtype"]]
    if case["op"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        return {"bytes": size * (m * k + n * k + m * n * (2 if case["residual"] else 1) + (n if case["bias"] else 0)),
                "flops": 2 * m * n * k}
    seqs, heads, dim = case["seqs"], case["kv_heads"], case["head_dim"]
    if case["op"] == "append":
        tokens = sum(lengths(seqs, case["new"])) if case["new"] > 1 else seqs
        return {"bytes": tokens * heads * dim * size * 4 + 8 * seqs, "flops": 0}
    lens = lengths(seqs, case["length"])
    if case["op"] == "attend":
        entries = sum(lens) * heads
        moved = entries * dim * size * 2 + 2 * seqs * case["q_heads"] * dim * size
        return {"bytes": moved + (8 * entries if case["weights"] else 0),
                "flops": 4 * sum(lens) * case["q_heads"] * dim}
    kept = sum(min(n, case["budget"]) for n in lens) * heads
    return {"bytes": kept * dim * size * 4 + sum(lens) * heads * 8 + kept * 4, "flops": 0}


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "linear":
        z = torch.mm(st["x"].double(), st["w"].double().T)
        if case["bias"]:
            z += st["bias"].double()
        if case["act"] == "relu":
            z = z.clamp_min(0)
        elif case["act"] == "silu":
            z = z * torch.special.expit(z)
        elif case["act"] == "gelu":
            z = z * torch.special.ndtr(z)
        elif case["act"] == "gelu_tanh":
            z = z * torch.special.expit(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
        return z + st["residual"].double() if case["residual"] else z
    lens, table = st["lens"].tolist(), st["table"].cpu().numpy().astype(np.int64)
    page = case["page"]

    def places(row, positions):
        return torch.from_numpy(row[positions // page]).cuda(), torch.from_numpy(positions % page).cuda()

    if case["op"] == "append":
        starts = st["starts"].tolist() if st["starts"] is not None else list(range(case["seqs"] + 1))
        for s, n in enumerate(lens):
            a, b = starts[s], starts[s + 1]
            p, o = places(table[s], np.arange(n, n + b - a))
            st["k_cache"][p, o], st["v_cache"][p, o] = st["k"][a:b], st["v"][a:b]
        return st["k_cache"], st["v_cache"]
    if case["op"] == "attend":
        y = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
        w = st["weights_out"].double() if case["weights"] else None
        group = case["q_heads"] // case["kv_heads"]
        for s, n in enumerate(lens):
            if n == 0:
                continue
            p, o = places(table[s], np.arange(n))
            for h in range(case["kv_heads"]):
                k, v = st["k_cache"][p, o, h].double(), st["v_cache"][p, o, h].double()
                q = st["q"][s, h * group:(h + 1) * group].double()
                prob = torch.softmax((q @ k.T) * case["head_dim"] ** -0.5, dim=1)
                y[s, h * group:(h + 1) * group] = prob @ v
                if w is not None:
                    w[s, h, :n] = st["weights"][s, h, :n].double() + prob.sum(0)
        return (y, w) if w is not None else y
    weights, out_table = st["weights"].cpu().numpy(), st["out_table"].cpu().numpy().astype(np.int64)
    w = st["weights_out"].cpu().numpy().astype(np.float64)
    kept = np.full((case["seqs"], case["kv_heads"], case["budget"]), -1, np.int32)
    new_lens = np.minimum(lens, case["budget"]).astype(np.int32)
    k_out, v_out = st["k_cache"].clone(), st["v_cache"].clone()
    for s, n in enumerate(lens):
        take = int(new_lens[s])
        old = n - min(case["recent"], take)
        for h in range(case["kv_heads"]):
            values = weights[s, h, :old].astype(np.float64)
            best = np.lexsort((np.arange(old), -np.where(np.isnan(values), -np.inf, values)))[:take - (n - old)]
            slots = np.concatenate([np.sort(best), np.arange(old, n)]).astype(np.int64)
            kept[s, h, :take] = slots
            w[s, h, :n] = 0
            w[s, h, :take] = weights[s, h, slots]
            if take:
                (p, o), (to, at) = places(table[s], slots), places(out_table[s], np.arange(take))
                k_out[to, at, h], v_out[to, at, h] = st["k_cache"][p, o, h], st["v_cache"][p, o, h]
    return torch.from_numpy(kept), torch.from_numpy(new_lens), torch.from_numpy(w), k_out, v_out
