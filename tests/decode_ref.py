"""Plain 64-bit restatements of the decoder-serving operators, and caches to run them on.

Every pool starts out as NaN, and only the tokens that a sequence holds are filled: an operator
that lets a slot past a length, an unused page or the padding of a row into its result shows it.
"""
import numpy as np
import torch

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


class Paged:
    """A paged cache with `lens` tokens per sequence (`room` more slots in the table), on `device`."""

    def __init__(self, dtype, lens, kv_heads, dim, page, seed=0, room=0, layout="nhd", device="cuda", spare=2):
        g = torch.Generator().manual_seed(seed)
        rng = np.random.default_rng(seed)
        self.lens_host, self.page, self.dim, self.heads = list(lens), page, dim, kv_heads
        need = [-(-(n + room) // page) for n in lens]
        total = sum(need) + spare
        order = rng.permutation(total)
        table, at = np.full((len(lens), max(max(need), 1) + 1), -1, np.int32), 0  # -1: never read
        for s, n in enumerate(need):
            table[s, :n] = order[at:at + n]
            at += n
        self.free = [int(x) for x in order[at:]]
        dt = DTYPES[dtype]

        def pool():
            if layout == "hnd":      # heads outside tokens
                return torch.full((total, kv_heads, page, dim), float("nan"), dtype=dt).permute(0, 2, 1, 3)
            if layout == "odd":      # rows at odd element offsets, off every alignment
                flat = torch.full((total * page * kv_heads * (dim + 1) + 1,), float("nan"), dtype=dt)
                return flat[1:].view(total, page, kv_heads, dim + 1)[..., :dim]
            return torch.full((total, page, kv_heads, dim), float("nan"), dtype=dt)

        if layout == "pair":         # keys and values of a page side by side in one tensor
            both = torch.full((total, 2, page, kv_heads, dim), float("nan"), dtype=dt)
            k, v = both[:, 0], both[:, 1]
        else:
            k, v = pool(), pool()
        for s, n in enumerate(lens):
            t = np.arange(n)
            p, o = torch.from_numpy(table[s, t // page].astype(np.int64)), torch.from_numpy(t % page)
            k[p, o] = torch.randn(n, kv_heads, dim, generator=g).to(dt)
            v[p, o] = torch.randn(n, kv_heads, dim, generator=g).to(dt)
        self.table_host = table

        def put(t):  # keeps strides and offset
            base = t._base if t._base is not None else t
            return base.to(device).as_strided(t.shape, t.stride(), t.storage_offset())

        if layout == "pair":
            both = put(both)
            self.k, self.v = both[:, 0], both[:, 1]
        else:
            self.k, self.v = put(k), put(v)
        self.table = torch.from_numpy(table).to(device)
        self.lens = torch.tensor(list(lens), dtype=torch.int32, device=device)

    def rows(self, pool, s, n, head):
        """Tokens 0 .. n - 1 of a sequence and head, [n, dim] in float64 on the host."""
        t = np.arange(n)
        pages = torch.from_numpy(self.table_host[s][t // self.page].astype(np.int64))
        return pool.cpu()[pages, torch.from_numpy(t % self.page), head].double()


def attention(c, q, scale):
    """(y, probabilities summed over each group, sum_t p |v|, bound of a score's error)."""
    q = q.cpu().double()
    seqs, q_heads, dim = q.shape
    group = q_heads // c.heads
    most = max(max(c.lens_host), 1)
    y, absum = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    mass = torch.zeros(seqs, c.heads, most, dtype=torch.float64)
    ds = torch.zeros(seqs, q_heads, 1, dtype=torch.float64)
    kc, vc = c.k.cpu(), c.v.cpu()
    for s, n in enumerate(c.lens_host):
        if n == 0:
            continue
        for h in range(c.heads):
            k, v = c.rows(kc, s, n, h), c.rows(vc, s, n, h)
            g = slice(h * group, (h + 1) * group)
            p = torch.softmax(q[s, g] @ k.T * scale, -1)
            y[s, g], absum[s, g] = p @ v, p @ v.abs()
            mass[s, h, :n] = p.sum(0)
            # a dot product of dim terms summed in fp32 is off by at most dim 2^-24 sum |q k|
            ds[s, g, 0] = (q[s, g].abs() @ k.abs().T).amax(-1) * abs(scale) * dim * 2.0 ** -24
    return y, mass, absum, ds


def evict(weights, lens, budget, recent):
    """(kept [seqs][heads] lists, new lengths): weights as a float32 array [seqs, heads, length]."""
    kept, new = [], []
    for s, n in enumerate(lens):
        take = min(n, budget)
        old = n - min(recent, take)
        new.append(take)
        rows = []
        for h in range(weights.shape[1]):
            w = weights[s, h, :old].astype(np.float64)
            w = np.where(np.isnan(w), -np.inf, w)
            best = sorted(range(old), key=lambda i: (-w[i], i))[:take - (n - old)]
            rows.append(sorted(best) + list(range(old, n)))
        kept.append(rows)
    return kept, new
