"""Paged attention where one token dominates and the many behind it, of little weight each, still make
up the result: none of their mass may be lost on the way through the product with the values."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
LN2 = 0.6931471805599453


@pytest.fixture(scope="module")
def rt(cuda_lib):
    from spinn_b200 import runtime
    return runtime


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("depth,spread,value,dim,group,weights", [
    (14.5, 0.0, 1.0, 64, 1, False), (20.0, 10.0, 16.0, 64, 4, True), (25.3, 0.0, 4.0, 128, 4, False),
    (26.0, 1.0, 16.0, 64, 16, False), (30.0, 2.0, 256.0, 64, 7, True), (36.0, 0.0, 16384.0, 192, 8, False)])
def test_mass_behind_a_dominating_token(rt, dtype, depth, spread, value, dim, group, weights):
    """Four of the first 64 tokens, one for each warp that reads them, take the weight and have values of
    zero; the other 32764, `depth` to `depth + spread` powers of two below, make up y.  The sequences
    share their pages, and there are enough of them that a CTA reads thousands of tokens behind those four."""
    if dtype == "fp32" and group > 8:
        group = 8 if weights else group
    dt, n, page, heads, seqs = DTYPES[dtype], 32768, 64, 4, 80
    g = torch.Generator(device="cuda").manual_seed(int(depth * 10) + group)
    k = torch.zeros(n // page, page, heads, dim, dtype=dt, device="cuda")
    low = -(depth + spread * torch.rand(n, heads, generator=g, device="cuda")) * LN2
    sink = torch.zeros(n, dtype=torch.bool, device="cuda")
    sink[:64:16] = True
    low[sink] = 0.0
    k[..., 0] = (low / 8).to(dt).view(n // page, page, heads)
    v = (value * (0.75 + 0.25 * torch.rand(n, heads, dim, generator=g, device="cuda"))).to(dt)
    v[sink] = 0.0
    v = v.view(n // page, page, heads, dim)
    table = torch.arange(n // page, dtype=torch.int32, device="cuda").expand(seqs, -1).contiguous()
    lens = torch.full((seqs,), n, dtype=torch.int32, device="cuda")
    q = torch.zeros(seqs, heads * group, dim, dtype=dt, device="cuda")
    q[..., 0] = 8.0
    y = torch.full_like(q, float("nan"))
    wout = torch.zeros(seqs, heads, n, device="cuda") if weights else None
    rt.paged_attention(q, k, v, table, lens, y, 1.0, None, wout)
    rt.stream_sync()
    s = 8.0 * k.double()[..., 0].reshape(n, heads)
    p = torch.softmax(s, 0)
    want = torch.einsum("th,thd->hd", p, v.double().view(n, heads, dim)).repeat_interleave(group, 0)
    # scores are exact but for the factor log2(e) and its product's rounding, 2^-23 of at most 64; exp2 is
    # good to 2^-22, a 16-bit type's two parts to 2^-16; a worker sums its tokens in chains of at most
    # n / 16 steps of one MMA, each off by a fp32 step of the sum (v > 0); y is rounded once.  fp16 parts of
    # the 15 tokens beside each of the four are off by up to 2^-32 of its weight, 1/4
    half = torch.finfo(dt).eps / 2
    rel = 2 * (64 * 2.0 ** -23 + 2.0 ** -22 + n / 16 * 2.0 ** -23) + (0.0 if dtype == "fp32" else 2.0 ** -16)
    tol = (half + rel * (1 + half)) * want + (2.0 ** -25 + 60 * 2.0 ** -34 * value if dtype == "fp16" else 0.0)
    err = (y.double() - want).abs()
    assert (err <= tol).all(), float((err / tol).max())
    if weights:
        assert ((wout.double() - group * p.T).abs() <= (rel + group * 2.0 ** -23) * group * p.T).all()
