"""Every kernel that a 16-bit linear layer may take -- each tile shape, alone, in pairs and with k split each way,
and the kernel for few rows -- on ragged sizes with the whole epilogue, aligned and off alignment.
The library's own choice is asked for each case, so that other choices do not quietly leave a kernel untested."""
import ctypes
import math
import random
import struct

import pytest

from spinn_b200 import lib

LINEAR = struct.Struct("<QQQQQqqqqiiiiii")  # SpinnCudaLinear
SMS = 148

# m, k, n, and the tile: rows of x (0: the kernel for few rows), CTAs of a pair, ways in which k is split
CASES = [
    (7, 333, 150, (0, 1, 1)), (13, 999, 261, (0, 1, 1)), (29, 520, 157, (0, 1, 1)),
    (36, 37, 151, (32, 1, 1)), (65, 1171, 2395, (32, 1, 2)), (35, 903, 155, (32, 1, 4)), (35, 1949, 169, (32, 1, 8)),
    (4877, 35, 257, (64, 1, 1)), (1239, 1667, 153, (64, 1, 2)), (561, 943, 151, (64, 1, 4)), (238, 1933, 151, (64, 1, 8)),
    (1438, 33, 7497, (128, 1, 1)), (132, 3487, 4481, (128, 1, 2)), (915, 2347, 257, (128, 1, 4)),
    (557, 4649, 155, (128, 1, 8)), (4765, 35, 5931, (128, 2, 1)), (1634, 2729, 269, (128, 2, 2)),
    (797, 2431, 267, (128, 2, 4)), (5529, 35, 8105, (256, 2, 1)), (1277, 1311, 5001, (128, 2, 1)),
]
ACTS = ["relu", "silu", "gelu", "gelu_tanh", "none"]


def plan(m, k, n, pad=0, at=4096):
    out = (ctypes.c_int * 5)()
    desc = LINEAR.pack(at, 4096, 0, 0, 4096, k + pad, k + pad, 0, n, m, n, k, lib.BF16, 0, 0)
    assert lib.lib().spinn_cuda_diag_linear_plan(desc, SMS, out) == 0
    return tuple(out[:3]), bool(out[3]), bool(out[4])


@pytest.mark.parametrize("m,k,n,tile", CASES)
def test_cases_take_the_kernel_that_they_are_for(m, k, n, tile):
    pad = -k % 8
    assert plan(m, k, n, pad) == (tile, False, False)
    if m <= 16 or tile[0]:
        shape, copy_x, copy_w = plan(m, k, n, pad + 1)
        assert shape == tile and (copy_x, copy_w) == ((tile[0] > 0,) * 2)


def test_no_size_takes_a_kernel_without_a_case():
    rng = random.Random(3)
    seen = set()
    for _ in range(40000):
        m, k, n = (int(round(math.exp(rng.uniform(math.log(a), math.log(b))))) for a, b in ((1, 9000), (8, 20000), (1, 40000)))
        seen.add(plan(m, k, n, rng.choice([0, 1, -k % 8]))[0])
    assert seen == {c[3] for c in CASES}


def test_plan_diagnostic_refuses_what_the_layer_refuses():
    out = (ctypes.c_int * 5)()
    bad = LINEAR.pack(4096, 4096, 0, 0, 4096, 8, 8, 0, 8, 0, 8, 8, lib.BF16, 0, 0)
    assert lib.lib().spinn_cuda_diag_linear_plan(bad, SMS, out) == lib.EINVAL
    assert lib.lib().spinn_cuda_diag_linear_plan(LINEAR.pack(4096, 4096, 0, 0, 4096, 8, 8, 0, 8, 8, 8, 8, lib.BF16, 0, 0), 0,
                                                 out) == lib.EINVAL


@pytest.mark.gpu
@pytest.mark.parametrize("m,k,n,tile", CASES)
@pytest.mark.parametrize("layout", ["aligned", "off", "copied"])
def test_every_kernel_matches_the_definition(cuda_lib, m, k, n, tile, layout):
    import torch

    from spinn_b200 import runtime as rt
    from test_gpu_linear import act64
    if layout == "copied" and m > 16 and tile[0] == 0:
        pytest.skip("rows of this number off alignment go to the tiles")
    dt = torch.float16 if (m + n) % 3 == 0 else torch.bfloat16
    act = ACTS[(m + k + n) % 5]
    torch.manual_seed(m + k)

    def rows(r, c, pad, shift, scale=1.0):
        """Rows `pad` elements apart beyond their length, `shift` elements into their storage, NaN between them."""
        flat = torch.full((r * (c + pad) + shift + 8,), float("nan"), dtype=dt, device="cuda")
        t = flat[shift:shift + r * (c + pad)].view(r, c + pad)
        t[:, :c] = (torch.randn(r, c, device="cuda") * scale).to(dt)
        return t[:, :c], t[:, c:]

    xpad = -k % 8 + (layout == "copied")
    ypad, shift = (-n % 8, 0) if layout == "aligned" else (2, 1)
    (x, _), (w, _) = rows(m, k, xpad, 0), rows(n, k, xpad, 0, k ** -0.5)
    (y, gaps), (res, _) = rows(m, n, ypad, shift), rows(m, n, ypad, shift)
    bias = torch.randn(n, device="cuda").to(dt)
    assert plan(m, k, n, xpad, x.data_ptr())[0] == tile
    rt.linear(x, w, y, bias, res, act)
    rt.stream_sync()
    first = y.clone()
    y.fill_(float("nan"))
    rt.linear(x, w, y, bias, res, act)
    rt.stream_sync()
    assert torch.equal(y, first) and bool(torch.isnan(gaps).all())
    z = x.double() @ w.double().T + bias.double()
    mass = x.double().abs() @ w.double().abs().T + bias.double().abs()
    want = act64(z, act) + res.double()
    # a sum of k + 1 products in fp32 in any order, the tensor core's truncating adder counted as a whole step:
    # (k + 1) 2^-23 of the sum of magnitudes; no activation is steeper than 1.13 and its arithmetic is good to 2^-20
    # of |z| + 1; then fp32 adds and one rounding, in steps of 2^-24 below fp16's 2^-14
    half = torch.finfo(dt).eps / 2
    slack = 1.13 * (k + 1) * 2.0 ** -23 * mass + 2.0 ** -20 * (z.abs() + 1) + 2.0 ** -22 * (z.abs() + want.abs())
    tol = half * want.abs() + (1 + half) * slack + (2.0 ** -25 if dt == torch.float16 else 0.0)
    err = (y.double() - want).abs()
    assert (err <= tol).all(), float((err / tol).max())
