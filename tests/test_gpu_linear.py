"""16-bit linear layers on the GPU against the same formula in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def rt(cuda_lib):
    from spinn_b200 import runtime
    return runtime


def act64(z, act):
    if act == "relu":
        return z.clamp_min(0)
    if act == "silu":
        return z * torch.sigmoid(z)
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z / math.sqrt(2)))
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    return z


def rows(shape, dtype, pad=0, shift=0, scale=1.0):
    """A matrix whose rows are `pad` elements apart beyond their length, `shift` elements into its
    storage; the gaps hold NaN."""
    m, k = shape
    flat = torch.full((m * (k + pad) + shift + 8,), float("nan"), dtype=dtype, device="cuda")
    t = flat[shift:shift + m * (k + pad)].view(m, k + pad)[:, :k]
    t.copy_((torch.randn(m, k, device="cuda") * scale).to(dtype))
    return t


CASES = [
    # dtype, m, k, n, act, bias, residual, (pad, shift) of x, w, y, residual
    ("fp16", 1, 1, 1, "none", False, False, (0, 0)),
    ("bf16", 1, 64, 16, "none", True, True, (0, 0)),
    ("fp16", 1, 2048, 1000, "none", True, False, (0, 0)),
    ("bf16", 3, 1001, 77, "gelu", True, True, (0, 0)),      # odd rows: element loads
    ("bf16", 8, 520, 100, "silu", True, False, (8, 8)),
    ("fp16", 9, 520, 100, "gelu_tanh", False, True, (3, 1)),
    ("bf16", 16, 4096, 48, "relu", True, True, (0, 0)),
    ("fp16", 16, 31, 5, "silu", True, True, (1, 1)),
    ("bf16", 17, 64, 128, "none", False, False, (0, 0)),    # first size of the tile kernel
    ("fp16", 17, 1, 1, "gelu", True, True, (0, 0)),
    ("bf16", 32, 40, 130, "silu", True, True, (0, 0)),
    ("bf16", 48, 4096, 512, "none", True, True, (0, 0)),    # k split over a cluster
    ("fp16", 33, 1000, 257, "gelu", True, True, (0, 0)),
    ("bf16", 64, 2048, 1000, "relu", False, True, (8, 16)),
    ("fp16", 65, 513, 129, "gelu_tanh", True, True, (0, 0)),  # operands copied to an aligned pitch
    ("bf16", 100, 777, 333, "none", True, True, (5, 3)),
    ("bf16", 128, 128, 128, "silu", False, False, (0, 0)),
    ("fp16", 129, 200, 64, "relu", True, True, (0, 0)),
    ("bf16", 777, 1001, 2047, "gelu", True, True, (0, 0)),
    ("fp16", 300, 4096, 130, "none", False, True, (0, 0)),
    ("bf16", 2100, 320, 2300, "silu", True, True, (0, 0)),  # CTA pairs, ragged on both sides
    ("fp16", 2048, 2048, 2304, "none", False, False, (0, 0)),
    ("bf16", 5000, 64, 1100, "gelu_tanh", True, True, (1, 1)),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{c[0]}-{c[1]}x{c[2]}x{c[3]}-{c[4]}-{c[7][0]}.{c[7][1]}")
def test_linear_matches_its_definition(rt, case):
    dtype, m, k, n, act, has_bias, has_res, (pad, shift) = case
    torch.manual_seed(m * 7 + k * 3 + n)
    dt = DTYPES[dtype]
    x, w = rows((m, k), dt, pad, shift), rows((n, k), dt, pad, shift, k ** -0.5)
    y, res = rows((m, n), dt, pad, shift), rows((m, n), dt, pad, shift) if has_res else None
    bias = torch.randn(n, device="cuda").to(dt) if has_bias else None
    gaps = y.as_strided((m, n + pad), (n + pad, 1), y.storage_offset())[:, n:].clone()
    rt.linear(x, w, y, bias, res, act)
    rt.stream_sync()
    z = x.double() @ w.double().T
    mass = x.double().abs() @ w.double().abs().T
    if has_bias:
        z = z + bias.double()
    want = act64(z, act)
    if has_res:
        want = want + res.double()
    # the sum of k exact products in fp32, in any order, the tensor core's truncating adder counted
    # as a whole step: k 2^-23 of the sum of their magnitudes; no activation is steeper than 1.13;
    # its own arithmetic is good to 2^-20 of |z| + 1; then fp32 adds and one rounding
    half = torch.finfo(dt).eps / 2
    slack = 1.13 * k * 2.0 ** -23 * mass + (0 if act == "none" else 2.0 ** -20) * (z.abs() + 1) + 2.0 ** -22 * (
        z.abs() + want.abs())
    tiny = 2.0 ** -25 if dtype == "fp16" else 0.0  # fp16 rounds in steps of 2^-24 below 2^-14
    tol = half * want.abs() + (1 + half) * slack + tiny
    err = (y.double() - want).abs()
    assert torch.isfinite(y).all()
    assert (err <= tol).all(), float((err / tol.clamp_min(1e-30)).max())
    after = y.as_strided((m, n + pad), (n + pad, 1), y.storage_offset())[:, n:]
    assert torch.equal(torch.isnan(after), torch.isnan(gaps))


def test_linear_in_place_of_its_residual(rt):
    for m in (5, 50, 700):
        x = rows((m, 256), torch.bfloat16)
        w = rows((384, 256), torch.bfloat16, scale=1 / 16)
        r = rows((m, 384), torch.bfloat16)
        y = torch.empty_like(r)
        rt.linear(x, w, y, None, r)
        rt.linear(x, w, r, None, r)
        rt.stream_sync()
        assert torch.equal(y, r)


@pytest.mark.parametrize("m,k,n,pad", [(1, 8192, 2048, 0), (8, 4096, 8192, 0), (16, 1024, 8200, 0), (16, 8192, 1024, 8),
                                       (1, 4095, 4100, 0), (12, 3001, 2304, 3), (5, 16000, 33, 0), (17, 1000, 1031, 0),
                                       (32, 520, 4096, 8), (25, 1024, 513, 0)])
def test_linear_few_rows_of_large_weights(rt, m, k, n, pad):
    """Few rows of x on both sides of the choice of a kernel, aligned or copied first, with the whole epilogue."""
    dtype = torch.bfloat16
    x, w, res = rows((m, k), dtype, pad), rows((n, k), dtype, pad, scale=k ** -0.5), rows((m, n), dtype)
    bias, y = torch.randn(n, device="cuda").to(dtype), torch.full((m + 1, n), 7.0, device="cuda", dtype=dtype)
    rt.linear(x, w, y[:m], bias, res, "relu")
    rt.stream_sync()
    z = x.double() @ w.double().T + bias.double()
    want = z.relu() + res.double()
    mass = x.double().abs() @ w.double().abs().T + bias.double().abs()
    # as above: k 2^-23 of the sum of magnitudes, fp32 adds, one rounding to bf16
    tol = 2.0 ** -8 * want.abs() + (1 + 2.0 ** -8) * (k * 2.0 ** -23 * mass + 2.0 ** -22 * (z.abs() + want.abs()))
    assert ((y[:m].double() - want).abs() <= tol).all()
    assert (y[m] == 7.0).all()


@pytest.mark.parametrize("m", [4, 40])
def test_linear_of_slices_of_one_buffer(rt, m):
    """x and y as column slices of the same rows; a y that reaches into what is read is refused."""
    from spinn_b200.lib import EINVAL, SpinnCudaError
    buf = torch.randn(m, 64 + 48, device="cuda").half()
    w = torch.randn(48, 64, device="cuda").half()
    want = torch.empty(m, 48, device="cuda").half()
    rt.linear(buf[:, :64].clone(), w, want)
    rt.linear(buf[:, :64], w, buf[:, 64:])
    rt.stream_sync()
    assert torch.equal(buf[:, 64:], want)
    res = torch.randn(m, 96, device="cuda").half()
    for args in ((buf[:, :64], w, buf[:, 56:104]), (w[:m, :48], torch.randn(48, 48, device="cuda").half(), w[:m, :48]),
                 (buf[:, :64], w, res[:, :48], None, res[:, 24:72]), (buf[:, :64], w, res[:, :48], res[0, 47:95])):
        with pytest.raises(SpinnCudaError, match="overlaps|apart") as e:
            rt.linear(*args)
        assert e.value.code == EINVAL


def test_linear_extreme_activations(rt):
    """Large and infinite pre-activations: the activations' limits, no NaN from inf - inf."""
    eye = torch.eye(16, device="cuda", dtype=torch.bfloat16)
    vals = torch.tensor([0.0, -0.0, 1.0, -1.0, 30.0, -30.0, 90.0, -90.0, 3e4, -3e4, 1e30, -1e30, 3e38, -3e38, 1e-30, -5.0],
                        device="cuda", dtype=torch.bfloat16)
    for m in (1, 40):
        x = vals.expand(m, 16).contiguous()
        for act in ("none", "relu", "silu", "gelu", "gelu_tanh"):
            y = torch.empty(m, 16, device="cuda", dtype=torch.bfloat16)
            rt.linear(x, eye, y, act=act)
            rt.stream_sync()
            want = act64(x.double(), act)
            # an infinite cube in 64 bits never occurs; bf16 keeps 8 bits
            tol = 2.0 ** -8 * want.abs() + 2.0 ** -20
            assert ((y.double() - want).abs() <= tol).all(), (act, m, y[0], want[0])


def test_linear_captured_and_replayed(rt):
    x, w = rows((77, 333), torch.float16), rows((200, 333), torch.float16, scale=0.05)  # with copies
    y, y2 = rows((77, 200), torch.float16), rows((77, 200), torch.float16)
    rt.linear(x, w, y, act="silu")
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        rt.linear(x, w, y2, act="silu")
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, y2)
    x.mul_(-1)
    rt.linear(x, w, y, act="silu")
    graph.replay()
    rt.stream_sync()
    assert torch.equal(y, y2)


def test_linear_rows_far_apart(rt):
    """Row strides that carry past 2^31 elements, in y, the residual and x."""
    far = (1 << 30) + 8
    big = torch.zeros(2 * far + 4096, dtype=torch.bfloat16, device="cuda")
    for m in (3, 20):
        step = 2 * far // (m - 1) // 8 * 8
        view = big.as_strided((m, 64), (step, 1))
        x = rows((m, 72), torch.bfloat16)
        w = rows((64, 72), torch.bfloat16, scale=0.1)
        y = torch.empty(m, 64, dtype=torch.bfloat16, device="cuda")
        view.copy_(torch.randn(m, 64, device="cuda"))
        res = view.clone()
        rt.linear(x, w, y, None, res)
        rt.linear(x, w, view, None, view)
        rt.stream_sync()
        assert torch.equal(view, y)
        z = torch.empty(m, 16, dtype=torch.bfloat16, device="cuda")
        rt.linear(view, w[:16, :64], z)                 # x with far rows; w off alignment
        want = y.double() @ w[:16, :64].double().T
        mass = y.double().abs() @ w[:16, :64].double().abs().T
        rt.stream_sync()
        assert ((z.double() - want).abs() <= 2.0 ** -8 * want.abs() + 64 * 2.0 ** -23 * mass).all()


@pytest.mark.parametrize("m", [1, 8, 9, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257])
def test_linear_around_the_tile_sizes(rt, m):
    for k, n in ((128, 128), (136, 256), (1032, 264), (4104, 40), (8, 1032)):
        torch.manual_seed(m + k + n)
        x, w = rows((m, k), torch.float16), rows((n, k), torch.float16, scale=k ** -0.5)
        y, r, b = rows((m, n), torch.float16), rows((m, n), torch.float16), torch.randn(n, device="cuda").half()
        rt.linear(x, w, y, b, r, "silu")
        rt.stream_sync()
        z = x.double() @ w.double().T + b.double()
        mass = x.double().abs() @ w.double().abs().T
        want = act64(z, "silu") + r.double()
        slack = 1.13 * k * 2.0 ** -23 * mass + 2.0 ** -20 * (z.abs() + 1) + 2.0 ** -22 * (z.abs() + want.abs())
        assert ((y.double() - want).abs() <= 2.0 ** -11 * want.abs() + 1.001 * slack + 2.0 ** -25).all(), (m, k, n)
