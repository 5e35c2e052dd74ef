"""Paged attention over every instantiated tile: head sizes, groups, ways of copying and of splitting the work,
with and without accumulated weights."""
import pytest

from test_gpu_cache import _attention_case, _check_attention, rt  # noqa: F401

pytestmark = pytest.mark.gpu

# head sizes of each tile, exact and ragged; groups of each block of heads; pages whose rows come by TMA boxes
# (16-byte rows, whole groups of them), by copies of the lanes, and element by element
DIMS = {"fp16": [64, 40, 128, 72, 192, 136, 256, 200], "bf16": [64, 56, 128, 120, 192, 184, 256, 248],
        "fp32": [64, 36, 96, 68, 128, 100, 256, 132]}
GROUPS = {"fp16": [1, 8, 11, 16], "bf16": [3, 7, 9, 16], "fp32": [1, 3, 4, 8]}
LAYOUTS = [(16, "nhd"), (64, "hnd"), (16, "pair"), (5, "nhd"), (16, "odd"), (7, "odd")]
LENGTHS = {"whole": [133, 0, 1, 256], "segments": [1999, 61], "workers": [430, 300, 0, 517, 290, 1, 611, 64, 333]}


@pytest.mark.parametrize("split", list(LENGTHS))
@pytest.mark.parametrize("page,layout", LAYOUTS)
@pytest.mark.parametrize("dtype", list(DIMS))
def test_every_tile(rt, dtype, page, layout, split):  # noqa: F811
    for i, dim in enumerate(DIMS[dtype]):
        for j, group in enumerate(GROUPS[dtype]):
            heads = 1 if split == "segments" else 2 + (i + j) % 2
            case = (dtype, LENGTHS[split], group * heads, heads, dim, page, layout, (i + j + page) % 2 == 0)
            _check_attention(case, *_attention_case(rt, case, seed=i * 10 + j))
