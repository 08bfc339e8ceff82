"""The lookup's gradient for up to 4096 ids over 16-bit rows that are read
eight values at a time: a usual batch of a bf16 table."""
import numpy as np
import pytest

from test_embedding_gpu import _grad_case, _zipf

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("rows,dim,count", [  # count * dim <= 2^20: compared, not sorted
    (1000, 8, 4096), (1000, 64, 4096), (20_000, 128, 4096), (300, 128, 1), (300, 136, 33), (500, 264, 3971),
    (3, 768, 1365), (2000, 768, 1365), (200_000, 64, 2048),
])
def test_grad(rows, dim, count, dtype, accumulate):
    rng = np.random.default_rng(count + dim)
    for idx in (rng.integers(0, rows, count), _zipf(rng, count, rows)):  # the latter with ids of far more than 32 entries
        idx[3::13] = -1
        _grad_case(rows, dim, idx, dtype, dtype, "int64", 1.25, accumulate=accumulate)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("repeats", [31, 32, 33, 64, 129, 1000])
def test_ids_around_a_warps_worth_of_entries(dtype, repeats):
    # four ids of as many entries, spread over the batch, and one id between each two
    idx = np.arange(8 * repeats) % 8
    idx[idx >= 4] = 4 + np.arange((idx >= 4).sum()) % 50
    _grad_case(60, 96, idx, dtype, dtype, "int32", 0.5, pad=8)
    _grad_case(60, 96, idx, dtype, dtype, "int32", 0.5, accumulate=True)
