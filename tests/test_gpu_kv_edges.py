"""Paged attention at its edges."""
import numpy as np
import pytest

import kvutil as K
from tuckmill_amd import hip as H

from q8util import require_gpu, upload_new
from test_gpu_kv import run_decode, run_prefill
from test_gpu_kv_many import many

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = require_gpu()
    yield c
    c.close()


@pytest.mark.parametrize("rows,heads", [(1, 2), (6, 2), (200, 64)])
def test_rows_whose_scores_all_overflow_are_zero_whatever_they_see(ctx, rows, heads):
    """Scores below the range of f32 are -infinity, and where all of a row's are its result is zero,
    though a value that it sees is NaN; among positions shared between workgroups too."""
    rng = np.random.default_rng(61)
    d, n = 64, 3000
    paged = K.Paged(rng, K.F16, 64, heads, d, [n])
    paged.keys[0][:] = -np.abs(paged.keys[0]) - 1
    paged.values[0][10, :, 3] = np.nan
    paged.values[0][1500, :, 5] = np.inf
    for j in range(n):
        paged.put(0, j)
    assert many(rows, 1, heads, heads) == (rows == 200)
    q = np.full((rows, heads * d), 3e37, np.float32)  # (64 products of -3e37 and less, times 0.5)
    attn = H.Attention(0.5)
    got = run_decode(ctx, paged, q, heads, attn) if rows == 1 else run_prefill(ctx, paged, q, heads, attn, np.array([0, rows]))
    assert not np.isnan(got).any() and not got.any()
