"""Rows' attention where queries, scales and caps lie near the ends of fp32's
range, and over values and keys that are not finite."""
import numpy as np
import pytest

import sheep_amd as sa
from test_gpu_rows import rows_case

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device():
    sa.init(0)


# ------------------------------------------------------------ small and large factors

@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads, kv, hd", [(8, 2, 128), (4, 1, 64)])
@pytest.mark.parametrize("mask", ["causal", "tree"])
@pytest.mark.parametrize("q_exp, scale", [(-140, 0.0), (-147, 0.0), (-120, 1e-5), (-20, 2.0 ** -130), (0, 2.0 ** -149), (-60, -2.0 ** -100)])
def test_scores_near_nothing(dtype, heads, kv, hd, mask, q_exp, scale):
    """Scores of some 2^-137 and less, beside masked ones and absent pages: a row is
    the mean of what it attends to, in the general bounds."""
    rows_case([40, 3, 9], [150, 3, 700], heads, kv, hd, dtype, 16, seed=hd, mask=mask, q_exp=q_exp, scale=scale, gone={2: [1, 20]})
