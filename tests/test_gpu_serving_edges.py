"""The operators of a step of many requests at the edges of what their header
allows, against the 64-bit forms of serving_oracle.py."""
import numpy as np
import pytest

import serving_oracle as so
import sheep_amd as sa
from sheep_amd import serving

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device():
    sa.init(0)


def ints(x):
    return sa.DevBuf.of(np.array(x, np.int32))


def within(got, want, tol, what=""):
    off = int((~(np.abs(got.astype(np.float64) - want) <= tol)).sum())
    assert off == 0, f"{what}: {off} of {got.size} off"


# ------------------------------------------------------------ adapters

def lora(n, n_in, n_out, rank, A, dtype, ids, x, base=None, in_place=False, a=None, b=None, y_pad=0):
    rng = np.random.default_rng(5)
    if a is None:
        a, b = (so.to_bits(rng.standard_normal(s), dtype) for s in ((A, rank, n_in), (A, n_out, rank)))
    bb = sa.DevBuf.of(base) if base is not None else None
    y = bb if in_place else sa.DevBuf.of(np.full((n, n_out + y_pad), 9.0, np.float32))
    work = sa.DevBuf.of(np.full(serving.lora_work_floats(rank, n), np.nan, np.float32))
    ad = serving.Adapters(sa.DevBuf.of(a), sa.DevBuf.of(b), A, rank, n_in, n_out, dtype)
    serving.lora(ad, sa.DevBuf.of(x), n, ints(ids), y, work, base=bb, y_stride=n_out + y_pad)
    return y.read(np.float32).reshape(n, n_out + y_pad), a, b


FORMS = [(8, 256, 70, 16, 4), (16, 520, 301, 64, 16), (20, 256, 70, 16, 3), (100, 256, 70, 16, 9), (130, 1032, 66, 64, 3),
         (300, 264, 131, 256, 4), (600, 264, 67, 24, 5)]


@pytest.mark.parametrize("n, n_in, n_out, rank, A", FORMS)
def test_bf16_adapters_of_the_largest_inputs(n, n_in, n_out, rank, A):
    """The largest finite inputs, and the same as the first product's results,
    with a second matrix that brings them down."""
    rng = np.random.default_rng(n)
    x = np.zeros((n, n_in), np.float32)
    x[np.arange(n), rng.integers(0, n_in, n)] = rng.choice([3.4028234e38, -3.4028234e38, 3.395e38, 2.0 ** 127], n)
    a = so.to_bits(rng.choice([-1, 1, 2.0 ** -20], (A, rank, n_in)), "bf16")
    b = so.to_bits(rng.choice([-1, 1], (A, n_out, rank)) * rng.uniform(0.5, 1, (A, n_out, rank)) * 2.0 ** -118, "bf16")
    ids = rng.integers(-1, A, n)
    got, _, _ = lora(n, n_in, n_out, rank, A, "bf16", ids, x, a=a, b=b)
    want, tol = so.lora(x, np.zeros((n, n_out)), so.from_bits(a, "bf16"), so.from_bits(b, "bf16"), np.ones(A, np.float32),
                        [rank] * A, ids)
    within(got, want, tol)
