"""Heads with an infinity in their projections, on the GPU (the rows of test_paged_host)."""
import numpy as np
import pytest

import paged_oracle as po
import test_paged_gpu as gpu

pytestmark = pytest.mark.gpu
_release = gpu._release  # the fixture


@pytest.mark.parametrize("kind", [gpu.F16, gpu.I8])
@pytest.mark.parametrize("hd", [128, 256, 80])
@pytest.mark.parametrize("rows", [[1, 1, 1], [3, 40, 2]])
def test_heads_with_an_infinity(kind, hd, rows):
    """x / sqrt(mean x^2 + eps) of a head with an infinity: 0, not a number where the infinity and its partner are.
    A page that no row began has no scale: any that is not a number counts as 0."""
    rng = np.random.default_rng(2)
    plan = gpu.Plan(rng, 32, [0, 31, 5], rows)
    pool = gpu.Pool(kind, 2, hd, 32, plan.pages, 3)
    for b in pool.open:
        b.zero()
    was = pool.raw()
    x = rng.normal(0, 1, (plan.total, 2 * 4 * hd + 4 * hd)).astype(np.float32)
    x[:, 3], x[1, 2 * hd + 70], x[:, 8 * hd + 7] = np.inf, -np.inf, np.inf  # of query heads, of a key's
    with np.errstate(invalid="ignore"):
        x, q, _, (qn, kn), cs = gpu.prep(rng, pool, plan, 4, 32, x=x)
        qx, _, kx, vx = gpu.split_heads(x, 4, 2, hd, 1)
        want, k = po.prepared(qx, qn, cs[:, None], gpu.EPS), po.prepared(kx, kn, cs[:, None], gpu.EPS)
    assert np.array_equal(np.isnan(q), np.isnan(want))
    assert (np.abs(q - want) <= 2**-23 * np.abs(want))[~np.isnan(want)].all()
    numbers = lambda raw: raw[:2] + [np.nan_to_num(s) for s in raw[2:4]] + raw[4:]  # noqa: E731
    assert gpu.same(numbers(pool.raw()), gpu.appended(numbers(was), plan, kind, k, vx))
