"""Rows of 8-bit pages that are not held, on the GPU: codes and scales of the others are those of the definition, whatever the
open pages and the pages held before."""
import numpy as np
import pytest

import test_paged_gpu as gpu
import test_paged_host as host

pytestmark = pytest.mark.gpu
_release = gpu._release  # the fixture


@pytest.mark.parametrize("stale,old", [(6e4, 0.5), (np.inf, 30), (np.nan, 0.5)])
@pytest.mark.parametrize("hd", [128, 256, 80])
@pytest.mark.parametrize("past,sizes,bad", host.HOLES, ids=[f"{p}_{'_'.join(map(str, s))}_{len(b)}" for p, s, b in host.HOLES])
def test_rows_that_are_not_held_do_not_count(past, sizes, bad, hd, stale, old):
    rng = np.random.default_rng(len(bad) + past)
    whole = gpu.Plan(rng, 32, [past], [sum(sizes)])
    pool = gpu.Pool(gpu.I8, 2, hd, 32, whole.pages, 1, *(rng.normal(0, old, (2, whole.pages, 2, 32, hd)).astype(np.float16)))
    for b in pool.open:
        b.upload(np.full((2, 32, hd), stale, np.float16))
    was = pool.raw()
    host.check_holes(pool, was, whole, host.steps_with_holes(None, rng, pool, whole, sizes, bad, on=gpu), bad)
