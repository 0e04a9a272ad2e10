"""Log probabilities of logits whose differences pass fp32's range, on the GPU (the rows of test_paged_host)."""
import numpy as np
import pytest

import test_paged_gpu as gpu
import test_paged_host as host

pytestmark = pytest.mark.gpu
_release = gpu._release  # the fixture


@pytest.mark.parametrize("vocab", [33, 1100, 8200, 20011, 70000])
@pytest.mark.parametrize("inv_t", [1e-38, 3e-39, 2e-38, 1e-30, 0.4])
def test_logprobs_of_logits_far_apart(vocab, inv_t):
    x, tokens = host.far_rows(vocab)
    for ld in (vocab + 3, (vocab + 3) // 4 * 4):
        gpu.check_logprobs(gpu.run_logprobs(x, tokens, np.float32(inv_t), 7, False, ld), x, tokens, inv_t, 7)
