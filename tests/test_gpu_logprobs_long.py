"""Log probabilities of many rows of the longest vocabularies, where one thread has thousands of values.

Tolerance: that of test_gpu_logprobs.py, whose count of additions in a row (256) is above what the kernel has for any length: 24 of a batch, 171
batches, five of a warp. Rows are one value behind their first HIGH tokens, which give every thread a larger one: the sums are known in closed
form, and as what is added is always the same, a sum of one addition after the other rounds to the same side all along."""
import numpy as np
import pytest
import torch

from tests.gpu_util import empty, host, runtime
from tests.test_gpu_logprobs import ABS, REL

pytestmark = pytest.mark.gpu
HIGH = 1100


@pytest.mark.parametrize("vocab", [1048576, 1048573, 300001])
@pytest.mark.parametrize("top", [0, 3])
def test_many_rows_of_a_long_vocabulary(vocab, top):
    rows = 320  # more than two for each SM: one CTA per row
    low = torch.linspace(-0.7, -0.05, rows, device="cuda")
    logits = low[:, None].expand(rows, vocab).contiguous()
    logits[:, :HIGH] = 0.0
    targets = torch.arange(rows, device="cuda", dtype=torch.int32) * 11 + 7
    lp, entropy, tokens, alternatives = empty(rows), empty(rows), empty((rows, top), torch.int32), empty((rows, top))
    runtime().logprobs_into(logits, rows, vocab, targets, lp, entropy, top, tokens, alternatives)
    x = low.double().cpu().numpy()
    ln_s = np.log(HIGH + (vocab - HIGH) * np.exp(x))
    want = np.where(targets.cpu().numpy() < HIGH, 0.0, x) - ln_s
    np.testing.assert_allclose(host(lp), want, rtol=REL, atol=ABS)
    mean = x * (vocab - HIGH) * np.exp(x - ln_s)
    np.testing.assert_allclose(host(entropy), ln_s - mean, rtol=REL, atol=ABS + 2 * ABS * np.abs(ln_s - mean).max())
    if top:
        np.testing.assert_array_equal(host(tokens), np.broadcast_to([0, 1, 2], (rows, 3)))
        np.testing.assert_allclose(host(alternatives), np.stack([-ln_s] * 3, 1), rtol=REL, atol=ABS)
