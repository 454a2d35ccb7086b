"""Rows of logits whose parts are of very different size, as masks of finite lowest values leave
them: the token and its share are those of the definition, and the same whether a row is drawn by
one workgroup among many rows or alone, cut into slices.

A workgroup reads a row in parts of 16384 tokens and follows the largest logit from part to part.
Tolerances are those of test_gpu_draft.py."""
import numpy as np
import pytest
from test_gpu_4bit import ops  # noqa: F401
from test_gpu_draft import SETTINGS, sample_ref

pytestmark = pytest.mark.gpu

PART = 16384
LOWEST = np.finfo(np.float32).min


def masked_rows(rng, vocab):
    """One row a layout; the likely tokens stand behind the first part."""
    def ordinary(n, top):
        x = np.float32(top) - np.abs(rng.standard_normal(n) * 3).astype(np.float32) - np.float32(0.1)
        x[rng.integers(0, n)] = top
        return x

    def after(top, *before):
        """Parts of one value each (those that leave no room for others are dropped), then ordinary logits."""
        head = [np.full(PART, v, np.float32) for v in before[:(vocab - 1) // PART]]
        return np.concatenate(head + [ordinary(vocab - PART * len(head), top)])
    rows = [after(5.0, LOWEST), after(0.0, -1e30), after(-3.0, LOWEST), after(0.0, -1e30, LOWEST),
            after(5.0, -np.inf, LOWEST), after(-3.0, LOWEST, -np.inf),
            # next to where the largest logit counts as far away (2^49 bins of T / 64), on both sides
            after(2.0, -1.2 * 2.0 ** 43, -0.9 * 2.0 ** 43), after(-1e30, LOWEST), after(-1e13, LOWEST, -1e30)]
    few = np.full(vocab, LOWEST, np.float32)
    few[vocab - 2000:vocab - 1995] = 2.0, 2.1, 2.2, 1.9, 2.15
    equal = np.full(vocab, -1e30, np.float32)
    equal[PART + 100:PART + 2900] = 0.0  # more than are sorted at once
    only = np.full(vocab, LOWEST, np.float32)
    only[-1] = 0.0
    scattered = after(5.0, LOWEST)
    scattered[PART + 1::3] = -1e30
    return np.stack(rows + [few, equal, only, scattered])


def same(a, b):
    return np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])


@pytest.mark.parametrize("t,k,p,m", SETTINGS)
@pytest.mark.parametrize("vocab,times", [(20000, 1), (50000, 7), (122753, 3)])
def test_sample_after_masked_parts(ops, vocab, times, t, k, p, m):
    rng = np.random.default_rng(vocab)
    x = masked_rows(rng, vocab)
    n = len(x)
    u = rng.random(n, dtype=np.float32)
    token, prob = (a.reshape(times, n) for a in ops.sample(np.tile(x, (times, 1)), np.tile(u, times), t, k, p, m))
    assert (token == token[0]).all() and (prob == prob[0]).all()
    for r in range(n):
        assert same(ops.sample(x[r:r + 1], u[r:r + 1], t, k, p, m), (token[0, r:r + 1], prob[0, r:r + 1])), r
        want, share, near = sample_ref(x[r], u[r], t, k, p, m)
        if near > 1e-8:
            assert token[0, r] == want, (r, token[0, r], want, near)
            assert abs(prob[0, r] - share) <= 2.0 ** -20 * max(share, 2.0 ** -40), (r, prob[0, r], share)
