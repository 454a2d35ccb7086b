"""The first token is always kept, wherever its logit falls among the bins of 1/64: top_p of 0 (and below) is
the argmax. Logits on a grid of quarters, as integers' quotients have them, fall next to a bin's border."""
import numpy as np
import pytest
from test_gpu_4bit import ops  # noqa: F401
from test_gpu_draft import sample_ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", [1.5, 0.3, 0.7, 1.0, 1e4, 3e38])
@pytest.mark.parametrize("rows,vocab", [(200, 50), (200, 20000), (6, 40000)])
@pytest.mark.parametrize("k,m", [(0, 0.0), (3000, 0.0), (0, 0.05)])
def test_sample_top_p_of_nothing(ops, rows, vocab, t, k, m):
    rng = np.random.default_rng(vocab)
    x = (np.round(rng.standard_normal((rows, vocab)) * 40) / 4).astype(np.float32)
    x -= rng.integers(0, 400, (rows, 1)).astype(np.float32) / 4
    x[0] = -1 - np.abs(x[0])
    x[0, 7] = 1e-12  # a positive one below all steps of the bins
    x[1, :] = -83.25
    x[2, 3:] = -83.5
    u = rng.random(rows, dtype=np.float32)
    for p in (0.0, -1.0):
        token, prob = ops.sample(x, u, np.float32(t), k, p, m)
        assert np.array_equal(token, x.argmax(1)) and (prob == 1).all()


def test_sample_next_to_a_bins_border(ops):
    """-83.25 x 64 / 1.5 is 3552 less 2e-13 in 64 bits."""
    rng = np.random.default_rng(7)
    for vocab in (9, 60000):
        x = np.full((40, vocab), -90.0, np.float32)
        x[:, 1:9] = -83.25 - np.arange(8)
        u = rng.random(40, dtype=np.float32)
        for k, p, m in ((0, 1.0, 0.0), (1, 1.0, 0.0), (0, 1e-30, 0.0), (2, 0.0, 0.0), (0, 1.0, 1.0), (5, 0.7, 0.3)):
            token, prob = ops.sample(x, u, 1.5, k, p, m)
            for r in range(40):
                want, share, near = sample_ref(x[r], u[r], 1.5, k, p, m)
                assert near < 1e-8 or (token[r] == want and abs(prob[r] - share) <= 2.0 ** -20)


@pytest.mark.parametrize("t", [1.0, 1e4, 1e10, 3e38])
@pytest.mark.parametrize("rows,vocab", [(3, 100), (300, 5000), (3, 40000)])
def test_sample_min_p_of_one(ops, rows, vocab, t):
    """The largest logit and its equals, and none of a lesser one, were it a step of f32 below and the weights
    alike in 64 bits."""
    rng = np.random.default_rng(vocab)
    x = (rng.standard_normal((rows, vocab)) * 3).astype(np.float32)
    for r in range(rows):
        top = x[r].max() + np.float32(1)
        at = rng.permutation(vocab)[:80]
        x[r, at[:3]] = top
        for i, j in enumerate(at[3:]):
            x[r, j] = top - (i + 1) * np.spacing(top)
    u = rng.random(rows, dtype=np.float32)
    token, prob = ops.sample(x, u, np.float32(t), min_p=1.0)
    for r in range(rows):
        equal = np.flatnonzero(x[r] == x[r].max())
        assert token[r] == equal[int(float(u[r]) * 3)] and abs(prob[r] * 3 - 1) <= 2.0 ** -20
