"""The weights' sum of the attention where positions' values are of any sizes beside each other: zeros and
tiny ones among large ones, single large ones, parts of the cache of one size each. What a position adds to
the sum depends on its score alone. Tolerances are those of test_gpu_draft.py."""
import numpy as np
import pytest
from test_gpu_4bit import new_model, ops, put  # noqa: F401
from test_gpu_draft import check_tree, random_tree, tree_ref

pytestmark = pytest.mark.gpu

SHAPES = [(1, 1, 64, 3000, 5), (4, 1, 128, 700, 8), (2, 2, 32, 1500, 3), (2, 1, 256, 900, 4), (7, 1, 64, 90, 9), (3, 1, 32, 40, 20)]


def check_sizes(ops, rng, H, Hkv, hd, n, S, size, top):
    """size [n + S]: what the positions' values are multiplied by."""
    k, v = rng.standard_normal((2, 1, n + S, Hkv * hd), dtype=np.float32)
    k *= np.float32(0.3)
    v *= size.astype(np.float32)[:, None]
    cap = -(-(n + S) // 32) * 32
    c, m = ops.Kv4Cache(1, Hkv, cap, hd), new_model(1, Hkv, cap, hd)
    c.append(k, v, [0])
    put(m, k[0], v[0], 0, 0, n + S, Hkv)
    q = rng.standard_normal((1, S, H * hd), dtype=np.float32)
    scale = float(np.float32(hd ** -0.5))
    for parent in (None, random_tree(rng, S, "late")[None]):
        out = c.attention_tree(q, [n], None, parent)
        assert np.abs(out).max() <= 5 * top
        check_tree(out, tree_ref(m, q, [n], [S], parent, Hkv, hd, scale))


@pytest.mark.parametrize("times", [2.0 ** 12, 2.0 ** 25, 2.0 ** 40, 2.0 ** 80, 2.0 ** 120])
@pytest.mark.parametrize("H,Hkv,hd,n,S", SHAPES)
@pytest.mark.parametrize("where", [0, 1])
def test_attention_one_large_value(ops, H, Hkv, hd, n, S, times, where):
    """A position at the start, or among the tokens, whose value all queries attend as the others'."""
    rng = np.random.default_rng(n)
    size = np.ones(n + S)
    size[[5, n][where]] = times
    check_sizes(ops, rng, H, Hkv, hd, n, S, size, times)


@pytest.mark.parametrize("top", [2.0 ** 4, 2.0 ** 30, 2.0 ** 60, 2.0 ** 124])
@pytest.mark.parametrize("low", [0.0, 2.0 ** -120, 2.0 ** -60, 1.0])
@pytest.mark.parametrize("H,Hkv,hd,n,S", SHAPES)
@pytest.mark.parametrize("kind", ["scattered", "first", "last", "halves", "blocks"])
def test_attention_values_of_two_sizes(ops, H, Hkv, hd, n, S, top, low, kind):
    rng = np.random.default_rng(n + hd)
    small = {"scattered": rng.random(n + S) < 0.3, "first": np.arange(n + S) < 40, "last": np.arange(n + S) >= n - 3,
             "halves": np.arange(n + S) < n // 2, "blocks": np.arange(n + S) // 32 % 3 == 1}[kind]
    check_sizes(ops, rng, H, Hkv, hd, n, S, np.where(small, low, top), top)


@pytest.mark.parametrize("hd", [64, 256])
def test_attention_values_that_grow(ops, hd):
    """Each block's values 2^6 times those before it, up and down again, in caches of few blocks a wave and of many."""
    rng = np.random.default_rng(hd)
    for n in (1300, 36 * 32 * 4):
        size = 2.0 ** np.clip(np.arange(n + 4) // (n // 40) * 6 - 120, -120, 118)
        for x in (size, size[::-1]):
            check_sizes(ops, rng, 2, 1, hd, n, 4, x, size.max())


@pytest.mark.parametrize("hd,H", [(64, 1), (128, 4), (32, 2), (256, 1)])
def test_attention_unseen_large_values_leave_no_trace(ops, hd, H):
    """Tokens of the largest values, and of none, beside those that a token sees: the same bits."""
    rng = np.random.default_rng(hd)
    S, pos0, cap = 6, 45, 64
    parent = np.array([[-1, 0, 0, 1, 2, 3]], np.int32)
    k, v = rng.standard_normal((2, 1, pos0 + S, hd), dtype=np.float32)
    v[0, 3::7] = 0
    q = rng.standard_normal((1, S, H * hd), dtype=np.float32)
    outs = []
    for other in (1.0, 0.0, 1e30, 3e37):
        vv = v.copy()
        vv[0, pos0 + 2] *= np.float32(other)
        vv[0, pos0 + 4] *= np.float32(other)
        c = ops.Kv4Cache(1, 1, cap, hd)
        c.append(k, vv, [0])
        outs.append(c.attention_tree(q, [pos0], None, parent)[0])
    for out in outs[1:]:
        assert np.array_equal(out[[0, 1, 3, 5]], outs[0][[0, 1, 3, 5]])


@pytest.mark.parametrize("far", [2.0 ** 12, 2.0 ** 24, 2.0 ** 33, 2.0 ** 60])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("size", [1.0, 2.0 ** 67, 2.0 ** -67])
@pytest.mark.parametrize("H,Hkv,hd,n,S", SHAPES)
def test_attention_far_scores_of_some_positions(ops, H, Hkv, hd, n, S, far, sign, size):
    """Scores far above and below the others' among ordinary ones: what a block of far scores adds to the sum stays
    finite. Where one of them is the largest score it takes all of the weight; where they are the lowest they have none."""
    rng = np.random.default_rng(n + S)
    k, v = rng.standard_normal((2, 1, n + S, Hkv * hd), dtype=np.float32)
    k[..., ::hd] = 0
    v *= np.float32(size)
    at = rng.permutation(n + S)[:6]
    at[0] = 7
    k[0, at, ::hd] = (-far if sign < 0 else far) * (1 + np.arange(6, dtype=np.float32)[:, None])
    k[0, at[:, None], np.arange(Hkv * hd) % hd != 0] = 0
    q = rng.standard_normal((1, S, H * hd), dtype=np.float32)
    q[..., ::hd] = 8  # (the far scores are whole numbers: one is larger than the next by far)
    cap = -(-(n + S) // 32) * 32
    c, m = ops.Kv4Cache(1, Hkv, cap, hd), new_model(1, Hkv, cap, hd)
    c.append(k, v, [0])
    put(m, k[0], v[0], 0, 0, n + S, Hkv)
    for parent in (None, random_tree(rng, S, "late")[None]):
        out = c.attention_tree(q, [n], None, parent, scale=0.125)
        ref, tol, live = tree_ref(m, q, [n], [S], parent, Hkv, hd, 0.125)
        # The bound of tree_ref with the largest ds of the ordinary positions in place of each one's, and t at most 100
        # (what lies further off has a weight below 2^-144): a far score's own error decides nothing, since the far
        # ones are whole steps apart from each other and from the rest.
        u = np.float64(2.0 ** -24)
        near = np.setdiff1d(np.arange(n + S), at)
        kmax = np.abs(m["k"][0][:, near]).max()
        ds = (2 * hd + 48) * u * 0.125 * kmax * np.abs(q[0]).reshape(S, H, hd).sum(-1).max()
        bound = (2 * (ds + (96 + n + S + 400) * u)) * np.abs(v).max()
        assert np.isfinite(out).all() and (np.abs(out - ref) <= bound).all(), (np.abs(out - ref) / bound).max()


@pytest.mark.parametrize("far", [2.0 ** 20, 2.0 ** 33, 2.0 ** 60])
@pytest.mark.parametrize("size", [1.0, 2.0 ** 67, 2.0 ** -67])
@pytest.mark.parametrize("H,Hkv,hd,n,S", [(1, 1, 64, 96, 6), (4, 1, 128, 32, 8), (2, 2, 32, 224, 3), (2, 1, 256, 64, 4), (1, 1, 64, 4064, 6)])
def test_attention_tokens_far_below_the_rest(ops, H, Hkv, hd, n, S, far, size):
    """Tokens in a block of their own that see themselves and what comes before: their own scores are far
    below all others, so that they have no weight."""
    rng = np.random.default_rng(n + S)
    k, v = rng.standard_normal((2, 1, n + S, Hkv * hd), dtype=np.float32)
    v[:, n:] *= np.float32(size)
    k[0, :n, ::hd] = 0
    k[0, n:] = 0
    k[0, n:, ::hd] = -far
    q = rng.standard_normal((1, S, H * hd), dtype=np.float32)
    q[..., ::hd] = 8
    cap = n + 32
    c, m = ops.Kv4Cache(1, Hkv, cap, hd), new_model(1, Hkv, cap, hd)
    c.append(k, v, [0])
    put(m, k[0], v[0], 0, 0, n + S, Hkv)
    parent = np.full((1, S), -1, np.int32)
    out = c.attention_tree(q, [n], None, parent, scale=0.125)
    # (nor does the bound take their values in, which could hide a part of the sum)
    m["v"][:, :, n:] = 0
    m["vm"][:, :, n:] = 0
    check_tree(out, tree_ref(m, q, [n], [S], parent, Hkv, hd, 0.125))
