"""Where the operators of a step with drafted tokens can go wrong: values, keys and queries of
unlike size, scores at the ends of f32, batches of unlike lengths, calls at once on streams
and in graphs, temperatures and vocabularies at their ends.

Tolerances are those of test_gpu_draft.py. Where scores are exact in every step (`exact`) their
error ds is left out: what remains are the exponent's and the sums' roundings."""
import ctypes as C

import numpy as np
import pytest
from test_gpu_4bit import U, dev, device_cache, filled, new_model, ops, put  # noqa: F401
from test_gpu_draft import check_sample, check_tree, random_tree, sample_ref, sees, spread, tree_ref

from sparrow_amd import VmlmError

pytestmark = pytest.mark.gpu


def stored(ops, k, v, Hkv, cap):
    B, n, hd = k.shape[0], k.shape[1], k.shape[2] // Hkv
    c, m = ops.Kv4Cache(B, Hkv, cap, hd), new_model(B, Hkv, cap, hd)
    c.append(k, v, np.zeros(B))
    for b in range(B):
        put(m, k[b], v[b], b, 0, n, Hkv)
    return c, m


def exact_ref(m, q, pos0, parent, Hkv, hd, scale):
    """tree_ref of whole sequences where the scores are exact."""
    B, S, H = q.shape[0], q.shape[1], q.shape[2] // hd
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    for b in range(B):
        lo, sc = spread(m["vm"][b])
        most = np.maximum(np.abs(lo), np.abs(lo + 15 * sc))
        for t in range(S):
            see = sees(None if parent is None else parent[b], pos0[b], S, t)
            for h in range(H):
                kv, at = h // (H // Hkv), slice(h * hd, (h + 1) * hd)
                s = m["k"][b, kv, see].astype(np.float64) @ q[b, t, at].astype(np.float64) * scale
                d = s.max() - s
                p = np.exp(-d)
                p /= p.sum()
                e = (96 + len(see) + 4 * d) * U
                out[b, t, at] = p @ m["v"][b, kv, see].astype(np.float64)
                tol[b, t, at] = np.repeat(((p * (e + p @ e))[:, None] * most[kv, see]).sum(0), 32) + 2.0 ** -130
    return out, tol, np.ones((B, S), bool)


# ------------------------------------------------------------------ attention
SHAPES = [(1, 1, 64, 200, 5), (4, 1, 128, 130, 8), (2, 2, 32, 100, 3), (2, 1, 256, 90, 4), (7, 1, 64, 60, 9),
          (1, 1, 64, 300, 40), (2, 2, 128, 1500, 2), (1, 1, 32, 700, 64)]


def case(rng, H, Hkv, hd, n, S):
    """(q, k, v, parent, pos0) of a tree at the end of n positions."""
    k, v = rng.standard_normal((2, 1, n, Hkv, hd), dtype=np.float32)
    q = rng.standard_normal((1, S, H, hd), dtype=np.float32)
    return q, k, v, random_tree(rng, S)[None], n - S


def run(ops, q, k, v, parent, pos0, scale=None):
    n, Hkv, hd = k.shape[1:]
    c, m = stored(ops, k.reshape(1, n, -1), v.reshape(1, n, -1), Hkv, -(-n // 32) * 32)
    q = q.reshape(1, q.shape[1], -1)
    scale = float(np.float32(hd ** -0.5)) if scale is None else scale
    out = c.attention_tree(q, [pos0], None, parent, scale=scale)
    return out, m, q, scale


@pytest.mark.parametrize("times", [1e3, 1e10, 1e20, 1e32, 1e36])
@pytest.mark.parametrize("H,Hkv,hd,n,S", SHAPES)
@pytest.mark.parametrize("where", [0, 1])
def test_attention_value_that_no_query_attends(ops, H, Hkv, hd, n, S, times, where):
    """A value that stands out at a position whose weight is nothing (e^-100 and less), in the
    first block and in the middle: the others keep all their bits."""
    rng = np.random.default_rng(n + hd)
    q, k, v, parent, pos0 = case(rng, H, Hkv, hd, n, S)
    base = rng.standard_normal((Hkv, hd))
    q = (base[None, None, np.arange(H) // (H // Hkv)] + 0.1 * q).astype(np.float32)
    scale = float(np.float32(hd ** -0.5))
    at = where * (pos0 // 2)
    k[0, at] = -(100 + np.log(times)) / scale * base / (base * base).sum(-1, keepdims=True) * 1.3
    v[0, at] *= np.float32(times)
    out, m, q, scale = run(ops, q, k, v, parent, pos0)
    check_tree(out, tree_ref(m, q, [pos0], [S], parent, Hkv, hd, scale))


@pytest.mark.parametrize("times", [1e-30, 1e-3, 1e3, 1e30])
@pytest.mark.parametrize("H,Hkv,hd,n,S", SHAPES)
def test_attention_values_of_other_magnitudes(ops, H, Hkv, hd, n, S, times):
    """Every other block's values, and every fourth block's keys, of another size; among a
    position's values one group a thousandth of the others."""
    rng = np.random.default_rng(n + hd + 1)
    q, k, v, parent, pos0 = case(rng, H, Hkv, hd, n, S)
    block = np.arange(n) // 32
    v[0, block % 2 == 1] *= np.float32(times)
    v[..., :32] *= np.float32(1e-3)
    k[0, block % 4 == 2] *= np.float32(1e-3)
    out, m, q, scale = run(ops, q, k, v, parent, pos0)
    check_tree(out, tree_ref(m, q, [pos0], [S], parent, Hkv, hd, scale))


@pytest.mark.parametrize("small", [0.0, 1e-30, 1e-6])
@pytest.mark.parametrize("H,Hkv,hd,n,S", SHAPES)
@pytest.mark.parametrize("where", [0, 1, 2])
def test_attention_weight_on_no_value(ops, H, Hkv, hd, n, S, small, where):
    """A position with nearly all the weight (e^60 times the others') whose values are 0, or next to it: what the
    others' weights bring keeps its bits."""
    rng = np.random.default_rng(n + hd + where)
    q, k, v, parent, pos0 = case(rng, H, Hkv, hd, n, S)
    base = rng.standard_normal((Hkv, hd))
    q = (base[None, None, np.arange(H) // (H // Hkv)] + 0.01 * q).astype(np.float32)
    scale = float(np.float32(hd ** -0.5))
    at = [0, pos0 // 2, pos0][where]
    k[0, at] = 60 / scale * base / (base * base).sum(-1, keepdims=True)
    v[0, at] *= np.float32(small)
    out, m, q, scale = run(ops, q, k, v, parent, pos0)
    check_tree(out, tree_ref(m, q, [pos0], [S], parent, Hkv, hd, scale))


@pytest.mark.parametrize("times", [1e4, 1e6, 1e12])
@pytest.mark.parametrize("H,Hkv,hd,n,S", [s for s in SHAPES if s[2] > 32])
def test_attention_query_groups_of_other_magnitudes(ops, H, Hkv, hd, n, S, times):
    """Queries whose first 32 channels are large against keys that are small there (and
    the other way round in the last 32): each group's products keep their bits."""
    rng = np.random.default_rng(hd + H)
    q, k, v, parent, pos0 = case(rng, H, Hkv, hd, n, S)
    q[..., :32] *= np.float32(times)
    k[..., :32] /= np.float32(times)
    q[..., -32:] /= np.float32(times)
    k[..., -32:] *= np.float32(times)
    out, m, q, scale = run(ops, q, k, v, parent, pos0)
    check_tree(out, tree_ref(m, q, [pos0], [S], parent, Hkv, hd, scale))


@pytest.mark.parametrize("times", [1e-37, 1e-20, 1e20, 1e36])
def test_attention_tiny_and_huge_queries(ops, times):
    """Queries and keys at opposite ends of f32, with a group of zeros and a zero token."""
    rng = np.random.default_rng(21)
    q, k, v, parent, pos0 = case(rng, 3, 1, 128, 170, 7)
    q *= np.float32(times)
    q[..., 32:64] = 0
    q[:, 2] = 0
    k /= np.float32(times)
    out, m, q, scale = run(ops, q, k, v, parent, pos0, 0.125)
    check_tree(out, tree_ref(m, q, [pos0], [7], parent, 1, 128, scale))


def test_attention_queries_of_unlike_size(ops):
    """Tokens of one tile from 1e-20 to 1e20 against the same keys: small ones see a mean, large ones
    one position, each to its own bits."""
    rng = np.random.default_rng(20)
    q, k, v, parent, pos0 = case(rng, 1, 1, 64, 250, 12)
    q *= np.float32(10.0) ** rng.integers(-20, 3, 12).astype(np.float32)[None, :, None, None]
    out, m, q, scale = run(ops, q, k, v, parent, pos0)
    check_tree(out, tree_ref(m, q, [pos0], [12], parent, 1, 64, scale))


@pytest.mark.parametrize("q,k,scale", [(2.0 ** -138, 2.0 ** 127, 2.0 ** 20), (2.0 ** -122, 2.0 ** 122, -200.0),
                                       (2.0 ** 100, 2.0 ** -60, 2.0 ** -45), (1.0, 1.0, 0.0)])
def test_attention_any_scale_of_the_scores(ops, q, k, scale):
    """Scales that bring scores of a few out of queries and keys near f32's ends: no
    step between leaves f32."""
    rng = np.random.default_rng(22)
    x, y, v, parent, pos0 = case(rng, 2, 1, 64, 170, 6)
    x = (x.astype(np.float64) * q / 8).astype(np.float32)
    y = (y.astype(np.float64) * k / 64).astype(np.float32)
    out, m, x, scale = run(ops, x, y, v, parent, pos0, scale)
    check_tree(out, tree_ref(m, x, [pos0], [6], parent, 1, 64, scale))


@pytest.mark.parametrize("H,Hkv,hd,n,S", SHAPES)
def test_attention_scores_of_minus_infinity(ops, H, Hkv, hd, n, S):
    """Finite queries and keys whose product leaves f32 downwards at the first 40
    positions: those have no weight, as in f32."""
    rng = np.random.default_rng(n)
    q, k, v, parent, pos0 = case(rng, H, Hkv, hd, n, S)
    q[..., 0] = 1e30
    k[..., :32] = 0
    k[0, :40, :, 0] = -1e30
    out, m, q, scale = run(ops, q, k, v, parent, pos0)
    part = {x: y[:, :, 40:] for x, y in m.items()}
    q.reshape(1, S, H, hd)[..., 0] = 0
    check_tree(out, tree_ref(part, q, [pos0 - 40], [S], parent, Hkv, hd, scale))


@pytest.mark.parametrize("H,Hkv,hd,n,S", SHAPES + [(1, 1, 64, 3000, 63)])
@pytest.mark.parametrize("far", [8192, 2 ** 20])
def test_attention_scores_far_from_zero(ops, H, Hkv, hd, n, S, far):
    """Scores of 15360 (and of two million) and a few more, exact in f32: the weights depend on their
    differences, so that log2(e) must not round the scores themselves."""
    rng = np.random.default_rng(n)
    q, k, v, parent, pos0 = case(rng, H, Hkv, hd, n, S)
    q[:], k[:] = 0, 0
    q[..., 0], q[..., 1] = far, 8
    k[..., 0] = 15
    k[..., 1] = rng.integers(0, 6, k.shape[:-1])
    out, m, q, scale = run(ops, q, k, v, parent, pos0, 0.125)
    assert np.array_equal(m["k"][0, :, :n], k[0].transpose(1, 0, 2))
    check_tree(out, exact_ref(m, q, [pos0], parent, Hkv, hd, scale))


@pytest.mark.parametrize("far", [2 ** 24, 2 ** 27, 2 ** 40, 2 ** 90])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("H,Hkv,hd,n,S", SHAPES)
def test_attention_scores_beyond_f32s_steps(ops, H, Hkv, hd, n, S, far, sign):
    """Scores so large that a step of f32 is more than a weight's exponent: 2^28 and more, whose steps are 32
    and more, so that what the largest ones' weights are to each other is within a rounding of the
    score. They are 2^21 and more from the others', which have none: the output lies between the least
    and the largest of the values at those positions, off by the sums' roundings."""
    rng = np.random.default_rng(n)
    q, k, v, parent, pos0 = case(rng, H, Hkv, hd, n, S)
    q[:], k[:] = 0, 0
    q[..., 0], q[..., 1] = np.float32(far) * sign, np.float32(far) / 8
    k[..., 0] = 15
    k[..., 1] = rng.integers(0, 6, k.shape[:-1])
    out, m, q, scale = run(ops, q, k, v, parent, pos0, 1.0)
    assert np.array_equal(m["k"][0, :, :n], k[0].transpose(1, 0, 2))
    out = out.reshape(S, Hkv, H // Hkv, hd)
    for t in range(S):
        see = sees(parent[0], pos0, S, t)
        for kv in range(Hkv):
            score = k[0, see, kv, 1]
            top = see[score == score.max()]
            x = m["v"][0, kv, top]
            tol = (96 + n) * U * np.abs(m["v"][0, kv, see]).max()
            assert (out[t, kv] >= x.min(0) - tol).all() and (out[t, kv] <= x.max(0) + tol).all()


@pytest.mark.parametrize("H,Hkv,hd", [(1, 1, 32), (1, 1, 64), (4, 1, 128), (3, 1, 256), (2, 1, 64)])
def test_attention_every_bit_of_the_weights(ops, H, Hkv, hd):
    """One position has nearly all the weight, and half of its channels hold an exact zero
    (u = 8, min = -8 scale): there the output is the sum of weights near 2^-15 of the largest.
    Those are off by e of themselves and half a step of their lower term, 2^-25 of the 2^9 at which the
    largest stands at least: 2^-34 of it, each times a code up to 8."""
    rng = np.random.default_rng(hd)
    n, S = 60, 3
    q = np.zeros((1, S, H, hd), np.float32)
    q[..., 0] = 8
    k = np.zeros((1, n, 1, hd), np.float32)
    k[0, 1:, 0, 0] = -rng.uniform(9, 12, n - 1)
    v = rng.integers(-8, 8, (1, n, 1, hd)).astype(np.float32)
    v[..., 0::32], v[..., 1::32] = -8, 7
    zero = np.arange(hd) % 2 == 0
    v[0, 0, 0, zero & (np.arange(hd) % 32 > 1)] = 0
    parent = np.array([[-1, 0, 0]], np.int32)
    out, m, q, scale = run(ops, q, k, v, parent, n - S, 0.125)
    assert np.array_equal(m["v"][0, 0, :n], v[0, :, 0])
    ref = tree_ref(m, q, [n - S], [S], parent, Hkv, hd, scale)
    check_tree(out, ref)
    see = v[0, 0, 0] == 0
    for t in range(S):
        s = m["k"][0, 0, sees(parent[0], n - S, S, t), 0].astype(np.float64)
        p = np.exp(s - s.max())
        p /= p.sum()
        e = (96 + n + 4 * 13 + (2 * hd + 48) * 13) * U  # (a score is above -13)
        bound = (2 * e * p[1:].sum() + (n - 1) * 2.0 ** -34) * 8
        d = np.abs(out - ref[0]).reshape(1, S, H, hd)[0, t][:, see]
        assert see.any() and d.max() <= bound


@pytest.mark.parametrize("n", [129, 300, 1025, 1200])
@pytest.mark.parametrize("H,Hkv,hd", [(1, 1, 64), (4, 1, 128), (2, 2, 32), (1, 1, 256)])
def test_attention_nan_keys_fill_blocks(ops, H, Hkv, hd, n):
    """Poisoned keys at every position of the last blocks, or of the first: all that see them are
    NaN, also where a wave has nothing else."""
    rng = np.random.default_rng(n)
    for bad in (slice((n - 4) // 128 * 128, n - 3), slice(0, 128), slice(32, 64)):
        q, k, v, parent, pos0 = case(rng, H, Hkv, hd, n, 3)
        k[0, bad, :, 3] = np.nan
        c = ops.Kv4Cache(1, Hkv, -(-n // 32) * 32, hd)
        c.append(k.reshape(1, n, -1), v.reshape(1, n, -1), [0])
        assert np.isnan(c.attention_tree(q.reshape(1, 3, -1), [pos0], None, parent)).all()


@pytest.mark.parametrize("kind", ["tree", "chain"])
@pytest.mark.parametrize("B,H,Hkv,hd,cap", [(1, 1, 1, 64, 4096), (70, 1, 1, 64, 1184), (130, 2, 1, 32, 1056),
                                            (5, 4, 2, 128, 4160), (3, 1, 1, 256, 2080)])
def test_attention_of_unlike_lengths(ops, B, H, Hkv, hd, cap, kind):
    """One long sequence among short, idle and empty ones, also more sequences than a wave has lanes:
    each gets its own shares of the positions."""
    rng = np.random.default_rng(B + hd)
    S = 3
    for long in {0, B // 2, B - 1}:
        pos0 = rng.choice([-1, 0, 1, 29, 31, 64, 100], B).astype(np.int32)
        count = rng.integers(-1, S + 2, B).astype(np.int32)
        pos0[long], count[long] = cap - S, S + 5
        n = np.clip(count, 0, S)
        c, m = filled(ops, rng, B, Hkv, cap, hd, np.where(pos0 >= 0, pos0 + n, 0))
        parent = np.stack([random_tree(rng, S) for _ in range(B)]) if kind == "tree" else None
        q = rng.standard_normal((B, S, H * hd), dtype=np.float32)
        out = c.attention_tree(q, pos0, count, parent)
        check_tree(out, tree_ref(m, q, pos0, n, parent, Hkv, hd, float(np.float32(hd ** -0.5))))
    for idle in (dict(pos0=[-1] * B, count=None), dict(pos0=[5] * B, count=[0] * B), dict(pos0=[5] * B, count=[-7] * B)):
        assert not c.attention_tree(q, idle["pos0"], idle["count"], parent).any()


def test_attention_long_among_many(ops):
    """More (sequence, kv head) pairs than the card takes workgroups at once, one sequence long."""
    rng = np.random.default_rng(77)
    B, H, hd, cap, S, n = 17, 32, 32, 8192, 2, 8100
    c = ops.Kv4Cache(B, H, cap, hd)
    one, few = new_model(1, H, cap, hd), new_model(B, H, 64, hd)
    at = 0
    while at < n:
        rows = min(600, n - at)
        k, v = np.zeros((2, B, rows, H * hd), np.float32)
        k[3], v[3] = rng.standard_normal((2, rows, H * hd), dtype=np.float32)
        pos = np.full(B, -1)
        pos[3] = at
        c.append(k, v, pos)
        put(one, k[3], v[3], 0, at, rows, H)
        at += rows
    k, v = rng.standard_normal((2, B, 40, H * hd), dtype=np.float32)
    pos = np.zeros(B, int)
    pos[3] = -1
    c.append(k, v, pos)
    for b in range(B):
        put(few, k[b], v[b], b, 0, 40, H)
    q = rng.standard_normal((B, S, H * hd), dtype=np.float32)
    pos0 = np.full(B, 38, np.int32)
    pos0[3], pos0[9] = n - S, -1
    out = c.attention_tree(q, pos0)
    scale = float(np.float32(hd ** -0.5))
    check_tree(out[3:4], tree_ref(one, q[3:4], [n - S], [S], None, H, hd, scale))
    pos0[3], out[3] = -1, 0
    check_tree(out, tree_ref(few, q, pos0, [S] * B, None, H, hd, scale))


@pytest.mark.parametrize("B", [1, 3])
def test_attention_shares_refused_on_the_device(ops, B):
    """Sequences whose positions are dealt out: tokens past the capacity and parents that are no earlier
    token trip the guard, the others are right."""
    rng = np.random.default_rng(78)
    cap, hd, S = 4096, 64, 4
    c, m = filled(ops, rng, B, 1, cap, hd, [cap] * B)
    q = rng.standard_normal((B, S, hd), dtype=np.float32)
    good = np.array([[-1, 0, 1, 0]] * B, np.int32)
    bad = good.copy()
    bad[0, 2] = 2
    at = [4000] * B
    for pos0, parent in (([cap - S + 1] + at[1:], good), ([2 ** 31 - 1] + at[1:], good), (at, bad)):
        with pytest.raises(VmlmError) as e:
            c.attention_tree(q, pos0, None, parent)
        assert e.value.code == 9
        out = np.full(q.shape, 3.0, np.float32)
        with pytest.raises(VmlmError):
            c.attention_tree(q, pos0, None, parent, out=out)
    for pos0 in (at, [cap - S] + at[1:], [-1] + at[1:]):
        check_tree(c.attention_tree(q, pos0, None, good), tree_ref(m, q, pos0, [S] * B, good, 1, hd, 0.125))


def test_attention_shares_and_refused_sequences(dev, ops):
    """On the device, past the guard: the refused sequence's rows stay, the others' are right."""
    rng = np.random.default_rng(79)
    B, cap, hd, S = 3, 4096, 64, 4
    c, m = filled(ops, rng, B, 1, cap, hd, [cap] * B)
    _, d = device_cache(dev, c)
    q = rng.standard_normal((B, S, hd), dtype=np.float32)
    parent = np.array([[-1, 0, 1, 0]] * B, np.int32)
    parent[1, 3] = 3
    pos0 = np.array([4090, 1000, 4093], np.int32)  # (the last one's tokens pass the capacity)
    dq, dp, dt, do = dev.up(q), dev.up(pos0), dev.up(parent), dev.up(np.full(q.shape, 3.0, np.float32))
    st = dev.stream()
    dev.sync()
    dev.check(dev.L.vmlm_hip_attention_tree_kv4(d, dq.ptr, hd, dp.ptr, None, dt.ptr, S, do.ptr, hd, 1, 0.125, None, 0, st))
    dev.sync()
    assert dev.L.vmlm_hip_check_guards() == 9
    out = do.get()
    assert (out[1:] == 3).all()
    check_tree(out[:1], tree_ref(m, q[:1], pos0[:1], [S], parent[:1], 1, hd, 0.125))


@pytest.mark.parametrize("G", [17, 63])
@pytest.mark.parametrize("S", [1, 64])
@pytest.mark.parametrize("hd", [32, 128])
def test_attention_many_queries_a_head(ops, G, S, hd):
    """Tiles that end inside a token's heads."""
    rng = np.random.default_rng(G + S)
    c, m = filled(ops, rng, 1, 1, 160, hd, [90 + S])
    q = rng.standard_normal((1, S, G * hd), dtype=np.float32)
    parent = random_tree(rng, S, "late")[None]
    out = c.attention_tree(q, [90], None, parent)
    check_tree(out, tree_ref(m, q, [90], [S], parent, 1, hd, float(np.float32(hd ** -0.5))))


@pytest.mark.parametrize("H,Hkv,hd", [(8, 4, 128), (4, 4, 64), (12, 4, 128), (8, 8, 256)])
def test_attention_chunks_that_fill_the_card(ops, H, Hkv, hd):
    """Many tiles of many sequences, of unlike lengths, that end inside a token's heads or behind the last."""
    rng = np.random.default_rng(H + hd)
    B, cap, S = 16, 480, 400
    pos0 = rng.integers(0, 80, B).astype(np.int32)
    count = rng.integers(1, S + 1, B).astype(np.int32)
    pos0[3], pos0[5], count[0], count[5], count[7], count[9] = -1, 80, 0, 400, 17, 1
    c, m = filled(ops, rng, B, Hkv, cap, hd, np.where(pos0 >= 0, pos0 + count, 0))
    q = rng.standard_normal((B, S, H * hd), dtype=np.float32)
    out = c.attention_tree(q, pos0, count)
    scale = float(np.float32(hd ** -0.5))
    for b in range(B):
        n = count[b] if pos0[b] >= 0 else 0
        assert not out[b, n:].any()
        for t in {0, 11, 15, 16, 23, 24, n // 2, n - 2, n - 1} & set(range(n)):
            one = {x: y[b:b + 1] for x, y in m.items()}
            check_tree(out[b:b + 1, t:t + 1],
                       tree_ref(one, q[b:b + 1, t:t + 1], [pos0[b] + t], [1], None, Hkv, hd, scale))


def test_attention_queries_in_the_output(dev, ops):
    """Two calls in a row whose second reads what the first wrote, and an unaligned output."""
    rng = np.random.default_rng(30)
    H, hd, S, cap = 2, 64, 4, 96
    c, m = filled(ops, rng, 1, H, cap, hd, [70])
    _, d = device_cache(dev, c)
    q = rng.standard_normal((1, S, H * hd), dtype=np.float32)
    dq, dp = dev.up(q), dev.up(np.array([66], np.int32))
    a, b = dev.zeros(S * H * hd + 1), dev.zeros(S * H * hd + 1)
    st = dev.stream()
    dev.sync()
    w = H * hd
    dev.check(dev.L.vmlm_hip_attention_tree_kv4(d, dq.ptr, w, dp.ptr, None, None, S, a.ptr + 4, w, H, 0.125, None, 0, st))
    dev.check(dev.L.vmlm_hip_attention_tree_kv4(d, a.ptr + 4, w, dp.ptr, None, None, S, b.ptr + 4, w, H, 0.125, None, 0, st))
    dev.sync()
    one, two = (x.get()[1:].reshape(1, S, w) for x in (a, b))
    check_tree(one, tree_ref(m, q, [66], [S], None, H, hd, 0.125))
    check_tree(two, tree_ref(m, one, [66], [S], None, H, hd, 0.125))


# ------------------------------------------------------------------ at once
def attention_job(dev, ops, rng, B, H, Hkv, hd, cap, S):
    c, m = filled(ops, rng, B, Hkv, cap, hd, [cap] * B)
    keep, d = device_cache(dev, c)
    q = rng.standard_normal((B, S, H * hd), dtype=np.float32)
    parent = np.stack([random_tree(rng, S) for _ in range(B)])
    need = C.c_size_t()
    dev.check(dev.L.vmlm_hip_attention_tree_kv4_work(d, H, S, C.byref(need)))
    dq, dp, dt = dev.up(q), dev.up(np.full(B, cap - S, np.int32)), dev.up(parent)
    work = dev.zeros(max(need.value, 16), dtype=np.uint8)
    outs = [dev.zeros(B, S, H * hd) for _ in range(6)]
    w = H * hd

    def call(out, ptr, n, st):
        return dev.L.vmlm_hip_attention_tree_kv4(d, dq.ptr, w, dp.ptr, None, dt.ptr, S, out.ptr, w, H, 0.125,
                                                 ptr, n, st)

    def ref(pos0):
        return tree_ref(m, q, pos0, [S] * B, parent, Hkv, hd, 0.125)
    return dict(call=call, ref=ref, outs=outs, work=work, need=need.value, pos=dp, B=B, cap=cap, S=S, keep=(keep, dq, dt))


JOBS = [(1, 1, 1, 64, 8192, 5), (3, 2, 1, 128, 2080, 20), (1, 4, 4, 64, 4096, 40), (2, 1, 1, 256, 1056, 3)]


def test_attention_on_streams_at_once(dev, ops):
    """Calls at once on streams of their own, split positions in the streams' own workspaces, give
    what they give alone."""
    rng = np.random.default_rng(40)
    jobs = [attention_job(dev, ops, rng, *j) for j in JOBS]
    assert all(j["need"] for j in jobs)
    streams = [dev.stream() for _ in jobs]
    dev.sync()
    for i in range(6):
        for j, st in zip(jobs, streams):
            dev.check(j["call"](j["outs"][i], None, 0, st))
    dev.sync()
    for j in jobs:
        got = [o.get() for o in j["outs"]]
        check_tree(got[0], j["ref"]([j["cap"] - j["S"]] * j["B"]))
        assert all(np.array_equal(g, got[0]) for g in got[1:])


def test_attention_captured(dev, ops):
    """A split launch under capture without a workspace is refused and leaves the capture usable;
    graphs with workspaces of their own run at once, over other positions than the captured
    ones, with eager calls of the same streams between."""
    rng = np.random.default_rng(41)
    jobs = [attention_job(dev, ops, rng, *j) for j in JOBS]
    for j in jobs:
        st, graph = dev.stream(), C.c_void_p()
        dev.sync()
        dev.check(dev.L.vmlm_hip_capture_begin(st))
        assert j["call"](j["outs"][0], None, 0, st) == 9
        assert j["call"](j["outs"][0], j["work"].ptr, j["need"] - 4, st) == 9
        assert j["call"](j["outs"][0], j["work"].ptr + 4, j["need"], st) == 9
        dev.check(j["call"](j["outs"][0], j["work"].ptr, j["work"].nbytes, st))
        dev.check(dev.L.vmlm_hip_capture_end(st, C.byref(graph)))
        j.update(st=st, graph=graph)
    for i in range(4):
        for j in jobs:
            j["at"] = [int(rng.integers(0, j["cap"] - j["S"])) for _ in range(j["B"])]
            if i == 2:
                j["at"][0] = -1
            j["pos"].put(np.array(j["at"], np.int32))
            j["outs"][0].put(np.zeros(j["outs"][0].shape, np.float32))
            j["outs"][1].put(np.zeros(j["outs"][1].shape, np.float32))
        dev.sync()
        for j in jobs:
            dev.check(dev.L.vmlm_hip_graph_launch(j["graph"], j["st"]))
        for j in jobs:
            dev.check(j["call"](j["outs"][1], None, 0, j["st"]))
        dev.sync()
        for j in jobs:
            ref = j["ref"](j["at"])
            check_tree(j["outs"][0].get(), ref)
            assert np.array_equal(j["outs"][0].get(), j["outs"][1].get())
    for j in jobs:
        dev.check(dev.L.vmlm_hip_graph_destroy(j["graph"]))


def sample_job(dev, rng, rows, vocab):
    x = rng.standard_normal((rows, vocab), dtype=np.float32) * 3
    u, t = rng.random(rows, dtype=np.float32), np.full(rows, 0.8, np.float32)
    p = np.full(rows, 0.95, np.float32)
    need = C.c_size_t()
    dev.check(dev.L.vmlm_hip_sample_work(rows, vocab, C.byref(need)))
    dx, du, dt, dp = (dev.up(a) for a in (x, u, t, p))
    work = dev.zeros(max(need.value, 16), dtype=np.uint8)
    outs = [(dev.zeros(rows, dtype=np.int32), dev.zeros(rows)) for _ in range(4)]

    def call(out, ptr, n, st):
        return dev.L.vmlm_hip_sample(dx.ptr, vocab, du.ptr, dt.ptr, None, dp.ptr, None, rows, vocab, out[0].ptr,
                                     out[1].ptr, ptr, n, st)
    return dict(call=call, outs=outs, work=work, need=need.value, x=x, u=u, du=du, keep=(dx, dt, dp))


def sample_right(job, out):
    token, prob = (b.get() for b in out)
    for r in range(len(token)):
        want, share, near = sample_ref(job["x"][r], job["u"][r], 0.8, 0, 0.95, 0.0)
        assert near < 1e-8 or (token[r] == want and abs(prob[r] - share) <= 2.0 ** -20)


@pytest.mark.parametrize("graphs", [False, True])
def test_sample_at_once(dev, graphs):
    """Sliced calls on streams of their own at once, in the streams' workspaces, or captured with
    workspaces of their own and replayed with other random numbers."""
    rng = np.random.default_rng(42)
    jobs = [sample_job(dev, rng, rows, vocab) for rows, vocab in ((1, 122753), (3, 70001), (8, 40000))]
    assert all(j["need"] for j in jobs)
    for j in jobs:
        j["st"] = dev.stream()
        if graphs:
            j["graph"] = C.c_void_p()
            dev.sync()
            dev.check(dev.L.vmlm_hip_capture_begin(j["st"]))
            assert j["call"](j["outs"][0], None, 0, j["st"]) == 9
            assert j["call"](j["outs"][0], j["work"].ptr, j["need"] - 1, j["st"]) == 9
            dev.check(j["call"](j["outs"][0], j["work"].ptr, j["need"], j["st"]))
            dev.check(dev.L.vmlm_hip_capture_end(j["st"], C.byref(j["graph"])))
    for i in range(3):
        for j in jobs:
            j["u"] = rng.random(j["u"].shape, dtype=np.float32)
            j["du"].put(j["u"])
        dev.sync()
        for j in jobs:
            if graphs:
                dev.check(dev.L.vmlm_hip_graph_launch(j["graph"], j["st"]))
            for out in j["outs"][1 if graphs else 0:]:
                dev.check(j["call"](out, None, 0, j["st"]))
        dev.sync()
        for j in jobs:
            sample_right(j, j["outs"][0])
            for out in j["outs"][1:]:
                assert all(np.array_equal(a.get(), b.get()) for a, b in zip(out, j["outs"][0]))
    for j in jobs if graphs else ():
        dev.check(dev.L.vmlm_hip_graph_destroy(j["graph"]))


# ------------------------------------------------------------------ sampling
@pytest.mark.parametrize("rows", [2, 300])
@pytest.mark.parametrize("t", [1e-45, 1e-38, 1e-30, 1e-10, 1e-4, 1e10, 3e38])
@pytest.mark.parametrize("size", [1e-30, 1.0, 1e8, 1e30])
def test_sample_temperatures_at_the_ends(ops, rows, t, size):
    """Temperatures far below a step of the logits leave the largest one and its equals, far above them all
    alike."""
    rng = np.random.default_rng(50)
    vocab = 40000 if rows == 2 else 3000
    x = (rng.standard_normal((4, vocab)) * size).astype(np.float32)
    x[1, rng.integers(0, vocab, 9)] = x[1].max()  # equal ones
    x[2] = np.round(x[2] / np.float32(size) * 4) * np.float32(size)  # many equal ones
    x[3, ::3] = -np.inf
    x = np.ascontiguousarray(np.tile(x, (-(-rows // 4), 1))[:rows] if rows > 4 else x[[1, 2]])
    u = rng.random(rows, dtype=np.float32)
    token, prob = ops.sample(x, u, np.float32(t))
    for r in range(min(rows, 8)):
        want, share, near = sample_ref(x[r], u[r], np.float32(t))
        if near > 1e-8:
            assert token[r] == want and abs(prob[r] - share) <= 2.0 ** -20 * max(share, 2.0 ** -40)


@pytest.mark.parametrize("vocab", [32769, 122753, 2 ** 20 - 1])
def test_sample_slices_of_every_kind(ops, vocab):
    """Slices without a token, with the only tokens, with a NaN or an infinity, with more tokens of the first bins
    than a slice lists; the largest one at either end."""
    rng = np.random.default_rng(51)
    base = rng.standard_normal(vocab, dtype=np.float32)
    rows = [base.copy() for _ in range(8)]
    rows[0][8192:] = -np.inf
    rows[1][:-8192] = -np.inf
    rows[2][:-1] = -np.inf
    rows[3][0] = rows[3][-1] = 9
    rows[4][:2000] = 3.0
    rows[4][-3000:] = 3.0 - 1e-4
    rows[5][9000:9300] += 20
    rows[6][-5] = np.nan
    rows[7][10000] = np.inf
    x = np.stack(rows)
    for i in range(8):
        for k, p, m in ((0, 1.0, 0.0), (50, 0.9, 0.0), (0, 0.5, 0.01), (3000, 1.0, 0.0)):
            u = rng.random(1, dtype=np.float32)
            if i < 6:
                check_sample(ops, x[i:i + 1], u, 0.9, k, p, m)
            else:
                token, prob = ops.sample(x[i:i + 1], u, 0.9, k, p, m)
                assert token[0] == -1 and np.isnan(prob[0])


@pytest.mark.parametrize("rows", [513, 1500])
def test_sample_more_rows_than_workgroups(ops, rows):
    rng = np.random.default_rng(52)
    x = rng.standard_normal((rows, 501), dtype=np.float32) * 4
    check_sample(ops, x, rng.random(rows, dtype=np.float32), 1.0, rng.integers(0, 60, rows),
                 rng.random(rows).astype(np.float32) * 1.2, 0.0)


@pytest.mark.parametrize("k,p,m", [(0, 1.0, 0.0), (40, 0.9, 0.0), (0, 1.0, 0.05), (20000, 0.99, 0.0)])
def test_sample_few_and_many_rows_agree(ops, k, p, m):
    """A row alone (in slices) and among hundreds (by one workgroup): the same token and share."""
    rng = np.random.default_rng(53)
    vocab, n = 50000, 300
    x = np.tile(rng.standard_normal((3, vocab), dtype=np.float32) * 2, (100, 1))
    u = rng.random(n, dtype=np.float32)
    token, prob = ops.sample(x, u, 1.0, k, p, m)
    for r in (0, 1, 2, 150, 299):
        one, share = ops.sample(x[r:r + 1], u[r:r + 1], 1.0, k, p, m)
        assert one[0] == token[r] and share[0] == prob[r]
