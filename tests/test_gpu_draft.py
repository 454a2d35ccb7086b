"""The operators of a step that verifies drafted tokens (rotation, attention of trees over
the 4-bit cache, sampling, acceptance) on the GPU against their definitions in 64 bits.

Tolerances (u = 2^-24, half a step of f32):
 * rotation: sine and cosine 4 u of their own, 2 pi u of the f32 angle and u of the
   factor's product, two products and a sum, against the pair's length: 16 u.
 * attention, per output channel: with p the weights, R the largest value that a position's
   32 channels can hold and t a score's distance from the largest one, sum_p p R (e + mean e)
   where e = ds + (96 + n + 4 t) u. The score is off by ds = (2 hd + 48) u scale
   sum_g |q_g|_1 K_g over the groups g of 32 channels (K the largest value its key's group can
   hold): queries to 22 bits (2 u of each), f32 sums of 2 hd products and a few more. 4 t u
   is the exponent's product with log2(e) and its rounding; n u sums over the positions;
   96 u the exponential, weights held in 22 bits (4 u), the conversions and the joins.
 * sampling, acceptance: tokens, paths and cache contents are equal; prob is off by 2^-20 (the
   bins' sums to 2^-30 of a weight, the roundings of f32)."""
import ctypes as C

import numpy as np
import pytest
from test_gpu_4bit import (U, Dev, cache_codes, dev, device_cache, filled, held,  # noqa: F401
                           new_model, ops, put)

from sparrow_amd import VmlmError

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ rotation
def rope_ref(x, pos, freq, hd, inter, factor):
    """(rotated rows in 64 bits, their bound)."""
    rot = 2 * len(freq)
    y = x.astype(np.float64).reshape(x.shape[0], -1, hd).copy()
    a, b = (slice(0, rot, 2), slice(1, rot, 2)) if inter else (slice(0, rot // 2), slice(rot // 2, rot))
    turn = (pos[:, None].astype(np.float64) * freq)[:, None]
    c, s = factor * np.cos(turn), factor * np.sin(turn)
    lo, hi = y[..., a].copy(), y[..., b].copy()
    tol = np.zeros_like(y)
    y[..., a], y[..., b] = lo * c - hi * s, lo * s + hi * c
    tol[..., a] = tol[..., b] = 16 * U * np.hypot(lo, hi) * factor
    return y.reshape(x.shape), tol.reshape(x.shape)


@pytest.mark.parametrize("rows,H,Hkv,hd,rot", [(1, 36, 36, 64, 64), (1, 1, 0, 2, 2), (2, 0, 3, 16, 8), (5, 4, 2, 80, 20),
                                               (3, 5, 5, 96, 24), (300, 8, 2, 128, 64), (7, 3, 1, 512, 512),
                                               (33, 2, 2, 6, 4), (65, 32, 8, 128, 128), (2, 257, 1, 30, 14)])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("far", [0, 1 << 20])
def test_rope(ops, rows, H, Hkv, hd, rot, inter, far):
    rng = np.random.default_rng(rows + hd)
    q, k = (rng.standard_normal((rows, h * hd), dtype=np.float32) for h in (H, Hkv))
    pos = (rng.integers(0, 5000, rows) + far).astype(np.int32)
    if rows > 2:
        pos[1] = -1
    freq, factor = ops.rope_freqs(rot, 10000.0, ("ramp", 16, 1, 8, 4096))
    got = ops.rope_qk(q, k, pos, freq, hd, inter, factor)
    for x, y in zip((q, k), got):
        ref, tol = rope_ref(x, pos, freq, hd, inter, factor)
        assert not y[pos < 0].any()
        assert (np.abs(y - ref)[pos >= 0] <= tol[pos >= 0]).all()


def test_rope_positions_and_values(ops):
    """Position 0 is the identity, the largest position and values that are not finite."""
    rng = np.random.default_rng(1)
    hd = 64
    q = rng.standard_normal((4, hd), dtype=np.float32)
    q[2, 3], q[3, 5] = np.inf, np.nan
    freq, _ = ops.rope_freqs(32)
    pos = np.array([0, 2 ** 31 - 1, 7, 7], np.int32)
    y, _ = ops.rope_qk(q, q[:, :0], pos, freq, hd, True)
    assert np.array_equal(y[0], q[0])
    with np.errstate(invalid="ignore"):
        ref, tol = rope_ref(q, pos, freq, hd, True, 1.0)
    # (the angle of position 2^31: 64 bits leave 2^-22 of a turn)
    assert (np.abs(y[1] - ref[1]) <= tol[1] + 2.0 ** -20).all()
    other = np.ones(hd, bool)
    other[[2, 3]] = False
    assert (np.abs(y[2] - ref[2]) <= tol[2])[other].all() and not np.isfinite(y[2, 2:4]).any()
    assert np.isnan(y[3, 4:6]).all() and np.array_equal(y[3, 32:], q[3, 32:])


@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("hd,rot", [(64, 32), (20, 6)])
def test_rope_strides_and_bounds(dev, ops, inplace, hd, rot):
    """q and k inside fused rows of an odd stride at an odd address; rows of idle positions and everything
    beside the heads stay as they were."""
    rng = np.random.default_rng(3)
    rows, H, Hkv = 9, 3, 2
    ld = (H + 2 * Hkv) * hd + 3
    x = rng.standard_normal(1 + rows * ld, dtype=np.float32)
    pos = np.array([5, -1, 0, 9, 4, 3, -1, 2, 77], np.int32)
    freq, _ = ops.rope_freqs(rot)
    dx, dp, df = dev.up(x), dev.up(pos), dev.up(freq)
    do = dx if inplace else dev.up(np.full_like(x, 3.0))
    src, dst = dx.ptr + 4, do.ptr + 4
    dev.check(dev.L.vmlm_hip_rope_qk(dst, ld, dst + 4 * H * hd, ld, src, ld, src + 4 * H * hd, ld, dp.ptr,
                                     df.ptr, rows, H, Hkv, hd, rot, False, 0.5, None))
    dev.sync()
    got, x = do.get()[1:].reshape(rows, ld), x[1:].reshape(rows, ld)
    w = (H + Hkv) * hd
    ref, tol = rope_ref(np.ascontiguousarray(x[:, :w]), pos, freq, hd, False, 0.5)
    live = pos >= 0
    assert (np.abs(got[:, :w] - ref)[live] <= tol[live]).all()
    kept = x if inplace else np.full_like(x, 3.0)
    assert np.array_equal(got[:, w:], kept[:, w:]) and np.array_equal(got[~live], kept[~live])


# ------------------------------------------------------------------ attention
def random_tree(rng, S, kind="any"):
    parent = np.full(S, -1, np.int32)
    for t in range(1, S):
        parent[t] = {"any": rng.integers(-1, t), "wide": 0, "deep": t - 1,
                     "late": max(0, t - 1 - int(rng.integers(0, 4)))}[kind]
    return parent


def sees(parent, pos0, n, t):
    """The positions that token t sees, ascending."""
    own = []
    at = t
    while at >= 0:
        own.append(pos0 + at)
        at = at - 1 if parent is None else parent[at]
    return np.concatenate([np.arange(pos0), np.array(own[::-1])]).astype(int)


def spread(meta):
    lo = (meta & np.uint32(0xFFFF0000)).view(np.float32).astype(np.float64)
    return lo, (meta << np.uint32(16)).view(np.float32).astype(np.float64)


def tree_ref(m, q, pos0, count, parent, Hkv, hd, scale):
    """(out in 64 bits, its bound, the rows that are live); m: a model of the cache."""
    B, S, H = q.shape[0], q.shape[1], q.shape[2] // hd
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    live = np.zeros((B, S), bool)
    for b in range(B):
        if pos0[b] < 0:
            continue
        most = []
        for name in ("km", "vm"):
            lo, sc = spread(m[name][b])
            most.append(np.maximum(np.abs(lo), np.abs(lo + 15 * sc)))
        for t in range(min(max(count[b], 0), S)):
            live[b, t] = True
            see = sees(None if parent is None else parent[b], pos0[b], count[b], t)
            for h in range(H):
                kv, at = h // (H // Hkv), slice(h * hd, (h + 1) * hd)
                x = q[b, t, at].astype(np.float64)
                s = m["k"][b, kv, see].astype(np.float64) @ x * scale
                d = s.max() - s
                p = np.exp(-d)
                p /= p.sum()
                e = (96 + len(see) + 4 * d) * U
                e += (2 * hd + 48) * U * abs(scale) * (most[0][kv, see] @ np.abs(x).reshape(-1, 32).sum(1))
                out[b, t, at] = p @ m["v"][b, kv, see].astype(np.float64)
                w = (p * (e + p @ e))[:, None] * most[1][kv, see] + 2.0 ** -126 * most[1][kv, see]
                tol[b, t, at] = np.repeat(w.sum(0), 32) + 2.0 ** -130
    return out, tol, live


def check_tree(out, ref, old=0.0):
    ref, tol, live = ref
    assert (out[~live] == old).all()
    d = np.abs(out - ref)[live]
    assert (d <= tol[live]).all(), (d / tol[live]).max()


TREES = [  # B, H, Hkv, hd, cap, pos0, S, counts
    (1, 1, 1, 64, 32, [0], 1, None), (1, 1, 1, 32, 32, [31], 1, None), (1, 36, 36, 64, 64, [50], 8, None),
    (3, 4, 4, 64, 256, [0, 100, 193], 63, [63, 40, 1]), (2, 6, 2, 128, 320, [250, 31], 16, [16, 9]),
    (4, 8, 1, 64, 192, [31, -1, 128, 64], 64, [64, 64, 0, 33]), (2, 16, 1, 256, 160, [77, 96], 7, [7, 5]),
    (1, 15, 3, 32, 544, [481], 62, None), (1, 20, 1, 128, 128, [3], 13, None), (1, 2, 1, 64, 4160, [4060], 33, None),
    (1, 2, 2, 128, 8192, [8128], 64, None), (2, 5, 1, 64, 5120, [5000, 3], 21, [21, 20]),
    (1, 1, 1, 256, 2080, [2000], 50, None), (9, 3, 3, 32, 96, [0, 1, 31, 32, 33, 63, 64, -1, 65], 31, None),
    (1, 34, 2, 64, 1024, [900], 5, None)]


@pytest.mark.parametrize("B,H,Hkv,hd,cap,pos0,S,count", TREES)
@pytest.mark.parametrize("kind", ["any", "wide", "deep", "late", "chain"])
def test_attention_tree(ops, B, H, Hkv, hd, cap, pos0, S, count, kind):
    rng = np.random.default_rng(cap + H + hd + S)
    n = np.full(B, S) if count is None else np.array(count)
    pos0 = np.array(pos0, np.int32)
    c, m = filled(ops, rng, B, Hkv, cap, hd, np.where(pos0 >= 0, pos0 + n, 0))
    q = rng.standard_normal((B, S, H * hd), dtype=np.float32)
    parent = None if kind == "chain" else np.stack([random_tree(rng, S, kind) for _ in range(B)])
    if parent is not None:
        for b in range(B):
            parent[b, n[b]:] = 99  # behind the last token: not looked at
    old = np.full_like(q, 3.0)
    out = c.attention_tree(q, pos0, count, parent, out=old)
    scale = float(np.float32(hd ** -0.5))
    check_tree(out, tree_ref(m, q, pos0, n, parent, Hkv, hd, scale), 3.0)


@pytest.mark.parametrize("H,Hkv,hd,S,pos0", [(4, 2, 64, 333, 100), (8, 1, 128, 70, 0), (1, 1, 32, 200, 31),
                                             (3, 3, 256, 90, 700), (2, 1, 64, 129, 4000)])
def test_attention_chunk(ops, H, Hkv, hd, S, pos0):
    """A prompt's chunk: every token sees those before it. The second sequence has fewer tokens."""
    rng = np.random.default_rng(S)
    cap = -(-(pos0 + S) // 32) * 32
    n = np.array([S, S // 3])
    at = np.array([pos0, pos0 // 2], np.int32)
    c, m = filled(ops, rng, 2, Hkv, cap, hd, at + n)
    q = rng.standard_normal((2, S, H * hd), dtype=np.float32)
    out = c.attention_tree(q, at, n)
    check_tree(out, tree_ref(m, q, at, n, None, Hkv, hd, float(np.float32(hd ** -0.5))))


@pytest.mark.parametrize("H,Hkv,hd", [(2, 1, 64), (4, 4, 32), (8, 2, 128), (1, 1, 256)])
def test_attention_equals_decoding(ops, H, Hkv, hd):
    """A chain of tokens gives what the decode attention gives token by token, to the
    sum of both bounds."""
    rng = np.random.default_rng(hd)
    S, pos0, cap = 9, 60, 96
    c, m = filled(ops, rng, 1, Hkv, cap, hd, [pos0 + S])
    q = rng.standard_normal((1, S, H * hd), dtype=np.float32)
    got = c.attention_tree(q, [pos0])
    _, tol, _ = tree_ref(m, q, [pos0], [S], None, Hkv, hd, float(np.float32(hd ** -0.5)))
    for t in range(S):
        assert (np.abs(got[0, t] - c.attention_decode(q[:, t], [pos0 + t])[0]) <= 2 * tol[0, t]).all()


def test_attention_scales_and_masks(ops):
    """Large scores, a negative scale and scale 0 (the mean of what is seen)."""
    rng = np.random.default_rng(5)
    c, m = filled(ops, rng, 1, 1, 160, 64, [140])
    q = rng.standard_normal((1, 12, 128), dtype=np.float32)
    parent = random_tree(rng, 12)[None]
    for scale in (40.0, -0.5, 0.0):
        out = c.attention_tree(q, [128], None, parent, scale=scale)
        check_tree(out, tree_ref(m, q, [128], [12], parent, 1, 64, scale))


@pytest.mark.parametrize("hd,G", [(64, 1), (128, 4), (32, 2), (256, 1)])
@pytest.mark.parametrize("pos0", [0, 40, 1200])
def test_attention_nonfinite(ops, hd, G, pos0):
    """A query head that is not finite is NaN alone; a key that is not, to the tokens that see it;
    a value that is not, in its 32 channels to those tokens."""
    rng = np.random.default_rng(hd + pos0)
    S, cap = 20, 1248
    parent = random_tree(rng, S, "late")[None]
    k, v = rng.standard_normal((2, 1, pos0 + S, hd), dtype=np.float32)
    k[0, pos0 + 5, 3] = np.nan
    v[0, pos0 + 8, 1] = np.inf
    v[0, pos0 + 11, hd - 1] = np.nan
    q = rng.standard_normal((1, S, G * hd), dtype=np.float32)
    q[0, 2, 7] = np.inf
    q[0, 3, hd * (G - 1) + 9] = np.nan
    c = ops.Kv4Cache(1, 1, cap, hd)
    c.append(k, v, [0])
    out = c.attention_tree(q, [pos0], None, parent).reshape(S, G, hd)
    m = new_model(1, 1, cap, hd)
    k, v = np.nan_to_num(k, nan=0, posinf=0), np.nan_to_num(v, nan=0, posinf=0)
    k[0, pos0 + 5] = v[0, pos0 + 8, :32] = v[0, pos0 + 11, -32:] = 0
    put(m, k[0], v[0], 0, 0, pos0 + S, 1)
    bad = np.zeros((S, G, hd), bool)
    bad[2, 0] = bad[3, G - 1] = True
    for t in range(S):
        own = sees(parent[0], pos0, S, t) - pos0
        bad[t] |= 5 in own
        bad[t, :, :32] |= 8 in own
        bad[t, :, -32:] |= 11 in own
    assert bad.any() and not bad.all()
    assert np.array_equal(np.isnan(out), bad)
    ref, tol, _ = tree_ref(m, np.nan_to_num(q, nan=0, posinf=0), [pos0], [S], parent, 1, hd,
                           float(np.float32(hd ** -0.5)))
    ok = ~bad.reshape(S, -1)
    assert (np.abs(out.reshape(S, -1) - ref[0])[ok] <= tol[0][ok]).all()


@pytest.mark.parametrize("hd,H", [(64, 1), (128, 4), (32, 2), (256, 1)])
def test_attention_unseen_tokens_leave_no_trace(ops, hd, H):
    """Siblings whose keys and values are poisoned or huge: a token that does not see them
    gives the same bits as with ordinary ones there."""
    rng = np.random.default_rng(hd)
    S, pos0, cap = 6, 45, 64
    parent = np.array([[-1, 0, 0, 1, 2, 3]], np.int32)
    k, v = rng.standard_normal((2, 1, pos0 + S, hd), dtype=np.float32)
    q = rng.standard_normal((1, S, H * hd), dtype=np.float32)
    outs = []
    for poison in (None, np.nan, np.inf, 1e30):
        kk, vv = k.copy(), v.copy()
        if poison is not None:
            kk[0, pos0 + 2], vv[0, pos0 + 2] = poison, poison
            vv[0, pos0 + 4] = poison
        c = ops.Kv4Cache(1, 1, cap, hd)
        c.append(kk, vv, [0])
        outs.append(c.attention_tree(q, [pos0], None, parent)[0])
    for out in outs[1:]:
        assert np.array_equal(out[[0, 1, 3, 5]], outs[0][[0, 1, 3, 5]])


@pytest.mark.parametrize("hd", [32, 64, 128, 256])
def test_attention_every_bit(ops, hd):
    """Integers that every step holds exactly: queries of 22 bits in two channels that nearly cancel, equal
    weights, values of 11 bits: the output is the mean of the values."""
    rng = np.random.default_rng(hd)
    S, pos0 = 4, 12
    q = np.zeros((1, S, hd), np.float32)
    big = rng.integers(2 ** 21, 2 ** 22, (S, hd // 32))
    q[0, :, 5::32], q[0, :, 20::32] = big, -(big - rng.integers(1, 4, big.shape))
    k = np.zeros((1, pos0 + S, hd), np.float32)
    k[0, :, 5::32] = k[0, :, 20::32] = 15
    v = rng.integers(0, 16, (1, pos0 + S, hd)) * np.float32(128)
    v[0, :, 0::32], v[0, :, 1::32] = 0, 15 * 128
    c, m = ops.Kv4Cache(1, 1, 32, hd), new_model(1, 1, 32, hd)
    c.append(k, v, [0])
    put(m, k[0], v[0], 0, 0, pos0 + S, 1)
    assert np.array_equal(m["k"][0, 0, :pos0 + S], k[0]) and np.array_equal(m["v"][0, 0, :pos0 + S], v[0])
    out = c.attention_tree(q, [pos0], scale=2.0 ** -4)
    for t in range(S):
        mean = v[0, :pos0 + t + 1].astype(np.float64).mean(0)
        assert (np.abs(out[0, t] - mean) <= 8 * U * 2048).all()


def test_attention_refused_on_the_device(ops):
    """Tokens past the capacity and parents that are no earlier token: the guard trips, the
    sequence's rows stay as they were, the others are right."""
    rng = np.random.default_rng(6)
    c, m = filled(ops, rng, 2, 1, 96, 64, [96, 40])
    q = rng.standard_normal((2, 4, 64), dtype=np.float32)
    parent = np.array([[-1, 0, 1, 0]] * 2, np.int32)
    from sparrow_amd import _abi, check, lib
    for at, par in (([93, 30], parent), ([2 ** 31 - 1, 30], parent), ([10, 30], [[-1, 0, 2, 0], [-1, 0, 1, 0]]),
                    ([10, 30], [[-1, 0, -2, 0], [-1, 0, 1, 0]]), ([10, 30], [[0, 0, 1, 0], [-1, 0, 1, 0]])):
        with pytest.raises(VmlmError) as e:
            c.attention_tree(q, at, None, par)
        assert e.value.code == 9
    out = c.attention_tree(q, [92, 30], None, parent)
    check_tree(out, tree_ref(m, q, [92, 30], [4, 4], parent, 1, 64, 0.125))


def test_attention_strides(dev, ops):
    """Queries inside fused rows of an odd stride at an odd address, outputs likewise; idle and
    padding rows and what lies beside the heads stay as they were."""
    rng = np.random.default_rng(12)
    B, H, Hkv, hd, cap, S = 3, 4, 2, 64, 1216, 5
    pos0, count = np.array([40, -1, 1200], np.int32), np.array([5, 5, 3], np.int32)
    c, m = filled(ops, rng, B, Hkv, cap, hd, np.where(pos0 >= 0, pos0 + count, 0))
    parent = np.stack([random_tree(rng, S) for _ in range(B)])
    ld, ldo = (H + 2 * Hkv) * hd + 3, H * hd + 1
    x = rng.standard_normal(1 + B * S * ld, dtype=np.float32)
    _, d = device_cache(dev, c)
    dx, dp, dn, dt = dev.up(x), dev.up(pos0), dev.up(count), dev.up(parent)
    do = dev.up(np.full(1 + B * S * ldo, 3.0, np.float32))
    st = dev.stream()
    dev.sync()
    dev.check(dev.L.vmlm_hip_attention_tree_kv4(d, dx.ptr + 4, ld, dp.ptr, dn.ptr, dt.ptr, S,
                                                do.ptr + 4, ldo, H, 0.125, None, 0, st))
    dev.sync()
    q = np.ascontiguousarray(x[1:].reshape(B, S, ld)[:, :, :H * hd])
    got = do.get()
    assert got[0] == 3
    got = got[1:].reshape(B, S, ldo)
    assert (got[..., -1] == 3).all()
    check_tree(got[..., :-1], tree_ref(m, q, pos0, count, parent, Hkv, hd, 0.125), 3.0)


def test_attention_offsets_past_32_bits(dev):
    """The last of five sequences whose caches are 1 GB of codes each: its rows lie
    past 2^32 bytes in every array of codes; the accepted ones move there."""
    from sparrow_amd import _abi
    B, H, cap, hd, S = 5, 8, 1 << 20, 256, 6
    ptrs = []
    for n in [B * H * cap * hd // 2] * 2 + [B * H * cap * hd // 8] * 2:
        p = C.c_void_p()
        dev.check(dev.L.vmlm_hip_malloc(C.byref(p), n))
        dev.bufs.append(p.value)
        ptrs.append(p.value)
    d = _abi.Kv4Cache(*ptrs, B, H, cap, hd)
    rng = np.random.default_rng(16)
    w = H * hd
    k, v, q = rng.standard_normal((3, B, S, w), dtype=np.float32)
    dk, dv, dq, out = dev.up(k), dev.up(v), dev.up(q), dev.zeros(B, S, w)
    pos = np.array([-1] * (B - 1) + [0], np.int32)
    dp, dn = dev.up(pos), dev.up(np.full(B, S, np.int32))
    need = C.c_size_t()
    dev.check(dev.L.vmlm_hip_attention_tree_kv4_work(d, H, S, C.byref(need)))
    work = dev.zeros(max(need.value, 16), dtype=np.uint8)
    dev.check(dev.L.vmlm_hip_kv4_append(d, dk.ptr, w, dv.ptr, w, dp.ptr, None, S, None))
    dev.check(dev.L.vmlm_hip_attention_tree_kv4(d, dq.ptr, w, dp.ptr, dn.ptr, None, S, out.ptr, w, H,
                                                0.0625, work.ptr, work.nbytes, None))
    dev.check(dev.L.vmlm_hip_check_guards())
    dev.sync()
    m = new_model(B, H, 32, hd)
    put(m, k[-1], v[-1], B - 1, 0, S, H)
    check_tree(out.get(), tree_ref(m, q, pos, [S] * B, None, H, hd, 0.0625))
    # a tree at the end of the capacity: tokens 2 and 5 after the first
    first = cap - S
    dp.put(np.array([-1] * (B - 1) + [first], np.int32))
    parent = np.tile(np.array([-1, 0, 0, 1, 1, 2], np.int32), (B, 1))
    drafted = np.tile(np.arange(S, dtype=np.int32) + 10, (B, 1))
    chosen = np.zeros((B, S), np.int32)
    chosen[:, 0], chosen[:, 2], chosen[:, 5] = 12, 15, 7
    dt, dd, dc = dev.up(parent), dev.up(drafted), dev.up(chosen)
    res = dev.zeros(B, S, dtype=np.int32), dev.zeros(B, dtype=np.int32), dev.zeros(B, dtype=np.int32)
    dev.check(dev.L.vmlm_hip_kv4_append(d, dk.ptr, w, dv.ptr, w, dp.ptr, None, S, None))
    dev.check(dev.L.vmlm_hip_tree_accept_kv4(d, 1, dp.ptr, None, dt.ptr, dd.ptr, dc.ptr, S,
                                             *(x.ptr for x in res), None))
    rk, rv = dev.zeros(B, S, w), dev.zeros(B, S, w)
    dev.check(dev.L.vmlm_hip_kv4_read(d, rk.ptr, w, rv.ptr, w, dp.ptr, None, S, None))
    dev.check(dev.L.vmlm_hip_check_guards())
    dev.sync()
    assert res[0].get()[-1].tolist() == [0, 2, 5, -1, -1, -1] and res[1].get()[-1] == 3 and res[2].get()[-1] == 7
    for got, x in ((rk.get()[-1], k[-1]), (rv.get()[-1], v[-1])):
        assert np.array_equal(got, held(x[[0, 2, 5, 3, 4, 5]])[2])


# ------------------------------------------------------------------ acceptance
def accept_ref(parent, drafted, chosen, n):
    path = [0]
    while True:
        want = chosen[path[-1]]
        nxt = [t for t in range(path[-1] + 1, n) if parent[t] == path[-1] and drafted[t] == want and want >= 0]
        if not nxt:
            return path, want
        path.append(nxt[0])


ACCEPTS = [(1, 1, 64, 32, 1, 1), (1, 36, 64, 96, 8, 2), (3, 2, 128, 160, 33, 1), (5, 3, 32, 128, 64, 17),
           (2, 1, 256, 96, 20, 3), (16, 2, 64, 96, 63, 4), (2, 1, 32, 64, 5, 33)]


@pytest.mark.parametrize("B,Hkv,hd,cap,S,layers", ACCEPTS)
@pytest.mark.parametrize("kind", ["any", "late", "deep", "chain", "twins"])
def test_accept(ops, B, Hkv, hd, cap, S, layers, kind):
    """Few distinct tokens, so that paths are long and siblings often hold the same one (the first
    counts); the moved rows' codes and meta are equal bit for bit, every other one untouched."""
    rng = np.random.default_rng(B + hd + S + layers)
    pos0 = rng.integers(0, cap - S + 1, B).astype(np.int32)
    count = rng.integers(1, S + 1, B).astype(np.int32)
    count[0] = S
    if B > 2:
        pos0[1], count[2] = -1, 0
    parent = None if kind == "chain" else np.stack([random_tree(rng, S, {"twins": "late"}.get(kind, kind))
                                                    for _ in range(B)])
    drafted = rng.integers(0, 3, (B, S)).astype(np.int32)
    chosen = rng.integers(-1 if kind == "any" else 0, 3, (B, S)).astype(np.int32)
    if kind in ("deep", "chain", "twins"):  # most of the tree is accepted
        drafted[:], chosen[:] = 1, np.where(rng.random((B, S)) < 0.04, 2, 1)
    caches, before = [], []
    for _ in range(layers):
        c = ops.Kv4Cache(B, Hkv, cap, hd)
        for a in (c.k, c.v):
            a[:] = rng.integers(0, 256, a.shape)
        for a in (c.k_meta, c.v_meta):
            a[:] = rng.integers(0, 2 ** 32, a.shape, dtype=np.uint32)
        caches.append(c)
        before.append([x.copy() for x in (*cache_codes(c), c.k_meta, c.v_meta)])
    path, kept, nxt = ops.tree_accept(caches, pos0, drafted, chosen, count, parent)
    for b in range(B):
        if pos0[b] < 0 or count[b] == 0:
            assert (path[b] == -1).all() and kept[b] == 0 and nxt[b] == -1
            continue
        par = np.arange(S) - 1 if parent is None else parent[b]
        want, token = accept_ref(par, drafted[b], chosen[b], count[b])
        assert path[b].tolist() == want + [-1] * (S - len(want)) and kept[b] == len(want) and nxt[b] == token
        src, dst = pos0[b] + np.array(want), pos0[b] + np.arange(len(want))
        for old in before:
            for x in old:
                x[b, :, dst] = x[b, :, src].copy()
    for c, old in zip(caches, before):
        for got, x in zip((*cache_codes(c), c.k_meta, c.v_meta), old):
            assert np.array_equal(got, x)


def test_accept_refused_on_the_device(ops):
    c = ops.Kv4Cache(1, 1, 64, 32)
    c.k[:] = 7
    for at, parent in (([62], [[-1, 0, 0]]), ([5], [[-1, 1, 0]]), ([5], [[-1, -3, 0]]), ([2 ** 31 - 2], None)):
        with pytest.raises(VmlmError) as e:
            ops.tree_accept([c], at, [[1, 1, 1]], [[1, 1, 1]], parent=parent)
        assert e.value.code == 9
    assert (c.k == 7).all()


# ------------------------------------------------------------------ sampling
def sample_ref(x, u, t, k=0, p=1.0, m=0.0):
    """(token, prob) by the definition, and how near the decisions came to a border (relative to
    the sums): a test's inputs keep away from it."""
    x = x.astype(np.float64)
    order = np.lexsort((np.arange(x.size), -x))
    if t == 0:
        return order[0], 1.0, 1.0
    near = 1.0
    if 0 < k < x.size:
        order = order[:k]
    w = np.exp((x[order] - x[order[0]]) / np.float64(np.float32(t)))
    if p < 1:
        c, goal = np.cumsum(w) - w, np.float64(np.float32(p)) * w.sum()
        near = min(near, np.abs(c / w.sum() - np.float64(np.float32(p))).min())
        w = w[:max(1, np.count_nonzero(c < goal))]
    w = w[w >= np.float64(np.float32(m))]
    c = np.cumsum(w)
    goal = np.float64(np.float32(u)) * c[-1]
    near = min(near, np.abs(c[:-1] / c[-1] - np.float64(np.float32(u))).min()) if w.size > 1 else near
    i = min(int(np.searchsorted(c, goal, side="right")), w.size - 1)
    return order[i], w[i] / c[-1], near


def check_sample(ops, x, u, t, k, p, m):
    rows = x.shape[0]
    each = [np.broadcast_to(np.asarray(a, d), rows) for a, d in ((u, np.float32), (t, np.float32), (k, np.int32),
                                                                 (p, np.float32), (m, np.float32))]
    token, prob = ops.sample(x, *each)
    for r in range(rows):
        want, share, near = sample_ref(x[r], *(a[r] for a in each))
        if near > 1e-8:  # (f64 of both sides, 2^-30 of a weight)
            assert token[r] == want, (r, token[r], want, near, [a[r] for a in each])
            assert abs(prob[r] - share) <= 2.0 ** -20 * max(share, 2.0 ** -40), (r, prob[r], share)


SETTINGS = [(1.0, 0, 1.0, 0.0), (0.7, 40, 1.0, 0.0), (1.0, 0, 0.9, 0.0), (1.3, 0, 1.0, 0.1), (0.8, 50, 0.95, 0.05),
            (1.0, 1, 1.0, 0.0), (0.0, 5, 0.5, 0.0), (1.0, 0, 0.0, 0.0), (1.0, 0, 1.0, 1.0), (2.0, 100000, 0.999, 1e-6),
            (0.05, 0, 0.99, 0.0), (30.0, 7, 0.6, 0.0), (1.0, 3000, 1.0, 0.0)]


@pytest.mark.parametrize("t,k,p,m", SETTINGS)
@pytest.mark.parametrize("vocab", [1, 2, 7, 64, 1000, 4097, 32001, 122753])
def test_sample(ops, vocab, t, k, p, m):
    rng = np.random.default_rng(vocab)
    rows = 5
    x = rng.standard_normal((rows, vocab), dtype=np.float32) * np.float32(3)
    x[1, rng.integers(0, vocab, 5)] += 12  # peaked
    x[2] = x[2] * np.float32(0.01)  # nearly flat
    if vocab > 8:
        x[3, rng.integers(0, vocab, vocab // 2)] = -np.inf  # masked
        x[4, ::2] = np.finfo(np.float32).min
    check_sample(ops, x, rng.random(rows, dtype=np.float32), t, k, p, m)


@pytest.mark.parametrize("vocab", [3, 2048, 2049, 5000, 122753])
@pytest.mark.parametrize("value", [0.0, -7.25, np.finfo(np.float32).min])
def test_sample_equal_logits(ops, vocab, value):
    """All the same: the lowest indices come first, so that the token is arithmetic."""
    x = np.full((4, vocab), value, np.float32)
    u = np.array([0.0, 0.2503, 0.7001, 1 - 2.0 ** -24], np.float32)
    token, prob = ops.sample(x, u, 1.0)
    want = np.floor(u.astype(np.float64) * vocab).astype(int)
    assert np.array_equal(token, want) and np.abs(prob * vocab - 1).max() <= 2.0 ** -20
    k = max(1, vocab // 3)
    token, prob = ops.sample(x, u, 0.5, top_k=k)
    assert np.array_equal(token, np.floor(u.astype(np.float64) * k).astype(int))
    p = 0.37
    kept = max(1, int(np.ceil(np.float64(np.float32(p)) * vocab)))
    token, prob = ops.sample(x, u, 2.0, top_p=p, min_p=1.0)
    assert np.array_equal(token, np.floor(u.astype(np.float64) * kept).astype(int))
    assert np.abs(prob * kept - 1).max() <= 2.0 ** -20


@pytest.mark.parametrize("vocab", [6000, 100000])
def test_sample_few_values(ops, vocab):
    """Many equal logits of a few values, a step of f32 apart, and values that differ in their last bits
    only: more tokens in a bin than are sorted at once."""
    rng = np.random.default_rng(vocab)
    x = np.empty((6, vocab), np.float32)
    x[0] = rng.choice(np.float32([1.0, 1.0 + 2 ** -23, 1.0 - 2 ** -24]), vocab)
    x[1] = rng.choice(np.float32([0.0, -0.0, 1e-30, -1e-30]), vocab)
    x[2] = 1 + rng.integers(0, 5000, vocab) * np.float32(2 ** -23)
    x[3] = rng.standard_normal(vocab) * 1e-6
    x[4] = rng.integers(-3, 3, vocab)
    x[5] = rng.standard_normal(vocab) * 1e-38
    for u in (0.0, 0.123456, 0.5001, 0.98765):
        for k, p in ((0, 1.0), (vocab // 2 + 1, 1.0), (0, 0.61803), (vocab // 3, 0.777)):
            check_sample(ops, x, u, 1.0, k, p, 0.0)


def test_sample_frequencies(ops):
    """u over a fine grid: each token comes as often as its share of the grid, to one."""
    rng = np.random.default_rng(3)
    x = np.repeat(rng.standard_normal((1, 50), dtype=np.float32), 4096, 0)
    u = ((np.arange(4096) + 0.5) / 4096).astype(np.float32)
    token, prob = ops.sample(x, u, 0.9, top_p=0.9)
    got = np.bincount(token, minlength=50) / 4096
    for i in np.flatnonzero(got):
        share = prob[token == i]
        assert (share == share[0]).all() and abs(got[i] - share[0]) <= 1 / 4096 + 2.0 ** -20


def test_sample_rows_without_a_token(ops):
    x = np.zeros((7, 300), np.float32)
    x[0] = -np.inf
    x[1, 7] = np.nan
    x[2, 8] = np.inf
    x[3, :299] = -np.inf
    x[4, 5] = -np.inf
    x[6, 299], x[6, 0] = np.inf, np.nan
    u = np.float32([0.5, 0.5, 0.5, 0.999, 0.0, -1.0, 0.2])
    for t in (0.0, 1.0):
        token, prob = ops.sample(x, u, t, top_k=20)
        assert token.tolist() == [-1, -1, -1, 299, 0, -1, -1]
        assert prob[0] == 0 and np.isnan(prob[[1, 2, 6]]).all() and prob[3] == 1 and prob[5] == 0


def test_sample_settings_out_of_range(ops):
    x = np.zeros((2, 10), np.float32)
    nan = float("nan")
    for bad in (dict(u=[1.0, 0.5]), dict(u=[nan, 0.5]), dict(temperature=[-1.0, 1.0]), dict(temperature=[nan, 1.0]),
                dict(temperature=[float("inf"), 1.0]), dict(top_p=[nan, 1.0]), dict(min_p=[1.5, 0.0]),
                dict(min_p=[-0.1, 0.0]), dict(min_p=[nan, 0.0])):
        with pytest.raises(VmlmError) as e:
            ops.sample(x, **{"u": [0.5, 0.5], "temperature": [1.0, 1.0], **bad})
        assert e.value.code == 9, bad
    token, _ = ops.sample(x, [0.5, -0.0], 1.0)
    assert token.tolist() == [5, 0]


@pytest.mark.parametrize("rows", [3, 300])
def test_sample_strides_and_bounds(dev, rows):
    """Rows at an odd address and stride with poison between them, no prob, a stream of its own;
    idle rows and what lies behind the last one stay as they were."""
    rng = np.random.default_rng(9)
    vocab, ld = 5003, 5010
    buf = np.full(1 + rows * ld, np.nan, np.float32)
    x = buf[1:].reshape(rows, ld)
    x[:, :vocab] = rng.standard_normal((rows, vocab)) * 4
    u = rng.random(rows, dtype=np.float32)
    u[1] = -0.5
    dx, du = dev.up(buf), dev.up(u)
    dt = dev.up(np.ones(rows, np.float32))
    tok, prob = dev.up(np.full(rows + 1, 77, np.int32)), dev.up(np.full(rows + 1, 7.0, np.float32))
    st = dev.stream()
    dev.sync()
    for out in (None, prob.ptr):
        dev.check(dev.L.vmlm_hip_sample(dx.ptr + 4, ld, du.ptr, dt.ptr, None, None, None, rows, vocab,
                                        tok.ptr, out, None, 0, st))
        dev.sync()
        got, share = tok.get(), prob.get()
        assert got[-1] == 77 and got[1] == 77 and share[-1] == 7 and share[1] == 7
        for r in set(range(rows)) - {1}:
            want, p, near = sample_ref(x[r, :vocab], u[r], 1.0)
            assert near < 1e-8 or got[r] == want
            if out:
                assert abs(share[r] - p) <= 2.0 ** -20
            else:
                assert share[r] == 7


# ------------------------------------------------------------------ together
@pytest.mark.parametrize("H,Hkv,hd,cap", [(4, 4, 64, 160), (8, 2, 128, 2112)])
def test_step_with_drafted_tokens(dev, ops, H, Hkv, hd, cap):
    """A verifying step of two layers as a program runs it: rotation of the drafted rows at their depths,
    the rows into the cache, the tree's attention, a token drawn at each node from logits, the
    accepted rows moved up; eagerly, then captured and replayed for further steps with eager work
    between. Every stage is checked against 64 bits on its own inputs."""
    rng = np.random.default_rng(cap)
    B, S, vocab, layers = 3, 11, 64, 2
    wq, wk = H * hd, Hkv * hd
    ld, scale = wq + 2 * wk, float(np.float32(hd ** -0.5))
    start = np.array([cap - 8 * S, 5, -1], np.int32)
    freq, factor = ops.rope_freqs(hd // 2, 10000.0, ("bands", 4, 1, 4, 512))
    caches, models, keep = [], [], []
    for _ in range(layers):
        c, m = filled(ops, rng, B, Hkv, cap, hd, np.maximum(start, 0))
        t, d = device_cache(dev, c)
        caches.append(d)
        models.append(m)
        keep.append(t)
    from sparrow_amd import _abi
    desc = (_abi.Kv4Cache * layers)(*caches)
    qkv = [dev.zeros(B * S, ld) for _ in range(layers)]
    out = [dev.zeros(B, S, wq) for _ in range(layers)]
    logits, u, temp = dev.zeros(B * S, vocab), dev.zeros(B * S), dev.up(np.full(B * S, 0.5, np.float32))
    top_p = dev.up(np.full(B * S, 0.9, np.float32))
    pos0, depth = dev.up(start), dev.zeros(B * S, dtype=np.int32)
    parent, drafted = dev.zeros(B, S, dtype=np.int32), dev.zeros(B, S, dtype=np.int32)
    token, prob = dev.zeros(B * S, dtype=np.int32), dev.zeros(B * S)
    path, kept, nxt = (dev.zeros(*s, dtype=np.int32) for s in ((B, S), (B,), (B,)))
    df = dev.up(freq)
    need = C.c_size_t()
    dev.check(dev.L.vmlm_hip_attention_tree_kv4_work(caches[0], H, S, C.byref(need)))
    work = dev.zeros(max(need.value, 16), dtype=np.uint8)
    dev.check(dev.L.vmlm_hip_sample_work(B * S, vocab, C.byref(need)))
    work2 = dev.zeros(max(need.value, 16), dtype=np.uint8)
    st = dev.stream()

    def step():
        for x, o, d in zip(qkv, out, caches):
            k = x.ptr + 4 * wq
            dev.check(dev.L.vmlm_hip_rope_qk(x.ptr, ld, k, ld, x.ptr, ld, k, ld, depth.ptr, df.ptr, B * S, H, Hkv,
                                             hd, hd // 2, True, factor, st))
            dev.check(dev.L.vmlm_hip_kv4_append(d, k, ld, k + 4 * wk, ld, pos0.ptr, None, S, st))
            dev.check(dev.L.vmlm_hip_attention_tree_kv4(d, x.ptr, ld, pos0.ptr, None, parent.ptr, S, o.ptr, wq, H,
                                                        scale, work.ptr, work.nbytes, st))
        dev.check(dev.L.vmlm_hip_sample(logits.ptr, vocab, u.ptr, temp.ptr, None, top_p.ptr, None, B * S, vocab,
                                        token.ptr, prob.ptr, work2.ptr, work2.nbytes, st))
        dev.check(dev.L.vmlm_hip_tree_accept_kv4(desc, layers, pos0.ptr, None, parent.ptr, drafted.ptr, token.ptr,
                                                 S, path.ptr, kept.ptr, nxt.ptr, st))

    def inputs(at):
        tree = np.stack([random_tree(rng, S, "late") for _ in range(B)])
        tree[:, 1:] = np.maximum(tree[:, 1:], 0)
        deep = np.zeros((B, S), np.int32)
        for t in range(1, S):
            deep[:, t] = deep[np.arange(B), tree[:, t]] + 1
        x = [rng.standard_normal((B * S, ld), dtype=np.float32) for _ in range(layers)]
        lg = rng.standard_normal((B * S, vocab), dtype=np.float32)
        draft = rng.integers(0, vocab, (B, S)).astype(np.int32)
        for b in range(B):  # most drafts are what the logits make likely
            for t in range(1, S):
                if rng.random() < 0.8:
                    lg[b * S + tree[b, t], draft[b, t]] += 6
        for buf, v in zip((*qkv, logits), (*x, lg)):
            buf.put(v)
        u.put(rng.random(B * S, dtype=np.float32))
        pos0.put(at)
        depth.put(np.where(at[:, None] >= 0, at[:, None] + deep, -1).reshape(-1).astype(np.int32))
        parent.put(tree)
        drafted.put(draft)
        return x, lg, tree, draft

    def check(at, x, lg, tree, draft):
        dev.check(dev.L.vmlm_hip_check_guards())
        dev.sync()
        dep = depth.get()
        rows = np.flatnonzero(dep >= 0)
        for n in range(layers):
            y = qkv[n].get()
            ref, tol = rope_ref(np.ascontiguousarray(x[n][:, :wq + wk]), dep, freq, hd, True, factor)
            assert (np.abs(y[:, :wq + wk] - ref)[rows] <= tol[rows]).all()
            y = y.reshape(B, S, ld)
            for b in np.flatnonzero(at >= 0):
                put(models[n], y[b, :, wq:wq + wk], y[b, :, wq + wk:], b, at[b], S, Hkv)
            check_tree(out[n].get(), tree_ref(models[n], np.ascontiguousarray(y[..., :wq]), at, [S] * B, tree, Hkv,
                                              hd, scale))
        tok, uu = token.get(), u.get()
        for r in range(B * S):
            want, _, near = sample_ref(lg[r], uu[r], 0.5, 0, 0.9, 0.0)
            assert near < 1e-8 or tok[r] == want
        hp, hk, hn = path.get(), kept.get(), nxt.get()
        moved = 0
        for b in np.flatnonzero(at >= 0):
            want, last = accept_ref(tree[b], draft[b], tok.reshape(B, S)[b], S)
            assert hp[b].tolist() == want + [-1] * (S - len(want)) and hk[b] == len(want) and hn[b] == last
            moved += want != list(range(len(want)))
            for m in models:
                for a in m.values():
                    a[b, :, at[b]:at[b] + len(want)] = a[b, :, at[b] + np.array(want)].swapaxes(0, 1).copy()
        for n in range(layers):  # what the caches hold now
            t, d = keep[n], caches[n]
            kd, vd = dev.zeros(B, S, wk), dev.zeros(B, S, wk)
            dev.check(dev.L.vmlm_hip_kv4_read(d, kd.ptr, wk, vd.ptr, wk, pos0.ptr, None, S, None))
            dev.sync()
            for b in np.flatnonzero(at >= 0):
                for got, name in ((kd, "k"), (vd, "v")):
                    want = models[n][name][b, :, at[b]:at[b] + S].swapaxes(0, 1).reshape(S, wk)
                    assert np.array_equal(got.get()[b], want)
        return np.where(at >= 0, at + hk, -1).astype(np.int32), moved

    got = inputs(start)
    dev.sync()
    step()
    at, moved = check(start, *got)
    graph = C.c_void_p()
    dev.check(dev.L.vmlm_hip_capture_begin(st))
    step()
    dev.check(dev.L.vmlm_hip_capture_end(st, C.byref(graph)))
    for _ in range(5):
        got = inputs(at)
        dev.sync()
        dev.check(dev.L.vmlm_hip_graph_launch(graph, st))
        at, more = check(at, *got)
        moved += more
    assert moved
    dev.check(dev.L.vmlm_hip_graph_destroy(graph))
