"""The 4-bit operators on the GPU where their arithmetic, their masks and their sizes
are at an edge, against their definitions in 64 bits.

Tolerances (u = 2^-24, half a step of f32), where no other is derived beside a test:
 * attention, per output channel: with p the weights, R the largest value that a
   position's 32 channels can hold and t a score's distance from the largest one,
   sum_p p R (e + mean e) where e = ds + (64 + n / 16 + 4 t) u. The score is off by
   ds = 33 u scale sum_g |q_g|_1 K_g over the groups g of 32 channels (K the largest
   value its key's group can hold): q to 2^-30 of its group's largest value, its sum, the
   products' conversions and the sums over groups, all below 33 roundings of that sum; 0
   where every step is exact. 4 t u is the exponent's product with log2(e) and its
   rounding; 64 u the exponential, the weights' fixed point (24 bits, and 2^-30 of the
   largest weight times scale of 128 positions, which is 3 u of sum_p p R), the
   conversions and the joins; n / 16 u the sums over the positions that a lane adds one
   after another."""
import ctypes as C

import numpy as np
import pytest
from test_gpu_4bit import (U, dev, device_cache, int4_case, int4_check, int4_ref,  # noqa: F401
                           new_model, nibbles, norm_ref, ops, put, same_cache)

pytestmark = pytest.mark.gpu


def spread(meta):
    """(min, scale) of each 32 channels, f64."""
    lo = (meta & np.uint32(0xFFFF0000)).view(np.float32).astype(np.float64)
    return lo, (meta << np.uint32(16)).view(np.float32).astype(np.float64)


def attn_exact(m, q, pos, Hkv, hd, scale, ds=True):
    """(out in 64 bits, its bound) for live rows; ds False: scores are exact in f32."""
    B, H = q.shape[0], q.shape[1] // hd
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    for b in range(B):
        n = pos[b] + 1
        for h in range(H if n > 0 else 0):
            kv, at = h // (H // Hkv), slice(h * hd, (h + 1) * hd)
            x = q[b, at].astype(np.float64)
            s = m["k"][b, kv, :n].astype(np.float64) @ x * scale
            t = s.max() - s
            p = np.exp(-t)
            p /= p.sum()
            most = []
            for name in ("km", "vm"):
                lo, sc = spread(m[name][b, kv, :n])
                most.append(np.maximum(np.abs(lo), np.abs(lo + 15 * sc)))
            e = (64 + n / 16 + 4 * t) * U
            if ds:
                e += 33 * U * abs(scale) * (most[0] @ np.abs(x).reshape(-1, 32).sum(1))
            out[b, at] = p @ m["v"][b, kv, :n].astype(np.float64)
            # (a weight below 2^-126 may be none)
            w = (p * (e + p @ e))[:, None] * most[1] + 2.0 ** -126 * most[1]
            tol[b, at] = np.repeat(w.sum(0), 32) + 2.0 ** -138
    return out, tol


def stored(ops, k, v, Hkv, cap):
    """Rows [B, n, Hkv * hd] in a cache and in its model."""
    B, n, hd = k.shape[0], k.shape[1], k.shape[2] // Hkv
    c, m = ops.Kv4Cache(B, Hkv, cap, hd), new_model(B, Hkv, cap, hd)
    c.append(k, v, np.zeros(B))
    for b in range(B):
        put(m, k[b], v[b], b, 0, n, Hkv)
    return c, m


def close(out, ref, tol):
    assert (np.abs(out - ref) <= tol).all(), (np.abs(out - ref) / tol).max()


# ------------------------------------------------------------------ attention
@pytest.mark.parametrize("times", [1e3, 1e6, 1e10, 1e20])
@pytest.mark.parametrize("H,Hkv,hd,n,at", [(1, 1, 64, 200, 77), (4, 1, 128, 130, 129), (2, 2, 32, 100, 0),
                                           (2, 1, 256, 90, 64), (7, 1, 64, 60, 59), (2, 2, 128, 2500, 1300)])
@pytest.mark.parametrize("append", [False, True])
def test_attention_value_that_no_query_attends(ops, H, Hkv, hd, n, at, times, append):
    """A value row that stands out at a position whose weight is nothing (e^-100):
    the others keep all their bits."""
    rng = np.random.default_rng(n + hd)
    base = rng.standard_normal((1, Hkv, 1, hd))
    q = (base + 0.1 * rng.standard_normal((1, Hkv, H // Hkv, hd))).astype(np.float32).reshape(1, -1)
    k, v = rng.standard_normal((2, 1, n, Hkv * hd), dtype=np.float32)
    scale = float(np.float32(hd ** -0.5))
    k[0, at] = (-100 / scale * base / (base * base).sum(-1, keepdims=True)).reshape(-1)
    v[0, at] *= np.float32(times)
    cap = -(-n // 32) * 32
    c, m = stored(ops, k, v, Hkv, cap)
    new = (k[:, -1], v[:, -1]) if append else ()
    if append:  # the last row again, by the attention itself
        c.k[:, :, n - 1] = 0
        c.k_meta[:, :, n - 1] = c.v_meta[:, :, n - 1] = 0x7FC07FC0
    out = c.attention_decode(q, [n - 1], *new)
    close(out, *attn_exact(m, q, [n - 1], Hkv, hd, scale))


@pytest.mark.parametrize("H,Hkv,hd", [(1, 1, 32), (1, 1, 64), (4, 1, 128), (3, 1, 256), (2, 1, 64)])
def test_attention_every_bit_of_the_weights(ops, H, Hkv, hd):
    """One position has nearly all the weight, and half of its channels hold an exact
    zero (u = 8, min = -8 scale): there the output is the sum of weights near 2^-15 of the
    largest, in fixed point below it. Off by half a step (2^-30 of the largest) each
    times a code up to 8, besides the roundings of the weights themselves; without their
    lowest byte it would be off by 1e-5, six times the bound."""
    rng = np.random.default_rng(hd)
    n = 60
    q = np.zeros((1, H, hd), np.float32)
    q[0, :, 0] = 8
    k = np.zeros((1, n, hd), np.float32)
    scale = 0.125
    k[0, 1:, 0] = -rng.uniform(9, 12, n - 1)
    v = rng.integers(-8, 8, (1, n, hd)).astype(np.float32)
    v[0, :, 0::32], v[0, :, 1::32] = -8, 7
    zero = np.arange(hd) % 2 == 0
    v[0, 0, zero & (np.arange(hd) % 32 > 1)] = 0
    c, m = stored(ops, k, v, Hkv, 64)
    assert np.array_equal(m["v"][0, 0, :n], v[0])
    out = c.attention_decode(q.reshape(1, -1), [n - 1], scale=scale).reshape(H, hd)
    ref, tol = attn_exact(m, q.reshape(1, -1), [n - 1], Hkv, hd, scale)
    close(out, ref.reshape(H, hd), tol.reshape(H, hd))
    see = v[0, 0] == 0
    s = m["k"][0, 0, :n, 0].astype(np.float64) * 8 * scale
    p = np.exp(s - s.max())
    p /= p.sum()
    e = (64 + n / 16 + 4 * 13 + 33 * 13) * U  # (a score is above -13)
    bound = (2 * e * p[1:].sum() + (n - 1) * 2.0 ** -30) * 8
    assert see.any() and np.abs(out - ref.reshape(H, hd))[:, see].max() <= bound


@pytest.mark.parametrize("H,Hkv,hd", [(1, 1, 64), (4, 1, 128), (2, 2, 256)])
@pytest.mark.parametrize("times", [1e4, 1e6, 1e12])
def test_attention_query_groups_of_other_magnitudes(ops, H, Hkv, hd, times):
    """Queries whose first 32 channels are large against keys that are small there (and
    the other way round in the last 32): each group's products keep their bits."""
    rng = np.random.default_rng(hd + H)
    n = 150
    q = rng.standard_normal((1, H, hd), dtype=np.float32)
    k, v = rng.standard_normal((2, 1, n, Hkv, hd), dtype=np.float32)
    q[..., :32] *= np.float32(times)
    k[..., :32] /= np.float32(times)
    q[..., -32:] /= np.float32(times)
    k[..., -32:] *= np.float32(times)
    c, m = stored(ops, k.reshape(1, n, -1), v.reshape(1, n, -1), Hkv, 160)
    q = q.reshape(1, -1)
    scale = float(np.float32(hd ** -0.5))
    close(c.attention_decode(q, [n - 1]), *attn_exact(m, q, [n - 1], Hkv, hd, scale))


@pytest.mark.parametrize("times", [1e-37, 1e-20, 1e20, 1e36])
def test_attention_tiny_and_huge_queries(ops, times):
    """Queries and keys at opposite ends of f32, with a group of zeros and a zero head."""
    rng = np.random.default_rng(21)
    n, hd = 70, 128
    q = rng.standard_normal((1, 3, hd), dtype=np.float32) * np.float32(times)
    q[:, :, 32:64] = 0
    q[:, 2] = 0
    k, v = rng.standard_normal((2, 1, n, hd), dtype=np.float32)
    k /= np.float32(times)
    c, m = stored(ops, k, v, 1, 96)
    q = q.reshape(1, -1)
    close(c.attention_decode(q, [n - 1], scale=0.125), *attn_exact(m, q, [n - 1], 1, hd, 0.125))


@pytest.mark.parametrize("q,k,scale", [(2.0 ** -138, 2.0 ** 127, 2.0 ** 20), (2.0 ** -122, 2.0 ** 122, -200.0),
                                       (2.0 ** 100, 2.0 ** -60, 2.0 ** -45), (1.0, 1.0, 0.0)])
def test_attention_any_scale_of_the_scores(ops, q, k, scale):
    """Scales that bring scores of a few out of queries and keys near f32's ends: no
    step between leaves f32."""
    rng = np.random.default_rng(22)
    n, hd = 70, 64
    x = (rng.standard_normal((1, 2 * hd)) * q / 8).astype(np.float32)
    y, v = rng.standard_normal((2, 1, n, hd), dtype=np.float32)
    y = (y.astype(np.float64) * k / 64).astype(np.float32)
    c, m = stored(ops, y, v, 1, 96)
    close(c.attention_decode(x, [n - 1], scale=scale), *attn_exact(m, x, [n - 1], 1, hd, scale))


@pytest.mark.parametrize("H,hd", [(1, 32), (1, 64), (4, 128), (3, 256)])
def test_attention_every_bit_of_the_queries(ops, H, hd):
    """Two channels of a group, 24 bits each, that nearly cancel against equal keys: the
    score is their difference, exact in every step."""
    rng = np.random.default_rng(hd)
    q = np.zeros((1, H, hd), np.float32)
    big = rng.integers(2 ** 23, 2 ** 24 - 2 ** 18, (H, hd // 32))
    q[0, :, 5::32] = big
    q[0, :, 20::32] = -(big - rng.integers(1, 4, big.shape))
    k = np.zeros((1, 3, hd), np.float32)
    k[0, 0, 5::32] = k[0, 0, 20::32] = 15
    k[0, 1, 5::32] = k[0, 1, 20::32] = 15
    k[0, 1, 3::32] = 1
    k[0, 2, 7::32] = 15
    v = rng.standard_normal((1, 3, hd), dtype=np.float32)
    c, m = stored(ops, k, v, 1, 32)
    assert np.array_equal(m["k"][0, 0, :3], k[0])
    q = q.reshape(1, -1)
    close(c.attention_decode(q, [2], scale=2.0 ** -7),
          *attn_exact(m, q, [2], 1, hd, 2.0 ** -7, ds=False))


@pytest.mark.parametrize("n", [129, 257, 300, 1025, 1200])
@pytest.mark.parametrize("H,Hkv,hd", [(1, 1, 64), (4, 1, 128), (2, 2, 32), (1, 1, 256)])
def test_attention_nan_keys_fill_a_chunk(ops, H, Hkv, hd, n):
    """Poisoned keys at every position of the last chunk, or of the first 128: the head
    is NaN, also where a wave has nothing else."""
    rng = np.random.default_rng(n)
    q = rng.standard_normal((1, H * hd), dtype=np.float32)
    for bad in (slice((n - 1) // 128 * 128, n), slice((n - 1) // 64 * 64, n), slice(0, 128)):
        k, v = rng.standard_normal((2, 1, n, Hkv * hd), dtype=np.float32)
        k[0, bad, 3::hd] = np.nan
        c = ops.Kv4Cache(1, Hkv, -(-n // 32) * 32, hd)
        c.append(k, v, [0])
        assert np.isnan(c.attention_decode(q, [n - 1])).all()


@pytest.mark.parametrize("B,Hkv,n", [(1, 1, 200), (16, 32, 1150), (1, 1, 5000)])
def test_attention_scores_of_minus_infinity(ops, B, Hkv, n):
    """Finite queries and keys whose product leaves f32 downwards at the first 128
    positions: those have no weight, as in f32."""
    rng = np.random.default_rng(n)
    hd, cap = 64, -(-n // 32) * 32
    q = rng.standard_normal((B, Hkv, hd), dtype=np.float32)
    q[..., 0] = 1e30
    k, v = rng.standard_normal((2, B, n, Hkv, hd), dtype=np.float32)
    k[..., :32] = 0
    k[:, :128, :, 0] = -1e30
    c, m = stored(ops, k.reshape(B, n, -1), v.reshape(B, n, -1), Hkv, cap)
    out = c.attention_decode(q.reshape(B, -1), [n - 1] * B)
    # the definition without those positions
    keep = slice(128, n)
    part = {x: y[:, :, keep] for x, y in m.items()}
    q[..., 0] = 0
    ref, tol = attn_exact(part, q.reshape(B, -1), [n - 129] * B, Hkv, hd, 0.125)
    close(out, ref, tol)


@pytest.mark.parametrize("H,Hkv,hd,n", [(1, 1, 64, 100), (4, 1, 128, 300), (2, 2, 32, 60), (2, 1, 256, 200),
                                        (1, 1, 64, 3000)])
def test_attention_scores_far_from_zero(ops, H, Hkv, hd, n):
    """Scores of 15360 and a few more, exact in f32: the weights depend on their
    differences, so that log2(e) must not round the scores themselves."""
    rng = np.random.default_rng(n)
    q = np.zeros((1, H, hd), np.float32)
    q[..., 0], q[..., 1] = 8192, 8
    k = np.zeros((1, n, Hkv, hd), np.float32)
    k[..., 0] = 15
    k[..., 1] = rng.integers(0, 6, (1, n, Hkv))
    v = rng.standard_normal((1, n, Hkv * hd), dtype=np.float32)
    c, m = stored(ops, k.reshape(1, n, -1), v, Hkv, -(-n // 32) * 32)
    assert np.array_equal(m["k"][0, :, :n], k[0].transpose(1, 0, 2))
    q = q.reshape(1, -1)
    close(c.attention_decode(q, [n - 1], scale=0.125),
          *attn_exact(m, q, [n - 1], Hkv, hd, 0.125, ds=False))


# ------------------------------------------------------------------ the cache
def nan_of(bits):
    return np.array([bits], np.uint32).view(np.float32)[0]


@pytest.mark.parametrize("bits", [0x7FC00000, 0xFFC00000, 0x7F800001, 0x7FFFFFFF, 0xFF800001, 0xFFFF0000,
                                  0xFFFF0001, 0xFFFFFFFF])
def test_cache_any_nan_poisons(ops, bits):
    """Every NaN, whatever its bits, and also 32 of them, gives NaN in its 32 channels
    alone; the same for a row that the attention appends."""
    rng = np.random.default_rng(6)
    x = rng.standard_normal((1, 4, 128), dtype=np.float32)
    x.view(np.uint32)[0, 0, 5] = bits
    x.view(np.uint32)[0, 1, 32:64] = bits
    x.view(np.uint32)[0, 2, 64] = bits
    poisoned = np.zeros((1, 4, 128), bool)
    poisoned[0, 0, :32] = poisoned[0, 1, 32:64] = poisoned[0, 2, 64:96] = True
    c = ops.Kv4Cache(1, 1, 32, 128)
    c.append(x, x, [0])
    for y in c.read([0], 4):
        assert np.isnan(y[poisoned]).all() and np.isfinite(y[~poisoned]).all()
    q = rng.standard_normal((1, 128), dtype=np.float32)
    for at in range(3):
        good = rng.standard_normal((1, 128), dtype=np.float32)
        c = ops.Kv4Cache(1, 1, 32, 128)
        out = c.attention_decode(q, [0], good, x[:, at])
        assert np.isnan(out[poisoned[:, at]]).all() and np.isfinite(out[~poisoned[:, at]]).all()
        c = ops.Kv4Cache(1, 1, 32, 128)
        assert np.isnan(c.attention_decode(q, [0], x[:, at], good)).all()


def test_cache_no_rows_to_drop(ops):
    """A sequence without a row trips no guard, wherever its first position lies."""
    c = ops.Kv4Cache(2, 1, 64, 64)
    x = np.ones((2, 3, 64), np.float32)
    c.append(x, x, [1000, 5], [0, 3])
    c.append(x, x, [2 ** 31 - 1, 5], [-4, 3])
    k, _ = c.read([65, 5], 3, [0, 3])
    assert not k[0].any() and (k[1] == 1).all()


# ------------------------------------------------------------------ the cache's end
@pytest.mark.parametrize("at", [60, 63, 64, 1000, 2 ** 31 - 1])
@pytest.mark.parametrize("append", [True, False])
def test_cache_rows_up_to_the_capacity(ops, at, append):
    """Of rows that run past cap the ones before it are stored, and read; the others
    are dropped and reported, and no other sequence sees it."""
    from sparrow_amd import VmlmError
    rng = np.random.default_rng(at % 1000)
    c, m = ops.Kv4Cache(2, 1, 64, 64), new_model(2, 1, 64, 64)
    k, v = rng.standard_normal((2, 2, 10, 64), dtype=np.float32)
    fit = max(0, min(10, 64 - at))
    where = np.zeros((2, 64), bool)
    for b, (p, n) in enumerate(((at, fit), (20, 10))):
        put(m, k[b], v[b], b, p, n, 1)
        where[b, p:p + n] = True
    if append:
        with pytest.raises(VmlmError) as e:
            c.append(k, v, [at, 20])
        assert e.value.code == 9
        same_cache(c, m, where)
        return
    c.append(k, v, [at, 20], [fit, 10])
    rk = np.full((2, 10, 64), 3, np.float32)
    rv, pos = rk.copy(), np.array([at, 20], np.int32)
    p = [x.ctypes.data_as(C.c_void_p) for x in (rk, rv, pos)]
    from sparrow_amd import lib
    assert lib().vmlm_kv4_read(c.descriptor(), *p, None, 10) == 9
    for got, name in ((rk, "k"), (rv, "v")):
        assert np.array_equal(got[0, :fit], m[name][0, 0, at:at + fit] if fit else got[0, :0])
        assert (got[0, fit:] == 3).all()
        assert np.array_equal(got[1], m[name][1, 0, 20:30])


# ------------------------------------------------------------------ a prompt, then its decode
def test_prompt_then_decode(dev, ops):
    """A prompt as the documentation has it, for as many kv heads as heads: the head
    norms alone for the prefill attention, which rotates; norm and rotation for the cache's
    rows; then decode steps over the cache. The prefill's outputs are checked against the
    rotated rows' attention, the cache's rows against the rotated rows, and the
    decode steps against 64 bits over what the cache holds."""
    rng = np.random.default_rng(17)
    H, hd, S, steps, cap, theta = 3, 64, 70, 4, 96, 10000.0
    w, scale = H * hd, 0.125
    x = rng.standard_normal((S + steps, 3 * w), dtype=np.float32)  # fused q, k, v
    g = (1 + rng.standard_normal((2, hd)) / 8).astype(np.float32)
    pos = np.arange(S + steps, dtype=np.int32)
    q, k, v = np.split(x, 3, 1)
    rot = [norm_ref(t, gg, pos, hd, 1e-5, theta)[0] for t, gg in ((q, g[0]), (k, g[1]))]
    dx, dg, dp = dev.up(x), dev.up(g), dev.up(pos)
    nq, nk, rk, out, vv = (dev.zeros(S, w) for _ in range(5))
    vv.put(v[:S])
    c = ops.Kv4Cache(1, H, cap, hd)
    keep, d = device_cache(dev, c)
    zero = dev.up(np.zeros(1, np.int32))
    dev.sync()

    def norm(qo, ko, first, rows, at):
        src = dx.ptr + first * 12 * w
        dev.check(dev.L.vmlm_hip_qk_norm_rope(qo.ptr, w, ko.ptr, w, src, 3 * w, src + 4 * w, 3 * w,
                                              dg.ptr, dg.ptr + 4 * hd, at, rows, H, H, hd, 1e-5, theta,
                                              None))
    norm(nq, nk, 0, S, None)
    dev.check(dev.L.vmlm_hip_attention_prefill(nq.ptr, nk.ptr, vv.ptr, out.ptr, S, H, hd, theta, 0,
                                               scale, True, None))
    norm(nq, rk, 0, S, dp.ptr)
    dev.check(dev.L.vmlm_hip_kv4_append(d, rk.ptr, w, dx.ptr + 8 * w, 3 * w, zero.ptr, None, S, None))
    dev.sync()
    got = out.get().astype(np.float64)
    for h in range(H):
        at = slice(h * hd, (h + 1) * hd)
        s = rot[0][:S, at] @ rot[1][:S, at].T * scale
        s = np.where(np.tril(np.ones((S, S), bool)), s, -np.inf)
        p = np.exp(s - s.max(1, keepdims=True))
        ref = p / p.sum(1, keepdims=True) @ v[:S, at].astype(np.float64)
        # the prefill's own bound: bf16 terms, 1e-4 of the RMS
        assert np.abs(got[:, at] - ref).max() <= 1e-4 * np.sqrt((ref ** 2).mean())
    m = new_model(1, H, cap, hd)
    hk = rk.get()
    close(hk, rot[1][:S], norm_ref(k[:S], g[1], pos[:S], hd, 1e-5, theta)[1])
    put(m, hk, v[:S], 0, 0, S, H)
    sq, sk, so = (dev.zeros(1, w) for _ in range(3))
    for i in range(S, S + steps):
        norm(sq, sk, i, 1, dp.ptr + 4 * i)
        dev.check(dev.L.vmlm_hip_attention_decode_kv4(
            d, sq.ptr, w, sk.ptr, dx.ptr + i * 12 * w + 8 * w, w, dp.ptr + 4 * i, so.ptr, w, H, scale,
            None, 0, None))
        dev.sync()
        put(m, sk.get(), v[i:i + 1], 0, i, 1, H)
        close(so.get(), *attn_exact(m, sq.get(), [i], H, hd, scale))


# ------------------------------------------------------------------ sizes past a launch's grid
def test_norm_rows_past_one_grid(dev):
    """More rows than a grid of 256 threads a row can have."""
    rng = np.random.default_rng(7)
    rows, hd, tile = (1 << 24) + 5, 8, 1 << 18
    x = rng.standard_normal((tile, hd), dtype=np.float32)
    p = rng.integers(0, 1000, tile).astype(np.int32)
    reps = -(-rows // tile)
    q, pos = (dev.up(np.concatenate([t] * reps)[:rows]) for t in (x, p))
    g = np.ones(hd, np.float32)
    dg, out = dev.up(g), dev.zeros(rows + 1, hd)
    dev.sync()
    dev.check(dev.L.vmlm_hip_qk_norm_rope(out.ptr, hd, None, 0, q.ptr, hd, None, 0, dg.ptr, None,
                                          pos.ptr, rows, 1, 0, hd, 1e-5, 1e4, None))
    dev.sync()
    got = out.get()
    assert not got[rows].any()
    ref, tol = norm_ref(x, g, p, hd, 1e-5, 1e4)
    for i in range(reps):
        part = got[i * tile:min(rows, (i + 1) * tile)]
        assert (np.abs(part - ref[:len(part)]) <= tol[:len(part)]).all(), i


def test_int4_rows_past_one_grid(dev):
    """More rows than the grid of the launch that splits them can have."""
    rng = np.random.default_rng(8)
    m, n, k, group, tile = (1 << 24) + 16, 16, 32, 64, 1 << 18
    a, w, s = int4_case(rng, tile, n, k, group)
    p = C.c_void_p()
    for count in (m * k, m * n + n):
        dev.check(dev.L.vmlm_hip_malloc(C.byref(p), count * 4))
        dev.bufs.append(p.value)
    pa, pc = dev.bufs[-2:]
    for r in range(0, m, tile):
        part = a[:min(tile, m - r)]
        dev.check(dev.L.vmlm_hip_memcpy_h2d(pa + r * k * 4, part.ctypes.data, part.nbytes))
    mark = np.full(n, 5, np.float32)
    dev.check(dev.L.vmlm_hip_memcpy_h2d(pc + m * n * 4, mark.ctypes.data, mark.nbytes))
    dw, ds = dev.up(w), dev.up(s)
    dev.sync()
    dev.check(dev.L.vmlm_hip_gemm_nt_int4(pa, dw.ptr, ds.ptr, pc, m, n, k, group, None))
    dev.sync()
    got = np.empty((m + 1, n), np.float32)
    dev.check(dev.L.vmlm_hip_memcpy_d2h(got.ctypes.data, pc, got.nbytes))
    assert (got[m] == 5).all()
    int4_check(got[:tile], a, w, s, group)
    for r in range(tile, m, tile):
        part = got[r:min(m, r + tile)]
        assert np.array_equal(part, got[:len(part)]), r


# ------------------------------------------------------------------ norms
def test_norm_alone_keeps_channels_apart(ops):
    """Without positions nothing is rotated: a channel whose gain or value is not
    finite leaves its partner in the other half as it is."""
    rng = np.random.default_rng(9)
    q = rng.standard_normal((2, 64), dtype=np.float32)
    g = np.ones(64, np.float32)
    g[3], g[40] = np.inf, np.nan
    got, _ = ops.qk_norm_rope(q, q[:, :0], g, g, None, 64)
    finite = np.ones(64, np.float32)
    ref, tol = norm_ref(q, finite, None, 64, 1e-5, 1e4)
    ok = np.isfinite(g)
    assert (np.abs(got - ref)[:, ok] <= tol[:, ok]).all()
    assert np.isinf(got[:, 3]).all() and np.isnan(got[:, 40]).all()


# ------------------------------------------------------------------ gemm_nt_int4
# In place with one, two and four tiles of columns, and over byte planes, with groups
# that end inside a wave's share of K.
PATHS = [(1, 50, 384, 128), (3, 70, 640, 32), (7, 5000, 256, 64), (1, 33000, 256, 64), (20, 40, 352, 32),
         (20, 5100, 384, 128), (21, 5100, 1280, 384), (18, 3500, 320, 64), (40, 2600, 3328, 640)]


@pytest.mark.parametrize("m,n,k,group", PATHS)
def test_int4_every_bit(ops, m, n, k, group):
    """One power of two in each weight row: the product is one activation times it, so
    all 24 bits come back. (Activations within 2^-6 of a power of two are left
    out: with the term that makes their bytes signed they need 25.)"""
    rng = np.random.default_rng(m * n + k)
    a = rng.integers(2 ** 23, 2 ** 24 - 2 ** 18, (m, k)) * rng.choice([-1, 1], (m, k))
    runs = -(-k // 128)
    a = a * np.repeat(2.0 ** rng.integers(-60, 20, (m, runs)), 128, 1)[:, :k]
    a = a.astype(np.float32)
    at, v = rng.integers(0, k, n), rng.choice([-8, -4, -1, 1, 2, 4], n)
    w = np.zeros((n, k), np.int8)
    w[np.arange(n), at] = v
    s = 2.0 ** rng.integers(-6, 7, (n, -(-k // group)))
    u = (w & 15).astype(np.uint8)
    got = ops.gemm_nt_int4(a, u[:, 0::2] | (u[:, 1::2] << 4), s, group)
    want = a[:, at].astype(np.float64) * (v * s[np.arange(n), at // group])
    assert np.array_equal(got, want)


@pytest.mark.parametrize("m,n,k,group", PATHS)
def test_int4_norm_of_the_error(ops, m, n, k, group):
    """Roundings of both signs: the split rounds each activation once (half a step, 0.3
    u in the mean of a uniform one), each run's sum is rounded at most five times and its
    addition once more, at the partial sums' magnitude, so the error is below
    sqrt(0.3 + 5 + k / 256) u of the result's norm, 4.5 u at k = 3328. Without the lowest two
    of the four bytes it would be 2^-16."""
    rng = np.random.default_rng(m + n * k)
    a, q, s = int4_case(rng, m, n, k, group)
    ref, _ = int4_ref(a, q, s, group)
    err = np.linalg.norm(ops.gemm_nt_int4(a, q, s, group) - ref)
    assert err <= (0.3 + 5 + k / 256) ** 0.5 * U * np.linalg.norm(ref)


@pytest.mark.parametrize("m,n,k,group", PATHS)
def test_int4_wide_rows(ops, m, n, k, group):
    """Rows from 1e-30 to 1e30, values that stand out by 1e4, a zero row and zero runs."""
    rng = np.random.default_rng(m + k)
    a, q, s = int4_case(rng, m, n, k, group)
    a[:, 5::97] *= np.float32(1e4)
    a *= np.float32(10.0) ** rng.integers(-30, 31, (m, 1)).astype(np.float32)
    a[0, 128:300] = 0
    a[m // 2] = 0
    got = ops.gemm_nt_int4(a, q, s, group)
    int4_check(got, a, q, s, group)
    assert not got[m // 2].any()


@pytest.mark.parametrize("m,n,k,group", [p for p in PATHS if p[0] > 2])
def test_int4_rows_that_are_not_finite(ops, m, n, k, group):
    """An infinity gives +-inf by its weight's sign (NaN against a zero weight), a
    NaN gives NaN; the other rows do not see them."""
    rng = np.random.default_rng(m * k)
    a, q, s = int4_case(rng, m, n, k, group)
    clean = ops.gemm_nt_int4(a, q, s, group)
    a[0, 130], a[1, 7], a[m - 1, k - 1] = np.inf, np.nan, -np.inf
    got = ops.gemm_nt_int4(a, q, s, group)
    w = nibbles(q).astype(np.float32)
    with np.errstate(invalid="ignore"):
        assert np.array_equal(got[0], np.float32(np.inf) * w[:, 130], equal_nan=True)
        assert np.array_equal(got[m - 1], -np.float32(np.inf) * w[:, k - 1], equal_nan=True)
    assert np.isnan(got[1]).all() and np.array_equal(got[2:m - 1], clean[2:m - 1])


@pytest.mark.parametrize("m,n,k,group", PATHS)
def test_int4_odd_addresses(dev, m, n, k, group):
    """Operands at odd addresses (the codes at any byte); what lies beside C stays."""
    rng = np.random.default_rng(m + n)
    a, q, s = int4_case(rng, m, n, k, group)
    buf = lambda x, pad: dev.up(np.concatenate([np.full(pad, 77, x.dtype), x.ravel()]))  # noqa: E731
    da, dq, ds = buf(a, 1), buf(q, 5), buf(s, 3)
    dc = dev.up(np.full(m * n + 10, 5.0, np.float32))
    dev.sync()
    dev.check(dev.L.vmlm_hip_gemm_nt_int4(da.ptr + 4, dq.ptr + 5, ds.ptr + 12, dc.ptr + 20, m, n, k,
                                          group, None))
    dev.sync()
    got = dc.get()
    assert (got[:5] == 5).all() and (got[5 + m * n:] == 5).all()
    int4_check(got[5:5 + m * n].reshape(m, n), a, q, s, group)
