"""The 4-bit operators on the GPU against their definitions in 64 bits.

Tolerances (u = 2^-24, half a step of f32):
 * int4 GEMM: an activation enters with an error of at most u times the largest of its
   128 neighbours; within 128 k the products are exact, the result of each is
   rounded a few times and the K/128 of them added. The bound (K/32 + 48) * u *
   sum(max|x| of the 128 * |w|) also covers an f32 sum in runs of 32.
 * norm and rotation: the sum of squares and its root 10 u (half of its relative
   error counts), three products and the rotation's sum 6 u, sine and cosine 4 u of
   their own and 2 pi u of the f32 angle, against the pair's length: 32 u.
 * cache: codes, meta and values are equal bit for bit (the definition is f32).
 * attention: a score is off by ds = (32 + hd/8) u scale sum|q||k| (q in 31 bits below
   its largest, a sum over hd/32 groups of exact products), a weight by twice that
   and the exponential's few u, and the sums over n positions by (n/128 + 64) u of the
   largest |v|: (4 ds + (n/128 + 64) u) * max|v|."""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.fixture(scope="module")
def ops(hip):
    from sparrow_amd import ops
    return ops


class Buf:
    """An array in device memory."""

    def __init__(self, dev, a):
        a = np.ascontiguousarray(a)
        self.dev, self.shape, self.dtype, self.nbytes = dev, a.shape, a.dtype, a.nbytes
        p = C.c_void_p()
        dev.check(dev.L.vmlm_hip_malloc(C.byref(p), max(a.nbytes, 16)))
        self.ptr = p.value
        dev.bufs.append(self.ptr)
        self.put(a)

    def put(self, a):
        a = np.ascontiguousarray(a, self.dtype)
        assert a.shape == self.shape
        self.dev.check(self.dev.L.vmlm_hip_memcpy_h2d(self.ptr, a.ctypes.data, a.nbytes))

    def get(self):
        out = np.empty(self.shape, self.dtype)
        self.dev.check(self.dev.L.vmlm_hip_memcpy_d2h(out.ctypes.data, self.ptr, out.nbytes))
        return out


class Dev:
    """Device memory and streams through the library (and the HIP runtime under it)."""

    def __init__(self, lib, check):
        self.L, self.check, self.bufs, self.streams = lib, check, [], []

    def up(self, a):
        return Buf(self, a)

    def zeros(self, *shape, dtype=np.float32):
        return Buf(self, np.zeros(shape, dtype))

    def stream(self):
        st = C.c_void_p()
        assert self.L.hipStreamCreateWithFlags(C.byref(st), 1) == 0
        self.streams.append(st)
        return st

    def sync(self):
        assert self.L.hipDeviceSynchronize() == 0

    def free(self):
        self.sync()
        for st in self.streams:
            self.L.hipStreamDestroy(st)
        for p in self.bufs:
            self.L.vmlm_hip_free(p)


@pytest.fixture
def dev(hip):
    import sparrow_amd
    sparrow_amd.init(0)
    d = Dev(hip, sparrow_amd.check)
    yield d
    d.free()


# ------------------------------------------------------------------ gemm_nt_int4
def nibbles(b):
    u = np.stack((b & 15, b >> 4), -1).reshape(*b.shape[:-1], -1)
    return (u.astype(np.int8) ^ 8) - 8


def int4_case(rng, m, n, k, group):
    a = rng.standard_normal((m, k), dtype=np.float32)
    q = rng.integers(0, 256, size=(n, k // 2), dtype=np.uint8)
    s = np.abs(rng.standard_normal((n, -(-k // group)), dtype=np.float32)) * np.float32(0.003)
    return a, q, s + np.float32(1e-5)


def int4_ref(a, q, s, group):
    """(C in 64 bits, its bound)."""
    k = a.shape[1]
    w = nibbles(q).astype(np.float64) * np.repeat(s.astype(np.float64), group, 1)[:, :k]
    x = np.abs(a).astype(np.float64)
    run = -(-k // 128)
    top = np.zeros((a.shape[0], run * 128))
    top[:, :k] = x
    top = np.repeat(top.reshape(-1, run, 128).max(-1), 128, 1)[:, :k]
    return a.astype(np.float64) @ w.T, (k / 32 + 48) * U * (top @ np.abs(w).T)


def int4_check(got, a, q, s, group):
    ref, tol = int4_ref(a, q, s, group)
    bad = np.abs(got - ref) > tol
    assert not bad.any(), (np.argwhere(bad)[:4], (np.abs(got - ref) / tol).max())


SHAPES = [(1, 1, 32, 32), (1, 16, 128, 128), (1, 2304, 2304, 128), (2, 17, 96, 64),
          (3, 33, 160, 32), (4, 130, 992, 64), (5, 48, 256, 128), (7, 100, 5760, 32),
          (16, 1537, 992, 32), (16, 64, 5760, 64), (16, 2304, 2304, 128), (17, 100, 416, 128),
          (33, 96, 1024, 256), (100, 200, 704, 1024), (129, 40, 64, 32), (1, 20000, 2304, 64),
          (8, 20011, 512, 128), (300, 300, 288, 64), (2, 5, 32, 1 << 40)]


@pytest.mark.parametrize("m,n,k,group", SHAPES)
def test_int4(ops, m, n, k, group):
    rng = np.random.default_rng(m + n + k)
    a, q, s = int4_case(rng, m, n, k, min(group, 1024))
    s = s[:, :-(-k // group)]
    int4_check(ops.gemm_nt_int4(a, q, s, group), a, q, s, min(group, 1024))


@pytest.mark.parametrize("m", [1, 6, 40])
def test_int4_integers_are_exact(ops, m):
    """Integer activations and power-of-two scales: every sum is a small integer."""
    rng = np.random.default_rng(1)
    a, q, s = int4_case(rng, m, 50, 384, 64)
    a = rng.integers(-100, 101, a.shape).astype(np.float32)
    s[:] = np.float32(2.0) ** rng.integers(-3, 4, s.shape)
    assert np.array_equal(ops.gemm_nt_int4(a, q, s, 64), int4_ref(a, q, s, 64)[0])


@pytest.mark.parametrize("m,group", [(1, 128), (5, 32), (16, 64), (20, 128)])
def test_int4_magnitudes(ops, m, group):
    """Rows from 1e-30 to 1e30, values that stand out by 1e4, a zero row and
    runs of zeros."""
    rng = np.random.default_rng(2)
    a, q, s = int4_case(rng, m, 70, 640, group)
    a[:, 5::97] *= np.float32(1e4)
    a *= np.float32(10.0) ** rng.integers(-30, 31, (m, 1)).astype(np.float32)
    a[0, 128:300] = 0
    if m > 1:
        a[1] = 0
    got = ops.gemm_nt_int4(a, q, s, group)
    int4_check(got, a, q, s, group)
    assert m == 1 or not got[1].any()


@pytest.mark.parametrize("m,group", [(1, 128), (3, 32), (16, 64), (18, 256)])
def test_int4_nonfinite(ops, m, group):
    """An infinity gives +-inf by its weight's sign (NaN against a zero weight), a
    NaN gives NaN; the other rows do not see it."""
    rng = np.random.default_rng(3)
    a, q, s = int4_case(rng, m, 40, 320, group)
    clean = ops.gemm_nt_int4(a, q, s, group)
    a[0, 130] = np.inf
    if m > 2:
        a[2, 7] = np.nan
        a[m - 1, 300] = -np.inf
    got = ops.gemm_nt_int4(a, q, s, group)
    w = nibbles(q).astype(np.float32)
    with np.errstate(invalid="ignore"):
        want = np.float32(np.inf) * w[:, 130]
        assert np.array_equal(got[0], want, equal_nan=True)
        if m > 2:
            assert np.isnan(got[2]).all()
            if m > 3:  # of three rows the last one holds the NaN too
                assert np.array_equal(got[m - 1], -np.float32(np.inf) * w[:, 300], equal_nan=True)
            rest = [i for i in range(m) if i not in (0, 2, m - 1)]
            assert np.array_equal(got[rest], clean[rest])


def test_int4_k_zero(ops):
    c = ops.gemm_nt_int4(np.zeros((2, 0), np.float32), np.zeros((3, 0), np.uint8),
                         np.zeros((3, 0), np.float32), 128)
    assert c.shape == (2, 3) and not c.any()


@pytest.mark.parametrize("m,n,k,group", [(1, 37, 352, 32), (9, 50, 384, 128), (40, 33, 128, 64)])
def test_int4_alignment_and_bounds(dev, m, n, k, group):
    """Operands at odd addresses (the codes at any byte); what lies beside C stays."""
    rng = np.random.default_rng(4)
    a, q, s = int4_case(rng, m, n, k, group)
    buf = lambda x, pad: dev.up(np.concatenate([np.full(pad, 77, x.dtype), x.ravel()]))  # noqa: E731
    da, dq, ds = buf(a, 1), buf(q, 3), buf(s, 3)
    dc = dev.up(np.full(m * n + 10, 5.0, np.float32))
    dev.sync()
    dev.check(dev.L.vmlm_hip_gemm_nt_int4(da.ptr + 4, dq.ptr + 3, ds.ptr + 12,
                                          dc.ptr + 20, m, n, k, group, None))
    dev.sync()
    got = dc.get()
    assert (got[:5] == 5).all() and (got[5 + m * n:] == 5).all()
    int4_check(got[5:5 + m * n].reshape(m, n), a, q, s, group)


def test_int4_two_streams(dev):
    """Calls at once on streams of their own give what they give alone."""
    rng = np.random.default_rng(5)
    jobs = []
    # (the last one's rows go through the stream's workspace)
    for m, n, k, group in ((1, 2304, 2304, 128), (16, 5760, 2304, 64), (70, 2304, 1024, 128),
                           (70, 2400, 1000 // 32 * 32, 64)):
        a, q, s = int4_case(rng, m, n, k, group)
        jobs.append((dev.stream(), dev.up(a), dev.up(q), dev.up(s),
                     [dev.zeros(m, n) for _ in range(20)], (m, n, k, group)))
    dev.sync()
    for i in range(20):
        for st, a, q, s, c, dims in jobs:
            dev.check(dev.L.vmlm_hip_gemm_nt_int4(a.ptr, q.ptr, s.ptr,
                                                  c[i].ptr, *dims, st))
    dev.sync()
    for st, a, q, s, c, dims in jobs:
        one = c[0].get()
        int4_check(one, a.get(), q.get(), s.get(), dims[3])
        for x in c[1:]:
            assert np.array_equal(x.get(), one)


@pytest.mark.parametrize("m,n,group", [(3, 500, 32), (16, 700, 128), (40, 5000, 128), (70, 3000, 64)])
def test_int4_captured(dev, m, n, group):
    """Captured calls take no workspace (two graphs may run at once) and agree with the
    definition on every replay, with eager calls of the same stream between them."""
    rng = np.random.default_rng(6)
    a, q, s = int4_case(rng, m, n, 416, group)
    da, dq, ds, dc, de = dev.up(a), dev.up(q), dev.up(s), dev.zeros(m, n), dev.zeros(m, n)
    st, graph = dev.stream(), C.c_void_p()

    def call(c):
        dev.check(dev.L.vmlm_hip_gemm_nt_int4(da.ptr, dq.ptr, ds.ptr, c.ptr, m, n, 416, group, st))
    call(dc)
    dev.check(dev.L.vmlm_hip_capture_begin(st))
    call(dc)
    dev.check(dev.L.vmlm_hip_capture_end(st, C.byref(graph)))
    for i in range(3):
        a = rng.standard_normal(a.shape, dtype=np.float32)
        dev.sync()
        da.put(a)
        dc.put(np.zeros((m, n)))
        dev.check(dev.L.vmlm_hip_graph_launch(graph, st))
        call(de)
        dev.sync()
        int4_check(dc.get(), a, q, s, group)
        int4_check(de.get(), a, q, s, group)
    dev.check(dev.L.vmlm_hip_graph_destroy(graph))


# ------------------------------------------------------------------ qk_norm_rope
def norm_ref(x, g, pos, hd, eps, theta):
    x = x.astype(np.float64).reshape(x.shape[0], -1, hd)
    y = x / np.sqrt((x * x).mean(-1, keepdims=True) + np.float32(eps)) * g
    i = np.arange(hd // 2)
    a = (np.zeros(len(x)) if pos is None else pos).astype(np.float64)[:, None, None] * \
        float(np.float32(theta)) ** (-2.0 * i / hd)
    lo, hi = y[..., :hd // 2], y[..., hd // 2:]
    r = np.concatenate((lo * np.cos(a) - hi * np.sin(a), lo * np.sin(a) + hi * np.cos(a)), -1)
    tol = 32 * U * np.tile(np.hypot(lo, hi), 2)
    return r.reshape(x.shape[0], -1), tol.reshape(x.shape[0], -1)


@pytest.mark.parametrize("rows,H,Hkv,hd", [(1, 36, 36, 64), (1, 1, 0, 8), (2, 0, 3, 16), (5, 4, 2, 80),
                                           (3, 8, 1, 128), (7, 3, 3, 32), (2, 5, 1, 256),
                                           (3, 2, 2, 96), (2, 1, 1, 512), (33, 32, 8, 128),
                                           (200, 36, 36, 64), (2, 100, 7, 24)])
@pytest.mark.parametrize("far", [0, 1 << 20])
def test_norm(ops, rows, H, Hkv, hd, far):
    rng = np.random.default_rng(rows + H + hd)
    q = rng.standard_normal((rows, H * hd), dtype=np.float32) * np.float32(3)
    k = rng.standard_normal((rows, Hkv * hd), dtype=np.float32)
    gq, gk = (1 + rng.standard_normal((2, hd), dtype=np.float32) / 4)
    pos = (rng.integers(0, 2000, rows) + far).astype(np.int32)
    for p in (pos, None):
        got = ops.qk_norm_rope(q, k, gq, gk, p, hd, theta=10000.0)
        for y, x, g in zip(got, (q, k), (gq, gk)):
            ref, tol = norm_ref(x, g, p, hd, 1e-5, 10000.0)
            assert (np.abs(y - ref) <= tol).all(), (np.abs(y - ref) / tol).max()


def test_norm_values(ops):
    """A zero head stays zero, a tiny one is governed by eps, a NaN or an infinity
    stays in its head."""
    rng = np.random.default_rng(1)
    q = rng.standard_normal((4, 2 * 64), dtype=np.float32)
    q[0, :64] = 0
    q[1, :64] *= np.float32(1e-12)
    q[2, 3] = np.nan
    q[3, 70] = np.inf
    one, pos = np.ones(64, np.float32), np.arange(4, dtype=np.int32)
    got, _ = ops.qk_norm_rope(q, q, one, one, pos, 64)
    assert not got[0, :64].any() and np.isfinite(got[:2]).all()
    ref, tol = norm_ref(q[:2], one, pos[:2], 64, 1e-5, 10000.0)
    assert (np.abs(got[:2] - ref) <= tol).all()
    assert np.isnan(got[2, :64]).all() and np.isfinite(got[2, 64:]).all()
    assert not np.isfinite(got[3, 64:]).all() and np.isfinite(got[3, :64]).all()


@pytest.mark.parametrize("inplace", [False, True])
def test_norm_strides_idle_rows_and_bounds(dev, inplace):
    """q and k inside fused rows of an odd stride, outputs likewise or in place; rows
    with a negative position, v and the padding stay as they were."""
    rng = np.random.default_rng(2)
    rows, H, Hkv, hd, ld = 6, 3, 1, 64, 3 * 64 + 2 * 64 + 5
    x = rng.standard_normal(1 + rows * ld, dtype=np.float32)
    g = (1 + rng.standard_normal((2, hd)) / 4).astype(np.float32)
    pos = np.array([5, -1, 0, 77, -3, 2 ** 31 - 1], np.int32)
    dx, dg, dp = dev.up(x), dev.up(g), dev.up(pos)
    do = dx if inplace else dev.up(np.full_like(x, 9.0))
    base, out = dx.ptr + 4, do.ptr + 4
    dev.sync()
    dev.check(dev.L.vmlm_hip_qk_norm_rope(out, ld, out + 4 * H * hd, ld, base, ld,
                                          base + 4 * H * hd, ld, dg.ptr,
                                          dg.ptr + 4 * hd, dp.ptr, rows, H, Hkv, hd,
                                          1e-5, 1e4, None))
    dev.sync()
    got, m = do.get()[1:].reshape(rows, ld), x[1:].reshape(rows, ld)
    was = m if inplace else np.full_like(m, 9.0)
    assert do.get()[0] == (x[0] if inplace else 9.0)
    w = (H + Hkv) * hd
    assert np.array_equal(got[:, w:], was[:, w:])
    for r in range(rows):
        if pos[r] < 0:
            assert np.array_equal(got[r], was[r])
            continue
        for a, b, gg in ((0, H * hd, g[0]), (H * hd, w, g[1])):
            ref, tol = norm_ref(m[r:r + 1, a:b], gg, pos[r:r + 1], hd, 1e-5, 1e4)
            assert (np.abs(got[r:r + 1, a:b] - ref) <= tol).all()


# ------------------------------------------------------------------ the cache
def held(x):
    """(codes 0..15, meta, values) of rows [..., hd], in the definition's f32 steps."""
    y = np.ascontiguousarray(x, np.float32).reshape(*x.shape[:-1], -1, 32)
    lo, hi = y.min(-1), y.max(-1)
    b = lo.view(np.uint32)
    mn = np.where(b >> 31, b + np.uint32(0xFFFF), b) & np.uint32(0xFFFF0000)
    low = mn.view(np.float32)
    sc = (((hi - low) / np.float32(15)).view(np.uint32) + np.uint32(0xFFFF)) & np.uint32(0xFFFF0000)
    step = sc.view(np.float32)[..., None]
    with np.errstate(divide="ignore", invalid="ignore"):
        u = np.where(step > 0, np.clip(np.rint((y - low[..., None]) / step), 0, 15), 0)
    u = u.astype(np.float32)
    val = step * u + low[..., None]
    return u.astype(np.uint8).reshape(x.shape), mn | (sc >> 16), val.reshape(x.shape)


def heads_of(x, Hkv):
    """Rows [S, Hkv * hd] as [Hkv, S, hd]."""
    return x.reshape(x.shape[0], Hkv, -1).transpose(1, 0, 2)


def put(model, k, v, b, p0, n, Hkv):
    """The same append on the test's model of the cache: dict of per-position arrays."""
    if n == 0:
        return
    for name, x in (("k", k), ("v", v)):
        u, m, val = held(heads_of(x[:n], Hkv))
        model[name + "u"][b, :, p0:p0 + n] = u
        model[name + "m"][b, :, p0:p0 + n] = m
        model[name][b, :, p0:p0 + n] = val


def new_model(B, Hkv, cap, hd):
    z = np.zeros
    return dict(ku=z((B, Hkv, cap, hd), np.uint8), vu=z((B, Hkv, cap, hd), np.uint8),
                km=z((B, Hkv, cap, hd // 32), np.uint32), vm=z((B, Hkv, cap, hd // 32), np.uint32),
                k=z((B, Hkv, cap, hd), np.float32), v=z((B, Hkv, cap, hd), np.float32))


def cache_codes(c):
    """(K, V) codes 0..15 of an ops.Kv4Cache by position."""
    k = (nibbles(c.k) + 8).astype(np.uint8)
    v = (nibbles(c.v) + 8).astype(np.uint8).transpose(0, 1, 2, 4, 3)
    return k, v.reshape(k.shape)


def same_cache(c, m, where):
    """Bit equality on the positions `where` [B, cap]; untouched ones are the empty
    cache's zero nibbles (u = 8)."""
    k, v = cache_codes(c)
    w = where[:, None, :, None]
    for got, u in ((k, m["ku"]), (v, m["vu"])):
        assert np.array_equal(got, np.where(w, u, 8))
    assert np.array_equal(c.k_meta, np.where(w, m["km"], 0))
    assert np.array_equal(c.v_meta, np.where(w, m["vm"], 0))


@pytest.mark.parametrize("B,Hkv,hd,cap,chunks", [
    (1, 1, 32, 32, [1, 1, 30]), (1, 2, 64, 96, [31, 1, 33, 31]), (2, 3, 64, 128, [32, 64, 5]),
    (3, 1, 128, 160, [100, 59]), (1, 2, 256, 64, [7, 57]), (2, 36, 64, 128, [128])])
def test_cache_append_and_read(ops, B, Hkv, hd, cap, chunks):
    """Chunks of other lengths a sequence, one after another, from positions inside a
    block; codes, meta and read values equal the definition's, and the positions
    behind stay as they were."""
    rng = np.random.default_rng(cap + hd)
    c, m = ops.Kv4Cache(B, Hkv, cap, hd), new_model(B, Hkv, cap, hd)
    at = np.zeros(B, np.int32)
    for S in chunks:
        k, v = (rng.standard_normal((2, B, S, Hkv * hd), dtype=np.float32) *
                np.exp(rng.standard_normal((1, 1, 1, Hkv * hd))).astype(np.float32))
        n = np.array([max(0, S - 3 * b) for b in range(B)], np.int32)
        c.append(k, v, at, n)
        for b in range(B):
            put(m, k[b], v[b], b, at[b], n[b], Hkv)
        rk, rv = c.read(at, S, n)
        for b in range(B):
            for got, name in ((rk, "k"), (rv, "v")):
                want = m[name][b, :, at[b]:at[b] + n[b]].transpose(1, 0, 2).reshape(n[b], -1)
                assert np.array_equal(got[b, :n[b]], want) and not got[b, n[b]:].any()
        at += n
        same_cache(c, m, np.arange(cap)[None] < at[:, None])


def test_cache_overwrites_and_idles(ops):
    """Positions written again take the new rows, their neighbours in a byte keep
    theirs; a sequence with a negative first position is left alone."""
    rng = np.random.default_rng(3)
    c, m = ops.Kv4Cache(3, 2, 64, 64), new_model(3, 2, 64, 64)
    k, v = rng.standard_normal((2, 3, 64, 128), dtype=np.float32)
    c.append(k, v, [0, 0, 0])
    for b in range(3):
        put(m, k[b], v[b], b, 0, 64, 2)
    k, v = rng.standard_normal((2, 3, 3, 128), dtype=np.float32)
    c.append(k, v, [31, -1, 6], [3, 3, 1])
    put(m, k[0], v[0], 0, 31, 3, 2)
    put(m, k[2], v[2], 2, 6, 1, 2)
    same_cache(c, m, np.ones((3, 64), bool))
    rk, _ = c.read([-5, 0, 0], 2)
    assert not rk[0].any() and rk[1].any()


def test_cache_past_the_capacity(ops):
    """Rows from cap on are dropped and reported; those before are stored."""
    from sparrow_amd import VmlmError
    rng = np.random.default_rng(4)
    for at in (60, 64, 1000, 2 ** 31 - 1):
        c, m = ops.Kv4Cache(2, 1, 64, 64), new_model(2, 1, 64, 64)
        k, v = rng.standard_normal((2, 2, 10, 64), dtype=np.float32)
        with pytest.raises(VmlmError) as e:
            c.append(k, v, [at, 20])
        assert e.value.code == 9
        c.append(k[:, :1], v[:, :1], [0, 0])  # the guard is down again



@pytest.mark.parametrize("case", ["flat", "wide", "tiny", "offset", "huge", "bad"])
def test_cache_values(ops, case):
    """One value 32 times; ranges from subnormal steps to past f32; channels beside a
    large offset; NaN and infinities, which poison their 32 channels alone."""
    rng = np.random.default_rng(5)
    x = rng.standard_normal((1, 9, 128), dtype=np.float32)
    if case == "flat":
        x[:] = rng.standard_normal((1, 9, 1), dtype=np.float32)
        x[0, 0] = 0
        x[0, 1] = -0.0
    elif case == "wide":
        x *= np.float32(10.0) ** rng.integers(-20, 21, x.shape).astype(np.float32)
    elif case == "tiny":
        x *= np.float32(1e-37)
    elif case == "offset":
        x += np.float32(1000)
    elif case == "huge":
        x[0, :, 0], x[0, :, 1] = 3e38, -3e38  # the range leaves f32
    else:
        x[0, 0, 3], x[0, 1, 40], x[0, 2, 77], x[0, 3, 100] = np.nan, np.inf, -np.inf, np.nan
    c = ops.Kv4Cache(1, 1, 32, 128)
    c.append(x, x, [0])
    got = c.read([0], 9)
    with np.errstate(all="ignore"):
        want = held(x)[2]
    groups = x.reshape(9, 4, 32)
    with np.errstate(over="ignore", invalid="ignore"):
        poisoned = ~np.isfinite(groups).all(-1) | ~np.isfinite(groups.max(-1) - groups.min(-1))
    poisoned = np.repeat(poisoned, 32, -1).reshape(1, 9, 128)
    for y in got:
        assert np.isnan(y[poisoned]).all()
        assert np.array_equal(y[~poisoned], want[~poisoned])


# ------------------------------------------------------------------ attention
def attn_ref(m, q, pos, Hkv, hd, scale):
    """(out in 64 bits, its bound) for live rows."""
    B, H = q.shape[0], q.shape[1] // hd
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    for b in range(B):
        n = pos[b] + 1
        if n <= 0:
            continue
        for h in range(H):
            k = m["k"][b, h // (H // Hkv), :n].astype(np.float64)
            v = m["v"][b, h // (H // Hkv), :n].astype(np.float64)
            x = q[b, h * hd:(h + 1) * hd].astype(np.float64)
            s = k @ x * scale
            p = np.exp(s - s.max())
            ds = (32 + hd / 8) * U * scale * (np.abs(k) @ np.full(hd, np.abs(x).max())).max()
            out[b, h * hd:(h + 1) * hd] = p @ v / p.sum()
            tol[b, h * hd:(h + 1) * hd] = (4 * ds + (n / 128 + 64) * U) * np.abs(v).max()
    return out, tol


def filled(ops, rng, B, Hkv, cap, hd, lens):
    c, m = ops.Kv4Cache(B, Hkv, cap, hd), new_model(B, Hkv, cap, hd)
    k, v = rng.standard_normal((2, B, cap, Hkv * hd), dtype=np.float32)
    k += rng.standard_normal((1, 1, Hkv * hd), dtype=np.float32)
    c.append(k, v, np.zeros(B), lens)
    for b in range(B):
        put(m, k[b], v[b], b, 0, lens[b], Hkv)
    # what was never written may hold anything: NaN ranges and any codes
    for b in range(B):
        n = lens[b]
        c.k[b, :, n:] = 0x5A
        c.k_meta[b, :, n:] = c.v_meta[b, :, n:] = 0x7FC07FC0
        u = nibbles(c.v[b])  # [Hkv, blocks, hd, 32]
        u = u.transpose(0, 1, 3, 2).reshape(Hkv, cap, hd)
        u[:, n:] = -6
        u = (u & 15).astype(np.uint8).reshape(Hkv, cap // 32, 32, hd).transpose(0, 1, 3, 2)
        c.v[b] = u[..., 0::2] | (u[..., 1::2] << 4)
    return c, m


ATTN = [(1, 1, 1, 32, 32, [0]), (1, 1, 1, 64, 32, [31]), (1, 36, 36, 64, 128, [127]),
        (4, 4, 4, 64, 256, [0, 1, 130, -1]), (2, 6, 2, 128, 320, [319, 127]),
        (3, 8, 1, 64, 192, [31, 32, 190]), (2, 16, 1, 256, 160, [77, 159]),
        (1, 15, 3, 32, 544, [543]), (2, 14, 2, 64, 96, [95, 5]), (1, 24, 2, 128, 1056, [1040]),
        (1, 2, 1, 64, 4128, [4100]), (1, 2, 2, 64, 8192, [8191]), (2, 5, 1, 128, 5120, [5000, 3]),
        (1, 3, 3, 32, 4096, [4000]), (3, 2, 1, 256, 1600, [1599, 700, -1]), (2, 9, 1, 64, 2080, [5, 2079]),
        # more sequences than a wave has lanes, some idle, most of them short
        (70, 1, 1, 64, 1152, [-1, 1151, 0, 64, 700, -1, 127, 128, 1000, 3] * 7),
        (130, 2, 1, 32, 1056, ([-1] * 60 + [1055, 31, 90, 500, 0]) * 2)]


@pytest.mark.parametrize("B,H,Hkv,hd,cap,pos", ATTN)
@pytest.mark.parametrize("append", [True, False])
def test_attention(ops, B, H, Hkv, hd, cap, pos, append):
    rng = np.random.default_rng(cap + H + hd)
    pos = np.array(pos, np.int32)
    c, m = filled(ops, rng, B, Hkv, cap, hd, np.maximum(pos + (0 if append else 1), 0))
    q = rng.standard_normal((B, H * hd), dtype=np.float32)
    new = [None, None]
    if append:
        new = list(rng.standard_normal((2, B, Hkv * hd), dtype=np.float32))
        for b in range(B):
            if pos[b] >= 0:
                put(m, new[0][b:b + 1], new[1][b:b + 1], b, pos[b], 1, Hkv)
    scale = float(np.float32(hd ** -0.5))
    out = c.attention_decode(q, pos, *new)
    ref, tol = attn_ref(m, q, pos, Hkv, hd, scale)
    assert (np.abs(out - ref) <= tol).all(), (np.abs(out - ref) / np.maximum(tol, 1e-30)).max()
    if append:  # the cache holds the new rows and what it held
        k, v = cache_codes(c)
        for b in range(B):
            n = pos[b] + 1
            assert np.array_equal(k[b, :, :max(n, 0)], m["ku"][b, :, :max(n, 0)])
            assert np.array_equal(v[b, :, :max(n, 0)], m["vu"][b, :, :max(n, 0)])
            assert (v[b, :, max(n, 0):] == 2).all()  # -6 + 8


@pytest.mark.parametrize("H,Hkv,hd", [(2, 2, 64), (8, 2, 64), (4, 1, 128)])
def test_attention_large_scores(ops, H, Hkv, hd):
    """Scores in the hundreds: the weights are nearly one-hot, and the position that
    wins may come first, last or in between."""
    rng = np.random.default_rng(8)
    cap, pos = 512, np.array([511, 300, 2], np.int32)
    c, m = filled(ops, rng, 3, Hkv, cap, hd, pos + 1)
    q = 60 * rng.standard_normal((3, H * hd), dtype=np.float32)
    out = c.attention_decode(q, pos)
    ref, tol = attn_ref(m, q, pos, Hkv, hd, float(np.float32(hd ** -0.5)))
    assert (np.abs(out - ref) <= tol).all(), (np.abs(out - ref) / tol).max()


def test_attention_magnitudes(ops):
    """Values whose scales differ by 1e20 between positions, and subnormal queries."""
    rng = np.random.default_rng(9)
    c, m = ops.Kv4Cache(1, 1, 256, 64), new_model(1, 1, 256, 64)
    k, v = rng.standard_normal((2, 1, 256, 64), dtype=np.float32)
    v *= np.float32(10.0) ** rng.integers(-10, 11, (1, 256, 1)).astype(np.float32)
    c.append(k, v, [0])
    put(m, k[0], v[0], 0, 0, 256, 1)
    q = rng.standard_normal((1, 128), dtype=np.float32)
    q[0, 64:] *= np.float32(1e-39)
    out = c.attention_decode(q, [255])
    ref, tol = attn_ref(m, q, [255], 1, 64, 0.125)
    assert (np.abs(out - ref) <= tol).all(), (np.abs(out - ref) / tol).max()


def test_attention_nonfinite(ops):
    """A poisoned value group gives NaN in its 32 channels, a poisoned key or query
    in the heads that read it, and no other head or sequence sees it."""
    rng = np.random.default_rng(10)
    k, v = rng.standard_normal((2, 2, 100, 256), dtype=np.float32)  # 4 kv heads of 64
    q = rng.standard_normal((2, 8 * 64), dtype=np.float32)
    pos = [99, 99]
    c = ops.Kv4Cache(2, 4, 128, 64)
    c.append(k, v, [0, 0])
    clean = c.attention_decode(q, pos)
    v[0, 40, 64 + 5] = np.inf   # kv head 1, channels 0..31
    k[0, 41, 128 + 50] = np.nan  # kv head 2
    q[0, 7 * 64 + 1] = np.nan   # head 7
    c.append(k, v, [0, 0])
    out = c.attention_decode(q, pos)
    bad = np.zeros(out.shape, bool)
    for h in (2, 3):
        bad[0, h * 64:h * 64 + 32] = True
    bad[0, 4 * 64:6 * 64] = bad[0, 7 * 64:] = True
    assert np.isnan(out[bad]).all()
    assert np.array_equal(out[~bad], clean[~bad])


def test_attention_position_past_the_capacity(ops):
    from sparrow_amd import VmlmError
    rng = np.random.default_rng(11)
    c = ops.Kv4Cache(2, 1, 64, 64)
    k, v = rng.standard_normal((2, 2, 64, 64), dtype=np.float32)
    c.append(k, v, [0, 0])
    q = rng.standard_normal((2, 64), dtype=np.float32)
    for p in (64, 2 ** 31 - 1):
        with pytest.raises(VmlmError) as e:
            c.attention_decode(q, [p, 63], q, q)
        assert e.value.code == 9
    assert np.isfinite(c.attention_decode(q, [63, 63])).all()


def test_attention_split_position_past_the_capacity(ops):
    """The same where the sequences are split."""
    from sparrow_amd import VmlmError
    rng = np.random.default_rng(15)
    c, m = filled(ops, rng, 2, 1, 2048, 64, [2048, 2048])
    q = rng.standard_normal((2, 64), dtype=np.float32)
    for p in (2048, 2 ** 31 - 1):
        with pytest.raises(VmlmError) as e:
            c.attention_decode(q, [2047, p])
        assert e.value.code == 9
    out = c.attention_decode(q, [2047, 1500])
    ref, tol = attn_ref(m, q, [2047, 1500], 1, 64, 0.125)
    assert (np.abs(out - ref) <= tol).all()


def test_offsets_past_32_bits(dev):
    """The last of five sequences whose caches are 1 GB of codes each: its rows lie
    past 2^32 bytes in every array of codes."""
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
    k, v = rng.standard_normal((2, B, S, H * hd), dtype=np.float32)
    q = rng.standard_normal((B, H * hd), dtype=np.float32)
    dk, dv, dq = dev.up(k), dev.up(v), dev.up(q)
    rk, rv, out = dev.zeros(*k.shape), dev.zeros(*v.shape), dev.zeros(*q.shape)
    need = C.c_size_t()
    dev.check(dev.L.vmlm_hip_attention_decode_kv4_work(d, H, C.byref(need)))
    work = dev.zeros(max(need.value, 16), dtype=np.uint8)
    w = H * hd
    for first in (cap - S, 0):
        pos = dev.up(np.array([-1] * (B - 1) + [first], np.int32))
        dev.check(dev.L.vmlm_hip_kv4_append(d, dk.ptr, w, dv.ptr, w, pos.ptr, None, S, None))
        dev.check(dev.L.vmlm_hip_kv4_read(d, rk.ptr, w, rv.ptr, w, pos.ptr, None, S, None))
        dev.sync()
        for got, x in ((rk.get(), k), (rv.get(), v)):
            assert not got[:-1].any() and np.array_equal(got[-1], held(x[-1])[2])
    pos = np.array([-1] * (B - 1) + [S - 1], np.int32)
    dp = dev.up(pos)
    dev.check(dev.L.vmlm_hip_attention_decode_kv4(d, dq.ptr, w, None, None, 0, dp.ptr, out.ptr, w, H,
                                                  0.0625, work.ptr, work.nbytes, None))
    dev.check(dev.L.vmlm_hip_check_guards())
    dev.sync()
    m = new_model(B, H, 32, hd)
    put(m, k[-1], v[-1], B - 1, 0, S, H)
    ref, tol = attn_ref(m, q, pos, H, hd, 0.0625)
    assert (np.abs(out.get() - ref) <= tol).all()


def device_cache(dev, c):
    from sparrow_amd import _abi
    t = [dev.up(x) for x in (c.k, c.v, c.k_meta, c.v_meta)]
    d = _abi.Kv4Cache(*(x.ptr for x in t), c.batch, c.n_kv_heads, c.cap, c.head_dim)
    return t, d


def test_attention_strides_and_idle_rows(dev, ops):
    """Queries and new rows inside fused rows of an odd stride, outputs likewise; idle
    rows and the padding stay as they were."""
    rng = np.random.default_rng(12)
    B, H, Hkv, hd, cap = 3, 4, 2, 64, 96
    pos = np.array([40, -1, 95], np.int32)
    c, m = filled(ops, rng, B, Hkv, cap, hd, np.maximum(pos, 0))
    ld, ldo = (H + 2 * Hkv) * hd + 3, H * hd + 1
    x = rng.standard_normal(1 + B * ld, dtype=np.float32)
    t, d = device_cache(dev, c)
    dx, dp, do = dev.up(x), dev.up(pos), dev.up(np.full(1 + B * ldo, 3.0, np.float32))
    base = dx.ptr + 4
    dev.sync()
    dev.check(dev.L.vmlm_hip_attention_decode_kv4(
        d, base, ld, base + 4 * H * hd, base + 4 * (H + Hkv) * hd, ld, dp.ptr,
        do.ptr + 4, ldo, H, 0.125, None, 0, None))
    dev.sync()
    r = x[1:].reshape(B, ld)
    for b in (0, 2):
        put(m, r[b:b + 1, H * hd:(H + Hkv) * hd], r[b:b + 1, (H + Hkv) * hd:(H + 2 * Hkv) * hd], b,
            pos[b], 1, Hkv)
    ref, tol = attn_ref(m, r[:, :H * hd], pos, Hkv, hd, 0.125)
    got = do.get()
    assert got[0] == 3
    got = got[1:].reshape(B, ldo)
    assert (got[:, -1] == 3).all() and (got[1] == 3).all()
    for b in (0, 2):
        assert (np.abs(got[b, :-1] - ref[b]) <= tol[b]).all()


# ------------------------------------------------------------------ together
def test_layer_of_a_decode_step(dev, ops):
    """One decode layer as a program runs it: q/k/v in one int4 product, head norms
    and rotation in place, the new rows into the cache and the attention, the o
    projection; eagerly, then captured and replayed over further tokens, with eager work
    between. Every stage is checked against 64 bits on the stage's own inputs."""
    rng = np.random.default_rng(13)
    B, H, Hkv, hd, hidden, cap, group = 3, 8, 2, 64, 512, 4160, 64
    wq, wk = H * hd, Hkv * hd
    ld, scale = wq + 2 * wk, 0.125
    qw, qs = ops.quantize_int4(rng.standard_normal((ld, hidden)) / 22, group)
    ow, osc = ops.quantize_int4(rng.standard_normal((hidden, wq)) / 22, group)
    g = (1 + rng.standard_normal((2, hd)) / 8).astype(np.float32)
    start = np.array([4100, 0, -1], np.int32)
    c, m = filled(ops, rng, B, Hkv, cap, hd, np.maximum(start, 0))
    keep, d = device_cache(dev, c)
    dw = [dev.up(x) for x in (qw, qs, ow, osc, g)]
    x = dev.up(rng.standard_normal((B, hidden), dtype=np.float32))
    qkv, rot, out, y = (dev.zeros(B, w) for w in (ld, ld, wq, hidden))
    pos = dev.up(start)
    need = C.c_size_t()
    dev.check(dev.L.vmlm_hip_attention_decode_kv4_work(d, H, C.byref(need)))
    work = dev.zeros(max(need.value, 16), dtype=np.uint8)
    st = dev.stream()

    def step():
        p, s = [v.ptr for v in (x, qkv, rot, out, y, pos)], st
        dev.check(dev.L.vmlm_hip_gemm_nt_int4(p[0], dw[0].ptr, dw[1].ptr, p[1], B, ld,
                                              hidden, group, s))
        dev.check(dev.L.vmlm_hip_qk_norm_rope(
            p[2], ld, p[2] + 4 * wq, ld, p[1], ld, p[1] + 4 * wq, ld, dw[4].ptr,
            dw[4].ptr + 4 * hd, p[5], B, H, Hkv, hd, 1e-5, 1e4, s))
        dev.check(dev.L.vmlm_hip_attention_decode_kv4(
            d, p[2], ld, p[2] + 4 * wq, p[1] + 4 * (wq + wk), ld, p[5], p[3], wq, H, scale,
            work.ptr, work.nbytes, s))
        dev.check(dev.L.vmlm_hip_gemm_nt_int4(p[3], dw[2].ptr, dw[3].ptr, p[4], B,
                                              hidden, wq, group, s))

    def check(at):
        dev.sync()
        hx, hq, hr, ho, hy = (v.get() for v in (x, qkv, rot, out, y))
        int4_check(hq, hx, qw, qs, group)
        for b in np.flatnonzero(at >= 0):
            for a, e, gg in ((0, wq, g[0]), (wq, wq + wk, g[1])):
                ref, tol = norm_ref(hq[b:b + 1, a:e], gg, at[b:b + 1], hd, 1e-5, 1e4)
                assert (np.abs(hr[b:b + 1, a:e] - ref) <= tol).all()
            put(m, hr[b:b + 1, wq:wq + wk], hq[b:b + 1, wq + wk:], b, at[b], 1, Hkv)
        assert not hr[at < 0].any() and not ho[at < 0].any()
        ref, tol = attn_ref(m, hr[:, :wq], at, Hkv, hd, scale)
        assert (np.abs(ho - ref) <= tol).all()
        int4_check(hy, ho, ow, osc, group)

    dev.sync()
    step()
    check(start)
    graph = C.c_void_p()
    dev.check(dev.L.vmlm_hip_capture_begin(st))
    step()
    dev.check(dev.L.vmlm_hip_capture_end(st, C.byref(graph)))
    for i in range(1, 5):
        at = np.where(start >= 0, start + i, -1).astype(np.int32)
        pos.put(at)
        x.put(np.roll(x.get(), 7, 1) * 0.5 + y.get() * 0.1)
        dev.check(dev.L.vmlm_hip_graph_launch(graph, st))
        check(at)
    dev.check(dev.L.vmlm_hip_graph_destroy(graph))


def test_captured_attention_needs_its_own_workspace(dev, ops):
    """A split launch under capture without a workspace is refused and leaves the
    capture usable; two graphs with workspaces of their own run at once."""
    rng = np.random.default_rng(14)
    B, H, hd, cap = 1, 1, 64, 8192
    graphs = []
    for i in range(2):
        c, m = filled(ops, rng, B, H, cap, hd, np.array([cap]))
        keep, d = device_cache(dev, c)
        q, pos = rng.standard_normal((B, hd), dtype=np.float32), np.array([cap - 1], np.int32)
        dq, dp, out = dev.up(q), dev.up(pos), dev.zeros(B, hd)
        need = C.c_size_t()
        dev.check(dev.L.vmlm_hip_attention_decode_kv4_work(d, H, C.byref(need)))
        work = dev.zeros(max(need.value, 16), dtype=np.uint8)
        st, graph = dev.stream(), C.c_void_p()
        dev.sync()

        def call(w, n):
            return dev.L.vmlm_hip_attention_decode_kv4(d, dq.ptr, hd, None, None, 0,
                                                       dp.ptr, out.ptr, hd, H, 0.125,
                                                       w, n, st)
        dev.check(dev.L.vmlm_hip_capture_begin(st))
        if need.value:
            assert call(None, 0) == 9
            assert call(work.ptr, need.value - 4) == 9
            assert call(work.ptr + 4, need.value) == 9
        dev.check(call(work.ptr, work.nbytes))
        dev.check(dev.L.vmlm_hip_capture_end(st, C.byref(graph)))
        graphs.append((st, graph, out, attn_ref(m, q, pos, H, hd, 0.125), (keep, dq, dp, work)))
    for _ in range(3):
        for st, graph, out, _, _ in graphs:
            out.put(np.zeros(out.shape))
        for st, graph, out, _, _ in graphs:
            dev.check(dev.L.vmlm_hip_graph_launch(graph, st))
        dev.sync()
        for st, graph, out, (ref, tol), _ in graphs:
            assert (np.abs(out.get() - ref) <= tol).all()
    for st, graph, *_ in graphs:
        dev.check(dev.L.vmlm_hip_graph_destroy(graph))
