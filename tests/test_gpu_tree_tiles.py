"""Attention of a chunk over few (sequence, kv head) pairs: as many tiles of queries as the accepted sizes
give, each computed once. Tolerances are those of test_gpu_draft.py."""
import ctypes as C

import numpy as np
import pytest
from test_gpu_4bit import dev, device_cache, filled, new_model, ops, put  # noqa: F401
from test_gpu_draft import check_tree, tree_ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,Hkv", [(1, 1), (1, 3), (7, 1), (2, 4), (3, 3), (1, 17)])
@pytest.mark.parametrize("hd", [32, 128])
def test_attention_pairs_and_tiles(ops, B, Hkv, hd):
    """Fewer pairs than XCDs, as many, and more; each with several tiles of the last one not full."""
    rng = np.random.default_rng(B + Hkv + hd)
    S, G, cap = 45, 3, 96
    pos0 = rng.integers(0, cap - S, B).astype(np.int32)
    n = rng.integers(1, S + 1, B)
    n[0] = S
    c, m = filled(ops, rng, B, Hkv, cap, hd, pos0 + n)
    q = rng.standard_normal((B, S, Hkv * G * hd), dtype=np.float32)
    out = c.attention_tree(q, pos0, n, out=np.full_like(q, 3.0))
    check_tree(out, tree_ref(m, q, pos0, n, None, Hkv, hd, float(np.float32(hd ** -0.5))), 3.0)


def test_attention_of_the_most_rows(dev, ops):
    """2^27 (token, head) pairs over one kv head, two million tiles: all but the first token are padding,
    whose queries are never looked at and whose outputs stay as they were."""
    S, H, hd, cap = 32768, 4096, 32, 32
    rng = np.random.default_rng(60)
    w = H * hd
    c, m = filled(ops, rng, 1, 1, cap, hd, [9])
    q = rng.standard_normal((1, 1, w), dtype=np.float32)
    _, d = device_cache(dev, c)
    ptrs = []
    for _ in range(2):
        p = C.c_void_p()
        dev.check(dev.L.vmlm_hip_malloc(C.byref(p), S * w * 4))
        dev.bufs.append(p.value)
        ptrs.append(p.value)
    old = np.full((2, w), 3.0, np.float32)
    dev.check(dev.L.vmlm_hip_memcpy_h2d(ptrs[0], q.ctypes.data, q.nbytes))
    dev.check(dev.L.vmlm_hip_memcpy_h2d(ptrs[1], old.ctypes.data, old.nbytes))
    dp, dn = dev.up(np.array([8], np.int32)), dev.up(np.array([1], np.int32))
    need = C.c_size_t(1)
    dev.check(dev.L.vmlm_hip_attention_tree_kv4_work(d, H, S, C.byref(need)))
    assert need.value == 0
    scale = float(np.float32(hd ** -0.5))
    dev.check(dev.L.vmlm_hip_attention_tree_kv4(d, ptrs[0], w, dp.ptr, dn.ptr, None, S, ptrs[1], w, H, scale, None, 0,
                                                None))
    dev.check(dev.L.vmlm_hip_check_guards())
    dev.sync()
    got = np.empty_like(old)
    dev.check(dev.L.vmlm_hip_memcpy_d2h(got.ctypes.data, ptrs[1], got.nbytes))
    assert (got[1] == 3).all()
    check_tree(got[None, :1], tree_ref(m, q, [8], [1], None, 1, hd, scale))


@pytest.mark.parametrize("B,Hkv,cap", [(513, 1, 8192), (512, 1, 8192), (1100, 1, 8192), (300, 4, 8192)])
def test_attention_long_caches_of_many_sequences(ops, B, Hkv, cap):
    """As many sequences as are dealt out by their lengths, and more, a long one among them."""
    rng = np.random.default_rng(B)
    hd, S, n = 32, 2, np.full(B, 2)
    pos0 = rng.integers(0, 40, B).astype(np.int32)
    pos0[[3, B // 2]], pos0[5] = [1500, 700], -1
    c, m = ops.Kv4Cache(B, Hkv, cap, hd), new_model(B, Hkv, 1536, hd)
    k, v = rng.standard_normal((2, B, 1502, Hkv * hd), dtype=np.float32)
    lens = np.where(pos0 >= 0, pos0 + 2, 0)
    c.append(k, v, np.zeros(B), lens)
    for b in range(B):
        put(m, k[b], v[b], b, 0, lens[b], Hkv)
    q = rng.standard_normal((B, S, Hkv * hd), dtype=np.float32)
    out = c.attention_tree(q, pos0, n, out=np.full_like(q, 3.0))
    check_tree(out, tree_ref(m, q, pos0, n, None, Hkv, hd, float(np.float32(hd ** -0.5))), 3.0)
