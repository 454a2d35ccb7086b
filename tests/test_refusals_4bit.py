"""What the 4-bit operators refuse, through the C ABI on the CPU: arguments are
checked before the library looks for a GPU, so a refused call returns 9 here too
and an accepted one of no work returns 0. Pointers are made up and never read."""
import ctypes as C

import numpy as np
import pytest

A, Q, S, Y, Z = (0x10000000 * (i + 1) for i in range(5))  # far apart


@pytest.fixture(scope="module")
def L():
    import sparrow_amd
    return sparrow_amd.lib()


def message(L):
    return L.vmlm_hip_last_error().decode()


# ------------------------------------------------------------------ gemm_nt_int4
def int4(L, a=A, q=Q, s=S, c=Y, m=2, n=64, k=128, group=128):
    return L.vmlm_hip_gemm_nt_int4(a, q, s, c, m, n, k, group, None)


@pytest.mark.parametrize("bad", [dict(k=100), dict(k=1), dict(group=0), dict(group=16),
                                 dict(group=96), dict(group=200), dict(a=None), dict(q=None),
                                 dict(s=None), dict(c=None), dict(m=2 ** 31), dict(n=2 ** 40),
                                 dict(k=2 ** 25), dict(c=A), dict(c=A + 4 * 128), dict(c=Q + 64),
                                 dict(c=S + 4), dict(a=Y + 4 * 127)])
def test_int4_refused(L, bad):
    assert int4(L, **bad) == 9, bad
    assert "int4 gemm" in message(L)


@pytest.mark.parametrize("empty", [dict(m=0), dict(n=0), dict(m=0, a=None, c=None)])
def test_int4_nothing_to_do(L, empty):
    assert int4(L, **empty) == 0


def test_int4_host_refused(L):
    f = np.zeros(256, np.float32)
    p = f.ctypes.data
    assert L.vmlm_gemm_nt_int4(p, p, p, p, 1, 1, 33, 32) == 9
    assert L.vmlm_gemm_nt_int4(p, p, None, p, 1, 1, 32, 32) == 9
    assert L.vmlm_gemm_nt_int4(p, p, p, p, 0, 1, 32, 32) == 0


# ------------------------------------------------------------------ qk_norm_rope
def norm(L, qo=Y, ldqo=256, ko=Z, ldko=128, q=A, ldq=256, k=Q, ldk=128, gq=S, gk=S + 4096,
         pos=S + 8192, rows=3, H=4, Hkv=2, hd=64, eps=1e-5, theta=1e4):
    return L.vmlm_hip_qk_norm_rope(qo, ldqo, ko, ldko, q, ldq, k, ldk, gq, gk, pos, rows, H, Hkv,
                                   hd, eps, theta, None)


@pytest.mark.parametrize("bad", [dict(hd=0), dict(hd=4), dict(hd=60), dict(hd=520), dict(theta=0.0),
                                 dict(theta=-1.0), dict(theta=float("nan")),
                                 dict(theta=float("inf")), dict(eps=-1.0), dict(eps=float("nan")),
                                 dict(q=None), dict(k=None), dict(gq=None), dict(gk=None),
                                 dict(qo=None), dict(ko=None), dict(ldq=255), dict(ldqo=255),
                                 dict(ldk=127), dict(ldko=0), dict(H=65536), dict(rows=2 ** 31),
                                 dict(qo=A + 4), dict(qo=A, ldqo=512), dict(ko=A), dict(qo=Q),
                                 dict(ko=Y + 4 * 255), dict(ko=Y + 128), dict(gq=Y + 64),
                                 dict(gk=Z)])
def test_norm_refused(L, bad):
    assert norm(L, **bad) == 9, bad


def test_norm_parts_of_one_row_are_no_overlap(L):
    """q and k normed in place inside fused rows share a span but no value; what is
    accepted goes on to the device (0 with one, 2 without) when there is work."""
    fused = dict(q=A, qo=A, k=A + 4 * 256, ko=A + 4 * 256, ldq=512, ldqo=512, ldk=512, ldko=512)
    assert norm(L, **fused, rows=0) == 0
    bad = dict(fused, ko=A + 4 * 200, k=A + 4 * 200)
    assert norm(L, **bad) == 9  # k's columns begin among q's
    bad = dict(fused, ko=A + 4 * 400, k=A + 4 * 400)
    assert norm(L, **bad) == 9  # and here run into the next row's q


@pytest.mark.parametrize("empty", [dict(rows=0), dict(H=0, Hkv=0)])
def test_norm_nothing_to_do(L, empty):
    assert norm(L, **empty) == 0


# ------------------------------------------------------------------ the cache
def cache(k=A, v=Q, k_meta=S, v_meta=S + 0x1000000, batch=2, n_kv_heads=2, cap=64, head_dim=64):
    from sparrow_amd import _abi
    return _abi.Kv4Cache(k=k, v=v, k_meta=k_meta, v_meta=v_meta, batch=batch,
                         n_kv_heads=n_kv_heads, cap=cap, head_dim=head_dim)


BAD_CACHES = [dict(head_dim=48), dict(head_dim=512), dict(cap=33), dict(cap=0), dict(cap=2 ** 31),
              dict(k=None), dict(v=None), dict(k_meta=None), dict(v_meta=None), dict(k=A + 8),
              dict(v=Q + 1), dict(k_meta=S + 2), dict(batch=65536), dict(n_kv_heads=65536)]


def rows(L, fn, c, k=Y, ldk=128, v=Z, ldv=128, pos0=A - 64, count=None, S=3):
    return getattr(L, fn)(c, k, ldk, v, ldv, pos0, count, S, None)


@pytest.mark.parametrize("fn", ["vmlm_hip_kv4_append", "vmlm_hip_kv4_read"])
def test_cache_rows_refused(L, fn):
    for bad in BAD_CACHES:
        assert rows(L, fn, cache(**bad)) == 9, bad
    for bad in (dict(k=None), dict(v=None), dict(pos0=None), dict(ldk=127), dict(ldv=0),
                dict(S=2 ** 31)):
        assert rows(L, fn, cache(), **bad) == 9, bad
    assert rows(L, fn, None) == 9
    assert rows(L, fn, cache(), S=0) == 0
    assert rows(L, fn, cache(batch=0)) == 0


def test_read_over_itself_refused(L):
    assert rows(L, "vmlm_hip_kv4_read", cache(), v=Y + 4) == 9


def attend(L, c, q=Y, ldq=256, k=Z, v=Z + 0x100000, ldkv=128, pos=A - 64, out=Y + 0x100000, ldo=256,
           H=4, scale=0.125, work=None, nbytes=0):
    return L.vmlm_hip_attention_decode_kv4(c, q, ldq, k, v, ldkv, pos, out, ldo, H, scale, work,
                                           nbytes, None)


def test_attention_refused(L):
    for bad in BAD_CACHES:
        assert attend(L, cache(**bad)) == 9, bad
    for bad in (dict(q=None), dict(pos=None), dict(out=None), dict(k=None), dict(v=None), dict(ldq=255),
                dict(ldo=255), dict(ldkv=127), dict(H=3), dict(H=34), dict(scale=float("nan")),
                dict(scale=float("inf")), dict(out=Y), dict(out=Y + 4 * 255), dict(out=Z + 4)):
        assert attend(L, cache(), **bad) == 9, bad
    assert attend(L, None) == 9
    assert attend(L, cache(n_kv_heads=0)) == 9
    assert attend(L, cache(batch=0)) == 0
    assert attend(L, cache(), H=0) == 0


def test_rows_over_the_cache_refused(L):
    """An output among the codes or the meta would be read back as them."""
    ends = (A, A + 8192 - 4, Q + 64, S, S + 4, S + 0x1000000 + 2048 - 4)  # 2 * 2 * 64 * 64 values
    for at in ends:
        for fn in ("vmlm_hip_kv4_append", "vmlm_hip_kv4_read"):
            assert rows(L, fn, cache(), k=at) == 9, hex(at)
            assert rows(L, fn, cache(), v=at) == 9, hex(at)
            assert "lie over the cache" in message(L)
        assert attend(L, cache(), out=at) == 9, hex(at)
        assert "over the cache" in message(L)


def test_sizes_past_64_bits_refused(L):
    """Products of sizes, each within its own limit, that would wrap."""
    huge = cache(batch=65535, n_kv_heads=32767, cap=2 ** 30, head_dim=256)
    assert rows(L, "vmlm_hip_kv4_append", huge, ldk=2 ** 23, ldv=2 ** 23) == 9
    assert attend(L, huge, H=32767, ldq=2 ** 23, ldo=2 ** 23) == 9
    assert L.vmlm_kv4_read(huge, A, Q, S, None, 1) == 9
    wide = cache(batch=65535, n_kv_heads=2, cap=32, head_dim=32)
    assert rows(L, "vmlm_hip_kv4_read", wide, S=2 ** 30) == 9


def test_attention_workspace(L):
    n = C.c_size_t(1)
    assert L.vmlm_hip_attention_decode_kv4_work(cache(), 4, None) == 9
    assert L.vmlm_hip_attention_decode_kv4_work(cache(), 3, C.byref(n)) == 9
    assert L.vmlm_hip_attention_decode_kv4_work(cache(cap=65536, batch=1), 4, C.byref(n)) == 0
    assert n.value > 0
    long, out = cache(cap=65536, batch=1), Y + 0x100000
    work = Z + 0x1000000
    for bad in (dict(work=work, nbytes=n.value - 1), dict(work=work + 4, nbytes=n.value),
                dict(work=out, nbytes=n.value), dict(work=out + 4 * 256 - 16, nbytes=n.value),
                dict(work=Y, nbytes=n.value), dict(work=A, nbytes=n.value),
                dict(work=S, nbytes=n.value)):
        assert attend(L, long, out=out, **bad) == 9, bad
        assert "workspace" in message(L)


def test_host_forms_refuse_before_any_copy(L):
    c = cache(cap=33)
    p = A  # never read
    assert L.vmlm_kv4_append(c, p, p, p, None, 1) == 9
    assert L.vmlm_kv4_read(c, p, p, p, None, 1) == 9
    assert L.vmlm_attention_decode_kv4(c, p, None, None, p, p, 2, 1.0) == 9
    assert L.vmlm_attention_decode_kv4(cache(), p, p, None, p, p, 2, 1.0) == 9
    assert L.vmlm_qk_norm_rope(p, p, p, p, p, p, None, 1, 1, 1, 12, 1e-5, 1e4) == 9


def test_quantize_int4_round_trip():
    from sparrow_amd import ops
    rng = np.random.default_rng(0)
    w = rng.standard_normal((5, 96), dtype=np.float32)
    w[2, 64:] = 0
    for group in (32, 64, 128):
        q, s = ops.quantize_int4(w, group)
        assert q.shape == (5, 48) and s.shape == (5, -(-96 // group))
        u = np.stack((q & 15, q >> 4), -1).reshape(5, 96)
        back = ((u.astype(np.int8) ^ 8) - 8) * np.repeat(s, group, 1)[:, :96]
        # half a step, and the rounding of w / s
        assert (np.abs(back - w) <= np.repeat(s, group, 1)[:, :96] * (0.5 + 1e-5)).all()


# ------------------------------------------------------------------ operands over each other
FAR = 0x60000000  # behind every operand of the calls above


def test_norm_output_over_the_positions_refused(L):
    """Rows that other workgroups have yet to look up would find values there."""
    for bad in (dict(pos=Y), dict(pos=Y + 4 * (3 * 256 - 1)), dict(pos=Z - 8), dict(pos=Z + 4 * 200)):
        assert norm(L, **bad) == 9, bad
        assert "over the positions" in message(L)


def test_cache_arrays_over_each_other_refused(L):
    """2 * 2 * 64 * 64 values: 8192 bytes of codes, 2048 of meta."""
    for bad in (dict(v=A), dict(v=A + 8176), dict(k_meta=A + 4096), dict(v_meta=A + 8188),
                dict(k_meta=Q), dict(v_meta=Q + 8188), dict(v_meta=S), dict(v_meta=S + 2044),
                dict(k_meta=S + 0x1000000 - 2044)):
        for fn in ("vmlm_hip_kv4_append", "vmlm_hip_kv4_read"):
            assert rows(L, fn, cache(**bad)) == 9, bad
            assert "over each other" in message(L)
        assert attend(L, cache(**bad)) == 9, bad
        n = C.c_size_t()
        assert L.vmlm_hip_attention_decode_kv4_work(cache(**bad), 4, C.byref(n)) == 9


def test_positions_over_what_is_written_refused(L):
    at_cache = (A, A + 8188, Q + 8188, S + 2044, S + 0x1000000)
    for at in at_cache:
        assert rows(L, "vmlm_hip_kv4_append", cache(), pos0=at) == 9, hex(at)
        assert rows(L, "vmlm_hip_kv4_append", cache(), count=at) == 9, hex(at)
        assert "positions or counts" in message(L)
        assert attend(L, cache(), pos=at) == 9, hex(at)
    # 2 x 3 rows of 128 floats
    for at in (Y, Y + 4 * 767, Z, Z + 4 * 767, Z - 4):
        assert rows(L, "vmlm_hip_kv4_read", cache(), pos0=at) == 9, hex(at)
        assert rows(L, "vmlm_hip_kv4_read", cache(), count=at) == 9, hex(at)
        assert "positions or counts" in message(L)
    assert attend(L, cache(), pos=Y + 0x100000 + 4 * 511) == 9
    assert "positions" in message(L)


def test_inputs_over_the_cache_that_takes_new_rows_refused(L):
    for at in (A, A + 8188, Q, S + 2044, S + 0x1000000):
        for bad in (dict(q=at), dict(k=at), dict(v=at)):
            assert attend(L, cache(), **bad) == 9, bad
            assert "over the cache" in message(L)


def test_workspace_over_any_operand_refused(L):
    n = C.c_size_t()
    long = cache(cap=65536, batch=1)
    assert L.vmlm_hip_attention_decode_kv4_work(long, 4, C.byref(n)) == 0 and n.value
    args = dict(q=FAR, k=FAR + 0x100000, v=FAR + 0x200000, pos=FAR + 0x300000, out=FAR + 0x400000)
    width = dict(q=1024, k=512, v=512, pos=4, out=1024)
    for name, at in args.items():
        for work in (at, at + width[name] // 16 * 16 - 16 if width[name] > 16 else at,
                     (at - n.value) // 16 * 16 + 16):
            assert attend(L, long, **args, work=work, nbytes=n.value) == 9, (name, hex(work))
            assert "workspace" in message(L)


def test_host_read_over_itself_refused(L):
    assert L.vmlm_kv4_read(cache(), Y, Y + 4, A - 64, None, 3) == 9
    assert "over each other" in message(L)


@pytest.mark.parametrize("fn", ["vmlm_hip_kv4_append", "vmlm_hip_kv4_read"])
def test_rows_past_a_grid_refused(L, fn):
    """A grid of 256 threads for each block of 32 positions ends at 2^24 blocks; one
    block of a long cache, or many rows of a short one, are no such call (a batch of 0
    has no work)."""
    wide = dict(k=1 << 40, v=1 << 41, k_meta=1 << 42, v_meta=1 << 43, n_kv_heads=1, head_dim=32)
    at = dict(k=1 << 44, v=1 << 45, ldk=32, ldv=32)
    big = cache(batch=1, cap=2 ** 30, **wide)
    assert rows(L, fn, big, **at, S=2 ** 29) == 9
    assert "capacity" in message(L)
    assert rows(L, fn, cache(batch=0, cap=2 ** 30, **wide), **at, S=2 ** 29 - 64) == 0
    assert rows(L, fn, cache(batch=0, cap=64, **wide), **at, S=2 ** 30) == 0
