"""What the operators of a step with drafted tokens refuse, through the C ABI on the CPU:
arguments are checked before the library looks for a GPU, so a refused call returns 9
here too and an accepted one of no work returns 0. Pointers are made up and never read."""
import ctypes as C

import numpy as np
import pytest

A, Q, S, Y, Z = (0x10000000 * (i + 1) for i in range(5))  # far apart
W, X = 0x60000000, 0x70000000


@pytest.fixture(scope="module")
def L():
    import sparrow_amd
    return sparrow_amd.lib()


def message(L):
    return L.vmlm_hip_last_error().decode()


# ------------------------------------------------------------------ rope_qk
def rope(L, qo=Y, ldqo=256, ko=Z, ldko=128, q=A, ldq=256, k=Q, ldk=128, pos=S, freq=W, rows=3, H=4,
         Hkv=2, hd=64, rot=32, inter=False, factor=1.0):
    return L.vmlm_hip_rope_qk(qo, ldqo, ko, ldko, q, ldq, k, ldk, pos, freq, rows, H, Hkv, hd, rot,
                              inter, factor, None)


@pytest.mark.parametrize("bad", [
    dict(hd=0), dict(hd=63), dict(hd=514, rot=64), dict(rot=0), dict(rot=31), dict(rot=66),
    dict(factor=float("nan")), dict(factor=float("inf")), dict(rows=2 ** 31), dict(H=70000, ldq=2 ** 23, ldqo=2 ** 23),
    dict(q=None), dict(qo=None), dict(k=None), dict(ko=None), dict(pos=None), dict(freq=None),
    dict(freq=W + 4), dict(ldq=255), dict(ldqo=255), dict(ldk=127), dict(ldko=127),
    dict(ldq=2 ** 62), dict(ldko=2 ** 61), dict(qo=A + 4), dict(qo=A, ldqo=260), dict(ko=Q + 512),
    dict(qo=Q), dict(ko=A + 256), dict(qo=Z), dict(pos=Y + 8), dict(pos=Z), dict(freq=Y + 2 * 1024),
    dict(freq=Z + 8)])
def test_rope_refused(L, bad):
    assert rope(L, **bad) == 9, bad
    assert "rope_qk" in message(L)


def test_rope_host_refused(L):
    f = np.zeros(64, np.float32)
    p = f.ctypes.data
    assert L.vmlm_rope_qk(p, p, p, p, p, p, 1, 1, 0, 63, 32, False, 1.0) == 9
    assert L.vmlm_rope_qk(p, None, p, None, None, p, 1, 1, 0, 64, 32, False, 1.0) == 9
    assert L.vmlm_rope_qk(None, None, None, None, None, None, 0, 4, 4, 64, 64, True, 1.0) == 0


@pytest.mark.parametrize("empty", [dict(rows=0), dict(H=0, Hkv=0)])
def test_rope_nothing_to_do(L, empty):
    assert rope(L, qo=None, ko=None, q=None, k=None, pos=None, freq=None, **empty) == 0


def test_rope_freqs(L):
    from sparrow_amd import VmlmError, ops
    for kw in (dict(rot_dim=0), dict(rot_dim=7), dict(rot_dim=514), dict(rot_dim=64, theta=0.0),
               dict(rot_dim=64, theta=float("nan")), dict(rot_dim=64, scaling=("linear", 0.5)),
               dict(rot_dim=64, scaling=("bands", 8, 4, 4, 8192)),
               dict(rot_dim=64, scaling=("bands", 8, 0, 4, 8192)),
               dict(rot_dim=64, scaling=("ramp", 8, 1, 4, 0)),
               dict(rot_dim=64, theta=1.0, scaling=("ramp", 8, 1, 4, 8192)),
               dict(rot_dim=64, scaling=("ramp", float("inf"), 1, 4, 8192))):
        with pytest.raises(VmlmError) as e:
            ops.rope_freqs(**kw)
        assert e.value.code == 9, kw
    assert L.vmlm_rope_freqs(None, None, 64, 1e4, None) == 9


@pytest.mark.parametrize("rot,theta", [(2, 10000.0), (20, 10000.0), (64, 500000.0), (128, 1.5)])
def test_rope_freqs_values(L, rot, theta):
    """Each rule against its definition: doubles, a few roundings apart (1e-14)."""
    from sparrow_amd import ops
    i = np.arange(rot // 2)
    base = theta ** (-2.0 * i / rot)

    def same(got, want, factor):
        assert np.abs(got[0] / want - 1).max() < 1e-14 and got[1] == np.float32(factor)
    same(ops.rope_freqs(rot, theta), base, 1)
    same(ops.rope_freqs(rot, theta, ("linear", 4)), base / 4, 1)
    for f, low, high, trained in ((8, 1, 4, 8192), (32, 1, 32, 4096), (2, 0.5, 1.0, 100)):
        n = trained * base / (2 * np.pi)
        keep = np.clip((n - low) / (high - low), 0, 1)
        assert set(keep[n >= high]) <= {1.0} and set(keep[n <= low]) <= {0.0}
        same(ops.rope_freqs(rot, theta, ("bands", f, low, high, trained)),
             base * keep + base / f * (1 - keep), 1)
        at = [rot * np.log(trained / (2 * np.pi * t)) / (2 * np.log(theta)) for t in (high, low)]
        a, b = max(np.floor(at[0]), 0), min(np.ceil(at[1]), rot - 1)
        away = np.clip((i - a) / max(b - a, 1e-3), 0, 1)
        same(ops.rope_freqs(rot, theta, ("ramp", f, low, high, trained)),
             base * (1 - away) + base / f * away, 0.1 * np.log(f) + 1)


# ------------------------------------------------------------------ the cache's operators
def cache(k=A, v=Q, k_meta=S, v_meta=S + 0x1000000, batch=2, n_kv_heads=2, cap=64, head_dim=64):
    from sparrow_amd import _abi
    return _abi.Kv4Cache(k=k, v=v, k_meta=k_meta, v_meta=v_meta, batch=batch,
                         n_kv_heads=n_kv_heads, cap=cap, head_dim=head_dim)


def attend(L, c=None, q=Y, ldq=256, pos0=W, count=W + 64, parent=W + 128, n=5, out=Z, ldo=256, H=4,
           scale=0.125, work=None, bytes_=0):
    return L.vmlm_hip_attention_tree_kv4(cache() if c is None else c, q, ldq, pos0, count, parent, n,
                                         out, ldo, H, scale, work, bytes_, None)


@pytest.mark.parametrize("bad", [
    dict(q=None), dict(out=None), dict(pos0=None), dict(H=3), dict(H=65536 * 2), dict(n=65),
    dict(n=65536, parent=None), dict(ldq=255), dict(ldo=255), dict(scale=float("inf")),
    dict(scale=float("nan")), dict(out=Y), dict(out=Y + 9 * 1024 + 1020), dict(out=A), dict(out=Q + 8),
    dict(out=S), dict(out=S + 0x1000000), dict(pos0=Z + 4), dict(count=Z), dict(parent=Z + 9 * 1024),
    dict(ldq=2 ** 60), dict(ldo=2 ** 61)])
def test_attention_refused(L, bad):
    assert attend(L, **bad) == 9, bad
    assert "tree attention" in message(L)


def test_attention_refused_caches(L):
    for c in (dict(head_dim=48), dict(cap=40), dict(k=None), dict(v=Q + 8), dict(batch=70000),
              dict(cap=0), dict(v=A + 64)):
        assert attend(L, cache(**c)) == 9, c
    assert attend(L, cache(n_kv_heads=0), H=0) == 9


def test_attention_sizes_at_their_limits(L):
    """More rows or heads than a grid takes."""
    far = dict(k=1 << 40, v=2 << 40, k_meta=3 << 40, v_meta=4 << 40)
    need = C.c_size_t()
    for c, H, n in ((dict(batch=64, n_kv_heads=64, cap=32, head_dim=32), 64, 32769),
                    (dict(batch=4096, n_kv_heads=1, cap=32, head_dim=32), 1024, 33),
                    (dict(batch=65535, n_kv_heads=33, cap=32, head_dim=32), 33, 1)):
        c = cache(**far, **c)
        w = H * 32
        assert attend(L, c, q=5 << 40, ldq=w, pos0=W, count=None, parent=None, n=n, out=9 << 40, ldo=w, H=H) == 9
        assert "limit" in message(L) or "2^21" in message(L)
        assert L.vmlm_hip_attention_tree_kv4_work(c, H, n, C.byref(need)) == 9
    # what a workspace holds does not grow with the sequences that are not split
    c = cache(**far, batch=2048, n_kv_heads=32, cap=8192, head_dim=128)
    assert L.vmlm_hip_attention_tree_kv4_work(c, 256, 64, C.byref(need)) == 0 and 0 < need.value < 64 << 20


@pytest.mark.parametrize("empty", [dict(n=0), dict(H=0), dict(c=dict(batch=0))])
def test_attention_nothing_to_do(L, empty):
    if "c" in empty:
        empty = dict(c=cache(**empty["c"]))
    assert attend(L, q=None, out=None, pos0=None if empty.get("H") != 0 else W, **empty) == 0


def test_attention_workspace(L):
    """A workspace that is too small, unaligned or over an operand (capacities where one is used)."""
    c = cache(v=0x1000000000, k_meta=0x2000000000, v_meta=0x3000000000, k=0x4000000000,
              batch=1, cap=1 << 20)
    need = C.c_size_t(1)
    assert L.vmlm_hip_attention_tree_kv4_work(c, 4, 5, C.byref(need)) == 0
    assert L.vmlm_hip_attention_tree_kv4_work(c, 3, 5, C.byref(need)) == 9
    assert L.vmlm_hip_attention_tree_kv4_work(c, 4, 5, None) == 9
    assert L.vmlm_hip_attention_tree_kv4_work(c, 4, 70000, C.byref(need)) == 9
    assert L.vmlm_hip_attention_tree_kv4_work(c, 4, 5, C.byref(need)) == 0
    if need.value == 0:
        return
    for work, n in ((X, need.value - 1), (X + 8, need.value), (Y, need.value), (Z + 16, need.value),
                    (W, need.value), (c.k, need.value), (c.v_meta + 64, need.value)):
        assert attend(L, c, work=work, bytes_=n) == 9, hex(work)
        assert "workspace" in message(L)


def accept(L, c=None, n=None, pos0=W, count=W + 64, parent=W + 0x100, drafted=W + 0x200,
           chosen=W + 0x300, s=5, path=Y, kept=Y + 64, nxt=Y + 128):
    from sparrow_amd import _abi
    c = [cache()] if c is None else c
    arr = (_abi.Kv4Cache * max(1, len(c)))(*c)
    return L.vmlm_hip_tree_accept_kv4(arr, len(c) if n is None else n, pos0, count, parent, drafted,
                                      chosen, s, path, kept, nxt, None)


@pytest.mark.parametrize("bad", [
    dict(n=0), dict(n=257), dict(s=65), dict(pos0=None), dict(drafted=None), dict(chosen=None), dict(path=None),
    dict(kept=None), dict(nxt=None), dict(path=W), dict(kept=W + 64), dict(nxt=W + 0x104),
    dict(path=W + 0x220), dict(kept=W + 0x300), dict(kept=Y + 36), dict(nxt=Y + 66), dict(path=A),
    dict(kept=Q + 16), dict(nxt=S), dict(pos0=S + 0x1000000), dict(drafted=A + 8), dict(count=Q)])
def test_accept_refused(L, bad):
    assert accept(L, **bad) == 9, bad
    assert "tree accept" in message(L)


def test_accept_refused_caches(L):
    far = dict(k=X, v=X + 0x1000000, k_meta=X + 0x2000000, v_meta=X + 0x3000000)
    for second in (dict(far, cap=96), dict(far, batch=1), dict(far, n_kv_heads=1), dict(far, head_dim=32),
                   dict(), dict(far, k=A + 2048), dict(far, v=Q + 64), dict(far, v_meta=S + 4), dict(far, k=None)):
        assert accept(L, [cache(), cache(**second)]) == 9, second
    assert L.vmlm_hip_tree_accept_kv4(None, 1, W, None, None, W, W, 5, Y, Y, Y, None) == 9
    assert accept(L, [cache(cap=0)]) == 9 and accept(L, [cache(n_kv_heads=0)]) == 9


def test_accept_nothing_to_do(L):
    assert accept(L, [cache(batch=0)]) == 0
    assert accept(L, s=0, path=None, kept=None, nxt=None) == 0


# ------------------------------------------------------------------ sample
def draw(L, logits=A, ld=1000, u=Q, t=S, k=W, p=W + 64, m=W + 128, rows=3, vocab=1000, token=Y,
         prob=Z, work=None, bytes_=0):
    return L.vmlm_hip_sample(logits, ld, u, t, k, p, m, rows, vocab, token, prob, work, bytes_, None)


@pytest.mark.parametrize("bad", [
    dict(vocab=0), dict(vocab=2 ** 20), dict(rows=2 ** 20 + 1), dict(logits=None), dict(u=None), dict(t=None),
    dict(token=None), dict(ld=999), dict(ld=2 ** 61), dict(token=Z + 8), dict(token=A + 11996), dict(prob=A),
    dict(token=Q), dict(prob=S + 8), dict(token=W), dict(prob=W + 64), dict(prob=W + 136)])
def test_sample_refused(L, bad):
    assert draw(L, **bad) == 9, bad
    assert "sample" in message(L)


def test_sample_nothing_to_do(L):
    assert draw(L, rows=0, logits=None, u=None, t=None, token=None) == 0


@pytest.mark.parametrize("rows,vocab", [(1, 122753), (16, 122753), (3, 1000)])
def test_sample_workspace(L, rows, vocab):
    need = C.c_size_t(1)
    assert L.vmlm_hip_sample_work(rows, vocab, C.byref(need)) == 0
    assert L.vmlm_hip_sample_work(rows, vocab, None) == 9
    assert L.vmlm_hip_sample_work(rows, 0, C.byref(need)) == 9
    assert L.vmlm_hip_sample_work(2 ** 21, 10, C.byref(need)) == 9
    assert L.vmlm_hip_sample_work(rows, vocab, C.byref(need)) == 0
    if need.value == 0:
        return
    for work, n in ((X, need.value - 1), (X + 4, need.value), (A, need.value), (Y, need.value),
                    (Z, need.value), (Q, need.value), (W, need.value)):
        assert draw(L, rows=rows, vocab=vocab, ld=vocab, work=work, bytes_=n) == 9, hex(work)
        assert "workspace" in message(L)
