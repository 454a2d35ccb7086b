"""Rotation of rows of more heads than one launch takes workgroups for. Tolerances are those
of test_gpu_draft.py."""
import numpy as np
import pytest
from test_gpu_4bit import ops  # noqa: F401
from test_gpu_draft import rope_ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("H,Hkv", [(65535, 300), (300, 65535)])
@pytest.mark.parametrize("inter", [False, True])
def test_rope_more_heads_than_a_launch(ops, H, Hkv, inter):
    """255 pairs a head: past 65535 workgroups of 256 threads a row."""
    rng = np.random.default_rng(H)
    hd, pos = 510, np.array([12345], np.int32)
    q, k = (rng.standard_normal((1, h * hd), dtype=np.float32) for h in (H, Hkv))
    freq, factor = ops.rope_freqs(hd)
    for x, y in zip((q, k), ops.rope_qk(q, k, pos, freq, hd, inter, factor)):
        ref, tol = rope_ref(x, pos, freq, hd, inter, factor)
        assert (np.abs(y - ref) <= tol).all()
