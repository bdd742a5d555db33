"""4-bit weights on the host: an image is not written over what it is made from (CPU)."""
import numpy as np
import pytest

import w4_ref

N, K = 40, 256


def sources(qattn):
    """{name: (the source arrays, the call with their addresses)}"""
    L = qattn.lib()
    codes, groups, scales = w4_ref.random_weights(np.random.default_rng(3), N, K)
    q4 = np.zeros(L.qattn_q4_compact_bytes(K, N), np.uint8)
    q4.reshape(-1, 20)[:, 0:2] = np.array([0.01], np.float16).view(np.uint8)
    rows = np.random.default_rng(4).standard_normal((N, K + 8)).astype(np.float32)
    return {
        "codes": ([w4_ref.nibbles(codes), groups, scales], lambda c, g, s, out, size: L.qattn_w4_pack(c, g, s, K, N, out, size)),
        "rows": ([rows], lambda w, out, size: L.qattn_w4_quantize(w, K + 8, K, N, out, size)),
        "q4": ([q4], lambda q, out, size: L.qattn_w4_from_q4(q, q4.nbytes, K, N, out, size)),
    }


@pytest.mark.parametrize("kind,which", [("codes", 0), ("codes", 1), ("codes", 2), ("rows", 0), ("q4", 0)])
def test_image_over_its_source_is_refused(qattn, kind, which):
    arrays, call = sources(qattn)[kind]
    need = qattn.lib().qattn_w4_bytes(K, N)
    size = arrays[which].nbytes - (32 if kind == "rows" else 0)  # a last row ends with its K columns
    arena = np.zeros(2 * need + size, np.uint8)
    arena[need:need + size] = arrays[which].reshape(-1).view(np.uint8)[:size]
    base = arena.ctypes.data
    given = [base + need if i == which else a.ctypes.data for i, a in enumerate(arrays)]
    before = arena.copy()
    for at in (1, need // 2, need - 1, need, need + 1, need + size - 1):
        assert call(*given, base + at, need) == qattn.EINVAL, at
        assert b"overlap" in qattn.lib().qattn_last_error(None)
        assert np.array_equal(arena, before), at
    # right before and right behind it
    want = np.zeros(need, np.uint8)
    assert call(*given, want.ctypes.data, need) == 0
    for at in (0, need + size):
        assert call(*given, base + at, need) == 0
        assert np.array_equal(arena[at:at + need], want)
        assert np.array_equal(arena[need:need + size], before[need:need + size])
