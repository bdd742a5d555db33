"""4-bit weights on the host: the image that the products read, quantising, Q4_0 tensors, refusals (CPU)."""
import ctypes

import numpy as np
import pytest

import w4_ref

rng_of = np.random.default_rng
SHAPES = [(1, 32), (1, 65536), (15, 96), (16, 128), (17, 160), (40, 1024), (333, 224)]


@pytest.mark.parametrize("N,K", SHAPES)
def test_image_is_as_described(qattn, N, K):
    codes, groups, scales = w4_ref.random_weights(rng_of(N + K), N, K)
    packed = qattn.w4_pack(w4_ref.nibbles(codes), groups, scales)
    assert packed.nbytes == qattn.lib().qattn_w4_bytes(K, N) == -(-N // 16) * (-(-K // 128) * 1088 + 64)
    assert np.array_equal(packed, w4_ref.image(codes, groups, scales))
    back = w4_ref.taken_apart(packed, K, N)
    assert all(np.array_equal(a, b) for a, b in zip(back, (codes, groups, scales)))


def test_padding_is_zero_weights_whatever_was_there(qattn):
    """Multipliers of the padding's groups are zero, also in an image that held something else."""
    N, K = 3, 32
    codes, groups, scales = w4_ref.random_weights(rng_of(1), N, K)
    out = np.full(qattn.lib().qattn_w4_bytes(K, N), 0xFF, np.uint8)
    nib = w4_ref.nibbles(codes)
    qattn._check(qattn.lib().qattn_w4_pack(nib.ctypes.data, groups.ctypes.data, scales.ctypes.data, K, N, out.ctypes.data, out.nbytes))
    assert np.array_equal(out, w4_ref.image(codes, groups, scales))
    out[:] = 0xFF
    w = rng_of(2).standard_normal((N, K)).astype(np.float32)
    qattn._check(qattn.lib().qattn_w4_quantize(w.ctypes.data, K, K, N, out.ctypes.data, out.nbytes))
    assert np.array_equal(out, qattn.w4_quantize(w))


def test_every_pair_that_fits_is_taken_and_no_other(qattn):
    codes, scale = np.zeros((1, 16), np.uint8), np.ones(1, np.float32)
    fitting = set(w4_ref.pairs().tolist())
    for b in range(256):
        m, z = b & 15, b >> 4
        group = np.array([[b]], np.uint8)
        if b in fitting:
            assert -128 <= -z * m and (15 - z) * m <= 127
            qattn.w4_pack(codes, group, scale)
        else:
            with pytest.raises(qattn.QattnError) as e:
                qattn.w4_pack(codes, group, scale)
            assert e.value.code == qattn.EINVAL and "8 bits" in str(e.value)


def some_rows(rng, N, K):
    w = rng.standard_normal((N, K)) * np.exp(0.7 * rng.standard_normal((N, K // 32, 1))).repeat(32, 1).reshape(N, K)
    w = w.astype(np.float32)
    w[0, :32] = 0                                   # a group of zeros
    if N > 1:
        w[1] = 0                                    # a row of zeros
    if N > 2:
        w[2] *= np.float32(2.0 ** -80)              # small, but a row
    if N > 3:
        w[3] = np.float32(2.0 ** -120)              # next to nothing
    if N > 4:
        w[4, :32], w[4, 32:] = 0.01, 50             # groups that a multiplier of 15 steps cannot tell apart
    if N > 5:
        w[5, ::2], w[5, 1::2] = 1.0, -1.0           # ties: the first value decides the zero point
    if N > 6:
        w[6] *= np.float32(1e38) / np.abs(w[6]).max()
    return w


@pytest.mark.parametrize("N,K", [(1, 32), (8, 64), (19, 160), (7, 4096)])
def test_quantize(qattn, N, K):
    w = some_rows(rng_of(N * K), N, K)
    got = w4_ref.taken_apart(qattn.w4_quantize(w), K, N)
    want = w4_ref.quantize(w)
    for a, b in zip(got, want):
        assert np.array_equal(a, b)
    assert set(np.unique(got[1])) <= set(w4_ref.pairs().tolist())
    # With the larger multiplier tried, which takes the value of the largest magnitude within 8 steps (1 + 2^-23), a
    # value is off by at most half a step, or by one where it is as large with the other sign, whose codes end at 7.
    W = w4_ref.values(*got)
    step = np.abs(got[2].astype(np.float64))[:, None]
    group = np.abs(w.astype(np.float64)).reshape(N, -1, 32).max(-1).repeat(32, 1)
    larger = step * np.clip(np.floor(group / 8 / np.where(step, step, 1)) + 1, 1, 15)
    squares = ((W - w) ** 2).reshape(N, -1, 32).sum(-1)
    live = np.abs(w).max(-1) >= 2.0 ** -100
    assert (squares <= 32 * (larger[:, ::32] * (1 + 1e-6)) ** 2)[live].all()
    assert (W[~live] == 0).all()


@pytest.mark.parametrize("N,K", [(32, 32), (50, 96), (33, 1024)])
def test_from_q4(qattn, oracle, N, K):
    rng = rng_of(N)
    tiles = -(-N // 32)
    rec = rng.integers(0, 256, (tiles, K // 32, 32, 20)).astype(np.uint8)
    scale = (rng.standard_normal((tiles, K // 32, 32)) * 0.02).astype(np.float16)
    scale[0, 0, 0], scale[0, 0, 1] = 0, np.float16(6e-8)  # none, the least
    rec[..., 0:2] = scale[..., None].view(np.uint8)
    packed = rec.reshape(-1)
    got = qattn.w4_from_q4(packed, K, N)
    # f32(scale) * (q - 8) is exact in f32
    q = rec[..., 4:20]
    vals = np.concatenate([(q & 15).astype(np.float32) - 8, (q >> 4).astype(np.float32) - 8], -1) * scale[..., None].astype(np.float32)
    w = vals.transpose(0, 2, 1, 3).reshape(-1, K)[:N]
    assert np.array_equal(got, qattn.w4_quantize(w))
    assert np.array_equal(w.astype(np.float16), oracle.q40_compact_weights(packed, K, N))


def test_from_q4_changes_a_models_weights_by_a_few_percent(qattn):
    """Normal values through Q4_0 (the value of the largest magnitude at -8 steps) and on: a group's scale becomes
    a multiple of a fifteenth of the row's largest, off by at most half of one; 3 % of the weights' size here."""
    rng = rng_of(5)
    N, K = 64, 1024
    w = rng.standard_normal((N, K // 32, 32))
    a = np.take_along_axis(w, np.abs(w).argmax(-1)[..., None], -1)
    d = (a / -8).astype(np.float16)
    q = np.clip(np.rint(w / d.astype(np.float64)) + 8, 0, 15)
    q4 = (d.astype(np.float64) * (q - 8)).reshape(N, K)
    W = w4_ref.values(*w4_ref.taken_apart(qattn.w4_quantize(q4.astype(np.float32)), K, N))
    size = np.sqrt((w ** 2).mean())
    added, left_out = np.sqrt(((W - q4) ** 2).mean()) / size, np.sqrt(((q4 - w.reshape(N, K)) ** 2).mean()) / size
    print(f"Q4_0 leaves out {left_out:.4f} of the weights' size, the whole-number scales {added:.4f}")
    assert 0.06 < left_out < 0.09 and added < 0.05


def test_refusals(qattn):
    L = qattn.lib()
    for K, N in ((0, 1), (31, 1), (48, 1), (-32, 4), (65568, 1), (32, 0), (32, -1), (32, (1 << 22) + 1)):
        assert L.qattn_w4_bytes(K, N) == -1
        with pytest.raises(qattn.QattnError):
            qattn.w4_quantize(np.zeros((max(N, 0), max(K, 0)) if N < 1 << 20 else (1, 33), np.float32))
    N, K = 2, 64
    codes, groups, scales = w4_ref.random_weights(rng_of(0), N, K)
    nib, out = w4_ref.nibbles(codes), np.full(L.qattn_w4_bytes(K, N), 7, np.uint8)
    w, q4 = np.ones((N, K), np.float32), np.zeros(L.qattn_q4_compact_bytes(K, N), np.uint8)

    def at(a):
        return None if a is None else a.ctypes.data

    def pack(c=nib, g=groups, s=scales, k=K, n=N, o=out, size=out.nbytes):
        return L.qattn_w4_pack(at(c), at(g), at(s), k, n, at(o), size)

    def quantize(x=w, stride=K, k=K, n=N, o=out, size=out.nbytes):
        return L.qattn_w4_quantize(at(x), stride, k, n, at(o), size)

    def from_q4(x=q4, x_size=q4.nbytes, k=K, n=N, o=out, size=out.nbytes):
        return L.qattn_w4_from_q4(at(x), x_size, k, n, at(o), size)

    bad_scale, bad_weight = scales.copy(), w.copy()
    bad_scale[1], bad_weight[1, 63] = np.inf, np.nan
    bad_q4 = q4.copy()
    bad_q4[20:22] = np.array([np.inf], np.float16).view(np.uint8)  # row 1, group 0
    calls = [lambda: pack(c=None), lambda: pack(g=None), lambda: pack(s=None), lambda: pack(o=None), lambda: pack(k=48),
             lambda: pack(n=0), lambda: pack(size=out.nbytes - 1), lambda: pack(s=bad_scale),
             lambda: pack(g=np.full_like(groups, 0x9F)), lambda: quantize(x=None), lambda: quantize(o=None),
             lambda: quantize(stride=K - 1), lambda: quantize(k=33), lambda: quantize(size=0), lambda: quantize(x=bad_weight),
             lambda: from_q4(x=None), lambda: from_q4(o=None), lambda: from_q4(x_size=q4.nbytes - 1), lambda: from_q4(n=-1),
             lambda: from_q4(size=out.nbytes - 1), lambda: from_q4(x=bad_q4)]
    for i, call in enumerate(calls):
        assert call() == qattn.EINVAL, i
        assert len(L.qattn_last_error(None)) > 10, i
        assert (out == 7).all(), i  # a refused call leaves the image as it was
    assert pack() == quantize() == from_q4() == 0
    with pytest.raises(ValueError):
        qattn.w4_pack(nib, groups[:, :1], scales)
    with pytest.raises(ValueError):
        qattn.w4_pack(nib, groups, scales[:1])
    assert isinstance(ctypes.c_int64(L.qattn_w4_bytes(65536, 1 << 22)).value, int)
