"""Limits of the descriptions of attention behind one shared prefix, on the CPU: the values next to them."""
import ctypes

import pytest

from test_shared_plan import make


def refused(qattn, desc):
    """The message of the refusal, or None."""
    try:
        qattn.shared_plan(desc)
    except qattn.QattnError as e:
        assert e.code == qattn.EINVAL
        return str(e)
    return None


@pytest.mark.parametrize("scale,fine", [
    (5e-324, False), (1e-100, False), (1e-46, False), (4.8e-46, False),  # times log2 e below half of 2^-149: 0 in f32
    (4.9e-46, True), (1e-45, True), (1e-40, True), (1e-30, True), (0.0, True), (9.9e29, True), (1e30, False)])
def test_scales_that_vanish_in_f32_are_refused(qattn, scale, fine):
    """A masked score is -inf; times a scale of 0 it would be NaN."""
    message = refused(qattn, make(qattn, 100, [3, 1], [5, 70], scale=scale)[0])
    assert (message is None) == fine, message
    assert fine or "scale" in message


def planned(qattn, prefix, queries, own, **kw):
    n, info = ctypes.c_int64(0), qattn.SharedInfo()
    desc = make(qattn, prefix, queries, own, **kw)[0]
    qattn._check(qattn.lib().qattn_shared_plan_describe(ctypes.byref(desc), None, 0, ctypes.byref(n), ctypes.byref(info)))
    return info


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("form", [0, 1, 2])
@pytest.mark.parametrize("queries", [1, 16, 128, 256])
def test_what_has_one_place_is_not_cut(qattn, dim, form, queries):
    """With 256 KV heads each has one of the chip's 256 places, so cutting an item gains nothing and costs a merge:
    one item of 16, 128 or 256 rows, however many tiles it has."""
    for tiles in range(1, 401):
        info = planned(qattn, 128 * tiles, [queries], [queries], heads=256, kv=256, dim=dim, form=form, paged=False)
        assert (info.items, info.merged_rows, info.partial_rows) == (1, 0, 0), (tiles, info.as_dict())


@pytest.mark.parametrize("form", [0, 1, 2])
def test_blocks_that_fill_the_chip_are_not_cut(qattn, form):
    """64 prompts of 64 tokens: 32 blocks of 256 rows a KV head, for 32 places, behind any prefix."""
    for prefix in (50, 100, 128, 200, 256, 300, 900, 1500, 2500, 5000):
        info = planned(qattn, prefix, [64] * 64, [64] * 64, form=form, paged=False)
        assert (info.items, info.merged_rows) == (32, 0), (prefix, info.as_dict())


def test_as_many_sequences_as_elsewhere(qattn):
    """65,536 sequences, as for the other launches; one more is refused."""
    assert planned(qattn, 20, [1] * 65536, [1] * 65536).tokens == 65536
    message = refused(qattn, make(qattn, 20, [1] * 65537, [1] * 65537)[0])
    assert message and "nseq=65537" in message and "65536" in message


def test_limits_that_the_header_states(qattn):
    """A launch has fewer than 2^23 workgroups, and merges fewer than 2^23 rows, over all KV heads."""
    queries = [1] * 65536
    assert planned(qattn, 100, queries, queries, heads=63 * 2, kv=63, page=16).merged_rows == 1 << 17
    message = refused(qattn, make(qattn, 100, queries, queries, heads=64 * 2, kv=64, page=16)[0])
    assert message and "too many rows for one launch" in message
