"""Limits of the descriptions of attention behind one shared prefix, on the CPU: the values next to them."""
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
