"""How 4-bit weights are rounded on the host: no value further off than a rounding, whichever sign a group's largest has."""
import numpy as np
import pytest

import juliavision_b200 as jv
from tests import decode_ref as ref


@pytest.mark.parametrize("group, most", [(32, 0.0935), (64, 0.0985), (128, 0.1060)])
def test_the_largest_weights_are_within_half_a_step(group, most):
    """Half a step and the scale's rounding to fp16, 2^-11 of up to eight and a half steps; and the whole no further off than where the largest stands at 8 and
    is cut to 7 (0.0938, 0.0990, 0.1056 of these values' 2-norm; for 128 with room for the sample)."""
    rng = np.random.default_rng(0)
    W = rng.standard_normal((256, 500)).astype(np.float16)
    W[:, 3] = np.abs(W[:, 3])
    W[:, 4] = -np.abs(W[:, 4])
    W[:group, 5] = 0
    W[:group, 6] = 0
    W[0, 6] = 1
    q, s, z = jv.quantise4(W, group)
    assert z is None and q.max() <= 15
    off = np.abs(ref.weight4(q, s, None, group) - W.astype(np.float64))
    step = np.abs(np.repeat(s.astype(np.float64), group, 0))
    assert np.all(off <= step * (0.5 + 8.5 * 2.0 ** -11))
    assert np.linalg.norm(off) <= most * np.linalg.norm(W.astype(np.float64))


@pytest.mark.parametrize("symmetric, most", [(True, 7 * 65519.0), (False, 15 * 65519.0)])
def test_weights_whose_scale_passes_fp16_are_refused(symmetric, most):
    """65520 rounds to infinity in fp16, and 0 times infinity is no weight; below it every weight is a number."""
    W = np.zeros((64, 3), np.float32)
    W[5, 1] = most
    q, s, z = jv.quantise4(W, 64, symmetric)
    assert np.isfinite(s).all() and abs(ref.weight4(q, s, z, 64)[5, 1] / most - 1) < 2.0 ** -4
    W[5, 1] = most * 1.001
    with pytest.raises(jv.B200Error) as e:
        jv.quantise4(W, 64, symmetric)
    assert e.value.code == 1
