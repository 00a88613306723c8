"""By parts is the schedule whose ramp is linear in the turns that a pair makes over the trained context; one that is linear in the
pair's index agrees with it outside the ramp and differs inside it. No kernel is launched."""
import ctypes as C
import math

import numpy as np
import pytest


@pytest.mark.parametrize("theta,rot,context,factor", [(1e4, 128, 4096.0, 4.0), (1e6, 64, 32768.0, 8.0), (1e4, 100, 2048.0, 2.0)])
def test_by_parts_ramps_in_turns(qh, theta, rot, context, factor):
    low, high = 1.0, 32.0
    got = np.empty(rot // 2)
    desc = qh.qh_rope_desc(theta, rot, qh.ROPE_PARTS, factor, context, low, high)
    assert qh.lib().qh_rope_turns(C.byref(desc), got.ctypes.data) == 0
    plain = np.array([theta ** (-2 * i / rot) / math.tau for i in range(rot // 2)])
    made = context * plain
    keep = np.clip((made - low) / (high - low), 0, 1)
    assert np.allclose(got, plain * (keep + (1 - keep) / factor), rtol=1e-14, atol=0)
    # by index: the ends are the pairs (not whole) that make `high` and `low` turns
    first, last = (rot * math.log(context / (n * math.tau)) / (2 * math.log(theta)) for n in (high, low))
    other = np.clip((last - np.arange(rot // 2)) / (last - first), 0, 1)
    by_index = plain * (other + (1 - other) / factor)
    ramp = (made > low) & (made < high)
    assert np.allclose(got[~ramp], by_index[~ramp], rtol=1e-12, atol=0) and ramp.sum() > 5
    assert (np.abs(got[ramp] / by_index[ramp] - 1) > 1e-3).all()
