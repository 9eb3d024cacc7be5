"""The range tests of window attention and the quantised cache on the CPU: the kernels' own source through tests/hostsim, by the C ABI."""
import pytest
import torch

import test_hostsim_long_context_cpu as sim
import test_zzp_long_context_range_gpu as rng
from test_hostsim_long_context_cpu import lib  # noqa: F401

pytestmark = sim.pytestmark
BOTH = sim.BOTH


@BOTH
@pytest.mark.parametrize("factor", [0.1])
@pytest.mark.parametrize("t,b,h,hk,d,window,sinks,ragged", [(100, 1, 2, 1, 64, 48, 0, False), (140, 2, 1, 1, 128, 90, 3, True)])
def test_d_is_that_of_the_output_before_its_rounding(lib, t, b, h, hk, d, window, sinks, ragged, factor, dtype):  # noqa: F811
    data = rng.alike(t, b, h, hk, d, factor, dtype)
    lengths = torch.tensor([t, t - 61][:b], dtype=torch.int32) if ragged else None
    got = sim.window(lib, *data, lengths, window, sinks, d ** -0.5, dtype)
    rng.check_d(got[1:3], *data, lengths, window, sinks, d ** -0.5)
    with pytest.raises(AssertionError, match="dq"):            # the check tells the two apart
        rng.check_d(sim.window(lib, *data, lengths, window, sinks, d ** -0.5, dtype, keep_rest=False)[1:3], *data, lengths, window, sinks, d ** -0.5)
