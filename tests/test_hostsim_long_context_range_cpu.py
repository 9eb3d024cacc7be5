"""The range tests of window attention and the quantised cache on the CPU: the kernels' own source through tests/hostsim, by the C ABI."""
import pytest
import torch

import test_hostsim_long_context_cpu as sim
import test_zzn_window_attention_gpu as wa
import test_zzp_long_context_range_gpu as rng
from test_hostsim_long_context_cpu import lib  # noqa: F401

pytestmark = sim.pytestmark
BOTH = sim.BOTH


@BOTH
@pytest.mark.parametrize("factor", [1e-3, 8.0, 64.0, 1000.0])
@pytest.mark.parametrize("t,b,h,hk,d,window,sinks,ragged", rng.MAGNITUDES)
def test_values_of_other_magnitudes(lib, t, b, h, hk, d, window, sinks, ragged, factor, dtype):  # noqa: F811
    q, k, v, dout, lengths = rng.scaled_inputs(t, b, h, hk, d, ragged, factor, dtype, "cpu")
    want, mag = wa.reference(*(torch.nan_to_num(x) for x in (q, k, v, dout)), lengths, window, sinks, d ** -0.5)
    wa.check(sim.window(lib, q, k, v, dout, lengths, window, sinks, d ** -0.5, dtype), want, mag, dtype)


@BOTH
@pytest.mark.parametrize("factor", [1e-3, 1.0, 64.0, 1000.0])
@pytest.mark.parametrize("t,b,h,hk,d,window,sinks,ragged", [(100, 1, 2, 1, 64, 48, 0, False), (140, 2, 1, 1, 128, 90, 3, True)])
def test_d_is_that_of_the_output_before_its_rounding(lib, t, b, h, hk, d, window, sinks, ragged, factor, dtype):  # noqa: F811
    data = rng.alike(t, b, h, hk, d, factor, dtype)
    lengths = torch.tensor([t, t - 61][:b], dtype=torch.int32) if ragged else None
    got = sim.window(lib, *data, lengths, window, sinks, d ** -0.5, dtype)
    rng.check_d(got[1:3], *data, lengths, window, sinks, d ** -0.5)
    with pytest.raises(AssertionError, match="dq"):            # the check tells the two apart
        rng.check_d(sim.window(lib, *data, lengths, window, sinks, d ** -0.5, dtype, keep_rest=False)[1:3], *data, lengths, window, sinks, d ** -0.5)


def test_smallest_and_largest_outputs(lib):  # noqa: F811
    """Outputs below the normal range of the type, in which every rounding is as large as any, and the largest of bf16."""
    for dtype, factor in ((torch.float16, 2.0 ** -22), (torch.bfloat16, 2.0 ** -125), (torch.bfloat16, 2.0 ** 120)):
        q, k, v, dout, _ = rng.scaled_inputs(70, 1, 1, 1, 64, False, factor, dtype, "cpu")
        dout = dout * 2.0 ** -20 if factor > 1 else dout
        got = sim.window(lib, q, k, v, dout, None, 20, 2, 0.125, dtype)
        assert all(torch.isfinite(x).all() for x in got)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype,d,lengths", [(torch.float16, 64, [70, 33]), (torch.float16, 128, [70, 2]), (torch.bfloat16, 128, [1, 1])])
def test_finite_values_are_attended_to_as_finite(lib, dtype, d, lengths, bits):  # noqa: F811
    cap = max(lengths)
    k, v, seen, q, scale = rng.top_of_the_type(cap, 2, 2, d, bits, dtype)
    cache = sim.qc.buffers(2, 2, cap, d, bits, "cpu")
    sim.write(lib, cache, k, v, None, 0)
    want, mag = sim.qc.attend_reference(q, *seen, lengths, 0, 0, scale)
    rng.check_attend(sim.attend(lib, q, cache, torch.tensor(lengths, dtype=torch.int32), cap, 0, 0, scale), want, mag, dtype,
                     lengths, torch.finfo(dtype).max)
    # a block that is not finite is still NaN, and no other
    v[0, 0, 0, 3] = float("inf")
    sim.write(lib, cache, k, v, None, 0)
    out = sim.attend(lib, q, cache, torch.tensor(lengths, dtype=torch.int32), cap, 0, 0, scale)
    assert torch.isnan(out[0, 0, :2, :32]).all() and torch.isfinite(out[0, 0, :2, 32:]).all() and torch.isfinite(out[0, 0, 2:]).all()


def test_one_position_has_no_stride(lib):  # noqa: F811
    q, k, v, dout = wa.inputs(1, 2, 2, 1, 64, torch.bfloat16, "cpu")
    out, rest, lse = torch.empty_like(q), sim.rest_of(q), torch.empty(2, 2, 1)
    grads = [torch.empty_like(x) for x in (q, k, v)]
    views = lambda *ts: (sim.ctypes.c_int64 * (3 * len(ts)))(*(s for x in ts for s in ((1 << 24) + 3, *x.stride()[1:3])))     # noqa: E731
    sizes = (1, 2, 2, 1, 64, 4, 1)
    sim.call(lib, "window_attn_fwd", q, k, v, out, rest, lse, None, views(q, k, v, out), *sizes, 0.125, sim._lib.BF16)
    ws = sim.bytes256(sim.call(lib, "window_attn_bwd_workspace_bytes", *sizes))
    sim.call(lib, "window_attn_bwd", dout, q, k, v, out, rest, lse, *grads, None, views(dout, q, k, v, out, *grads), *sizes, 0.125, sim._lib.BF16, ws, ws.numel())
    assert torch.equal(out, v.expand_as(q))
    wa.check((out, *grads), *wa.reference(q, k, v, dout, None, 4, 1, 0.125), torch.bfloat16)


def test_launches_beyond_32_bits_are_refused(lib):  # noqa: F811
    """A launch holds less than 2^32 threads: 2^24 blocks of 256. Refused before anything runs, the backward's later launches too."""
    x = torch.zeros(64, dtype=torch.bfloat16)
    st = lambda n: (sim.ctypes.c_int64 * (3 * n))(*([0, 64, 64] * n))                       # noqa: E731
    lse = torch.zeros(1)
    for sizes in ((1, 60000, 300, 300, 64, 4, 0), (1 << 20, 2, 60000, 60000, 64, 4, 0)):
        assert "too many blocks" in sim.call(lib, "window_attn_fwd", x, x, x, x, None, lse, None, st(4), *sizes, 0.125, sim._lib.BF16, expect=-1)
    # the forward fits, the chunks and parts of dK and dV do not
    sizes = (8192, 128, 1024, 1024, 64, 1, 8192)
    ws = sim.bytes256(256)
    huge = sim.call(lib, "window_attn_bwd_workspace_bytes", *sizes)
    assert "too many blocks" in sim.call(lib, "window_attn_bwd", x, x, x, x, x, None, lse, x, x, x, None, st(8), *sizes, 0.125, sim._lib.BF16, ws, huge, expect=-1)
    # rows of a broadcast key written to 2^31 - 1 positions
    codes, scales = torch.zeros(64, dtype=torch.uint8), torch.zeros(2, dtype=torch.uint8)
    n = (1 << 30) - 1
    assert "too many rows" in sim.call(lib, "kv_cache_write", x, 0, 0, 0, x, 0, 0, 0, codes, scales, codes, scales, None, 0, n, 4, 1, 64, n, 8, sim._lib.BF16, expect=-1)
