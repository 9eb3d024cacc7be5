"""Linear attention and the norms with rotation at the ends of their range and precision, executed on the CPU: the kernels' own source through tests/hostsim, called by the
C ABI, against the definition in 64 bits."""
import pytest
import torch

import test_zzr_linear_attention_gpu as la
import test_zzs_linear_states_gpu as ends
import test_zzt_norm_calls_gpu as calls
from test_hostsim_linear_attention_cpu import linear, norm
from test_hostsim_long_context_cpu import hostsim_build, lib      # noqa: F401 (a fixture among them)

pytestmark = pytest.mark.skipif(not hostsim_build.available(), reason="no clang++ to build the CPU simulator")
F16, BF16 = torch.float16, torch.bfloat16


@pytest.mark.parametrize("t,d", [(40, 64), (100, 128)])
@pytest.mark.parametrize("size", [1e24, 1e28, 3e37])
def test_large_states_meet_small_rows_in_fp16(lib, t, d, size):     # noqa: F811
    """A state of a finite size stays finite whatever the rows behind it are: zeros, or some that grow again."""
    (q, k, v, dout), (s0, dlast) = la.inputs(t, 1, 6, d, F16, "cpu", 21)
    s0, dlast = s0.clamp(-3, 3) * size, dlast.clamp(-3, 3) * size
    ld = la.decays(6)
    for rows in (torch.zeros(t), (torch.arange(t) >= 33).float(), (torch.arange(t) < 7).float() * 2.0 ** -20):
        vv, gg = (x * rows.to(F16)[:, None, None, None] for x in (v, dout))
        got = linear(lib, q, k, vv, gg, ld, None, 1.0, F16, s0, dlast, True)
        want, mag = la.reference(q, k, vv, gg, ld, None, 1.0, s0, dlast)
        la.check({n: got[n] for n in ("last", "dstate")}, want, mag)


@pytest.mark.parametrize("size", [1e10, 1e30])
def test_large_columns_leave_small_ones_their_bits_in_fp16(lib, size):     # noqa: F811
    (q, k, v, dout), (s0, dlast) = la.inputs(70, 1, 6, 64, F16, "cpu", 22)
    for x in (s0, dlast):
        x[..., 3] *= size
    ld = la.decays(6)
    got = linear(lib, q, k, v, dout, ld, None, 1.0, F16, s0, dlast, True)
    want, mag = la.reference(q, k, v, dout, ld, None, 1.0, s0, dlast)
    la.check({n: got[n] for n in ("last", "dstate")}, want, mag)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("states", [0.0, 1.0])
@pytest.mark.parametrize("t,d", [(5, 64), (200, 64), (130, 128), (1100, 64)])
def test_states_have_their_bits(lib, t, d, states, dtype):     # noqa: F811
    rows, (s0, dlast), ld = ends.few_rows(t, 3, d, dtype, "cpu", states)
    got = linear(lib, *rows, ld, None, 0.3, dtype, s0, dlast, True)
    want, mag = la.reference(*rows, ld, None, 0.3, s0, dlast)
    ends.check_bits({n: got[n] for n in ("last", "dstate")}, want, mag)


@pytest.mark.parametrize("dtype,size", [(BF16, 1e12), (BF16, 1e-12), (F16, 200.0), (F16, 1e-3)])
def test_magnitudes(lib, dtype, size):     # noqa: F811
    rows, scale, ld = ends.magnitudes(dtype, size, "cpu")
    got = linear(lib, *rows, ld, None, scale, dtype, states=True)
    want, mag = la.reference(*rows, ld, None, scale)
    ends.check_by_type({n: x for n, x in got.items() if x.dtype != F16 or want[n].abs().max() < 6e4}, want, mag)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_magnitudes_of_norms(lib, dtype):     # noqa: F811
    x, pos = calls.magnitudes(dtype, "cpu"), calls.tables(8, 64, "cpu")
    g = torch.ones_like(x)
    out, grads, _ = norm(lib, x, x, g, g, [None, None], *pos, None, dtype)
    want, mag = calls.reference(x, None, g, *pos, calls.rows_of(len(x), 1, None), 1e-6)
    calls.check_by_type("out", out[0], want[0], mag[0])
    calls.check_by_type("dx", grads[0], want[1], mag[1])
