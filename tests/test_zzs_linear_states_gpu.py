"""Linear attention at the ends of the range of its numbers and at the ends of its precision, against the definition in 64 bits.

Tolerances: those of test_zzr_linear_attention_gpu.py, but with an absolute part that goes by the result's type (SLACK), so that small results
are held to their own size, and for states BITS, which tells 24 bits from 16:

A state to which two rows of values add, in units of 2^-24 of the sum of the terms' magnitudes. What is added, a value times its weight, in two
numbers of fp16 or three of bf16: 4 (2^-22) or 1. Two additions of either row's parts at the state's own size, rounded by the matrix cores, whose
rounding is not said to be to nearest: 2 each, 8. The weight: three exponentials (2 each, 2^-23 being their error), their arguments (products with
a decay whose own rounding counts with it, of weights that are 2^-4 at least: 3 ln 2 * 4 = 8), five products: 19. A sequence in segments: four sums of a product
with an exponential and a rounding each, 20. A gradient: its division and its product with the scale, and one more, 3. In all 54 at most, of which 64 are
granted: 2^-18. Two numbers of bf16 where three are meant are off by up to 2^-17 in either row, and
found to be by 1.9 of the bound.
"""
import pytest
import torch

from nmtgminor_amd.modules.linear_attention import linear_attn_func
from test_zzr_linear_attention_gpu import U, check, decays, inputs, reference

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16
BITS = 2.0 ** -18
# fp16 rounds its smallest values absolutely; the others' smallest normal number, below which products may be flushed
SLACK = {F16: 2.0 ** -25, BF16: 2.0 ** -126, torch.float32: 2.0 ** -126}


def check_by_type(got, want, mag):
    for name, x in got.items():
        u, slack = U[x.dtype], SLACK[x.dtype]
        x = x.detach().cpu().double()
        assert x.shape == want[name].shape and torch.isfinite(x).all(), name
        worst = ((x - want[name]).abs() / ((u + 1e-5) * mag[name] + u * want[name].abs() + slack)).max().item()
        assert worst <= 1.0, f"{name}: {worst:.3f} of the bound"


def few_rows(t, h, d, dtype, dev, states):
    """-> rows, states, decays: values and output gradients that are zero but for two positions, decays of less than four powers of two in all"""
    (q, k, v, dout), (s0, dlast) = inputs(t, 1, h, d, dtype, dev, 23)
    kept = torch.zeros(t, 1, 1, 1, dtype=dtype)
    kept[[t // 3, t - 2]] = 1
    kept = kept.to(dev)
    ld = -torch.linspace(0.3, 2.6, h, device=dev) / t
    return (q, k, v * kept, dout * kept), (s0 * states, dlast * states), ld


def check_bits(got, want, mag):
    for name, x in got.items():
        assert x.dtype == torch.float32
        worst = ((x.detach().cpu().double() - want[name]).abs() / (BITS * mag[name] + 2.0 ** -126)).max().item()
        assert worst <= 1.0, f"{name}: {worst:.3f} of the bound"


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("states", [0.0, 1.0])
@pytest.mark.parametrize("t,d", [(5, 64), (32, 128), (200, 64), (130, 128), (1100, 64), (1500, 128)])
def test_states_have_their_bits(dev, t, d, states, dtype):
    (q, k, v, dout), (s0, dlast), ld = few_rows(t, 3, d, dtype, dev, states)
    s0.requires_grad_()
    out, last = linear_attn_func(q, k, v, ld, scale=0.3, state=s0, return_state=True)
    dstate, = torch.autograd.grad((out, last), s0, (dout, dlast))
    want, mag = reference(q, k, v, dout, ld, None, 0.3, s0, dlast)
    check_bits(dict(last=last, dstate=dstate), want, mag)


def magnitudes(dtype, size, dev):
    (q, k, v, dout), _ = inputs(90, 1, 2, 64, dtype, dev, 7)
    return (q * size, k * size, v, dout), min(max(0.125 / size ** 2, 1e-6), 1e6), decays(2, dev)


@pytest.mark.parametrize("dtype,size", [(BF16, 1e12), (BF16, 1e-12), (F16, 200.0), (F16, 1e-3)])
def test_magnitudes(dev, dtype, size):
    """Every result to its own size; in fp16 those within its range."""
    (q, k, v, dout), scale, ld = magnitudes(dtype, size, dev)
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    out, last = linear_attn_func(*leaves, ld, scale=scale, return_state=True)
    got = dict(zip(("out", "last", "dq", "dk", "dv"), (out, last, *torch.autograd.grad(out, leaves, dout))))
    want, mag = reference(q, k, v, dout, ld, None, scale)
    check_by_type({n: x for n, x in got.items() if x.dtype != F16 or want[n].abs().max() < 6e4}, want, mag)


@pytest.mark.parametrize("t,d", [(40, 64), (100, 128), (1500, 128), (1100, 64)])
@pytest.mark.parametrize("size", [1e24, 1e28, 3e37])
def test_large_states_meet_small_rows_in_fp16(dev, t, d, size):
    """A state of a finite size stays finite whatever the rows behind it are: zeros, or some that grow again."""
    (q, k, v, dout), (s0, dlast) = inputs(t, 1, 3, d, F16, dev, 21)
    s0, dlast = s0.clamp(-3, 3) * size, dlast.clamp(-3, 3) * size
    ld = decays(6, dev)[:3].contiguous()
    s0.requires_grad_()
    for rows in (torch.zeros(t), (torch.arange(t) >= 33).float(), (torch.arange(t) < 7).float() * 2.0 ** -20):
        vv, gg = (x * rows.to(F16).to(dev)[:, None, None, None] for x in (v, dout))
        out, last = linear_attn_func(q, k, vv, ld, scale=1.0, state=s0, return_state=True)
        dstate, = torch.autograd.grad((out, last), s0, (gg, dlast))
        want, mag = reference(q, k, vv, gg, ld, None, 1.0, s0, dlast)
        check(dict(last=last, dstate=dstate), want, mag)


@pytest.mark.parametrize("size", [1e10, 1e30])
def test_large_columns_leave_small_ones_their_bits_in_fp16(dev, size):
    (q, k, v, dout), (s0, dlast) = inputs(70, 1, 6, 64, F16, dev, 22)
    for x in (s0, dlast):
        x[..., 3] *= size
    ld = decays(6, dev)
    s0.requires_grad_()
    out, last = linear_attn_func(q, k, v, ld, scale=1.0, state=s0, return_state=True)
    dstate, = torch.autograd.grad((out, last), s0, (dout, dlast))
    want, mag = reference(q, k, v, dout, ld, None, 1.0, s0, dlast)
    check(dict(last=last, dstate=dstate), want, mag)
