"""States of linear attention at the ends of their range, against the definition in 64 bits, with the bounds of test_zzr_linear_attention_gpu.py."""
import pytest
import torch

from nmtgminor_amd.modules.linear_attention import linear_attn_func
from test_zzr_linear_attention_gpu import check, decays, inputs, reference

pytestmark = pytest.mark.gpu
F16 = torch.float16


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
