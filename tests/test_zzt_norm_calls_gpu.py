"""Calls of the norms with rotation, of linear attention's step and of the modules around them that their documentation allows or refuses."""
import pytest
import torch

from nmtgminor_amd.modules.linear_attention import LinearSelfMultiheadAttn, linear_attn_step
from nmtgminor_amd.modules.qk_norm import qk_norm_rotary_func
from nmtgminor_amd.modules.window_attention import WindowSelfMultiheadAttn
from test_zzq_qk_norm_gpu import U, reference, rows_of

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def tables(rows, d, dev, dtype=torch.float32):
    angles = torch.arange(rows, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
    angles = torch.cat((angles, angles), 1)
    return angles.cos().to(dtype).to(dev), angles.sin().to(dtype).to(dev)


def rows(t, b, h, d, dtype, dev, seed=0):
    gen = torch.Generator().manual_seed(seed)
    return [torch.randn(t, b, h, d, generator=gen).to(dtype).to(dev) for _ in range(3)]


@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("grad", [False, True])
def test_tangents_of_the_tables_are_refused(dev, which, grad):
    q, k, _ = rows(3, 1, 2, 64, F16, dev)
    q.requires_grad_(grad)
    pos = list(tables(4, 64, dev))
    with torch.autograd.forward_ad.dual_level():
        pos[which] = torch.autograd.forward_ad.make_dual(pos[which], torch.ones_like(pos[which]))
        with pytest.raises(RuntimeError, match="jvp"):
            qk_norm_rotary_func(q, k, None, None, *pos)


def test_tables_that_learn_elsewhere(dev):
    """Where nothing is recorded they are tables like others."""
    q, k, _ = rows(3, 1, 2, 64, F16, dev)
    pos = tables(4, 64, dev)
    want = qk_norm_rotary_func(q, k, None, None, *pos)
    learned = [x.clone().requires_grad_() for x in pos]
    with torch.no_grad():
        assert all(torch.equal(x, y) for x, y in zip(qk_norm_rotary_func(q, k, None, None, *learned), want))
    with pytest.raises(RuntimeError, match="no gradient"):
        qk_norm_rotary_func(q, k, None, None, *learned)


def test_step_under_autocast(dev):
    q, k, v = rows(2, 3, 2, 64, torch.float32, dev)
    decay, states = torch.tensor([-0.1, -0.01], device=dev), [torch.ones(3, 2, 64, 64, device=dev) for _ in range(2)]
    want = linear_attn_step(q.bfloat16(), k.bfloat16(), v.bfloat16(), decay, states[0])
    with torch.autocast("cuda", dtype=BF16):
        got = linear_attn_step(q, k, v, decay, states[1])
    assert got.dtype == BF16 and torch.equal(got, want) and torch.equal(*states) and states[1].dtype == torch.float32


def test_weights_and_tables_of_another_type_under_autocast(dev):
    """Weights and tables in 32 bits stay what they are, others take autocast's type as the rows do."""
    q, k, g = rows(5, 2, 2, 64, F16, dev)
    w = [torch.linspace(0.5, 1.5, 64, device=dev).half().requires_grad_() for _ in range(2)]
    pos = tables(8, 64, dev, F16)
    same = [x.detach().bfloat16().requires_grad_() for x in w]
    want = qk_norm_rotary_func(q.bfloat16(), k.bfloat16(), *same, *(x.bfloat16() for x in pos))
    with torch.autocast("cuda", dtype=BF16):
        got = qk_norm_rotary_func(q, k, *w, *pos)
    assert all(x.dtype == BF16 and torch.equal(x, y) for x, y in zip(got, want))
    one, two = (torch.autograd.grad(x, y, (g.bfloat16(), g.bfloat16())) for x, y in ((got, w), (want, same)))
    assert all(x.dtype == F16 and torch.equal(x, y.half()) for x, y in zip(one, two))
    x = torch.randn(6, 2, 128, device=dev).half()
    for m in (LinearSelfMultiheadAttn(128, 2), WindowSelfMultiheadAttn(128, 2, window=4, qk_norm=True)):
        m = m.to(dev).half()
        with torch.autocast("cuda", dtype=BF16):
            out = m(x, pos_emb=pos)
        assert out.dtype == BF16 and torch.isfinite(out).all()


def test_rows_far_apart_are_read_where_they_are(dev):
    t, b, h, d, far = 2, 64, 64, 64, 1 << 24
    q, k, g = rows(t, b, h, d, BF16, dev, 3)
    room = torch.empty(t * far, dtype=BF16, device=dev)
    apart = [room.as_strided(x.shape, (far, h * d, d, 1), b * h * d * i).copy_(x) for i, x in enumerate((q, k, g))]
    pos = tables(t, d, dev)
    want = qk_norm_rotary_func(q, k, None, None, *pos)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    got = qk_norm_rotary_func(*apart[:2], None, None, *pos)
    assert torch.cuda.max_memory_allocated() - before < 3 * q.numel() * 2          # the two results, no copies of the rows
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    near, leaves = q.requires_grad_(), apart[0].detach().requires_grad_()
    one, two = (torch.autograd.grad(qk_norm_rotary_func(x, k, None, None, *pos)[0], x, y)[0] for x, y in ((near, g), (leaves, apart[2])))
    assert torch.equal(one, two)


@pytest.mark.parametrize("norm", [True, False])
def test_modules_without_positions(dev, norm):
    pos = tables(8, 64, dev) if norm else None
    for m in (LinearSelfMultiheadAttn(128, 2, qk_norm=norm), WindowSelfMultiheadAttn(128, 2, window=4, qk_norm=norm)):
        m = m.to(dev).bfloat16()
        for t, b in ((0, 2), (3, 0)):
            x = torch.randn(t, b, 128, device=dev).bfloat16().requires_grad_()
            out = m(x, pos_emb=pos)
            assert out.shape == x.shape and torch.autograd.grad(out.sum(), x)[0].shape == x.shape


SIZES = {BF16: (3e38, 1e30, 1e19, 1.0, 1e-20, 0.0), F16: (6e4, 1.0, 6e-5, 1e-7, 0.0)}


def magnitudes(dtype, dev):
    base = torch.randn(len(SIZES[dtype]), 1, 2, 64, generator=torch.Generator().manual_seed(2)).clamp(-1, 1)
    return (base * torch.tensor(SIZES[dtype]).view(-1, 1, 1, 1)).to(dtype).to(dev)


def check_by_type(name, got, want, mag):
    """As test_zzq_qk_norm_gpu.check, with an absolute part that goes by the type: fp16 rounds its smallest values to 2^-25, bf16's
    smallest normal number is 2^-126."""
    u, slack = U[got.dtype], {F16: 2.0 ** -25, BF16: 2.0 ** -126}[got.dtype]
    got = got.detach().cpu().double()
    worst = ((got - want).abs() / (u * want.abs() + 1e-5 * mag + slack)).max().item()
    assert torch.isfinite(got).all() and worst <= 1.0, f"{name}: {worst:.3f} of the bound"


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_magnitudes(dev, dtype):
    """Rows of the largest and smallest numbers, every result to its own size."""
    x, pos = magnitudes(dtype, dev).requires_grad_(), tables(8, 64, dev)
    g = torch.ones_like(x)
    out = qk_norm_rotary_func(x, x.detach(), None, None, *pos)[0]
    dx, = torch.autograd.grad(out, x, g)
    want, mag = reference(x, None, g, *pos, rows_of(len(x), 1, None), 1e-6)
    check_by_type("out", out, want[0], mag[0])
    check_by_type("dx", dx, want[1], mag[1])
