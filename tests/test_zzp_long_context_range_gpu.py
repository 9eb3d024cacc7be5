"""Window attention and the quantised cache over the range of what they are given: magnitudes far from one, and D = dO . O of the
output before its rounding, told apart from D of the rounded one.

Magnitudes: the bounds of test_zzn_window_attention_gpu, which scale with the terms they are sums of.

D. Keys that are all alike make every visible probability 1 / n, and sum_j dS_ij = sum_j P_ij (dP_ij - D_i) = 0: the true dQ is
zero, and what the kernels leave is scale * key * (minus D's error + the sum of dS's roundings). Values of one large vector m plus small ones:
the error of D of the rounded output is e_i = sum_d dO_id (round(O_id) - O_id), known exactly, about m u / 2 per element; dS's are
those of the small part only, times 1 / sqrt(n). With |m| = 10 and a small part of 0.5 they are 4% of e (dQ) and 5% (dK, plus its own rounding,
u of a value as small as they). The rest of the output is held in 8 bits, to a sixteenth of itself at worst: 3.6% in the mean square of
a uniform error (2^-4 / sqrt(3)). Together below 10%; a quarter of what D of the rounded output would leave, in the 2-norm, is asked for.
"""
import pytest
import torch

import test_zzn_window_attention_gpu as wa
import test_zzo_quantized_cache_gpu as qc
from nmtgminor_amd import _lib as L
from nmtgminor_amd.modules.window_attention import window_attn_func

pytestmark = pytest.mark.gpu
BOTH = pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])

MAGNITUDES = [
    # t, b, h, hk, d, window, sinks, ragged
    (150, 1, 2, 1, 64, 40, 3, False),
    (200, 2, 2, 2, 128, 33, 70, True),
]


def scaled_inputs(t, b, h, hk, d, ragged, factor, dtype, dev):
    """-> q, k, v * factor, dout, lengths; not a number behind the lengths"""
    q, k, v, dout = wa.inputs(t, b, h, hk, d, torch.float32, "cpu", 11)
    q, k, v, dout = (x.to(dtype).to(dev) for x in (q, k, v * factor, dout))
    lengths = torch.tensor([(t, t // 2)[i % 2] for i in range(b)], dtype=torch.int32, device=dev) if ragged else None
    if ragged:
        for x in (q, k, v, dout):
            for s in range(b):
                x[int(lengths[s]):, s] = float("nan")
    return q, k, v, dout, lengths


def alike(t, b, h, hk, d, factor, dtype, seed=21):
    """Keys all alike, values of one large vector and small ones. -> q, k, v, dout on the CPU"""
    gen = torch.Generator().manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=gen)                                        # noqa: E731
    key = (4 * torch.sign(rand(d))).expand(t, b, hk, d)
    v = (10 * (1 + 0.3 * rand(b, hk, d)).clamp(0.5, 1.5) * torch.sign(rand(b, hk, d)) + 0.5 * rand(t, b, hk, d)) * factor
    return [x.to(dtype).contiguous() for x in (rand(t, b, h, d), key, v, rand(t, b, h, d))]


def errors_of_rounded_d(q, k, v, dout, lengths, window, sinks, scale):
    """What D of the rounded output adds to dQ and dK, in 64 bits"""
    dtype = q.dtype
    (out, *_), _ = wa.reference(q, k, v, dout, lengths, window, sinks, scale)
    t, b, h, _ = q.shape
    group = h // k.shape[2]
    e = (dout.double() * (out.to(dtype).double() - out)).sum(-1)                            # [t, b, h]
    dq, dk = torch.zeros_like(out), torch.zeros(k.shape, dtype=torch.float64)
    for s in range(b):
        sees = wa.visible(t if lengths is None else int(lengths[s]), t, window, sinks).double()
        p = sees / sees.sum(1, keepdim=True).clamp_min(1.0)
        for x in range(h):
            ds = -p * e[:, s, x][:, None]
            dq[:, s, x] = ds @ k[:, s, x // group].double() * scale
            dk[:, s, x // group] += ds.t() @ q[:, s, x].double() * scale
    return dq, dk


def check_d(grads, q, k, v, dout, lengths, window, sinks, scale):
    want, _ = wa.reference(q, k, v, dout, lengths, window, sinks, scale)
    for name, got, true, lost in zip(("dq", "dk"), grads, want[1:3], errors_of_rounded_d(q, k, v, dout, lengths, window, sinks, scale)):
        left = (got.detach().cpu().double() - true).norm() / lost.norm()
        assert left <= 0.25, f"{name}: {left:.3f} of the error that the rounded output's D leaves"


@BOTH
@pytest.mark.parametrize("factor", [1e-3, 8.0, 64.0, 1000.0])
@pytest.mark.parametrize("t,b,h,hk,d,window,sinks,ragged", MAGNITUDES)
def test_values_of_other_magnitudes(dev, t, b, h, hk, d, window, sinks, ragged, factor, dtype):
    q, k, v, dout, lengths = scaled_inputs(t, b, h, hk, d, ragged, factor, dtype, dev)
    clean = [torch.nan_to_num(x) for x in (q, k, v, dout)]
    want, mag = wa.reference(*clean, lengths, window, sinks, d ** -0.5)
    for x in (q, k, v):
        x.requires_grad_()
    out = window_attn_func(q, k, v, window, sinks, lengths=lengths)
    wa.check((out, *torch.autograd.grad(out, (q, k, v), dout)), want, mag, dtype)
    # the same as slots of one projection
    lin = torch.cat((q, k, v), 2).detach().flatten(2).requires_grad_()
    out = L.host().window_attention_projection(lin, h, hk, window, sinks, None, lengths)
    dlin, = torch.autograd.grad(out, lin, dout)
    wa.check((out, *dlin.view(t, b, -1, d).split((h, hk, hk), 2)), want, mag, dtype)


@BOTH
@pytest.mark.parametrize("factor", [1e-3, 1.0, 64.0, 1000.0])
@pytest.mark.parametrize("t,b,h,hk,d,window,sinks,ragged", [(200, 1, 2, 1, 64, 48, 0, False), (300, 2, 2, 2, 128, 90, 3, True)])
def test_d_is_that_of_the_output_before_its_rounding(dev, t, b, h, hk, d, window, sinks, ragged, factor, dtype):
    data = alike(t, b, h, hk, d, factor, dtype)
    lengths = torch.tensor([t, t - 61][:b], dtype=torch.int32) if ragged else None
    leaves = [x.to(dev).requires_grad_() for x in data[:3]]
    out = window_attn_func(*leaves, window, sinks, lengths=None if lengths is None else lengths.to(dev))
    grads = torch.autograd.grad(out, leaves[:2], data[3].to(dev))
    check_d(grads, *data, lengths, window, sinks, d ** -0.5)


@BOTH
def test_rows_of_no_magnitude_and_of_none_that_is_finite(dev, dtype):
    """An output of zeros has gradients like any other; one that is not finite spoils its own query's gradients, and no other head's."""
    q, k, v, dout = wa.inputs(100, 1, 2, 2, 64, dtype, dev, 6)
    for x in (q, k, v):
        x.requires_grad_()
    zero = torch.zeros_like(v).requires_grad_()
    out = window_attn_func(q, k, zero, 30, 2)
    assert not out.any()
    grads = torch.autograd.grad(out, (q, k, zero), dout)
    assert not grads[0].any() and not grads[1].any() and torch.isfinite(grads[2]).all()
    poisoned = v.detach().clone()
    poisoned[50, 0, 1, 3] = float("inf")
    bad = torch.autograd.grad(window_attn_func(q, k, poisoned.requires_grad_(), 30, 2), (q, k, poisoned), dout)
    good = torch.autograd.grad(window_attn_func(q, k, v, 30, 2), (q, k, v), dout)
    assert all(torch.equal(x[:, :, 0], y[:, :, 0]) for x, y in zip(bad, good))
    assert not torch.isfinite(bad[0][50, 0, 1]).all()


# ------------------------------------------------------------------------------------------------------ quantised cache
def check_attend(got, want, mag, dtype, lengths, largest):
    """Probabilities rounded once (u each, their sum that of the rounded ones) times values exact in the type, rounded once: 2 u of the terms'
    magnitudes and u of the result, 1e-5 of the magnitudes for sums and exponentials in 32 bits (u: 2^-8 for bf16, 2^-11 for fp16). Probabilities
    below fp16's normal range, relative to a largest of at least 1, are off by up to 2^-25 each, times at most the largest value."""
    got = got.cpu().double()
    assert got.shape == want.shape and torch.isfinite(got).all()
    small = 2.0 ** -25 * largest * torch.tensor(lengths, dtype=torch.float64)[None, :, None, None] if dtype == torch.float16 else 0.0
    worst = ((got - want).abs() / ((2 * wa.U[dtype] + 1e-5) * mag + wa.U[dtype] * want.abs() + 1e-6 + small)).max().item()
    assert worst <= 1.0, f"{worst:.3f} of the bound"


def top_of_the_type(cap, b, hk, d, bits, dtype):
    """Keys and values up to the type's largest. A block whose largest magnitude rounds up is held as a power of two beyond it, which the
    attention takes as the type's largest. -> k, v, their values as the attention sees them, q, softmax scale"""
    gen = torch.Generator().manual_seed(31)
    top = torch.finfo(dtype).max
    k, v = ((2 * torch.rand(cap, b, hk, d, generator=gen, dtype=torch.float64) - 1) * top for _ in range(2))
    k[..., 5], v[..., 7] = top, -top
    k[1::3, ..., :32] *= 2.0 ** -9                                # blocks of ordinary magnitude among them
    k, v = k.to(dtype), v.to(dtype)
    seen = [qc.held(x, bits)[0].clamp(-top, top) for x in (k, v)]
    assert (qc.held(k, bits)[0].abs() > top).any() and (qc.held(v, bits)[0].abs() > top).any()
    # scores of some units: sums of head_dim products of q and numbers up to the largest
    q = (torch.randn(1, b, 2 * hk, d, generator=gen) * (2.0 ** -4 if dtype == torch.float16 else 2.0 ** -120)).to(dtype)
    return k, v, seen, q, 2.0 ** -12 if dtype == torch.float16 else 2.0 ** -8


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype,d,lengths", [(torch.float16, 64, [70, 33]), (torch.float16, 128, [70, 2]), (torch.float16, 64, [2500, 40]),
                                             (torch.bfloat16, 128, [1, 1])])          # (bf16: sums of two such values leave 32 bits)
def test_finite_values_are_attended_to_as_finite(dev, dtype, d, lengths, bits):
    cap = max(lengths)
    k, v, seen, q, scale = top_of_the_type(cap, 2, 2, d, bits, dtype)
    cache = qc.buffers(2, 2, cap, d, bits, dev)
    qc.kv_cache_write(*cache, k.to(dev), v.to(dev), 0)
    want, mag = qc.attend_reference(q, *seen, lengths, 0, 0, scale)
    got = qc.kv_cache_attend(q.to(dev), *cache, torch.tensor(lengths, dtype=torch.int32, device=dev), cap, 0, 0, scale)
    check_attend(got, want, mag, dtype, lengths, torch.finfo(dtype).max)


def test_int64_positions_beyond_32_bits(dev):
    """Starts that lie outside the cache are outside it however far, and a length is clamped, not wrapped."""
    far = [1 << 32, -(1 << 32), (1 << 32) + 3, -(1 << 31) - 1, 2]
    b, hk, d, cap = len(far), 1, 64, 8
    k, v = (torch.randn(2, b, hk, d, device=dev).to(torch.bfloat16) for _ in range(2))
    cache = qc.buffers(b, hk, cap, d, 8, dev, fill=7)
    starts = torch.tensor(far, dtype=torch.int64, device=dev)
    qc.kv_cache_write(*cache, k, v, starts)
    for x in cache:
        assert (x[:4] == 7).all() and (x[4, :, :2] == 7).all() and (x[4, :, 4:] == 7).all()
    got = qc.kv_cache_read(*cache, starts, 2, torch.bfloat16)
    assert not got[0][:, :4].any() and not got[1][:, :4].any() and got[0][:, 4].any()
    qc.kv_cache_write(*cache, *(torch.randn(cap, b, hk, d, device=dev).to(torch.bfloat16) for _ in range(2)), 0)
    q = torch.randn(1, b, 2, d, device=dev).to(torch.bfloat16)
    lengths = torch.tensor([1 << 32, -(1 << 32), (1 << 32) + 3, -(1 << 31) - 1, 5], dtype=torch.int64, device=dev)
    want = qc.kv_cache_attend(q, *cache, torch.tensor([cap, 0, cap, 0, 5], dtype=torch.int32, device=dev), cap)
    assert torch.equal(qc.kv_cache_attend(q, *cache, lengths, cap), want)
    x, y, z, _ = wa.inputs(20, b, 2, 1, 64, torch.bfloat16, dev)
    want = window_attn_func(x, y, z, 5, 1, lengths=torch.tensor([20, 0, 20, 0, 5], dtype=torch.int32, device=dev))
    assert torch.equal(window_attn_func(x, y, z, 5, 1, lengths=lengths), want)


# ----------------------------------------------------------------------------------------------------- what is refused
def test_tracing_is_refused(dev):
    """torch.jit.trace does not see the native layer's results and would keep those of the recording."""
    cache = qc.QuantizedKVCache(1, 2, 64, 8, dtype=torch.float16, device=dev)
    q, k, v, _ = wa.inputs(3, 1, 2, 2, 64, torch.float16, dev)
    m = wa.WindowSelfMultiheadAttn(128, 2, window=4).to(dev).half().requires_grad_(False)
    x = torch.randn(3, 1, 128, device=dev).half()
    with torch.no_grad():
        for call, arg in ((lambda y: window_attn_func(y, k, v, 4), q), (m, x), (lambda y: m(y, cache=cache), x),
                          (lambda y: cache.append(y, v) or y, k), (lambda y: cache.read()[0] + y, q), (lambda y: cache.attend(y), q)):
            with pytest.raises(RuntimeError, match="cannot be traced"):
                torch.jit.trace(call, (arg,), check_trace=False)
        assert cache.longest == 0 and not cache.k_codes.any()
        m(x)


def test_tangents_are_refused(dev):
    """A forward-mode dual's tangent would be dropped without a word."""
    from torch.autograd import forward_ad
    cache = qc.QuantizedKVCache(1, 2, 64, 8, dtype=torch.float16, device=dev)
    q, k, v, t = wa.inputs(3, 1, 2, 2, 64, torch.float16, dev)
    lin = torch.cat((q, k, v), 2).flatten(2)
    with torch.no_grad(), forward_ad.dual_level():
        dual = forward_ad.make_dual(q, t)
        for call in (lambda: qc.kv_cache_write(*cache.tensors, dual, v, 0), lambda: qc.kv_cache_write(*cache.tensors, k, dual, 0),
                     lambda: cache.append(k, dual), lambda: cache.attend(dual), lambda: window_attn_func(q, dual, v, 2),
                     lambda: L.host().window_attention_projection(forward_ad.make_dual(lin, lin), 2, 2, 2, 0, None, None)):
            with pytest.raises(RuntimeError, match="(?i)jvp"):
                call()
        assert cache.longest == 0 and not cache.k_codes.any()
        cache.append(k, v)
        cache.attend(q)


# ---------------------------------------------------------------------------------------------------------- the module
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_module_in_32_bits_decodes_under_autocast(dev, dtype):
    torch.manual_seed(4)
    m = wa.WindowSelfMultiheadAttn(256, 4, window=12, sinks=2, num_kv_heads=2, cache_bits=8).to(dev).eval()
    half = wa.WindowSelfMultiheadAttn(256, 4, window=12, sinks=2, num_kv_heads=2, cache_bits=8).to(dev).eval()
    half.load_state_dict(m.state_dict())
    half.to(dtype)
    x = torch.randn(30, 2, 256, device=dev)
    with torch.no_grad():
        with torch.autocast("cuda", dtype=dtype):
            cache = m.make_cache(2, 32)
            got = [m(x[:25], cache=cache)] + [m(x[i:i + 1], cache=cache) for i in range(25, 30)]
        other = half.make_cache(2, 32)
        want = [half(x[:25].to(dtype), cache=other)] + [half(x[i:i + 1].to(dtype), cache=other) for i in range(25, 30)]
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert cache.dtype == dtype and all(torch.equal(a, b) for a, b in zip(cache.read(), other.read()))


def test_module_prompt_lengths_beyond_the_prompt(dev):
    """Attention and cache agree on what a sequence holds."""
    torch.manual_seed(5)
    m = wa.WindowSelfMultiheadAttn(128, 2, window=6, sinks=1, cache_bits=8).to(dev).to(torch.bfloat16).eval()
    x = torch.randn(12, 3, 128, device=dev).to(torch.bfloat16)
    with torch.no_grad():
        res = []
        for lengths in ([10, 0, 10], [1 << 33, -5, 400]):
            cache = m.make_cache(3, 16)
            first = m(x[:10], torch.tensor(lengths, device=dev), cache=cache)
            res.append((first, cache.lengths.clone(), m(x[10:11], cache=cache), m(x[11:], cache=cache)))
    assert all(torch.equal(a, b) for a, b in zip(*res)) and res[0][1].tolist() == [10, 0, 10]


def test_one_position_of_many_heads(dev):
    """A single position has no stride to the next one: what that stride would be limits nothing."""
    b, h, hk, d = 4096, 64, 64, 64
    q, k, v, dout = (torch.randn(1, b, h, d, device=dev, dtype=torch.bfloat16) for _ in range(4))
    assert q.stride(0) >= 1 << 24
    for x in (q, k, v):
        x.requires_grad_()
    out = window_attn_func(q, k, v, 3, 1)
    dq, dk, dv = torch.autograd.grad(out, (q, k, v), dout)
    assert torch.equal(out, v) and torch.equal(dv, dout)
    # dS = dP - D is zero but for the order of the sums in 32 bits
    terms = 2e-5 * (dout.double() * v.detach().double()).abs().sum(-1, keepdim=True) * d ** -0.5
    assert (dq.double().abs() <= terms * k.detach().double().abs() + 1e-6).all() and (dk.double().abs() <= terms * q.detach().double().abs() + 1e-6).all()
    lin = torch.cat((q, k, v), 2).detach().flatten(2)
    assert torch.equal(L.host().window_attention_projection(lin, h, hk, 3, 1, None, None), v)
    with pytest.raises(RuntimeError, match="position stride below"):
        window_attn_func(*(x.detach().expand(2, b, h, d).contiguous() for x in (q, k, v)), 3, 1)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("d,lengths", [(64, [70, 33]), (128, [95, 64])])
def test_scales_at_any_address(dev, d, lengths, bits):
    """Scale bytes are a dense tensor of bytes, which may begin anywhere."""
    b, hk, cap = 2, 2, max(lengths)
    k, v = (torch.randn(cap, b, hk, d, device=dev).to(torch.bfloat16) for _ in range(2))
    q = torch.randn(1, b, 4, d, device=dev).to(torch.bfloat16)
    n = torch.tensor(lengths, dtype=torch.int32, device=dev)
    dense = qc.buffers(b, hk, cap, d, bits, dev)
    qc.kv_cache_write(*dense, k, v, 0)
    want = qc.kv_cache_attend(q, *dense, n, cap)
    for offset in (1, 3):
        moved = [torch.zeros(x.numel() + 16, dtype=torch.uint8, device=dev)[offset if i % 2 else 0:][:x.numel()].view(x.shape) for i, x in enumerate(dense)]
        qc.kv_cache_write(*moved, k, v, 0)
        assert all(torch.equal(x, y) for x, y in zip(moved, dense)) and torch.equal(qc.kv_cache_attend(q, *moved, n, cap), want)
        assert all(torch.equal(x, y) for x, y in zip(qc.kv_cache_read(*moved, 0, cap), qc.kv_cache_read(*dense, 0, cap)))


def test_module_parameter_gradients(dev):
    """Against the same module in 64 bits on the parameters as they are, in the 2-norm: every tensor on the way (projection, context, their gradients,
    probabilities and score gradients) is rounded to bf16 once, u = 2^-8 of an element at worst and 0.41 u in the mean square; some six such
    roundings lie behind each parameter gradient: 6 * 0.41 u if they all added up. Twice that is asked for."""
    torch.manual_seed(7)
    t, b, e, h, hk, window, sinks = 60, 2, 256, 4, 2, 15, 2
    m = wa.WindowSelfMultiheadAttn(e, h, window=window, sinks=sinks, num_kv_heads=hk).to(dev).to(torch.bfloat16)
    with torch.no_grad():
        for p in (m.in_proj_bias, m.out_proj_bias):
            p.normal_()
    x, dy = (torch.randn(t, b, e, device=dev).to(torch.bfloat16) for _ in range(2))
    lengths = torch.tensor([60, 37], device=dev)
    m(x, lengths).backward(dy)
    params = [p.detach().cpu().double().requires_grad_() for p in (m.in_proj_weight, m.in_proj_bias, m.out_proj_weight, m.out_proj_bias)]
    d = e // h
    q, k, v = torch.nn.functional.linear(x.cpu().double(), *params[:2]).view(t, b, -1, d).split((h, hk, hk), 2)
    out = []
    for s in range(b):
        sees = wa.visible(int(lengths[s]), t, window, sinks)
        rows = sees.any(1)
        for i in range(h):
            score = (q[:, s, i] @ k[:, s, i * hk // h].t() * d ** -0.5)[rows].masked_fill(~sees[rows], -torch.inf)
            out.append(torch.zeros(t, d, dtype=torch.float64).index_put((rows.nonzero()[:, 0],), torch.softmax(score, 1) @ v[:, s, i * hk // h]))
    context = torch.stack(out).view(b, h, t, d).permute(2, 0, 1, 3).reshape(t, b, e)
    torch.nn.functional.linear(context, *params[2:]).backward(dy.cpu().double())
    for got, want in zip((m.in_proj_weight, m.in_proj_bias, m.out_proj_weight, m.out_proj_bias), params):
        off = (got.grad.cpu().double() - want.grad).norm() / want.grad.norm()
        assert off <= 12 * 0.41 * 2.0 ** -8, off
