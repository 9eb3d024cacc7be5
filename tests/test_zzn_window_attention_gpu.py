"""Attention with a sliding window and sinks (nmtg_window_attn_fwd / _bwd, modules/window_attention.py) against the definition in 64 bits.

Tolerances, from the roundings on the way (u: unit roundoff of the 16-bit type, 2^-8 for the 8 significant bits
of bf16, 2^-11 for the 11 of fp16): the output is a sum
of probabilities (rounded once, u each) times values, rounded once: at most 2 u sum_j p_j |v_j| per element, and 1e-5 of the
same for fp32 sums and exponentials. Gradients are sums over products of two factors of which one is rounded once, of score
gradients that contain the output rounded once (D = dO . O), rounded once themselves: 4 u times the sum of the terms' magnitudes,
which the reference computes along.
"""
import pytest
import torch

from nmtgminor_amd.modules.window_attention import WindowSelfMultiheadAttn, window_attn_func

pytestmark = pytest.mark.gpu
U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def visible(n, t, window, sinks):
    i, j = torch.arange(t)[:, None], torch.arange(t)[None, :]
    return (j <= i) & ((j > i - window) | (j < sinks)) & (i < n) & (j < n)


def reference(q, k, v, dout, lengths, window, sinks, scale):
    """-> (out, dq, dk, dv) and the sums of the magnitudes of their terms, in 64 bits on the CPU"""
    q, k, v, dout = (x.detach().cpu().double() for x in (q, k, v, dout))
    t, b, h, _ = q.shape
    g = h // k.shape[2]
    res = [torch.zeros_like(x) for x in (q, q, k, v)]
    mag = [torch.zeros_like(x) for x in (q, q, k, v)]
    for s in range(b):
        sees = visible(t if lengths is None else int(lengths[s]), t, window, sinks)
        for x in range(h):
            qq, kk, vv, do = q[:, s, x], k[:, s, x // g], v[:, s, x // g], dout[:, s, x]
            sc = (qq @ kk.t() * scale).masked_fill(~sees, -torch.inf)
            top = sc.amax(1, keepdim=True)
            p = torch.exp(sc - torch.where(top == -torch.inf, torch.zeros_like(top), top))
            p = p / p.sum(1, keepdim=True).clamp_min(1e-300)
            o = p @ vv
            do = do * sees.any(1, keepdim=True)
            dp = do @ vv.t()
            delta = (do * o).sum(1, keepdim=True)
            ds = p * (dp - delta)
            dsm = p * (do.abs() @ vv.abs().t() + (do.abs() * o.abs()).sum(1, keepdim=True))
            for i, (val, m, at) in enumerate(((o, p @ vv.abs(), x), (ds @ kk * scale, dsm @ kk.abs() * abs(scale), x),
                                              (ds.t() @ qq * scale, dsm.t() @ qq.abs() * abs(scale), x // g), (p.t() @ do, p.t() @ do.abs(), x // g))):
                res[i][:, s, at] += val
                mag[i][:, s, at] += m
    return res, mag


def check(got, want, mag, dtype, factors=(2, 4, 4, 2)):
    for name, a, e, m, f in zip(("out", "dq", "dk", "dv"), got, want, mag, factors):
        a = a.detach().cpu().double()
        assert a.shape == e.shape and torch.isfinite(a).all(), name
        # the last rounding is of the value itself; the smallest values of fp16 round absolutely
        bound = (f * U[dtype] + 1e-5) * m + U[dtype] * e.abs() + 1e-6
        worst = ((a - e).abs() / bound).max().item() if a.numel() else 0.0
        assert worst <= 1.0, f"{name}: {worst:.3f} of the bound"


def inputs(t, b, h, hk, d, dtype, dev, seed=0):
    gen = torch.Generator().manual_seed(seed)
    make = lambda heads: torch.randn(t, b, heads, d, generator=gen).to(dtype).to(dev)      # noqa: E731
    return make(h), make(hk), make(hk), make(h)


CASES = [
    # t, b, h, hk, d, window, sinks, ragged
    (1, 2, 2, 2, 64, 1, 0, False),
    (2, 1, 2, 1, 128, 1, 1, False),
    (63, 2, 2, 2, 64, 17, 3, False),
    (64, 1, 4, 1, 64, 64, 0, True),
    (65, 2, 2, 1, 128, 5, 64, False),
    (129, 3, 2, 2, 64, 1000, 0, True),
    (200, 2, 4, 2, 128, 33, 70, True),
    (257, 1, 2, 2, 64, 100, 4, False),
    (300, 3, 2, 1, 64, 7, 130, True),
    (520, 1, 2, 1, 128, 129, 1, False),
    (700, 2, 2, 2, 64, 64, 37, True),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("t,b,h,hk,d,window,sinks,ragged", CASES)
def test_forward_and_gradients(dev, t, b, h, hk, d, window, sinks, ragged, dtype):
    q, k, v, dout = inputs(t, b, h, hk, d, dtype, dev)
    lengths = torch.tensor([(t, t // 2, 0)[i % 3] for i in range(b)], dtype=torch.int32, device=dev) if ragged else None
    if ragged:                                      # what lies behind a sequence's end is nobody's business
        for x in (q, k, v, dout):
            for s in range(b):
                x[int(lengths[s]):, s] = float("nan")
    for x in (q, k, v):
        x.requires_grad_()
    out = window_attn_func(q, k, v, window, sinks, lengths=lengths)
    grads = torch.autograd.grad(out, (q, k, v), dout)
    clean = [torch.nan_to_num(x.detach()) for x in (q, k, v, dout)]
    want, mag = reference(*clean, lengths, window, sinks, d ** -0.5)
    check((out, *grads), want, mag, dtype)
    with torch.no_grad():
        assert torch.equal(window_attn_func(q, k, v, window, sinks, lengths=lengths), out)


@pytest.mark.parametrize("t,b,h,hk,d,window,sinks,ragged", [
    (1500, 1, 4, 1, 64, 40, 2, False),               # a head's sinks in eleven chunks
    (900, 2, 4, 1, 128, 30, 300, True),              # more sinks than a block's keys, in longer chunks
])
def test_sinks_in_many_chunks(dev, t, b, h, hk, d, window, sinks, ragged):
    test_forward_and_gradients(dev, t, b, h, hk, d, window, sinks, ragged, torch.bfloat16)


@pytest.mark.parametrize("scale", [0.0, -0.25, 1.0])
def test_other_scales(dev, scale):
    q, k, v, dout = inputs(90, 1, 2, 2, 64, torch.bfloat16, dev, 3)
    for x in (q, k, v):
        x.requires_grad_()
    out = window_attn_func(q, k, v, 20, 2, softmax_scale=scale)
    grads = torch.autograd.grad(out, (q, k, v), dout)
    want, mag = reference(q, k, v, dout, None, 20, 2, scale)
    # scores of up to some 40 (scale 1): the fp32 sum of 64 products is off by up to 64 * 2^-24 * 40 in the exponent
    mag = [m * 1.05 for m in mag]
    check((out, *grads), want, mag, torch.bfloat16)


def test_heads_of_one_projection_and_other_strides(dev):
    """Slots of one tensor, batch-first tensors, and layouts that the kernels cannot take (copied)."""
    t, b, h, hk, d = 150, 2, 4, 2, 64
    lin = torch.randn(t, b, h + 2 * hk, d, device=dev).to(torch.bfloat16)
    q, k, v = lin.split((h, hk, hk), 2)
    want = window_attn_func(q.contiguous(), k.contiguous(), v.contiguous(), 40, 4)
    assert torch.equal(window_attn_func(q, k, v, 40, 4), want)
    first = lambda x: x.transpose(0, 1).contiguous().transpose(0, 1)                    # noqa: E731
    assert torch.equal(window_attn_func(first(q), first(k), v, 40, 4), want)
    odd = torch.empty(t, b, h, d + 1, device=dev, dtype=torch.bfloat16)[..., 1:]
    odd.copy_(q)
    swapped = k.transpose(2, 3).contiguous().transpose(2, 3)
    assert torch.equal(window_attn_func(odd, swapped, v, 40, 4), want)
    # a gradient that is broadcast (no strides of its own)
    leaves = [x.detach().clone().requires_grad_() for x in (q, k, v)]
    out = window_attn_func(*leaves, 40, 4)
    one = torch.autograd.grad(out.sum(), leaves, retain_graph=True)
    two = torch.autograd.grad(out, leaves, torch.ones_like(out))
    assert all(torch.equal(x, y) for x, y in zip(one, two))


def test_a_window_over_everything_is_causal_attention(dev):
    q, k, v, _ = inputs(333, 2, 2, 2, 64, torch.float16, dev, 5)
    assert torch.equal(window_attn_func(q, k, v, 333, 0), window_attn_func(q, k, v, 1 << 35, 1 << 35))
    # with sinks everywhere the window does not matter (up to the order of the tiles, which is the same)
    assert torch.equal(window_attn_func(q, k, v, 1, 333), window_attn_func(q, k, v, 333, 0))


def test_gradients_against_differences(dev):
    """Directional derivative of a scalar by central differences of the 64-bit definition."""
    t, b, h, hk, d, window, sinks = 40, 1, 2, 1, 64, 9, 2
    q, k, v, dout = inputs(t, b, h, hk, d, torch.float16, dev, 9)
    for x in (q, k, v):
        x.requires_grad_()
    grads = torch.autograd.grad(window_attn_func(q, k, v, window, sinks), (q, k, v), dout)
    base = [x.detach().cpu().double() for x in (q, k, v)]
    do = dout.cpu().double()
    for at in range(3):
        step = torch.randn(base[at].shape, dtype=torch.float64, generator=torch.Generator().manual_seed(at))
        values = []
        for sign in (1, -1):
            moved = [x + sign * 1e-5 * step if i == at else x for i, x in enumerate(base)]
            values.append((reference(*moved, do, None, window, sinks, d ** -0.5)[0][0] * do).sum())
        slope = (values[0] - values[1]) / 2e-5
        mine = (grads[at].cpu().double() * step).sum()
        # the sum's error: independent errors of at most ~4 u of each term's magnitude, against its 2-norm
        _, mag = reference(*base, do, None, window, sinks, d ** -0.5)
        assert abs(mine - slope) <= 6 * U[torch.float16] * 4 * (mag[at + 1] * step.abs()).norm() + 1e-6


def test_infinities_at_masked_positions(dev):
    """Inf and NaN in keys and values of tiles that no query sees, or behind a length, reach nothing."""
    q, k, v, dout = inputs(640, 1, 2, 2, 64, torch.bfloat16, dev, 2)
    want = window_attn_func(q[300:], k[300:], v[300:], 30, 0)
    k2, v2 = k.clone(), v.clone()
    k2[:192], v2[:192] = float("nan"), float("inf")
    got = window_attn_func(q, k2, v2, 30, 0)
    assert torch.isfinite(got[256:]).all()
    # the same rows without the poison (their tiles differ, so do the orders of their sums)
    assert torch.allclose(got[340:].float(), want[40:].float(), rtol=2e-2, atol=2e-2)
    # the lowest value of the type as a mask of one's own
    low = torch.finfo(torch.bfloat16).min
    q2 = q.clone()
    q2[:] = 1.0
    k2 = torch.zeros_like(k)
    k2[100:] = low
    out = window_attn_func(q2, k2, v, 640, 0)
    assert torch.isfinite(out).all()
    assert torch.allclose(out[500].float(), v[:100].float().mean(0), atol=2e-2)


def test_runs_on_the_current_stream(dev):
    q, k, v, dout = inputs(300, 2, 2, 2, 64, torch.bfloat16, dev, 4)
    want = window_attn_func(q, k, v, 50, 4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = window_attn_func(q, k, v, 50, 4)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


def test_a_captured_call_replays(dev):
    q, k, v, dout = inputs(200, 2, 4, 2, 64, torch.bfloat16, dev, 4)
    leaves = [x.requires_grad_() for x in (q, k, v)]

    def step():
        out = window_attn_func(*leaves, 50, 4)
        return (out, *torch.autograd.grad(out, leaves, dout))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = step()
    for seed in range(3):
        for x, y in zip((*leaves, dout), inputs(200, 2, 4, 2, 64, torch.bfloat16, dev, seed)):
            x.data.copy_(y)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(res, step()))


def test_empty(dev):
    for shape in ((0, 2), (3, 0)):
        q, k = (torch.empty(*shape, n, 64, device=dev, dtype=torch.float16, requires_grad=True) for n in (4, 2))
        out = window_attn_func(q, k, k.detach(), 5)
        assert out.shape == q.shape
        out.sum().backward()
        assert q.grad.shape == q.shape and k.grad.shape == k.shape
    q, k, v, dout = inputs(70, 2, 2, 2, 64, torch.float16, dev)
    none = torch.zeros(2, dtype=torch.int64, device=dev)
    assert not window_attn_func(q, k, v, 5, 1, lengths=none).any()


def test_refusals(dev):
    q, k, v, _ = inputs(8, 2, 4, 2, 64, torch.float16, dev)
    for args, text in (((q.cpu(), k, v, 4), "device memory"), ((q.float(), k, v, 4), "fp16 or bf16"), ((q, k.to(torch.bfloat16), v, 4), "one dtype"),
                       ((q, k[:4], v[:4], 4), "positions"), ((q, k, v, 0), "window"), ((q, k, v, 4, -1), "sinks"),
                       ((q[:, :, :3], k, v, 4), "evenly"), ((q[..., :32], k[..., :32], v[..., :32], 4), "head dimension 32")):
        with pytest.raises(RuntimeError, match=text):
            window_attn_func(*args)
    for bad in (torch.ones(3, dtype=torch.int32, device=dev), torch.ones(2, device=dev), torch.ones(2, dtype=torch.int32)):
        with pytest.raises(RuntimeError):
            window_attn_func(q, k, v, 4, lengths=bad)


# ------------------------------------------------------------------------------------------------------------ the module
def test_module_trains(dev):
    torch.manual_seed(1)
    m = WindowSelfMultiheadAttn(256, 4, window=20, sinks=2, num_kv_heads=2).to(dev).to(torch.bfloat16)
    x = torch.randn(70, 3, 256, device=dev).to(torch.bfloat16).requires_grad_()
    dy = torch.randn(70, 3, 256, device=dev).to(torch.bfloat16)
    lengths = torch.tensor([70, 33, 1], device=dev)
    y = m(x, lengths)
    y.backward(dy)
    # the same with the operators one by one
    y2_in = x.detach().clone().requires_grad_()
    lin = torch.nn.functional.linear(y2_in.double(), m.in_proj_weight.double(), m.in_proj_bias.double())
    heads = lin.to(torch.bfloat16).view(70, 3, 8, 64)
    q, k, v = (t.contiguous() for t in heads.split((4, 2, 2), 2))
    ctx = window_attn_func(q, k, v, 20, 2, lengths=lengths)
    y2 = torch.nn.functional.linear(ctx.reshape(70, 3, 256).double(), m.out_proj_weight.double(), m.out_proj_bias.double())
    y2.backward(dy.double())
    for got, want in ((y, y2), (x.grad, y2_in.grad)):
        got, want = got.detach().double(), want.detach().double()
        assert (got - want).norm() <= 2e-2 * want.norm()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in m.parameters())


@pytest.mark.parametrize("bits,close", [(8, 0.05), (4, 0.25)])
def test_module_decodes_from_its_quantised_cache(dev, bits, close):
    """Prompt and steps against the whole sequence at once. What the cache's rounding costs: 8 bits hold an element to 2^-4 of
    itself at worst (2^-4 / sqrt(12) on average), 4 bits to a quarter."""
    torch.manual_seed(2)
    m = WindowSelfMultiheadAttn(256, 4, window=24, sinks=3, num_kv_heads=2, cache_bits=bits).to(dev).to(torch.bfloat16).eval()
    x = torch.randn(90, 2, 256, device=dev).to(torch.bfloat16)
    with torch.no_grad():
        whole = m(x)
        cache = m.make_cache(2, 96)
        parts = [m(x[:60], cache=cache)] + [m(x[i:i + n], cache=cache) for i, n in ((60, 1), (61, 1), (62, 3), (65, 1))]
        parts += [m(x[i:i + 1], cache=cache) for i in range(66, 90)]
    got = torch.cat(parts)
    assert cache.longest == 90 and cache.lengths.tolist() == [90, 90]
    assert torch.equal(got[:60], whole[:60])
    a, e = got[60:].double(), whole[60:].double()
    assert (a - e).norm() <= close * e.norm()


def test_module_prompts_of_several_lengths(dev):
    torch.manual_seed(3)
    m = WindowSelfMultiheadAttn(256, 4, window=10, sinks=1, cache_bits=8).to(dev).to(torch.bfloat16).eval()
    x = torch.randn(40, 2, 256, device=dev).to(torch.bfloat16)
    with torch.no_grad():
        cache = m.make_cache(2, 64)
        m(x[:30], torch.tensor([30, 17], device=dev), cache=cache)
        step = m(x[30:31], cache=cache)
        for s, n in enumerate((30, 17)):
            alone = m.make_cache(1, 64)
            m(x[:n, s:s + 1], cache=alone)
            assert torch.equal(m(x[30:31, s:s + 1], cache=alone), step[:, s:s + 1])
        assert cache.lengths.tolist() == [31, 18]
        with pytest.raises(RuntimeError, match="lengths go with the prompt"):
            m(x[:1], torch.tensor([1, 1], device=dev), cache=cache)
    with pytest.raises(RuntimeError, match="no gradient"):
        m(x[:1], cache=cache)
