"""The quantised key / value cache (nmtg_kv_cache_write / _read / _attn, modules/quantized_cache.py) against its definition in 64 bits.

What a cache holds is compared exactly: the scale is a power of two, so the definition has one answer. Attention: a sum of
probabilities (rounded once to the 16-bit type, u each) times held values (exact in that type), rounded once: 2 u sum_j p_j |v_j|
plus u of the value, and 1e-5 of the same for fp32 sums and exponentials (u: 2^-9 for bf16, 2^-12 for fp16).
"""
import pytest
import torch

from nmtgminor_amd.modules.quantized_cache import QuantizedKVCache, kv_cache_attend, kv_cache_read, kv_cache_write

pytestmark = pytest.mark.gpu
U = {torch.float16: 2.0 ** -12, torch.bfloat16: 2.0 ** -9}
FOUR = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
EIGHT = [(m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)) for e in range(16) for m in range(8)][:127]


def held(x, bits):
    """-> (values in 64 bits, scale bytes, codes of one element each) for x [..., D] on the CPU"""
    grid = torch.tensor(FOUR if bits == 4 else EIGHT, dtype=torch.float64)
    limit, lowest = (7.0 if bits == 4 else 464.0), -126
    b = x.double().unflatten(-1, (-1, 32))
    top = b.abs().amax(-1)
    bad = ~torch.isfinite(top)
    e = torch.full(top.shape, lowest, dtype=torch.int64)
    for s in range(lowest, 128):                    # the smallest that fits
        e = torch.where(top > limit * 2.0 ** s, s + 1, e)
    scale = torch.pow(2.0, e.double())[..., None]
    y = torch.nan_to_num(b / scale, posinf=0, neginf=0).abs()
    lo = (torch.searchsorted(grid, y.contiguous(), right=True) - 1).clamp(max=len(grid) - 2)
    up = (y - grid[lo] > grid[lo + 1] - y) | ((y - grid[lo] == grid[lo + 1] - y) & (lo % 2 == 1))
    code = lo + up
    values = grid[code] * torch.where(torch.signbit(b), -1.0, 1.0) * scale
    values = torch.where(bad[..., None], torch.full_like(values, float("nan")), values)
    code = torch.where(bad[..., None], 0, code + (8 if bits == 4 else 128) * torch.signbit(b))
    return values.flatten(-2), torch.where(bad, 255, e + 127).to(torch.uint8), code.flatten(-2)


def buffers(b, hk, cap, d, bits, dev, fill=0):
    return [torch.full((b, hk, cap, w), fill, dtype=torch.uint8, device=dev) for w in (d * bits // 8, d // 32) * 2]


def unpack(codes, bits):
    codes = codes.cpu().long()
    return codes if bits == 8 else torch.stack((codes & 15, codes >> 4), -1).flatten(-2)


ROWS = [
    # count, b, hk, d, cap
    (1, 1, 1, 64, 1), (1, 5, 3, 128, 7), (3, 2, 2, 64, 40), (37, 3, 1, 128, 50), (130, 2, 4, 64, 131),
]


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("count,b,hk,d,cap", ROWS)
def test_write_and_read(dev, count, b, hk, d, cap, dtype, bits):
    gen = torch.Generator().manual_seed(count)
    k, v = (torch.randn(count, b, hk, d, generator=gen) * torch.exp2(torch.randint(-8, 6, (count, b, hk, 1), generator=gen).float()) for _ in range(2))
    k[..., 3] *= 30
    k, v = k.to(dtype), v.to(dtype)
    v[0, 0, 0, :32] = 0
    cache = buffers(b, hk, cap, d, bits, dev, fill=7)
    start = (cap - count) // 2
    kv_cache_write(*cache, k.to(dev), v.to(dev), start)
    for x, codes, scales in ((k, cache[0], cache[1]), (v, cache[2], cache[3])):
        values, byte, code = held(x.permute(1, 2, 0, 3), bits)
        nonzero = x.permute(1, 2, 0, 3).unflatten(-1, (-1, 32)).abs().amax(-1) > 0
        got = scales[:, :, start:start + count].cpu()
        assert torch.equal(got[nonzero], byte[nonzero])
        assert torch.equal(unpack(codes[:, :, start:start + count], bits), code)
        # nothing else is touched
        for t in (codes, scales):
            assert (t[:, :, :start] == 7).all() and (t[:, :, start + count:] == 7).all()
    kk, vv = kv_cache_read(*cache, start, count, dtype)
    for x, got in ((k, kk), (v, vv)):
        want = held(x, bits)[0]
        assert got.dtype == dtype and torch.equal(got.cpu().double(), want)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_ties_edges_and_what_is_not_finite(dev, dtype, bits):
    """Every midpoint of the format, the upper ends of a scale's range, the smallest numbers, inf and NaN."""
    grid = torch.tensor(FOUR if bits == 4 else EIGHT, dtype=torch.float64)
    mids = (grid[1:] + grid[:-1]) / 2
    rows = []
    for anchor in (6.0, 7.0, 7.03125) if bits == 4 else (448.0, 464.0, 466.0):
        for part in mids.split(31):
            row = torch.zeros(32, dtype=torch.float64)
            row[0], row[1:1 + len(part)] = anchor, part
            row[2::3] *= -1
            rows.append(row)
    fine = torch.finfo(dtype)
    for extreme in (fine.max, fine.tiny, fine.smallest_normal / 8 if dtype == torch.float16 else fine.tiny):
        rows.append(torch.linspace(-1, 1, 32, dtype=torch.float64) * extreme)
    for bad in (float("inf"), float("-inf"), float("nan")):
        row = torch.ones(32, dtype=torch.float64)
        row[17] = bad
        rows.append(row)
    rows = torch.stack(rows + [torch.zeros(32, dtype=torch.float64)] * (-len(rows) % 2)).to(dtype).view(-1, 1, 1, 64)
    cache = buffers(1, 1, len(rows), 64, bits, dev)
    kv_cache_write(*cache, rows.to(dev), -rows.to(dev), 0)
    kk, vv = kv_cache_read(*cache, 0, len(rows), dtype)
    want = held(rows, bits)[0]
    # (a held value below the normal range of fp16 may need more bits than that type keeps: rounded there, to nearest)
    assert torch.equal(torch.nan_to_num(kk.cpu().double(), nan=-1e300), torch.nan_to_num(want.to(dtype).double(), nan=-1e300))
    assert torch.equal(torch.isnan(vv.cpu()), torch.isnan(want))


@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
def test_starts_of_their_own(dev, kind):
    """Rows that a tensor of starts puts outside the cache are dropped and read as zeros."""
    count, b, hk, d, cap = 4, 5, 2, 64, 10
    k, v = (torch.randn(count, b, hk, d, device=dev).to(torch.bfloat16) for _ in range(2))
    cache = buffers(b, hk, cap, d, 8, dev)
    starts = torch.tensor([0, 3, 8, -2, 1 << 30], dtype=kind, device=dev)
    kv_cache_write(*cache, k, v, starts)
    kk, vv = kv_cache_read(*cache, starts, count, torch.bfloat16)
    want = held(k.cpu(), 8)[0]
    for s, at in enumerate(starts.tolist()):
        for i in range(count):
            row = kk[i, s].cpu().double()
            assert torch.equal(row, want[i, s] if 0 <= at + i < cap else torch.zeros_like(row))
    assert (kv_cache_read(*cache, 0, cap, torch.bfloat16)[0][:, 4] == 0).all()


def test_strided_rows(dev):
    lin = torch.randn(6, 2, 8, 64, device=dev).to(torch.float16)
    q, k, v = lin.split((4, 2, 2), 2)
    one, two = buffers(2, 2, 6, 64, 4, dev), buffers(2, 2, 6, 64, 4, dev)
    kv_cache_write(*one, k, v, 0)
    kv_cache_write(*two, k.contiguous(), v.transpose(2, 3).contiguous().transpose(2, 3), 0)
    assert all(torch.equal(x, y) for x, y in zip(one, two))


# ------------------------------------------------------------------------------------------------------------- attention
def fill(b, hk, cap, d, bits, dtype, dev, seed):
    gen = torch.Generator().manual_seed(seed)
    k, v = (torch.randn(cap, b, hk, d, generator=gen).to(dtype) for _ in range(2))
    k[..., ::16] *= 4
    cache = buffers(b, hk, cap, d, bits, dev)
    kv_cache_write(*cache, k.to(dev), v.to(dev), 0)
    return cache, held(k, bits)[0], held(v, bits)[0]


def attend_reference(q, k, v, lengths, window, sinks, scale):
    q = q.cpu().double()
    tq, b, h, d = q.shape
    g = h // k.shape[2]
    out, mag = torch.zeros_like(q), torch.zeros_like(q)
    for s in range(b):
        n = min(max(int(lengths[s]), 0), k.shape[0])
        for i in range(tq):
            at = n - tq + i
            keys = [j for j in range(0, at + 1) if window == 0 or j > at - window or j < sinks]
            if not keys:
                continue
            for x in range(h):
                p = torch.softmax(k[keys, s, x // g] @ q[i, s, x] * scale, 0)
                out[i, s, x] = p @ v[keys, s, x // g]
                mag[i, s, x] = p @ v[keys, s, x // g].abs()
    return out, mag


def check(got, want, mag, dtype):
    got = got.cpu().double()
    assert got.shape == want.shape and torch.isfinite(got).all()
    bound = (2 * U[dtype] + 1e-5) * mag + U[dtype] * want.abs() + 1e-6
    assert ((got - want).abs() <= bound).all(), ((got - want).abs() / bound).max().item()


ATTEND = [
    # tq, b, h, hk, d, cap, lengths, window, sinks
    (1, 1, 1, 1, 64, 1, [1], 0, 0),
    (1, 4, 4, 2, 64, 33, [33, 1, 0, 17], 0, 0),
    (1, 3, 8, 1, 128, 95, [95, 64, 31], 0, 0),
    (3, 2, 4, 4, 128, 70, [70, 2], 0, 0),
    (2, 2, 16, 1, 64, 200, [200, 111], 0, 0),
    (5, 2, 8, 2, 64, 131, [131, 40], 9, 2),
    (1, 3, 4, 2, 64, 500, [500, 321, 5], 40, 4),
    (1, 2, 2, 2, 128, 500, [499, 100], 64, 37),
    (4, 1, 32, 4, 128, 300, [300], 100, 1),
    (1, 2, 2, 1, 64, 1500, [1500, 1499], 0, 0),
    (1, 1, 2, 1, 128, 3001, [2999], 2000, 65),
]


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("tq,b,h,hk,d,cap,lengths,window,sinks", ATTEND)
def test_attend(dev, tq, b, h, hk, d, cap, lengths, window, sinks, dtype, bits):
    cache, k, v = fill(b, hk, cap, d, bits, dtype, dev, cap)
    q = torch.randn(tq, b, h, d, generator=torch.Generator().manual_seed(7)).to(dtype).to(dev)
    n = torch.tensor(lengths, dtype=torch.int32, device=dev)
    want, mag = attend_reference(q, k, v, lengths, window, sinks, d ** -0.5)
    check(kv_cache_attend(q, *cache, n, max(lengths), window, sinks), want, mag, dtype)
    # `longest` is a bound: a larger one shares the work out differently
    check(kv_cache_attend(q, *cache, n, cap, window, sinks), want, mag, dtype)
    # the same call gives the same bits
    assert torch.equal(kv_cache_attend(q, *cache, n, cap, window, sinks), kv_cache_attend(q, *cache, n, cap, window, sinks))


@pytest.mark.parametrize("d,lengths", [(64, [26000, 3]), (128, [40, 66000])])
def test_attend_joins_many_parts(dev, d, lengths):
    """Few rows over long reaches: a hundred parts and the most there are, many of them empty for the short sequence."""
    cap = max(lengths)
    cache, k, v = fill(2, 1, cap, d, 8, torch.float16, dev, 9)
    q = torch.randn(1, 2, 3, d, generator=torch.Generator().manual_seed(8)).to(torch.float16).to(dev)
    n = torch.tensor(lengths, dtype=torch.int32, device=dev)
    want, mag = attend_reference(q, k, v, lengths, 0, 0, d ** -0.5)
    check(kv_cache_attend(q, *cache, n, cap, 0, 0), want, mag, torch.float16)


def test_attend_takes_strided_queries_other_scales_and_long_lengths(dev):
    cache, k, v = fill(2, 2, 100, 64, 8, torch.bfloat16, dev, 3)
    lin = torch.randn(1, 2, 8, 64, device=dev).to(torch.bfloat16)
    q = lin[:, :, :4]
    n = torch.tensor([100, 400], device=dev)                     # clamped to the capacity
    for scale in (0.0, -0.5, 0.2):
        want, mag = attend_reference(q, k, v, [100, 400], 30, 2, scale)
        check(kv_cache_attend(q, *cache, n, 100, 30, 2, scale), want, mag, torch.bfloat16)


def test_what_is_not_finite_reaches_only_who_sees_it(dev):
    cap, d = 200, 64
    k, v = (torch.randn(cap, 2, 1, d, device=dev).to(torch.float16) for _ in range(2))
    q = torch.randn(1, 2, 2, d, device=dev).to(torch.float16)
    n = torch.tensor([120, 120], dtype=torch.int32, device=dev)
    clean = buffers(2, 1, cap, d, 4, dev)
    kv_cache_write(*clean, k, v, 0)
    want = kv_cache_attend(q, *clean, n, cap, 40, 3)
    for lo, hi in ((3, 80), (120, 200)):                         # between sinks and window, behind the end
        k2, v2 = k.clone(), v.clone()
        k2[lo:hi], v2[lo:hi] = float("nan"), float("inf")
        cache = buffers(2, 1, cap, d, 4, dev)
        kv_cache_write(*cache, k2, v2, 0)
        assert torch.equal(kv_cache_attend(q, *cache, n, cap, 40, 3), want)
    v2 = v.clone()
    v2[100, 1, 0, 40] = float("nan")                             # seen by sequence 1: its second block of 32
    cache = buffers(2, 1, cap, d, 4, dev)
    kv_cache_write(*cache, k, v2, 0)
    got = kv_cache_attend(q, *cache, n, cap, 40, 3)
    assert torch.equal(got[:, 0], want[:, 0]) and torch.equal(got[:, 1, :, :32], want[:, 1, :, :32]) and torch.isnan(got[:, 1, :, 32:]).all()


def test_offsets_beyond_32_bits(dev):
    """A cache whose last rows lie more than 4 GB behind its first ones."""
    b, hk, cap, d = 3, 8, 1 << 21, 128                           # 64 bytes a row: 3.2 GB of codes each
    cache = buffers(b, hk, cap, d, 4, dev)
    assert cache[0].numel() > 1 << 31
    k, v = (torch.randn(40, b, hk, d, device=dev).to(torch.bfloat16) for _ in range(2))
    kv_cache_write(*cache, k, v, cap - 40)
    kk, vv = kv_cache_read(*cache, cap - 40, 40, torch.bfloat16)
    assert torch.equal(kk.cpu().double(), held(k.cpu(), 4)[0])
    q = torch.randn(1, b, hk, d, device=dev).to(torch.bfloat16)
    n = torch.full((b,), cap, dtype=torch.int32, device=dev)
    want, mag = attend_reference(q, held(k.cpu(), 4)[0], held(v.cpu(), 4)[0], [40] * b, 0, 0, d ** -0.5)
    check(kv_cache_attend(q, *cache, n, cap, 40, 0), want, mag, torch.bfloat16)


def test_cache_class_appends_reorders_and_refuses(dev):
    cache = QuantizedKVCache(3, 2, 64, 20, bits=8, dtype=torch.float16, device=dev)
    k, v = (torch.randn(20, 3, 2, 64, device=dev).to(torch.float16) for _ in range(2))
    cache.append(k[:5], v[:5], torch.tensor([5, 3, 0], device=dev))
    cache.append(k[5:6], v[5:6])
    assert cache.lengths.tolist() == [6, 4, 1] and cache.longest == 6
    kk, vv = cache.read()
    want = held(k.cpu(), 8)[0]
    assert torch.equal(kk[:6, 0].cpu().double(), want[:6, 0]) and torch.equal(kk[3, 1].cpu().double(), want[5, 1])
    assert torch.equal(kk[0, 2].cpu().double(), want[5, 2])
    q = torch.randn(1, 3, 4, 64, device=dev).to(torch.float16)
    out = cache.attend(q)
    cache.reorder(torch.tensor([2, 0, 0, 1], device=dev))
    assert cache.lengths.tolist() == [1, 6, 6, 4]
    assert torch.equal(cache.attend(q[:, [2, 0, 0, 1]]), out[:, [2, 0, 0, 1]])
    with pytest.raises(RuntimeError, match="do not fit"):
        cache.append(k[:, [0, 0, 0, 0]], v[:, [0, 0, 0, 0]])
    for args in (dict(bits=3), dict(head_dim=32), dict(dtype=torch.float32)):
        with pytest.raises(ValueError):
            QuantizedKVCache(**{**dict(batch=1, kv_heads=1, head_dim=64, capacity=4, device=dev), **args})


def test_refusals(dev):
    cache = buffers(2, 2, 10, 64, 4, dev)
    k = torch.randn(3, 2, 2, 64, device=dev).to(torch.bfloat16)
    for call, text in ((lambda: kv_cache_write(*cache, k, k, 8), "rows 8 .. 11"), (lambda: kv_cache_write(*cache, k, k, -1), "rows -1"),
                       (lambda: kv_cache_write(*cache, k[:, :1], k[:, :1], 0), "must be"), (lambda: kv_cache_write(*cache, k.float(), k, 0), "fp16 or bf16"),
                       (lambda: kv_cache_write(*cache, k.cpu(), k, 0), "device memory"), (lambda: kv_cache_write(*cache, k, k, torch.zeros(3, device=dev)), "integers"),
                       (lambda: kv_cache_write(cache[0][..., :20], *cache[1:], k, k, 0), "contiguous"), (lambda: kv_cache_write(*cache, k.requires_grad_(), k, 0), "no gradient"),
                       (lambda: kv_cache_read(*cache, 5, 6), "rows 5 .. 11"), (lambda: kv_cache_read(*cache, 0, 2, torch.float32), "fp16 or bf16"),
                       (lambda: kv_cache_attend(k.detach()[:1, :, :1], *cache, torch.zeros(2, dtype=torch.int32, device=dev), 10), "evenly"),
                       (lambda: kv_cache_attend(k.detach(), *cache, torch.zeros(2, dtype=torch.int32, device=dev), 11), "longest"),
                       (lambda: kv_cache_attend(k.detach(), *cache, torch.zeros(2, dtype=torch.int32, device=dev), 10, -1), "window")):
        with pytest.raises(RuntimeError, match=text):
            call()


def test_a_captured_step_replays(dev):
    cache = buffers(2, 2, 64, 64, 4, dev)
    starts = torch.tensor([0, 5], dtype=torch.int32, device=dev)
    k, v, q = (torch.randn(1, 2, n, 64, device=dev).to(torch.bfloat16) for n in (2, 2, 4))

    def step():
        kv_cache_write(*cache, k, v, starts)
        return kv_cache_attend(q, *cache, starts + 1, 64, 16, 2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = step()
    for i in range(4):
        for x in (k, v, q):
            x.copy_(torch.randn_like(x))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(res, step())
        starts += 1
