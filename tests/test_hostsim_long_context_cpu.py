"""Window attention and the quantised cache executed on the CPU: the kernels' own source through tests/hostsim, called by the C ABI,
against the same 64-bit definitions and bounds as on the GPU."""
import ctypes
import os
import sys

import pytest
import torch

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path.insert(0, os.path.join(HERE, "hostsim"))
import harness  # noqa: E402
import hostsim_build  # noqa: E402
import test_zzn_window_attention_gpu as wa  # noqa: E402
import test_zzo_quantized_cache_gpu as qc  # noqa: E402
from nmtgminor_amd import _lib  # noqa: E402
from test_marshalling_cpu import SIGS  # noqa: E402

pytestmark = pytest.mark.skipif(not hostsim_build.available(), reason="no clang++ to build the CPU simulator")
F16, BF16 = torch.float16, torch.bfloat16
BOTH = pytest.mark.parametrize("dtype", [F16, BF16])
WRAP = {"i64": _lib.i64, "i32": _lib.i32, "f32": _lib.f32}


@pytest.fixture(scope="module")
def lib():
    return harness.library()


@pytest.fixture(params=["late", "early"])
def dma(request, monkeypatch):
    monkeypatch.setenv("HOSTSIM_DMA", request.param)


def call(lib, name, *args, expect=0):
    """Arguments wrapped as the header declares them; tensors by their address."""
    kinds = SIGS["nmtg_" + name]
    assert len(kinds) == len(args) + (kinds[-1] == "ptr" and len(args) == len(kinds) - 1)
    args = list(args) + [None] * (len(kinds) - len(args))           # the stream
    wrapped = [WRAP[k](a) if k in WRAP else ctypes.c_void_p(a.data_ptr()) if isinstance(a, torch.Tensor) else a for k, a in zip(kinds, args)]
    fn = getattr(lib, "nmtg_" + name)
    fn.restype = ctypes.c_int64 if name.endswith("_bytes") else ctypes.c_int
    rc = fn(*wrapped)
    if name.endswith("_bytes"):
        return rc
    assert rc == expect, lib.nmtg_last_error()
    return lib.nmtg_last_error().decode()


def bytes256(n):
    buf = torch.full((n + 512,), 0xff, dtype=torch.uint8)           # fp32 NaN: what a kernel reads it has written
    return buf[(-buf.data_ptr()) % 256:][:max(n, 1)]


def strides(*tensors):
    flat = [s for t in tensors for s in t.stride()[:3]]
    return (ctypes.c_int64 * len(flat))(*flat)


def rest_of(q):
    t, b, h, d = q.shape
    return torch.full((b * h * ((t + 31) // 32) * 32 * d,), 0x7f, dtype=torch.uint8)          # NaN where nothing is written


def window(lib, q, k, v, dout, lengths, w, sinks, scale, dtype, keep_rest=True):
    t, b, h, d = q.shape
    sizes = (t, b, h, k.shape[2], d, w, sinks)
    out, rest, lse = torch.full_like(q, float("nan")), rest_of(q) if keep_rest else None, torch.full((b, h, t), float("nan"))
    call(lib, "window_attn_fwd", q, k, v, out, rest, lse, lengths, strides(q, k, v, out), *sizes, scale, _lib.dtype_code(dtype))
    grads = [torch.full_like(x, float("nan")) for x in (q, k, v)]
    ws = bytes256(call(lib, "window_attn_bwd_workspace_bytes", *sizes))
    call(lib, "window_attn_bwd", dout, q, k, v, out, rest, lse, *grads, lengths, strides(dout, q, k, v, out, *grads), *sizes, scale, _lib.dtype_code(dtype),
         ws, ws.numel())
    return [out, *grads]


CASES = [
    # t, b, h, hk, d, window, sinks, ragged
    (1, 1, 1, 1, 64, 1, 0, False),
    (65, 2, 2, 1, 128, 5, 64, True),
    (130, 2, 2, 1, 64, 33, 3, True),
    (200, 1, 1, 1, 128, 500, 0, False),
    (270, 1, 2, 1, 64, 7, 130, False),
    (330, 1, 1, 1, 128, 40, 4, False),
]


@BOTH
@pytest.mark.parametrize("t,b,h,hk,d,w,sinks,ragged", CASES)
def test_window_attention(lib, dma, t, b, h, hk, d, w, sinks, ragged, dtype):
    q, k, v, dout = wa.inputs(t, b, h, hk, d, dtype, "cpu", t)
    lengths = torch.tensor([(t, t // 2)[i % 2] for i in range(b)], dtype=torch.int32) if ragged else None
    want, mag = wa.reference(q, k, v, dout, lengths, w, sinks, d ** -0.5)
    if ragged:
        for x in (q, k, v, dout):
            for s in range(b):
                x[int(lengths[s]):, s] = float("nan")
    wa.check(window(lib, q, k, v, dout, lengths, w, sinks, d ** -0.5, dtype), want, mag, dtype)


@pytest.mark.parametrize("order", ["reverse", "random", "interleave"])
def test_window_attention_whatever_the_wavefronts_order(lib, order, monkeypatch):
    monkeypatch.setenv("HOSTSIM_ORDER", order)
    q, k, v, dout = wa.inputs(200, 1, 2, 1, 64, BF16, "cpu", 8)
    want, mag = wa.reference(q, k, v, dout, None, 20, 3, -0.2)
    wa.check(window(lib, q, k, v, dout, None, 20, 3, -0.2, BF16), want, mag, BF16)


def test_window_attention_without_the_rest(lib):
    """The rest of the output left out: the same output, gradients with D of the rounded one (within the same bounds)."""
    q, k, v, dout = wa.inputs(150, 1, 2, 1, 64, BF16, "cpu", 4)
    want, mag = wa.reference(q, k, v, dout, None, 40, 3, 0.125)
    got = window(lib, q, k, v, dout, None, 40, 3, 0.125, BF16, keep_rest=False)
    wa.check(got, want, mag, BF16)
    whole = window(lib, q, k, v, dout, None, 40, 3, 0.125, BF16)
    assert torch.equal(got[0], whole[0]) and torch.equal(got[3], whole[3]) and not torch.equal(got[1], whole[1])
    error = lambda x: (x[1].double() - want[1]).norm()                                          # noqa: E731
    assert error(whole) < error(got)


def test_window_attention_of_slots(lib):
    """Queries, keys and values as slots of one projection, gradients into the slots of another."""
    t, b, h, hk, d = 70, 2, 2, 1, 64
    lin, dlin = torch.randn(t, b, h + 2 * hk, d).to(BF16), torch.full((t, b, h + 2 * hk, d), float("nan"), dtype=BF16)
    q, k, v = lin.split((h, hk, hk), 2)
    dout = torch.randn(t, b, h, d).to(BF16)
    dense = window(lib, q.contiguous(), k.contiguous(), v.contiguous(), dout, None, 9, 2, 0.125, BF16)
    out, rest, lse = torch.empty(t, b, h, d, dtype=BF16), rest_of(q), torch.empty(b, h, t)
    sizes = (t, b, h, hk, d, 9, 2)
    call(lib, "window_attn_fwd", q, k, v, out, rest, lse, None, strides(q, k, v, out), *sizes, 0.125, _lib.BF16)
    ws = bytes256(call(lib, "window_attn_bwd_workspace_bytes", *sizes))
    grads = dlin.split((h, hk, hk), 2)
    call(lib, "window_attn_bwd", dout, q, k, v, out, rest, lse, *grads, None, strides(dout, q, k, v, out, *grads), *sizes, 0.125, _lib.BF16, ws, ws.numel())
    for x, y in zip((out, *grads), dense):
        assert torch.equal(x, y)


def test_window_attention_refuses(lib):
    q, k, v, dout = wa.inputs(4, 1, 2, 1, 64, BF16, "cpu")
    out, lse = torch.empty_like(q), torch.empty(1, 2, 4)
    good = dict(t=4, b=1, h=2, hk=1, d=64, w=3, s=0, scale=0.125, dtype=_lib.BF16)

    def run(**change):
        c = {**good, **change}
        st = c.pop("strides", strides(q, k, v, out))
        p = c.pop("q", q)
        return call(lib, "window_attn_fwd", p, k, v, out, None, lse, None, st, *c.values(), expect=c.pop("rc", -1))
    for change, text in ((dict(d=32), "head dimension 32"), (dict(h=3, hk=2), "evenly"), (dict(w=0), "window 0"), (dict(s=-1), "sinks -1"),
                         (dict(dtype=_lib.F32), "fp16 or bf16"), (dict(scale=float("nan")), "scale"), (dict(t=-1), "bad shape"),
                         (dict(b=70000), "65535"), (dict(q=None), "null pointer"), (dict(strides=(ctypes.c_int64 * 12)(*([4] * 12))), "multiples of 8")):
        assert text in run(**change)
    grads = [torch.empty_like(x) for x in (q, k, v)]
    assert "workspace" in call(lib, "window_attn_bwd", dout, q, k, v, out, None, lse, *grads, None, strides(dout, q, k, v, out, *grads), 4, 1, 2, 1, 64, 3, 0, 0.125,
                               _lib.BF16, bytes256(64), 16, expect=-1)
    call(lib, "window_attn_fwd", None, None, None, None, None, None, None, None, 0, 1, 2, 1, 64, 3, 0, 0.125, _lib.BF16)      # nothing to do


# ------------------------------------------------------------------------------------------------------ quantised cache
def cache_sizes(cache):
    b, hk, cap, _ = cache[0].shape
    d = 32 * cache[1].shape[-1]
    return b, hk, d, cap, cache[0].shape[-1] * 8 // d


def write(lib, cache, k, v, starts, start, expect=0):
    b, hk, d, cap, bits = cache_sizes(cache)
    return call(lib, "kv_cache_write", k, *k.stride()[:3], v, *v.stride()[:3], *cache, starts, start, k.shape[0], b, hk, d, cap, bits,
                _lib.dtype_code(k), expect=expect)


def read(lib, cache, starts, start, count, dtype):
    b, hk, d, cap, bits = cache_sizes(cache)
    k, v = (torch.full((count, b, hk, d), float("nan"), dtype=dtype) for _ in range(2))
    call(lib, "kv_cache_read", *cache, k, v, starts, start, count, b, hk, d, cap, bits, _lib.dtype_code(dtype))
    return k, v


def attend(lib, q, cache, lengths, longest, w, sinks, scale, expect=0):
    tq, b, h, d = q.shape
    _, hk, _, cap, bits = cache_sizes(cache)
    out = torch.full_like(q, float("nan"))
    ws = bytes256(call(lib, "kv_cache_attn_workspace_bytes", tq, b, h, hk, d, longest, w, sinks))
    said = call(lib, "kv_cache_attn", q, *q.stride()[:3], *cache, lengths, out, *out.stride()[:3], tq, b, h, hk, d, cap, longest, w, sinks, scale, bits,
                _lib.dtype_code(q), ws, ws.numel(), expect=expect)
    return said if expect else out


@BOTH
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("count,b,hk,d,cap", [(1, 3, 2, 64, 5), (11, 2, 1, 128, 13), (35, 1, 3, 64, 40)])
def test_rows_written_and_read(lib, count, b, hk, d, cap, bits, dtype):
    k, v = (torch.randn(count, b, hk, d) * torch.exp2(torch.randint(-6, 6, (count, b, hk, 1)).float()) for _ in range(2))
    k, v = k.to(dtype), v.to(dtype)
    k[0, 0, 0, 5] = float("inf")
    cache = qc.buffers(b, hk, cap, d, bits, "cpu", fill=7)
    starts = torch.tensor([cap - count - i for i in range(b)], dtype=torch.int32)      # a sequence may begin in front of the cache
    write(lib, cache, k, v, starts, 0)
    for x, got in zip((k, v), read(lib, cache, starts, 0, count, dtype)):
        want = qc.held(x, bits)[0]
        for s in range(b):
            skip = max(0, -int(starts[s]))
            assert not got[:skip, s].any()
            assert torch.equal(torch.nan_to_num(got[skip:, s].double(), nan=-9.0), torch.nan_to_num(want[skip:, s], nan=-9.0))
    assert "rows" in write(lib, cache, k, v, None, cap - count + 1, expect=-1)


@BOTH
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("tq,b,h,hk,d,cap,lengths,w,sinks", [
    (1, 3, 2, 1, 64, 45, [45, 0, 31], 0, 0),
    (3, 2, 8, 1, 128, 77, [77, 2], 9, 3),
    (1, 1, 2, 1, 64, 2113, [2100], 0, 0),
])
def test_attention_over_the_cache(lib, tq, b, h, hk, d, cap, lengths, w, sinks, bits, dtype):
    gen = torch.Generator().manual_seed(cap)
    k, v = (torch.randn(cap, b, hk, d, generator=gen).to(dtype) for _ in range(2))
    for s in range(b):                              # not written yet: nobody's business
        k[lengths[s]:, s], v[lengths[s]:, s] = float("nan"), float("inf")
    cache = qc.buffers(b, hk, cap, d, bits, "cpu")
    write(lib, cache, k, v, None, 0)
    q = torch.randn(tq, b, h, d, generator=gen).to(dtype)
    kk, vv = (torch.nan_to_num(qc.held(torch.nan_to_num(x, posinf=0.0), bits)[0]) for x in (k, v))
    want, mag = qc.attend_reference(q, kk, vv, lengths, w, sinks, d ** -0.5)
    qc.check(attend(lib, q, cache, torch.tensor(lengths, dtype=torch.int32), max(lengths), w, sinks, d ** -0.5), want, mag, dtype)


def test_cache_refuses(lib):
    cache = qc.buffers(1, 1, 8, 64, 4, "cpu")
    q = torch.zeros(1, 1, 2, 64, dtype=BF16)
    n = torch.tensor([3], dtype=torch.int32)
    assert "longest" in attend(lib, q, cache, n, 9, 0, 0, 0.1, expect=-1)
    assert "window" in attend(lib, q, cache, n, 8, -1, 0, 0.1, expect=-1)
    assert "null pointer" in call(lib, "kv_cache_read", *cache, None, None, None, 0, 1, 1, 1, 64, 8, 4, _lib.BF16, expect=-1)
    assert "bits" in call(lib, "kv_cache_read", *cache, q, q, None, 0, 1, 1, 1, 64, 8, 5, _lib.BF16, expect=-1)
    assert "workspace" in call(lib, "kv_cache_attn", q, 128, 128, 64, *cache, n, q, 128, 128, 64, 1, 1, 2, 1, 64, 4096, 4096, 0, 0, 0.1, 4, _lib.BF16, None, 0,
                               expect=-1)
