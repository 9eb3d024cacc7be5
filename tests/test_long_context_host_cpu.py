"""What window attention and the quantised cache decide before they touch a GPU."""
import pytest
import torch

from nmtgminor_amd.modules import quantized_cache as qc
from nmtgminor_amd.modules.window_attention import WindowSelfMultiheadAttn, window_attn_func


def test_tracing_is_refused():
    q = torch.zeros(3, 1, 2, 64, dtype=torch.bfloat16)
    cache = qc.QuantizedKVCache(1, 2, 64, 8, device="cpu")
    m = WindowSelfMultiheadAttn(128, 2, window=4).bfloat16().requires_grad_(False)
    for call, arg in ((lambda y: window_attn_func(y, q, q, 4), q), (m, torch.zeros(3, 1, 128, dtype=torch.bfloat16)),
                      (lambda y: cache.append(y, q) or y, q), (lambda y: cache.read()[0], q), (lambda y: cache.attend(y), q)):
        with pytest.raises(RuntimeError, match="cannot be traced"):
            torch.jit.trace(call, (arg,), check_trace=False)
    assert cache.longest == 0


def test_a_module_in_32_bits_has_a_cache():
    """Of the type that its rows will have: autocast's, or bf16 outside of it; another by name. (torch.autocast does nothing for a GPU that is
    not there: its state is set by hand.)"""
    m = WindowSelfMultiheadAttn(128, 2, window=4, num_kv_heads=1)
    assert m.make_cache(3, 8).dtype == torch.bfloat16
    for dtype in (torch.float16, torch.bfloat16):
        before = torch.get_autocast_dtype("cuda")
        torch.set_autocast_enabled("cuda", True)
        torch.set_autocast_dtype("cuda", dtype)
        try:
            cache = m.make_cache(3, 8)
        finally:
            torch.set_autocast_enabled("cuda", False)
            torch.set_autocast_dtype("cuda", before)
        assert cache.dtype == dtype and cache.k_codes.shape == (3, 1, 8, 32)
        assert m.make_cache(3, 8, dtype=dtype).dtype == dtype
        half = WindowSelfMultiheadAttn(128, 2, window=4).to(dtype)
        assert half.make_cache(1, 4).dtype == dtype
    with pytest.raises(ValueError, match="fp16 or bf16"):
        m.make_cache(3, 8, dtype=torch.float32)


def test_appended_counts_are_those_of_rows_that_were_appended(monkeypatch):
    """As in window_attn_func, whose lengths are clamped to the positions there are."""
    monkeypatch.setattr(qc, "kv_cache_write", lambda *a: None)
    rows = torch.zeros(5, 4, 2, 64, dtype=torch.bfloat16)
    for kind in (torch.int32, torch.int64):
        cache = qc.QuantizedKVCache(4, 2, 64, 16, device="cpu")
        cache.append(rows, rows, torch.tensor([9, -2, 3, 5], dtype=kind))
        assert cache.lengths.tolist() == [5, 0, 3, 5] and cache.lengths.dtype == torch.int32 and cache.longest == 5
        cache.append(rows[:1], rows[:1], torch.tensor([True, False, False, True]))
        assert cache.lengths.tolist() == [6, 0, 3, 6]
    cache.append(rows, rows, torch.tensor([1 << 32, -(1 << 32), (1 << 32) + 1, 0]))
    assert cache.lengths.tolist() == [11, 0, 8, 6]
