"""A key / value cache in 4 or 8 bits for incremental decoding.

Caches of the working dtype cost 2 * 2 * head_dim bytes per position and head, and a decoding step is bound by reading
them. Here a block of 32 neighbouring elements of a row keeps one scale byte (a power of two) and 32 elements of 4 bits
(E2M1) or 8 bits (E4M3): 0.53 or 1.03 bytes per element. include/nmtg_hip.h has the format.

    kv_cache_write(k_codes, k_scales, v_codes, v_scales, k, v, start)       rows k, v [count, B, H_kv, D] from position
                                                                            start (an int, or int32 [B] on the device)
    kv_cache_read(k_codes, k_scales, v_codes, v_scales, start, count, dtype)   -> k, v [count, B, H_kv, D]
    kv_cache_attend(q, k_codes, k_scales, v_codes, v_scales, lengths, longest, window, sinks, softmax_scale)
                                                                            -> [tq, B, H, D] of the newest tq positions

    QuantizedKVCache                                                        the four buffers with their lengths

Inference only: nothing here has a gradient, and torch.jit.trace is refused. Every call enqueues on the current stream and returns.
"""
import torch

from .. import _lib as L


def _start(start):
    """-> (device tensor or None, int)"""
    return (start, 0) if isinstance(start, torch.Tensor) else (None, int(start))


def kv_cache_write(k_codes, k_scales, v_codes, v_scales, k, v, start):
    """Quantises k and v [count, B, H_kv, D] (fp16 or bf16, any strides with a contiguous D that are multiples of 8) into
    the cache rows start .. start + count of every sequence. With a tensor of starts, rows outside the cache are dropped;
    with an int they are an error."""
    L.refuse_tracing("kv_cache_write")
    L.host().kv_cache_write(k_codes, k_scales, v_codes, v_scales, k, v, *_start(start))


def kv_cache_read(k_codes, k_scales, v_codes, v_scales, start, count, dtype=torch.bfloat16):
    """The values that cache rows start .. start + count stand for, k and v [count, B, H_kv, D]. With a tensor of starts,
    positions outside the cache read as zeros."""
    L.refuse_tracing("kv_cache_read")
    return L.host().kv_cache_read(k_codes, k_scales, v_codes, v_scales, *_start(start), count, dtype)


def kv_cache_attend(q, k_codes, k_scales, v_codes, v_scales, lengths, longest, window=0, sinks=0, softmax_scale=None):
    """q [tq, B, H, D]: the newest tq positions of every sequence, which hold lengths[b] positions (int32 on the device,
    these included), at most `longest`. Position p sees positions up to p; with window > 0 the last `window` of them (itself
    included) and the first `sinks` positions only. H is a multiple of the cache's heads, softmax_scale defaults to D^-0.5."""
    L.refuse_tracing("kv_cache_attend")
    return L.host().kv_cache_attend(q, k_codes, k_scales, v_codes, v_scales, lengths, longest, window, sinks, softmax_scale)


class QuantizedKVCache:
    """Buffers for `capacity` positions of `batch` sequences and what they hold: `lengths` (int32 [batch] on the device) and
    `longest` (an upper bound of them that the host knows without asking the device)."""

    def __init__(self, batch, kv_heads, head_dim, capacity, bits=4, dtype=torch.bfloat16, device="cuda"):
        if bits not in (4, 8):
            raise ValueError(f"quantised cache: {bits} bits per element (4 and 8 are built)")
        if head_dim not in (64, 128):
            raise ValueError(f"quantised cache: head dimension {head_dim} (64 and 128 are built)")
        if dtype not in (torch.float16, torch.bfloat16):
            raise ValueError("quantised cache: fp16 or bf16 tensors required")
        shape = (batch, kv_heads, capacity)
        self.bits, self.dtype, self.capacity = bits, dtype, capacity
        self.k_codes, self.v_codes = (torch.zeros(shape + (head_dim * bits // 8,), dtype=torch.uint8, device=device) for _ in range(2))
        self.k_scales, self.v_scales = (torch.zeros(shape + (head_dim // 32,), dtype=torch.uint8, device=device) for _ in range(2))
        self.lengths = torch.zeros(batch, dtype=torch.int32, device=device)
        self.longest = 0

    @property
    def tensors(self):
        return self.k_codes, self.k_scales, self.v_codes, self.v_scales

    def append(self, k, v, counts=None):
        """Writes k, v [T, B, H_kv, D] behind what every sequence holds. counts (integers [B] on the device, clamped to [0, T]): how
        many of the T rows are a sequence's own; those behind are written and not counted, the next rows go over them."""
        t = k.shape[0]
        if self.longest + t > self.capacity:
            raise RuntimeError(f"quantised cache: {self.longest} + {t} positions do not fit a capacity of {self.capacity}")
        kv_cache_write(*self.tensors, k, v, self.lengths)
        if counts is not None and counts.dtype != torch.bool:
            counts = counts.clamp(0, t)
        self.lengths += t if counts is None else counts.to(self.lengths)
        self.longest += t

    def read(self, start=0, count=None):
        return kv_cache_read(*self.tensors, start, self.longest - start if count is None else count, self.dtype)

    def attend(self, q, window=0, sinks=0, softmax_scale=None):
        return kv_cache_attend(q, *self.tensors, self.lengths, self.longest, window, sinks, softmax_scale)

    def reorder(self, index):
        """Sequence i becomes what sequence index[i] was (beam search); the number of sequences may change."""
        self.k_codes, self.k_scales, self.v_codes, self.v_scales, self.lengths = (
            x.index_select(0, index) for x in (*self.tensors, self.lengths))
