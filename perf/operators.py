"""The operators of long-context decoders that this library is timed on: attention with a sliding window and a few first tokens
that stay visible (sinks), forward and in training, and the quantised key / value cache that such a decoder is served from: rows
written in 4 or 8 bits, read back, and attended to by the newest positions.

`listed()` are the representative cases, `draw(rng)` gives more of the same ranges; `prepare(case, seed)` makes what the program
has in hand (projections, a filled cache), `run(state)` is one pass and returns everything it computes, `work(case)` the bytes
and operations a pass cannot do without, `exact(case, seed)` the results in 64 bits from the operators' definitions.

Where `own` is false, `run` computes the same in elementary torch operations in 32 bits, rounded once at the end.

The operators:
  window attention   query i of a sequence sees key j where j <= i and (j > i - window or j < sinks); positions at and behind
                     a sequence's length see nothing and are seen by nobody (output and gradients zero). Several query heads may
                     share a key / value head.
  cache              rows of blocks of 32 elements, each with a power-of-two scale 2^(byte - 127) and elements of 4 bits (sign,
                     2 exponent and 1 mantissa bits: 0, 0.5, 1, 1.5, 2, 3, 4, 6) or 8 bits (4 exponent and 3 mantissa bits, up to
                     448). The scale of a block is the smallest power of two under which its largest magnitude is at most 7
                     (464): no element is further from its held value than half a step. Ties round to even.
  cache attention    the newest positions of every sequence, query i of n at position length - n + i, under the same rule of
                     visibility (window 0: every position up to its own).

Sizes follow the benchmark (bench.py, nmtgminor_amd/synthetic.py) where it has them: model dimension 512 with 8 heads of 64 and
1024 with 16, up to 512 positions and 32 sentences, 1500 speech frames, a beam of 5; heads of 128 shared by four query heads and
lengths up to 32768 stand for long documents.
"""
import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
BLOCK = 32
TOP = {4: (2, 0.875, 6.0), 8: (8, 0.90625, 448.0)}     # exponent of the largest element, where frexp's mantissa moves the scale up, largest
MOST_FLOPS = 9.0e11                                     # of the largest listed attention
MOST_CACHE = 1 << 30                                    # elements of the largest listed cache, keys alone
MOST_WRITE = 1 << 26


def listed():
    return [
        # A beam of 5 short sentences through one layer without gradients: latency counts.
        dict(name="window_short", kind="window", train=False, t=61, b=5, heads=8, kv_heads=8, dim=64, window=32, sinks=4, ragged=True, dtype="f16"),
        # The prompt of a long document, heads shared by four: the forward pass as serving runs it.
        dict(name="window_prompt", kind="window", train=False, t=16384, b=1, heads=32, kv_heads=8, dim=128, window=4096, sinks=4, ragged=False, dtype="bf16"),
        # Training on a small ragged batch of odd sizes, gradients of shared heads.
        dict(name="window_train_ragged", kind="window", train=True, t=509, b=13, heads=8, kv_heads=2, dim=64, window=100, sinks=1, ragged=True, dtype="f16"),
        # Training of the large model's self-attention (16 heads of 64) on documents of 2048 positions.
        dict(name="window_train_large", kind="window", train=True, t=2048, b=8, heads=16, kv_heads=16, dim=64, window=512, sinks=4, ragged=False, dtype="bf16"),
        # Training on long documents, heads of 128 shared by four.
        dict(name="window_train_long", kind="window", train=True, t=8192, b=2, heads=32, kv_heads=8, dim=128, window=1024, sinks=4, ragged=False, dtype="bf16"),
        # The cache rows of one decoding step, every sentence at a position of its own: latency counts.
        dict(name="write_step", kind="write", count=1, b=32, kv_heads=16, dim=64, bits=8, cap=512, dtype="f16"),
        # The cache rows of a batch of long prompts.
        dict(name="write_prompt", kind="write", count=8192, b=8, kv_heads=8, dim=128, bits=4, cap=8200, dtype="bf16"),
        # A speech encoder's 1500 frames read back for an operator that takes 16-bit tensors.
        dict(name="read_speech", kind="read", count=1500, b=16, kv_heads=16, dim=64, bits=8, cap=1500, dtype="f16"),
        # A long prompt's rows read back.
        dict(name="read_long", kind="read", count=32768, b=4, kv_heads=8, dim=128, bits=4, cap=32768, dtype="bf16"),
        # One decoding step of a beam of 5 over a short cache: latency counts.
        dict(name="attend_beam5", kind="attend", tq=1, longest=61, cap=320, b=5, heads=8, kv_heads=8, dim=64, window=0, sinks=0, bits=4, dtype="f16"),
        # One decoding step of a batch whose layers see a window and the first tokens.
        dict(name="attend_window", kind="attend", tq=1, longest=8191, cap=8192, b=64, heads=16, kv_heads=4, dim=64, window=1024, sinks=4, bits=8, dtype="bf16"),
        # One decoding step of a full batch of long documents, all of the cache.
        dict(name="attend_long", kind="attend", tq=1, longest=32768, cap=32768, b=32, heads=32, kv_heads=8, dim=128, window=0, sinks=0, bits=4, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("window", "window", "window", "write", "read", "attend", "attend"))
    heads, kv_heads = rng.choice(((8, 8), (16, 16), (8, 2), (16, 4), (32, 8), (8, 1)))
    dim, dtype, bits = rng.choice((64, 128)), rng.choice(("f16", "bf16")), rng.choice((4, 8))
    sinks = rng.choice((0, 1, 4, 4, 37))
    if kind == "window":
        # (training from 16 positions: where every position sees one key, the gradients of queries and keys are zero)
        train = rng.random() < 0.6
        case = dict(kind=kind, train=train, t=_log(rng, 16 if train else 1, 16384), b=_log(rng, 1, 32), heads=heads, kv_heads=kv_heads, dim=dim,
                    window=_log(rng, 8, 4096), sinks=sinks, ragged=rng.random() < 0.5, dtype=dtype)
        while case["b"] > 1 and (work(case)["flops"] > MOST_FLOPS or case["t"] * case["b"] > 16384):
            case["b"] //= 2
        while work(case)["flops"] > MOST_FLOPS:
            case["window"] = case["window"] // 2 + 1
        return case
    if kind in ("write", "read"):
        case = dict(kind=kind, count=_log(rng, 1, 32768), b=_log(rng, 1, 64), kv_heads=kv_heads, dim=dim, bits=bits, cap=0, dtype=dtype)
        while case["b"] > 1 and case["count"] * case["b"] * kv_heads * dim > MOST_WRITE:
            case["b"] //= 2
        case["cap"] = case["count"] + _log(rng, 1, 512)
        return case
    case = dict(kind=kind, tq=rng.choice((1, 1, 1, 2, 5)), longest=_log(rng, 1, 32768), cap=0, b=_log(rng, 1, 64), heads=heads, kv_heads=kv_heads,
                dim=dim, window=rng.choice((0, _log(rng, 8, 4096))), sinks=sinks, bits=bits, dtype=dtype)
    while case["b"] > 1 and case["longest"] * case["b"] * kv_heads * dim > MOST_CACHE:
        case["b"] //= 2
    case["cap"] = case["longest"] + _log(rng, 1, 512)
    return case


# ------------------------------------------------------------------------------------------------------------- inputs
def _spread(n, b, ragged=True):
    """Lengths between half of n and all of it, the first the longest: the same for every seed, so that work() knows them."""
    return [max(1, n - (i * (n // 2)) // max(1, b - 1)) if ragged else n for i in range(b)]


def _keys(shape, dtype):
    """Keys have a few channels of large magnitude in every head, values have not."""
    k = torch.randn(shape, device=DEVICE)
    k[..., ::16] *= 4.0
    return k.to(dtype)


def _held(case):
    """Codes and scales of a filled cache: [b, kv_heads, cap, dim * bits / 8] and [b, kv_heads, cap, dim / 32] bytes."""
    shape = (case["b"], case["kv_heads"], case["cap"], case["dim"])
    return [t for x in (_keys(shape, DTYPES[case["dtype"]]), torch.randn(shape, device=DEVICE, dtype=DTYPES[case["dtype"]]))
            for t in _encode(x.float(), case["bits"])]


def prepare(case, seed):
    torch.manual_seed(seed)
    torch.cuda.manual_seed_all(seed)
    s, dtype = dict(case), DTYPES[case["dtype"]]
    b, dim = case["b"], case["dim"]
    if case["kind"] == "window":
        # the heads of one projection, side by side: queries, keys, values
        h, hk, t = case["heads"], case["kv_heads"], case["t"]
        lin = torch.randn(t, b, h + 2 * hk, dim, device=DEVICE, dtype=dtype)
        lin[:, :, h:h + hk, ::16] *= 2.0
        s["q"], s["k"], s["v"] = (x.detach().requires_grad_(case["train"]) for x in lin.split((h, hk, hk), dim=2))
        s["lengths"] = torch.tensor(_spread(t, b), dtype=torch.int32, device=DEVICE) if case["ragged"] else None
        s["dout"] = torch.randn(t, b, h, dim, device=DEVICE, dtype=dtype) if case["train"] else None
        return s
    if case["kind"] == "write":
        rows = (case["count"], b, case["kv_heads"])
        s["k"], s["v"] = _keys(rows + (dim,), dtype), torch.randn(rows + (dim,), device=DEVICE, dtype=dtype)
        held = (b, case["kv_heads"], case["cap"])
        s["cache"] = [torch.zeros(held + (w,), dtype=torch.uint8, device=DEVICE) for w in (dim * case["bits"] // 8, dim // BLOCK) * 2]
        # every sequence continues where it is; the longest fills the cache
        s["start"] = torch.tensor([n - 1 for n in _spread(case["cap"] - case["count"] + 1, b)], dtype=torch.int32, device=DEVICE)
        return s
    s["cache"] = _held(case)
    if case["kind"] == "read":
        return s
    s["q"] = torch.randn(case["tq"], b, case["heads"], dim, device=DEVICE, dtype=dtype)
    s["lengths"] = torch.tensor(_spread(case["longest"], b), dtype=torch.int32, device=DEVICE)
    return s


# --------------------------------------------------------------------------------------------------------------- passes
def run(s):
    if own:
        return _own(s)
    if s["kind"] == "window":
        return _window(s)
    if s["kind"] == "attend":
        with torch.no_grad():
            return _attend(s)
    with torch.no_grad():
        if s["kind"] == "write":
            _write(s)
            rows = s["start"].long()[:, None] + torch.arange(s["count"], device=DEVICE)
        else:
            rows = torch.arange(s["count"], device=DEVICE).expand(s["b"], -1)
        return [x.permute(2, 0, 1, 3).to(DTYPES[s["dtype"]]).contiguous() for x in _rows(s, rows)]


def _own(s):
    from nmtgminor_amd.modules.quantized_cache import kv_cache_attend, kv_cache_read, kv_cache_write
    from nmtgminor_amd.modules.window_attention import window_attn_func
    if s["kind"] == "window":
        out = window_attn_func(s["q"], s["k"], s["v"], s["window"], s["sinks"], lengths=s["lengths"])
        if not s["train"]:
            return [out]
        return [out.detach(), *torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["dout"])]
    if s["kind"] == "attend":
        return [kv_cache_attend(s["q"], *s["cache"], s["lengths"], s["longest"], s["window"], s["sinks"])]
    if s["kind"] == "write":
        kv_cache_write(*s["cache"], s["k"], s["v"], s["start"])
        return list(kv_cache_read(*s["cache"], s["start"], s["count"], s["k"].dtype))
    return list(kv_cache_read(*s["cache"], 0, s["count"], DTYPES[s["dtype"]]))


def _window(s):
    """Chunks of query positions against the band of keys that their windows reach, the sinks in front of it."""
    q, k, v = (s[n].detach().float() for n in "qkv")
    (t, b, h, d), hk, w, sinks = q.shape, k.shape[2], s["window"], min(s["sinks"], q.shape[0])
    c = min(t, max(128, w))
    n, g, scale = -(-t // c), h // k.shape[2], q.shape[3] ** -0.5
    qpos = torch.arange(n * c, device=DEVICE).view(n, c)
    kpos = torch.cat((torch.arange(sinks, device=DEVICE).expand(n, -1),
                      torch.arange(n, device=DEVICE)[:, None] * c - w + 1 + torch.arange(w + c - 1, device=DEVICE)), 1)
    ends = torch.full((b,), t, device=DEVICE) if s["lengths"] is None else s["lengths"].long()
    first = qpos[:, :, None] - w + 1                                     # of each position's window
    at = kpos[:, None, :]
    slot = torch.arange(kpos.shape[1], device=DEVICE) < sinks            # in front of the window only, or they would count twice
    sees = torch.where(slot, at < first, (at >= first) & (at >= 0)) & (at <= qpos[:, :, None])
    sees = sees[:, None] & (at[:, None] < ends[None, :, None, None]) & (qpos[:, None, :, None] < ends[None, :, None, None])
    sees = sees[:, :, None, None]                                        # [n, b, 1, 1, c, p]
    rows, cols = qpos.clamp(max=t - 1), kpos.clamp(0, t - 1)
    qc = q[rows].view(n, c, b, hk, g, d).permute(0, 2, 3, 4, 1, 5)       # [n, b, hk, g, c, d]
    kc, vc = (x[cols].permute(0, 2, 3, 1, 4).unsqueeze(3) for x in (k, v))   # [n, b, hk, 1, p, d]
    flat = lambda x: x.reshape(n, b, hk, g * c, x.shape[-1])             # noqa: E731
    p = (flat(qc) @ kc.squeeze(3).transpose(-1, -2)).view(n, b, hk, g, c, -1) * scale
    p = p.masked_fill(~sees, -math.inf)
    top = p.amax(-1, keepdim=True)
    p = torch.exp(p - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, torch.ones_like(total), total)
    back = lambda x: x.reshape(n, b, hk, g, c, d).permute(0, 4, 1, 2, 3, 5).reshape(n * c, b, h, d)[:t]   # noqa: E731
    out = flat(p) @ vc.squeeze(3)
    if not s["train"]:
        return [back(out).to(s["q"].dtype)]
    do = s["dout"].float()[rows].view(n, c, b, hk, g, d).permute(0, 2, 3, 4, 1, 5)
    dp = (flat(do) @ vc.squeeze(3).transpose(-1, -2)).view(p.shape)
    ds = p * (dp - (flat(do) * out).sum(-1).view(n, b, hk, g, c, 1))
    del dp
    dq = flat(ds) @ kc.squeeze(3) * scale
    dkc, dvc = flat(ds).transpose(-1, -2) @ flat(qc) * scale, flat(p).transpose(-1, -2) @ flat(do)
    dk, dv = (torch.zeros(t, b, hk, d, device=DEVICE).index_add_(0, cols.reshape(-1), x.permute(0, 3, 1, 2, 4).reshape(-1, b, hk, d)) for x in (dkc, dvc))
    return [x.to(s["q"].dtype) for x in (back(out), back(dq), dk, dv)]


def _encode(x, bits):
    """x [..., dim] in fp32 -> codes [..., dim * bits / 8] and scales [..., dim / 32], bytes."""
    top, up, most = TOP[bits]
    blocks = x.view(*x.shape[:-1], -1, BLOCK)
    amax = blocks.abs().amax(-1)
    mantissa, exponent = torch.frexp(amax)
    byte = (exponent - 1 - top + (mantissa > up).int() + 127).clamp(1, 254)
    y = torch.ldexp(blocks, (127 - byte)[..., None])
    if bits == 8:
        return y.clamp(-most, most).to(torch.float8_e4m3fn).view(torch.uint8).view(x.shape), byte.to(torch.uint8)
    magnitude = y.abs()
    step = torch.where(magnitude < 2, 0.5, torch.where(magnitude < 4, 1.0, 2.0))
    magnitude = (torch.round(magnitude / step) * step).clamp(max=most)
    code = ((magnitude[..., None] >= torch.tensor([0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=x.device)).sum(-1) + 8 * torch.signbit(y)).to(torch.uint8)
    code = code.view(*x.shape[:-1], -1, 2)
    return code[..., 0] | (code[..., 1] << 4), byte.to(torch.uint8)


def _decode(codes, scales, bits):
    """-> fp32 [..., dim]"""
    if bits == 8:
        x = codes.view(torch.float8_e4m3fn).float()
    else:
        table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=codes.device)
        nibbles = torch.stack((codes & 15, codes >> 4), -1).view(*codes.shape[:-1], -1)
        x = table[(nibbles & 7).int()] * (1.0 - 2.0 * (nibbles >> 3).float())
    x = x.view(*scales.shape, BLOCK)
    return torch.ldexp(x, (scales.int() - 127)[..., None]).view(*scales.shape[:-1], -1)


def _rows(s, rows):
    """Keys and values in fp32, [b, kv_heads, n, dim], of the cache rows [b, n]."""
    kc, ks, vc, vs = s["cache"]
    at = (torch.arange(s["b"], device=DEVICE)[:, None, None], torch.arange(s["kv_heads"], device=DEVICE)[None, :, None], rows[:, None, :])
    return _decode(kc[at], ks[at], s["bits"]), _decode(vc[at], vs[at], s["bits"])


def _write(s):
    rows = s["start"].long()[:, None] + torch.arange(s["count"], device=DEVICE)
    at = (torch.arange(s["b"], device=DEVICE)[:, None, None], torch.arange(s["kv_heads"], device=DEVICE)[None, :, None], rows[:, None, :])
    new = [t for x in (s["k"], s["v"]) for t in _encode(x.permute(1, 2, 0, 3).float().contiguous(), s["bits"])]
    s["cache"][0][at], s["cache"][1][at], s["cache"][2][at], s["cache"][3][at] = new


def _attend(s):
    tq, b, h, d = s["q"].shape
    hk, g, n = s["kv_heads"], h // s["kv_heads"], s["lengths"].long()
    w = s["window"] or s["longest"]
    span, sinks = min(s["longest"], w + tq - 1), min(s["sinks"] if s["window"] else 0, s["longest"])
    # the sinks, then the positions that the windows reach
    rows = torch.cat((torch.arange(sinks, device=DEVICE).expand(b, -1), n[:, None] - span + torch.arange(span, device=DEVICE)), 1)
    k, v = _rows(s, rows.clamp(0, s["cap"] - 1))
    qpos = (n[:, None] - tq + torch.arange(tq, device=DEVICE))[:, :, None]
    at, first = rows[:, None, :], qpos - w + 1
    slot = torch.arange(rows.shape[1], device=DEVICE) < sinks
    sees = torch.where(slot, at < torch.minimum(first, n[:, None, None]), (at >= first) & (at >= 0)) & (at <= qpos)
    q = s["q"].float().view(tq, b, hk, g, d).permute(1, 2, 3, 0, 4).reshape(b, hk, g * tq, d)
    p = (q @ k.transpose(-1, -2)).view(b, hk, g, tq, -1) * d ** -0.5
    p = p.masked_fill(~sees[:, None, None], -math.inf)
    top = p.amax(-1, keepdim=True)
    p = torch.exp(p - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, torch.ones_like(total), total)
    out = p.view(b, hk, g * tq, -1) @ v
    return [out.view(b, hk, g, tq, d).permute(3, 0, 1, 2, 4).reshape(tq, b, h, d).to(s["q"].dtype)]


# ----------------------------------------------------------------------------------------------------------- accounting
def _pairs(first, last, window, sinks):
    """Visible (query, key) pairs of the query positions first .. last - 1."""
    total, full = 0, lambda n: n * (n + 1) // 2       # positions 0 .. n - 1 see 1 .. n keys
    edge = window + min(sinks, 1 << 30)
    for a, sign in ((last, 1), (first, -1)):          # position i sees min(i + 1, window + sinks) keys
        a = max(a, 0)
        total += sign * (full(a) if a <= edge else full(edge) + (a - edge) * edge)
    return total


def work(case):
    """Every input read once, every output written once; products at two operations per multiply-add."""
    b, dim = case["b"], case["dim"]
    if case["kind"] == "window":
        t, h, hk = case["t"], case["heads"], case["kv_heads"]
        lens = _spread(t, b, case["ragged"])
        pairs = sum(_pairs(0, n, case["window"], case["sinks"]) for n in lens)
        live, rows = sum(lens) * dim * 2, t * b * dim * 2
        # queries, keys and values in, the output; in training its gradient in and three gradients out
        size = live * (h + 2 * hk) + rows * h
        if case["train"]:
            size += live * h + rows * (h + 2 * hk)
        return dict(bytes=size, flops=(14.0 if case["train"] else 4.0) * pairs * h * dim)
    held = dim * case["bits"] / 8 + dim / BLOCK
    if case["kind"] in ("write", "read"):
        rows = 2.0 * case["count"] * b * case["kv_heads"]
        return dict(bytes=rows * (held + dim * (4 if case["kind"] == "write" else 2)), flops=4.0 * rows * dim)
    lens = _spread(case["longest"], b)
    w = case["window"] or case["longest"]
    sinks = case["sinks"] if case["window"] else 0
    seen = sum(min(n, w + min(case["tq"], n) - 1 + min(sinks, max(0, n - w))) for n in lens)
    pairs = sum(_pairs(n - case["tq"], n, w, sinks) for n in lens)
    return dict(bytes=2.0 * seen * case["kv_heads"] * held + 4.0 * case["tq"] * b * case["heads"] * dim, flops=4.0 * pairs * case["heads"] * dim)


# ---------------------------------------------------------------------------------------------------------------- exact
_FOUR = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
_EIGHT = [(m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)) for e in range(16) for m in range(8)][:127]


def _exact_values(codes, scales, bits):
    magnitudes = torch.tensor(_FOUR if bits == 4 else _EIGHT + [math.nan], dtype=torch.float64, device=codes.device)
    table = torch.cat((magnitudes, -magnitudes))
    if bits == 4:
        pairs = torch.empty(*codes.shape, 2, dtype=torch.long, device=codes.device)
        pairs[..., 0], pairs[..., 1] = codes % 16, codes // 16
        codes = pairs.flatten(-2)
    return table[codes.long()] * torch.pow(2.0, scales.double() - 127.0).repeat_interleave(BLOCK, dim=-1)


def _exact_held(x, bits):
    """What a cache holds for x, by the nearest of the format's values."""
    values = torch.tensor(_FOUR if bits == 4 else _EIGHT, dtype=torch.float64, device=x.device)
    blocks = x.double().unflatten(-1, (-1, BLOCK))
    largest = blocks.abs().amax(-1, keepdim=True)
    limit = 7.0 if bits == 4 else 464.0
    e = torch.ceil(torch.log2(largest / limit))
    e = torch.where(largest > limit * torch.pow(2.0, e), e + 1, e)
    e = torch.where(largest <= limit * torch.pow(2.0, e - 1), e - 1, e)
    scale = torch.pow(2.0, torch.where(largest == 0, torch.zeros_like(e), e.clamp(-126, 127)))
    y = (blocks / scale).abs()
    below = (torch.searchsorted(values, y.contiguous(), right=True) - 1).clamp(max=len(values) - 2)
    lo, hi = values[below], values[below + 1]
    nearer = (y - lo > hi - y) | ((y - lo == hi - y) & (below % 2 == 1))
    return (torch.where(nearer, hi, lo) * torch.sign(blocks) * scale).flatten(-2)


def _exact_attention(q, k, v, sees):
    """q [h, n, d], k and v [hk, m, d], sees [n, m], all in 64 bits -> [h, n, d]; a row that sees nothing gives zeros."""
    g = q.shape[0] // k.shape[0]
    scores = q @ k.repeat_interleave(g, 0).transpose(1, 2) / math.sqrt(q.shape[2])
    p = torch.softmax(torch.where(sees, scores, scores.new_tensor(-1e300)), -1)
    return (p * sees) @ v.repeat_interleave(g, 0)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "write":
        return [_exact_held(s[n], case["bits"]) for n in "kv"]
    if case["kind"] == "read":
        kc, ks, vc, vs = (x[:, :, :case["count"]] for x in s["cache"])
        return [_exact_values(c, z, case["bits"]).permute(2, 0, 1, 3).contiguous() for c, z in ((kc, ks), (vc, vs))]
    if case["kind"] == "attend":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEVICE)
        for i, n in enumerate(s["lengths"].tolist()):
            kc, ks, vc, vs = (x[i, :, :n] for x in s["cache"])
            k, v = _exact_values(kc, ks, case["bits"]), _exact_values(vc, vs, case["bits"])
            pos = torch.arange(n - case["tq"], n, device=DEVICE)[:, None]
            out[:, i] = _exact_attention(s["q"][:, i].double().transpose(0, 1), k, v, _visible(pos, n, case["window"] or n, case["sinks"])).transpose(0, 1)
        return [out]
    q, k, v = (s[n].detach().double().requires_grad_(case["train"]) for n in "qkv")
    out = torch.zeros(q.shape, dtype=torch.float64, device=DEVICE)
    for i, n in enumerate(_spread(case["t"], case["b"], case["ragged"])):
        for a in range(0, n, 1024):
            z = min(n, a + 1024)
            sees = _visible(torch.arange(a, z, device=DEVICE)[:, None], z, case["window"], case["sinks"])
            part = _exact_attention(q[a:z, i].transpose(0, 1), k[:z, i].transpose(0, 1), v[:z, i].transpose(0, 1), sees).transpose(0, 1)
            if case["train"]:
                part.backward(s["dout"][a:z, i].double())
            out[a:z, i] = part.detach()
    return [out, q.grad, k.grad, v.grad] if case["train"] else [out]


def _visible(positions, n, window, sinks):
    keys = torch.arange(n, device=DEVICE)
    return (keys <= positions) & ((keys > positions - window) | (keys < sinks))
