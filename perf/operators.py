"""Operators of a long-context KV cache, measured: a cache of 8-bit floats as it
is written and read back, and the attention of single new tokens and of chunks
of them over such a cache, or over a 16-bit one, with a sliding window whose
first tokens stay visible.

Kinds of case
  write    the new tokens' K and V rows, quantised into their cache slots.
  read     cached rows, named by their slots, back as 16-bit K and V.
  decode   one new token per sequence against the sequence's visible context.
  prefill  a chunk of new tokens per sequence, already in the cache, against the
           visible context of each.

The quantised cache.  A row x of one token and kv head (head_size values) is held
as e4m3 codes c and one exponent byte b, and stands for the values c * 2^(b-127):
  z = x with its magnitudes held to 15/16 of the type's range, 61440 for float16
      and 15/16 * 2^128 for bfloat16, so that what the row stands for is finite;
  e = the least whole number with max|z| <= 448 * 2^e, at least -126;
  c = z / 2^e rounded to e4m3 (ties to even), b = e + 127.

The visible context.  A query at position p sees the keys j <= p with j < F or
j > p - W, for F first tokens and a window of W; W = 0 is the whole context.  In a
decode p is the sequence's last position.

`own` false computes them in elementary torch operations, in 32 bits; true calls the
framework.
"""
import functools
import math
import random
import sys
from pathlib import Path
from types import SimpleNamespace

import torch

own = False

DEV = "cuda"
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
TOP = {torch.float16: 61440.0, torch.bfloat16: 0.9375 * 2.0 ** 128}


def listed():
    """The fixed cases, smallest first inside a kind."""
    return [
        # The new tokens of a decode step: latency counts.
        dict(name="write-step", kind="write", tokens=32, kv=8, dim=128, dtype="bf16", block=16,
             layout="vllm", pad=0),
        # The chunk of a prefill step: four times 512 tokens, engine layout.
        dict(name="write-chunk", kind="write", tokens=2048, kv=8, dim=128, dtype="fp16", block=16,
             layout="kernel", pad=0),
        # A batch of long prompts, padded to a captured size (slots of -1), an odd
        # number of tokens.
        dict(name="write-prompts", kind="write", tokens=24573, kv=8, dim=128, dtype="bf16",
             block=16, layout="vllm", pad=259),
        # One conversation's cached rows, to be moved to another cache.
        dict(name="read-context", kind="read", tokens=2557, kv=8, dim=128, dtype="fp16", block=16,
             layout="vllm", pad=0),
        # The rows of a long shared prompt.
        dict(name="read-long", kind="read", tokens=65536, kv=8, dim=128, dtype="bf16", block=16,
             layout="kernel", pad=0),
        # A small model answering four short conversations: latency and launches.
        dict(name="decode-tiny-q8", kind="decode", q8=True, seqs=4, lo=16, hi=512, heads=14, kv=2,
             dim=64, dtype="fp16", block=16, layout="vllm", window=0, first=0),
        # The benchmark's headline over a quantised cache: 32 contexts of 8192.
        dict(name="decode-32x8k-q8", kind="decode", q8=True, seqs=32, lo=8192, hi=8192, heads=32,
             kv=8, dim=128, dtype="bf16", block=16, layout="kernel", window=0, first=0),
        # Long conversations of a model with a sliding window, 16-bit cache, a few of
        # them still shorter than the window; four first tokens stay visible.
        dict(name="decode-window", kind="decode", q8=False, seqs=27, lo=100, hi=32000, heads=32,
             kv=8, dim=128, dtype="fp16", block=16, layout="vllm", window=4096, first=4),
        # The same of a larger batch, its cache quantised.
        dict(name="decode-window-q8", kind="decode", q8=True, seqs=64, lo=4096, hi=32768, heads=32,
             kv=8, dim=128, dtype="bf16", block=16, layout="vllm", window=4096, first=4),
        # Short ragged chunks of a small model with a short window.
        dict(name="prefill-ragged-q8", kind="prefill", q8=True, seqs=7, prefix=150, lo=3, hi=77,
             heads=14, kv=2, dim=64, dtype="fp16", block=16, layout="vllm", window=128, first=4),
        # Chunked prefill over a quantised cache: four times 512 new over 2048.
        dict(name="prefill-chunk-q8", kind="prefill", q8=True, seqs=4, prefix=2048, lo=512, hi=512,
             heads=32, kv=8, dim=128, dtype="bf16", block=16, layout="vllm", window=0, first=0),
        # Two chunks of 2048 deep inside long documents, sliding window, 16-bit cache.
        dict(name="prefill-window", kind="prefill", q8=False, seqs=2, prefix=12000, lo=2048,
             hi=2048, heads=32, kv=8, dim=128, dtype="bf16", block=16, layout="kernel",
             window=4096, first=4),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    """One more case of the same ranges: every kind, type and layout, sizes over
    their logarithm, odd ones and short blocks among them."""
    kind = rng.choice(["write", "read", "decode", "decode", "prefill", "prefill"])
    heads, kv, dim = rng.choice([(14, 2, 64), (32, 8, 128), (28, 4, 128), (16, 16, 64), (64, 8, 64),
                                 (32, 32, 96), (16, 2, 128), (8, 4, 80), (4, 4, 32), (20, 1, 128)])
    c = dict(kind=kind, kv=kv, dim=dim, dtype=rng.choice(["fp16", "bf16"]),
             block=rng.choice([16, 16, 16, 32, 64, 8]), layout=rng.choice(["vllm", "kernel"]))
    if kind in ("write", "read"):
        most = min(65536 if kind == "read" else 24573, (1 << 26) // (kv * dim))
        c["tokens"] = _log(rng, 1, most)
        c["pad"] = rng.choice([0, c["tokens"] // 9])
        return c
    c.update(heads=heads, q8=rng.random() < 0.6)
    windowed = not c["q8"] or rng.random() < 0.5
    c["window"] = _log(rng, 16, 8192) if windowed else 0
    c["first"] = rng.choice([0, 1, 4, 16, 100]) if windowed else 0
    if kind == "decode":
        c["seqs"] = _log(rng, 1, 64)
        seen = (1 << 28) // (c["seqs"] * kv * dim)  # the headline's K values
        c["hi"] = _log(rng, 16, min(32768, seen))
        c["lo"] = rng.randint(1, c["hi"])
    else:
        c["seqs"] = _log(rng, 1, 16)
        c["hi"] = _log(rng, 2, max(2, 4096 // c["seqs"]))
        c["lo"] = rng.randint(1, c["hi"])
        sees = (1 << 36) // (c["seqs"] * c["hi"] * heads * dim * 2)
        c["prefix"] = _log(rng, 1, max(2, min(16000, sees)))
        if not windowed:
            c["prefix"] = min(c["prefix"], 8000)
    return c


# ------------------------------------------------------------------- inputs


def _two(e):
    """2^e in 32 bits, exactly, for -126 <= e <= 127."""
    return ((e + 127).to(torch.int32) << 23).view(torch.float32)


def _quantise(x):
    """(codes, exponent bytes) of the rows of x, by the definition above."""
    z = x.float().clamp(-TOP[x.dtype], TOP[x.dtype])
    top = z.abs().amax(-1)
    # log2 in 64 bits: a row whose largest value is 448 * 2^k is on a border.
    e = torch.ceil(torch.log2(top.double() / 448)).clamp(min=-126).to(torch.int32)
    codes = (z * _two(-e)[..., None]).to(torch.float8_e4m3fn)
    return codes, (e + 127).to(torch.uint8)


def _rows(c, shape, g):
    """K-like rows: normal values, some channels of a head several times larger."""
    chan = torch.exp(0.5 * torch.randn((c["kv"], c["dim"]), generator=g, device=DEV))
    if c["layout"] == "kernel" and len(shape) == 4:
        chan = chan[:, None]
    return (torch.randn(shape, generator=g, device=DEV) * chan).to(TYPES[c["dtype"]])


def _caches(c, blocks, g, q8, clean=False):
    """(key cache, value cache, their exponents or None): filled, or empty."""
    kv, d, bs = c["kv"], c["dim"], c["block"]
    shape = (blocks, kv, bs, d) if c["layout"] == "kernel" else (blocks, bs, kv, d)
    got = []
    for k in range(2):
        if clean:
            got.append((torch.zeros(shape, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn),
                        torch.zeros(shape[:-1], dtype=torch.uint8, device=DEV)))
            continue
        x = _rows(c, shape, g) if k == 0 else \
            torch.randn(shape, generator=g, device=DEV).to(TYPES[c["dtype"]])
        got.append(_quantise(x) if q8 else (x, None))
        del x
    (k, ke), (v, ve) = got
    return k, v, ke, ve


def _lens(lo, hi, n, g):
    return torch.randint(lo, hi + 1, (n,), generator=g, device=DEV).tolist()


def _chunks(c):
    """The sequences' new tokens: of the case, so that its output has one shape."""
    r = random.Random(c["lo"] * 65537 + c["hi"])
    return [r.randint(c["lo"], c["hi"]) for _ in range(c["seqs"])]


def prepare(case, seed):
    """What a serving program has in hand: caches, tables and lengths on the GPU, the
    lengths on the host too, the new rows or queries, and the output buffers."""
    c, t = case, TYPES[case["dtype"]]
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = SimpleNamespace(case=c)
    if c["kind"] in ("write", "read"):
        n = c["tokens"]
        blocks = -(-n // c["block"]) + 3
        s.slots = torch.randperm(blocks, generator=g, device=DEV)[:, None] * c["block"]
        s.slots = (s.slots + torch.arange(c["block"], device=DEV)).reshape(-1)[:n].contiguous()
        if c["pad"]:
            s.slots[n - c["pad"]:] = -1
        s.kc, s.vc, s.ke, s.ve = _caches(c, blocks, g, True, clean=c["kind"] == "write")
        if c["kind"] == "write":
            s.key = _rows(c, (n, c["kv"], c["dim"]), g)
            s.value = torch.randn((n, c["kv"], c["dim"]), generator=g, device=DEV).to(t)
        else:
            s.key = torch.empty((n, c["kv"], c["dim"]), dtype=t, device=DEV)
            s.value = torch.empty_like(s.key)
        return s
    if c["kind"] == "decode":
        s.lens = _lens(c["lo"], c["hi"], c["seqs"], g)
        new = [1] * c["seqs"]
    else:
        new = _chunks(c)
        s.lens = [c["prefix"] + n for n in new]
    need = [-(-n // c["block"]) for n in s.lens]
    blocks = sum(need) + 3
    perm = torch.randperm(blocks, generator=g, device=DEV).to(torch.int32)
    s.table = torch.full((c["seqs"], max(need)), -1, dtype=torch.int32, device=DEV)
    at = 0
    for i, n in enumerate(need):
        s.table[i, :n] = perm[at:at + n]
        at += n
    s.kc, s.vc, s.ke, s.ve = _caches(c, blocks, g, c["q8"])
    s.seq_lens = torch.tensor(s.lens, dtype=torch.int32, device=DEV)
    s.longest, s.scale, s.new = max(s.lens), c["dim"] ** -0.5, max(new)
    s.q = torch.randn((sum(new), c["heads"], c["dim"]), generator=g, device=DEV).to(t)
    s.out = torch.empty_like(s.q)
    starts = torch.tensor([0] + new, device=DEV).cumsum(0).to(torch.int32)
    s.starts = starts
    s.seq_of = torch.repeat_interleave(torch.arange(c["seqs"], device=DEV),
                                       torch.tensor(new, device=DEV)).to(torch.int32)
    t_in = torch.arange(sum(new), device=DEV) - starts[s.seq_of.long()]
    news = torch.tensor(new, device=DEV)
    s.positions = (s.seq_lens[s.seq_of.long()] - news[s.seq_of.long()] + t_in).to(torch.int32)
    return s


# --------------------------------------------------------------------- runs


@functools.cache
def _kernels():
    root = str(Path.cwd() / "vllm-apple_amd")
    if root not in sys.path:
        sys.path.insert(1, root)
    from vllm_apple_amd import kernels
    return kernels


def run(s):
    c = s.case
    if c["kind"] == "write":
        (_write_own if own else _write_plain)(s)
        return {"key": s.kc, "value": s.vc, "key_exps": s.ke, "value_exps": s.ve}
    if c["kind"] == "read":
        key, value = (_read_own if own else _read_plain)(s)
        return {"key": key, "value": value}
    return (_attend_own if own else _attend_plain)(s)


def _write_own(s):
    _kernels().kv_write_slots(s.key, s.value, s.kc, s.vc, s.slots, key_exps=s.ke, value_exps=s.ve,
                             layout=s.case["layout"])


def _read_own(s):
    return _kernels().kv_read_slots(s.kc, s.vc, s.ke, s.ve, s.slots, key=s.key, value=s.value,
                                   layout=s.case["layout"])


def _attend_own(s):
    c = s.case
    more = dict(scale=s.scale, layout=c["layout"], output=s.out, window=c["window"],
                first_tokens=c["first"], key_exps=s.ke, value_exps=s.ve, max_seq_len=s.longest)
    if c["kind"] == "decode":
        return _kernels().paged_decode(s.q, s.kc, s.vc, s.table, s.seq_lens, seq_lens_host=s.lens,
                                       **more)
    return _kernels().paged_prefill(s.q, s.kc, s.vc, s.table, s.seq_of, s.positions, **more)


def _put(cache, c, block, off, rows):
    if c["layout"] == "kernel":
        cache[block, :, off] = rows
    else:
        cache[block, off] = rows


def _write_plain(s):
    c = s.case
    real = s.slots[:c["tokens"] - c["pad"]]
    block, off = real // c["block"], real % c["block"]
    for x, codes, exps in ((s.key, s.kc, s.ke), (s.value, s.vc, s.ve)):
        q, e = _quantise(x[:real.numel()])
        _put(codes.view(torch.uint8), c, block, off, q.view(torch.uint8))
        _put(exps, c, block, off, e)


def _take(cache, exps, c, block, off):
    """The rows (block, off) of every kv head, [..., KV, D], in 32 bits."""
    raw = cache.view(torch.uint8) if exps is not None else cache
    x = raw[block, :, off] if c["layout"] == "kernel" else raw[block, off]
    if exps is None:
        return x.float()
    e = exps[block, :, off] if c["layout"] == "kernel" else exps[block, off]
    return x.view(torch.float8_e4m3fn).float() * _two(e.int() - 127)[..., None]


def _read_plain(s):
    c = s.case
    ok = s.slots >= 0
    real = s.slots.clamp(min=0)
    block, off = real // c["block"], real % c["block"]
    return tuple(torch.where(ok[:, None, None], _take(x, e, c, block, off), 0.0).to(s.key.dtype)
                 for x, e in ((s.kc, s.ke), (s.vc, s.ve)))


def _visible(s):
    """(positions [S, K], which of them a sequence has): the first tokens, and the rest
    from the oldest key that a window still shows."""
    c = s.case
    rest = min(s.longest, c["window"] + s.new - 1 if c["window"] else s.longest)
    low = (s.seq_lens.long() - rest).clamp(min=0)[:, None]
    pos = low + torch.arange(rest, device=DEV)
    fine = pos < s.seq_lens[:, None]
    if c["window"] and c["first"]:
        head = torch.arange(c["first"], device=DEV).expand(c["seqs"], -1)
        pos = torch.cat([head, pos], 1)
        fine = torch.cat([(head < low), fine], 1)
    return pos, fine


def _attend_plain(s):
    """Batched over the sequences, queries padded to the longest chunk."""
    c = s.case
    n, h, kv, d = c["seqs"], c["heads"], c["kv"], c["dim"]
    pos, fine = _visible(s)
    at = pos.clamp(max=s.table.shape[1] * c["block"] - 1)
    block = torch.gather(s.table.long(), 1, at // c["block"]).clamp(min=0)
    k, v = (_take(x, e, c, block, at % c["block"]).transpose(1, 2)  # [S, KV, K, D]
            for x, e in ((s.kc, s.ke), (s.vc, s.ve)))
    row = s.starts[:-1, None].long() + torch.arange(s.new, device=DEV)
    real = row < s.starts[1:, None]
    row = row.clamp(max=s.q.shape[0] - 1)
    p = s.positions[row]  # [S, N]
    q = s.q[row].float().view(n, s.new, kv, h // kv, d).permute(0, 2, 1, 3, 4)
    x = q.reshape(n, kv, -1, d) @ k.transpose(2, 3) * s.scale
    x = x.view(n, kv, s.new, h // kv, -1)
    sees = fine[:, None] & (pos[:, None] <= p[:, :, None])
    if c["window"]:
        sees &= (pos[:, None] < c["first"]) | (pos[:, None] > p[:, :, None] - c["window"])
    x = torch.where(sees[:, None, :, None], x, -math.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True))
    total = x.sum(-1, keepdim=True)
    o = x.view(n, kv, -1, x.shape[-1]) @ v
    o = o.view(n, kv, s.new, h // kv, d) / total
    o = o.permute(0, 2, 1, 3, 4).reshape(n, s.new, h, d)
    s.out[row[real]] = o[real].to(s.out.dtype)
    return s.out


# --------------------------------------------------------------------- work


def work(case):
    """Rows that a call sees, once each, with their exponents; the new rows, queries
    and results.  The lengths are the ranges' means."""
    c = case
    row = c["kv"] * c["dim"]
    if c["kind"] in ("write", "read"):
        n = c["tokens"] - c["pad"]
        wide, narrow = 2 * 2 * row * n, 2 * (row + c["kv"]) * n
        if c["kind"] == "read":
            wide = 2 * 2 * row * c["tokens"]  # padded rows are cleared
        return {"bytes": wide + narrow + 8 * c["tokens"], "flops": 0}
    held = 2 * (row + c["kv"]) if c["q8"] else 2 * 2 * row
    mean = (c["lo"] + c["hi"]) / 2
    new = 1 if c["kind"] == "decode" else mean
    if c["kind"] == "decode":
        sees = mean
        if c["window"]:  # the mean of min(L, F + W) over lo..hi
            top, span = c["window"] + c["first"], c["hi"] - c["lo"] + 1
            under = min(max(top - c["lo"], 0), span)
            sees = (under * (c["lo"] + c["lo"] + under - 1) / 2 + (span - under) * top) / span
        rows = pairs = c["seqs"] * sees
    else:
        longest = c["prefix"] + new
        pairs = new * (c["prefix"] + (new + 1) / 2)
        rows = longest
        if c["window"]:
            top = c["window"] + c["first"]
            whole = min(new, max(0, top - c["prefix"]))  # queries that see all before them
            pairs = whole * (c["prefix"] + (whole + 1) / 2) + (new - whole) * top
            rows = min(longest, top + new - 1)
        rows, pairs = c["seqs"] * rows, c["seqs"] * pairs
    q = c["seqs"] * new * c["heads"] * c["dim"] * 2
    return {"bytes": rows * held + 2 * q + rows / c["block"] * 4,
            "flops": pairs * c["heads"] * c["dim"] * 4}


# -------------------------------------------------------------------- exact


def _power(e):
    """2^e in 64 bits, exactly."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _e4m3(x):
    """x in 64 bits, rounded to the nearest e4m3 value, ties to even."""
    _, e = torch.frexp(x)  # |x| in [2^(e-1), 2^e)
    step = _power((e - 1).clamp(min=-6) - 3)
    return torch.round(x / step) * step


def _held(x):
    """(codes, exponent bytes) that the definition gives for rows in 64 bits."""
    z = x.double().clamp(-TOP[x.dtype], TOP[x.dtype])
    m, e = torch.frexp(z.abs().amax(-1))  # max = m 2^e, m in [1/2, 1); 448 = 7/8 2^9
    e = torch.where(m == 0, -126, torch.where(m <= 0.875, e - 9, e - 8).clamp(min=-126))
    return _e4m3(z * _power(-e)[..., None]), e + 127


def _values(cache, exps):
    if exps is None:
        return cache.double()
    return cache.to(torch.float64) * _power(exps.long() - 127)[..., None]


def exact(case, seed):
    """One sequence and kv head after another, in 64 bits."""
    c, s = case, prepare(case, seed)
    if c["kind"] == "write":
        got = {}
        for name, x, cache in (("key", s.key, s.kc), ("value", s.value, s.vc)):
            codes, exps = _held(x)
            full = torch.zeros(cache.shape, dtype=torch.float64, device=DEV)
            bytes_ = torch.zeros(cache.shape[:-1], dtype=torch.uint8, device=DEV)
            if c["layout"] == "kernel":
                full, bytes_ = full.transpose(1, 2), bytes_.transpose(1, 2)
            keep = s.slots >= 0
            at = s.slots[keep]
            full[at // c["block"], at % c["block"]] = codes[keep]
            bytes_[at // c["block"], at % c["block"]] = exps[keep].to(torch.uint8)
            if c["layout"] == "kernel":
                full, bytes_ = full.transpose(1, 2), bytes_.transpose(1, 2)
            got[name], got[name + "_exps"] = full.contiguous(), bytes_.contiguous()
        return got
    token_first = (lambda x: x.transpose(1, 2)) if c["layout"] == "kernel" else (lambda x: x)
    if c["kind"] == "read":
        got = {}
        for name, cache, exps in (("key", s.kc, s.ke), ("value", s.vc, s.ve)):
            rows = token_first(_values(cache, exps)).reshape(-1, c["kv"], c["dim"])
            got[name] = rows[s.slots.clamp(min=0)] * (s.slots >= 0)[:, None, None]
        return got
    out = torch.zeros(s.q.shape, dtype=torch.float64, device=DEV)
    group = c["heads"] // c["kv"]
    start = s.starts.tolist()
    for i, length in enumerate(s.lens):
        rows = s.table[i, :-(-length // c["block"])].long()
        p = s.positions[start[i]:start[i + 1]].double()[:, None]
        j = torch.arange(length, device=DEV, dtype=torch.float64)[None]
        sees = j <= p
        if c["window"]:
            sees = sees & ((j < c["first"]) | (p - j < c["window"]))
        seen = sees.any(0)
        sees = sees[:, seen]
        k, v = (token_first(_values(x[rows], None if e is None else e[rows]))
                .reshape(-1, c["kv"], c["dim"])[:length][seen]
                for x, e in ((s.kc, s.ke), (s.vc, s.ve)))
        for head in range(c["heads"]):
            q = s.q[start[i]:start[i + 1], head].double()
            x = (q @ k[:, head // group].T) * s.scale
            w = torch.softmax(x.masked_fill(~sees, -math.inf), -1)
            out[start[i]:start[i + 1], head] = w @ v[:, head // group]
    return out
