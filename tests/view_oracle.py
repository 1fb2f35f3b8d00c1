"""Plain 64-bit forms of the quantised cache and of attention over a cache view, and
the tolerances that follow from the kernels' roundings."""
from __future__ import annotations

import math

import torch

TOP = {torch.float16: 61440.0, torch.bfloat16: 0.9375 * 2.0 ** 128}
UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}  # half a step, relative
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def two(e):
    """2^e in 64 bits, exactly."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def e4m3(x):
    """x (64 bits) rounded to the nearest e4m3 value, ties to even; NaN stays."""
    _, e = torch.frexp(torch.nan_to_num(x))
    step = two((e - 1).clamp(min=-6) - 3)
    return torch.round(x / step) * step


def quantise(x):
    """(codes in 64 bits, exponent bytes) of rows x (fp16 or bf16)."""
    z = x.double().clamp(-TOP[x.dtype], TOP[x.dtype])
    m, e = torch.frexp(torch.nan_to_num(z).abs().amax(-1))  # m in [1/2, 1)
    e = torch.where(m == 0, -126, torch.where(m <= 0.875, e - 9, e - 8).clamp(min=-126))
    return e4m3(z * two(-e)[..., None]), (e + 127).to(torch.uint8)


def values(codes, exps):
    """What a quantised cache stands for, in 64 bits."""
    return codes.double() * two(exps.int() - 127)[..., None]


def rows_of(cache, layout):
    """[num_blocks, block_size, KV, ...] of a cache or its exponents."""
    return cache.transpose(1, 2) if layout == "kernel" else cache


class Case:
    """Sequences in shuffled blocks of a pool with spare ones, seen from their last
    new[s] positions (1 each: a decode)."""

    def __init__(self, lens, H, KV, D, *, dtype="bf16", q8=True, layout="kernel", bs=16, window=0,
                 first=0, new=None, seed=0, spread=1.0):
        g = torch.Generator().manual_seed(seed)
        if not q8 and not window:
            first = max(first, 1)  # the whole context, still by the view's kernels
        self.H, self.KV, self.D, self.bs, self.layout = H, KV, D, bs, layout
        self.window, self.first, self.lens = window, first, list(lens)
        self.dtype, self.q8, self.scale = DTYPES[dtype], q8, D ** -0.5
        self.new = [1] * len(lens) if new is None else list(new)
        need = [-(-n // bs) for n in lens]
        nb = sum(need) + 3
        shape = (nb, KV, bs, D) if layout == "kernel" else (nb, bs, KV, D)
        raw = [(spread * torch.randn(shape, generator=g)).to(self.dtype) for _ in range(2)]
        # The pool's first block stays unused: an unread entry must not stand for it.
        perm = (1 + torch.randperm(nb - 1, generator=g)).to(torch.int32)
        self.table = torch.full((len(lens), max(max(need), 1)), -1, dtype=torch.int32)
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = perm[at:at + n]
            at += n
        self.seq_lens = torch.tensor(self.lens, dtype=torch.int32)
        T = sum(self.new)
        self.q = torch.randn(T, H, D, generator=g).to(self.dtype)
        self.tok, pos = [], []
        for s, (n, k) in enumerate(zip(self.lens, self.new)):
            self.tok += [s] * k
            pos += range(n - k, n)
        self.tok = torch.tensor(self.tok, dtype=torch.int32)
        self.pos = torch.tensor(pos, dtype=torch.int32)
        if q8:
            (kc, self.ke), (vc, self.ve) = map(quantise, raw)
            self.kc, self.vc = (c.float().to(torch.float8_e4m3fn) for c in (kc, vc))
        else:
            (self.kc, self.vc), self.ke, self.ve = raw, None, None

    def cached(self, s):
        """(K, V) [L, KV, D] of sequence s in 64 bits."""
        rows = self.table[s, :-(-self.lens[s] // self.bs)].long()
        ok = (rows >= 0) & (rows < self.kc.shape[0])
        got = []
        for c, e in ((self.kc, self.ke), (self.vc, self.ve)):
            c = rows_of(c, self.layout)[rows * ok]
            x = values(c, rows_of(e, self.layout)[rows * ok]) if self.q8 else c.double()
            got.append(x.reshape(-1, self.KV, self.D)[:self.lens[s]])
        return got

    def sees(self, s, p):
        """[queries at p, L]: which keys of sequence s they see."""
        j = torch.arange(self.lens[s])[None]
        p = p[:, None]
        m = j <= p
        if self.window:
            m &= (j < self.first) | (j > p - self.window)
        rows = self.table[s, :-(-self.lens[s] // self.bs)].long()
        ok = ((rows >= 0) & (rows < self.kc.shape[0])).repeat_interleave(self.bs)[:self.lens[s]]
        return m & ok[None]

    def attend(self, prefill):
        """(reference, tolerance) [T, H, D], by the formula in 64 bits."""
        out = torch.zeros(self.q.shape, dtype=torch.float64)
        tol = torch.zeros_like(out)
        for s in range(len(self.lens)):
            if self.lens[s] <= 0:
                continue
            mine = (self.tok == s).nonzero()[:, 0]
            if not len(mine):
                continue
            k, v = self.cached(s)
            m = self.sees(s, self.pos[mine].long())
            k, v = (torch.where(m.any(0)[:, None, None], x, 0.0) for x in (k, v))
            for h in range(self.H):
                kv = h // (self.H // self.KV)
                q = self.q[mine, h].double()
                x = (q @ k[:, kv].T * self.scale).masked_fill(~m, -math.inf)
                some = m.any(1)
                w = torch.zeros_like(x)
                w[some] = torch.softmax(x[some], -1)
                a = (q.abs() @ k[:, kv].abs().T * self.scale).masked_fill(~m, 0).amax(1)
                out[mine, h] = w @ v[:, kv]
                tol[mine, h] = self.tolerance(out[mine, h], w @ v[:, kv].abs(), a, q,
                                              v[:, kv].abs().max(), m.sum(1), prefill)
        return out, tol

    def tolerance(self, ref, mass, a, q, vmax, n, prefill):
        """How far the kernels' roundings can put an output from ref.

        mass = sum w |v|.  The result is rounded once to its type (unit u, 2^-25 below
        fp16's normals).  A weight is off, relatively, by the fp32 error of its
        score (D + 8 roundings of terms whose magnitudes sum to a nats), the error of
        exp2 (2^-22) and the rounding of P: the decode's pair of 16-bit values and
        the prefill's bf16 pair are good to u^2, its single fp16 value to 2^-11, and
        below fp16's normals to 2^-25 absolutely, for each of n keys of magnitude
        up to vmax (a quantised V, held relative to its group's exponent: twice
        that).  Numerator and normaliser each take it; the fp32 sums over n keys add n
        roundings.  fp16 K and V below the normals are off by 2^-25 each."""
        u = UNIT[self.dtype]
        fp16_p = prefill and (self.q8 or self.dtype == torch.float16)
        score = (self.D + 8) * 2.0 ** -24 * a
        if self.dtype == torch.float16:
            score = score + 2.0 ** -25 * self.scale * q.abs().sum(1)
        rel = score + 2.0 ** -22 + (2.0 ** -11 if fp16_p else u * u) + (n + 8) * 2.0 ** -24
        tiny = n * 2.0 ** -25 * 2 * vmax * (1 if fp16_p else 2.0 ** -10)
        if self.dtype == torch.float16:
            tiny = tiny + 2.0 ** -24
        return (u * ref.abs() + (rel[:, None] * (mass + ref.abs()) + tiny[:, None]) * (1 + u))

    def cuda(self):
        """The operands on the GPU, as keyword arguments of the wrappers."""
        return dict(query=self.q.cuda(), key_cache=self.kc.cuda(), value_cache=self.vc.cuda(),
                    block_table=self.table.cuda(), scale=self.scale, layout=self.layout,
                    window=self.window, first_tokens=self.first,
                    key_exps=self.ke.cuda() if self.q8 else None,
                    value_exps=self.ve.cuda() if self.q8 else None)

    def poison(self):
        """NaN in every cached row that no query sees, and table entries that name no
        block where a whole block is unseen."""
        used = torch.zeros(rows_of(self.kc, self.layout).shape[:2], dtype=torch.bool)
        for s in range(len(self.lens)):
            mine = (self.tok == s).nonzero()[:, 0]
            seen = self.sees(s, self.pos[mine].long()).any(0) if self.lens[s] > 0 else None
            for b in range(self.table.shape[1]):
                e = int(self.table[s, b])
                part = seen[b * self.bs:(b + 1) * self.bs] if seen is not None else []
                if e < 0 or not len(part) or not bool(part.any()):
                    self.table[s, b] = [-7, 1 << 30, -1][b % 3]
                else:
                    used[e, :len(part)] |= part
        for c, e in ((self.kc, self.ke), (self.vc, self.ve)):
            raw = rows_of(c.view(torch.uint8) if self.q8 else c.view(torch.int16), self.layout)
            raw[~used] = 0x7F if self.q8 else 0x7FFF
            if self.q8:
                rows_of(e, self.layout)[~used] = 255
        return self


def check(got, ref, tol, what=""):
    got = got.detach().double().cpu()
    assert got.shape == ref.shape
    assert torch.isfinite(got).all(), f"{what}: {int((~torch.isfinite(got)).sum())} not finite"
    over = (got - ref).abs() - tol
    if over.numel() and over.max() > 0:
        i = int(over.argmax())
        raise AssertionError(f"{what}: {int((over > 0).sum())} of {over.numel()} off; worst "
                             f"{got.flatten()[i]} for {ref.flatten()[i]}, tolerance "
                             f"{tol.flatten()[i]}")
