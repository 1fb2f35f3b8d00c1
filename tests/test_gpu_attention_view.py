"""Decode and chunked prefill over quantised caches and with sliding windows, against
the formula in 64 bits."""
import pytest
import torch

from helpers import canaried, tail_ok
from view_oracle import Case, check, rows_of

pytestmark = pytest.mark.gpu


def _decode(c, **kw):
    from vllm_apple_amd import kernels

    args = dict(max_seq_len=max(max(c.lens), 1))
    args.update(kw)
    return kernels.paged_decode(seq_lens=c.seq_lens.cuda(), **c.cuda(), **args)


def _prefill(c, **kw):
    from vllm_apple_amd import kernels

    return kernels.paged_prefill(token_to_seq=c.tok.cuda(), positions=c.pos.cuda(), **c.cuda(),
                                 **kw)


# Lengths of one token, of whole tiles and beside them, of windows that begin and end
# inside tiles and blocks, of windows longer than the context, of first tokens that
# meet the window.
LENS = [1, 2, 16, 17, 31, 32, 33, 64, 65, 100, 257, 700]
VIEWS = [(0, 0), (1, 0), (16, 4), (33, 1), (100, 16), (64, 70), (600, 100), (5000, 4)]


@pytest.mark.parametrize("window,first", VIEWS)
@pytest.mark.parametrize("q8,dtype", [(True, "bf16"), (True, "fp16"), (False, "bf16"),
                                      (False, "fp16")])
def test_decode_windows(gpu, q8, dtype, window, first):
    c = Case(LENS, 8, 2, 128, dtype=dtype, q8=q8, window=window, first=first, seed=1).poison()
    ref, tol = c.attend(False)
    for part in (0, 128, 256, -1):
        check(_decode(c, partition_size=part), ref, tol, f"partition {part}")
    check(_decode(c, seq_lens_host=c.lens), ref, tol, "host lengths")


SHAPES = [  # H, KV, D, block size, layout
    (14, 2, 64, 16, "vllm"), (4, 4, 32, 16, "kernel"), (6, 2, 96, 32, "vllm"),
    (20, 1, 128, 16, "kernel"), (32, 1, 64, 64, "vllm"), (4, 2, 80, 16, "vllm"),
    (3, 1, 48, 8, "kernel"), (8, 4, 112, 5, "vllm"), (5, 5, 16, 1, "kernel"),
    (8, 2, 128, 24, "vllm"), (2, 1, 64, 100, "kernel"),
]


@pytest.mark.parametrize("H,KV,D,bs,layout", SHAPES)
@pytest.mark.parametrize("q8,dtype", [(True, "bf16"), (True, "fp16"), (False, "bf16"),
                                      (False, "fp16")])
def test_decode_shapes(gpu, q8, dtype, H, KV, D, bs, layout):
    for window, first in ((0, 0), (70, 5)):
        c = Case([1, 15, 40, 130, 301], H, KV, D, dtype=dtype, q8=q8, layout=layout, bs=bs,
                 window=window, first=first, seed=D + bs).poison()
        ref, tol = c.attend(False)
        for part in (0, 128, -1):
            check(_decode(c, partition_size=part), ref, tol, f"partition {part}")


@pytest.mark.parametrize("D", [8, 24, 40, 72, 104])
def test_sixteen_bit_head_sizes(gpu, D):
    """Multiples of 8 that no multiple of 16 is: 16-bit caches take them."""
    c = Case([1, 50, 200], 4, 2, D, q8=False, dtype="fp16", window=60, first=3).poison()
    ref, tol = c.attend(False)
    check(_decode(c), ref, tol)
    p = Case([20, 50, 200], 4, 2, D, q8=False, dtype="bf16", window=60, first=3, new=[20, 3, 40])
    check(_prefill(p.poison()), *p.attend(True))


def test_decode_empty_rows_and_missing_blocks(gpu):
    """Sequences without tokens give zeros; a key in a missing block is not seen, and a
    sequence that sees none gives zeros; rows behind the last sequence stay."""
    c = Case([0, 40, 100, 5, 70], 8, 2, 64, dtype="fp16", window=30, first=2, layout="vllm")
    c.table[1] = -1
    c.table[2, 5] = 10 ** 6  # inside the window
    c.seq_lens[3] = c.lens[3] = 0
    ref, tol = c.attend(False)
    assert bool((ref[[0, 1, 3]] == 0).all())
    for part in (0, 128, -1):
        out = torch.full((7, 8, 64), 7.0).half().cuda()
        q = torch.cat([c.q, c.q[:2]]).cuda()
        args = {**c.cuda(), "query": q}
        from vllm_apple_amd import kernels
        kernels.paged_decode(seq_lens=c.seq_lens.cuda(), max_seq_len=100, output=out,
                             partition_size=part, **args)
        check(out[:5], ref, tol, f"partition {part}")
        assert bool((out[5:] == 7).all())


@pytest.mark.parametrize("q8", [True, False])
def test_decode_long_context(gpu, q8):
    """A context of several thousand tokens next to short ones, every split of it."""
    c = Case([5000, 3, 1024, 2049], 8, 2, 64, dtype="bf16", q8=q8, layout="vllm", seed=3,
             window=0 if q8 else 4000, first=0 if q8 else 40).poison()
    ref, tol = c.attend(False)
    for part in (0, 128, 512, 2048, -1):
        check(_decode(c, partition_size=part), ref, tol, f"partition {part}")
    # A bound below the lengths only sizes the split: the last piece takes the rest.
    check(_decode(c, partition_size=128, max_seq_len=300), ref, tol, "short bound")


CHUNKS = [  # context lengths, new tokens of each
    ([1], [1]), ([40], [40]), ([300, 17, 90], [45, 17, 1]), ([129, 64, 65, 700], [129, 1, 65, 33]),
]


@pytest.mark.parametrize("window,first", VIEWS)
@pytest.mark.parametrize("q8,dtype", [(True, "bf16"), (True, "fp16"), (False, "bf16"),
                                      (False, "fp16")])
def test_prefill_windows(gpu, q8, dtype, window, first):
    for lens, new in CHUNKS:
        c = Case(lens, 8, 2, 128, dtype=dtype, q8=q8, window=window, first=first, new=new, seed=2)
        check(_prefill(c.poison()), *c.attend(True), f"{lens} {new}")


@pytest.mark.parametrize("H,KV,D,bs,layout", SHAPES)
@pytest.mark.parametrize("q8,dtype", [(True, "bf16"), (True, "fp16"), (False, "bf16"),
                                      (False, "fp16")])
def test_prefill_shapes(gpu, q8, dtype, H, KV, D, bs, layout):
    for window, first in ((0, 0), (70, 5)):
        c = Case([200, 33, 131], H, KV, D, dtype=dtype, q8=q8, layout=layout, bs=bs,
                 window=window, first=first, new=[37, 33, 2], seed=D + bs)
        check(_prefill(c.poison()), *c.attend(True))


@pytest.mark.parametrize("q8", [True, False])
def test_prefill_split_and_whole(gpu, q8):
    """Few rows over a long context, whose keys are split, and many, whose are not: a
    row's result is the same formula's either way."""
    few = Case([3000], 8, 2, 64, dtype="bf16", q8=q8, new=[3], layout="vllm",
               window=0 if q8 else 2500, first=9)
    check(_prefill(few.poison()), *few.attend(True))
    many = Case([700] * 8, 32, 8, 64, dtype="fp16", q8=q8, new=[600] * 8, window=130, first=9)
    got = _prefill(many)
    pick = torch.arange(0, 4800, 97)
    ref, tol = _some(many, pick)
    check(got[pick.cuda()], ref, tol)


def _some(c, pick):
    """The reference at some of the query rows."""
    c.q, c.tok, c.pos = c.q[pick], c.tok[pick], c.pos[pick]
    return c.attend(True)


def test_prefill_rows_left_alone(gpu):
    """Rows of no sequence, of a negative position or of a context past the table stay
    as they were, in any token order; keys in a missing block are not seen; nothing
    is written behind the output."""
    from vllm_apple_amd import kernels

    for lens, new in (([90, 200, 40], [30, 100, 40]), ([2000, 30], [8, 4])):
        c = Case(lens, 4, 2, 64, dtype="bf16", new=new, seed=9, layout="vllm", window=50, first=6)
        g = torch.Generator().manual_seed(0)
        order = torch.randperm(sum(new), generator=g)
        c.q, c.tok, c.pos = c.q[order], c.tok[order], c.pos[order]
        c.table[0, (lens[0] - 20) // 16] = -1
        ref, tol = c.attend(True)
        tok, pos = c.tok.clone(), c.pos.clone()
        n = len(tok)
        tok[1], tok[2], pos[3], pos[4] = -1, len(lens), -1, c.table.shape[1] * 16
        buf, out = canaried(torch.full((n, 4, 64), 7.0).bfloat16())
        kernels.paged_prefill(token_to_seq=tok.cuda(), positions=pos.cuda(), output=out, **c.cuda())
        left = torch.zeros(n, dtype=torch.bool)
        left[1:5] = True
        assert bool((out[left.cuda()] == 7).all())
        check(out[~left.cuda()], ref[~left], tol[~left])
        assert tail_ok(buf)


@pytest.mark.parametrize("prefill", [False, True])
def test_values_far_apart(gpu, prefill):
    """bf16 rows of magnitudes from 2^-30 to 2^30, past fp16's range, quantised: the V
    groups' exponents differ widely."""
    c = Case([300, 40], 4, 2, 64, dtype="bf16", new=[20, 20] if prefill else None, seed=4)
    g = torch.Generator().manual_seed(5)
    lift = torch.randint(-30, 31, c.ve.shape, generator=g)
    c.ve = (c.ve.int() + lift).to(torch.uint8)
    ref, tol = c.attend(prefill)
    check(_prefill(c) if prefill else _decode(c), ref, tol)


def test_no_queries(gpu):
    from vllm_apple_amd import kernels

    c = Case([20], 4, 2, 64)
    args = {**c.cuda(), "query": c.q[:0].cuda()}
    none = torch.zeros(0, dtype=torch.int32).cuda()
    assert kernels.paged_prefill(token_to_seq=none, positions=none, **args).shape == (0, 4, 64)
    args["block_table"] = args["block_table"][:0]
    assert kernels.paged_decode(seq_lens=none, max_seq_len=1, **args).shape == (0, 4, 64)


@pytest.mark.parametrize("window,first", [(0, 0), (20, 3)])
@pytest.mark.parametrize("new", [[40, 30], [3, 2]])
@pytest.mark.parametrize("q8,dtype", [(True, "bf16"), (False, "bf16"), (False, "fp16")])
def test_infinities_that_some_rows_see(gpu, q8, dtype, new, window, first):
    """Infinities and NaN in rows that part of a chunk sees: rows that do not see them
    are what they are without, the others have them where the formula has."""
    lens = [120, 1500]
    c = Case(lens, 4, 2, 64, dtype=dtype, q8=q8, new=new, window=window, first=first, seed=6,
             layout="vllm")
    ref, tol = c.attend(True)

    def row(cache, s, j):
        return rows_of(cache, c.layout)[c.table[s, j // 16], j % 16]

    bad = {0: (lens[0] - 2, 1), 1: (lens[1] - 1, 0)}  # position and kv head
    marks = [(3, "nan")] if q8 else [(3, "nan"), (7, "inf"), (40, "-inf")]
    for s, (j, kv) in bad.items():
        for d, x in marks:
            if q8:
                row(c.vc.view(torch.uint8), s, j)[kv, d] = 0x7F
            else:
                row(c.vc, s, j)[kv, d] = float(x)
    got = _prefill(c).double().cpu()
    hit = torch.zeros(ref.shape, dtype=torch.bool)
    for s, (j, kv) in bad.items():
        rows = (c.tok == s) & (c.pos >= j)
        for d, x in marks:
            for h in (2 * kv, 2 * kv + 1):
                hit[rows, h, d] = True
                want = torch.full((int(rows.sum()),), float(x), dtype=torch.float64)
                assert torch.equal(got[rows, h, d].nan_to_num(nan=5.0), want.nan_to_num(nan=5.0))
    assert bool(hit.any()) and not bool(hit.all())
    check(torch.where(hit, 0.0, got), torch.where(hit, 0.0, ref), tol)
    # A NaN key: every value of the rows that see it, and nothing else.
    c = Case(lens, 4, 2, 64, dtype=dtype, q8=q8, new=new, window=window, first=first, seed=6,
             layout="vllm")
    for s, (j, kv) in bad.items():
        if q8:
            row(c.kc.view(torch.uint8), s, j)[kv, 5] = 0x7F
        else:
            row(c.kc, s, j)[kv, 5] = float("nan")
    got = _prefill(c).double().cpu()
    hit = torch.zeros(ref.shape, dtype=torch.bool)
    for s, (j, kv) in bad.items():
        hit[(c.tok == s) & (c.pos >= j), 2 * kv:2 * kv + 2] = True
    assert bool(torch.isnan(got[hit]).all())
    check(torch.where(hit, 0.0, got), torch.where(hit, 0.0, ref), tol)
