"""The quantised KV write and its read back, against the definition in 64 bits."""
import pytest
import torch

from helpers import canaried, tail_ok
from view_oracle import DTYPES, quantise, rows_of, values

pytestmark = pytest.mark.gpu


def _empty(nb, kv, bs, d, layout):
    shape = (nb, kv, bs, d) if layout == "kernel" else (nb, bs, kv, d)
    cache = torch.full(shape, 0x2A, dtype=torch.uint8).cuda()
    return cache.view(torch.float8_e4m3fn), torch.full(shape[:-1], 9, dtype=torch.uint8).cuda()


def _compare(cache, exps, layout, bs, slots, x):
    """The named rows hold x's quantisation, every other byte what it held."""
    codes, want_e = quantise(x.cpu())
    c = rows_of(cache.view(torch.uint8).cpu(), layout).reshape(-1, x.shape[1], x.shape[2])
    e = rows_of(exps.cpu(), layout).reshape(-1, x.shape[1])
    real = (slots >= 0) & (slots < c.shape[0])
    at = slots[real].long()
    assert torch.equal(e[at], want_e[real])
    got = c[at].contiguous().view(torch.float8_e4m3fn).double()
    want = codes[real]
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    ok = ~torch.isnan(want)
    assert torch.equal(got[ok], want[ok])
    assert torch.equal(torch.signbit(got[ok]), torch.signbit(want[ok]))
    rest = torch.ones(c.shape[0], dtype=torch.bool)
    rest[at] = False
    assert bool((c[rest] == 0x2A).all()) and bool((e[rest] == 9).all())


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("layout", ["kernel", "vllm"])
@pytest.mark.parametrize("kv,d,bs,n", [(8, 128, 16, 300), (2, 64, 16, 1), (4, 96, 8, 77),
                                       (1, 32, 7, 33), (3, 80, 16, 50), (2, 8, 1, 19),
                                       (2, 100, 16, 31), (1, 136, 16, 9), (5, 1, 4, 6)])
def test_write_slots(gpu, dtype, layout, kv, d, bs, n):
    """Every row size, the ones without 16-byte pieces among them; padding and slots
    past the cache are skipped."""
    from vllm_apple_amd import kernels

    g = torch.Generator().manual_seed(n)
    nb = -(-n // bs) + 2
    key, value = (torch.randn(n, kv, d, generator=g).to(DTYPES[dtype]).cuda() for _ in range(2))
    slots = torch.randperm(nb * bs, generator=g)[:n]
    slots[::5] = -1
    if n > 6:
        slots[6] = nb * bs + 3
    for index in (torch.int64, torch.int32):
        kc, ke = _empty(nb, kv, bs, d, layout)
        vc, ve = _empty(nb, kv, bs, d, layout)
        kernels.kv_write_slots(key, value, kc, vc, slots.to(index).cuda(), key_exps=ke,
                               value_exps=ve, layout=layout)
        _compare(kc, ke, layout, bs, slots, key)
        _compare(vc, ve, layout, bs, slots, value)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_write_every_value(gpu, dtype):
    """All 65536 bit patterns: alone in a row (so that each sets its row's exponent),
    and in shared rows whose exponent another value sets.  Infinities, NaN, zeros and
    subnormal numbers among them."""
    from vllm_apple_amd import kernels

    bits = torch.arange(-32768, 32768, dtype=torch.int32).to(torch.int16).view(DTYPES[dtype])
    alone = torch.zeros(65536, 1, 8).to(DTYPES[dtype])
    alone[:, 0, 3] = bits
    g = torch.Generator().manual_seed(1)
    shared = bits[torch.randperm(65536, generator=g)].view(-1, 1, 8)
    sorted_ = bits.view(-1, 1, 8)
    x = torch.cat([alone, shared, sorted_])
    n = x.shape[0]
    kc, ke = _empty(n // 16, 1, 16, 8, "kernel")
    vc, ve = _empty(n // 16, 1, 16, 8, "kernel")
    slots = torch.arange(n)
    kernels.kv_write_slots(x.cuda(), x.flip(0).cuda(), kc, vc, slots.cuda(), key_exps=ke,
                           value_exps=ve)
    _compare(kc, ke, "kernel", 16, slots, x)
    _compare(vc, ve, "kernel", 16, slots, x.flip(0))


def test_write_strided_rows(gpu):
    """K and V as views into a fused projection's rows, and a cache that is a view
    with spare room in every row; nothing lands beside the rows."""
    from vllm_apple_amd import kernels

    g = torch.Generator().manual_seed(4)
    T, H, kv, d, nb, bs = 100, 4, 2, 64, 16, 16
    qkv = torch.randn(T, (H + 2 * kv) * d, generator=g).bfloat16().cuda()
    key = qkv[:, H * d:(H + kv) * d].view(T, kv, d)
    value = qkv[:, (H + kv) * d:].view(T, kv, d)
    big = torch.full((nb, bs, kv, d + 16), 0x2A, dtype=torch.uint8).cuda()
    kc = big[..., :d].view(torch.float8_e4m3fn)
    vc, ve = _empty(nb, kv, bs, d, "vllm")
    ke = torch.full((nb, bs, 2 * kv), 9, dtype=torch.uint8).cuda()[..., ::2]
    slots = torch.randperm(nb * bs, generator=g)[:T]
    kernels.kv_write_slots(key, value, kc, vc, slots.cuda(), key_exps=ke, value_exps=ve,
                           layout="vllm")
    _compare(kc.contiguous(), ke.contiguous(), "vllm", bs, slots, key)
    _compare(vc, ve, "vllm", bs, slots, value)
    assert bool((big[..., d:] == 0x2A).all())


@pytest.mark.parametrize("layout", ["kernel", "vllm"])
def test_write_decode_positions(gpu, layout):
    """Each sequence's token at its last position; sequences without one, past their
    table, or with a missing block write nothing."""
    from vllm_apple_amd import kernels

    g = torch.Generator().manual_seed(5)
    nb, bs, kv, d = 12, 16, 2, 64
    lens = torch.tensor([1, 16, 17, 0, -3, 40, 33, 20], dtype=torch.int32)
    table = torch.tensor([[3, -1], [4, -1], [5, 6], [7, 8], [9, 10], [0, 1], [2, 11], [11, 99]],
                         dtype=torch.int32)
    slots = torch.tensor([3 * 16, 4 * 16 + 15, 6 * 16, -1, -1, -1, -1, -1])
    new = [torch.randn(8, kv, d, generator=g).half().cuda() for _ in range(2)]
    kc, ke = _empty(nb, kv, bs, d, layout)
    vc, ve = _empty(nb, kv, bs, d, layout)
    kernels.kv_write_decode(*new, kc, vc, table.cuda(), lens.cuda(), key_exps=ke, value_exps=ve,
                            layout=layout)
    _compare(kc, ke, layout, bs, slots, new[0])
    _compare(vc, ve, layout, bs, slots, new[1])


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_read_every_code(gpu, dtype):
    """All 256 codes under every exponent a written row can have, to the nearest value
    of the type."""
    from vllm_apple_amd import kernels

    exps = torch.arange(1, 248, dtype=torch.uint8)
    codes = torch.arange(256, dtype=torch.uint8).view(2, 128).repeat(247, 1)
    e = exps.repeat_interleave(2)
    nb = -(-len(e) // 16)
    kc = torch.zeros(nb * 16, 128, dtype=torch.uint8)
    ke = torch.ones(nb * 16, dtype=torch.uint8)
    kc[:len(e)], ke[:len(e)] = codes, e
    kc = kc.view(nb, 1, 16, 128).view(torch.float8_e4m3fn)
    ke = ke.view(nb, 1, 16)
    slots = torch.arange(len(e)).cuda()
    for name in ("key", "value"):
        got = dict(zip(("key", "value"), kernels.kv_read_slots(
            kc.cuda(), kc.flip(0).contiguous().cuda() if name == "key" else kc.cuda(), ke.cuda(),
            ke.flip(0).contiguous().cuda() if name == "key" else ke.cuda(), slots,
            dtype=DTYPES[dtype])))[name].cpu()[:, 0]
        want64 = values(kc.view(-1, 128)[:len(e)], ke.view(-1)[:len(e)])
        want = want64.float().to(DTYPES[dtype])  # 32 bits hold every one of them
        nan = torch.isnan(want64)
        assert torch.equal(torch.isnan(got), nan)
        assert torch.equal(got[~nan], want[~nan])


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("layout", ["kernel", "vllm"])
@pytest.mark.parametrize("kv,d,bs,n", [(8, 128, 16, 301), (2, 64, 16, 1), (3, 80, 8, 77),
                                       (2, 100, 7, 31), (5, 1, 4, 6)])
def test_read_slots(gpu, dtype, layout, kv, d, bs, n):
    """Rows in any order, some twice, padding and slots past the cache as zeros,
    outputs that are views."""
    from vllm_apple_amd import kernels

    g = torch.Generator().manual_seed(n)
    nb = 9
    x = [torch.randn(nb, bs, kv, d, generator=g).to(DTYPES[dtype]) for _ in range(2)]
    held = [quantise(t) for t in x]
    caches = [rows_of(c.float().to(torch.float8_e4m3fn), layout).contiguous() for c, _ in held]
    exps = [rows_of(e, layout).contiguous() for _, e in held]
    slots = torch.randint(0, nb * bs, (n,), generator=g)
    slots[::4] = -1
    if n > 6:
        slots[6] = nb * bs
    want = [values(c, e).reshape(-1, kv, d)[slots.clamp(0, nb * bs - 1)]
            * ((slots >= 0) & (slots < nb * bs))[:, None, None] for c, e in held]
    want = [w.float().to(DTYPES[dtype]) for w in want]
    for index in (torch.int32, torch.int64):
        got = kernels.kv_read_slots(*(t.cuda() for t in caches + exps), slots.to(index).cuda(),
                                    dtype=DTYPES[dtype], layout=layout)
        assert all(torch.equal(a.cpu(), b) for a, b in zip(got, want))
    bufs = [canaried(torch.zeros(n, kv, d).to(DTYPES[dtype])) for _ in range(2)]
    kernels.kv_read_slots(*(t.cuda() for t in caches + exps), slots.cuda(), key=bufs[0][1],
                          value=bufs[1][1], layout=layout)
    for (buf, view), b in zip(bufs, want):
        assert torch.equal(view.cpu(), b) and tail_ok(buf)


def test_no_tokens(gpu):
    from vllm_apple_amd import kernels

    kc, ke = _empty(2, 1, 16, 64, "kernel")
    x = torch.zeros(0, 1, 64).half().cuda()
    none = torch.zeros(0, dtype=torch.int64).cuda()
    kernels.kv_write_slots(x, x, kc, kc, none, key_exps=ke, value_exps=ke)
    k, v = kernels.kv_read_slots(kc, kc, ke, ke, none)
    assert k.shape == v.shape == (0, 1, 64)


def test_offsets_past_32_bits(gpu):
    """Slots whose codes lie beyond 2^32 bytes from the cache's start."""
    from vllm_apple_amd import kernels

    nb, bs, kv, d = 36000, 128, 8, 128  # 4.7e9 bytes
    kc = torch.empty((nb, kv, bs, d), dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    ke = torch.empty((nb, kv, bs), dtype=torch.uint8, device="cuda")
    g = torch.Generator().manual_seed(6)
    x = torch.randn(40, kv, d, generator=g).bfloat16()
    slots = torch.randint(33000 * bs, nb * bs, (40,), generator=g).unique()[:30]
    x = x[:len(slots)]
    kernels.kv_write_slots(x.cuda(), x.cuda(), kc, kc, slots.cuda(), key_exps=ke, value_exps=ke)
    k, v = kernels.kv_read_slots(kc, kc, ke, ke, slots.cuda(), dtype=torch.bfloat16)
    want = values(*quantise(x)).bfloat16()
    assert torch.equal(k.cpu(), want) and torch.equal(v.cpu(), want)
    block, off = slots // bs, slots % bs
    assert torch.equal(kc.view(torch.uint8)[block.cuda(), :, off.cuda()].cpu().view(
        torch.float8_e4m3fn).double(), quantise(x)[0])
