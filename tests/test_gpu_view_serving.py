"""The quantised cache and the windows as a serving program uses them: a prompt
written and prefilled in chunks, tokens decoded behind it, rows read back; through
the wrappers, the engine ops, captured graphs and several streams."""
import pytest
import torch

from view_oracle import Case, check, quantise, values

pytestmark = pytest.mark.gpu

H, KV, D, BS = 8, 2, 64, 16
SCALE = D ** -0.5


class Model:
    """Sequences' tokens, K/V rows and queries, and the paged cache they go through."""

    def __init__(self, lens, dtype, q8, seed=0):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.dtype, self.q8 = lens, dtype, q8
        self.k, self.v = ([torch.randn(n, KV, D, generator=g).to(dtype) for n in lens]
                          for _ in range(2))
        self.q = [torch.randn(n, H, D, generator=g).to(dtype) for n in lens]
        need = [-(-n // BS) for n in lens]
        perm = torch.randperm(sum(need) + 2, generator=g).to(torch.int32)
        self.table = torch.full((len(lens), max(need)), -1, dtype=torch.int32)
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = perm[at:at + n]
            at += n
        self.blocks = sum(need) + 2

    def slots(self, s, lo, hi):
        p = torch.arange(lo, hi)
        return self.table[s, p // BS].long() * BS + p % BS

    def reference(self, s, lo, hi, window, first):
        """(output, tolerance) of the queries at lo .. hi - 1 of sequence s."""
        c = Case([hi], H, KV, D, dtype={torch.float16: "fp16", torch.bfloat16: "bf16"}[self.dtype],
                 q8=self.q8, bs=BS, window=window, first=first, new=[hi - lo])
        c.q = self.q[s][lo:hi]
        rows = [x[s][:hi] for x in (self.k, self.v)]
        rows = [values(*quantise(x)) if self.q8 else x.double() for x in rows]
        c.cached = lambda _: rows
        return c


@pytest.mark.parametrize("q8,dtype,window,first,engine", [
    (True, torch.bfloat16, 0, 0, False), (True, torch.float16, 40, 4, False),
    (False, torch.bfloat16, 40, 4, False),  # the engine ops take fp16 alone
    (True, torch.float16, 0, 0, True), (True, torch.float16, 40, 4, True),
    (False, torch.float16, 40, 0, True)])
def test_prompt_then_tokens(gpu, q8, dtype, window, first, engine):
    from vllm_apple_amd import kernels
    from vllm_apple_amd.engine import KVWriteOp, PagedAttentionOp
    from vllm_apple_amd.kv_cache import HipKVCache, KVCacheDescriptor

    m = Model([150, 37, 90], dtype, q8)
    cache = HipKVCache(KVCacheDescriptor(m.blocks, BS, KV, D, 2,
                                         dtype=torch.float8_e4m3fn if q8 else dtype))
    kc, vc = cache.get_buffers(1)
    ke, ve = cache.get_exponents(1) if q8 else (None, None)
    bt = m.table.cuda()
    view = dict(window=window, first_tokens=first)
    write, attn = KVWriteOp(None, KV, D, BS), PagedAttentionOp(None, KV, H, D, BS)
    exps = dict(key_exps_buffer=ke, value_exps_buffer=ve)

    def chunk(spans):
        n = [hi - lo for lo, hi in spans]
        slots = torch.cat([m.slots(s, *x) for s, x in enumerate(spans)]).cuda()
        k, v, q = (torch.cat([t[s][lo:hi] for s, (lo, hi) in enumerate(spans)]).cuda()
                   for t in (m.k, m.v, m.q))
        tok = torch.repeat_interleave(torch.arange(len(n)), torch.tensor(n)).to(torch.int32).cuda()
        pos = torch.cat([torch.arange(*x) for x in spans]).to(torch.int32).cuda()
        out = torch.zeros_like(q)
        longest = max(hi for _, hi in spans)
        if engine:
            write.encode_prefill(None, k, v, kc, vc, slots, len(q), **exps)
            attn.encode_prefill(None, q, kc, vc, bt, tok, pos, out, len(q), len(n), longest,
                                bt.shape[1], **view, **exps)
        else:
            kernels.kv_write_slots(k, v, kc, vc, slots, key_exps=ke, value_exps=ve)
            kernels.paged_prefill(q, kc, vc, bt, tok, pos, scale=SCALE, output=out, key_exps=ke,
                                  value_exps=ve, max_seq_len=longest, **view)
        at = 0
        for s, (lo, hi) in enumerate(spans):
            check(out[at:at + hi - lo], *m.reference(s, lo, hi, window, first).attend(True),
                  f"chunk {spans} sequence {s}")
            at += hi - lo

    def token(p):
        lens = torch.tensor([x + 1 for x in p], dtype=torch.int32).cuda()
        k, v, q = (torch.stack([t[s][x] for s, x in enumerate(p)]).cuda()
                   for t in (m.k, m.v, m.q))
        out = torch.empty_like(q)
        if engine:
            attn.encode_decode_fused(None, q, k, v, kc, vc, bt, lens, out, len(p), max(p) + 1,
                                     bt.shape[1], **view, **exps)
            again = torch.empty_like(q)
            attn.encode_decode(None, q, kc, vc, bt, lens, again, len(p), max(p) + 1, bt.shape[1],
                               **view, **exps)
            assert torch.equal(again, out)
        else:
            kernels.kv_write_decode(k, v, kc, vc, bt, lens, key_exps=ke, value_exps=ve)
            kernels.paged_decode(q, kc, vc, bt, lens, scale=SCALE, max_seq_len=max(p) + 1,
                                 output=out, key_exps=ke, value_exps=ve, **view)
        for s, x in enumerate(p):
            check(out[s:s + 1], *m.reference(s, x, x + 1, window, first).attend(False),
                  f"token {p} sequence {s}")

    chunk([(0, 100), (0, 20), (0, 33)])
    chunk([(100, 140), (20, 30), (33, 80)])
    for i in range(7):
        token([140 + i, 30 + i, 80 + i])
    if q8:
        got = kernels.kv_read_slots(kc, vc, ke, ve, m.slots(0, 0, 147).cuda(), dtype=dtype)
        for a, b in zip(got, (m.k, m.v)):
            assert torch.equal(a.cpu(), values(*quantise(b[0][:147])).to(dtype))
        cache.write_kv(1, int(m.table[1, 0]), 3, m.k[0][5], m.v[0][5])
        slot = m.slots(1, 3, 4).cuda()
        a, b = kernels.kv_read_slots(kc, vc, ke, ve, slot, dtype=dtype)
        assert torch.equal(a.cpu()[0], values(*quantise(m.k[0][5:6])).to(dtype)[0])


def _step(c, kind, out, part=0):
    """One call on a case whose operands are on the GPU already."""
    from vllm_apple_amd import kernels

    if kind == "decode":
        return lambda stream=None: kernels.paged_decode(
            seq_lens=c["seq_lens"], max_seq_len=c["longest"], output=out, partition_size=part,
            stream=stream, **c["ops"])
    return lambda stream=None: kernels.paged_prefill(
        token_to_seq=c["tok"], positions=c["pos"], max_seq_len=c["longest"], output=out,
        stream=stream, **c["ops"])


def _on_gpu(c):
    return dict(ops=c.cuda(), seq_lens=c.seq_lens.cuda(), tok=c.tok.cuda(), pos=c.pos.cuda(),
                longest=max(c.lens))


@pytest.mark.parametrize("kind,part", [("decode", 0), ("decode", 128), ("decode", -1),
                                       ("prefill", 0)])
@pytest.mark.parametrize("q8", [True, False])
def test_captured_and_replayed(gpu, kind, part, q8):
    """Two graphs and an eager call in turns, lengths and queries changed in between:
    every replay is the eager result, bit for bit."""
    from vllm_apple_amd import kernels

    made = []
    for seed in (1, 2):
        c = Case([900, 40, 333], H, KV, D, dtype="bf16", q8=q8, seed=seed, window=400, first=5,
                 new=None if kind == "decode" else [4, 1, 2], layout="vllm")
        g = _on_gpu(c)
        out, eager = torch.zeros_like(c.q.cuda()), torch.zeros_like(c.q.cuda())
        x = torch.randn(3, KV, D).bfloat16().cuda()
        kc, vc = g["ops"]["key_cache"], g["ops"]["value_cache"]
        exps = dict(key_exps=g["ops"]["key_exps"], value_exps=g["ops"]["value_exps"])
        slots = torch.tensor([0, 1, -1]).cuda()  # the unused block's first rows

        def run(o, g=g, x=x, kc=kc, vc=vc, exps=exps, slots=slots):
            if q8:
                kernels.kv_write_slots(x, x, kc, vc, slots, layout="vllm", **exps)
            _step(g, kind, o, part)()
        run(out)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            run(out)
        made.append((g, out, eager, run, graph))
    for i in range(4):
        for g, out, eager, run, graph in made:
            g["ops"]["query"].copy_(torch.randn_like(g["ops"]["query"]))
            g["seq_lens"].sub_(3 * (i % 2))
            out.zero_()
            graph.replay()
        for g, out, eager, run, graph in made:
            run(eager)
        torch.cuda.synchronize()
        for g, out, eager, run, graph in made:
            assert torch.equal(out, eager) and bool(out.any())


@pytest.mark.parametrize("kind,part", [("decode", 128), ("decode", -1), ("prefill", 0)])
def test_two_streams_at_once(gpu, kind, part):
    """Calls in flight on two streams, given explicitly and as the current stream, do
    not share scratch memory."""
    cases, want = [], []
    for seed in (1, 2):
        c = Case([3000, 200], H, KV, D, dtype="fp16", seed=seed, layout="vllm",
                 new=None if kind == "decode" else [5, 9])
        g = _on_gpu(c)
        out = torch.zeros_like(c.q.cuda())
        _step(g, kind, out, part)()
        cases.append((g, c))
        want.append(out)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[torch.zeros_like(w) for _ in range(8)] for w in want]
    torch.cuda.synchronize()
    for i in range(8):
        for (g, c), s, o in zip(cases, streams, got):
            if i % 2:
                _step(g, kind, o[i], part)(stream=s)
            else:
                with torch.cuda.stream(s):
                    _step(g, kind, o[i], part)()
    torch.cuda.synchronize()
    for o, w in zip(got, want):
        assert all(torch.equal(x, w) for x in o)


@pytest.mark.parametrize("q8", [True, False])
def test_native_path_and_wrapper_agree(gpu, monkeypatch, q8):
    """The same bits and the same refusals with the native host path and without it."""
    from vllm_apple_amd import _lib, kernels

    class Declines:
        def __getattr__(self, name):
            return lambda *a: False

    results = []
    for native in (True, False):
        if not native:
            monkeypatch.setattr(_lib, "host", lambda: Declines())
        c = Case([400, 30], H, KV, D, dtype="fp16", q8=q8, window=100, first=3, layout="vllm")
        p = Case([400, 30], H, KV, D, dtype="fp16", q8=q8, window=100, first=3, new=[20, 4])
        g, gp = _on_gpu(c), _on_gpu(p)
        got = []
        for part in (0, 128, -1):
            out = torch.zeros_like(c.q.cuda())
            _step(g, "decode", out, part)()
            got.append(out)
        out = torch.zeros_like(p.q.cuda())
        _step(gp, "prefill", out)()
        got.append(out)
        got.append(kernels.paged_decode(seq_lens=g["seq_lens"], max_seq_len=400,
                                        seq_lens_host=[400, 30], **g["ops"]))
        got.append(kernels.paged_prefill(token_to_seq=gp["tok"], positions=gp["pos"], **gp["ops"]))
        if q8:
            x = torch.randn(2, KV, D, generator=torch.Generator().manual_seed(3)).half().cuda()
            slots = torch.tensor([0, 1]).cuda()
            o = g["ops"]
            kernels.kv_write_slots(x, x, o["key_cache"], o["value_cache"], slots,
                                   key_exps=o["key_exps"], value_exps=o["value_exps"],
                                   layout="vllm")
            got += kernels.kv_read_slots(o["key_cache"], o["value_cache"], o["key_exps"],
                                         o["value_exps"], slots, layout="vllm")
        results.append([t.cpu() for t in got])
        o = dict(g["ops"], output=torch.zeros_like(c.q.cuda()))
        with pytest.raises(ValueError, match="multiple of 128"):
            kernels.paged_decode(seq_lens=g["seq_lens"], max_seq_len=400, partition_size=100, **o)
        with pytest.raises(ValueError, match="workspace"):
            kernels.paged_decode(seq_lens=g["seq_lens"], max_seq_len=400, partition_size=128,
                                 workspace=torch.zeros(16, dtype=torch.uint8).cuda(), **o)
        with pytest.raises(ValueError, match="scale"):
            kernels.paged_decode(seq_lens=g["seq_lens"], max_seq_len=400, **dict(o, scale=-1.0))
        with pytest.raises(ValueError, match="head_size"):
            kernels.paged_decode(seq_lens=g["seq_lens"], max_seq_len=400,
                                 **dict(o, query=o["query"][..., :32], output=None))
        with pytest.raises(ValueError, match="rows|shape"):
            kernels.paged_decode(seq_lens=g["seq_lens"], max_seq_len=400,
                                 **dict(o, query=o["query"][:1], output=o["output"][:1]))
    for a, b in zip(*results):
        assert torch.equal(a, b)


def test_strided_operands(gpu):
    """Queries and outputs that are views into wider rows, a cache that is every
    second block of a larger one, exponents in a tensor of their own order."""
    from vllm_apple_amd import kernels

    for kind in ("decode", "prefill"):
        c = Case([70, 300], H, KV, D, dtype="bf16", layout="vllm", window=64, first=2,
                 new=None if kind == "decode" else [33, 20])
        ref, tol = c.attend(kind == "prefill")
        g = _on_gpu(c)
        n = len(c.q)
        wide = torch.zeros(n, 3 * H * D).bfloat16().cuda()
        q = wide[:, H * D:2 * H * D].view(n, H, D)
        q.copy_(c.q)
        big = torch.full((n, H, 2, D), 7.0).bfloat16().cuda()
        out = big[:, :, 0]
        nb = c.kc.shape[0]
        ops = dict(g["ops"], query=q)
        for name in ("key_cache", "value_cache"):
            x = torch.full((nb, 2, *c.kc.shape[1:]), 0x7F, dtype=torch.uint8).cuda()
            x[:, 0] = ops[name].view(torch.uint8)
            ops[name] = x.view(torch.float8_e4m3fn)[:, 0]
        for name in ("key_exps", "value_exps"):
            ops[name] = ops[name].permute(2, 1, 0).contiguous().permute(2, 1, 0)
        g["ops"] = ops
        _step(g, kind, out)()
        check(out, ref, tol, kind)
        assert bool((big[:, :, 1] == 7).all())


@pytest.mark.parametrize("q8", [True, False])
def test_caches_past_32_bits(gpu, q8):
    """Blocks whose bytes lie beyond 2^32 from the cache's start, for both kernels."""
    from vllm_apple_amd import kernels

    D8, KV8 = 128, 8
    nb = 320000 if q8 else 160000  # blocks of 16 tokens x 8 heads: 2^14 values each
    c = Case([100, 45], 8, KV8, D8, dtype="bf16", q8=q8, layout="vllm", window=60, first=3)
    p = Case([100, 45], 8, KV8, D8, dtype="bf16", q8=q8, layout="vllm", window=60, first=3,
             new=[30, 2])
    for case, prefill in ((c, False), (p, True)):
        ref, tol = case.attend(prefill)
        g = _on_gpu(case)
        ops = dict(g["ops"])
        far = nb - case.kc.shape[0]
        dt = torch.uint8 if q8 else torch.bfloat16
        for name in ("key_cache", "value_cache"):
            small = ops[name].view(dt) if q8 else ops[name]
            x = torch.empty((nb, *small.shape[1:]), dtype=dt, device="cuda")
            x[far:] = small
            ops[name] = x.view(torch.float8_e4m3fn) if q8 else x
        if q8:
            for name in ("key_exps", "value_exps"):
                x = torch.empty((nb, *ops[name].shape[1:]), dtype=dt, device="cuda")
                x[far:] = ops[name]
                ops[name] = x
        ops["block_table"] = torch.where(ops["block_table"] >= 0, ops["block_table"] + far, -1)
        g["ops"] = ops
        out = torch.zeros_like(ops["query"])
        _step(g, "prefill" if prefill else "decode", out)()
        check(out, ref, tol, "prefill" if prefill else "decode")
        del ops, g
        torch.cuda.empty_cache()


def test_another_device_is_refused(gpu):
    """Operands on several devices (here: one on the host) raise before a launch."""
    from vllm_apple_amd import kernels

    c = Case([40], H, KV, D)
    for name in ("block_table", "key_exps", "value_cache"):
        ops = dict(c.cuda())
        ops[name] = ops[name].cpu()
        with pytest.raises(ValueError, match="one ROCm device"):
            kernels.paged_decode(seq_lens=c.seq_lens.cuda(), max_seq_len=40, **ops)
