"""What the quantised-cache and window operators refuse, and the C struct's layout.
No GPU: every refusal comes before a launch, and the pointers are never read."""
import ctypes
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

from vllm_apple_amd import _lib, kernels
from vllm_apple_amd.kv_cache import HipKVCache, KVCacheDescriptor

REPO = Path(__file__).resolve().parent.parent
PTR = 0x10000  # an aligned address that nothing reads


def _params(**kw):
    p = _lib.VaaAttnParams()
    d = dict(scale=0.125, num_seqs=2, max_seq_len=100, max_blocks_per_seq=8, head_size=64,
             block_size=16, num_kv_heads=2, num_query_heads=8, queries_per_kv=4, num_blocks=32,
             k_stride_block=2048, k_stride_head=1024, k_stride_token=64, v_stride_block=2048,
             v_stride_head=1024, v_stride_token=64, q_stride_token=512, q_stride_head=64,
             o_stride_token=512, o_stride_head=64, new_kv_stride_token=128, new_kv_stride_head=64)
    d.update(kw)
    for k, v in d.items():
        setattr(p, k, v)
    return p


def _view(**kw):
    v = _lib.VaaKvView()
    d = dict(cache_type=1, key_exps=PTR, value_exps=PTR, ke_stride_block=32, ke_stride_head=16,
             ke_stride_token=1, ve_stride_block=32, ve_stride_head=16, ve_stride_token=1)
    d.update(kw)
    for k, x in d.items():
        setattr(v, k, x)
    return v


def _calls(lib, p, v, ptr=PTR, ws=None, ws_bytes=0):
    """The status of the decode and of the prefill."""
    p, v = ctypes.byref(p), ctypes.byref(v)
    return (lib.vaa_paged_attention_decode_view(p, v, ptr, ptr, ptr, ptr, ptr, ptr, ws, ws_bytes,
                                                None),
            lib.vaa_paged_attention_prefill_view(p, v, ptr, ptr, ptr, ptr, ptr, ptr, ptr, 3, ws,
                                                 ws_bytes, None))


BAD = _lib.VAA_ERR_INVALID_ARG
NO = _lib.VAA_ERR_UNSUPPORTED


@pytest.mark.parametrize("params,view,status", [
    (dict(head_size=72), {}, NO), (dict(head_size=136), {}, NO), (dict(head_size=0), {}, NO),
    (dict(head_size=100), dict(cache_type=0), NO), ({}, dict(cache_type=2), NO),
    (dict(dtype=5), {}, NO), (dict(block_size=0), {}, BAD), (dict(num_query_heads=7), {}, BAD),
    (dict(num_kv_heads=0), {}, BAD), (dict(num_blocks=0), {}, BAD), ({}, dict(window=-1), BAD),
    ({}, dict(first_tokens=-1), BAD), ({}, dict(key_exps=None), BAD),
    ({}, dict(value_exps=None), BAD), (dict(k_stride_token=72), {}, BAD),
    (dict(v_stride_block=-16), {}, BAD), (dict(q_stride_token=12), {}, BAD),
    (dict(o_stride_head=4), {}, BAD), ({}, dict(ke_stride_token=-1), BAD),
    ({}, dict(ve_stride_token=1 << 24), BAD), (dict(k_stride_token=1 << 24), {}, BAD),
    (dict(k_stride_block=1 << 31), {}, NO), (dict(v_stride_token=1 << 23, block_size=256), {}, NO),
    (dict(scale=0.0), {}, BAD), (dict(scale=-1.0), {}, BAD), (dict(scale=float("nan")), {}, BAD),
    (dict(scale=float("inf")), {}, BAD), (dict(max_blocks_per_seq=0), {}, BAD),
    (dict(num_seqs=-1), {}, BAD),
])
def test_attention_refusals(params, view, status):
    lib = _lib.load()
    p, v = _params(**params), _view(**view)
    assert _calls(lib, p, v) == (status, status), _lib.last_error()
    assert lib.vaa_paged_attention_decode_view_workspace_size(
        ctypes.byref(p), ctypes.byref(v), None) == 0
    assert lib.vaa_paged_attention_prefill_view_workspace_size(
        ctypes.byref(p), ctypes.byref(v), 3) == 0


def test_attention_pointers_and_partitions():
    lib = _lib.load()
    p, v = _params(), _view()
    for ptr in (None, PTR + 8):
        assert _calls(lib, p, v, ptr) == (BAD, BAD)
    assert lib.vaa_paged_attention_decode_view(None, ctypes.byref(v), *[PTR] * 6, None, 0,
                                               None) == BAD
    assert lib.vaa_paged_attention_decode_view(ctypes.byref(p), None, *[PTR] * 6, None, 0,
                                               None) == BAD

    def decode(ws=None, n=0, **kw):
        return lib.vaa_paged_attention_decode_view(ctypes.byref(_params(**kw)), ctypes.byref(v),
                                                   *[PTR] * 6, ws, n, None)

    assert decode(partition_size=100) == BAD
    assert decode(partition_size=-2) == NO and decode(partition_size=-9) == NO
    assert decode(num_seqs=65536) == NO
    assert decode(partition_size=-1, num_seqs=8193) == NO
    # A split needs its workspace: present, large enough, aligned.
    split = _params(partition_size=128, max_seq_len=128 * 8, max_blocks_per_seq=64)
    part = ctypes.c_int32()
    need = lib.vaa_paged_attention_decode_view_workspace_size(ctypes.byref(split),
                                                              ctypes.byref(v), ctypes.byref(part))
    assert need == 2 * 8 * 8 * (64 + 2) * 4 and part.value == 128
    args = dict(partition_size=128, max_seq_len=128 * 8, max_blocks_per_seq=64)
    assert decode(**args) == _lib.VAA_ERR_WORKSPACE
    assert decode(PTR, need - 1, **args) == _lib.VAA_ERR_WORKSPACE
    assert decode(PTR + 4, need, **args) == BAD
    # No sequences, no tokens: nothing to do, nothing read.
    assert decode(num_seqs=0) == _lib.VAA_OK
    assert lib.vaa_paged_attention_prefill_view(ctypes.byref(p), ctypes.byref(v), *[None] * 7, 0,
                                                None, 0, None) == _lib.VAA_OK
    assert lib.vaa_paged_attention_prefill_view(ctypes.byref(p), ctypes.byref(v), *[PTR] * 7, -1,
                                                None, 0, None) == BAD


def test_window_bounds_the_workspace():
    """Partitions count the tokens that are seen, whatever the longest context."""
    lib = _lib.load()
    sizes = []
    for longest in (5000, 50000):
        p = _params(partition_size=128, max_seq_len=longest, max_blocks_per_seq=4000)
        sizes.append(lib.vaa_paged_attention_decode_view_workspace_size(
            ctypes.byref(p), ctypes.byref(_view(window=1000, first_tokens=4)), None))
    assert sizes[0] == sizes[1] > 0


def test_row_refusals():
    lib = _lib.load()
    good, v = _params(), _view()

    def rows(p=good, view=v, n=3, ptr=PTR, slots=PTR, itype=0):
        args = (ctypes.byref(p), ctypes.byref(view), ptr, ptr, slots, itype, ptr, ptr, n, None)
        got = {lib.vaa_kv_write_slots_q8(*args), lib.vaa_kv_read_slots_q8(*args)}
        assert len(got) == 1
        return got.pop()

    assert rows(view=_view(cache_type=0)) == NO
    assert rows(_params(dtype=7)) == NO
    assert rows(_params(block_size=0)) == BAD and rows(_params(num_kv_heads=0)) == BAD
    assert rows(_params(head_size=0)) == BAD
    assert rows(n=-1) == BAD and rows(ptr=None) == BAD and rows(slots=None) == BAD
    assert rows(view=_view(key_exps=None)) == BAD and rows(itype=2) == BAD
    assert rows(n=0, ptr=None, slots=None) == _lib.VAA_OK
    dec = (ctypes.byref(good), ctypes.byref(v), PTR, PTR)
    assert lib.vaa_kv_write_decode_q8(*dec, None, PTR, PTR, PTR, None) == BAD
    assert lib.vaa_kv_write_decode_q8(*dec, PTR, None, PTR, PTR, None) == BAD
    assert lib.vaa_kv_write_decode_q8(None, ctypes.byref(v), *[PTR] * 6, None) == BAD
    none = ctypes.byref(_params(num_seqs=0))
    assert lib.vaa_kv_write_decode_q8(none, ctypes.byref(v), *[None] * 6, None) == _lib.VAA_OK


def test_view_struct_layout_matches_header(tmp_path):
    if shutil.which("gcc") is None:
        pytest.skip("gcc not available")
    names = [f[0] for f in _lib.VaaKvView._fields_]
    prog = tmp_path / "layout.c"
    prog.write_text(
        "#include <stdio.h>\n#include <stddef.h>\n#include \"vllm_apple_amd.h\"\n"
        "int main(void) {\n  printf(\"%zu\\n\", sizeof(vaa_kv_view));\n"
        + "".join(f'  printf("%zu\\n", offsetof(vaa_kv_view, {n}));\n' for n in names)
        + "  return 0;\n}\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c99", f"-I{REPO / 'include'}", str(prog), "-o", str(exe)],
                   check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True,
                                          check=True).stdout.split()]
    assert got[0] == ctypes.sizeof(_lib.VaaKvView)
    assert got[1:] == [getattr(_lib.VaaKvView, n).offset for n in names]


def test_wrappers_refuse_host_tensors():
    c = torch.zeros(4, 2, 16, 64, dtype=torch.uint8).view(torch.float8_e4m3fn)
    e = torch.ones(4, 2, 16, dtype=torch.uint8)
    x = torch.zeros(3, 2, 64).half()
    q = torch.zeros(3, 8, 64).half()
    i = torch.zeros(3, dtype=torch.int32)
    t = torch.zeros(3, 4, dtype=torch.int32)
    for call in (
            lambda: kernels.kv_write_slots(x, x, c, c, i, key_exps=e, value_exps=e),
            lambda: kernels.kv_read_slots(c, c, e, e, i),
            lambda: kernels.kv_read_slots(c, c, e, e, i, key=x, value=x),
            lambda: kernels.kv_write_decode(x, x, c, c, t, i, key_exps=e, value_exps=e),
            lambda: kernels.paged_decode(q, c, c, t, i, scale=0.1, max_seq_len=9, key_exps=e,
                                         value_exps=e),
            lambda: kernels.paged_prefill(q, c, c, t, i, i, scale=0.1, window=4)):
        with pytest.raises(ValueError, match="ROCm device"):
            call()
    with pytest.raises(ValueError, match="go together"):
        kernels.kv_read_slots(c, c, e, e, i, key=x)
    with pytest.raises(ValueError, match="write the new token before"):
        kernels.paged_decode(q, c, c, t, i, scale=0.1, max_seq_len=9, window=4, new_keys=x,
                             new_values=x)
    with pytest.raises(ValueError, match="split_keys"):
        kernels.paged_prefill(q, c, c, t, i, i, scale=0.1, window=4, split_keys=64)


def test_view_checks():
    c = torch.zeros(4, 2, 16, 64, dtype=torch.uint8).view(torch.float8_e4m3fn)
    e = torch.ones(4, 2, 16, dtype=torch.uint8)
    h = torch.zeros(4, 2, 16, 64).half()
    for args, kw, match in (
            ((c, c, e, None, "kernel"), {}, "go together"),
            ((c, c, None, None, "kernel"), {}, "needs key_exps"),
            ((h, h, e, e, "kernel"), {}, "float8_e4m3fn"),
            ((c, c, e[:2], e, "kernel"), {}, "must be uint8"),
            ((c, c, e.int(), e, "kernel"), {}, "must be uint8"),
            ((c, c, e, e, "other"), {}, "layout"),
            ((h, h, None, None, "kernel"), dict(window=-1), "window"),
            ((h, h, None, None, "kernel"), dict(first_tokens=1 << 31), "first_tokens")):
        with pytest.raises(ValueError, match=match):
            kernels._kv_view(*args, **kw)
    v = kernels._kv_view(c, c, e, e, "vllm", 5, 2)
    assert (v.cache_type, v.window, v.first_tokens) == (1, 5, 2)
    assert (v.ke_stride_block, v.ke_stride_head, v.ke_stride_token) == (32, 1, 16)


@pytest.mark.parametrize("name,count", [("rows_q8", 11), ("decode_view", 17),
                                        ("prefill_view", 17)])
def test_native_path_declines_other_objects(name, count):
    fn = getattr(_lib.host(), name)
    t = torch.zeros(4, 4, 8, dtype=torch.float16)
    for a in (None, t, t[0], 3, "x", 2.5, object()):
        assert fn(*[a] * count) is False
    with pytest.raises(TypeError):
        fn(t)


def test_partition_choice_counts_what_is_seen(monkeypatch):
    monkeypatch.setattr(kernels, "device_cus", lambda device=None: 256)
    q = torch.zeros(4, 32, 128)
    lens = [30000, 20000, 9000, 25000]
    kernels._view_partition_cache.clear()
    window = kernels._view_partition(lens, q, 8, 1000, 24, False)
    assert window == kernels._decode_partition(q, 8, [1024] * 4, False)
    q8 = kernels._view_partition(lens, q, 8, 2000, 48, True)
    assert q8 == 2 * kernels._decode_partition(q, 8, [1024] * 4, False)
    assert kernels._view_partition(lens, q, 8, 1000, 24, False) == window  # remembered


def test_quantised_cache_descriptor():
    d = KVCacheDescriptor(num_blocks=3, block_size=16, num_kv_heads=2, head_size=64, num_layers=2,
                          dtype=torch.float8_e4m3fn, device="cpu")
    assert d.quantised and d.block_size_bytes == 2 * 2 * 16 * 65
    assert d.total_cache_bytes == 2 * 3 * d.block_size_bytes
    cache = HipKVCache(d)
    k, v = cache.get_buffers(1)
    ke, ve = cache.get_exponents(1)
    assert k.dtype == v.dtype == torch.float8_e4m3fn and k.shape == (3, 2, 16, 64)
    assert ke.dtype == torch.uint8 and ke.shape == ve.shape == (3, 2, 16)
    ke.fill_(5)
    cache.reset()
    assert int(ke.sum()) == 0
    plain = HipKVCache(KVCacheDescriptor(3, 16, 2, 64, 1, device="cpu"))
    with pytest.raises(ValueError, match="no exponents"):
        plain.get_exponents(0)
    for block, off in ((3, 0), (-1, 0), (0, -1), (0, 16)):
        with pytest.raises(ValueError):
            cache.write_kv(0, block, off, torch.zeros(2, 64), torch.zeros(2, 64))
