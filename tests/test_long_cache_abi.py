"""include/bz_long_cache.h on the CPU: struct layouts, and the host-side checks' status codes and Python refusals. No call
here launches a kernel (every case fails validation first)."""
import ctypes
import subprocess
from pathlib import Path

import pytest
import torch

REPO = Path(__file__).resolve().parents[1]


@pytest.fixture(scope="module")
def lib(pkg):
    return pkg.load()


@pytest.fixture(scope="module")
def K(pkg):
    from breeze_tts_2_flash_amd import kernels
    return kernels


STRUCTS = {"bz_gqa_window_args": "GqaWindowArgs", "bz_kv4_cache": "Kv4CacheArgs", "bz_gqa_kv4_args": "GqaKv4Args",
           "bz_gqa_tracked_args": "GqaTrackedArgs", "bz_kv_select_args": "KvSelectArgs", "bz_kv_tensor": "KvTensor"}


def test_struct_layouts_match_c(K, tmp_path):
    src = ["#include <stddef.h>", "#include <stdio.h>", '#include "bz_long_cache.h"', "int main(void) {"]
    for c, py in STRUCTS.items():
        src.append(f'  printf("{c} %zu\\n", sizeof({c}));')
        src += [f'  printf("{c}.{f} %zu\\n", offsetof({c}, {f}));' for f, _ in getattr(K, py)._fields_]
    src += [f'  printf("tensors %d\\n", BZ_KV_TENSORS);', "  return 0;", "}"]
    (tmp_path / "layout.c").write_text("\n".join(src))
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c11", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", f"-I{REPO / 'include'}",
                    str(tmp_path / "layout.c"), "-o", str(exe)], check=True)
    got = dict(ln.split() for ln in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines())
    for c, py in STRUCTS.items():
        cls = getattr(K, py)
        assert int(got[c]) == ctypes.sizeof(cls), c
        for f, _ in cls._fields_:
            assert int(got[f"{c}.{f}"]) == getattr(cls, f).offset, (c, f)
    assert int(got["tensors"]) == K.KV_TENSORS


def _base(K, **over):
    """Plausible sizes with fake (never dereferenced) device addresses."""
    a = K.GqaDecodeArgs()
    a.q, a.q_stride_b, a.q_stride_h, a.q_stride_t = 0x10000, 16 * 128, 128, 16 * 128
    a.k_cache, a.v_cache = 0x100000, 0x200000
    a.kv_stride_b, a.kv_stride_h, a.kv_stride_s = 8 * 256 * 128, 256 * 128, 128
    a.seq_lens, a.scale = 0x30000, 128 ** -0.5
    a.out, a.out_stride_b, a.out_stride_h = 0x40000, 16 * 128, 128
    a.batch, a.num_q_heads, a.num_kv_heads, a.head_dim, a.capacity = 2, 16, 8, 128, 4096
    a.kv_stride_b, a.kv_stride_h = 8 * 4096 * 128, 4096 * 128
    a.num_splits, a.tokens_per_row = 4, 1
    for k, v in over.items():
        setattr(a, k, v)
    return a


def _cache(K, **over):
    c = K.Kv4CacheArgs()
    c.k, c.v, c.k_scale, c.v_scale = 0x100000, 0x200000, 0x300000, 0x400000
    c.stride_b, c.stride_h, c.stride_s = 8 * 4096 * 64, 4096 * 64, 64
    c.scale_stride_b, c.scale_stride_h = 8 * 4096 * 4, 4096 * 4
    c.batch, c.num_kv_heads, c.capacity, c.head_dim = 2, 8, 4096, 128
    for k, v in over.items():
        setattr(c, k, v)
    return c


COMMON = [
    (dict(q=None), -1), (dict(out=None), -1), (dict(seq_lens=None), -1), (dict(mask=0x50000), -3), (dict(mask_dtype=1), -3),
    (dict(q=0x10008), -4), (dict(q_stride_h=132), -4), (dict(tokens_per_row=2, q_stride_t=4), -4), (dict(out=0x40001), -4),
    (dict(seq_lens=0x30002), -4), (dict(kv_start=0x30001), -4), (dict(num_splits=-1), -2), (dict(num_splits=257), -2),
    (dict(tokens_per_row=-1), -2), (dict(num_q_heads=24), -3), (dict(workspace=None), -5),
    (dict(workspace=0x60000, workspace_bytes=16), -5), (dict(workspace=0x60010, workspace_bytes=1 << 30), -4),
]


@pytest.mark.parametrize("over,code", COMMON + [
    (dict(k_cache=None), -1), (dict(v_cache=0x200008), -4), (dict(kv_stride_s=132), -4), (dict(kv_stride_s=64), -2),
    (dict(batch=0), -2), (dict(num_kv_heads=5), -2), (dict(capacity=0), -2), (dict(head_dim=96), -3),
    (dict(capacity=1 << 23), -2), (dict(window=-1), -2), (dict(sinks=-1), -2),
])
def test_window_refusals(lib, K, over, code):
    over = dict(over)
    w = K.GqaWindowArgs()
    w.window, w.sinks = over.pop("window", 1024), over.pop("sinks", 4)
    w.base = _base(K, **over)
    assert lib.bz_gqa_window(ctypes.byref(w), None) == code


@pytest.mark.parametrize("over,cover,code", [(o, {}, c) for o, c in COMMON] + [
    ({}, dict(k=None), -1), ({}, dict(v_scale=None), -1), ({}, dict(head_dim=32), -3), ({}, dict(k=0x100008), -4),
    ({}, dict(stride_s=72), -4), ({}, dict(stride_s=32), -2), ({}, dict(k_scale=0x300002), -4),
    ({}, dict(scale_stride_h=4096 * 4 + 1), -4), ({}, dict(capacity=1 << 25), -2), ({}, dict(batch=0), -2),
    (dict(tokens_per_row=17), {}, -3),
])
def test_kv4_refusals(lib, K, over, cover, code):
    ka = K.GqaKv4Args()
    ka.base, ka.cache = _base(K, **over), _cache(K, **cover)
    assert lib.bz_gqa_decode_kv4(ctypes.byref(ka), None) == code


@pytest.mark.parametrize("over,mine,code", [(o, {}, c) for o, c in COMMON if "tokens_per_row" not in o] + [
    ({}, dict(weights=None), -1), ({}, dict(weights_out=None), -1), ({}, dict(weights=0x70001), -4),
    (dict(tokens_per_row=2, q_stride_t=128), {}, -3),
])
def test_tracked_refusals(lib, K, over, mine, code):
    ta = K.GqaTrackedArgs()
    ta.base = _base(K, **over)
    ta.weights = ta.weights_out = 0x70000
    ta.w_stride_b = ta.wo_stride_b = 8 * 4096
    ta.w_stride_h = ta.wo_stride_h = 4096
    for k, v in mine.items():
        setattr(ta, k, v)
    assert lib.bz_gqa_decode_tracked(ctypes.byref(ta), None) == code


@pytest.mark.parametrize("over,code", [
    (dict(k=None), -1), (dict(slots=None), -1), (dict(tokens=0), -2), (dict(sb=4), -4), (dict(k=0x10008), -4),
    (dict(cache=dict(batch=32768)), -2), (dict(cache=dict(head_dim=256)), -3), (dict(cache=dict(v=0x200004)), -4),
    (dict(cache=dict(stride_s=48)), -2), (dict(cache=dict(k_scale=None)), -1),
])
def test_store_load_refusals(lib, K, over, code):
    c = _cache(K, **over.get("cache", {}))
    x = dict(k=0x10000, v=0x20000, sb=1024, sh=128, st=1024, tokens=1, slots=0x30000)
    x.update({k: v for k, v in over.items() if k != "cache"})
    assert lib.bz_kv4_store(x["k"], x["v"], x["sb"], x["sh"], x["st"], x["tokens"], x["slots"], None, ctypes.byref(c),
                            None) == code
    assert lib.bz_kv4_load(ctypes.byref(c), x["slots"], x["tokens"], x["k"], x["v"], x["sb"], x["sh"], x["st"],
                           None) == code


@pytest.mark.parametrize("over,code", [
    (dict(weights=None), -1), (dict(index=None), -1), (dict(lens=None), -1), (dict(seq_lens=None), -1), (dict(keep=0), -2),
    (dict(keep=4097), -2), (dict(sinks=-1), -2), (dict(sinks=60, recent=41), -2), (dict(batch=0), -2),
    (dict(weights_out=0x70002), -4), (dict(index=0x80001), -4),
])
def test_select_refusals(lib, K, over, code):
    a = K.KvSelectArgs()
    a.weights, a.w_stride_b, a.w_stride_h = 0x70000, 8 * 4096, 4096
    a.seq_lens, a.index, a.lens = 0x30000, 0x80000, 0x90000
    a.batch, a.num_kv_heads, a.capacity, a.keep, a.sinks, a.recent = 2, 8, 4096, 100, 4, 16
    for k, v in over.items():
        setattr(a, k, v)
    assert lib.bz_kv_select(ctypes.byref(a), None) == code


@pytest.mark.parametrize("over,num,code", [
    ({}, 0, -2), ({}, 5, -2), (dict(src=None), 1, -1), (dict(dst=None), 1, -1), (dict(row_bytes=0), 1, -2),
    (dict(src_stride_s=128), 1, -2), (dict(dst=0x100000, dst_stride_s=512), 1, -2),
])
def test_compact_refusals(lib, K, over, num, code):
    arr = (K.KvTensor * 4)()
    t = arr[0]
    t.src, t.dst, t.row_bytes = 0x100000, 0x900000, 256
    t.src_stride_b = t.dst_stride_b = 8 * 4096 * 256
    t.src_stride_h = t.dst_stride_h = 4096 * 256
    t.src_stride_s = t.dst_stride_s = 256
    for k, v in over.items():
        setattr(t, k, v)
    assert lib.bz_kv_compact(arr, num, 0x80000, 0x90000, 2, 8, 4096, 100, None) == code


def test_sizes_past_32_bits(lib, K):
    """Lengths whose sums with a tile's would pass 32 bits, and lens shifted over what the call reads."""
    big = 2**31 - 1
    w = K.GqaWindowArgs()
    w.base = _base(K, tokens_per_row=big, q_stride_t=0)
    assert lib.bz_gqa_window(ctypes.byref(w), None) == -2
    c = _cache(K)
    assert lib.bz_kv4_store(0x10000, 0x20000, 1024, 128, 1024, big, 0x30000, None, ctypes.byref(c), None) == -2
    c.capacity = big
    assert lib.bz_kv4_load(ctypes.byref(c), 0x30000, 1, 0x10000, 0x20000, 1024, 128, 1024, None) == -2
    a = K.KvSelectArgs()
    a.weights, a.seq_lens, a.index, a.lens = 0x70000, 0x30000, 0x80000, 0x90000
    a.batch, a.num_kv_heads, a.capacity, a.keep = 2, 8, big, 100
    assert lib.bz_kv_select(ctypes.byref(a), None) == -2
    a.capacity, a.lens = 4096, 0x30004
    assert lib.bz_kv_select(ctypes.byref(a), None) == -2
    a.lens, a.kv_start = 0x90000, 0x8fffc
    assert lib.bz_kv_select(ctypes.byref(a), None) == -2
    arr = (K.KvTensor * 4)()
    arr[0].src, arr[0].dst, arr[0].row_bytes = 0x100000, 0x900000, 256
    arr[0].src_stride_s = arr[0].dst_stride_s = 256
    assert lib.bz_kv_compact(arr, 1, 0x80000, 0x90000, 2, 8, big, 100, None) == -2


def test_workspace_size(lib, K):
    n = ctypes.c_size_t(0)
    size = lambda *a: lib.bz_long_workspace_size(*a, ctypes.byref(n))  # noqa: E731
    assert size(0, 2, 16, 8, 128, 4096, 1, 1024, 4, 8, 0) == 0 and n.value > 0
    assert size(0, 2, 16, 8, 128, 4096, 1, 1024, 4, 1, 0) == 0 and n.value == 0  # one split: nothing to merge
    assert size(2, 2, 16, 8, 128, 4096, 1, 0, 0, 1, 0) == 0 and n.value >= 2 * 16 * 4096 * 4  # the scores
    assert size(3, 2, 16, 8, 128, 4096, 1, 0, 0, 1, 0) == -2
    assert size(0, 2, 16, 8, 96, 4096, 1, 0, 0, 1, 0) == -3
    assert size(2, 2, 16, 8, 128, 2**31 - 1, 1, 0, 0, 1, 0) == -2
    assert size(0, 2, 16, 8, 128, 4096, 1, -1, 0, 1, 0) == -2
    assert lib.bz_long_workspace_size(0, 2, 16, 8, 128, 4096, 1, 0, 0, 1, 0, None) == -1


def test_python_refusals_on_cpu_tensors(pkg):
    q = torch.zeros(2, 16, 128, dtype=torch.bfloat16)
    k = torch.zeros(2, 8, 64, 128, dtype=torch.bfloat16)
    lens = torch.zeros(2, dtype=torch.int32)
    w = torch.zeros(2, 8, 64)
    cache = pkg.kv4_cache(2, 8, 64, 128, "cpu")
    assert [tuple(t.shape) for t in cache] == [(2, 8, 64, 64)] * 2 + [(2, 8, 64, 4)] * 2
    for call in (lambda: pkg.gqa_window(q, k, k, lens, 0.1, 8), lambda: pkg.gqa_decode_kv4(q, cache, lens, 0.1),
                 lambda: pkg.kv4_store(k, k, cache, lens), lambda: pkg.kv4_load(cache, lens, 1),
                 lambda: pkg.gqa_decode_tracked(q, k, k, lens, 0.1, w), lambda: pkg.kv_select(w, lens, 8),
                 lambda: pkg.kv_compact((k,), torch.zeros(2, 8, 8, dtype=torch.int32), lens),
                 lambda: pkg.kv4_cache(1, 1, 16, 96, "cpu"), lambda: pkg.long_workspace("other", torch.device("cuda", 0), 1, 1,
                                                                                        1, 64, 16)):
        with pytest.raises(RuntimeError):
            call()
