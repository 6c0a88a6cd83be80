"""include/bz_paged_cache.h on the CPU: struct layouts, the host-side checks' status codes, and Python refusals. No call here launches a
kernel (every case fails validation first)."""
import ctypes
import subprocess
from pathlib import Path

import pytest
import torch

REPO = Path(__file__).resolve().parents[1]
STRUCTS = {"bz_paged_cache": "PagedCacheArgs", "bz_rope": "RopeSpec", "bz_rope_args": "RopeArgs",
           "bz_paged_store_args": "PagedStoreArgs", "bz_gqa_paged_args": "GqaPagedArgs"}


@pytest.fixture(scope="module")
def lib(pkg):
    return pkg.load()


@pytest.fixture(scope="module")
def K(pkg):
    from breeze_tts_2_flash_amd import kernels
    return kernels


def test_struct_layouts_match_c(K, tmp_path):
    src = ["#include <stddef.h>", "#include <stdio.h>", '#include "bz_paged_cache.h"', "int main(void) {"]
    for c, py in STRUCTS.items():
        src.append(f'  printf("{c} %zu\\n", sizeof({c}));')
        src += [f'  printf("{c}.{f} %zu\\n", offsetof({c}, {f}));' for f, _ in getattr(K, py)._fields_]
    src += ["  return 0;", "}"]
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


def _cache(K, **over):
    """Plausible sizes with fake (never dereferenced) device addresses."""
    c = K.PagedCacheArgs()
    c.k, c.v, c.k_scale, c.v_scale = 0x100000, 0x200000, 0x300000, 0x400000
    c.stride_page, c.stride_h, c.stride_s = 8 * 64 * 128, 64 * 128, 128
    c.scale_stride_page, c.scale_stride_h = 8 * 64, 64
    c.pages, c.num_kv_heads, c.page_size, c.head_dim, c.bits = 40, 8, 64, 128, 8
    c.page_table, c.table_stride, c.batch, c.max_pages = 0x500000, 20, 2, 20
    c.seq_lens, c.q_start, c.tokens = 0x600000, 0x700000, 5
    for k, v in over.items():
        setattr(c, k, v)
    return c


CACHE = [
    (dict(k=None), -1), (dict(v=None), -1), (dict(page_table=None), -1), (dict(k_scale=None), -1), (dict(v_scale=None), -1),
    (dict(pages=0), -2), (dict(num_kv_heads=0), -2), (dict(batch=0), -2), (dict(max_pages=0), -2), (dict(max_pages=1 << 25), -2),
    (dict(stride_s=112), -2), (dict(stride_s=1 << 24), -2), (dict(bits=16), -2),
    (dict(page_size=8), -3), (dict(page_size=48), -3), (dict(page_size=2048), -3), (dict(head_dim=96), -3), (dict(bits=4), -3),
    (dict(k=0x100008), -4), (dict(stride_page=8 * 64 * 128 + 8), -4), (dict(stride_h=8200), -4), (dict(stride_s=136), -4),
    (dict(k_scale=0x300002), -4), (dict(scale_stride_h=66), -4), (dict(page_table=0x500002), -4),
]
ROWS = [(dict(seq_lens=None), -1), (dict(tokens=0), -2), (dict(tokens=(1 << 30) + 1), -2), (dict(q_start=None), -2),
        (dict(seq_lens=0x600001), -4), (dict(q_start=0x700002), -4)]


@pytest.mark.parametrize("over,status", CACHE + ROWS, ids=str)
def test_cache_checks(lib, K, over, status):
    c = _cache(K, **over)
    a = K.GqaPagedArgs(cache=c, q=0x10000, q_stride_t=2048, q_stride_h=128, out=0x20000, out_stride_t=2048, out_stride_h=128,
                       scale=0.1, num_q_heads=16, workspace=0x800000, workspace_bytes=1 << 40)
    assert lib.bz_gqa_paged(ctypes.byref(a), None) == status
    s = K.PagedStoreArgs(cache=c, k=0x10000, v=0x20000, k_stride_t=1024, k_stride_h=128, v_stride_t=1024, v_stride_h=128)
    assert lib.bz_paged_store(ctypes.byref(s), None) == status
    if (over, status) in CACHE:
        assert lib.bz_paged_load(ctypes.byref(c), 0x10000, 4, 0x20000, 0x30000, 8 * 4 * 128, 4 * 128, 128, None) == status


@pytest.mark.parametrize("over,status", [
    (dict(q=None), -1), (dict(out=None), -1), (dict(num_q_heads=12), -2), (dict(num_q_heads=0), -2), (dict(max_tokens=-1), -2),
    (dict(max_seq_len=-1), -2), (dict(num_q_heads=24), -3), (dict(num_q_heads=128), -3), (dict(q=0x10008), -4), (dict(q_stride_h=132), -4),
    (dict(out=0x20001), -4)], ids=str)
def test_attention_checks(lib, K, over, status):
    a = K.GqaPagedArgs(cache=_cache(K), q=0x10000, q_stride_t=2048, q_stride_h=128, out=0x20000, out_stride_t=2048, out_stride_h=128,
                       scale=0.1, num_q_heads=16, workspace=0x800000, workspace_bytes=1 << 40)
    for k, v in over.items():
        setattr(a, k, v)
    assert lib.bz_gqa_paged(ctypes.byref(a), None) == status
    assert lib.bz_gqa_paged(None, None) == -1


@pytest.mark.parametrize("over,rope,status", [
    (dict(k=None), {}, -1), (dict(v=None), {}, -1), (dict(q_out=None), {}, -1), (dict(k=0x10004), {}, -4), (dict(v_stride_h=129), {}, -4),
    (dict(q=0x30002), {}, -4), (dict(q_out_stride_t=4), {}, -4), (dict(k_norm_weight=0x40008), {}, -4), (dict(positions=0x50002), {}, -4),
    (dict(positions=0x50004, positions_64=1), {}, -4), (dict(q=None), {}, -2), (dict(num_q_heads=-1), {}, -2), (dict(num_q_heads=0), {}, -2),
    ({}, dict(inv_freq=None), -3), (dict(q=None, num_q_heads=0, k_norm_weight=0x40000), dict(inv_freq=None), -3),
    ({}, dict(rotary_dim=0), -2), ({}, dict(rotary_dim=24), -2), ({}, dict(rotary_dim=144), -2), ({}, dict(inv_freq=0x60004), -4)], ids=str)
def test_store_checks(lib, K, over, rope, status):
    s = K.PagedStoreArgs(cache=_cache(K), k=0x10000, v=0x20000, k_stride_t=1024, k_stride_h=128, v_stride_t=1024, v_stride_h=128,
                         q=0x30000, q_stride_t=2048, q_stride_h=128, q_out=0x38000, q_out_stride_t=2048, q_out_stride_h=128,
                         num_q_heads=16, eps=1e-6)
    s.rope = K.RopeSpec(inv_freq=0x60000, rotary_dim=128, factor=1.0)
    for k, v in over.items():
        setattr(s, k, v)
    for k, v in rope.items():
        setattr(s.rope, k, v)
    assert lib.bz_paged_store(ctypes.byref(s), None) == status
    assert lib.bz_paged_store(None, None) == -1


@pytest.mark.parametrize("over,status", [
    (dict(x=None), -1), (dict(out=None), -1), (dict(positions=None), -1), (dict(tokens=0), -2), (dict(heads=0), -2), (dict(head_dim=96), -3),
    (dict(x=0x10002), -4), (dict(x_stride_h=4), -4), (dict(out_stride_t=9), -4), (dict(positions=0x50002), -4),
    (dict(tokens=1 << 30, heads=1 << 10), -2), (dict(tokens=1 << 20, heads=1 << 10), -2)], ids=str)
def test_rope_checks(lib, K, over, status):
    a = K.RopeArgs(x=0x10000, x_stride_t=1024, x_stride_h=128, out=0x20000, out_stride_t=1024, out_stride_h=128, positions=0x50000,
                   tokens=3, heads=8, head_dim=128)
    a.rope = K.RopeSpec(inv_freq=0x60000, rotary_dim=64, factor=1.0)
    for k, v in over.items():
        setattr(a, k, v)
    assert lib.bz_rope_apply(ctypes.byref(a), None) == status
    assert lib.bz_rope_apply(None, None) == -1


def test_load_and_workspace_checks(lib, K):
    c = _cache(K)
    load = lambda starts=0x10000, n=4, k=0x20000, v=0x30000, st=128: lib.bz_paged_load(  # noqa: E731
        ctypes.byref(c), starts, n, k, v, 8 * 4 * 128, 4 * 128, st, None)
    assert [load(starts=None), load(k=None), load(v=None), load(n=0), load(k=0x20008), load(st=132), load(starts=0x10002)] == [-1, -1, -1, -2, -4, -4, -4]
    assert load(n=1 << 28) == -2  # 2^32 threads
    n = ctypes.c_size_t(0)
    size = lambda *a: lib.bz_paged_workspace_size(*a, ctypes.byref(n))  # noqa: E731
    assert [size(96, 2, 1), size(64, 3, 1), size(64, 2, -1), lib.bz_paged_workspace_size(64, 2, 1, None)] == [-3, -3, -2, -1]


def test_python_refusals_without_a_device(pkg):
    x = torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    f = pkg.rope_frequencies(64, 1e4, "cpu")
    cache = pkg.paged_cache(4, 4, 16, 64, "cpu", torch.float8_e4m3fn)
    table, lens = torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    for call in (lambda: pkg.rope(x, lens, f), lambda: pkg.paged_store(x, x, cache, table, lens), lambda: pkg.gqa_paged(x, cache, table, lens, 0.1),
                 lambda: pkg.rope_store(x, x, x, cache, table, lens, f), lambda: pkg.paged_load(cache, table, lens, 3),
                 lambda: pkg.rope(None, lens, f), lambda: pkg.paged_store(x, 3, cache, table, lens)):
        with pytest.raises(RuntimeError):
            call()
    assert cache.k.dtype == torch.float8_e4m3fn and (cache.k_scale == 127).all() and pkg.paged_cache(1, 1, 16, 128, "cpu").k_scale is None
