"""C ABI and host-side contract of the paged cache and its attention (no GPU needed)."""

import ctypes
import re
import subprocess
from pathlib import Path

import pytest
import torch

import b200_attention as b2
from b200_attention import _native
from b200_attention.build import LIB_PATH, build_native, build_torch_op

ROOT = Path(__file__).resolve().parents[1]
HEADER = ROOT / "include" / "b200_paged.h"


@pytest.fixture(scope="module")
def lib():
    build_native()
    build_torch_op()
    return _native.load_library()


def test_header_declarations_are_mirrored_and_exported(lib):
    names = re.findall(r"B200_ATTN_API\s+[\w\s\*]+?\b(b200_(?:cache|tree_attn)_\w+)\s*\(", HEADER.read_text())
    assert set(names) == set(_native.PAGED_SYMBOLS)
    out = subprocess.run(["nm", "-D", "--defined-only", str(LIB_PATH)], capture_output=True,
                         text=True, check=True).stdout
    assert set(names) <= set(re.findall(r"\bT\s+(b200_\w+)", out))


@pytest.mark.parametrize("c_name,mirror", [("b200_cache", _native.Cache),
                                           ("b200_cache_rows", _native.CacheRows),
                                           ("b200_tree_attn_params", _native.TreeAttnParams)])
def test_struct_layouts_match_c(tmp_path, c_name, mirror):
    fields = [f for f, _ in mirror._fields_]
    body = "\n".join(f'  printf("{f} %zu\\n", offsetof({c_name}, {f}));' for f in fields)
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "b200_paged.h"\n'
                   f'int main(void) {{\n  printf("size %zu\\n", sizeof({c_name}));\n'
                   f'  printf("batch_limit %d\\n", B200_CACHE_MAX_BATCH);\n{body}\n  return 0;\n}}\n')
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c11", f"-I{ROOT / 'include'}", str(src), "-o", str(exe)], check=True)
    lines = dict(l.split() for l in subprocess.run([str(exe)], capture_output=True, text=True,
                                                   check=True).stdout.splitlines())
    assert int(lines["size"]) == ctypes.sizeof(mirror)
    assert int(lines["batch_limit"]) == _native.CACHE_MAX_BATCH
    for f in fields:
        assert int(lines[f]) == getattr(mirror, f).offset, f


def cache(**kw):
    c = _native.Cache()
    c.k, c.v = 0x10000000, 0x100000000
    c.layers, c.pages, c.kv_heads, c.page_size, c.head_dim = 2, 100, 4, 16, 64
    for s in (c.k_stride, c.v_stride):
        s[:] = (100 * 4 * 16 * 64, 4 * 16 * 64, 16 * 64, 64)
    c.page_table, c.batch, c.slots, c.table_stride = 0x20000000, 3, 8, 8
    c.seq_lens, c.page_refs, c.dtype = 0x30000000, 0x40000000, _native.DTYPE_BF16
    for k, v in kw.items():
        if isinstance(v, tuple):
            getattr(c, k)[:] = v
        else:
            setattr(c, k, v)
    return c


OK, INVALID, UNSUPPORTED, ALIGNMENT = (_native.OK, _native.ERR_INVALID_ARGUMENT,
                                       _native.ERR_UNSUPPORTED, _native.ERR_ALIGNMENT)


@pytest.mark.parametrize("kw,code", [
    ({}, OK),
    (dict(head_dim=128, k_stride=(1 << 30, 8192, 2048, 128), v_stride=(1 << 30, 8192, 2048, 128)), OK),
    (dict(dtype=_native.DTYPE_FP32, head_dim=8), OK),
    (dict(page_size=1), OK),
    (dict(k=None), INVALID),
    (dict(page_table=None), INVALID),
    (dict(layers=0), INVALID),
    (dict(pages=0), INVALID),
    (dict(page_size=0), INVALID),
    (dict(batch=0), INVALID),
    (dict(batch=_native.CACHE_MAX_BATCH + 1), INVALID),
    (dict(slots=0), INVALID),
    (dict(slots=1 << 24, page_size=1 << 20, table_stride=1 << 24), INVALID),
    (dict(table_stride=7), INVALID),
    (dict(reserved=1), INVALID),
    (dict(head_dim=12), UNSUPPORTED),
    (dict(head_dim=136), UNSUPPORTED),
    (dict(dtype=9), UNSUPPORTED),
    (dict(k=0x10000008), ALIGNMENT),
    (dict(v_stride=(409600, 4096, 1024, 68)), ALIGNMENT),
    (dict(k_stride=(409600, 4096, -1024, 64)), ALIGNMENT),
    (dict(page_table=0x20000002), ALIGNMENT),
])
def test_cache_check(lib, kw, code):
    assert lib.b200_cache_check(ctypes.byref(cache(**kw))) == code


def test_operations_refuse_before_any_launch(lib):
    c, p = cache(), ctypes.c_void_p
    rows = _native.CacheRows()
    rows.k, rows.v, rows.tokens = 0x50000000, 0x60000000, 5
    for s in (rows.k_stride, rows.v_stride):
        s[:] = (3 * 4 * 5 * 64, 4 * 5 * 64, 5 * 64, 64)
    ref = ctypes.byref

    def append(cc=c, **kw):
        r = _native.CacheRows.from_buffer_copy(rows)
        for k, v in kw.items():
            setattr(r, k, v)
        return lib.b200_cache_append(ref(cc), ref(r), None)

    assert append(k=None) == INVALID and append(tokens=0) == INVALID
    assert append(k=0x50000004) == ALIGNMENT and append(counts=0x70000001) == ALIGNMENT
    assert append(k=0x10000400) == INVALID  # rows inside the pool
    assert append(cache(seq_lens=None)) == INVALID
    assert lib.b200_cache_append(ref(c), None, None) == INVALID
    accept = lambda paths, width, counts, out: lib.b200_cache_accept(  # noqa: E731
        ref(c), p(paths), width, width, p(counts), p(out), None)
    assert accept(None, 4, 0x700, 0x800) == INVALID and accept(0x600, 0, 0x700, 0x800) == INVALID
    assert accept(0x600, 4, 0x700, 0x30000000) == INVALID  # new lengths over the old ones
    assert accept(0x601, 4, 0x700, 0x800) == ALIGNMENT
    size = lib.b200_cache_workspace_bytes(ref(c))
    assert size > 0 and lib.b200_cache_workspace_bytes(ref(cache(batch=0))) == 0
    reserve = lambda cc, n, ws, bytes_: lib.b200_cache_reserve(  # noqa: E731
        ref(cc), None, n, p(0x900), p(ws), bytes_, None)
    assert reserve(c, -1, 0xa00, size) == INVALID
    assert reserve(c, 1, 0xa00, size - 1) == INVALID and reserve(c, 1, None, size) == INVALID
    assert reserve(c, 1, 0xa08, size) == ALIGNMENT
    assert reserve(cache(page_refs=None), 1, 0xa00, size) == INVALID
    fork = lambda n: lib.b200_cache_fork(ref(c), p(0x600), p(0x700), n, None)  # noqa: E731
    assert fork(-1) == INVALID and fork(4) == INVALID and fork(0) == OK
    assert lib.b200_cache_free(ref(c), None, 1, None) == INVALID
    assert lib.b200_cache_free(ref(c), None, 0, None) == OK
    assert lib.b200_cache_compact(ref(c), None, p(0xa00), size, None) == INVALID


def attn(cache_kw=None, **kw):
    t = _native.TreeAttnParams()
    t.cache = cache(layers=1, **(cache_kw or {}))
    t.q, t.o, t.heads, t.tokens, t.scale = 0x70000000, 0x80000000, 8, 5, 0.125
    for s in (t.q_stride, t.o_stride):
        s[:] = (8 * 5 * 64, 5 * 64, 64)
    for k, v in kw.items():
        if isinstance(v, tuple):
            getattr(t, k)[:] = v
        else:
            setattr(t, k, v)
    return t


@pytest.mark.parametrize("kw,code", [
    ({}, OK),
    (dict(tokens=300, heads=4), OK),
    (dict(mask=0x90000000, mask_stride=(25, 5, 1)), OK),
    (dict(mask=0x90000000, mask_stride=(0, 5, 1)), OK),
    (dict(cache_kw=dict(page_size=7)), OK),
    (dict(q=None), INVALID),
    (dict(o=None), INVALID),
    (dict(tokens=0), INVALID),
    (dict(heads=6), INVALID),
    (dict(heads=0), INVALID),
    (dict(scale=0.0), INVALID),
    (dict(scale=float("nan")), INVALID),
    (dict(scale=float("inf")), INVALID),
    (dict(reserved=1), INVALID),
    (dict(mask=0x90000000, mask_stride=(25, -5, 1)), INVALID),
    (dict(tokens=1 << 24), INVALID),
    (dict(cache_kw=dict(seq_lens=None)), INVALID),
    (dict(q=0x70000004), ALIGNMENT),
    (dict(o_stride=(8 * 5 * 64, 5 * 64, 60)), ALIGNMENT),
    (dict(draft_lens=0x90000001), ALIGNMENT),
    (dict(counters=0x90000002), ALIGNMENT),
    (dict(cache_kw=dict(head_dim=132)), UNSUPPORTED),
])
def test_attention_check(lib, kw, code):
    t = attn(**kw)
    assert lib.b200_tree_attn_check(ctypes.byref(t)) == code
    size = lib.b200_tree_attn_workspace_bytes(ctypes.byref(t))
    assert (size > 0) == (code == OK)
    if code == OK:
        t.workspace, t.workspace_bytes = 0xa0000000, size - 1
        assert lib.b200_tree_attn_fwd(ctypes.byref(t), None) == INVALID
        t.workspace, t.workspace_bytes = 0xa0000008, size
        assert lib.b200_tree_attn_fwd(ctypes.byref(t), None) == ALIGNMENT


def test_one_layer_only(lib):
    t = attn()
    t.cache.layers = 2
    assert lib.b200_tree_attn_check(ctypes.byref(t)) == INVALID


def tensors():
    i32 = torch.int32
    return dict(k=torch.zeros(2, 9, 2, 4, 16), v=torch.zeros(2, 9, 2, 4, 16),
                table=torch.zeros(3, 5, dtype=i32), lens=torch.zeros(3, dtype=i32),
                refs=torch.zeros(9, dtype=i32))


def test_python_entry_points_refuse_cpu_tensors_and_bad_types(lib):
    t = tensors()
    k_new = torch.zeros(2, 3, 2, 1, 16)
    with pytest.raises(ValueError, match="CUDA"):
        b2.b200_cache_append(k_new, k_new, t["k"], t["v"], t["table"], t["lens"])
    with pytest.raises(ValueError, match="CUDA"):
        b2.b200_cache_reserve(t["k"], t["v"], t["table"], t["lens"], t["refs"], 1)
    with pytest.raises(ValueError, match="CUDA"):
        b2.b200_cache_fork(t["table"], t["lens"], t["refs"], t["lens"][:1], t["lens"][1:2], 4)
    with pytest.raises(ValueError, match="CUDA"):
        b2.b200_cache_free(t["table"], t["lens"], t["refs"], t["lens"][:1])
    with pytest.raises(ValueError, match="CUDA"):
        b2.b200_cache_compact(t["k"], t["v"], t["table"], t["refs"])
    with pytest.raises(ValueError, match="CUDA"):
        b2.b200_cache_accept(t["k"], t["v"], t["table"], t["lens"], t["table"], t["lens"])
    with pytest.raises(ValueError, match="CUDA"):
        b2.b200_tree_attention(torch.zeros(3, 2, 1, 16), t["k"][0], t["v"][0], t["table"], t["lens"])
    with pytest.raises(TypeError, match="int32"):
        b2.b200_cache_free(t["table"].long(), t["lens"], t["refs"], t["lens"][:1])
    with pytest.raises(TypeError, match="dtype"):
        b2.b200_cache_reserve(t["k"], t["v"].half(), t["table"], t["lens"], t["refs"], 1)
    with pytest.raises(ValueError, match="shape"):
        b2.b200_cache_reserve(t["k"][0, 0], t["v"][0, 0], t["table"], t["lens"], t["refs"], 1)
    with pytest.raises(ValueError, match="positive"):
        b2.PagedKVCache(1, 0, 1, 16, 64, 1, 1, device="cpu")
