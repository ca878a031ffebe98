"""C ABI and host-side contract of the 4-bit cache and of the check of drafted tokens (no GPU
needed)."""

import ctypes
import re
import subprocess
from pathlib import Path

import pytest
import torch

import b200_attention as b2
from b200_attention import _native
from b200_attention.build import LIB_PATH, build_native, build_torch_op
from cache4_reference import quantise

ROOT = Path(__file__).resolve().parents[1]
OK, INVALID, UNSUPPORTED, ALIGNMENT = (_native.OK, _native.ERR_INVALID_ARGUMENT,
                                       _native.ERR_UNSUPPORTED, _native.ERR_ALIGNMENT)
BF16, FP16, FP32 = _native.DTYPE_BF16, _native.DTYPE_FP16, _native.DTYPE_FP32


@pytest.fixture(scope="module")
def lib():
    build_native()
    build_torch_op()
    return _native.load_library()


@pytest.mark.parametrize("header,symbols", [("b200_cache4.h", _native.CACHE4_SYMBOLS),
                                            ("b200_verify.h", _native.VERIFY_SYMBOLS)])
def test_header_declarations_are_mirrored_and_exported(lib, header, symbols):
    text = (ROOT / "include" / header).read_text()
    names = re.findall(r"B200_ATTN_API\s+[\w\s\*]+?\b(b200_(?:cache4|verify)_\w+)\s*\(", text)
    assert set(names) == set(symbols)
    out = subprocess.run(["nm", "-D", "--defined-only", str(LIB_PATH)], capture_output=True,
                         text=True, check=True).stdout
    assert set(names) <= set(re.findall(r"\bT\s+(b200_\w+)", out))


def test_struct_layout_matches_c(tmp_path):
    fields = [f for f, _ in _native.VerifyParams._fields_]
    body = "\n".join(f'  printf("{f} %zu\\n", offsetof(b200_verify_params, {f}));' for f in fields)
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "b200_verify.h"\n#include "b200_cache4.h"\n'
                   'int main(void) {\n  printf("size %zu\\n", sizeof(b200_verify_params));\n'
                   '  printf("most_nodes %d\\n", B200_VERIFY_MAX_NODES);\n'
                   f'  printf("most_vocab %d\\n", B200_VERIFY_MAX_VOCAB);\n{body}\n  return 0;\n}}\n')
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c11", f"-I{ROOT / 'include'}", str(src), "-o", str(exe)], check=True)
    lines = dict(l.split() for l in subprocess.run([str(exe)], capture_output=True, text=True,
                                                   check=True).stdout.splitlines())
    assert int(lines["size"]) == ctypes.sizeof(_native.VerifyParams)
    assert int(lines["most_nodes"]) == _native.VERIFY_MAX_NODES
    assert int(lines["most_vocab"]) == _native.VERIFY_MAX_VOCAB
    for f in fields:
        assert int(lines[f]) == getattr(_native.VerifyParams, f).offset, f


def test_row_bytes(lib):
    assert [lib.b200_cache4_row_bytes(d) for d in (8, 40, 64, 72, 128)] == [48, 48, 48, 80, 80]
    assert [lib.b200_cache4_row_bytes(d) for d in (0, -8, 7, 12, 136, 1 << 40)] == [0] * 6


def cache(**kw):
    c = _native.Cache()
    c.k, c.v = 0x10000000, 0x100000000
    c.layers, c.pages, c.kv_heads, c.page_size, c.head_dim = 1, 100, 4, 16, 24
    for s in (c.k_stride, c.v_stride):
        s[:] = (100 * 4 * 16 * 24, 4 * 16 * 24, 16 * 24, 24)
    c.page_table, c.batch, c.slots, c.table_stride = 0x20000000, 3, 8, 8
    c.seq_lens, c.page_refs, c.dtype = 0x30000000, 0x40000000, BF16
    return change(c, kw)


def change(c, kw):
    for k, v in kw.items():
        if isinstance(v, tuple):
            getattr(c, k)[:] = v
        else:
            setattr(c, k, v)
    return c


def test_rows_in_and_out_refuse_before_any_launch(lib):
    def call(entry, head_dim=64, dtype=BF16, cc=None, **kw):
        r = _native.CacheRows()
        r.k, r.v, r.tokens = 0x500000000, 0x600000000, 5
        for s in (r.k_stride, r.v_stride):
            s[:] = (3 * 4 * 5 * 64, 4 * 5 * 64, 5 * 64, 64)
        return entry(ctypes.byref(cc or cache()), head_dim, dtype, ctypes.byref(change(r, kw)), None)

    for entry in (lib.b200_cache4_append, lib.b200_cache4_read):
        assert call(entry, 60) == UNSUPPORTED and call(entry, 64, 7) == UNSUPPORTED
        assert call(entry, 72) == INVALID                       # rows of 80 bytes
        assert call(entry, cc=cache(head_dim=32)) == INVALID    # a pool of another kind
        assert call(entry, cc=cache(dtype=FP32)) == INVALID
        assert call(entry, cc=cache(seq_lens=None)) == INVALID
        assert call(entry, cc=cache(batch=0)) == INVALID
        assert call(entry, k=None) == INVALID and call(entry, tokens=0) == INVALID
        assert call(entry, tokens=1 << 30) == INVALID
        assert call(entry, k=0x500000008) == ALIGNMENT
        assert call(entry, v_stride=(0, 1280, 320, 60)) == ALIGNMENT
        assert call(entry, counts=0x700000001) == ALIGNMENT
        assert call(entry, k=0x10000400) == INVALID             # rows inside the pool
        assert entry(ctypes.byref(cache()), 64, BF16, None, None) == INVALID
    assert call(lib.b200_cache4_read, v=0x500000000) == INVALID  # both outputs in one place
    assert call(lib.b200_cache4_read, k_stride=(0, 0, 320, 64)) == INVALID
    assert call(lib.b200_cache4_read, k=0x30000000) == INVALID   # over the lengths
    assert call(lib.b200_cache4_read, counts=0x500000010) == INVALID


def attn(cache_kw=None, **kw):
    t = _native.TreeAttnParams()
    t.cache = cache(**(cache_kw or {}))
    t.q, t.o, t.heads, t.tokens, t.scale = 0x70000000, 0x80000000, 8, 5, 0.125
    for s in (t.q_stride, t.o_stride):
        s[:] = (8 * 5 * 64, 5 * 64, 64)
    return change(t, kw)


@pytest.mark.parametrize("kw,code", [
    ({}, OK),
    (dict(tokens=300, heads=4, q_stride=(4 * 300 * 64, 300 * 64, 64), o_stride=(4 * 300 * 64, 300 * 64, 64)), OK),
    (dict(mask=0x90000000, mask_stride=(25, 5, 1)), OK),
    (dict(cache_kw=dict(page_size=7)), OK),
    (dict(o=0x70000000), OK),               # in the queries' place
    (dict(o=0x70000010), INVALID),          # beside it
    (dict(o=0x10000000), INVALID),          # over the pool
    (dict(o_stride=(8 * 5 * 64, 0, 64)), INVALID),
    (dict(q=None), INVALID),
    (dict(tokens=0), INVALID),
    (dict(heads=6), INVALID),
    (dict(scale=0.0), INVALID),
    (dict(scale=float("inf")), INVALID),
    (dict(reserved=1), INVALID),
    (dict(mask=0x90000000, mask_stride=(25, -5, 1)), INVALID),
    (dict(cache_kw=dict(seq_lens=None)), INVALID),
    (dict(cache_kw=dict(layers=2)), INVALID),
    (dict(cache_kw=dict(head_dim=40)), INVALID),
    (dict(cache_kw=dict(dtype=FP16)), INVALID),
    (dict(q=0x70000004), ALIGNMENT),
    (dict(o_stride=(8 * 5 * 64, 5 * 64, 60)), ALIGNMENT),
    (dict(draft_lens=0x90000001), ALIGNMENT),
    (dict(cache_kw=dict(k=0x10000008)), ALIGNMENT),
])
def test_attention_check(lib, kw, code):
    t = attn(**kw)
    assert lib.b200_cache4_attn_check(ctypes.byref(t), 64, BF16) == code
    size = lib.b200_cache4_attn_workspace_bytes(ctypes.byref(t), 64, BF16)
    assert (size > 0) == (code == OK)
    if code == OK:
        t.workspace, t.workspace_bytes = 0xa0000000, size - 1
        assert lib.b200_cache4_attn_fwd(ctypes.byref(t), 64, BF16, None) == INVALID
        t.workspace, t.workspace_bytes = 0xa0000008, size
        assert lib.b200_cache4_attn_fwd(ctypes.byref(t), 64, BF16, None) == ALIGNMENT


def test_attention_types(lib):
    t = ctypes.byref(attn())
    assert lib.b200_cache4_attn_check(t, 64, FP16) == OK
    assert lib.b200_cache4_attn_check(t, 64, FP32) == UNSUPPORTED
    assert lib.b200_cache4_attn_check(t, 60, BF16) == UNSUPPORTED
    assert lib.b200_cache4_attn_check(t, 128, BF16) == INVALID
    assert lib.b200_cache4_attn_check(None, 64, BF16) == INVALID


def verify(**kw):
    p = _native.VerifyParams()
    p.logits, p.draft_probs, p.tokens, p.uniforms = 0x100000000, 0x200000000, 0x300000000, 0x400000000
    p.parents, p.draft_lens = 0x500000000, 0x600000000
    p.paths, p.counts, p.next = 0x700000000, 0x800000000, 0x900000000
    p.batch, p.nodes, p.vocab, p.temperature = 4, 6, 1001, 1.0
    p.logits_stride[:], p.draft_stride[:] = (6 * 1001, 1001), (5 * 1001, 1001)
    p.token_stride = p.uniform_stride = p.parent_stride = 6
    p.dtype, p.draft_dtype, p.wide_tokens = FP32, FP32, 1
    return change(p, kw)


@pytest.mark.parametrize("kw,code", [
    ({}, OK),
    (dict(draft_probs=None, parents=None, draft_lens=None, temperature=0.0, wide_tokens=0), OK),
    (dict(parent_stride=0), OK),
    (dict(nodes=1), OK),
    (dict(dtype=BF16, draft_dtype=FP16, logits=0x100000002), OK),
    (dict(logits=None), INVALID),
    (dict(tokens=None), INVALID),
    (dict(uniforms=None), INVALID),
    (dict(paths=None), INVALID),
    (dict(next=None), INVALID),
    (dict(batch=0), INVALID),
    (dict(batch=65536), INVALID),
    (dict(nodes=0), INVALID),
    (dict(nodes=1025), INVALID),
    (dict(vocab=0), INVALID),
    (dict(vocab=(1 << 24) + 1), INVALID),
    (dict(temperature=-1.0), INVALID),
    (dict(temperature=float("nan")), INVALID),
    (dict(temperature=float("inf")), INVALID),
    (dict(temperature=5e-324), INVALID),
    (dict(reserved=1), INVALID),
    (dict(wide_tokens=2), INVALID),
    (dict(logits_stride=(-1, 1001)), INVALID),
    (dict(token_stride=-6), INVALID),
    (dict(paths=0x100000100), INVALID),   # over the logits
    (dict(counts=0x200000100), INVALID),
    (dict(next=0x700000000), INVALID),    # over the paths
    (dict(paths=0x600000000), INVALID),
    (dict(dtype=5), UNSUPPORTED),
    (dict(draft_dtype=-1), UNSUPPORTED),
    (dict(logits=0x100000002), ALIGNMENT),
    (dict(tokens=0x300000004), ALIGNMENT),
    (dict(next=0x900000004), ALIGNMENT),
    (dict(uniforms=0x400000001), ALIGNMENT),
])
def test_verify_check(lib, kw, code):
    assert lib.b200_verify_check(ctypes.byref(verify(**kw))) == code
    if code != OK:
        assert lib.b200_verify_drafts(ctypes.byref(verify(**kw)), None) == code


def test_python_entry_points_refuse(lib):
    i32 = torch.int32
    pool = torch.zeros(2, 9, 2, 4, 48, dtype=torch.uint8)
    table, lens = torch.zeros(3, 5, dtype=i32), torch.zeros(3, dtype=i32)
    x = torch.zeros(2, 3, 2, 1, 16)
    with pytest.raises(ValueError, match="CUDA"):
        b2.b200_cache_append(x, x, pool, pool, table, lens)
    with pytest.raises(ValueError, match="CUDA"):
        b2.b200_cache_read(pool, pool, table, lens, 1, 16)
    with pytest.raises(TypeError, match="4-bit"):
        b2.b200_cache_read(pool.half(), pool.half(), table, lens, 1, 16)
    with pytest.raises(TypeError, match="uint8"):
        b2.b200_cache_append(x, x, pool.int(), pool.int(), table, lens)
    with pytest.raises(ValueError, match="CUDA"):
        b2.b200_verify_drafts(torch.zeros(1, 2, 9), torch.zeros(1, 2, dtype=torch.int64), torch.zeros(1, 2))
    with pytest.raises(ValueError, match="shape"):
        b2.b200_verify_drafts(torch.zeros(2, 9), torch.zeros(1, 2, dtype=torch.int64), torch.zeros(1, 2))


def test_cache_of_4_bits():
    c = b2.PagedKVCache(2, 5, 3, 16, 40, 2, 4, dtype=torch.float16, device="cpu", bits=4)
    assert c.k_pages.shape == (2, 5, 3, 16, 48) and c.k_pages.dtype == torch.uint8
    assert c.page_size == 16 and c.head_dim == 40 and c.dtype == torch.float16
    assert b2.PagedKVCache(1, 1, 1, 16, 72, 1, 1, device="cpu", bits=4).v_pages.shape[-1] == 80
    with pytest.raises(ValueError, match="bits"):
        b2.PagedKVCache(1, 1, 1, 16, 64, 1, 1, device="cpu", bits=8)
    for d in (12, 136):
        with pytest.raises(ValueError, match="head_dim"):
            b2.PagedKVCache(1, 1, 1, 16, d, 1, 1, device="cpu", bits=4)


def test_the_format_is_within_half_a_step():
    x = torch.randn(50, 96, generator=torch.Generator().manual_seed(0)) + 5
    value, step = quantise(x)
    assert ((value - x.double()).abs() <= step / 2 + 1e-15).all() and (step < 0.5).all()
