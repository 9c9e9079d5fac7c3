"""The paged cache's C ABI without a GPU: exports, the ctypes mirrors' layout, what each
entry point refuses before any launch, workspace sizes, and the Python checks."""
import ctypes
import os
import re
import shutil
import subprocess

import numpy as np
import pytest

from mugen_amd import _capi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "mugen_attn_paged.h")
STRUCTS = {
    "KvPages": "mugen_attn_kv_pages",
    "KvPagedAppendArgs": "mugen_attn_kv_paged_append_args",
    "GqaDecodePagedArgs": "mugen_attn_gqa_decode_paged_args",
    "PageSelectArgs": "mugen_attn_page_select_args",
    "GqaPrefillPagedArgs": "mugen_attn_gqa_prefill_paged_args",
}


def test_exports_and_structs_are_mirrored():
    src = open(HEADER).read()
    assert set(re.findall(r"typedef struct (\w+) \{", src)) == set(STRUCTS.values())
    src = re.sub(r"/\*.*?\*/", "", src, flags=re.S)
    declared = sorted(set(re.findall(r"\b(mugen_attn_\w+)\s*\(", src)))
    assert declared == sorted(_capi.EXPORTS_PAGED)
    for name in declared:
        assert hasattr(_capi.lib(), name)
    assert f"#define MUGEN_ATTN_PAGED_MAX_Q {_capi.PAGED_MAX_Q}" in src


def test_struct_layout(tmp_path):
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no host C compiler")
    lines = ["#include <stddef.h>", "#include <stdio.h>", '#include "mugen_attn_paged.h"', "int main(void) {"]
    for py, c in STRUCTS.items():
        lines.append(f'  printf("{py} sizeof %zu\\n", sizeof({c}));')
        for name, _ in getattr(_capi, py)._fields_:
            lines.append(f'  printf("{py} {name} %zu\\n", offsetof({c}, {name}));')
    (tmp_path / "layout.c").write_text("\n".join(lines + ["  return 0;", "}"]) + "\n")
    exe = str(tmp_path / "layout")
    subprocess.run([cc, "-std=c11", "-I", os.path.join(ROOT, "include"), str(tmp_path / "layout.c"), "-o", exe], check=True)
    for line in subprocess.run([exe], check=True, capture_output=True, text=True).stdout.splitlines():
        py, field, at = line.split()
        cls = getattr(_capi, py)
        assert int(at) == (ctypes.sizeof(cls) if field == "sizeof" else getattr(cls, field).offset), line


def store(**kw):
    s = _capi.KvPages()
    s.k_pages = s.v_pages = s.k_exp = s.v_exp = s.tail_k = s.tail_v = s.k_range = s.page_table = 0x1000
    s.n_seq, s.n_pages, s.page_tokens, s.page_bits, s.ring = 2, 64, 64, 8, 128
    s.n_kv_heads, s.head_dim, s.max_seq_len, s.dtype = 4, 128, 4096, _capi.F16
    s.table_stride, s.tail_seq_stride = 64, 128 * 4 * 128
    for k, v in kw.items():
        setattr(s, k, v)
    return s


def make(cls, **kw):
    a = cls()
    a.store = store(**{k[2:]: v for k, v in kw.items() if k.startswith("s_")})
    a.n_heads = 28
    if cls is _capi.KvPagedAppendArgs:
        a.k_new = a.v_new = a.q = a.q_out = a.seq_lens = 0x1000
        a.k_stride = a.v_stride = 512
        a.q_stride, a.n_new, a.rope_dim = 28 * 128, 3, 128
        a.rope = _capi.RopeParams(1e4, 1.0, 0)
    elif cls is _capi.GqaDecodePagedArgs:
        a.q = a.out = a.seq_lens = 0x1000
        a.q_len, a.out_dtype = 1, _capi.F16
    elif cls is _capi.PageSelectArgs:
        a.q = a.pages = a.seq_lens = 0x1000
        a.q_len, a.n_select, a.n_first, a.n_last = 1, 8, 1, 2
    else:
        a.q = a.out = 0x1000
        a.n_tokens, a.start_pos, a.out_dtype = 100, 50, _capi.F16
    for k, v in kw.items():
        if not k.startswith("s_"):
            setattr(a, k, v)
    return a


def call(a, ws=None, nbytes=0):
    L = _capi.lib()
    if isinstance(a, _capi.KvPagedAppendArgs):
        return L.mugen_attn_kv_paged_append(ctypes.byref(a), None)
    name = {_capi.GqaDecodePagedArgs: "gqa_decode_paged", _capi.PageSelectArgs: "page_select",
            _capi.GqaPrefillPagedArgs: "gqa_prefill_paged"}[type(a)]
    return getattr(L, f"mugen_attn_{name}")(ctypes.byref(a), ws, nbytes, None)


ALL = [_capi.KvPagedAppendArgs, _capi.GqaDecodePagedArgs, _capi.PageSelectArgs, _capi.GqaPrefillPagedArgs]
I, U = _capi.E_INVALID, _capi.E_UNSUPPORTED


@pytest.mark.parametrize("cls", ALL)
@pytest.mark.parametrize("kw,code", [
    (dict(s_n_seq=0), I), (dict(s_n_pages=0), I), (dict(s_n_kv_heads=0), I), (dict(s_max_seq_len=0), I),
    (dict(s_head_dim=96), U), (dict(s_page_tokens=16), U), (dict(s_page_tokens=48), U), (dict(s_page_bits=4), U),
    (dict(s_dtype=_capi.F32), U), (dict(s_page_table=0), I), (dict(s_table_stride=63), I), (dict(s_k_range=0x1008), I),
    (dict(s_max_seq_len=2 ** 27 + 1, s_table_stride=2 ** 22), U), (dict(n_heads=30), I), (dict(n_heads=68), U), (dict(n_heads=0), I),
])
def test_refusals_of_the_store(cls, kw, code):
    assert call(make(cls, **kw), 0x1000, 1 << 40) == code
    assert _capi.lib().mugen_attn_last_error().decode()


@pytest.mark.parametrize("cls", [c for c in ALL if c is not _capi.PageSelectArgs])
@pytest.mark.parametrize("kw", [dict(s_k_pages=0), dict(s_v_pages=0), dict(s_k_pages=0x1008), dict(s_k_exp=0), dict(s_v_exp=0),
                                dict(s_tail_k=0), dict(s_tail_v=0x1004), dict(s_ring=64), dict(s_ring=192), dict(s_ring=0),
                                dict(s_tail_seq_stride=128 * 512 - 8), dict(s_tail_seq_stride=128 * 512 + 4)])
def test_refusals_of_the_8bit_store(cls, kw):
    assert call(make(cls, **kw), 0x1000, 1 << 40) == I


@pytest.mark.parametrize("kw,code", [
    (dict(n_new=-1), I), (dict(k_new=0), I), (dict(v_new=0x1002), I), (dict(k_stride=516), I), (dict(v_stride=504), I),
    (dict(seq_lens=0), I), (dict(seq_lens_out=0x1000), I), (dict(q_out=0), I), (dict(q=0x1008), I), (dict(q_stride=28 * 128 - 8), I),
    (dict(rope_dim=136), U), (dict(rope_dim=24), U), (dict(rope_dim=-16), U), (dict(n_new=0, seq_lens_out=0x2000), I),
    (dict(rope=_capi.RopeParams(0.0, 1.0, 0)), I), (dict(rope=_capi.RopeParams(float("nan"), 1.0, 0)), I),
    (dict(rope=_capi.RopeParams(1.0, 4.0, 4096)), I), (dict(rope=_capi.RopeParams(1e4, 4.0, 0)), I), (dict(n_new=2 ** 24), U),
])
def test_append_refusals(kw, code):
    assert call(make(_capi.KvPagedAppendArgs, **kw)) == code


def test_refusals_of_too_large_launches():
    """2^32 threads and more: 134 million page jobs, 5 million work items of 768 threads."""
    big = dict(s_n_seq=65535, s_n_kv_heads=1024, s_tail_seq_stride=128 * 1024 * 128)
    assert call(make(_capi.KvPagedAppendArgs, n_new=1, q=0, k_stride=1024 * 128, v_stride=1024 * 128, **big)) == U
    big = dict(s_n_seq=5000, s_n_kv_heads=1000, s_tail_seq_stride=128 * 1000 * 128)
    assert call(make(_capi.GqaDecodePagedArgs, n_heads=16000, q_len=3, **big), 0x1000, 1 << 60) == U


def test_append_of_nothing():
    assert call(make(_capi.KvPagedAppendArgs, n_new=0)) == _capi.OK
    # a call without tokens checks the store and the rotation all the same
    assert call(make(_capi.KvPagedAppendArgs, n_new=0, rope_dim=136)) == U


@pytest.mark.parametrize("kw,code", [
    (dict(q=0), I), (dict(out=0), I), (dict(seq_lens=0), I), (dict(q=0x1008), I), (dict(out=0x1008), I), (dict(q_len=0), U), (dict(q_len=65), U),
    (dict(num_splits=-1), I), (dict(num_splits=129), I), (dict(out_dtype=7), U), (dict(pages=0x1000, n_select=0), I),
    (dict(scale=float("nan")), I), (dict(scale=float("inf")), I),
])
def test_decode_refusals(kw, code):
    a = make(_capi.GqaDecodePagedArgs, **kw)
    assert call(a, 0x1000, 1 << 40) == code
    assert _capi.lib().mugen_attn_gqa_decode_paged_workspace_size(ctypes.byref(a)) == 0


@pytest.mark.parametrize("kw,code", [
    (dict(s_k_range=0), I), (dict(q=0), I), (dict(pages=0), I), (dict(seq_lens=0), I), (dict(q_len=65), U), (dict(n_first=-1), I),
    (dict(n_last=0), I), (dict(n_select=0), I), (dict(n_first=7), I), (dict(n_first=2 ** 31 - 1), I),
    (dict(s_max_seq_len=64 * 16384 + 1, s_table_stride=16385), U),
])
def test_select_refusals(kw, code):
    a = make(_capi.PageSelectArgs, **kw)
    assert call(a, 0x1000, 1 << 40) == code
    assert _capi.lib().mugen_attn_page_select_workspace_size(ctypes.byref(a)) == 0


@pytest.mark.parametrize("kw,code", [
    (dict(q=0), I), (dict(out=0x1008), I), (dict(seq=2), I), (dict(seq=-1), I), (dict(n_tokens=-1), I), (dict(start_pos=-1), I),
    (dict(start_pos=3997), I), (dict(start_pos=2 ** 31 - 1), I), (dict(out_dtype=9), U), (dict(scale=float("nan")), I),
])
def test_prefill_refusals(kw, code):
    a = make(_capi.GqaPrefillPagedArgs, **kw)
    assert call(a, 0x1000, 1 << 40) == code
    assert _capi.lib().mugen_attn_gqa_prefill_paged_workspace_size(ctypes.byref(a)) == 0


def test_null_arguments():
    L = _capi.lib()
    for rc in (L.mugen_attn_kv_paged_append(None, None), L.mugen_attn_gqa_decode_paged(None, None, 0, None),
               L.mugen_attn_page_select(None, None, 0, None), L.mugen_attn_gqa_prefill_paged(None, None, 0, None)):
        assert rc == I


@pytest.mark.parametrize("cls", ALL[1:])
def test_a_workspace_is_asked_for(cls):
    a = make(cls)
    if cls is _capi.GqaPrefillPagedArgs:
        assert call(make(cls, n_tokens=0)) == _capi.OK
    assert call(a) == _capi.E_WORKSPACE
    assert call(a, 0x1000, 16) == _capi.E_WORKSPACE
    assert "workspace of" in _capi.lib().mugen_attn_last_error().decode()


@pytest.mark.parametrize("q_len,pages,heads", [(1, 0, 28), (5, 0, 28), (1, 64, 28), (3, 7, 4), (64, 0, 4)])
def test_a_workspace_asked_for_without_lengths_covers_every_copy(q_len, pages, heads):
    rng = np.random.default_rng(q_len)
    L = _capi.lib()
    for B in (1, 2, 7, 40, 300):
        for T in (64, 1000, 20000, 131072):
            kw = dict(q_len=q_len, n_heads=heads, s_n_seq=B, s_max_seq_len=T, s_table_stride=T // 64 + 1)
            if pages:
                kw.update(pages=0x1000, n_select=pages)
            a = make(_capi.GqaDecodePagedArgs, **kw)
            bound = L.mugen_attn_gqa_decode_paged_workspace_size(ctypes.byref(a))
            for lens in ([T] * B, [0] * B, rng.integers(0, T + 1, B), [T] + [1] * (B - 1), [2 ** 31 - 1] + [-5] * (B - 1)):
                host = np.ascontiguousarray(lens, dtype=np.int32)
                a.seq_lens_host = host.ctypes.data
                assert L.mugen_attn_gqa_decode_paged_workspace_size(ctypes.byref(a)) <= bound


def splits(lens, H=28, Hk=4, D=128, bits=8, q_len=1, n_select=0, cache=16384):
    """The plan's splits, from its workspace size (0: one, no partials)."""
    host = np.ascontiguousarray(lens, np.int32)
    a = make(_capi.GqaDecodePagedArgs, q_len=q_len, n_heads=H, s_n_seq=len(host), s_n_kv_heads=Hk, s_head_dim=D, s_page_bits=bits,
             s_max_seq_len=cache, s_table_stride=cache // 64, s_tail_seq_stride=128 * Hk * D)
    a.seq_lens_host = host.ctypes.data
    if n_select:
        a.pages, a.n_select = 0x1000, n_select
    size = _capi.lib().mugen_attn_gqa_decode_paged_workspace_size(ctypes.byref(a))
    return (size - 512) // (len(host) * q_len * H * (4 * D + 8)) if size else 1


# short ranges, and batches that fill the card, are not cut; few long ones are
@pytest.mark.parametrize("kw,whole", [
    (dict(lens=[256]), True), (dict(lens=[512]), True), (dict(lens=[1024]), False), (dict(lens=[256], bits=16), True),
    (dict(lens=[384], bits=16), False), (dict(lens=[1024] * 32), True), (dict(lens=[4096] * 8), False),
    (dict(lens=[1024] * 32, H=32, Hk=8, D=64), True), (dict(lens=[256], H=16, Hk=8, D=256, bits=16), False),
    (dict(lens=[9000] * 4, n_select=3), True), (dict(lens=[9000] * 4, n_select=64), False),
    (dict(lens=[0]), True), (dict(lens=[1] * 200), True),
])
def test_plan_of_short_and_long_ranges(kw, whole):
    assert (splits(**kw) == 1) == whole
