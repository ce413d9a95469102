"""CPU: rotary positions, the paged cache and attention over it: struct layouts, what the C ABI and the Python surface refuse before
anything touches a device, the rotary table."""
import ctypes
import importlib
import math
import os
import subprocess

import pytest
import torch

from conftest import ROOT


@pytest.fixture(scope="module")
def lib():
    L = importlib.import_module("int-flashattention_b200._lib")
    if not os.path.exists(L.LIB_PATH):
        importlib.import_module("int-flashattention_b200.build").build()
    return L


@pytest.mark.parametrize("name", ["IntfaRotaryParams", "IntfaPagedCache", "IntfaAppendParams", "IntfaPagedParams"])
def test_struct_layouts(lib, name, tmp_path):
    cls = getattr(lib, name)
    fields = [f[0] for f in cls._fields_]
    c = ['#include <stdio.h>', '#include <stddef.h>', '#include "intfa.h"', 'int main(void){', 'printf("%%zu\\n", sizeof(%s));' % name]
    c += ['printf("%%zu\\n", offsetof(%s, %s));' % (name, f) for f in fields] + ['return 0;}']
    (tmp_path / "layout.c").write_text("\n".join(c))
    exe = str(tmp_path / "layout")
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), str(tmp_path / "layout.c"), "-o", exe])
    nums = [int(x) for x in subprocess.check_output([exe]).split()]
    assert nums == [ctypes.sizeof(cls)] + [getattr(cls, f).offset for f in fields]


def cache(lib, **kw):
    c = lib.IntfaPagedCache()
    c.k = c.v = c.k_scale = c.v_scale = c.block_table = c.seq_lens = 1 << 20
    c.S, c.pages, c.H_kv, c.D, c.page_size, c.block, c.table_width, c.table_stride = 3, 10, 2, 128, 16, 4, 5, 5
    for n in ("k_stride", "v_stride"):
        setattr(c, n, lib._i64x3(2 * 16 * 128, 16 * 128, 128))
    c.ks_stride = c.vs_stride = lib._i64x3(8, 4, 1)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


BAD_CACHES = [(dict(D=32), "head_dim"), (dict(D=96), "head_dim"), (dict(page_size=48), "page_size"), (dict(page_size=4, block=1), "page_size"),
              (dict(page_size=512), "page_size"), (dict(block=3), "block"), (dict(block=32), "block"), (dict(block=0), "block"), (dict(S=0), "positive"),
              (dict(pages=0), "positive"), (dict(table_width=0), "positive"), (dict(k=None), "k_cache is NULL"), (dict(v=(1 << 20) + 8), "v_cache"),
              (dict(k_scale=None), "k_scale"), (dict(block_table=None), "block_table"), (dict(seq_lens=None), "seq_lens")]


@pytest.mark.parametrize("change,word", BAD_CACHES)
def test_c_abi_refuses_bad_caches(lib, change, word):
    h = lib.load()
    for cls, f in ((lib.IntfaAppendParams, h.intfa_paged_append), (lib.IntfaPagedParams, h.intfa_paged_attention)):
        P = cls()
        P.cache = cache(lib, **change)
        P.tokens, P.H = 3, 4
        assert f(ctypes.byref(P), None) in (lib.ERR_INVALID_ARG, lib.ERR_UNSUPPORTED)
        assert word in lib.last_error()
    assert h.intfa_paged_workspace_bytes(ctypes.byref(P)) == 0


def test_c_abi_refuses_sizes_past_its_counters(lib):
    h = lib.load()
    A, P = lib.IntfaAppendParams(), lib.IntfaPagedParams()
    for X, f in ((A, h.intfa_paged_append), (P, h.intfa_paged_attention)):
        X.cache, X.tokens, X.H = cache(lib, table_width=(1 << 26) + 1), 3, 4
        assert f(ctypes.byref(X), None) == lib.ERR_TOO_LARGE and "block_table" in lib.last_error()
        X.cache, X.cu_seqlens, X.tokens = cache(lib), 1 << 20, (1 << 30) + 1
        assert f(ctypes.byref(X), None) == lib.ERR_TOO_LARGE and "too many" in lib.last_error()
    P.tokens = (1 << 28) + 1                          # (4 heads of them)
    assert h.intfa_paged_attention(ctypes.byref(P), None) == lib.ERR_TOO_LARGE and "too many" in lib.last_error()


def test_c_abi_refuses_bad_arguments(lib):
    h = lib.load()
    for f in (h.intfa_rotary, h.intfa_paged_append, h.intfa_paged_attention):
        assert f(None, None) == lib.ERR_INVALID_ARG and "NULL" in lib.last_error()
    A = lib.IntfaAppendParams()
    A.cache, A.tokens, A.H = cache(lib), 3, 4
    A.k = A.v = A.q = A.q8 = A.q_scale = 1 << 20
    A.k_stride = A.v_stride = lib._i64x2(256, 128)
    A.q_stride = lib._i64x2(512, 128)

    def refused(word, **kw):
        was = {k: lib._i64x2(*v) if isinstance(v, lib._i64x2) else v for k, v in ((k, getattr(A, k)) for k in kw)}
        for k, v in kw.items():
            setattr(A, k, v)
        assert h.intfa_paged_append(ctypes.byref(A), None) != lib.OK and word in lib.last_error(), lib.last_error()
        for k, v in was.items():
            setattr(A, k, v)

    refused("tokens", tokens=0)
    refused("one token a sequence", tokens=4)
    refused("dtype", dtype=lib.TYPE_FP32)
    refused("k is NULL", k=None)
    refused("v stride", v_stride=lib._i64x2(256, 124))
    refused("q8", q8=None)
    refused("rot_dim", table=1 << 20, table_rows=10, rot_dim=130)
    refused("rot_dim", table=1 << 20, table_rows=10, rot_dim=7)
    refused("no rows", table=1 << 20, table_rows=0, rot_dim=64)
    P = lib.IntfaPagedParams()
    P.cache, P.tokens, P.H = cache(lib), 3, 4
    P.q = P.o = P.q_scale = 1 << 20
    P.q_stride = P.o_stride = lib._i64x2(512, 128)
    P.qs_stride = lib._i64x2(4, 1)
    n = h.intfa_paged_workspace_bytes(ctypes.byref(P))
    assert n > 0
    assert h.intfa_paged_attention(ctypes.byref(P), None) == lib.ERR_INVALID_ARG and "workspace" in lib.last_error()
    P.H = 3
    assert h.intfa_paged_attention(ctypes.byref(P), None) == lib.ERR_INVALID_ARG and "multiple of H_kv" in lib.last_error()
    P.H, P.o_dtype = 4, 7
    assert h.intfa_paged_attention(ctypes.byref(P), None) == lib.ERR_INVALID_ARG and "o_dtype" in lib.last_error()
    P.o_dtype, P.tokens = 0, 5
    assert h.intfa_paged_attention(ctypes.byref(P), None) == lib.ERR_INVALID_ARG and "one row a sequence" in lib.last_error()
    P.tokens, P.o = 3, (1 << 20) + 2
    assert h.intfa_paged_attention(ctypes.byref(P), None) == lib.ERR_INVALID_ARG and "o must be" in lib.last_error()
    R = lib.IntfaRotaryParams()
    R.q = R.q_out = R.table = R.positions = 1 << 20
    R.B, R.H, R.N, R.D, R.table_rows, R.rot_dim = 1, 2, 3, 64, 5, 64
    R.q_stride = R.q_out_stride = lib._i64x3(384, 192, 64)
    for field, bad, word in (("D", 48, "head_dim"), ("dtype", 3, "dtype"), ("N", 0, "positive"), ("q_out", None, "q_out"), ("rot_dim", 66, "rot_dim"),
                             ("table", None, "table"), ("table", (1 << 20) + 4, "aligned"), ("positions", None, "positions"),
                             ("q_stride", lib._i64x3(384, 192, 60), "stride")):
        was = lib._i64x3(*getattr(R, field)) if field == "q_stride" else getattr(R, field)
        setattr(R, field, bad)
        assert h.intfa_rotary(ctypes.byref(R), None) != lib.OK and word in lib.last_error(), (field, lib.last_error())
        setattr(R, field, was)


def paged_args(T=3, H=4, Hkv=2, D=64, pages=6, page=16, block=4, S=3):
    i32 = dict(dtype=torch.int32)
    return dict(q=torch.zeros(T, H, D, dtype=torch.int8), k_cache=torch.zeros(pages, Hkv, page, D, dtype=torch.int8),
                v_cache=torch.zeros(pages, Hkv, page, D, dtype=torch.int8), q_scale=torch.ones(T, H), k_scale=torch.ones(pages, Hkv, page // block),
                v_scale=torch.ones(pages, Hkv, page // block), block_table=torch.zeros(S, 2, **i32), seq_lens=torch.ones(S, **i32), cu_seqlens=None,
                causal=True, sm_scale=1.0)


@pytest.mark.parametrize("change,error,word", [
    (dict(), RuntimeError, "CUDA"),
    (dict(q=torch.zeros(3, 4, 64)), TypeError, "int8"),
    (dict(q=torch.zeros(3, 3, 64, dtype=torch.int8), q_scale=torch.ones(3, 3)), ValueError, "multiple"),
    (dict(q=torch.zeros(4, 4, 64, dtype=torch.int8), q_scale=torch.ones(4, 4)), ValueError, "one token a sequence"),
    (dict(q_scale=torch.ones(3, 4).half()), TypeError, "q_scale"),
    (dict(q_scale=torch.ones(3, 3)), ValueError, "q_scale"),
    (dict(k_cache=torch.zeros(6, 2, 16, 64)), TypeError, "int8"),
    (dict(v_cache=torch.zeros(6, 2, 32, 64, dtype=torch.int8)), ValueError, "v_cache"),
    (dict(k_scale=torch.ones(6, 2, 3)), ValueError, "k_scale"),
    (dict(k_scale=torch.ones(6, 2, 32)), ValueError, "k_scale"),
    (dict(v_scale=torch.ones(6, 2, 8)), ValueError, "same block"),
    (dict(block_table=torch.zeros(3, 2)), TypeError, "block_table"),
    (dict(block_table=torch.zeros(3, dtype=torch.int32)), ValueError, "block_table"),
    (dict(seq_lens=torch.ones(4, dtype=torch.int32)), ValueError, "seq_lens"),
    (dict(seq_lens=torch.ones(3, dtype=torch.int64)), TypeError, "seq_lens"),
    (dict(cu_seqlens=torch.zeros(3, dtype=torch.int32)), ValueError, "cu_seqlens"),
    (dict(out_dtype=torch.float32), TypeError, "out_dtype"),
    (dict(out=torch.zeros(3, 4, 64)), TypeError, "out"),
    (dict(out=torch.zeros(3, 4, 32).half()), ValueError, "out"),
    (dict(out=torch.zeros(3, 4, 64).half(), out_dtype=torch.bfloat16), TypeError, "out_dtype"),
])
def test_attention_refuses(pkg, change, error, word):
    with pytest.raises(error, match=word):
        pkg.attention_int8_paged(**{**paged_args(), **change})


@pytest.mark.parametrize("D,page", [(32, 16), (96, 16), (64, 24), (64, 4), (64, 512)])
def test_caches_that_are_refused(pkg, D, page):
    with pytest.raises(ValueError, match="head dim|page_size"):
        pkg.attention_int8_paged(**paged_args(D=D, page=page, block=1))


@pytest.mark.parametrize("change,error,word", [
    (dict(), RuntimeError, "CUDA"),
    (dict(k=torch.zeros(3, 2, 64)), TypeError, "float16 or bfloat16"),
    (dict(v=torch.zeros(3, 2, 64).bfloat16()), TypeError, "same type"),
    (dict(v=torch.zeros(2, 2, 64).half()), ValueError, "shape of k"),
    (dict(k=torch.zeros(3, 1, 64).half(), v=torch.zeros(3, 1, 64).half()), ValueError, "heads"),
    (dict(q=torch.zeros(2, 4, 64).half()), ValueError, "q must"),
    (dict(q=torch.zeros(3, 4, 64)), TypeError, "same type"),
    (dict(table=torch.zeros(5, 33, 2)), ValueError, "66 channels"),
    (dict(table=torch.zeros(5, 32, 2).half()), TypeError, "table"),
    (dict(table=torch.zeros(0, 32, 2)), ValueError, "table"),
    (dict(k_scale=torch.ones(1, 1, 4).expand(6, 2, 4)), ValueError, "strides"),
    (dict(k_cache=torch.zeros(6, 2, 64, 16, dtype=torch.int8).transpose(2, 3)), ValueError, "contiguous last dim"),
])
def test_append_refuses(pkg, change, error, word):
    a = paged_args()
    args = dict(k=torch.zeros(3, 2, 64).half(), v=torch.zeros(3, 2, 64).half(), **{n: a[n] for n in ("k_cache", "v_cache", "k_scale", "v_scale", "block_table", "seq_lens", "cu_seqlens")})
    args.update(change)
    with pytest.raises(error, match=word):
        pkg.append_int8_paged(**args)


@pytest.mark.parametrize("change,error,word", [
    (dict(), RuntimeError, "CUDA"),
    (dict(q=torch.zeros(1, 2, 3, 48)), ValueError, "head dim"),
    (dict(q=torch.zeros(1, 2, 3, 64).double()), TypeError, "q must"),
    (dict(q=torch.zeros(2, 64)), ValueError, "q must"),
    (dict(k=torch.zeros(1, 2, 4, 64)), ValueError, "k must"),
    (dict(k=torch.zeros(1, 2, 3, 64).half()), TypeError, "type of q"),
    (dict(positions=torch.zeros(4, dtype=torch.int32)), ValueError, "positions"),
    (dict(positions=torch.zeros(3)), TypeError, "positions"),
    (dict(positions=torch.zeros(2, 3, dtype=torch.int32)), ValueError, "positions"),
    (dict(table=torch.zeros(5, 64, 2)), ValueError, "128 channels"),
    (dict(table=torch.zeros(5, 64)), ValueError, "table"),
])
def test_rotary_refuses(pkg, change, error, word):
    args = dict(q=torch.zeros(1, 2, 3, 64), k=None, table=torch.zeros(5, 32, 2), positions=torch.zeros(3, dtype=torch.int32))
    with pytest.raises(error, match=word):
        pkg.rotary(**{**args, **change})


def test_rotary_table(pkg):
    t = pkg.rotary_table(70000, 64)
    assert t.shape == (70000, 32, 2) and t.dtype == torch.float32 and t.is_contiguous()
    for pos, j in ((0, 0), (1, 0), (17, 5), (69999, 0), (69999, 1), (69999, 31)):
        a = pos * 10000.0 ** (-2 * j / 64)
        # (half a step of a value up to 1, and of the angle in 64 bits)
        assert abs(t[pos, j, 0].item() - math.cos(a)) <= 2 ** -24 + 1e-10 and abs(t[pos, j, 1].item() - math.sin(a)) <= 2 ** -24 + 1e-10
    lin = pkg.rotary_table(100, 64, scaling=("linear", 4.0))
    assert torch.equal(lin[::4], pkg.rotary_table(25, 64))
    ntk = pkg.rotary_table(9, 8, 100.0, scaling=("ntk", 2.0))
    assert torch.equal(ntk[:, 0], pkg.rotary_table(9, 8, 100.0)[:, 0])                # the fastest pair as before
    a = 8 * 100.0 ** (-6 / 8) / 2.0                                                   # the slowest twice slower
    assert abs(ntk[8, 3, 1].item() - math.sin(a)) < 1e-7
    parts = pkg.rotary_table(50, 64, scaling=("by_parts", 8.0, 4096, 32.0, 1.0, 1.0))
    plain = pkg.rotary_table(50, 64)
    assert torch.equal(parts[:, 0], plain[:, 0])                                      # 652 turns in 4096 positions: stays
    a = 49 * 10000.0 ** (-62 / 64) / 8                                                # 0.09 turns: divided
    assert abs(parts[49, 31, 1].item() - math.sin(a)) < 1e-7
    loud = pkg.rotary_table(50, 64, scaling=("by_parts", 8.0, 4096))
    assert torch.allclose(loud, parts * (0.1 * math.log(8.0) + 1), atol=1e-6, rtol=0)
    for bad in (dict(rot_dim=7), dict(rot_dim=0), dict(n=0), dict(scaling=("linear",)), dict(scaling=("other", 2.0)), dict(scaling=("linear", -1.0)),
                dict(scaling=("by_parts", 2.0)), dict(scaling=("by_parts", 2.0, 4096, 1.0, 2.0)), dict(rot_dim=2, scaling=("ntk", 2.0))):
        with pytest.raises(ValueError):
            pkg.rotary_table(**{**dict(n=4, rot_dim=8), **bad})
