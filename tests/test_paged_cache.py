"""CPU tests of the paged cache's boundary: refusals of the public functions, error codes of the C entries before any CUDA call,
and the layout of their parameter structs."""
import ctypes
import os
import subprocess

import pytest
import torch

import triton_flashattn_b200 as fa
from triton_flashattn_b200 import _cabi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BF = torch.bfloat16


@pytest.mark.parametrize("name,mirror", [("fa_paged_params", _cabi.FaPagedParams), ("fa_kv_write_params", _cabi.FaKvWriteParams),
                                         ("fa_kv_table_params", _cabi.FaKvTableParams)])
def test_struct_layouts_match_the_header(name, mirror, tmp_path):
    fields = [f[0] for f in mirror._fields_]
    src = tmp_path / "sz.c"
    src.write_text('#include "fa_sm100.h"\n#include <stdio.h>\n#include <stddef.h>\nint main(void){printf("%zu", sizeof(' + name + "));"
                   + "".join(f'printf(" %zu", offsetof({name}, {f}));' for f in fields) + "return 0;}\n")
    exe = tmp_path / "sz"
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)])
    c = [int(x) for x in subprocess.check_output([str(exe)]).split()]
    assert c == [ctypes.sizeof(mirror)] + [getattr(mirror, f).offset for f in fields]


# ---------------------------------------------------------------------------------- C entries
def _filled(cls, **kw):
    """Parameters that pass every check; the pointers are never followed: device -1 is refused by the first CUDA call."""
    p = cls()
    p.struct_size, p.device = ctypes.sizeof(cls), -1
    for name, t in cls._fields_:
        if t is ctypes.c_void_p:
            setattr(p, name, 4096)
        elif name.endswith("_stride"):
            setattr(p, name, 64 if t is ctypes.c_int64 else t(*([512] * t._length_)))
    for k, v in kw.items():
        setattr(p, k, v)
    return p


def _paged(**kw):
    return _filled(_cabi.FaPagedParams, **{**dict(B=2, H=8, Hkv=2, D=64, page_size=16, width=4, num_pages=9, dtype=1, bias_kind=1), **kw})


def _write(**kw):
    return _filled(_cabi.FaKvWriteParams, **{**dict(T=5, Hkv=2, D=64, page_size=16, num_pages=9), **kw})


def _table(**kw):
    return _filled(_cabi.FaKvTableParams, **{**dict(B=3, width=4, page_size=16, capacity=9, T=5), **kw})


def test_paged_attention_error_codes():
    lib = _cabi.load()

    def rc(p, ws=4096, n=1 << 40):
        return lib.fa_paged_fwd(ctypes.byref(p), ws, n, None)

    assert lib.fa_paged_fwd(None, None, 0, None) == 2
    assert rc(_paged()) == 6  # nothing to complain about but the device
    assert rc(_paged(), ws=4100) == 5
    assert rc(_paged(struct_size=8)) == 1
    for bad in (dict(B=0), dict(H=0), dict(Hkv=0), dict(H=7), dict(D=48), dict(page_size=0), dict(width=0), dict(num_pages=0)):
        assert rc(_paged(**bad)) == 3, bad
    assert rc(_paged(dtype=2)) == 4 and rc(_paged(bias_kind=4)) == 4
    for name in ("q", "k_cache", "v_cache", "o", "block_table", "seq_lens", "bias"):
        assert rc(_paged(**{name: None})) == 2, name
    assert rc(_paged(bias=None, bias_kind=0)) == 6
    for name in ("q", "k_cache", "v_cache", "o"):
        assert rc(_paged(**{name: 4096 + 8})) == 5, name
    for name in ("block_table", "seq_lens"):
        assert rc(_paged(**{name: 4096 + 2})) == 5, name
    assert rc(_paged(bias=4097)) == 5 and rc(_paged(bias=4097, bias_kind=2)) == 6 and rc(_paged(bias=4098, bias_kind=3)) == 5
    assert rc(_paged(k_stride=_cabi._I64x3(512, 4, 64))) == 5 and rc(_paged(q_stride=_cabi._I64x2(4, 64))) == 5
    assert rc(_paged(width=1 << 20, page_size=1 << 12)) == 9
    assert lib.fa_paged_workspace_bytes(ctypes.byref(_paged(B=0))) == 0


def test_cache_row_error_codes():
    lib = _cabi.load()

    def rc(p):
        return lib.fa_kv_write(ctypes.byref(p), None)

    assert lib.fa_kv_write(None, None) == 2
    assert rc(_write()) == 6 and rc(_write(struct_size=8)) == 1
    assert rc(_write(T=0, k=None)) == 0  # nothing to do
    for bad in (dict(T=-1), dict(Hkv=0), dict(D=24), dict(page_size=0), dict(num_pages=0)):
        assert rc(_write(**bad)) == 3, bad
    for name in ("k", "v", "k_cache", "v_cache", "slots"):
        assert rc(_write(**{name: None})) == 2, name
        assert rc(_write(**{name: 4096 + 4})) == 5, name
    for name in ("k_cache_stride", "v_cache_stride"):
        for i in range(3):
            st = [512, 512, 512]
            for bad in (0, -512, 4):
                st[i] = bad
                assert rc(_write(**{name: _cabi._I64x3(*st)})) == 5
        assert rc(_write(**{name: _cabi._I64x3(512, 512, 0)}, Hkv=1)) == 6  # a stride over one element says nothing


@pytest.mark.parametrize("entry", ["fa_kv_extend", "fa_kv_release"])
def test_table_error_codes(entry):
    fn = getattr(_cabi.load(), entry)
    extend = entry == "fa_kv_extend"

    def rc(**kw):
        return fn(ctypes.byref(_table(**kw)), None)

    assert fn(None, None) == 2
    assert rc() == 6 and rc(struct_size=8) == 1
    for bad in (dict(B=-1), dict(width=0), dict(page_size=0), dict(capacity=-1), dict(table_stride=3)):
        assert rc(**bad) == 3, bad
    assert rc(T=-1) == (3 if extend else 6)
    for name in ("block_table", "lens", "free_pages", "count", "lens_out", "count_out"):
        assert rc(**{name: None}) == 2, name
        assert rc(**{name: 4098}) == 5, name
    assert rc(change=None) == (2 if extend else 6) and rc(finished=None) == (6 if extend else 2)
    assert rc(slots=None) == (2 if extend else 6) and rc(slots=4100) == (5 if extend else 6)
    assert rc(width=1 << 20, page_size=1 << 12, table_stride=1 << 20) == 9
    assert rc(B=0, block_table=None, lens=None, lens_out=None, change=None, finished=None, free_pages=None, capacity=0) == 6


# ---------------------------------------------------------------------------------- public functions
def _attend_args(**kw):
    a = dict(q=torch.zeros(2, 8, 64, dtype=BF), k_cache=torch.zeros(9, 16, 2, 64, dtype=BF), v_cache=torch.zeros(9, 16, 2, 64, dtype=BF),
             block_table=torch.zeros(2, 4, dtype=torch.int32), seq_lens=torch.zeros(2, dtype=torch.int32), bias=None, sm_scale=None)
    a.update(kw)
    return a


@pytest.mark.parametrize("change,error,text", [
    ({}, ValueError, "no CPU path"),
    (dict(q=torch.zeros(2, 1, 8, 64, dtype=BF)), ValueError, "3-D"),
    (dict(q=None), TypeError, "must be a torch.Tensor"),
    (dict(q=torch.zeros(2, 7, 64, dtype=BF)), ValueError, "multiple of those of the caches"),
    (dict(q=torch.zeros(2, 8, 32, dtype=BF)), AssertionError, "share the head dimension"),
    (dict(q=torch.zeros(2, 8, 64, dtype=torch.float16)), TypeError, "share one dtype"),
    (dict(q=torch.zeros(2, 8, 64)), TypeError, "share one dtype"),
    (dict(k_cache=torch.zeros(9, 16, 2, 48, dtype=BF), v_cache=torch.zeros(9, 16, 2, 48, dtype=BF)), AssertionError, "head dimension"),
    (dict(v_cache=torch.zeros(9, 16, 1, 64, dtype=BF)), ValueError, "shape of k_cache"),
    (dict(k_cache=torch.zeros(9, 16, 64, dtype=BF)), ValueError, "4-D"),
    (dict(k_cache=torch.zeros(0, 16, 2, 64, dtype=BF), v_cache=torch.zeros(0, 16, 2, 64, dtype=BF)), ValueError, "at least one page"),
    (dict(k_cache=torch.zeros(9, 16, 2, 68, dtype=BF)[..., :64]), ValueError, "multiples of 16 bytes"),
    (dict(v_cache=torch.zeros(9, 16, 64, 2, dtype=BF).transpose(2, 3)), ValueError, "unit inner stride"),
    (dict(block_table=torch.zeros(2, 4, dtype=torch.int64)), TypeError, "block_table must be an int32"),
    (dict(block_table=torch.zeros(3, 4, dtype=torch.int32)), ValueError, "block_table must be"),
    (dict(block_table=torch.zeros(2, 0, dtype=torch.int32)), ValueError, "block_table must be"),
    (dict(seq_lens=torch.zeros(2, dtype=torch.int64)), TypeError, "seq_lens must be an int32"),
    (dict(seq_lens=torch.zeros(3, dtype=torch.int32)), ValueError, "seq_lens must have shape"),
    (dict(bias=torch.zeros(2, 8, 63, dtype=BF)), ValueError, "no CPU path"),  # (the device is looked at first)
    (dict(sm_scale="x"), ValueError, "no CPU path"),
])
def test_paged_attention_refusals(change, error, text):
    with pytest.raises(error, match=text):
        fa.paged_attention_fn(**_attend_args(**change))


def _row_args(**kw):
    a = dict(k=torch.zeros(5, 2, 64, dtype=BF), v=torch.zeros(5, 2, 64, dtype=BF), k_cache=torch.zeros(9, 16, 2, 64, dtype=BF),
             v_cache=torch.zeros(9, 16, 2, 64, dtype=BF), slot_mapping=torch.zeros(5, dtype=torch.int64))
    a.update(kw)
    return a


@pytest.mark.parametrize("change,error,text", [
    ({}, ValueError, "no CPU path"),
    (dict(k=torch.zeros(5, 3, 64, dtype=BF)), ValueError, "k must have shape"),
    (dict(v=torch.zeros(4, 2, 64, dtype=BF)), ValueError, "v must have shape"),
    (dict(k=torch.zeros(5, 128, dtype=BF)), ValueError, "3-D"),
    (dict(slot_mapping=torch.zeros(5, dtype=torch.int32)), TypeError, "int64"),
    (dict(slot_mapping=torch.zeros(4, dtype=torch.int64)), ValueError, "slot_mapping must have shape"),
    (dict(v=torch.zeros(5, 2, 64, dtype=torch.float16)), TypeError, "share one dtype"),
    (dict(v_cache=torch.zeros(9, 16, 2, 64, dtype=torch.float16)), TypeError, "share one dtype"),
    (dict(k_cache=torch.zeros(9, 1, 2, 64, dtype=BF).expand(9, 16, 2, 64)), ValueError, "expanded"),
    (dict(v_cache=torch.zeros(9, 16, 2, 65, dtype=BF)[..., :64]), ValueError, "multiples of 16 bytes"),
])
def test_cache_row_refusals(change, error, text):
    with pytest.raises(error, match=text):
        fa.paged_kv_write(**_row_args(**change))


def _i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


@pytest.mark.parametrize("change,error,text", [
    ({}, ValueError, "no CPU path"),
    (dict(block_table=_i32(12)), ValueError, "block_table must be"),
    (dict(block_table=_i32(3, 0)), ValueError, "block_table must be"),
    (dict(block_table=_i32(3, 4).long()), TypeError, "block_table must be an int32"),
    (dict(seq_lens=_i32(2)), ValueError, "seq_lens must have shape"),
    (dict(seq_lens=_i32(3).long()), TypeError, "seq_lens must be an int32"),
    (dict(free_pages=_i32(18)[::2]), ValueError, "dense 1-D"),
    (dict(free_pages=_i32(9).long()), TypeError, "free_pages must be an int32"),
    (dict(free_count=_i32(2)), ValueError, "one number"),
    (dict(free_count=_i32(1).long()), TypeError, "free_count must be an int32"),
    (dict(page_size=0), ValueError, "page_size"),
    (dict(page_size=1.5), TypeError, "whole number"),
    (dict(page_size=1 << 30), ValueError, "32 bits"),
])
def test_table_refusals(change, error, text):
    common = dict(block_table=_i32(3, 4), seq_lens=_i32(3), free_pages=_i32(9), free_count=_i32(1), page_size=16)
    with pytest.raises(error, match=text):
        fa.paged_kv_extend(**{**common, "new_lens": _i32(3), "num_tokens": 5, **change})
    with pytest.raises(error, match=text):
        fa.paged_kv_release(**{**common, "finished": torch.zeros(3, dtype=torch.bool), **change})


def test_inputs_that_want_a_gradient_are_refused():
    q = torch.zeros(2, 8, 64, dtype=BF, requires_grad=True)
    with pytest.raises(NotImplementedError, match="no backward"):
        fa.paged_attention_fn(**_attend_args(q=q))
    with pytest.raises(NotImplementedError, match="no backward"):
        fa.paged_attention_fn(**_attend_args(bias=torch.zeros(2, 8, 64, requires_grad=True)))
    with pytest.raises(NotImplementedError, match="no backward"):
        fa.paged_kv_write(**_row_args(k=torch.zeros(5, 2, 64, dtype=BF, requires_grad=True)))
    with torch.no_grad(), pytest.raises(ValueError, match="no CPU path"):
        fa.paged_attention_fn(**_attend_args(q=q))
    with pytest.raises(RuntimeError, match="functorch transforms"):
        torch.func.vmap(lambda q: fa.paged_attention_fn(**_attend_args(q=q)))(torch.zeros(3, 2, 8, 64, dtype=BF))


@pytest.mark.parametrize("change,error", [(dict(num_pages=0), ValueError), (dict(head_dim=48), AssertionError),
                                          (dict(dtype=torch.float32), TypeError), (dict(max_len=0), ValueError)])
def test_cache_constructor_refusals(change, error):
    with pytest.raises(error):
        fa.PagedKVCache(**{**dict(num_layers=1, num_pages=4, page_size=16, num_kv_heads=2, head_dim=64, max_seqs=2, max_len=40,
                                  device="cpu"), **change})


def test_cache_tensors():
    c = fa.PagedKVCache(3, 7, 16, 2, 32, 5, 40, torch.float16, "cpu")
    assert c.k.shape == c.v.shape == (3, 7, 16, 2, 32) and c.k.dtype == torch.float16
    assert c.block_table.shape == (5, 3) and c.seq_lens.shape == (5,) and c.free_count.tolist() == [7]
    assert sorted(c.free_pages.tolist()) == list(range(7))
    assert all(t.dtype == torch.int32 for t in (c.block_table, c.seq_lens, c.free_pages, c.free_count))


def test_operators_are_registered_with_shape_only_implementations():
    from torch._subclasses.fake_tensor import FakeTensorMode

    ops = torch.ops.triton_flashattn_b200
    with FakeTensorMode():
        q = torch.empty(2, 8, 64, dtype=BF, device="cuda")
        cache = torch.empty(9, 16, 2, 64, dtype=BF, device="cuda")
        table, lens = torch.empty(2, 4, dtype=torch.int32, device="cuda"), torch.empty(2, dtype=torch.int32, device="cuda")
        out = ops.paged_attn(q, cache, cache, table, lens, None, 0.125)
        assert out.shape == q.shape and out.dtype == q.dtype and out.is_contiguous()
        rows = torch.empty(5, 2, 64, dtype=BF, device="cuda")
        assert ops.paged_kv_write(rows, rows, cache, cache, torch.empty(5, dtype=torch.int64, device="cuda")) is None
