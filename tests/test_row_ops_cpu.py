"""Row operators, checks that need no GPU: arguments are refused with status codes before a device is touched, and the
python entry points refuse operands that do not fit together."""
import ctypes

import pytest

F, U = ctypes.c_void_p(4096), ctypes.c_void_p(4097)  # never dereferenced: argument checks come first


def _lookup(L, n=4, vocab=8, width=16, ids=F, id_type=1, table=F, ld_table=16, dtype=1, scale=1.0, out=F, ld_out=16):
    return L.hpspmm_embedding_lookup(n, vocab, width, ids, id_type, table, ld_table, dtype, scale, out, ld_out, None)


@pytest.mark.parametrize("bad", [
    {"n": -1}, {"vocab": -1}, {"n": 2**31 - 1}, {"vocab": 2**31 - 1}, {"width": 0}, {"width": 2**20 + 1, "ld_table": 2**21, "ld_out": 2**21},
    {"ids": None}, {"ids": ctypes.c_void_p(4100)}, {"id_type": 2}, {"id_type": -1}, {"table": None}, {"table": U},
    {"ld_table": 15}, {"ld_table": 2**41}, {"dtype": 3}, {"dtype": -1}, {"out": None}, {"out": U}, {"ld_out": 15}],
    ids=str)
def test_lookup_refuses(pkg, bad):
    L = pkg.capi.lib()
    assert _lookup(L, **bad) == pkg.capi.ERR_INVALID_ARG
    assert L.hpspmm_last_error() != b""


def test_lookup_of_nothing_is_fine(pkg):
    assert _lookup(pkg.capi.lib(), n=0, ids=None, out=None) == pkg.capi.OK


def _grad(L, plan=None, n=4, vocab=8, width=16, ids=F, id_type=1, grad=F, ld_grad=16, grad_type=1, table=F, ld_table=16,
          table_type=0):
    return L.hpspmm_embedding_grad(plan, n, vocab, width, ids, id_type, grad, ld_grad, grad_type, 1.0, table, ld_table,
                                   table_type, 0, None)


@pytest.mark.parametrize("bad", [
    {}, {"n": -1}, {"vocab": 2**31 - 1}, {"width": 0}, {"ids": None}, {"id_type": 7}, {"grad": None}, {"grad": U},
    {"ld_grad": 3}, {"grad_type": 9}, {"table": None}, {"table": ctypes.c_void_p(4098)}, {"ld_table": 0}, {"table_type": 4}],
    ids=str)
def test_lookup_gradient_refuses(pkg, bad):
    """(with no plan at all in every case: a call without one is refused too)"""
    L = pkg.capi.lib()
    assert _grad(L, **bad) == pkg.capi.ERR_INVALID_ARG
    assert (L.hpspmm_last_error() == b"plan is NULL") == (bad == {})


def test_group_rows_refuses(pkg):
    capi = pkg.capi
    L = capi.lib()
    for n, groups, ids, kind, order, offsets in ((-1, 4, F, 1, F, F), (4, -1, F, 1, F, F), (4, 4, None, 1, F, F),
                                                 (4, 4, F, 5, F, F), (4, 4, F, 1, None, F), (4, 4, F, 1, F, None),
                                                 (4, 4, F, 1, U, F), (4, 4, F, 1, F, U), (2**31 - 1, 4, F, 1, F, F),
                                                 (4, 4, F, 1, F, F)):
        assert L.hpspmm_group_rows(None, n, groups, ids, kind, order, offsets, None) == capi.ERR_INVALID_ARG


def test_plan_refuses(pkg):
    capi = pkg.capi
    L = capi.lib()
    h = ctypes.c_void_p()
    for rows, ids, width in ((-1, 4, 4), (4, -1, 4), (4, 4, -1), (2**31 - 1, 4, 4), (4, 2**31 - 1, 4), (4, 4, 2**20 + 1)):
        assert L.hpspmm_rows_plan_create(rows, ids, width, ctypes.byref(h)) == capi.ERR_INVALID_ARG
        assert not h.value
    assert L.hpspmm_rows_plan_create(4, 4, 4, None) == capi.ERR_INVALID_ARG
    assert L.hpspmm_rows_plan_destroy(None) == capi.OK


def _grouped(name):
    def call(L, rows=8, groups=2, k=16, m=32, a=F, lda=None, b=F, ldb=None, stride=None, offsets=F, c=F, ldc=None, dtype=1,
             dw_type=1):
        wide_a, wide_c = (k, m) if name == "forward" else (m, k)
        lda, ldc = wide_a if lda is None else lda, wide_c if ldc is None else ldc
        ldb, stride = k if ldb is None else ldb, m * k if stride is None else stride
        if name == "forward":
            return L.hpspmm_grouped_mm(rows, groups, k, m, a, lda, b, ldb, stride, offsets, c, ldc, dtype, None)
        if name == "grad_x":
            return L.hpspmm_grouped_mm_grad_x(rows, groups, k, m, a, lda, b, ldb, stride, offsets, c, ldc, dtype, None)
        return L.hpspmm_grouped_mm_grad_w(None, rows, groups, k, m, a, lda, b, ldb, offsets, c, ldc, stride, dtype, dw_type,
                                          0, None)
    return call


@pytest.mark.parametrize("name", ["forward", "grad_x", "grad_w"])
@pytest.mark.parametrize("bad", [
    {"rows": -1}, {"rows": 2**31 - 1}, {"groups": -1}, {"groups": 65536}, {"k": 0}, {"m": 0}, {"k": 2**20 + 1}, {"m": 2**20 + 1},
    {"a": None}, {"a": U}, {"lda": 3}, {"b": None}, {"b": U}, {"ldb": 3}, {"stride": -1}, {"offsets": None},
    {"offsets": ctypes.c_void_p(4098)}, {"c": None}, {"c": U}, {"ldc": 3}, {"dtype": 3}], ids=str)
def test_grouped_products_refuse(pkg, name, bad):
    L = pkg.capi.lib()
    assert _grouped(name)(L, **bad) == pkg.capi.ERR_INVALID_ARG
    assert L.hpspmm_last_error() not in (b"", b"plan is NULL")


def test_gradient_of_the_weights_refuses(pkg):
    """No plan, a type that is neither the operands' nor 32 bits, matrices that would lie in one another."""
    L = pkg.capi.lib()
    call = _grouped("grad_w")
    for bad in ({}, {"dw_type": 2}, {"stride": 16 * 32 - 1}):
        assert call(L, **bad) == pkg.capi.ERR_INVALID_ARG


def test_products_of_nothing_are_fine(pkg):
    L = pkg.capi.lib()
    for name in ("forward", "grad_x"):
        assert _grouped(name)(L, rows=0, a=None, c=None) == pkg.capi.OK
        assert _grouped(name)(L, groups=0, b=None, offsets=None) == pkg.capi.OK


def test_python_entry_points_refuse_host_tensors(pkg):
    import torch
    capi = pkg.capi
    ids, table = torch.zeros(4, dtype=torch.int64), torch.zeros(8, 16)
    with pytest.raises(TypeError, match="GPU memory"):
        capi.embedding_lookup(table, ids, torch.zeros(4, 16))
    with pytest.raises(TypeError, match="GPU memory"):
        capi.grouped_mm(table, torch.zeros(2, 3, 16), torch.zeros(3, dtype=torch.int32), torch.zeros(8, 3))
    with pytest.raises(TypeError, match="GPU memory"):
        capi.grouped_mm_grad_x(torch.zeros(8, 3), torch.zeros(2, 3, 16), torch.zeros(3, dtype=torch.int32), table)
