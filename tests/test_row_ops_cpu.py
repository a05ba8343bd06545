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


# Sizes (rows, groups, k, m) of grouped products that between them are cut in every way there is; the GPU tests run them.
TILED = [(300, 5, 129, 65), (1000, 7, 256, 384), (700, 16, 1032, 1032), (9000, 5, 264, 4104), (9000, 5, 4104, 264),
         (9000, 5, 1028, 2052), (9000, 5, 1001, 1003), (12000, 3, 1004, 1148), (12000, 3, 1003, 1149), (2000, 16, 1016, 1000),
         (2000, 16, 1001, 1003), (12000, 3, 520, 1032), (9000, 2, 200, 89)]


def tilings(capi, kind, size, case):
    """{(product, whole rows, edge, in parts)} of one case; rows are whole where both lengths are multiples of 16 bytes."""
    rows, groups, k, m = case
    whole = k * size % 16 == 0 and m * size % 16 == 0
    cut = {q: capi.grouped_tiling(q, rows, groups, k, m, kind, whole) for q in capi.PRODUCTS}
    return {(q, whole, edge, parts > 1) for q, (edge, parts) in cut.items()}


@pytest.mark.parametrize("kind, size", [(0, 4), (1, 2), (2, 2)])
def test_the_tested_products_are_cut_in_every_way(pkg, kind, size):
    """Every tile kernel that a call can reach is reached by a size in TILED (a rule that is changed must not leave a
    kernel behind untested)."""
    capi = pkg.capi
    reached = set().union(*(tilings(capi, kind, size, case) for case in TILED))
    edges = {True: (256, 128, 64) if size == 2 else (128, 64), False: (128, 64)}
    every = {(q, whole, edge, False) for q in capi.PRODUCTS for whole in edges for edge in edges[whole]}
    every |= {("grouped_mm_grad_w", whole, 128, True) for whole in edges}
    assert reached == every, (sorted(every - reached), sorted(reached - every))


def test_tiling_refuses(pkg):
    capi = pkg.capi
    edge, parts = ctypes.c_int(), ctypes.c_int()
    call = lambda *a, e=ctypes.byref(edge), p=ctypes.byref(parts): capi.lib().hpspmm_grouped_tiling(*a, e, p)  # noqa: E731
    assert call(0, 8, 2, 16, 32, 1, 1) == capi.OK and edge.value and parts.value == 1
    for bad in ((3, 8, 2, 16, 32, 1, 1), (-1, 8, 2, 16, 32, 1, 1), (0, -1, 2, 16, 32, 1, 1), (0, 8, -1, 16, 32, 1, 1),
                (0, 8, 2, 0, 32, 1, 1), (0, 8, 2, 16, 0, 1, 1), (0, 8, 2, 16, 32, 3, 1)):
        assert call(*bad) == capi.ERR_INVALID_ARG and (edge.value, parts.value) == (0, 0)
    assert call(0, 8, 2, 16, 32, 1, 1, e=None) == capi.ERR_INVALID_ARG
    assert call(0, 8, 2, 16, 32, 1, 1, p=None) == capi.ERR_INVALID_ARG
    # nothing is launched for no groups, and for no rows but to clear the gradient of the weights
    assert capi.grouped_tiling("grouped_mm", 0, 2, 16, 32, capi.BF16) == (0, 0)
    assert capi.grouped_tiling("grouped_mm_grad_w", 8, 0, 16, 32, capi.BF16) == (0, 0)
    assert capi.grouped_tiling("grouped_mm_grad_w", 0, 2, 16, 32, capi.BF16) == (64, 1)
