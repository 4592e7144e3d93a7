"""Refusals of the 16-bit operators and their empty calls, without a GPU: the C
entry points check before they touch a device, the Python functions before they
call them."""
import ctypes as C

import pytest
import torch

from dense_ref import KERNEL_SHAPES, grouping, plan


@pytest.fixture(scope="module")
def lib():
    from winmoe_amd import _lib
    return _lib.load()


def desc(**kw):
    """A sound product of 4 rows, 16 x 8 weights, at made-up addresses that no check follows."""
    from winmoe_amd import _lib
    d = _lib.ProductDesc()
    d.dtype, d.rows, d.inn, d.out, d.n_groups, d.x_rows, d.y_type = _lib.BF16, 4, 8, 16, 1, 4, _lib.BF16
    d.x, d.w, d.y = 4096, 8192, 16384
    d.ldx, d.ldw, d.ldy = 8, 8, 16
    for k, v in kw.items():
        setattr(d, k, v)
    return d


BAD = [dict(dtype=0), dict(dtype=8), dict(rows=-1), dict(rows=(1 << 30) + 1), dict(inn=0), dict(out=0),
       dict(inn=(1 << 26) + 1), dict(n_groups=0), dict(n_groups=2), dict(n_groups=(1 << 16) + 1, offsets=64),
       dict(offsets=66), dict(token=65), dict(x_rows=3), dict(x_rows=-1, token=64), dict(ldx=7), dict(ldw=7),
       dict(n_groups=2, offsets=64, w_stride=127), dict(act=-1), dict(act=6), dict(x=None), dict(w=None), dict(y=None),
       dict(x=4097), dict(w=8193), dict(y=16385), dict(y_type=1), dict(y_type=0, y=16386), dict(ldy=15),
       dict(bias=65), dict(residual=65, ld_residual=16), dict(residual=64, ld_residual=15), dict(pre=64, ld_pre=15),
       dict(pre=65, ld_pre=16), dict(act=4, out=15), dict(act=4, ldy=7)]


@pytest.mark.parametrize("kw", BAD, ids=str)
def test_product_refuses(lib, kw):
    assert lib.wm_product(C.byref(desc(**kw)), None, 0, None) == -2


@pytest.mark.parametrize("kw", [b for b in BAD if set(b) <= {"dtype", "rows", "inn", "n_groups", "ldx", "ldw", "x_rows"}], ids=str)
def test_product_workspace_and_backward_refuse(lib, kw):
    d = desc(**kw)
    assert lib.wm_product_workspace_size(C.byref(d), 0) < 0
    d.dz, d.ld_dz = 64, 16
    assert lib.wm_product_workspace_size(C.byref(d), 1) < 0
    assert lib.wm_product_backward(C.byref(d), 64, 8, None, 0, None, None, 0, None) == -2


def test_product_backward_refuses(lib):
    d = desc()
    def call(d, dz=64, ldz=16, dx=None, ldx=8, dw=None, wt=30, db=None):
        d.dz, d.ld_dz = dz, ldz
        return lib.wm_product_backward(C.byref(d), dx, ldx, dw, wt, db, None, 0, None)

    assert call(desc(act=1), dx=64) == -2                    # the activation's gradient is a step of its own
    assert call(d, dz=None, dx=64) == -2
    assert call(d, dz=65, dx=64) == -2
    assert call(d, ldz=15, dx=64) == -2
    assert call(d, dx=65) == -2
    assert call(d, dx=64, ldx=7) == -2
    assert call(desc(w=None), dx=64) == -2
    assert call(desc(x=None), dw=64) == -2
    assert call(d, dw=64, wt=1) == -2                        # fp16 gradients of bf16 weights
    assert call(d, dw=66, wt=0) == -2
    assert call(d, db=66) == -2
    assert lib.wm_product(None, None, 0, None) == -2


def test_pair_operators_refuse(lib):
    bf, f32 = 30, 0
    assert lib.wm_act_backward(f32, 1, 4, 8, 64, 8, 64, 8, 64, 8, None) == -2
    assert lib.wm_act_backward(bf, 7, 4, 8, 64, 8, 64, 8, 64, 8, None) == -2
    assert lib.wm_act_backward(bf, 4, 4, 8, 64, 8, 64, 8, 64, 16, None) == -2       # pre must be twice as wide
    assert lib.wm_act_backward(bf, 1, 4, 0, 64, 8, 64, 8, 64, 8, None) == -2
    assert lib.wm_act_backward(bf, 1, -1, 8, 64, 8, 64, 8, 64, 8, None) == -2
    assert lib.wm_act_backward(bf, 1, 4, 8, None, 8, 64, 8, 64, 8, None) == -2
    g = lib.wm_group_by_expert
    assert g(64, 1, 0, 4, 64, 64, 64, None) == -2
    assert g(64, 1, 1, 0, 64, 64, 64, None) == -2
    assert g(64, 1 << 20, 1 << 11, 4, 64, 64, 64, None) == -2
    assert g(64, 1, 1, 4, None, 64, 64, None) == -2
    assert g(None, 1, 1, 4, 64, 64, 64, None) == -2
    assert g(66, 1, 1, 4, 64, 64, 64, None) == -2
    c = lib.wm_combine_rows
    assert c(f32, 64, 8, 4, 64, 64, 2, 2, 8, None, 0, 64, 8, f32, None) == -2
    assert c(bf, 64, 8, 4, 64, 64, 2, 2, 8, None, 0, 64, 8, 1, None) == -2
    assert c(bf, 64, 7, 4, 64, 64, 2, 2, 8, None, 0, 64, 8, bf, None) == -2
    assert c(bf, 64, 8, 4, 64, 64, 2, 2, 8, 64, 7, 64, 8, bf, None) == -2
    assert c(bf, 64, 8, 4, None, 64, 2, 2, 8, None, 0, 64, 8, bf, None) == -2
    assert c(bf, 64, 8, 4, 64, 64, 2, 2, 8, None, 0, 66, 8, f32, None) == -2
    b = lib.wm_combine_rows_backward
    assert b(bf, 64, 8, 1, 64, 8, 4, 64, 64, 2, 2, 8, 64, 8, None, None) == -2
    assert b(bf, 64, 7, bf, 64, 8, 4, 64, 64, 2, 2, 8, 64, 8, None, None) == -2
    assert b(bf, 64, 8, bf, None, 8, 4, 64, 64, 2, 2, 8, None, 8, 64, None) == -2
    assert b(bf, 64, 8, bf, 64, 8, 4, 64, 64, 2, 2, 8, 64, 7, None, None) == -2


def test_empty_calls_return_at_once(lib):
    """No rows, no tokens or nothing asked for: 0, before any device is needed."""
    assert lib.wm_product(C.byref(desc(rows=0, x=None, w=None, y=None)), None, 0, None) == 0
    assert lib.wm_act_backward(30, 1, 0, 8, None, 0, None, 0, None, 0, None) == 0
    assert lib.wm_combine_rows(30, None, 0, 0, None, None, 0, 2, 8, None, 0, None, 0, 30, None) == 0
    assert lib.wm_combine_rows_backward(30, 64, 8, 30, 64, 8, 4, 64, 64, 2, 2, 8, None, 8, None, None) == 0


def test_descriptor_is_as_long_as_the_headers(lib):
    from winmoe_amd import _lib
    assert C.sizeof(_lib.ProductDesc) == 8 * 4 + 16 * 8


def test_python_refuses_host_tensors():
    from winmoe_amd import dense
    x = torch.zeros(4, 8, dtype=torch.bfloat16)
    for call in (lambda: dense.linear(x, x), lambda: dense.group_by_expert(torch.zeros(2, 2, dtype=torch.int32), 4),
                 lambda: dense.act_backward(x, x, "silu"), lambda: dense.combine(x, torch.zeros(2, 2, dtype=torch.int32)),
                 lambda: dense.grouped_matmul(x, x.view(1, 4, 8), torch.zeros(2, dtype=torch.int32))):
        with pytest.raises(ValueError, match="HIP"):
            call()


def test_reference_grouping():
    """The tests' own sorting, on a case small enough to see."""
    off, token, row = grouping(torch.tensor([[2, 0], [-1, 2], [0, 3]]), 3)
    assert off.tolist() == [0, 2, 2, 4] and token.tolist() == [0, 2, 0, 1, -1, -1]
    assert row.tolist() == [[2, 0], [-1, 3], [1, -1]]


def test_kernel_shapes_run_every_kernel(lib):
    """The shapes of the GPU tests reach every kernel, whole and in parts, plain and grouped, that any of a wide
    range of shapes reaches; wm_product_plan knows the same names as the Python binding."""
    import itertools
    import re

    from winmoe_amd import _lib
    header = open(_lib.os.path.join(_lib.PKG, "..", "include", "winmoe_hip.h")).read()
    names = re.search(r"#define WM_PRODUCT_KERNELS (.*)", header).group(1)
    assert tuple(re.findall(r'"(\w+)"', names)) == _lib.PRODUCT_KERNELS
    reach, have = set(), set()
    for i, direction in enumerate(("forward", "dx", "dw")):
        for rows, inn, out, groups in KERNEL_SHAPES[direction]:
            p = []
            have.add((direction, plan(lib, rows, inn, out, groups, i, p), p[0] > 1, groups > 1))
        for rows, inn, out, groups in itertools.product((1, 3, 16, 17, 50, 130, 700, 2000, 4000), (64, 71, 264, 1032, 4096),
                                                        (16, 57, 136, 520, 2056, 8200), (1, 3, 9, 64)):
            p = []
            reach.add((direction, plan(lib, rows, inn, out, groups, i, p), p[0] > 1, groups > 1))
    assert not reach - have, sorted(reach - have)


def test_workspace_is_asked_for_and_checked(lib):
    """A call whose size query is not 0 refuses a missing, short or unaligned workspace."""
    parts = []
    plan(lib, 3000, 4104, 136, 1, 0, parts)
    d = desc(rows=3000, x_rows=3000, inn=4104, out=136, ldx=4104, ldw=4104, ldy=136)
    need = lib.wm_product_workspace_size(C.byref(d), 0)
    assert parts[0] > 1 and need >= parts[0] * 3000 * 136 * 4
    for ws, n in ((None, need), (4096, need - 1), (4096 + 128, need)):
        assert lib.wm_product(C.byref(d), ws, n, None) == -2
    d = desc(inn=4095, ldx=4095, ldw=4095, out=8192, ldy=8192, rows=4000, x_rows=4000)  # odd rows: copies
    assert lib.wm_product_workspace_size(C.byref(d), 0) >= (4000 + 8192) * 4096 * 2
    d.dz, d.ld_dz = 4096, 8192
    assert lib.wm_product_workspace_size(C.byref(d), 1) >= (4000 + 8192) * 4096 * 2
    assert lib.wm_product_backward(C.byref(d), 4096, 4095, None, 0, None, None, 0, None) == -2
    p = C.c_int()
    assert lib.wm_product_plan(C.byref(d), 3, C.byref(p)) == -2 and lib.wm_product_plan(C.byref(d), 0, None) == -2


@pytest.mark.parametrize("kw", [dict(n_groups=1 << 16, offsets=64, w_stride=1 << 20), dict(ldw=(1 << 40) + 1),
                                dict(ldx=(1 << 40) + 1), dict(inn=1 << 26, out=1 << 26, ldx=1 << 26, ldw=1 << 26, ldy=1 << 26)],
                         ids=str)
def test_sizes_beyond_any_memory_are_refused(lib, kw):
    d = desc(**kw)
    assert lib.wm_product(C.byref(d), None, 0, None) == -2
    assert lib.wm_product_workspace_size(C.byref(d), 0) < 0


def test_combine_refuses_more_tokens_than_a_launch_holds(lib):
    T = 1 << 24
    assert lib.wm_combine_rows(30, 4096, 8, 4, 64, None, T, 1, 8, None, 0, 8192, 8, 30, None) == -2
    for t, k in ((T // 2, 5), (T // 4, 6)):
        assert lib.wm_combine_rows_backward(30, 4096, 8, 30, 8192, 8, 4, 64, None, t, k, 8, 16384, 8, 64, None) == -2


@pytest.mark.parametrize("E, rows, out, inn", [(1, 65536, 64, 8), (3, 10000, 100, 64), (1, 4096, 262144, 8), (64, 2000, 16, 256)])
def test_workspace_covers_a_bias_gradient_alone(lib, E, rows, out, inn):
    """db without dw is a product with one column of x, in parts of its own."""
    d = desc(n_groups=E, offsets=64 if E > 1 else None, rows=rows, x_rows=rows, inn=inn, out=out, ldx=inn, ldw=inn, ldy=out,
             w_stride=out * inn)
    d.dz, d.ld_dz = 1 << 20, out
    one = _copy(d)
    one.inn = 1
    parts = C.c_int()
    assert lib.wm_product_plan(C.byref(one), 2, C.byref(parts)) >= 0
    assert parts.value == 1 or lib.wm_product_workspace_size(C.byref(d), 1) >= 4 * E * out * 2 * parts.value


def _copy(d):
    return type(d).from_buffer_copy(d)
