"""Plain 64-bit forms of the 16-bit operators and the error bounds their tests
use (not collected).

Bounds.  A product's fp32 sum of n exact terms, in any order, is off by at most
(n - 1) 2^-24 sum|terms| (1 + small); the bounds here take (n + 2) 2^-23, twice
that, for matrix instructions that cut instead of rounding inside.  An
activation with slope at most L passes an error on L times; its own evaluation
adds a few 2^-24 of its value (16 are allowed, the functions used are good to
a few).  Storing rounds by at most eps / 2 of the stored value, or half a step
of the smallest one."""
import math

import torch

TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}
SLOPE = {"none": 1.0, "relu": 1.0, "silu": 1.1, "gelu": 1.13, "sigmoid": 0.25}


def rounding(v, dtype):
    """Largest error of storing values of magnitude up to |v|."""
    return torch.finfo(dtype).eps / 2 * v + TINY[dtype]


def act(z, name):
    if name == "swiglu":
        g, u = z.chunk(2, 1)
        return g * torch.sigmoid(g) * u
    if name == "sigmoid":
        return torch.sigmoid(z)
    if name == "silu":
        return z * torch.sigmoid(z)
    if name == "gelu":
        return 0.5 * z * torch.special.erfc(-z * math.sqrt(0.5))
    return torch.relu(z) if name == "relu" else z            # slope 0 at 0


def act_grad(dy, z, name):
    z = z.detach().clone().requires_grad_(True)
    act(z, name).backward(dy)
    return z.grad


def product(x, w, bias, name, dtype):
    """(z, bound of z, y, bound of y before rounding) of act(x w^T + bias) for one group."""
    x, w = x.double().cpu(), w.double().cpu()
    z, mag = x @ w.T, x.abs() @ w.abs().T
    if bias is not None:
        z, mag = z + bias.double().cpu(), mag + bias.double().cpu().abs()
    dz = (x.shape[1] + 2) * 2.0 ** -23 * mag
    y = act(z, name)
    if name == "swiglu":
        (g, u), (dg, du) = z.chunk(2, 1), dz.chunk(2, 1)
        dy = 1.1 * dg * (u.abs() + du) + (g * torch.sigmoid(g)).abs() * du
    else:
        dy = SLOPE[name] * dz
    return z, dz, y, dy + 16 * 2.0 ** -24 * y.abs()


def within(got, want, bound, what=""):
    """|got - want| <= bound + the rounding of got's type, everywhere."""
    got64 = got.detach().double().cpu()
    lim = bound + rounding(want.abs() + bound, got.dtype)
    err = (got64 - want).abs()
    bad = ~(err <= lim)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} outside; worst {float((err / lim).max()):.2f} bounds"


def grouping(ids, E):
    """(offsets, token, row) by a loop over the picks."""
    T, K = ids.shape
    rows = [[] for _ in range(E)]
    for t in range(T):
        for k in range(K):
            if 0 <= int(ids[t, k]) < E:
                rows[int(ids[t, k])].append((t, k))
    offsets, token, row = [0], [], torch.full((T, K), -1, dtype=torch.int32)
    for r in rows:
        for t, k in r:
            row[t, k] = len(token)
            token.append(t)
        offsets.append(len(token))
    token += [-1] * (T * K - len(token))
    return torch.tensor(offsets, dtype=torch.int32), torch.tensor(token, dtype=torch.int32), row


# Shapes (rows, in, out, groups) that between them run every kernel of the
# products, whole and in parts, plain and grouped: test_dense_host.py checks
# that they still do.  Ragged in every dimension where the kernel allows it.
KERNEL_SHAPES = {
    "forward": [(1, 72, 40, 1), (3000, 200, 4104, 1), (4000, 264, 2056, 9), (4000, 136, 1032, 1), (4000, 72, 1032, 3),
                (130, 200, 8200, 3), (17, 2056, 8200, 1), (16, 2056, 520, 9), (4000, 136, 520, 1), (4000, 136, 520, 3),
                (3000, 4104, 136, 1), (3000, 4104, 136, 3), (16, 136, 4104, 9), (16, 2056, 264, 9), (19, 136, 24, 1),
                (5, 136, 24, 3), (17, 1032, 16, 1), (2, 2056, 24, 3), (2000, 136, 520, 1), (4000, 136, 264, 3),
                (1000, 2056, 16, 1), (1000, 2056, 24, 3), (200, 71, 56, 3), (50, 71, 56, 3), (5, 71, 57, 3), (700, 71, 57, 1),
                (3, 2056, 2056, 3), (1000, 136, 8200, 9), (2000, 2056, 24, 3),
           (4000, 264, 136, 1), (17, 4096, 8200, 1), (130, 4096, 520, 3), (4000, 1032, 8200, 9),
           (2000, 4096, 57, 3), (50, 264, 16, 3), (2000, 4096, 57, 64), (700, 4096, 136, 1), (700,
           4096, 136, 3), (2000, 71, 2056, 1), (2000, 71, 2056, 3), (700, 71, 2056, 1), (130, 71,
           2056, 3), (2000, 264, 136, 64), (700, 4096, 136, 9),
           (50, 4096, 2056, 3)],
    "dx": [(3000, 2056, 72, 1), (4000, 1032, 136, 9), (4000, 2056, 200, 9), (3000, 4104, 136, 1), (2000, 520, 8200, 1),
           (2000, 520, 8200, 3), (260, 4104, 72, 9), (3, 2056, 8200, 1), (130, 264, 4104, 9), (4000, 520, 72, 1),
           (4000, 520, 72, 3), (3000, 136, 4104, 1), (2000, 72, 8200, 9), (16, 4104, 72, 9), (1, 2056, 2056, 1),
           (16, 264, 2056, 9), (5, 72, 24, 1), (5, 72, 24, 3), (3, 72, 1032, 1), (3, 72, 2056, 3), (2000, 520, 72, 1),
           (2000, 520, 72, 3), (1000, 72, 2056, 1), (1000, 72, 2056, 3), (50, 71, 57, 3), (700, 71, 57, 1),
           (130, 200, 4104, 9), (3000, 4104, 136, 3),
           (2000, 264, 136, 1), (700, 71, 2056, 3), (700, 64, 8200, 1), (700, 64, 8200, 3), (4000,
           1032, 57, 1), (4000, 1032, 57, 3), (700, 71, 2056, 9), (700, 71, 8200, 3), (2000, 1032, 8200, 3),
           (1, 4096, 2056, 1), (50, 1032, 8200, 3)],
    "dw": [(200, 4104, 520, 1), (300, 4104, 24, 9), (4000, 72, 8200, 1), (130, 2056, 8200, 1), (700, 1032, 1032, 9),
           (70, 72, 24, 1), (70, 72, 24, 3), (1000, 72, 24, 1), (4000, 72, 24, 3), (1000, 71, 57, 1), (130, 264, 8200, 1),
           (700, 4096, 2056, 3)],
}


def plan(lib, rows, inn, out, groups, direction, parts):
    """The kernel a product of contiguous bf16 operands runs on (wm_product_plan)."""
    import ctypes as C

    from winmoe_amd import _lib
    d = _lib.ProductDesc()
    d.dtype, d.rows, d.inn, d.out, d.n_groups, d.x_rows, d.y_type = _lib.BF16, rows, inn, out, groups, rows, _lib.BF16
    d.x, d.w, d.y, d.dz, d.offsets = 4096, 4096, 4096, 4096, 4096 if groups > 1 else None
    d.ldx, d.ldw, d.w_stride, d.ldy, d.ld_dz = inn, inn, inn * out, out, out
    p = C.c_int()
    k = lib.wm_product_plan(C.byref(d), direction, C.byref(p))
    assert k >= 0
    parts.append(p.value)
    return _lib.PRODUCT_KERNELS[k]
