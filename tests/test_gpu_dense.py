"""The 16-bit operators on the GPU against plain 64-bit forms (dense_ref.py, with the bounds)."""
import pytest
import torch

import dense_ref as ref

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
DT = [BF16, F16]


@pytest.fixture(scope="module")
def dense():
    assert torch.cuda.is_available(), "GPU tests need a HIP device"
    from winmoe_amd import _lib, dense
    _lib.load()
    return dense


def rnd(seed, *shape, dt=BF16, scale=1.0, wide=0):
    """N(0, scale) values; wide > 0: a column range of a matrix that much wider, one element in."""
    g = torch.Generator().manual_seed(seed)
    v = (torch.randn(*shape[:-1], shape[-1] + wide, generator=g) * scale).to(dt).cuda()
    return v[..., 1:1 + shape[-1]] if wide else v


def case(*a):
    print("[case]", *a, flush=True)


# ------------------------------------------------------------------ linear

SIZES = [(1, 64, 16), (1, 4096, 40), (3, 7, 5), (4, 1, 1), (16, 72, 130), (17, 1001, 33), (33, 8, 300), (65, 256, 130),
         (64, 520, 128), (130, 72, 257), (129, 136, 512), (257, 1024, 96), (300, 264, 1100), (600, 2048, 264),
         (2, 8192, 64), (40, 3000, 24)]


@pytest.mark.parametrize("dt", DT, ids=["bf16", "fp16"])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_linear(dense, size, dt):
    T, K, N = size
    case("linear", size, dt)
    x, w = rnd(1, T, K, dt=dt), rnd(2, N, K, dt=dt, scale=0.1)
    _, _, y, by = ref.product(x, w, None, "none", dt)
    ref.within(dense.linear(x, w), y, by, "plain")
    ref.within(dense.linear(x, w, out_dtype=F32), y, by, "fp32")


@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu", "swiglu", "sigmoid"])
@pytest.mark.parametrize("size", [(1, 256, 64), (5, 96, 34), (40, 1000, 130), (200, 128, 258), (300, 576, 512)], ids=str)
def test_linear_epilogue(dense, size, act):
    """Bias, activation, residual, pre-activation, output in place of the residual, strided rows."""
    T, K, N = size
    for n, (dt, wide) in enumerate([(BF16, 0), (F16, 9)]):
        case("linear epilogue", size, act, dt, wide)
        x, w, b = rnd(3, T, K, dt=dt, wide=wide), rnd(4, N, K, dt=dt, scale=0.1, wide=wide), rnd(5, 1, N, dt=dt)[0]
        cols = N // 2 if act == "swiglu" else N
        r = rnd(6, T, cols, dt=dt, wide=wide)
        z, bz, y, by = ref.product(x, w, b, act, dt)
        pre = torch.full((T, N + 3), 7.0, dtype=dt, device="cuda")
        got = dense.linear(x, w, bias=b, act=act, residual=r, pre=pre[:, :N])
        want = y + r.double().cpu()
        bound = by + 2.0 ** -24 * want.abs()                # the residual's addition in fp32
        ref.within(got, want, bound, "y")
        ref.within(pre[:, :N], z, bz, "pre")
        assert (pre[:, N:] == 7.0).all()
        wide_out = torch.full((T, cols + 5), 3.0, dtype=dt, device="cuda")
        o = wide_out[:, 2:2 + cols]
        o.copy_(r)
        dense.linear(x, w, bias=b, act=act, residual=o, out=o)
        assert torch.equal(o, got)
        assert (wide_out[:, :2] == 3.0).all() and (wide_out[:, 2 + cols:] == 3.0).all()
        assert torch.equal(dense.linear(x, w, bias=b, act=act, residual=r), got)       # the same bits again


@pytest.mark.parametrize("dt", DT, ids=["bf16", "fp16"])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_linear_backward(dense, size, dt):
    T, K, N = size
    case("linear backward", size, dt)
    x, w, dz = rnd(7, T, K, dt=dt), rnd(8, N, K, dt=dt, scale=0.1), rnd(9, T, N, dt=dt, scale=0.1)
    dx, dw, db = dense.linear_backward(dz, x, w, need_db=True)
    dw32 = dense.linear_backward(dz, x, w, need_dx=False, dw_dtype=F32)
    assert dw32[0] is None and dw32[2] is None
    x64, w64, d64 = (t.double().cpu() for t in (x, w, dz))
    ref.within(dx, d64 @ w64, (N + 2) * 2.0 ** -23 * (d64.abs() @ w64.abs()), "dx")
    want, bound = d64.T @ x64, (T + 2) * 2.0 ** -23 * (d64.abs().T @ x64.abs())
    ref.within(dw, want, bound, "dw")
    ref.within(dw32[1], want, bound, "dw fp32")
    ref.within(db, d64.sum(0), (T + 2) * 2.0 ** -23 * d64.abs().sum(0), "db")
    only = dense.linear_backward(dz, x, w, need_dx=False, need_dw=False, need_db=True)
    assert only[0] is None and only[1] is None
    ref.within(only[2], d64.sum(0), (T + 2) * 2.0 ** -23 * d64.abs().sum(0), "db alone")


def mm64(a, b):
    """(a b, |a| |b|) in 64 bits on the device."""
    a, b = a.double(), b.double()
    return torch.mm(a, b).cpu(), torch.mm(a.abs(), b.abs()).cpu()


@pytest.mark.parametrize("direction", ["forward", "dx", "dw"])
def test_every_kernel(dense, direction):
    """KERNEL_SHAPES, even groups with an empty one, ragged tokens: each kernel, whole and in parts, against 64 bits."""
    for n, (R, K, N, E) in enumerate(ref.KERNEL_SHAPES[direction]):
        dt = DT[n % 2]
        case("every kernel", direction, R, K, N, E, dt)
        x, w, dz = rnd(80, R, K, dt=dt), rnd(81, E, N, K, dt=dt, scale=0.1), rnd(82, R, N, dt=dt, scale=0.1)
        cut = [0, *(R * e // E for e in range(1, E)), R]
        if E > 2:
            cut[1] = 0                                      # the first expert gets nothing
        off = torch.tensor(cut, dtype=torch.int32, device="cuda") if E > 1 else None
        tok = torch.randperm(R, generator=torch.Generator().manual_seed(n)).int().cuda() if E > 1 and n % 3 else None
        xg = x if tok is None else x[tok.long()]
        b = rnd(83, E, N, dt=dt)
        if direction == "forward":
            y = (dense.linear(x, w[0], bias=b[0]) if E == 1 else
                 dense.grouped_matmul(x, w, off, token=tok, bias=b, out=torch.zeros(R, N, dtype=dt, device="cuda")))
            gated = (dense.linear(x, w[0], act="swiglu", out_dtype=F32) if E == 1 else
                     dense.grouped_matmul(x, w, off, token=tok, act="swiglu", out_dtype=F32)) if N % 2 == 0 else None
        elif E == 1:
            dx, dw, db = dense.linear_backward(dz, x, w[0], need_db=direction == "dw", need_dx=direction == "dx",
                                               need_dw=direction == "dw", dw_dtype=F32 if n % 2 else dt)
        else:
            dx, dw, db = dense.grouped_matmul_backward(dz, x, w, off, token=tok, need_db=direction == "dw", need_dx=direction == "dx",
                                                       need_dw=direction == "dw", dw_dtype=F32 if n % 2 else dt)
        for e in range(E):
            r = slice(cut[e], cut[e + 1])
            rows = r.stop - r.start
            what = f"{direction} {(R, K, N, E)} group {e}"
            if direction == "forward" and rows:
                z, mag = mm64(xg[r], w[e].T)
                bias = b[e].double().cpu()
                ref.within(y[r], z + bias, (K + 3) * 2.0 ** -23 * (mag + bias.abs()), what)
                if gated is not None:
                    (g, u), (dg, du) = z.chunk(2, 1), ((K + 2) * 2.0 ** -23 * mag).chunk(2, 1)
                    s = g * torch.sigmoid(g)
                    ref.within(gated[r], s * u, 1.1 * dg * (u.abs() + du) + s.abs() * du + 2.0 ** -20 * (s * u).abs(), what + " swiglu")
            elif direction == "dx" and rows:
                want, mag = mm64(dz[r], w[e])
                ref.within(dx[r], want, (N + 2) * 2.0 ** -23 * mag, what)
            elif direction == "dw":
                want, mag = mm64(dz[r].T.contiguous(), xg[r])
                ref.within(dw if E == 1 else dw[e], want, (rows + 2) * 2.0 ** -23 * mag, what)
                d64 = dz[r].double().cpu()
                ref.within(db if E == 1 else db[e], d64.sum(0), (rows + 2) * 2.0 ** -23 * d64.abs().sum(0), what + " db")


def test_linear_extremes(dense):
    """Infinities and NaN stay in their row and column, also next to a ragged end."""
    for T, K, N in ((5, 70, 19), (150, 70, 150)):
        x, w = rnd(10, T, K), rnd(11, N, K)
        clean = dense.linear(x, w)
        x[2, 3], x[T - 1, K - 1] = float("nan"), float("inf")
        y = dense.linear(x, w)
        keep = [t for t in range(T) if t not in (2, T - 1)]
        assert torch.equal(y[keep], clean[keep])
        assert y[2].isnan().all() and not y[T - 1].isfinite().any()
        assert torch.equal(y[T - 1].float().sign(), w[:, K - 1].float().sign())
    big = torch.full((2, 64), 60000.0, dtype=F16, device="cuda")
    y = dense.linear(big, torch.ones(16, 64, dtype=F16, device="cuda"))
    assert (y == float("inf")).all()                        # past fp16's range: infinity
    y = dense.linear(big, torch.ones(16, 64, dtype=F16, device="cuda"), out_dtype=F32)
    assert (y == 64 * 60000.0 - (64 * 60000.0 - 64 * float(big[0, 0]))).all()


# ------------------------------------------------------------------ grouped


def groups(kind, E, R, seed=0):
    """Offsets with empty groups, and rows of no group before the first and behind the last."""
    if kind == "one":
        cut = [0] * (E // 2) + [R] * (E + 1 - E // 2)
    elif kind == "ragged":
        g = torch.Generator().manual_seed(seed)
        inner = torch.randint(2, R - 1, (E - 1,), generator=g).sort().values.tolist() if R > 4 else [R // 2] * (E - 1)
        cut = [min(2, R // 2), *inner, R - 1 if R > 4 else R]
        cut[1] = cut[0]                                     # the first group is empty
    else:
        cut = [R * e // E for e in range(E + 1)]
    return torch.tensor(sorted(cut), dtype=torch.int32)


GROUPED = [("even", 4, 37, 64, 48), ("ragged", 5, 90, 104, 34), ("one", 3, 140, 72, 66), ("ragged", 70, 300, 136, 130),
           ("even", 130, 131, 64, 32), ("ragged", 3, 700, 264, 256), ("one", 1, 1, 4096, 64), ("ragged", 9, 1500, 33, 57),
           ("even", 2, 520, 512, 264), ("even", 300, 40, 64, 64)]


@pytest.mark.parametrize("dt", DT, ids=["bf16", "fp16"])
@pytest.mark.parametrize("g", GROUPED, ids=str)
def test_grouped(dense, g, dt):
    kind, E, R, K, N = g
    off = groups(kind, E, R)
    case("grouped", g, dt)
    x, w, b = rnd(12, R, K, dt=dt), rnd(13, E, N, K, dt=dt, scale=0.1), rnd(14, E, N, dt=dt)
    first, last = int(off[0]), int(off[-1])
    x[:first], x[last:] = float("nan"), float("inf")        # rows of no group must not matter
    for act in ("none", "swiglu"):
        cols = N // 2 if act == "swiglu" else N
        if act == "swiglu" and N % 2:
            continue
        for ot in (dt, F32):
            out = torch.full((R, cols), 5.0, dtype=ot, device="cuda")
            pre = torch.full((R, N), 6.0, dtype=dt, device="cuda")
            dense.grouped_matmul(x, w, off.cuda(), bias=b, act=act, out=out, pre=pre)
            assert (out[:first] == 5.0).all() and (out[last:] == 5.0).all()
            assert (pre[:first] == 6.0).all() and (pre[last:] == 6.0).all()
            for e in range(E):
                r = slice(int(off[e]), int(off[e + 1]))
                if r.start < r.stop:
                    z, bz, y, by = ref.product(x[r], w[e], b[e], act, dt)
                    ref.within(out[r], y, by, f"y of group {e}")
                    ref.within(pre[r], z, bz, f"pre of group {e}")


@pytest.mark.parametrize("dt", DT, ids=["bf16", "fp16"])
@pytest.mark.parametrize("g", GROUPED, ids=str)
def test_grouped_backward(dense, g, dt):
    kind, E, R, K, N = g
    off = groups(kind, E, R)
    case("grouped backward", g, dt)
    x, w, dz = rnd(15, R, K, dt=dt), rnd(16, E, N, K, dt=dt, scale=0.1), rnd(17, R, N, dt=dt, scale=0.1)
    first, last = int(off[0]), int(off[-1])
    x[:first], dz[last:] = float("nan"), float("nan")
    dx = torch.full((R, K), 5.0, dtype=dt, device="cuda")
    _, dw, db = dense.grouped_matmul_backward(dz, x, w, off.cuda(), need_db=True, dx=dx)
    dw32 = dense.grouped_matmul_backward(dz, x, w, off.cuda(), need_dx=False, dw_dtype=F32)[1]
    assert (dx[:first] == 5.0).all() and (dx[last:] == 5.0).all()
    for e in range(E):
        r = slice(int(off[e]), int(off[e + 1]))
        x64, w64, d64 = (t.double().cpu() for t in (x[r], w[e], dz[r]))
        n = r.stop - r.start
        if n:
            ref.within(dx[r], d64 @ w64, (N + 2) * 2.0 ** -23 * (d64.abs() @ w64.abs()), f"dx of group {e}")
        want, bound = d64.T @ x64, (n + 2) * 2.0 ** -23 * (d64.abs().T @ x64.abs())
        ref.within(dw[e], want, bound, f"dw of group {e}")
        ref.within(dw32[e], want, bound, f"dw fp32 of group {e}")
        ref.within(db[e], d64.sum(0), (n + 2) * 2.0 ** -23 * d64.abs().sum(0), f"db of group {e}")
    again = dense.grouped_matmul_backward(dz, x, w, off.cuda(), need_db=True, dx=dx.clone())
    assert torch.equal(again[1], dw) and torch.equal(again[2], db)


@pytest.mark.parametrize("T", [1, 9, 150])
def test_grouped_token(dense, T):
    """Rows gathered from x, forward and in dw; a token outside x counts as zeros."""
    E, K, N = 4, 72, 40
    g = torch.Generator().manual_seed(3)
    R = 3 * T
    off = groups("even", E, R)
    token = torch.randint(0, T, (R,), generator=g, dtype=torch.int32)
    token[0], token[R - 1] = -1, T
    for K in (72, 71):
        case("grouped token", T, K)
        x, w, dz = rnd(18, T, K), rnd(19, E, N, K, scale=0.1), rnd(20, R, N, scale=0.1)
        xg = x[token.clamp(0, T - 1).long().cuda()].clone()
        xg[0], xg[R - 1] = 0, 0
        args = (off.cuda(), token.cuda())
        assert torch.equal(dense.grouped_matmul(x, w, *args), dense.grouped_matmul(xg, w, args[0]))
        a = dense.grouped_matmul_backward(dz, x, w, *args, need_db=True)
        b = dense.grouped_matmul_backward(dz, xg, w, args[0], need_db=True)
        assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_grouped_strided_weights(dense):
    """Experts, rows, inputs and outputs apart from each other."""
    E, R, K, N = 3, 50, 56, 24
    off = groups("even", E, R).cuda()
    big = rnd(21, E, N + 2, K + 5)
    w = big[:, 1:1 + N, 2:2 + K]
    x, dz = rnd(22, R, K, wide=7), rnd(23, R, N, wide=3)
    wc, xc, dzc = w.contiguous(), x.contiguous(), dz.contiguous()
    assert torch.equal(dense.grouped_matmul(x, w, off), dense.grouped_matmul(xc, wc, off))
    a, b = dense.grouped_matmul_backward(dz, x, w, off), dense.grouped_matmul_backward(dzc, xc, wc, off)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_offsets_out_of_bounds_are_taken_as_the_bounds(dense):
    E, R, K, N = 4, 40, 64, 32
    x, w = rnd(24, R, K), rnd(25, E, N, K)
    good = torch.tensor([0, 10, 10, 25, 40], dtype=torch.int32, device="cuda")
    wild = torch.tensor([-5, 10, 10, 25, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    assert torch.equal(dense.grouped_matmul(x, w, good), dense.grouped_matmul(x, w, wild))
    a, b = dense.grouped_matmul_backward(x[:, :N].contiguous(), x, w, good), dense.grouped_matmul_backward(
        x[:, :N].contiguous(), x, w, wild)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_no_rows(dense):
    """No rows: empty results, and gradients of the matrices that are zeros."""
    E, K, N = 3, 64, 32
    x, w, off = rnd(26, 0, K), rnd(27, E, N, K), torch.zeros(E + 1, dtype=torch.int32, device="cuda")
    assert dense.grouped_matmul(x, w, off).shape == (0, N)
    dx, dw, db = dense.grouped_matmul_backward(rnd(28, 0, N), x, w, off, need_db=True)
    assert dx.shape == (0, K) and (dw == 0).all() and (db == 0).all()
    g = dense.group_by_expert(torch.zeros(0, 2, dtype=torch.int32, device="cuda"), 5)
    assert g.offsets.tolist() == [0] * 6 and g.token.numel() == 0
    y = rnd(29, 4, 8)
    assert dense.combine(y, torch.zeros(0, 2, dtype=torch.int32, device="cuda")).shape == (0, 8)
    none = torch.zeros(3, 0, dtype=torch.int32, device="cuda")
    assert (dense.combine(y, none) == 0).all()


def test_past_32_bits(dense):
    """Element offsets past 2^31 in the weights, the inputs and the outputs."""
    E, N, K = 9, 16384, 16384                               # 2.4e9 weights
    w = torch.zeros(E, N, K, dtype=BF16, device="cuda")
    w[E - 1, N - 3:].normal_(0, 0.1)
    x = rnd(30, 3, K)
    off = torch.tensor([0] * E + [3], dtype=torch.int32, device="cuda")
    y = dense.grouped_matmul(x, w, off)
    _, _, want, bound = ref.product(x, w[E - 1, N - 3:], None, "none", BF16)
    assert (y[:, :N - 3] == 0).all()
    ref.within(y[:, N - 3:], want, bound)
    dz = rnd(31, 3, N)
    dx, _, _ = dense.grouped_matmul_backward(dz, x, w, off, need_dw=False)
    d64, w64 = dz[:, N - 3:].double().cpu(), w[E - 1, N - 3:].double().cpu()
    ref.within(dx, d64 @ w64, 5 * 2.0 ** -23 * (d64.abs() @ w64.abs()))
    dense.grouped_matmul_backward(dz, x, w, off, need_dx=False, dw=w)
    x64 = x.double().cpu()
    assert (w[:E - 1] == 0).all()
    d64 = dz[:, N - 3:].double().cpu()
    ref.within(w[E - 1, N - 3:], d64.T @ x64, 5 * 2.0 ** -23 * (d64.abs().T @ x64.abs()))
    del w
    T, K = 300000, 8192                                     # 2.5e9 inputs, gathered and in order
    x = torch.zeros(T, K, dtype=BF16, device="cuda")
    x[T - 2:].normal_(0, 1)
    w = rnd(32, 1, 24, K, scale=0.1)
    _, _, want, bound = ref.product(x[T - 2:], w[0], None, "none", BF16)
    tok = torch.tensor([T - 2, T - 1], dtype=torch.int32, device="cuda")
    ref.within(dense.grouped_matmul(x, w, torch.tensor([0, 2], dtype=torch.int32, device="cuda"), token=tok), want, bound)
    y = dense.linear(x, w[0])
    ref.within(y[T - 2:], want, bound)
    assert (y[:T - 2] == 0).all()
    out = dense.combine(x, tok.view(2, 1), out_dtype=F32)
    assert torch.equal(out, x[T - 2:].float())


# ------------------------------------------------------------------ grouping


@pytest.mark.parametrize("T,K,E", [(1, 1, 1), (1, 10, 512), (7, 3, 5), (64, 4, 64), (333, 10, 512), (2000, 2, 3), (5000, 7, 70),
                                   (40, 1, 1000)])
def test_group_by_expert(dense, T, K, E):
    g = torch.Generator().manual_seed(T + E)
    for lo, hi in ((0, E), (-2, E + 2)):
        ids = torch.randint(lo, hi, (T, K), generator=g, dtype=torch.int32)      # an expert may be picked twice by a token
        case("group", T, K, E, lo)
        got = dense.group_by_expert(ids.cuda(), E)
        for a, b in zip(got, ref.grouping(ids, E)):
            assert torch.equal(a.cpu(), b)


def test_group_extreme_ids(dense):
    ids = torch.tensor([[2 ** 31 - 1, -2 ** 31, 3], [3, 0, 4]], dtype=torch.int32)
    for a, b in zip(dense.group_by_expert(ids.cuda(), 4), ref.grouping(ids, 4)):
        assert torch.equal(a.cpu(), b)


# ------------------------------------------------------------------ combine


COMBINE = [(1, 10, 64), (5, 3, 7), (33, 1, 264), (64, 4, 2048), (70, 10, 4096), (9, 20, 2051), (3, 2, 9000)]


def combine_case(T, K, H, dt, seed=0, wide=0):
    g = torch.Generator().manual_seed(seed)
    rows = T * K + 3
    row = torch.randperm(rows, generator=g)[:T * K].int().view(T, K)
    row[T // 2:, K // 2] = -1
    row[0, 0] = rows                                        # one past the end
    w = torch.rand(T, K, generator=g)
    w[T // 2:, K // 2] = float("nan")                       # the weight of a pick that is not there
    y = rnd(40, rows, H, dt=dt, wide=wide)
    used = torch.zeros(rows, dtype=torch.bool)
    used[row[(row >= 0) & (row < rows)].long()] = True
    y[~used.cuda()] = float("nan")
    return row, w, y, used


@pytest.mark.parametrize("dt", DT, ids=["bf16", "fp16"])
@pytest.mark.parametrize("size", COMBINE, ids=str)
def test_combine(dense, size, dt):
    T, K, H = size
    for wide, ot in ((0, dt), (3, F32)):
        case("combine", size, dt, ot, wide)
        row, w, y, _ = combine_case(T, K, H, dt, wide=wide)
        live = (row >= 0) & (row < y.shape[0])
        yg = y.double().cpu()[row.clamp(0, y.shape[0] - 1).long()] * live[..., None]
        yg = torch.where(live[..., None], yg, 0.0)
        res = rnd(41, T, H, dt=ot, wide=wide)
        for weights, r in ((w, None), (w, res), (None, res)):
            f = torch.where(live, w.double() if weights is not None else torch.ones_like(w).double(), 0.0)[..., None]
            want, mag = (yg * f).sum(1), (yg * f).abs().sum(1)
            if r is not None:
                want, mag = want + r.double().cpu(), mag + r.double().cpu().abs()
            args = (y, row.cuda(), None if weights is None else weights.cuda())
            got = dense.combine(*args, residual=r, out_dtype=ot)
            ref.within(got, want, (K + 1) * 2.0 ** -24 * 1.01 * mag)
        o = res.clone()
        dense.combine(y, row.cuda(), residual=o, out=o)
        assert torch.equal(o, got)


@pytest.mark.parametrize("dt", DT, ids=["bf16", "fp16"])
@pytest.mark.parametrize("size", COMBINE, ids=str)
def test_combine_backward(dense, size, dt):
    T, K, H = size
    for wide, gt in ((0, dt), (3, F32)):
        case("combine backward", size, dt, gt, wide)
        row, w, y, used = combine_case(T, K, H, dt, wide=wide)
        live = (row >= 0) & (row < y.shape[0])
        dout = rnd(42, T, H, dt=gt, scale=0.1, wide=wide)
        dy = torch.full(y.shape, 5.0, dtype=dt, device="cuda")
        _, dw = dense.combine_backward(dout, y, row.cuda(), w.cuda(), dy=dy)
        assert (dy[~used.cuda()] == 5.0).all()
        g64, y64 = dout.double().cpu(), y.double().cpu()
        want = torch.zeros(T, K, dtype=torch.float64)
        mag = torch.zeros_like(want)
        for t in range(T):
            for k in range(K):
                if live[t, k]:
                    r = int(row[t, k])
                    want[t, k], mag[t, k] = g64[t] @ y64[r], g64[t].abs() @ y64[r].abs()
                    p = g64[t] * float(w[t, k])
                    ref.within(dy[r], p, 2.0 ** -24 * p.abs(), f"dy {t} {k}")
        ref.within(dw, want, H * 2.0 ** -24 * 1.01 * mag, "dw")
        none, dw2 = dense.combine_backward(dout, y, row.cuda(), w.cuda(), need_dy=False)
        assert none is None and torch.equal(dw, dw2)
        ones, none = dense.combine_backward(dout, y, row.cuda(), need_dw=False, dy=dy.clone())
        assert none is None
        for t in range(T):
            for k in range(K):
                if live[t, k]:
                    assert torch.equal(ones[int(row[t, k])], dout[t].to(dt))


# ------------------------------------------------------------------ activation gradient


@pytest.mark.parametrize("dt", DT, ids=["bf16", "fp16"])
@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu", "swiglu", "sigmoid"])
@pytest.mark.parametrize("size", [(1, 8), (3, 5), (23, 4096), (70, 1001)], ids=str)
def test_act_backward(dense, size, act, dt):
    """Bound: sums of two terms of at most 1.2 |dy| (|u|), each good to 16 steps of fp32."""
    T, n = size
    for wide in (0, 5):
        case("act backward", size, act, dt, wide)
        m = 2 * n if act == "swiglu" else n
        dy, pre = rnd(50, T, n, dt=dt, wide=wide), rnd(51, T, m, dt=dt, scale=3.0, wide=wide)
        pre[0, 0], pre[0, n - 1], pre[0, n // 2] = 60.0, -60.0, 0.0
        want = ref.act_grad(dy.double().cpu(), pre.double().cpu(), act)
        mag = dy.double().cpu().abs()
        if act == "swiglu":
            g, u = pre.double().cpu().chunk(2, 1)
            mag = torch.cat([mag * u.abs(), mag * g.abs()], 1)
        got = dense.act_backward(dy, pre, act)
        ref.within(got, want, 40 * 2.0 ** -24 * mag)
        p = pre.clone()
        assert torch.equal(dense.act_backward(dy, p, act, out=p), got) and torch.equal(p, got)


# ------------------------------------------------------------------ refusals, streams, graphs


def test_refusals(dense):
    x, w = rnd(60, 4, 8), rnd(61, 16, 8)
    off = torch.tensor([0, 4], dtype=torch.int32, device="cuda")
    bad = [lambda: dense.linear(x.float(), w), lambda: dense.linear(x, w.half()), lambda: dense.linear(x, w[:, :7]),
           lambda: dense.linear(x, w, act="tanh"), lambda: dense.linear(x, w[:15], act="swiglu"),
           lambda: dense.linear(x.T, w), lambda: dense.linear(x[0], w), lambda: dense.linear(x, w, bias=w[0, :8]),
           lambda: dense.linear(x, w, residual=x), lambda: dense.linear(x, w, out_dtype=F16),
           lambda: dense.linear(x, w, pre=x), lambda: dense.linear(x, w, out=torch.empty(4, 16, device="cuda").T),
           lambda: dense.linear(x[:1].expand(4, 8), w), lambda: dense.linear(x, w[:0]),
           lambda: dense.linear_backward(x, x, w), lambda: dense.linear_backward(rnd(1, 4, 16), x, w, dw_dtype=F16),
           lambda: dense.linear_backward(rnd(1, 4, 16), x, w, dw=w.T),
           lambda: dense.grouped_matmul(x, w, off), lambda: dense.grouped_matmul(x, w[None], off.long()),
           lambda: dense.grouped_matmul(x, w[None], off[:1]), lambda: dense.grouped_matmul(x, w[None], off.cpu()),
           lambda: dense.grouped_matmul(x, w[None], off, token=off.long()),
           lambda: dense.group_by_expert(off, 4), lambda: dense.group_by_expert(off.view(1, 2), 0),
           lambda: dense.group_by_expert(off.view(1, 2).long(), 4),
           lambda: dense.combine(x, off.view(1, 2), w=torch.ones(2, 1, device="cuda")),
           lambda: dense.combine(x, off.view(1, 2), residual=x), lambda: dense.combine(x.float(), off.view(1, 2)),
           lambda: dense.combine_backward(x, x, off.view(1, 2)), lambda: dense.act_backward(x, x, "swiglu"),
           lambda: dense.act_backward(x, x, "tanh"), lambda: dense.act_backward(x.half(), x, "silu")]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was accepted")


def chain(dense, x, ids, p, gu, down, E, T, K):
    g = dense.group_by_expert(ids, E)
    pre = torch.zeros(T * K, gu.shape[1], dtype=x.dtype, device="cuda")
    h = dense.grouped_matmul(x, gu, g.offsets, token=g.token, act="swiglu", pre=pre)
    y = dense.grouped_matmul(h, down, g.offsets)
    return g, pre, h, y, dense.combine(y, g.row, p, residual=x)


@pytest.mark.parametrize("size", [(1, 2056, 520), (17, 4096, 8200), (130, 4096, 520), (3000, 200, 4104), (50, 71, 57), (700, 4096, 136)],
                         ids=str)
@pytest.mark.parametrize("act", ["none", "swiglu"])
def test_residual_in_place(dense, size, act):
    """residual may be the result: whole tiles, parts joined afterwards and few rows give the bits of a result of its own."""
    T, K, N = size
    x, w, b = rnd(91, T, K), rnd(92, 2 * N, K, scale=0.1), rnd(93, 2 * N)
    cols = N if act == "swiglu" else 2 * N
    res = rnd(94, T, cols + 24)[:, :cols]
    pre = torch.empty(T, 2 * N, dtype=x.dtype, device="cuda")
    want = dense.linear(x, w, bias=b, act=act, residual=res, pre=pre)
    again = torch.empty_like(pre)
    got = dense.linear(x, w, bias=b, act=act, residual=res, out=res, pre=again)
    assert got is res and torch.equal(got, want) and torch.equal(again, pre)


def test_activation_gradient_in_place(dense):
    """dz may be pre, for wide and narrow rows alike."""
    for T, n in ((5, 1001), (300, 512)):
        for act in ("gelu", "swiglu"):
            pre, dy = rnd(95, T, 2 * n if act == "swiglu" else n), rnd(96, T, n)
            want = dense.act_backward(dy, pre, act)
            assert torch.equal(dense.act_backward(dy, pre, act, out=pre), want)


def test_combine_residual_in_place(dense):
    y, p, res = rnd(97, 70, 1001), torch.rand(23, 3, device="cuda"), rnd(98, 23, 1001)
    row = torch.randint(-1, 70, (23, 3), dtype=torch.int32, device="cuda")
    want = dense.combine(y, row, p, residual=res)
    assert torch.equal(dense.combine(y, row, p, residual=res, out=res), want)


def test_popular_experts_first(dense):
    """Groups of very different sizes in descending order, some empty: every tile of every group is computed once."""
    sizes = [700, 260, 257, 256, 130, 129, 64, 33, 16, 5, 1, 0, 0, 1, 0, 40, 0, 3, 0]
    E, H, N, R = len(sizes), 264, 520, sum(sizes) + 7
    off = torch.tensor([0] + sizes).cumsum(0).int().cuda()
    x, w, dz = rnd(99, R, H), rnd(100, E, N, H, scale=0.1), rnd(101, R, N)
    y, dx = torch.full((R, N), 7.0, dtype=x.dtype, device="cuda"), torch.full((R, H), 7.0, dtype=x.dtype, device="cuda")
    dense.grouped_matmul(x, w, off, out=y)
    _, dw, _ = dense.grouped_matmul_backward(dz, x, w, off, dx=dx, dw_dtype=torch.float32)
    assert bool((y[-7:] == 7).all()) and bool((dx[-7:] == 7).all())
    at = 0
    for e, n in enumerate(sizes):
        r = slice(at, at + n)
        X, W, Z = x[r].double(), w[e].double(), dz[r].double()
        # a result's rounding to bf16, and its fp32 sum of up to 700 products in any order
        for got, want, size, half in ((y[r], X @ W.T, X.abs() @ W.abs().T, 2.0 ** -8), (dx[r], Z @ W, Z.abs() @ W.abs(), 2.0 ** -8),
                                      (dw[e], Z.T @ X, Z.abs().T @ X.abs(), 0.0)):
            assert bool(((got.double() - want).abs() <= half * want.abs() + 1.01 * 700 * 2.0 ** -24 * size).all()), e
        at += n


def test_on_another_stream(dense):
    x, w = rnd(62, 300, 512), rnd(63, 384, 512, scale=0.1)
    want = dense.linear(x, w, act="silu")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    got = dense.linear(x, w, act="silu", stream=s)
    with torch.cuda.stream(s):
        also = dense.linear(x, w, act="silu")
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want) and torch.equal(also, want)


def test_a_stream_of_another_device_is_refused(dense):
    from types import SimpleNamespace
    x, w = rnd(62, 5, 64), rnd(63, 24, 64)
    out = torch.empty(5, 24, dtype=x.dtype, device="cuda")
    with pytest.raises(ValueError, match="stream"):
        dense.linear(x, w, out=out, stream=SimpleNamespace(cuda_stream=0, device_index=x.get_device() + 1))


def test_memory_of_the_current_stream_is_not_written_on_another(dense):
    """What a call on another stream writes does not lie where the current stream may still be reading."""
    x, w = rnd(62, 300, 512), rnd(63, 384, 512, scale=0.1)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    held = torch.empty(300, 384, dtype=x.dtype, device="cuda")
    at = held.data_ptr()
    del held                                                # its last use may still be queued
    got = dense.linear(x, w, stream=s)
    assert got.data_ptr() != at
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, dense.linear(x, w))


def test_captured_and_replayed(dense):
    """The block and its gradients under a graph: every replay, with eager work between, gives the eager bits."""
    T, K, E, H, I = 37, 3, 6, 128, 64
    x, p = rnd(64, T, H), torch.rand(T, K, device="cuda")
    gu, down, dout = rnd(65, E, 2 * I, H, scale=0.1), rnd(66, E, H, I, scale=0.1), rnd(67, T, H, scale=0.1)
    ids = torch.randint(-1, E, (T, K), dtype=torch.int32, device="cuda")

    def step():
        g, pre, h, y, out = chain(dense, x, ids, p, gu, down, E, T, K)
        dy, dp = dense.combine_backward(dout, y, g.row, p, dy=torch.zeros_like(y))
        dh, dd, db = dense.grouped_matmul_backward(dy, h, down, g.offsets, need_db=True, dx=torch.zeros_like(h))
        dz = dense.act_backward(dh, pre, "swiglu")
        dxr, dg, _ = dense.grouped_matmul_backward(dz, x, gu, g.offsets, token=g.token)
        return out, dp, dd, db, dg, dense.combine(dxr, g.row), dense.linear(x, down[0].T.contiguous(), act="gelu")

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for n in range(4):
        x.copy_(rnd(70 + n, T, H))
        ids.copy_(torch.randint(-1, E, (T, K), dtype=torch.int32))
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        for i, (a, b) in enumerate(zip(held, want)):
            assert torch.equal(a, b), (n, i)


def test_two_streams_at_once(dense):
    """The same products, in parts and whole, on two streams together: each keeps its own workspace."""
    cases = [(rnd(90, 1000, 2056), rnd(91, 16, 2056, scale=0.1)), (rnd(92, 40, 71), rnd(93, 57, 71, scale=0.1)),
             (rnd(94, 600, 1024), rnd(95, 512, 1024, scale=0.1))]
    want = [(dense.linear(x, w), *dense.linear_backward(rnd(96, x.shape[0], w.shape[0]), x, w, need_db=True)) for x, w in cases]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    dz = [rnd(96, x.shape[0], w.shape[0]) for x, w in cases]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(3):
        for s, keep in zip(streams, got):
            for (x, w), g in zip(cases, dz):
                with torch.cuda.stream(s):
                    keep.append((dense.linear(x, w), *dense.linear_backward(g, x, w, need_db=True)))
    torch.cuda.synchronize()
    for keep in got:
        for i, r in enumerate(keep):
            assert all(torch.equal(a, b) for a, b in zip(r, want[i % len(cases)]))


def test_parts_and_copies_captured(dense):
    """A product in parts and one whose operands are copied, under a graph, replayed between eager calls."""
    x, w, dz = rnd(97, 1000, 2055), rnd(98, 16, 2055, scale=0.1), rnd(99, 1000, 16)
    step = lambda: (dense.linear(x, w, act="silu"), *dense.linear_backward(dz, x, w, need_db=True, dw_dtype=F32))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for n in range(4):
        x.copy_(rnd(100 + n, 1000, 2055))
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want)), n
