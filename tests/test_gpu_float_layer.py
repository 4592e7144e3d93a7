"""FloatMoELayer: the 16-bit operators run together, forward and backward,
against the same block in 64 bits.

Bounds are carried through the chain element by element: every stage's result
is rounded to 16 bits (eps / 2 of its value), a product passes an input's error
on through the other operand's magnitudes and adds its own sums' error
(dense_ref.py), an activation passes it on with its largest slope (1.1 for
silu, whose own slope changes by at most 0.5 per unit)."""
import numpy as np
import pytest
import torch

from dense_ref import rounding, within

pytestmark = pytest.mark.gpu

DT = [torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def dense():
    assert torch.cuda.is_available(), "GPU tests need a HIP device"
    from winmoe_amd import _lib, dense
    _lib.load()
    return dense


def rnd(seed, *shape, dt, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dt).cuda()


def d(t):
    return t.detach().double().cpu()


class Err:
    """A 64-bit value and a bound of what the 16-bit chain's value may be off by."""

    def __init__(self, v, e=None, dt=None):
        self.v, self.e = v, torch.zeros_like(v) if e is None else e
        if dt is not None:
            self.e = self.e + rounding(v.abs() + self.e, dt)

    def mm(self, w, dt=None):
        """self @ w (w exact or with a bound), sums in fp32, rounded to dt."""
        w = w if isinstance(w, Err) else Err(w)
        a, n = self.v.abs() + self.e, self.v.shape[1]
        e = self.e @ (w.v.abs() + w.e) + self.v.abs() @ w.e + (n + 2) * 2.0 ** -23 * (a @ (w.v.abs() + w.e))
        return Err(self.v @ w.v, e, dt)

    @property
    def T(self):
        return Err(self.v.T, self.e.T)


def silu(g):
    return g * torch.sigmoid(g)


def ffn(x, gu, down, dt):
    """(pre, h, y) of one expert's rows x."""
    z = Err(x).mm(gu.T)
    g, u = z.v.chunk(2, 1)
    dg, du = z.e.chunk(2, 1)
    h = Err(silu(g) * u, 1.1 * dg * (u.abs() + du) + silu(g).abs() * du + 2.0 ** -20 * (silu(g) * u).abs(), dt)
    return Err(z.v, z.e, dt), h, h.mm(down.T, dt)


def ffn_backward(x, gu, down, pre, h, dy, dt):
    """(dx rows, dgu, ddown) given dy."""
    dh = dy.mm(down, dt)
    g, u = pre.v.chunk(2, 1)
    eg, eu = pre.e.chunk(2, 1)
    s = torch.sigmoid(g)
    slope = s * (1 + g * (1 - s))
    vg, vu = dh.v * u * slope, dh.v * silu(g)
    a = dh.v.abs() + dh.e
    fg = dh.e * (u * slope).abs() + a * eu * 1.1 + a * (u.abs() + eu) * 0.5 * eg + 2.0 ** -20 * a * u.abs()
    fu = dh.e * silu(g).abs() + a * 1.1 * eg + 2.0 ** -20 * a * g.abs()
    dz = Err(torch.cat([vg, vu], 1), torch.cat([fg, fu], 1), dt)
    return dz.mm(gu, dt), dz.T.mm(x), dy.T.mm(h)


def make(dense, dt, T, E, K, H, I, shared, seed=0):
    Is = I + 8
    L = dense.FloatMoELayer(rnd(seed + 1, E, 2 * I, H, dt=dt, scale=0.1), rnd(seed + 2, E, H, I, dt=dt, scale=0.1), K,
                            router=rnd(seed + 7, E, H, dt=torch.float32),
                            shared_gate_up=rnd(seed + 3, 2 * Is, H, dt=dt, scale=0.1) if shared else None,
                            shared_down=rnd(seed + 4, H, Is, dt=dt, scale=0.1) if shared else None,
                            shared_gate=rnd(seed + 5, 1, H, dt=dt, scale=0.1) if shared == 2 else None)
    g = torch.Generator().manual_seed(seed)
    ids = torch.stack([torch.randperm(E, generator=g)[:K] for _ in range(T)]).int() if T else torch.zeros(0, K).int()
    if T > 4:
        ids[T - 2:] = -1                                    # padding
        ids[1, 0] = ids[1, K - 1]                           # the same expert twice
    w = torch.rand(T, K, generator=g)
    return L, rnd(seed + 6, T, H, dt=dt), ids, w


@pytest.mark.parametrize("dt", DT, ids=["bf16", "fp16"])
@pytest.mark.parametrize("T,E,K,H,I,shared", [(1, 8, 2, 64, 32, 0), (1, 16, 4, 512, 128, 2), (9, 4, 3, 72, 40, 1),
                                              (60, 8, 2, 136, 64, 2), (150, 3, 2, 67, 33, 2), (300, 2, 1, 256, 128, 0)])
def test_layer(dense, T, E, K, H, I, shared, dt):
    print("[case] layer", T, E, K, H, I, shared, dt, flush=True)
    L, x, ids, w = make(dense, dt, T, E, K, H, I, shared)
    res, dout = rnd(20, T, H, dt=torch.float32), rnd(21, T, H, dt=torch.float32, scale=0.1)
    out, kept = L.forward(x, ids.cuda(), w.cuda(), residual=res, keep=True)
    assert torch.equal(out, L.forward(x, ids.cuda(), w.cuda(), residual=res))
    G = L.backward(dout, kept, dw_dtype=torch.float32)

    x64, do = d(x), d(dout)
    want, bound = d(res), torch.zeros(T, H, dtype=torch.float64)
    dx, bdx = torch.zeros(T, H, dtype=torch.float64), torch.zeros(T, H, dtype=torch.float64)
    wdw, bdw = torch.zeros(T, K, dtype=torch.float64), torch.zeros(T, K, dtype=torch.float64)
    zero = torch.zeros(0)
    for e in range(E):
        tk = (ids == e).nonzero()
        gu, down = d(L.gate_up[e]), d(L.down[e])
        if not len(tk):
            assert (G.gate_up[e] == 0).all() and (G.down[e] == 0).all()
            continue
        t, k = tk[:, 0], tk[:, 1]
        wt = w[t, k].double()[:, None]
        pre, h, y = ffn(x64[t], gu, down, dt)
        want.index_add_(0, t, wt * y.v)
        bound.index_add_(0, t, wt * y.e + 2.0 ** -22 * wt * y.v.abs())
        wdw[t, k], bdw[t, k] = (do[t] * y.v).sum(1), (do[t].abs() * (y.e + H * 2.0 ** -23 * y.v.abs())).sum(1)
        dxr, dgu, ddown = ffn_backward(x64[t], gu, down, pre, h, Err(wt * do[t], 2.0 ** -23 * (wt * do[t]).abs(), dt), dt)
        dx.index_add_(0, t, dxr.v)
        bdx.index_add_(0, t, dxr.e + 2.0 ** -22 * dxr.v.abs())
        within(G.gate_up[e], dgu.v, dgu.e, f"gate_up {e}")
        within(G.down[e], ddown.v, ddown.e, f"down {e}")
    if shared:
        gu, down = d(L.shared_gate_up), d(L.shared_down)
        pre, h, y = ffn(x64, gu, down, dt)
        s, bs = torch.ones(T, 1, dtype=torch.float64), torch.zeros(T, 1, dtype=torch.float64)
        if shared == 2:
            z = Err(x64).mm(d(L.shared_gate).T)
            s, bs = torch.sigmoid(z.v), 0.25 * z.e + 2.0 ** -21
        want += s * y.v
        bound += s * y.e + bs * (y.v.abs() + y.e) + 2.0 ** -22 * y.v.abs()
        dy = Err(s * do, bs * do.abs() + 2.0 ** -23 * do.abs(), dt)
        dxr, dgu, ddown = ffn_backward(x64, gu, down, pre, h, dy, dt)
        dx, bdx = dx + dxr.v, bdx + dxr.e + 2.0 ** -22 * dxr.v.abs()
        within(G.shared_gate_up, dgu.v, dgu.e, "shared gate_up")
        within(G.shared_down, ddown.v, ddown.e, "shared down")
        if shared == 2:
            ds, es = (do * y.v).sum(1, keepdim=True), (do.abs() * (y.e + H * 2.0 ** -23 * y.v.abs())).sum(1, keepdim=True)
            dz = Err(ds * s * (1 - s), es * 0.25 + bs * (ds.abs() + es) + 2.0 ** -22 * ds.abs(), dt)
            dxg, dg = dz.mm(d(L.shared_gate), dt), dz.T.mm(x64)
            dx, bdx = dx + dxg.v, bdx + dxg.e + 2.0 ** -22 * dxg.v.abs()
            within(G.shared_gate, dg.v, dg.e, "shared gate")
    within(out, want, bound + 2.0 ** -22 * want.abs(), "out")
    within(G.w, wdw, bdw, "dw")
    within(G.x, dx, bdx, "dx")


def plain(p, x, ids, w):
    """The block in 64 bits (routed experts)."""
    out = torch.zeros_like(x)
    for e in range(p["gate_up"].shape[0]):
        tk = (ids == e).nonzero()
        if len(tk):
            g, u = (x[tk[:, 0]] @ p["gate_up"][e].T).chunk(2, 1)
            out = out.index_add(0, tk[:, 0], w[tk[:, 0], tk[:, 1]][:, None] * ((silu(g) * u) @ p["down"][e].T))
    return out


def test_gradients_against_differences(dense):
    """<gradient, v> against (f(p + s v) - f(p - s v)) / 2 s of the block in 64
    bits, along the gradient itself and a random direction.

    The gradient passes six roundings of 2^-12 (fp16) and its fp32 sums; along
    itself their effects add up to at most 7 * 2^-12 of the product of the norms
    of what they multiply, which the factor 4 (norms of products of the chain's
    factors against the product's own norm, here of well-mixed random values)
    covers; the same limit holds for any direction, relative to |gradient| |v|."""
    dt, T, E, K, H, I = torch.float16, 40, 4, 2, 96, 48
    L, x, ids, w = make(dense, dt, T, E, K, H, I, 0, seed=50)
    dout = rnd(60, T, H, dt=torch.float32, scale=0.1)
    _, kept = L.forward(x, ids.cuda(), w.cuda(), keep=True)
    G = L.backward(dout, kept, dw_dtype=torch.float32)
    p = {"gate_up": d(L.gate_up), "down": d(L.down)}
    args, do = {"x": d(x), "w": w.double(), **p}, d(dout)

    def loss(a):
        return float((plain(a, a["x"], ids, a["w"]) * do).sum())

    for name, grad in (("x", G.x), ("w", G.w), ("gate_up", G.gate_up), ("down", G.down)):
        grad = d(grad)
        for v in (grad / grad.norm(), torch.randn(grad.shape, generator=torch.Generator().manual_seed(3), dtype=torch.float64)):
            s = 1e-5 / float(v.abs().max())
            hi, lo = loss({**args, name: args[name] + s * v}), loss({**args, name: args[name] - s * v})
            diff = (hi - lo) / (2 * s)
            assert abs(float((grad * v).sum()) - diff) <= 4 * 7 * 2.0 ** -12 * float(grad.norm() * v.norm()), name


def test_no_tokens_and_refusals(dense):
    L, x, ids, w = make(dense, torch.bfloat16, 0, 4, 2, 64, 32, 2)
    out, kept = L.forward(x, ids.cuda(), w.cuda(), keep=True)
    assert out.shape == (0, 64)
    G = L.backward(out, kept)
    assert (G.gate_up == 0).all() and (G.shared_down == 0).all() and G.x.shape == (0, 64)
    L, x, ids, w = make(dense, torch.bfloat16, 6, 4, 2, 64, 32, 0)
    for bad in (lambda: L.forward(x.float(), ids.cuda(), w.cuda()), lambda: L.forward(x, ids.cuda()[:, :1], w.cuda()),
                lambda: L.forward(x, ids.cuda(), w.cuda().double()), lambda: L.forward(x[:, :8], ids.cuda(), w.cuda()),
                lambda: dense.FloatMoELayer(L.gate_up, L.down, 5), lambda: dense.FloatMoELayer(L.gate_up, L.gate_up, 2),
                lambda: dense.FloatMoELayer(L.gate_up, L.down, 2, shared_down=L.down[0])):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize("ggml_type", [1, 30])
@pytest.mark.parametrize("shared", [False, True])
def test_layer_from_gguf(dense, tmp_path, ggml_type, shared):
    """A file's F16 or BF16 experts make the layer that its tensors make directly; its router picks as router_topk."""
    from winmoe_amd import gguf
    dt = torch.float16 if ggml_type == 1 else torch.bfloat16
    E, K, H, I, Is = 4, 2, 64, 32, 48
    raw = lambda t: t.cpu().contiguous().view(torch.int16).numpy().tobytes()
    t = {n: rnd(70 + i, *s, dt=dt, scale=0.1) for i, (n, s) in enumerate(
        {"ffn_gate_exps": (E, I, H), "ffn_up_exps": (E, I, H), "ffn_down_exps": (E, H, I), "ffn_gate_shexp": (Is, H),
         "ffn_up_shexp": (Is, H), "ffn_down_shexp": (H, Is)}.items()) if shared or "shexp" not in n}
    router, gi = rnd(80, E, H, dt=torch.float32), rnd(81, H, dt=torch.float32, scale=0.1)
    tensors = [(f"blk.0.{n}.weight", tuple(reversed(v.shape)), ggml_type, raw(v)) for n, v in t.items()]
    tensors.append(("blk.0.ffn_gate_inp.weight", (H, E), 0, router.cpu().numpy().tobytes()))
    if shared:
        tensors.append(("blk.0.ffn_gate_inp_shexp.weight", (H,), 0, gi.cpu().numpy().tobytes()))
    path = str(tmp_path / "m.gguf")
    gguf.write_gguf(path, {"general.architecture": "t", "t.expert_used_count": K}, tensors)
    L = gguf.moe_layer_from_gguf(gguf.GGUFFile(path), 0)
    assert isinstance(L, dense.FloatMoELayer) and L.K == K
    cat = lambda a, b: torch.cat([t[a], t[b]], -2).contiguous()
    sh = dict(shared_gate_up=cat("ffn_gate_shexp", "ffn_up_shexp"), shared_down=t["ffn_down_shexp"],
              shared_gate=gi.to(dt).view(1, H)) if shared else {}
    M = dense.FloatMoELayer(cat("ffn_gate_exps", "ffn_up_exps"), t["ffn_down_exps"], K, router=router, **sh)
    x = rnd(90, 5, H, dt=dt)
    ids, w = L.route(x)
    logits = d(x) @ d(router).T
    assert np.array_equal(np.sort(ids.cpu().numpy()), np.sort(logits.topk(K, 1).indices.numpy().astype(np.int32)))
    assert torch.allclose(d(w), torch.softmax(logits.gather(1, ids.cpu().long()), 1), atol=1e-5)
    assert torch.equal(L.forward(x, ids, w), M.forward(x, ids, w))


def test_gguf_of_mixed_types_is_refused(dense, tmp_path):
    from winmoe_amd import gguf
    E, H, I = 2, 64, 32
    z = lambda n: bytes(n * 2)
    tensors = [("blk.0.ffn_gate_exps.weight", (H, I, E), 1, z(E * H * I)), ("blk.0.ffn_up_exps.weight", (H, I, E), 30, z(E * H * I)),
               ("blk.0.ffn_down_exps.weight", (I, H, E), 1, z(E * H * I))]
    path = str(tmp_path / "m.gguf")
    gguf.write_gguf(path, {"general.architecture": "t", "t.expert_used_count": 1}, tensors)
    with pytest.raises(gguf.GGUFError, match="not supported"):
        gguf.moe_layer_from_gguf(gguf.GGUFFile(path), 0)
