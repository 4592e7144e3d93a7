"""The products of an expert layer whose weights are held in 16 bits, as cases that can be timed and checked.

Five operators, as a mixture-of-experts block in fp16 or bf16 runs them for one token, for a prompt and in training:
grouping the (token, pick) pairs by expert, the products grouped by expert with their gradients, the plain product with
bias, activation and residual with its gradients, the activation's gradient, and the weighted sum over a token's picks
with its gradients.  Sizes are those of the layers that the library's benchmark names (64 experts, hidden 2048, inner
512, 4 picks; 512 experts, hidden 4096, inner 1024, 10 picks).  Weights are N(0, 0.02), activations N(0, 1), gradients
N(0, 0.01); experts are picked by a skewed popularity (r^-0.456 over a random order), as in that benchmark.
"""
import math

import numpy as np
import torch

own = False

DTYPE = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


# ------------------------------------------------------------------ cases


def listed():
    return [
        # the pairs of one generated token: the shortest call there is, all latency
        {"name": "group_1", "do": "group", "T": 1, "K": 10, "E": 512, "pad": 0},
        # the pairs of a long prompt in a padded batch (the picks of padding are -1)
        {"name": "group_4096", "do": "group", "T": 4096, "K": 10, "E": 512, "pad": 96},
        # gate and up with SwiGLU for one generated token: ten experts' matrices are streamed for one row each
        {"name": "grouped_1_swiglu", "do": "grouped", "T": 1, "K": 10, "E": 512, "in": 4096, "out": 1024, "pad": 0,
         "dtype": "bf16", "act": "swiglu", "bias": False, "pre": False, "gather": True, "y": "bf16"},
        # the down projection of a prompt chunk: about ten rows an expert, every matrix read
        {"name": "grouped_512_down", "do": "grouped", "T": 512, "K": 10, "E": 512, "in": 1024, "out": 4096, "pad": 0,
         "dtype": "fp16", "act": "none", "bias": False, "pre": False, "gather": False, "y": "fp16"},
        # training: gradients of a small layer's gate/up inputs, matrices and biases for a whole batch
        {"name": "grouped_bwd_4096", "do": "grouped_bwd", "T": 4096, "K": 4, "E": 64, "in": 2048, "out": 1024,
         "pad": 0, "dtype": "bf16", "gather": True, "db": True, "dw": "bf16"},
        # a projection of one generated token: bias and residual in the same call
        {"name": "linear_1", "do": "linear", "T": 1, "in": 4096, "out": 4096, "dtype": "bf16", "act": "none",
         "bias": True, "res": True, "pre": False, "strided": False, "y": "bf16"},
        # a dense block's gate and up for a long prompt: the largest product
        {"name": "linear_4096_swiglu", "do": "linear", "T": 4096, "in": 4096, "out": 8192, "dtype": "bf16",
         "act": "swiglu", "bias": False, "res": False, "pre": False, "strided": False, "y": "bf16"},
        # training: gradients of a projection of odd sizes, the matrix's in fp32 for sums over several batches
        {"name": "linear_bwd_1001", "do": "linear_bwd", "T": 1001, "in": 4096, "out": 2047, "dtype": "fp16",
         "db": True, "dw": "fp32"},
        # the activation's gradient for a few rows
        {"name": "act_bwd_23_gelu", "do": "act_bwd", "T": 23, "out": 4096, "act": "gelu", "dtype": "fp16"},
        # SwiGLU's gradient for all pairs of a batch
        {"name": "act_bwd_16384_swiglu", "do": "act_bwd", "T": 16384, "out": 1024, "act": "swiglu", "dtype": "bf16"},
        # the weighted sum over the picks of a padded prompt chunk, added to the residual stream
        {"name": "combine_512", "do": "combine", "T": 512, "K": 10, "H": 4096, "dtype": "bf16", "pad": 31,
         "y": "fp32", "res": True},
        # its gradients for a whole batch: the rows' and the routing weights'
        {"name": "combine_bwd_4096", "do": "combine_bwd", "T": 4096, "K": 10, "H": 4096, "dtype": "bf16", "pad": 96,
         "y": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def _size(rng, lo, hi):
    """A matrix dimension: a multiple of 64 mostly, else of 8, else any."""
    n, kind = _log(rng, lo, hi), rng.random()
    step = 64 if kind < 0.6 else 8 if kind < 0.85 else 1
    return max(step, min(hi, n // step * step))


def _drawn(rng):
    do = rng.choice(["group", "grouped", "grouped", "grouped", "grouped_bwd", "grouped_bwd", "linear", "linear", "linear",
                     "linear_bwd", "act_bwd", "combine", "combine_bwd"])
    dt = rng.choice(["bf16", "fp16"])
    T = _log(rng, 1, 4096)
    if do == "act_bwd":
        return {"do": do, "T": _log(rng, 1, 16384), "out": _size(rng, 64, 4096),
                "act": rng.choice(["relu", "silu", "gelu", "swiglu", "swiglu"]), "dtype": dt}
    if do in ("linear", "linear_bwd"):
        c = {"do": do, "T": T, "in": _size(rng, 64, 8192), "out": _size(rng, 16, 16384), "dtype": dt}
        if do == "linear":
            c.update(act=rng.choice(["none", "none", "relu", "silu", "gelu", "swiglu"]), bias=rng.random() < 0.5,
                     res=rng.random() < 0.4, pre=rng.random() < 0.3, strided=rng.random() < 0.3,
                     y=rng.choice([dt, dt, "fp32"]))
        else:
            c.update(db=rng.random() < 0.5, dw=rng.choice([dt, "fp32"]))
        return c
    E = _log(rng, 4, 512)
    c = {"do": do, "T": T, "K": rng.randint(1, min(10, E)), "E": E, "pad": rng.randint(0, T // 4)}
    if do == "group":
        return c
    if do in ("combine", "combine_bwd"):
        c.update(H=_size(rng, 256, 4096), dtype=dt, y=rng.choice([dt, "fp32"]))
        if do == "combine":
            c["res"] = rng.random() < 0.5
        del c["E"]
        return c
    c.update({"in": _size(rng, 128, 4096), "out": _size(rng, 128, 4096), "dtype": dt, "gather": rng.random() < 0.5})
    if do == "grouped":
        c.update(act=rng.choice(["none", "none", "silu", "gelu", "swiglu", "swiglu"]), bias=rng.random() < 0.3,
                 pre=rng.random() < 0.3, y=rng.choice([dt, dt, "fp32"]))
    else:
        c.update(db=rng.random() < 0.5, dw=rng.choice([dt, "fp32"]))
    return c


def draw(rng):
    # what moves or computes more than the largest listed cases is drawn again
    while True:
        c = _drawn(rng)
        w = work(c)
        if w["bytes"] <= 4.4e9 and w["flops"] <= 5.6e11 and _weights(c) <= 1 << 32:
            return c


# ------------------------------------------------------------------ inputs


def _rows(c):
    """Rows of the weight matrix: twice the outputs where gate and up are stacked."""
    return c["out"] * (2 if c.get("act") == "swiglu" else 1)


def _weights(c):
    return c.get("E", 1) * c["in"] * _rows(c) if "in" in c else 0


def _picks(c, rng):
    """Skewed picks without repeats [T][K]; those of the last `pad` tokens are -1."""
    T, K, E = c["T"], c["K"], c["E"]
    p = np.arange(1, E + 1) ** -0.456
    keys = np.log(p)[rng.permutation(E)] + rng.gumbel(size=(T, E))
    ids = np.argsort(-keys, axis=1)[:, :K].astype(np.int32)
    ids[T - c["pad"]:] = -1
    return ids


def _grouping(ids, E):
    """Pairs sorted by expert on the host: (offsets [E+1], token of each row, row of each pair)."""
    key = np.where((ids >= 0) & (ids < E), ids, E).reshape(-1)
    order = np.argsort(key, kind="stable").astype(np.int32)
    offsets = np.zeros(E + 1, np.int32)
    offsets[1:] = np.cumsum(np.bincount(key, minlength=E + 1)[:E])
    token = np.where(np.arange(key.size) < offsets[E], order // ids.shape[1], -1).astype(np.int32)
    row = np.empty(key.size, np.int32)
    row[order] = np.arange(key.size, dtype=np.int32)
    return offsets, token, np.where(key < E, row, -1).astype(np.int32).reshape(ids.shape)


def _normal(shape, scale, dt, g):
    t = torch.empty(shape, dtype=DTYPE[dt], device="cuda")
    v = t.view(shape[0], -1)
    step = max(1, (1 << 28) // v.shape[1])
    for i in range(0, shape[0], step):
        v[i:i + step].normal_(0.0, scale, generator=g)
    return t


def _inputs(c, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    rng = np.random.default_rng(seed)
    do, T, dt = c["do"], c["T"], c.get("dtype")
    dev = lambda a: torch.from_numpy(a).cuda()
    s = {}
    if do == "act_bwd":
        s["dy"] = _normal((T, c["out"]), 0.01, dt, g)
        s["pre"] = _normal((T, _rows(c)), 1.0, dt, g)
    elif do == "group":
        s["ids"] = dev(_picks(c, rng))
    elif do in ("linear", "linear_bwd"):
        s["w"] = _normal((_rows(c), c["in"]), 0.02, dt, g)
        if do == "linear":
            # a strided input is a column range of a wider tensor, as a fused projection's output is split
            s["x"] = _normal((T, c["in"] + (64 if c["strided"] else 0)), 1.0, dt, g)[:, :c["in"]]
            s["bias"] = _normal((1, _rows(c)), 0.5, dt, g).view(-1) if c["bias"] else None
            s["res"] = _normal((T, c["out"]), 1.0, dt, g) if c["res"] else None
        else:
            s["x"] = _normal((T, c["in"]), 1.0, dt, g)
            s["dz"] = _normal((T, _rows(c)), 0.01, dt, g)
    elif do in ("combine", "combine_bwd"):
        T, K = c["T"], c["K"]
        row = rng.permutation(T * K).astype(np.int32).reshape(T, K)
        row[T - c["pad"]:] = -1
        p = np.exp(rng.standard_normal((T, K)))
        s.update(row=dev(row), w=dev((p / p.sum(1, keepdims=True)).astype(np.float32)),
                 y=_normal((T * K, c["H"]), 1.0, dt, g))
        if do == "combine":
            s["res"] = _normal((T, c["H"]), 1.0, c["y"], g) if c["res"] else None
        else:
            s["dout"] = _normal((T, c["H"]), 0.01, c["y"], g)
    else:
        offsets, token, _ = _grouping(_picks(c, rng), c["E"])
        R = token.size
        s.update(offsets=dev(offsets), token=dev(token) if c["gather"] else None,
                 x=_normal((T if c["gather"] else R, c["in"]), 1.0, dt, g),
                 w=_normal((c["E"], _rows(c), c["in"]), 0.02, dt, g))
        if do == "grouped":
            s["bias"] = _normal((c["E"], _rows(c)), 0.5, dt, g) if c["bias"] else None
        else:
            s["dz"] = _normal((R, _rows(c)), 0.01, dt, g)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    c = s["case"] = case
    do, dt, T = c["do"], c.get("dtype"), c["T"]
    zeros = lambda shape, t: torch.zeros(shape, dtype=DTYPE[t], device="cuda")
    # buffers that a program keeps from call to call; rows that no expert takes stay as they are
    if do == "grouped":
        R = T * c["K"]
        s["out"] = zeros((R, c["out"]), c["y"])
        s["pre"] = zeros((R, _rows(c)), dt) if c["pre"] else None
    elif do == "grouped_bwd":
        s["dx"] = zeros((T * c["K"], c["in"]), dt)
    elif do == "linear":
        s["pre"] = zeros((T, _rows(c)), dt) if c["pre"] else None
    elif do == "combine_bwd":
        s["dy"] = zeros((T * c["K"], c["H"]), dt)
    return s


# ------------------------------------------------------------------ one pass


def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    from winmoe_amd import dense
    c, do = s["case"], s["case"]["do"]
    if do == "group":
        return tuple(dense.group_by_expert(s["ids"], c["E"]))
    if do == "act_bwd":
        return dense.act_backward(s["dy"], s["pre"], c["act"])
    if do == "linear":
        y = dense.linear(s["x"], s["w"], bias=s["bias"], act=c["act"], residual=s["res"], pre=s["pre"],
                         out_dtype=DTYPE[c["y"]])
        return (y, s["pre"]) if c["pre"] else y
    if do == "linear_bwd":
        dx, dw, db = dense.linear_backward(s["dz"], s["x"], s["w"], need_db=c["db"], dw_dtype=DTYPE[c["dw"]])
        return (dx, dw, db) if c["db"] else (dx, dw)
    if do == "combine":
        return dense.combine(s["y"], s["row"], s["w"], residual=s["res"], out_dtype=DTYPE[c["y"]])
    if do == "combine_bwd":
        return dense.combine_backward(s["dout"], s["y"], s["row"], s["w"], dy=s["dy"])
    if do == "grouped":
        dense.grouped_matmul(s["x"], s["w"], s["offsets"], token=s["token"], bias=s["bias"], act=c["act"],
                             out=s["out"], pre=s["pre"])
        return (s["out"], s["pre"]) if c["pre"] else s["out"]
    dx, dw, db = dense.grouped_matmul_backward(s["dz"], s["x"], s["w"], s["offsets"], token=s["token"],
                                               need_db=c["db"], dw_dtype=DTYPE[c["dw"]], dx=s["dx"])
    return (dx, dw, db) if c["db"] else (dx, dw)


def _act(z, act):
    if act == "swiglu":
        n = z.shape[1] // 2
        return z[:, :n] * torch.sigmoid(z[:, :n]) * z[:, n:]
    if act == "silu":
        return z * torch.sigmoid(z)
    if act == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    return z.clamp(min=0) if act == "relu" else z


def _act_grad(dy, z, act):
    """dL/dz of y = act(z)."""
    if act == "relu":
        return torch.where(z > 0, dy, torch.zeros_like(dy))
    if act == "gelu":
        return dy * (0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi))
    g = z[:, :dy.shape[1]]
    sg = torch.sigmoid(g)
    dsilu = sg * (1.0 + g * (1.0 - sg))
    if act == "silu":
        return dy * dsilu
    return torch.cat([dy * z[:, dy.shape[1]:] * dsilu, dy * g * sg], 1)


def _run_plain(s):
    c, do = s["case"], s["case"]["do"]
    dt = DTYPE.get(c.get("dtype"))
    if do == "group":
        ids, E, K = s["ids"], c["E"], c["K"]
        key = torch.where((ids >= 0) & (ids < E), ids, torch.full_like(ids, E)).view(-1)
        order = torch.argsort(key, stable=True)
        offsets = torch.zeros(E + 1, dtype=torch.int32, device=ids.device)
        offsets[1:] = torch.cumsum(torch.bincount(key, minlength=E + 1)[:E], 0)
        at = torch.arange(key.numel(), dtype=torch.int32, device=ids.device)
        token = torch.where(at < offsets[E], (order // K).int(), torch.full_like(at, -1))
        row = torch.empty_like(at)
        row[order] = at
        return offsets, token, torch.where(key < E, row, torch.full_like(row, -1)).view(ids.shape)
    if do == "act_bwd":
        return _act_grad(s["dy"].float(), s["pre"].float(), c["act"]).to(dt)
    if do == "linear":
        z = s["x"].float() @ s["w"].float().T
        if c["bias"]:
            z = z + s["bias"].float()
        y = _act(z, c["act"])
        if c["res"]:
            y = y + s["res"].float()
        y = y.to(DTYPE[c["y"]])
        return (y, z.to(dt)) if c["pre"] else y
    if do == "linear_bwd":
        dz = s["dz"].float()
        out = ((dz @ s["w"].float()).to(dt), (dz.T @ s["x"].float()).to(DTYPE[c["dw"]]))
        return out + (dz.sum(0),) if c["db"] else out
    if do == "combine":
        y = torch.zeros((c["T"], c["H"]), device="cuda") if s["res"] is None else s["res"].float()
        for k in range(c["K"]):
            r = s["row"][:, k]
            y = y + torch.where((r >= 0)[:, None], s["w"][:, k, None] * s["y"][r.clamp(min=0)].float(), 0.0)
        return y.to(DTYPE[c["y"]])
    if do == "combine_bwd":
        dout, dy = s["dout"].float(), s["dy"]
        dw = torch.zeros_like(s["w"])
        for k in range(c["K"]):
            r = s["row"][:, k]
            live = (r >= 0).nonzero().view(-1)
            at = r[live].long()
            dy[at] = (s["w"][live, k, None] * dout[live]).to(dt)
            dw[live, k] = (dout[live] * s["y"][at].float()).sum(1)
        return dy, dw
    x, w, token, off = s["x"], s["w"], s["token"], s["offsets"].tolist()
    rows = lambda a, b: x[a:b].float() if token is None else x[token[a:b].long()].float()
    if do == "grouped":
        for e in range(c["E"]):
            a, b = off[e], off[e + 1]
            if a == b:
                continue
            z = rows(a, b) @ w[e].float().T
            if c["bias"]:
                z = z + s["bias"][e].float()
            s["out"][a:b] = _act(z, c["act"]).to(DTYPE[c["y"]])
            if c["pre"]:
                s["pre"][a:b] = z.to(dt)
        return (s["out"], s["pre"]) if c["pre"] else s["out"]
    dw = torch.zeros(w.shape, dtype=DTYPE[c["dw"]], device="cuda")
    db = torch.zeros(w.shape[:2], device="cuda")
    for e in range(c["E"]):
        a, b = off[e], off[e + 1]
        if a == b:
            continue
        dz = s["dz"][a:b].float()
        s["dx"][a:b] = (dz @ w[e].float()).to(dt)
        dw[e] = (dz.T @ rows(a, b)).to(dw.dtype)
        db[e] = dz.sum(0)
    return (s["dx"], dw, db) if c["db"] else (s["dx"], dw)


# ------------------------------------------------------------------ what a pass needs


def _used(c):
    """Experts that a call's picks reach, in expectation."""
    p = np.arange(1, c["E"] + 1) ** -0.456
    return float(np.sum(1.0 - (1.0 - np.minimum(1.0, c["K"] * p / p.sum())) ** (c["T"] - c["pad"])))


def work(case):
    c, do, T = case, case["do"], case["T"]
    b = BYTES.get(c.get("dtype"), 0)
    if do == "group":
        n = T * c["K"]
        return {"bytes": 12 * n + 4 * (c["E"] + 1), "flops": n}
    if do == "act_bwd":
        n = T * c["out"]
        return {"bytes": b * (n + 2 * T * _rows(c)), "flops": 10 * n}
    if do in ("combine", "combine_bwd"):
        K, H, Tv = c["K"], c["H"], T - c["pad"]
        yb = BYTES[c["y"]]
        if do == "combine":
            return {"bytes": Tv * K * H * b + T * H * yb * (2 if c["res"] else 1) + 8 * T * K, "flops": 2 * Tv * K * H}
        return {"bytes": 2 * Tv * K * H * b + Tv * H * yb + 12 * T * K, "flops": 3 * Tv * K * H}
    K, N = c["in"], _rows(c)
    if do in ("linear", "linear_bwd"):
        if do == "linear":
            n = b * (T * K + N * K) + T * c["out"] * BYTES[c["y"]]
            n += b * (N * c["bias"] + T * c["out"] * c["res"] + T * N * c["pre"])
            return {"bytes": n, "flops": 2 * T * N * K}
        return {"bytes": b * (2 * T * K + N * K + T * N) + N * K * BYTES[c["dw"]] + 4 * N * c["db"], "flops": 4 * T * N * K}
    E, R = c["E"], (T - c["pad"]) * c["K"]
    used, xr = _used(c), (T - c["pad"]) if c["gather"] else R
    if do == "grouped":
        n = b * (xr * K + used * N * K) + R * c["out"] * BYTES[c["y"]] + b * (used * N * c["bias"] + R * N * c["pre"])
        return {"bytes": int(n + 4 * R * c["gather"]), "flops": 2 * R * N * K}
    n = b * (xr * K + used * N * K + R * N + R * K) + E * N * K * BYTES[c["dw"]] + 4 * E * N * c["db"]
    return {"bytes": int(n + 4 * R * c["gather"]), "flops": 4 * R * N * K}


# ------------------------------------------------------------------ the same in 64 bits


def _act64(z, n, act):
    if act == "relu":
        return z * (z > 0)
    if act == "gelu":
        return z * 0.5 * torch.special.erfc(-z / 2.0 ** 0.5)
    if act in ("silu", "swiglu"):
        h = z[:, :n] / (1.0 + torch.exp(-z[:, :n]))
        return h * z[:, n:] if act == "swiglu" else h
    return z


def exact(case, seed):
    c, do = case, case["do"]
    s = _inputs(case, seed)
    d = lambda t: t.to(torch.float64)
    if do == "group":
        return tuple(torch.from_numpy(a).cuda() for a in _grouping(s["ids"].cpu().numpy(), c["E"]))
    if do == "act_bwd":
        # by the product and chain rules on y = act(z), through the 64-bit derivative that autograd forms
        out = torch.empty(s["pre"].shape, dtype=torch.float64, device="cuda")
        for i in range(0, c["T"], 2048):
            z = d(s["pre"][i:i + 2048]).requires_grad_(True)
            _act64(z, c["out"], c["act"]).backward(d(s["dy"][i:i + 2048]))
            out[i:i + 2048] = z.grad
        return out
    if do == "linear":
        z = torch.mm(d(s["x"]), d(s["w"]).t())
        if c["bias"]:
            z += d(s["bias"])
        y = _act64(z, c["out"], c["act"])
        if c["res"]:
            y = y + d(s["res"])
        return (y, z) if c["pre"] else y
    if do == "linear_bwd":
        dz = d(s["dz"])
        out = (torch.mm(dz, d(s["w"])), torch.mm(dz.t(), d(s["x"])))
        return out + (dz.sum(0),) if c["db"] else out
    if do in ("combine", "combine_bwd"):
        T, K, H = c["T"], c["K"], c["H"]
        live = (s["row"] >= 0).view(T, K)
        at = s["row"].clamp(min=0).long()
        if do == "combine":
            out = torch.zeros((T, H), dtype=torch.float64, device="cuda")
            for t in range(0, T, 256):
                v = d(s["y"])[at[t:t + 256]] if T * K * H < 1 << 24 else d(s["y"][at[t:t + 256]])
                out[t:t + 256] = (v * (d(s["w"]) * live)[t:t + 256, :, None]).sum(1)
            return out if s["res"] is None else out + d(s["res"])
        dy = torch.zeros((T * K, H), dtype=torch.float64, device="cuda")
        dw = torch.zeros((T, K), dtype=torch.float64, device="cuda")
        for t in range(0, T, 256):
            g = d(s["dout"][t:t + 256])
            dw[t:t + 256] = (d(s["y"][at[t:t + 256]]) * g[:, None, :]).sum(2) * live[t:t + 256]
            m = live[t:t + 256]
            dy[at[t:t + 256][m]] = (g[:, None, :] * d(s["w"][t:t + 256])[:, :, None])[m]
        return dy, dw
    R, N, K, E = c["T"] * c["K"], _rows(c), c["in"], c["E"]
    off = s["offsets"].cpu().numpy()
    pick = np.arange(R) if s["token"] is None else s["token"].cpu().numpy()
    zeros = lambda *shape: torch.zeros(shape, dtype=torch.float64, device="cuda")
    if do == "grouped":
        y, z = zeros(R, c["out"]), zeros(R, N) if c["pre"] else None
    else:
        if E * N * K > 1 << 30:
            return None        # the matrices' gradients in 64 bits are too large to keep
        dx, dw, db = zeros(R, K), zeros(E, N, K), zeros(E, N)
    for e in np.nonzero(off[1:] > off[:-1])[0].tolist():
        r = slice(int(off[e]), int(off[e + 1]))
        x = d(s["x"][torch.from_numpy(pick[r].astype(np.int64)).cuda()])
        w = d(s["w"][e])
        if do == "grouped":
            v = torch.mm(x, w.t())
            if c["bias"]:
                v += d(s["bias"][e])
            y[r] = _act64(v, c["out"], c["act"])
            if c["pre"]:
                z[r] = v
        else:
            g = d(s["dz"][r])
            dx[r], dw[e], db[e] = torch.mm(g, w), torch.mm(g.t(), x), g.sum(0)
    if do == "grouped":
        return (y, z) if c["pre"] else y
    return (dx, dw, db) if c["db"] else (dx, dw)
