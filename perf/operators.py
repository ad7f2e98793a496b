"""Cases of the layer and optimizer operators: the linear layer with its epilogue, layer norm, and the Newton-Schulz
update, each in its plain form (elementary torch operations in 32 bits) and through the library's entry points.

The library works on pool buffers; `Buf` is one of them, seen as a torch tensor.  With `own` set, prepare() puts the
inputs into such buffers once, as a program that trains or serves with the library has them, and run() makes the one call.
"""
import math

import torch

own = False

ACTS = ("none", "relu", "gelu", "silu")
NS = (3.4445, -4.7750, 2.0315)


# ---- cases ----
def listed():
    return [
        # one token through a square layer while serving: the weights are read once
        {"name": "linear_token_f32", "op": "linear", "M": 1, "K": 4096, "N": 4096, "act": "silu", "bias": True, "residual": False, "keep_z": False, "f16": False},
        # the widening layer of a block in training, pre-activation kept for the backward pass
        {"name": "linear_train_f32", "op": "linear", "M": 4096, "K": 1024, "N": 4096, "act": "gelu", "bias": True, "residual": False, "keep_z": True, "f16": False},
        # a prompt through a square layer in half storage, added to the stream it came from
        {"name": "linear_prompt_f16", "op": "linear", "M": 8192, "K": 4096, "N": 4096, "act": "none", "bias": True, "residual": True, "keep_z": False, "f16": True},
        # LeNet's first fully connected layer at its batch of 512
        {"name": "linear_bwd_lenet_f32", "op": "linear_bwd", "M": 512, "K": 400, "N": 120, "act": "relu", "f16": False},
        # the widening layer again, backward
        {"name": "linear_bwd_train_f32", "op": "linear_bwd", "M": 4096, "K": 1024, "N": 4096, "act": "gelu", "f16": False},
        # a ragged handful of half rows before a classifier
        {"name": "norm_odd_f16", "op": "norm", "rows": 77, "cols": 1001, "f16": True, "affine": True},
        # the norm of a whole training batch
        {"name": "norm_train_f32", "op": "norm", "rows": 16384, "cols": 2048, "f16": False, "affine": True},
        # backward of the ragged one ...
        {"name": "norm_bwd_odd_f16", "op": "norm_bwd", "rows": 777, "cols": 1001, "f16": True, "affine": True},
        # ... and of the batch
        {"name": "norm_bwd_train_f32", "op": "norm_bwd", "rows": 16384, "cols": 2048, "f16": False, "affine": True},
        # optimizer step of LeNet's first fully connected layer
        {"name": "muon_lenet", "op": "muon", "rows": 400, "cols": 120, "steps": 5, "nesterov": True},
        # optimizer step of the widening layer
        {"name": "muon_wide", "op": "muon", "rows": 1024, "cols": 4096, "steps": 5, "nesterov": True},
        # the orthogonalisation alone, at the size of the square benchmark product
        {"name": "orthogonal_square", "op": "orthogonal", "rows": 4096, "cols": 4096, "steps": 5},
    ]


def _spread(rng, lo, hi):
    """A whole number, even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("linear", "linear", "linear_bwd", "norm", "norm_bwd", "muon", "orthogonal"))
    if op in ("linear", "linear_bwd"):
        c = {"op": op, "M": _spread(rng, 1, 8192), "K": _spread(rng, 8, 4096), "N": _spread(rng, 8, 4096), "act": rng.choice(ACTS), "f16": rng.random() < 0.5}
        if rng.random() < 0.5:      # half of the layers have the round sizes that layers mostly have
            c["K"], c["N"] = (max(8, (c[k] + 63) // 64 * 64) for k in ("K", "N"))
        if op == "linear":
            c.update(bias=rng.random() < 0.8, residual=rng.random() < 0.5, keep_z=rng.random() < 0.4)
        return c
    if op in ("norm", "norm_bwd"):
        cols = _spread(rng, 8, 16384)
        return {"op": op, "rows": _spread(rng, 1, max(1, min(16384, (1 << 25) // cols))), "cols": cols, "f16": rng.random() < 0.5, "affine": rng.random() < 0.9}
    c = {"op": op, "rows": _spread(rng, 8, 4096), "cols": _spread(rng, 8, 4096), "steps": rng.choice((3, 5, 5))}
    if op == "muon":
        c["nesterov"] = rng.random() < 0.7
    return c


def work(case):
    op = case["op"]
    size = 2 if case.get("f16") else 4
    if op in ("linear", "linear_bwd"):
        M, K, N = case["M"], case["K"], case["N"]
        if op == "linear":
            vals = M * K + K * N + M * N * (1 + case["residual"] + case["keep_z"]) + N * case["bias"]
            return {"bytes": size * vals, "flops": 2 * M * N * K}
        vals = 2 * (M * K + K * N) + M * N * (1 + (case["act"] != "none")) + N
        return {"bytes": size * vals, "flops": 4 * M * N * K}
    rows, cols = case["rows"], case["cols"]
    if op == "norm":
        return {"bytes": size * (2 * rows * cols + 2 * cols * case["affine"]) + 8 * rows, "flops": 8 * rows * cols}
    if op == "norm_bwd":
        return {"bytes": size * (3 * rows * cols + 3 * cols * case["affine"]) + 8 * rows, "flops": 14 * rows * cols}
    m, n = min(rows, cols), max(rows, cols)
    # both squares are symmetric: half of their values suffice
    flops = case["steps"] * (m * m * n + m * m * m + 2 * m * m * n)
    return {"bytes": 4 * rows * cols * (5 if op == "muon" else 2), "flops": flops}


# ---- inputs ----
def _inputs(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dt = torch.float16 if case.get("f16") else torch.float32

    def normal(*shape, scale=1.0, shift=0.0, to=dt):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale + shift).to(to)

    op = case["op"]
    if op == "linear":
        M, K, N = case["M"], case["K"], case["N"]
        t = {"x": normal(M, K), "w": normal(K, N, scale=K ** -0.5)}
        if case["bias"]:
            t["bias"] = normal(N, scale=0.1)
        if case["residual"]:
            t["residual"] = normal(M, N)
        return t
    if op == "linear_bwd":
        M, K, N = case["M"], case["K"], case["N"]
        t = {"dy": normal(M, N, scale=0.02), "x": normal(M, K), "w": normal(K, N, scale=K ** -0.5)}
        if case["act"] != "none":
            t["z"] = normal(M, N)
        return t
    rows, cols = case["rows"], case["cols"]
    if op in ("norm", "norm_bwd"):
        t = {"x": normal(rows, cols, scale=1.5, shift=0.3)}
        if op == "norm_bwd":
            t["dy"] = normal(rows, cols, scale=0.02)
            x = t["x"].double()                         # the statistics that the forward pass kept
            mean = x.mean(1)
            t["mean"] = mean.float()
            t["rstd"] = ((x - mean[:, None]).square().mean(1) + EPS).rsqrt().float()
        if case["affine"]:
            t["gamma"] = normal(cols, scale=0.1, shift=1.0)
            if op == "norm":
                t["beta"] = normal(cols, scale=0.1)
        return t
    # gradients of layers: a few strong directions over a floor of noise
    r = min(8, rows, cols)
    low = normal(rows, r) @ normal(r, cols)
    g = (0.3 * low + normal(rows, cols)) * 1e-3
    if op == "orthogonal":
        return {"g": g}
    return {"g": g, "mom": normal(rows, cols, scale=2e-3), "p": normal(rows, cols, scale=rows ** -0.5)}


EPS = 1e-5
LR, MU, DECAY = 0.02, 0.95, 0.01


class _Memory:
    """A buffer of the library's pool; tensors that lie in it keep it alive."""

    def __init__(self, shape, dtype):
        be = _backend()
        size = 2 if dtype is torch.float16 else 4
        self.lib, self.id = be.lib, be.alloc(max(math.prod(shape) * size, 512))
        self.__cuda_array_interface__ = {"shape": tuple(shape), "typestr": "<f%d" % size, "data": (self.lib.thvm_cuda_buf_ptr(self.id), False), "version": 3}

    def __del__(self):
        self.lib.thvm_cuda_buf_free(self.id)


class Buf:
    """A buffer's id, and the tensor that lies in it."""

    def __init__(self, shape, dtype):
        memory = _Memory(shape, dtype)
        self.id, self.t = memory.id, torch.as_tensor(memory, device="cuda")


_be = None


def _backend():
    global _be
    if _be is None:
        import tinyhvm_b200
        _be = tinyhvm_b200.CudaBackend()
    return _be


def _outputs(case):
    """Names, shapes and types of what a call writes, in the order that run() returns."""
    op = case["op"]
    dt = torch.float16 if case.get("f16") else torch.float32
    if op == "linear":
        return [("y", (case["M"], case["N"]), dt)] + ([("z", (case["M"], case["N"]), dt)] if case["keep_z"] else [])
    if op == "linear_bwd":
        return [("dx", (case["M"], case["K"]), dt), ("dw", (case["K"], case["N"]), dt), ("dbias", (case["N"],), dt)]
    shape = (case["rows"], case["cols"])
    if op == "norm":
        return [("y", shape, dt), ("mean", shape[:1], torch.float32), ("rstd", shape[:1], torch.float32)]
    if op == "norm_bwd":
        return [("dx", shape, dt)] + ([("dgamma", shape[1:], dt), ("dbeta", shape[1:], dt)] if case["affine"] else [])
    return [("out", shape, torch.float32)] if op == "orthogonal" else []


def prepare(case, seed):
    state = {"case": case, "t": _inputs(case, seed)}
    if own:
        lib = state["lib"] = _backend().lib
        b = state["b"] = {name: Buf(t.shape, t.dtype) for name, t in state["t"].items()}
        b.update({name: Buf(shape, dt) for name, shape, dt in _outputs(case)})
        lib.thvm_cuda_sync()            # fresh buffers are cleared on the library's stream
        for name, t in state["t"].items():
            b[name].t.copy_(t)
        state["t"] = None
        torch.cuda.synchronize()
    return state


# ---- the library's calls ----
def _own(state):
    case, b, lib = state["case"], state["b"], state["lib"]
    op = case["op"]
    i = {name: x.id for name, x in b.items()}
    dt = 1 if case.get("f16") else 0
    if op == "linear":
        rc = lib.thvm_cuda_linear(i["y"], i.get("z", 0), i["x"], i["w"], i.get("bias", 0), i.get("residual", 0), case["M"], case["K"], case["N"], ACTS.index(case["act"]), dt)
    elif op == "linear_bwd":
        rc = lib.thvm_cuda_linear_backward(i["dx"], i["dw"], i["dbias"], i["dy"], i.get("z", 0), i["x"], i["w"], case["M"], case["K"], case["N"], ACTS.index(case["act"]), dt)
    elif op == "norm":
        rc = lib.thvm_cuda_layernorm(i["y"], i["mean"], i["rstd"], i["x"], i.get("gamma", 0), i.get("beta", 0), case["rows"], case["cols"], EPS, dt)
    elif op == "norm_bwd":
        rc = lib.thvm_cuda_layernorm_backward(i["dx"], i.get("dgamma", 0), i.get("dbeta", 0), i["dy"], i["x"], i.get("gamma", 0), i["mean"], i["rstd"], case["rows"], case["cols"], dt)
    elif op == "orthogonal":
        rc = lib.thvm_cuda_newton_schulz(i["out"], i["g"], case["rows"], case["cols"], case["steps"])
    else:
        rc = lib.thvm_cuda_muon_step(i["p"], i["g"], i["mom"], case["rows"], case["cols"], LR, MU, DECAY, int(case["nesterov"]), case["steps"])
    if rc:
        raise RuntimeError(_backend().last_error())
    if op == "muon":
        return {"p": b["p"].t, "mom": b["mom"].t}
    return {name: b[name].t for name, _, _ in _outputs(case)}


# ---- the plain forms ----
def _act(kind, z):
    if kind == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if kind == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if kind == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _act_slope(kind, z):
    if kind == "relu":
        return (z > 0).float()
    if kind == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    s = 1 / (1 + torch.exp(-z))
    return s * (1 + z * (1 - s))


def _newton_schulz(g, steps):
    a, b, c = NS
    x = g / (torch.sqrt((g * g).sum()) + 1e-7)
    flip = g.shape[0] > g.shape[1]
    x = x.T if flip else x
    for _ in range(steps):
        s = x @ x.T
        x = a * x + (b * s + c * (s @ s)) @ x
    return (x.T if flip else x).contiguous()


def run(state):
    if own:
        return _own(state)
    case, t = state["case"], state["t"]
    op = case["op"]
    dt = torch.float16 if case.get("f16") else torch.float32
    if op == "linear":
        z = t["x"].float() @ t["w"].float()
        if "bias" in t:
            z = z + t["bias"].float()
        y = _act(case["act"], z)
        if "residual" in t:
            y = y + t["residual"].float()
        return {"y": y.to(dt), "z": z.to(dt)} if case["keep_z"] else {"y": y.to(dt)}
    if op == "linear_bwd":
        dz = t["dy"].float()
        if case["act"] != "none":
            dz = dz * _act_slope(case["act"], t["z"].float())
        return {"dx": (dz @ t["w"].float().T).to(dt), "dw": (t["x"].float().T @ dz).to(dt), "dbias": dz.sum(0).to(dt)}
    if op == "norm":
        x = t["x"].float()
        mean = x.mean(1, keepdim=True)
        d = x - mean
        rstd = torch.rsqrt((d * d).mean(1, keepdim=True) + EPS)
        y = d * rstd
        if case["affine"]:
            y = y * t["gamma"].float() + t["beta"].float()
        return {"y": y.to(dt), "mean": mean[:, 0], "rstd": rstd[:, 0]}
    if op == "norm_bwd":
        rstd = t["rstd"][:, None]
        xh = (t["x"].float() - t["mean"][:, None]) * rstd
        dy = t["dy"].float()
        g = dy * t["gamma"].float() if case["affine"] else dy
        dx = rstd * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
        if not case["affine"]:
            return {"dx": dx.to(dt)}
        return {"dx": dx.to(dt), "dgamma": (dy * xh).sum(0).to(dt), "dbeta": dy.sum(0).to(dt)}
    if op == "orthogonal":
        return {"out": _newton_schulz(t["g"], case["steps"])}
    t["mom"].mul_(MU).add_(t["g"])
    u = t["g"] + MU * t["mom"] if case["nesterov"] else t["mom"]
    scale = LR * math.sqrt(max(1.0, case["rows"] / case["cols"]))
    t["p"].mul_(1 - LR * DECAY).sub_(scale * _newton_schulz(u, case["steps"]))
    return {"p": t["p"], "mom": t["mom"]}


# ---- the definitions in 64 bits ----
def exact(case, seed):
    t = {name: x.double() for name, x in _inputs(case, seed).items()}
    op = case["op"]
    normal = torch.distributions.Normal(torch.zeros((), dtype=torch.float64, device="cuda"), torch.ones((), dtype=torch.float64, device="cuda"))
    if op == "linear":
        z = torch.matmul(t["x"], t["w"]) + t.get("bias", 0.0)
        y = {"none": lambda: z, "relu": lambda: z.clamp(min=0), "gelu": lambda: z * normal.cdf(z), "silu": lambda: z * torch.sigmoid(z)}[case["act"]]()
        y = y + t.get("residual", 0.0)
        return {"y": y, "z": z} if case["keep_z"] else {"y": y}
    if op == "linear_bwd":
        dz = t["dy"]
        if case["act"] != "none":
            z = t["z"]
            sig = torch.sigmoid(z)
            dz = dz * {"relu": lambda: (z > 0).double(), "gelu": lambda: normal.cdf(z) + z * normal.log_prob(z).exp(), "silu": lambda: sig + z * sig * (1 - sig)}[case["act"]]()
        return {"dx": torch.einsum("mn,kn->mk", dz, t["w"]), "dw": torch.einsum("mk,mn->kn", t["x"], dz), "dbias": torch.einsum("mn->n", dz)}
    if op == "norm":
        var, mean = torch.var_mean(t["x"], dim=1, correction=0)
        rstd = (var + EPS) ** -0.5
        y = torch.einsum("ij,i->ij", t["x"] - mean[:, None], rstd)
        return {"y": torch.addcmul(t["beta"], y, t["gamma"]) if case["affine"] else y, "mean": mean, "rstd": rstd}
    if op == "norm_bwd":
        n = case["cols"]
        xh = torch.einsum("ij,i->ij", t["x"] - t["mean"][:, None], t["rstd"])
        g = torch.einsum("ij,j->ij", t["dy"], t["gamma"]) if case["affine"] else t["dy"]
        dx = (g - g.sum(1)[:, None] / n - xh * (torch.einsum("ij,ij->i", g, xh) / n)[:, None]) * t["rstd"][:, None]
        if not case["affine"]:
            return {"dx": dx}
        return {"dx": dx, "dgamma": torch.einsum("ij,ij->j", t["dy"], xh), "dbeta": torch.einsum("ij->j", t["dy"])}
    u = t["g"]
    if op == "muon":
        mom = MU * t["mom"] + t["g"]
        u = t["g"] + MU * mom if case["nesterov"] else mom
    # the polynomial acts on the eigenvalues of the smaller square: x p(s), s = x^T x or x x^T
    a, b, c = NS
    x = u / (torch.linalg.vector_norm(u) + 1e-7)
    wide = x.shape[0] <= x.shape[1]
    for _ in range(case["steps"]):
        s = torch.einsum("ik,jk->ij", x, x) if wide else torch.einsum("ki,kj->ij", x, x)
        q = a * torch.eye(s.shape[0], dtype=s.dtype, device=s.device) + torch.addmm(b * s, s, s, alpha=c)
        x = torch.einsum("ij,jk->ik", q, x) if wide else torch.einsum("ij,jk->ik", x, q)
    if op == "orthogonal":
        return {"out": x}
    scale = LR * max(1.0, case["rows"] / case["cols"]) ** 0.5
    return {"p": t["p"] - LR * DECAY * t["p"] - scale * x, "mom": mom}
