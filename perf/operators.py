"""The 16-bit training and serving operators of the library, as cases to be timed and compared:
group norm + activation on channels-last tensors, the connected layer (matrix product with bias,
residual and activation) with its backward, softmax cross entropy over a large number of classes
straight from the connected layer's inputs, and the SGD update that takes 16-bit gradients into fp32
weights and leaves their 16-bit copy for the next step.

`own = False` computes each operator from elementary torch operations in fp32; `own = True` calls
darknet_zig_b200.gpu. Deltas follow darknet's sign (truth - prediction: minus the loss's gradient).
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
ACT_CODE = {"logistic": 0, "relu": 1, "linear": 3, "leaky": 7}
EPS = 1e-5
LEARNING_RATE, MOMENTUM, DECAY, BATCH = 0.1, 0.9, 5e-4, 128


# ---- cases -------------------------------------------------------------------------------

def listed():
    return [
        # one image's 7x7x1024 plane in fp32 before a head: a launch's latency counts
        {"name": "gn_fwd_small", "op": "gn_fwd", "type": "f32", "batch": 1, "spatial": 49, "filters": 1024,
         "groups": 32, "act": "leaky"},
        # a training layer, 128 images of 28x28x256
        {"name": "gn_fwd_large", "op": "gn_fwd", "type": "bf16", "batch": 128, "spatial": 784, "filters": 256,
         "groups": 32, "act": "leaky"},
        # its backward
        {"name": "gn_bwd_large", "op": "gn_bwd", "type": "bf16", "batch": 128, "spatial": 784, "filters": 256,
         "groups": 32, "act": "logistic"},
        # serving: one token through a square projection, bound by reading the weights
        {"name": "connected_token", "op": "connected_fwd", "type": "bf16", "batch": 1, "inputs": 4096,
         "outputs": 4096, "act": "leaky", "biases": True, "residual": False, "pad": 0},
        # ragged rows, odd inputs (rows that start off a 16-byte boundary), 1000 outputs
        {"name": "connected_ragged", "op": "connected_fwd", "type": "f16", "batch": 777, "inputs": 1023,
         "outputs": 1000, "act": "relu", "biases": True, "residual": True, "pad": 0},
        # the second product of a wide block, with its residual
        {"name": "connected_large", "op": "connected_fwd", "type": "bf16", "batch": 8192, "inputs": 16384,
         "outputs": 4096, "act": "linear", "biases": True, "residual": True, "pad": 0},
        # a training step's backward: delta through the activation, input delta, weight and bias updates
        {"name": "connected_bwd_large", "op": "connected_bwd", "type": "bf16", "batch": 8192, "inputs": 4096,
         "outputs": 4096, "act": "relu", "biases": True, "pad": 0},
        # a classifier head: 256 images, 1000 classes
        {"name": "xent_fwd_head", "op": "xent_fwd", "type": "f16", "batch": 256, "inputs": 1024, "classes": 1000,
         "biases": True, "ignored": 0.0},
        # evaluation of a ragged batch over a large odd vocabulary, a tenth of the rows padding
        {"name": "xent_fwd_ragged", "op": "xent_fwd", "type": "bf16", "batch": 1021, "inputs": 2048,
         "classes": 50001, "biases": False, "ignored": 0.1},
        # the gradient of a training step over a large vocabulary
        {"name": "xent_bwd_large", "op": "xent_bwd", "type": "bf16", "batch": 8192, "inputs": 4096,
         "classes": 32768, "biases": False, "ignored": 0.0},
        # a head's update; its 16-bit rows start on 16-byte boundaries, one element longer than they need
        {"name": "sgd_small", "op": "sgd", "type": "f16", "rows": 1000, "cols": 1023, "pad": 1},
        # the update of a 64M-element weight vector
        {"name": "sgd_large", "op": "sgd", "type": "bf16", "rows": 8192, "cols": 8192, "pad": 0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["gn_fwd", "gn_bwd", "connected_fwd", "connected_fwd", "connected_bwd", "xent_fwd", "xent_bwd",
                     "sgd"])
    if op in ("gn_fwd", "gn_bwd"):
        per = rng.choice([1, 2, 4, 5, 8, 10, 16, 32, 48, 64])
        groups = rng.choice([1, 2, 7, 8, 16, 32, 33])
        spatial = _log(rng, 8, 4096)
        batch = max(1, min(_log(rng, 1, 128), (1 << 24) // (spatial * per * groups)))
        return {"op": op, "type": rng.choice(["f32", "bf16", "f16"]), "batch": batch, "spatial": spatial,
                "filters": per * groups, "groups": groups,
                "act": rng.choice(["linear", "leaky", "relu", "logistic"])}
    if op in ("connected_fwd", "connected_bwd"):
        case = {"op": op, "type": rng.choice(["bf16", "f16"]), "batch": _log(rng, 1, 8192),
                "inputs": _log(rng, 32, 8192), "outputs": _log(rng, 16, 8192),
                "act": rng.choice(["linear", "leaky", "relu", "logistic"]), "biases": rng.random() < 0.7,
                "pad": rng.choice([0, 0, 1, 8])}
        while case["batch"] * case["inputs"] * case["outputs"] > 1 << 36:
            case["batch"] = (case["batch"] + 1) // 2
        if rng.random() < 0.6:  # most models' sizes are whole multiples of 64
            case["inputs"] = max(64, case["inputs"] // 64 * 64)
            case["outputs"] = max(64, case["outputs"] // 64 * 64)
        if op == "connected_fwd":
            case["residual"] = rng.random() < 0.5
        return case
    if op in ("xent_fwd", "xent_bwd"):
        case = {"op": op, "type": rng.choice(["bf16", "f16"]), "batch": _log(rng, 1, 8192),
                "inputs": _log(rng, 64, 4096), "classes": _log(rng, 10, 131072), "biases": rng.random() < 0.5,
                "ignored": rng.choice([0.0, 0.0, 0.1, 0.5])}
        while case["batch"] * case["inputs"] * case["classes"] > 1 << 38:
            case["batch"] = (case["batch"] + 1) // 2
        if rng.random() < 0.6:
            case["inputs"] = max(64, case["inputs"] // 64 * 64)
        return case
    return {"op": op, "type": rng.choice(["bf16", "f16"]), "rows": _log(rng, 1, 8192), "cols": _log(rng, 16, 8192),
            "pad": rng.choice([0, 1, 7, 8])}


# ---- inputs ------------------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _normal(g, shape, std=1.0, mean=0.0):
    return torch.randn(shape, generator=g, device="cuda") * std + mean


def _rows(values, dtype, pad):
    """The matrix `values` in `dtype`, its rows `pad` elements further apart than they are long."""
    out = torch.zeros(values.shape[0], values.shape[1] + pad, device="cuda", dtype=dtype)[:, :values.shape[1]]
    out.copy_(values)
    return out


def _empty_rows(rows, cols, dtype, pad=0):
    return torch.empty(rows, cols + pad, device="cuda", dtype=dtype)[:, :cols]


def prepare(case, seed):
    g, op = _gen(seed), case["op"]
    if op in ("gn_fwd", "gn_bwd"):
        dtype = TYPES[case["type"]]
        B, S, C, G = case["batch"], case["spatial"], case["filters"], case["groups"]
        s = dict(case=case, x=_normal(g, (B, S, C), 1.2, 0.4).to(dtype), scales=_normal(g, (C,), 0.3, 1.0),
                 biases=_normal(g, (C,), 0.2), mean=torch.empty(B, G, device="cuda"),
                 rstd=torch.empty(B, G, device="cuda"))
        if op == "gn_fwd":
            s["y"] = torch.empty_like(s["x"])
            return s
        # what the forward left: the statistics, and its output where the activation's gradient needs its sign
        v = s["x"].double().view(B, S, G, C // G)
        mean = v.mean(dim=(1, 3))
        rstd = 1 / torch.sqrt(((v - mean[:, None, :, None]) ** 2).mean(dim=(1, 3)) + EPS)
        s["mean"], s["rstd"], s["y"] = mean.float(), rstd.float(), None
        if case["act"] in ("relu", "leaky"):
            z = ((v - mean[:, None, :, None]) * rstd[:, None, :, None]).reshape(B, S, C)
            z = z * s["scales"] + s["biases"]
            s["y"] = torch.where(z > 0, z, z * (0.1 if case["act"] == "leaky" else 0.0)).to(dtype)
        s["delta"] = _normal(g, (B, S, C)).to(dtype)
        s["dx"] = torch.empty_like(s["x"])
        s["bias_updates"], s["scale_updates"] = torch.empty(C, device="cuda"), torch.empty(C, device="cuda")
        return s
    if op in ("connected_fwd", "connected_bwd"):
        dtype = TYPES[case["type"]]
        M, K, N, pad = case["batch"], case["inputs"], case["outputs"], case["pad"]
        s = dict(case=case, x=_rows(_normal(g, (M, K)), dtype, pad),
                 w=_rows(_normal(g, (N, K), 1 / math.sqrt(K)), dtype, pad),
                 biases=_normal(g, (N,), 0.5) if case["biases"] else None)
        if op == "connected_fwd":
            s["residual"] = _rows(_normal(g, (M, N)), dtype, pad) if case["residual"] else None
            s["y"] = _empty_rows(M, N, dtype, pad)
            return s
        z = _normal(g, (M, N))
        y = {"linear": lambda: None, "relu": lambda: torch.relu(z), "leaky": lambda: torch.where(z > 0, z, 0.1 * z),
             "logistic": lambda: torch.sigmoid(z)}[case["act"]]()
        s["y"] = None if y is None else _rows(y, dtype, pad)
        s["delta"] = _rows(_normal(g, (M, N)), dtype, pad)
        s["dz"] = None if y is None else _empty_rows(M, N, dtype, pad)
        s["dx"] = _empty_rows(M, K, dtype, pad)
        s["weight_updates"] = _empty_rows(N, K, dtype, pad)
        s["bias_updates"] = torch.empty(N, device="cuda") if case["biases"] else None
        return s
    if op in ("xent_fwd", "xent_bwd"):
        dtype = TYPES[case["type"]]
        M, K, N = case["batch"], case["inputs"], case["classes"]
        s = dict(case=case, x=_normal(g, (M, K)).to(dtype), w=_normal(g, (N, K), 1.5 / math.sqrt(K)).to(dtype),
                 biases=_normal(g, (N,), 0.5) if case["biases"] else None)
        labels = torch.randint(0, N, (M,), generator=g, device="cuda", dtype=torch.int32)
        drop = torch.rand(M, generator=g, device="cuda") < case["ignored"]
        drop[0] = False
        s["labels"] = torch.where(drop, torch.full_like(labels, -1), labels)
        s["lse"] = torch.empty(M, device="cuda")
        if op == "xent_fwd":
            s["loss"] = torch.empty(M, device="cuda")
            return s
        s["lse"] = _plain_xent_fwd(s)[1]  # what the forward left
        # a mean over the rows in bf16; a sum in fp16, whose range holds no small means
        s["scale"] = 1.0 / M if case["type"] == "bf16" else 1.0
        s["dx"] = torch.empty_like(s["x"])
        s["weight_updates"] = torch.empty_like(s["w"])
        s["bias_updates"] = torch.empty(N, device="cuda") if case["biases"] else None
        return s
    dtype, rows, cols = TYPES[case["type"]], case["rows"], case["cols"]
    return dict(case=case, w=_normal(g, (rows, cols), 0.1), wu=_normal(g, (rows, cols), 0.5),
                gradients=_rows(_normal(g, (rows, cols)), dtype, case["pad"]),
                w16=_empty_rows(rows, cols, dtype, case["pad"]))


# ---- the plain forms -----------------------------------------------------------------------

def _act(z, act):
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if act == "leaky":
        return torch.where(z > 0, z, 0.1 * z)
    if act == "logistic":
        return 1 / (1 + torch.exp(-z))
    return z


def _act_gradient(y, act):
    """The activation's derivative from its output."""
    if act == "relu":
        return (y > 0).to(y.dtype)
    if act == "leaky":
        return torch.where(y > 0, torch.ones_like(y), torch.full_like(y, 0.1))
    if act == "logistic":
        return (1 - y) * y
    return torch.ones_like(y)


def _plain_gn_fwd(s):
    c = s["case"]
    B, S, C, G = c["batch"], c["spatial"], c["filters"], c["groups"]
    v = s["x"].float().view(B, S, G, C // G)
    mean = v.mean(dim=(1, 3))
    centred = v - mean[:, None, :, None]
    rstd = 1 / torch.sqrt((centred * centred).mean(dim=(1, 3)) + EPS)
    z = (centred * rstd[:, None, :, None]).reshape(B, S, C) * s["scales"] + s["biases"]
    return _act(z, c["act"]).to(s["x"].dtype), mean, rstd


def _plain_gn_bwd(s):
    c = s["case"]
    B, S, C, G = c["batch"], c["spatial"], c["filters"], c["groups"]
    v = s["x"].float().view(B, S, G, C // G)
    xh = ((v - s["mean"][:, None, :, None]) * s["rstd"][:, None, :, None]).reshape(B, S, C)
    y = s["y"].float() if s["y"] is not None else _act(xh * s["scales"] + s["biases"], c["act"])
    d = s["delta"].float() * _act_gradient(y, c["act"])
    t = d * s["scales"]
    group = lambda a: a.reshape(B, S, G, C // G)  # noqa: E731
    m0 = group(t).mean(dim=(1, 3))
    m1 = group(t * xh).mean(dim=(1, 3))
    dx = (group(t) - m0[:, None, :, None] - group(xh) * m1[:, None, :, None]) * s["rstd"][:, None, :, None]
    return dx.reshape(B, S, C).to(s["x"].dtype), d.sum(dim=(0, 1)), (d * xh).sum(dim=(0, 1))


def _plain_connected_fwd(s):
    z = s["x"].float() @ s["w"].float().t()
    if s["biases"] is not None:
        z = z + s["biases"]
    if s["residual"] is not None:
        z = z + s["residual"].float()
    return _act(z, s["case"]["act"]).to(s["x"].dtype)


def _plain_connected_bwd(s):
    dtype = s["x"].dtype
    dz = s["delta"].float()
    if s["y"] is not None:
        dz = dz * _act_gradient(s["y"].float(), s["case"]["act"])
    out = {"dx": (dz @ s["w"].float()).to(dtype), "weight_updates": (dz.t() @ s["x"].float()).to(dtype)}
    if s["y"] is not None:
        out["dz"] = dz.to(dtype)
    if s["bias_updates"] is not None:
        out["bias_updates"] = dz.sum(dim=0)
    return out


def _plain_logits(s):
    z = s["x"].float() @ s["w"].float().t()
    return z if s["biases"] is None else z + s["biases"]


def _plain_xent_fwd(s):
    z = _plain_logits(s)
    top = z.max(dim=1, keepdim=True).values
    lse = top[:, 0] + torch.log(torch.exp(z - top).sum(dim=1))
    valid = s["labels"] >= 0
    at = z.gather(1, s["labels"].clamp(min=0).long()[:, None])[:, 0]
    zero = torch.zeros_like(lse)
    return torch.where(valid, lse - at, zero), torch.where(valid, lse, zero)


def _plain_xent_bwd(s):
    dtype = s["x"].dtype
    d = -torch.exp(_plain_logits(s) - s["lse"][:, None])
    rows = torch.arange(d.shape[0], device=d.device)
    d[rows, s["labels"].clamp(min=0).long()] += 1
    d = torch.where((s["labels"] >= 0)[:, None], d, torch.zeros_like(d)) * s["scale"]
    out = {"dx": (d @ s["w"].float()).to(dtype), "weight_updates": (d.t() @ s["x"].float()).to(dtype)}
    if s["bias_updates"] is not None:
        out["bias_updates"] = d.sum(dim=0)
    return out


def _plain_sgd(s):
    wu = s["wu"] + s["gradients"].float() - DECAY * BATCH * s["w"]
    s["w"].copy_(s["w"] + LEARNING_RATE / BATCH * wu)
    s["wu"].copy_(wu * MOMENTUM)
    return s["w"], s["wu"], s["w"].to(s["gradients"].dtype)


PLAIN = {"gn_fwd": _plain_gn_fwd, "gn_bwd": _plain_gn_bwd, "connected_fwd": _plain_connected_fwd,
         "connected_bwd": _plain_connected_bwd, "xent_fwd": _plain_xent_fwd, "xent_bwd": _plain_xent_bwd,
         "sgd": _plain_sgd}


# ---- the library's calls -------------------------------------------------------------------

def _own_gn_fwd(gpu, s):
    c = s["case"]
    gpu.gnActForward(s["x"], s["y"], c["batch"], c["spatial"], c["filters"], c["groups"], s["scales"], s["biases"],
                     EPS, s["mean"], s["rstd"], ACT_CODE[c["act"]])
    return s["y"], s["mean"], s["rstd"]


def _own_gn_bwd(gpu, s):
    c = s["case"]
    gpu.gnActBackward(s["x"], s["y"], s["delta"], s["dx"], c["batch"], c["spatial"], c["filters"], c["groups"],
                      s["scales"], s["biases"], s["mean"], s["rstd"], s["bias_updates"], s["scale_updates"],
                      ACT_CODE[c["act"]], accumulate=0)
    return s["dx"], s["bias_updates"], s["scale_updates"]


def _own_connected_fwd(gpu, s):
    c = s["case"]
    gpu.connectedActForward(s["x"], s["w"], s["biases"], s["residual"], s["y"], c["batch"], c["inputs"],
                            c["outputs"], ACT_CODE[c["act"]])
    return s["y"]


def _own_connected_bwd(gpu, s):
    c = s["case"]
    gpu.connectedActBackward(s["x"], s["w"], s["y"], s["delta"], s["dz"], s["dx"], s["bias_updates"],
                             s["weight_updates"], c["batch"], c["inputs"], c["outputs"], ACT_CODE[c["act"]],
                             accumulate=0)
    out = {"dx": s["dx"], "weight_updates": s["weight_updates"]}
    if s["dz"] is not None:
        out["dz"] = s["dz"]
    if s["bias_updates"] is not None:
        out["bias_updates"] = s["bias_updates"]
    return out


def _own_xent_fwd(gpu, s):
    c = s["case"]
    gpu.connectedXentForward(s["x"], s["w"], s["biases"], s["labels"], s["loss"], s["lse"], c["batch"], c["inputs"],
                             c["classes"])
    return s["loss"], s["lse"]


def _own_xent_bwd(gpu, s):
    c = s["case"]
    gpu.connectedXentBackward(s["x"], s["w"], s["biases"], s["labels"], s["lse"], None, s["scale"], s["dx"],
                              s["bias_updates"], s["weight_updates"], c["batch"], c["inputs"], c["classes"],
                              accumulate=0)
    out = {"dx": s["dx"], "weight_updates": s["weight_updates"]}
    if s["bias_updates"] is not None:
        out["bias_updates"] = s["bias_updates"]
    return out


def _own_sgd(gpu, s):
    c = s["case"]
    gpu.sgdMomentumMixed(s["w"], s["wu"], s["gradients"], s["w16"], c["rows"], c["cols"], LEARNING_RATE, MOMENTUM,
                         DECAY, BATCH)
    return s["w"], s["wu"], s["w16"]


OWN = {"gn_fwd": _own_gn_fwd, "gn_bwd": _own_gn_bwd, "connected_fwd": _own_connected_fwd,
       "connected_bwd": _own_connected_bwd, "xent_fwd": _own_xent_fwd, "xent_bwd": _own_xent_bwd,
       "sgd": _own_sgd}


def run(state):
    if own:
        from darknet_zig_b200 import gpu

        return OWN[state["case"]["op"]](gpu, state)
    return PLAIN[state["case"]["op"]](state)


# ---- what a pass cannot do without -----------------------------------------------------------

def work(case):
    op = case["op"]
    if op in ("gn_fwd", "gn_bwd"):
        n, e = case["batch"] * case["spatial"] * case["filters"], SIZE[case["type"]]
        stats = 8 * case["batch"] * case["groups"] + 8 * case["filters"]
        if op == "gn_fwd":
            return {"bytes": 2 * n * e + stats, "flops": 8 * n}
        tensors = 4 if case["act"] in ("relu", "leaky") else 3
        return {"bytes": tensors * n * e + stats + 8 * case["filters"], "flops": 16 * n}
    if op in ("connected_fwd", "connected_bwd"):
        M, K, N = case["batch"], case["inputs"], case["outputs"]
        mk, nk, mn = 2 * M * K, 2 * N * K, 2 * M * N
        vec = 4 * N if case["biases"] else 0
        if op == "connected_fwd":
            return {"bytes": mk + nk + mn * (2 if case["residual"] else 1) + vec, "flops": 2 * M * N * K}
        return {"bytes": 2 * mk + 2 * nk + mn * (1 if case["act"] == "linear" else 3) + vec, "flops": 4 * M * N * K}
    if op in ("xent_fwd", "xent_bwd"):
        M, K, N = case["batch"], case["inputs"], case["classes"]
        once = 2 * M * K + 2 * N * K
        vec = 4 * N if case["biases"] else 0
        if op == "xent_fwd":
            return {"bytes": once + 12 * M + vec, "flops": 2 * M * N * K}
        return {"bytes": 2 * once + 8 * M + 2 * vec, "flops": 6 * M * N * K}
    n = case["rows"] * case["cols"]
    return {"bytes": 20 * n, "flops": 6 * n}


# ---- the definitions in 64 bits ----------------------------------------------------------------

def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    slope = {"relu": 0.0, "leaky": 0.1, "linear": 1.0}

    def activated(z):
        return torch.sigmoid(z) if case["act"] == "logistic" else z.clamp(min=0) + slope[case["act"]] * z.clamp(max=0)

    def through(delta, y):
        if case["act"] == "linear":
            return delta
        return delta * (y - y * y) if case["act"] == "logistic" else delta.where(y > 0, delta * slope[case["act"]])

    if op in ("gn_fwd", "gn_bwd"):
        B, G = case["batch"], case["groups"]
        # [batch, group, everything in the group]
        cut = lambda a: a.unflatten(2, (G, -1)).transpose(1, 2).flatten(2)  # noqa: E731
        back = lambda a: a.unflatten(2, (case["spatial"], -1)).transpose(1, 2).flatten(2)  # noqa: E731
        x = s["x"].double()
        if op == "gn_fwd":
            var, mean = torch.var_mean(cut(x), dim=2, correction=0)
            xh = back((cut(x) - mean[..., None]) * torch.rsqrt(var + EPS)[..., None])
            return activated(torch.addcmul(s["biases"].double(), xh, s["scales"].double())), mean, torch.rsqrt(var + EPS)
        mean, rstd = s["mean"].double()[..., None], s["rstd"].double()[..., None]
        xh = (cut(x) - mean) * rstd
        flat = back(xh)
        y = activated(torch.addcmul(s["biases"].double(), flat, s["scales"].double())) if s["y"] is None else s["y"].double()
        d = through(s["delta"].double(), y)
        t = cut(d * s["scales"].double())
        n = t.shape[2]
        dx = rstd * (t - t.sum(2, keepdim=True) / n - xh * (t * xh).sum(2, keepdim=True) / n)
        return back(dx), torch.einsum("bsc->c", d), torch.einsum("bsc,bsc->c", d, flat)
    if op == "connected_fwd":
        z = torch.einsum("mk,nk->mn", s["x"].double(), s["w"].double())
        z = z if s["biases"] is None else z + s["biases"].double()
        return activated(z if s["residual"] is None else z + s["residual"].double())
    if op == "connected_bwd":
        dz = s["delta"].double() if s["y"] is None else through(s["delta"].double(), s["y"].double())
        out = {"dx": torch.einsum("mn,nk->mk", dz, s["w"].double()),
               "weight_updates": torch.einsum("mn,mk->nk", dz, s["x"].double())}
        if s["y"] is not None:
            out["dz"] = dz
        if s["bias_updates"] is not None:
            out["bias_updates"] = torch.einsum("mn->n", dz)
        return out
    if op in ("xent_fwd", "xent_bwd"):
        z = torch.einsum("mk,nk->mn", s["x"].double(), s["w"].double())
        if s["biases"] is not None:
            z += s["biases"].double()
        kept = (s["labels"] >= 0).double()
        one = torch.arange(case["classes"], device="cuda")[None, :] == s["labels"][:, None]
        if op == "xent_fwd":
            lse = torch.logsumexp(z, dim=1)
            return kept * (lse - z.masked_fill(~one, 0).sum(dim=1)), kept * lse
        z = torch.exp_(z.sub_(s["lse"].double()[:, None]))
        d = torch.neg_(z.sub_(one.double())).mul_(kept[:, None] * s["scale"])
        out = {"dx": torch.einsum("mn,nk->mk", d, s["w"].double()),
               "weight_updates": torch.einsum("mn,mk->nk", d, s["x"].double())}
        if s["bias_updates"] is not None:
            out["bias_updates"] = torch.einsum("mn->n", d)
        return out
    w, wu = s["w"].double(), s["wu"].double() + s["gradients"].double() - BATCH * DECAY * s["w"].double()
    w = w + wu * LEARNING_RATE / BATCH
    return w, MOMENTUM * wu, w
