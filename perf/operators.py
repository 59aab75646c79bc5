"""Cases of the training operators that keep a full-batch step small: layer norm in both directions, activation
checkpoints in 8 bits and what the backward pass computes from them, and the negative log-likelihood of a linear
classifier over many classes whose logits are never kept.

``run`` computes them in elementary torch operations, or (``own``) through the framework's entry points.
"""
import math

import torch

own = False

EPS = 1e-5
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZES = {"fp32": 4, "bf16": 2, "fp16": 2}


def listed():
    return [
        # one request's worth of nodes through the normalisation of a served model: latency
        {"name": "norm_serve_64x256", "kind": "norm_forward", "n": 64, "width": 256, "dtype": "fp32", "affine": "fp32"},
        # a hidden layer of the 600 k-node benchmark graph, both directions
        {"name": "norm_train_600k_fp32", "kind": "norm", "n": 600_000, "width": 256, "dtype": "fp32", "affine": "fp32"},
        # features 602 wide (no multiple of 4: rows start at odd places), half-precision activations
        {"name": "norm_train_602_bf16", "kind": "norm", "n": 100_003, "width": 602, "dtype": "bf16", "affine": "fp32"},
        # the same hidden layer with its input kept in 8 bits for the backward pass
        {"name": "norm_checkpoint_600k", "kind": "norm_checkpoint", "n": 600_000, "width": 256, "dtype": "fp32",
         "affine": "fp32"},
        # activations of a small graph: 100 input channels, latency
        {"name": "checkpoint_1000x100", "kind": "checkpoint", "n": 1000, "width": 100, "dtype": "fp32"},
        # [aggregated | input] rows of a hidden layer kept in 8 bits and brought back
        {"name": "checkpoint_300k_512", "kind": "checkpoint", "n": 300_000, "width": 512, "dtype": "fp32"},
        # weight gradient of a hidden layer's two linear maps, [aggregated | input] kept in 8 bits
        {"name": "weight_grad_600k_fp32", "kind": "weight_grad", "n": 600_000, "width": 512, "out": 256, "dtype": "fp32"},
        # the last layer's: 47 classes, 100 channels, half-precision gradients, an odd number of nodes
        {"name": "weight_grad_47_bf16", "kind": "weight_grad", "n": 99_991, "width": 100, "out": 47, "dtype": "bf16"},
        # validation loss of a few nodes over a thousand classes: latency
        {"name": "nll_eval_128x1000", "kind": "nll", "n": 128, "width": 256, "classes": 1000, "dtype": "fp32", "on": 0.9},
        # a batch of nodes against a very large label set, as in label spaces built from node ids
        {"name": "nll_train_few_rows", "kind": "nll_train", "n": 64, "width": 256, "classes": 131_072, "dtype": "bf16",
         "on": 1.0},
        # full-batch training in fp32, odd sizes, part of the nodes in the loss
        {"name": "nll_train_5003_fp32", "kind": "nll_train", "n": 5003, "width": 200, "classes": 20_011, "dtype": "fp32",
         "on": 0.6},
        # the largest: 16 k nodes in the loss, 64 k classes, [aggregated | input] rows of 512
        {"name": "nll_train_64k_bf16", "kind": "nll_train", "n": 16_384, "width": 512, "classes": 65_536, "dtype": "bf16",
         "on": 1.0},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["norm_forward", "norm", "norm_checkpoint", "checkpoint", "weight_grad", "nll", "nll_train"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    if kind.startswith("norm"):
        width = _log(rng, 16, 2100)
        return {"kind": kind, "n": _log(rng, 1, min(600_000, 150_000_000 // width)), "width": width, "dtype": dtype,
                "affine": rng.choice([dtype, "fp32"])}
    if kind == "checkpoint":
        width = _log(rng, 1, 2100)
        return {"kind": kind, "n": _log(rng, 1, min(600_000, 150_000_000 // width)), "width": width, "dtype": dtype}
    if kind == "weight_grad":
        return {"kind": kind, "n": _log(rng, 1, 600_000), "width": _log(rng, 1, 512), "out": _log(rng, 1, 260),
                "dtype": rng.choice(["fp32", "bf16"])}
    return {"kind": kind, "n": _log(rng, 32, 16_384), "width": _log(rng, 4, 512), "classes": _log(rng, 16, 65_536),
            "dtype": rng.choice(["fp32", "bf16"]), "on": round(rng.uniform(0.3, 1.0), 3)}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    n, width, dtype = case["n"], case["width"], DTYPES[case["dtype"]]
    s = {"case": case}
    if case["kind"].startswith("nll"):
        classes = case["classes"]
        s["x"] = normal(n, width).to(dtype)
        s["weight"] = (normal(classes, width) * (2.0 / math.sqrt(width))).to(dtype)
        s["bias"] = (normal(classes) * 0.5).to(dtype)
        s["labels"] = torch.randint(0, classes, (n,), generator=gen, device="cuda")
        s["mask"] = torch.rand(n, generator=gen, device="cuda") < case["on"]
        s["inv_count"] = 1.0 / max(1.0, n * case["on"])
        return s
    # rows of different size and centre, as activations of nodes of different degree have
    x = normal(n, width)
    x = x * torch.exp(0.5 * normal(n, 1)) + 0.5 * normal(n, 1)
    if case["kind"] in ("checkpoint", "weight_grad"):
        x = torch.relu(x)
    s["x"] = x.to(dtype)
    if case["kind"] == "weight_grad":
        s["g"] = (normal(n, case["out"]) * 0.01).to(dtype)
    if case["kind"].startswith("norm"):
        affine = DTYPES[case["affine"]]
        s["gamma"] = (1.0 + 0.2 * normal(width)).to(affine)
        s["beta"] = (0.2 * normal(width)).to(affine)
        if case["kind"] != "norm_forward":
            s["gy"] = normal(n, width).to(dtype)
    return s


def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    from super_gnn_b200 import supergnn_ops as ops

    kind = s["case"]["kind"]
    if kind == "norm_forward":
        return ops.layer_norm_forward(s["x"], s["gamma"], s["beta"], EPS)[0]
    if kind == "norm":
        y, stats = ops.layer_norm_forward(s["x"], s["gamma"], s["beta"], EPS)
        return (y,) + ops.layer_norm_backward(s["gy"], s["x"], stats, s["gamma"])
    if kind == "norm_checkpoint":
        y, stats, codes, params = ops.layer_norm_forward(s["x"], s["gamma"], s["beta"], EPS, checkpoint=True)
        return (y,) + ops.layer_norm_backward_checkpoint(s["gy"], codes, params, stats, s["gamma"])
    if kind == "checkpoint":
        codes, params = ops.checkpoint_pack_rows(s["x"])
        return ops.checkpoint_unpack_rows(codes, params, s["x"].dtype)
    if kind == "weight_grad":
        codes, params = ops.checkpoint_pack_rows(s["x"])
        return ops.checkpoint_weight_grad(s["g"], codes, params)
    if kind == "nll":
        return ops.linear_nll_loss(s["x"], s["weight"], s["bias"], s["labels"], s["mask"], s["inv_count"])
    return ops.linear_nll_loss_grad(s["x"], s["weight"], s["bias"], s["labels"], s["mask"], s["inv_count"])


# ---- plain forms, in 32 bits, rounded once at the end ----
def _quantised(x):
    """The values that the 8-bit codes of the rows of ``x`` stand for."""
    low, high = x.amin(1, keepdim=True), x.amax(1, keepdim=True)
    scale = (high - low) / torch.full_like(low, 255.0)  # a division: by a number it would be a product
    scale = torch.where(scale == 0, torch.ones_like(scale), scale)
    return torch.round((x - low) / scale) * scale + low


def _run_plain(s):
    kind = s["case"]["kind"]
    x = s["x"].float()
    if kind.startswith("norm"):
        gamma, beta = s["gamma"].float(), s["beta"].float()
        mean = x.mean(1, keepdim=True)
        rstd = torch.rsqrt((x - mean).square().mean(1, keepdim=True) + EPS)
        y = ((x - mean) * rstd * gamma + beta).to(s["x"].dtype)
        if kind == "norm_forward":
            return y
        xhat = ((_quantised(x) if kind == "norm_checkpoint" else x) - mean) * rstd
        gy = s["gy"].float()
        gxhat = gy * gamma
        gx = rstd * (gxhat - gxhat.mean(1, keepdim=True) - xhat * (gxhat * xhat).mean(1, keepdim=True))
        return (y, gx.to(s["x"].dtype), (gy * xhat).sum(0).to(s["gamma"].dtype), gy.sum(0).to(s["beta"].dtype))
    if kind == "checkpoint":
        return _quantised(x).to(s["x"].dtype)
    if kind == "weight_grad":
        return s["g"].float().t() @ _quantised(x)
    weight, bias = s["weight"].float(), s["bias"].float()
    labels, inv = s["labels"], s["inv_count"]
    logits = x @ weight.t() + bias
    top = logits.amax(1, keepdim=True)
    lse = torch.log(torch.exp(logits - top).sum(1, keepdim=True)) + top
    picked = logits.gather(1, labels[:, None])
    on = s["mask"][:, None]
    loss = (torch.where(on, lse - picked, torch.zeros_like(lse)).sum() * inv).reshape(1)
    if kind == "nll":
        return loss, torch.where(on, lse, torch.zeros_like(lse))[:, 0]
    grad = torch.exp(logits - lse)
    grad = torch.where(on, grad.scatter_add(1, labels[:, None], torch.full_like(lse, -1.0)) * inv,
                       torch.zeros_like(grad))
    dtype = s["x"].dtype
    return loss, (grad @ weight).to(dtype), (grad.t() @ x).to(dtype), grad.sum(0).to(dtype)


# ---- the same from the definitions, in 64 bits ----
def _to32(v):
    """``v`` rounded to 32 bits, held in 64."""
    return v.float().double()


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    x = s["x"].to(torch.float64)
    if kind.startswith("nll"):
        on = s["mask"].nonzero()[:, 0]
        logits = torch.addmm(s["bias"].double(), x[on], s["weight"].double().T)
        logp = torch.log_softmax(logits, dim=1)
        lse = torch.zeros(case["n"], dtype=torch.float64, device="cuda")
        lse[on] = (logits[:, 0] - logp[:, 0])
        rows = torch.arange(on.numel(), device="cuda")
        loss = -logp[rows, s["labels"][on]].sum().reshape(1) * s["inv_count"]
        if kind == "nll":
            return loss, lse
        del logits
        prob = logp.exp_()
        prob[rows, s["labels"][on]] -= 1.0
        prob *= s["inv_count"]
        gx = torch.zeros_like(x)
        gx[on] = prob.mm(s["weight"].double())
        return loss, gx, prob.T.mm(x[on]), prob.sum(0)
    kept = x
    if kind in ("checkpoint", "weight_grad", "norm_checkpoint"):
        # which code a value gets is defined by the 32-bit roundings of the range, the step and the quotient
        low = x.min(1, keepdim=True).values
        step = _to32(_to32(x.max(1, keepdim=True).values - low) / 255)
        step[step == 0] = 1.0
        kept = low + step * torch.round(_to32(_to32(x - low) / step))
    if kind == "checkpoint":
        return kept
    if kind == "weight_grad":
        return torch.einsum("nm,nk->mk", s["g"].double(), kept)
    gamma, beta = s["gamma"].double(), s["beta"].double()
    var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
    std = (var + EPS).sqrt()
    y = torch.addcmul(beta, (x - mean) / std, gamma)
    if kind == "norm_forward":
        return y
    gy, z = s["gy"].double(), (kept - mean) / std
    a = gy * gamma
    h = float(case["width"])
    gx = (a - (a.sum(1, keepdim=True) + z * (a * z).sum(1, keepdim=True)) / h) / std
    return y, gx, torch.einsum("nk,nk->k", gy, z), gy.sum(0)


def work(case):
    n, width, size = case["n"], case["width"], SIZES[case["dtype"]]
    kind = case["kind"]
    if kind.startswith("norm"):
        affine = 2 * width * SIZES[case["affine"]]
        if kind == "norm_forward":
            return {"bytes": 2 * n * width * size + affine, "flops": 8 * n * width}
        # x and gy read, y and gx written; the checkpoint itself is neither an input nor an output of the pass
        return {"bytes": 4 * n * width * size + 2 * affine, "flops": 20 * n * width}
    if kind == "checkpoint":
        return {"bytes": 2 * n * width * size, "flops": 6 * n * width}
    if kind == "weight_grad":
        out = case["out"]
        return {"bytes": n * (width + out) * size + 4 * width * out, "flops": 2 * n * width * out}
    classes, rows = case["classes"], n * case["on"]
    if kind == "nll":
        return {"bytes": rows * width * size + classes * (width + 1) * size + n * 13,
                "flops": 2 * rows * classes * width}
    return {"bytes": (rows + n) * width * size + 2 * classes * (width + 1) * size + n * 9,
            "flops": 6 * rows * classes * width}
