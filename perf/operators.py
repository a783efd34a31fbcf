"""The operators between the MAM layers of a transformer block: what is measured of them.

Layer norm, GELU with dropout, dropout with the residual addition, and the residual addition with dropout and the layer
norm that follows it: forward alone, as in serving, and forward with backward, as in training.  Sizes are rows (tokens)
by width (features); a row of the residual stream is a model's width, a row of the GELU the width inside its MLP.
"""
import math

import numpy as np
import torch

own = False

_DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_GOLDEN, _MIX1, _MIX2 = 0x9E3779B97F4A7C15, 0xBF58476D1CE4E5B9, 0x94D049BB133111EB


def listed():
    def case(name, op, rows, width, dtype, train, rate=0.0, params="same", eps=1e-5):
        return {"name": name, "op": op, "rows": rows, "width": width, "dtype": dtype, "train": train, "rate": rate,
                "params": params, "eps": eps}

    return [
        # one image's class token through an encoder's last norm: latency
        case("norm_token", "layer_norm", 1, 768, "fp32", False, eps=1e-12),
        # the norm before the MLP in a ViT training step: 64 images of 197 tokens, width 768
        case("norm_vit_train", "layer_norm", 12608, 768, "fp32", True, eps=1e-12),
        # a width that is no multiple of anything, rows of a ragged batch, fp32 parameters beside bf16 activations
        case("norm_odd_train", "layer_norm", 5003, 1283, "bf16", True, params="fp32"),
        # a long-context batch at the width of a large language model
        case("norm_large_train", "layer_norm", 32768, 4096, "bf16", True),
        # a serving step of eight sequences: residual addition and norm, no dropout
        case("add_norm_tokens", "dropout_add_layer_norm", 8, 4096, "bf16", False),
        # between two encoder blocks of the ViT training step
        case("add_norm_vit_train", "dropout_add_layer_norm", 12608, 768, "fp32", True, rate=0.1, eps=1e-12),
        # between two blocks of a large language model
        case("add_norm_large_train", "dropout_add_layer_norm", 16384, 5120, "bf16", True, rate=0.1),
        # the activation for one image, no dropout: serving
        case("gelu_image", "gelu", 197, 4096, "bf16", False),
        # an odd width, half precision
        case("gelu_odd_train", "gelu", 7001, 2731, "fp16", True, rate=0.15),
        # the activation inside the MLP in training
        case("gelu_train", "gelu", 12608, 4096, "fp32", True, rate=0.1),
        # the end of a block for one image: dropout and the residual
        case("residual_image_train", "dropout", 197, 768, "fp32", True, rate=0.1),
        # the same for a long-context batch
        case("residual_large_train", "dropout", 32768, 4096, "bf16", True, rate=0.1),
    ]


def draw(rng):
    op = rng.choice(("layer_norm", "layer_norm", "dropout_add_layer_norm", "dropout_add_layer_norm", "gelu", "dropout"))
    dtype = rng.choice(("fp32", "bf16", "fp16"))
    train = rng.random() < 0.7
    width = int(round(math.exp(rng.uniform(math.log(40), math.log(16384)))))
    if rng.random() < 0.6:   # most models' widths are round numbers
        width = (width + 63) // 64 * 64
    most = min(65536, (1 << 25) // width)
    rows = int(round(math.exp(rng.uniform(0.0, math.log(most)))))
    rate = rng.choice((0.0, 0.05, 0.1, 0.25, 0.5)) if op != "layer_norm" else 0.0
    if op == "dropout" and rate == 0.0:
        rate = 0.1
    # fp32 parameters beside narrower activations for the plain norm alone: where the norm reads a rounded sum, a tie
    # that falls to the other side (x / 0.9 of a short x is often next to one) shows in an fp32 weight gradient
    params = rng.choice(("same", "fp32")) if op == "layer_norm" else "same"
    return {"op": op, "rows": rows, "width": width, "dtype": dtype, "train": train, "rate": rate, "params": params,
            "eps": rng.choice((1e-12, 1e-6, 1e-5))}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rows, width, dtype, train = case["rows"], case["width"], _DTYPES[case["dtype"]], case["train"]

    def normal(*shape, to=dtype):
        return torch.randn(*shape, generator=gen, device="cuda").to(to)

    def leaf(t):
        return t.requires_grad_(train)

    s = {"op": case["op"], "rate": case["rate"], "eps": case["eps"], "train": train,
         "drop_seed": int(torch.randint(0, 2 ** 62, (1,), generator=torch.Generator().manual_seed(seed)).item())}
    x = torch.randn(rows, width, generator=gen, device="cuda")
    if "norm" in case["op"]:
        # a residual stream: features of different means and sizes
        x = x * (0.5 + torch.rand(width, generator=gen, device="cuda")) + 0.5 * normal(width, to=torch.float32)
        kind = torch.float32 if case["params"] == "fp32" else dtype
        s["weight"] = leaf((1 + 0.2 * normal(width, to=torch.float32)).to(kind))
        s["bias"] = leaf((0.1 * normal(width, to=torch.float32)).to(kind))
    if case["op"] in ("dropout", "dropout_add_layer_norm"):
        s["residual"] = leaf(x.to(dtype))
        x = torch.randn(rows, width, generator=gen, device="cuda")
    s["x"] = leaf(x.to(dtype))
    if train:
        s["gy"] = normal(rows, width)
        if case["op"] == "dropout_add_layer_norm":
            s["gs"] = normal(rows, width)
    return s


def run(s):
    if own:
        return _run_own(s)
    with torch.no_grad():
        return _run_plain(s)


def _run_own(s):
    from mamtorch_b200.nn import functional as MF

    op, x = s["op"], s["x"]
    if op == "layer_norm":
        y = MF.layer_norm(x, s["weight"], s["bias"], s["eps"])
        if not s["train"]:
            return y
        return [y, *torch.autograd.grad(y, (x, s["weight"], s["bias"]), s["gy"])]
    if op == "dropout_add_layer_norm":
        y, total = MF.dropout_add_layer_norm(x, s["residual"], s["weight"], s["bias"], s["eps"], s["rate"], s["drop_seed"])
        if not s["train"]:
            return [y, total]
        return [y, total, *torch.autograd.grad((y, total), (x, s["residual"], s["weight"], s["bias"]), (s["gy"], s["gs"]))]
    if op == "gelu":
        y = MF.gelu(x, s["rate"], s["drop_seed"])
        return [y, *torch.autograd.grad(y, (x,), s["gy"])] if s["train"] else y
    y = MF.dropout(x, s["rate"], s["drop_seed"], residual=s["residual"])
    return [y, *torch.autograd.grad(y, (x, s["residual"]), s["gy"])] if s["train"] else y


# ---------------------------------------------------------------- the plain forms

def _signed(v):
    return v - (1 << 64) if v >> 63 else v


def _shifted(z, k):
    return (z >> k) & ((1 << (64 - k)) - 1)   # int64 shifts keep the sign


def _keep(shape, rate, seed, device):
    """Element i of the tensor's order is kept where its 32 bits are at least rate * 2^32: the low half (i even) or
    the high half (i odd) of a 64-bit mix of seed + (i // 2) * golden ratio."""
    n = math.prod(shape)
    z = torch.arange((n + 1) // 2, device=device) * _signed(_GOLDEN) + seed
    z = (z ^ _shifted(z, 30)) * _signed(_MIX1)
    z = (z ^ _shifted(z, 27)) * _signed(_MIX2)
    z = z ^ _shifted(z, 31)
    bits = torch.stack((z & 0xFFFFFFFF, _shifted(z, 32)), 1).reshape(-1)[:n].reshape(shape)
    return bits >= int(float(np.float32(rate)) * 2.0 ** 32)


def _dropped(x, keep, rate):
    return x if keep is None else torch.where(keep, x * (1.0 / (1.0 - rate)), torch.zeros((), device=x.device))


def _norm(x, weight, bias, eps):
    centred = x - x.mean(1, keepdim=True)
    rstd = 1.0 / torch.sqrt((centred * centred).mean(1, keepdim=True) + eps)
    h = centred * rstd
    return h * weight.float() + bias.float(), h, rstd


def _norm_grads(g, h, rstd, weight):
    a = g * weight.float()
    dx = rstd * (a - a.mean(1, keepdim=True) - h * (a * h).mean(1, keepdim=True))
    return dx, (g * h).sum(0).to(weight.dtype), g.sum(0).to(weight.dtype)


def _run_plain(s):
    op, x, rate = s["op"], s["x"].detach(), s["rate"]
    dtype = x.dtype
    keep = _keep(x.shape, rate, s["drop_seed"], x.device) if rate > 0 else None
    if op == "layer_norm":
        y, h, rstd = _norm(x.float(), s["weight"].detach(), s["bias"].detach(), s["eps"])
        if not s["train"]:
            return y.to(dtype)
        dx, dw, db = _norm_grads(s["gy"].float(), h, rstd, s["weight"].detach())
        return [y.to(dtype), dx.to(dtype), dw, db]
    if op == "dropout_add_layer_norm":
        total = (s["residual"].detach().float() + _dropped(x.float(), keep, rate)).to(dtype)
        y, h, rstd = _norm(total.float(), s["weight"].detach(), s["bias"].detach(), s["eps"])
        if not s["train"]:
            return [y.to(dtype), total]
        ds, dw, db = _norm_grads(s["gy"].float(), h, rstd, s["weight"].detach())
        ds = ds + s["gs"].float()
        return [y.to(dtype), total, _dropped(ds, keep, rate).to(dtype), ds.to(dtype), dw, db]
    if op == "gelu":
        u = x.float()
        cdf = 0.5 * (1.0 + torch.erf(u * math.sqrt(0.5)))
        y = _dropped(u * cdf, keep, rate).to(dtype)
        if not s["train"]:
            return y
        slope = cdf + u * torch.exp(-0.5 * u * u) * (1.0 / math.sqrt(2.0 * math.pi))
        return [y, (_dropped(s["gy"].float(), keep, rate) * slope).to(dtype)]
    y = (s["residual"].detach().float() + _dropped(x.float(), keep, rate)).to(dtype)
    if not s["train"]:
        return y
    return [y, _dropped(s["gy"].float(), keep, rate).to(dtype), s["gy"]]


# ---------------------------------------------------------------- the definition in 64 bits

def _mask64(shape, rate, seed):
    n = int(np.prod(shape))
    draws = np.empty((n + 1) // 2 * 2, dtype=np.uint32)
    with np.errstate(over="ignore"):
        z = np.arange(len(draws) // 2, dtype=np.uint64)
        z *= np.uint64(_GOLDEN)
        z += np.uint64(seed)
        z ^= z >> np.uint64(30)
        z *= np.uint64(_MIX1)
        z ^= z >> np.uint64(27)
        z *= np.uint64(_MIX2)
        z ^= z >> np.uint64(31)
    draws[0::2] = (z & np.uint64(0xFFFFFFFF)).astype(np.uint32)
    draws[1::2] = (z >> np.uint64(32)).astype(np.uint32)
    keep = draws[:n] >= np.uint32(int(float(np.float32(rate)) * 4294967296))
    return torch.from_numpy(keep.reshape(shape)).cuda()


def exact(case, seed):
    s = prepare(case, seed)
    rate, width = case["rate"], case["width"]
    t = {k: v.detach().double() for k, v in s.items() if isinstance(v, torch.Tensor)}
    # what each element of x is multiplied by on its way
    gate = _mask64(t["x"].shape, rate, s["drop_seed"]).double() / (1 - rate) if rate > 0 else torch.ones((), device="cuda")
    if case["op"] == "gelu":
        below = torch.erfc(-t["x"] / math.sqrt(2)) / 2
        out = [t["x"] * below * gate]
        if case["train"]:
            bell = torch.exp(-t["x"] ** 2 / 2) / math.sqrt(2 * math.pi)
            out.append(t["gy"] * gate * (below + t["x"] * bell))
        return out if case["train"] else out[0]
    if case["op"] == "dropout":
        out = t["residual"] + gate * t["x"]
        return [out, t["gy"] * gate, t["gy"]] if case["train"] else out
    v = t["x"]
    if case["op"] == "dropout_add_layer_norm":
        # the norm reads the sum as it is stored
        total = t["residual"] + gate * t["x"]
        v = total.to(s["x"].dtype).double()
    var, mu = torch.var_mean(v, dim=-1, unbiased=False, keepdim=True)
    scale = (var + case["eps"]).rsqrt()
    h = (v - mu) * scale
    y = torch.addcmul(t["bias"], h, t["weight"])
    out = [y] if case["op"] == "layer_norm" else [y, total]
    if not case["train"]:
        return out[0] if len(out) == 1 else out
    a = t["gy"] * t["weight"]
    dv = (a - (a.sum(-1, keepdim=True) + h * torch.einsum("rc,rc->r", a, h)[:, None]) / width) * scale
    if case["op"] == "dropout_add_layer_norm":
        dv = dv + t["gs"]
        out.append(gate * dv)
    return [*out, dv, torch.einsum("rc,rc->c", t["gy"], h), t["gy"].sum(0)]


def work(case):
    n, size = case["rows"] * case["width"], 4 if case["dtype"] == "fp32" else 2
    train, params = case["train"], 0
    if "norm" in case["op"]:
        params = case["width"] * (4 if case["params"] == "fp32" or case["dtype"] == "fp32" else 2) * (4 if train else 2)
    # tensors read and written once: in training the upstream gradients and the gradients too
    passes = {"layer_norm": (2, 4), "dropout_add_layer_norm": (4, 8), "gelu": (2, 4), "dropout": (3, 5)}[case["op"]][train]
    flops = {"layer_norm": (8, 23), "dropout_add_layer_norm": (10, 27), "gelu": (12, 30), "dropout": (2, 3)}[case["op"]][train]
    return {"bytes": n * size * passes + params, "flops": n * flops}
