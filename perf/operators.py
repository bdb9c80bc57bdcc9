"""Cases of the head operators: matrix product with epilogue, linear cross entropy, gradient norm and clipping.

With own = False run() computes the plain forms with elementary torch operations in 32 bits; with own = True it
makes the calls of rocal_b200.plugin.pytorch that a training or serving program makes."""
import math

import torch

own = False

_TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"fp32": 4, "fp16": 2, "bf16": 2}
_MAX_LINEAR = 50176 * 768 * 1024        # rows * in * out of the largest linear case
_MAX_LOSS = 8192 * 2048 * 128000        # rows * features * classes of the largest loss case
_IGNORE = -100


def listed():
    return [
        # serving: the class scores of one image
        {"name": "linear_one_row", "op": "linear", "rows": 1, "fin": 2048, "fout": 1000, "dtype": "fp16", "act": "none",
         "bias": True, "period": 0, "train": False},
        # odd sizes: nothing is a multiple of a tile or of 16 bytes
        {"name": "linear_odd", "op": "linear", "rows": 777, "fin": 1001, "fout": 515, "dtype": "bf16", "act": "relu",
         "bias": True, "period": 777, "train": False},
        # a hidden layer of a head, forward and backward
        {"name": "linear_hidden_train", "op": "linear", "rows": 8192, "fin": 1024, "fout": 4096, "dtype": "bf16", "act": "gelu",
         "bias": True, "period": 0, "train": True},
        # 16x16 patches of 256 images of 224x224, projected, the position table added; forward and backward
        {"name": "linear_patches_train", "op": "linear", "rows": 50176, "fin": 768, "fout": 1024, "dtype": "fp16", "act": "none",
         "bias": True, "period": 196, "train": True},
        # evaluation of a batch of 64 over a large class table, a loss for each sample
        {"name": "loss_eval", "op": "loss", "rows": 64, "fin": 2048, "classes": 21841, "dtype": "fp16", "smooth": 0.0,
         "bias": True, "ignored": 0.1, "reduction": "none", "train": False},
        # a classification batch of 1024 images, 1000 classes, label smoothing
        {"name": "loss_batch_train", "op": "loss", "rows": 1024, "fin": 2048, "classes": 1000, "dtype": "fp16", "smooth": 0.1,
         "bias": True, "ignored": 0.02, "reduction": "mean", "train": True},
        # the 8732 anchors of 32 detection samples, 81 classes, most anchors left out of the loss
        {"name": "loss_anchors_train", "op": "loss", "rows": 279424, "fin": 256, "classes": 81, "dtype": "bf16", "smooth": 0.0,
         "bias": True, "ignored": 0.7, "reduction": "sum", "train": True},
        # a large class table and many rows: the case whose logits nobody wants to keep
        {"name": "loss_large_train", "op": "loss", "rows": 8192, "fin": 2048, "classes": 128000, "dtype": "bf16", "smooth": 0.0,
         "bias": False, "ignored": 0.05, "reduction": "mean", "train": True},
        # a small head's gradients: latency
        {"name": "clip_small", "op": "clip", "tensors": 6, "elements": 60000, "dtype": "fp32", "out": "fp32", "clips": True, "packed": False},
        # the gradients of an image classifier
        {"name": "clip_classifier", "op": "clip", "tensors": 161, "elements": 25600000, "dtype": "fp32", "out": "fp32", "clips": True, "packed": False},
        # fp16 gradients under a loss scale, unscaled and clipped into 32-bit ones
        {"name": "clip_unscale", "op": "clip", "tensors": 200, "elements": 90000001, "dtype": "fp16", "out": "fp32", "clips": False, "packed": True},
        # a large model's gradients
        {"name": "clip_large", "op": "clip", "tensors": 300, "elements": 700000000, "dtype": "bf16", "out": "bf16", "clips": True, "packed": False},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["linear", "loss", "clip"])
    if op == "linear":
        c = {"op": op, "rows": _log(rng, 1, 60000), "fin": _log(rng, 16, 8192), "fout": _log(rng, 16, 8192)}
        if rng.random() < 0.5:      # half of them with sizes of ordinary programs, the others any
            c["fin"], c["fout"] = (c["fin"] + 15) // 16 * 16, (c["fout"] + 15) // 16 * 16
        c["rows"] = max(1, min(c["rows"], _MAX_LINEAR // (c["fin"] * c["fout"])))
        period = rng.choice([0, 0, 1, 2])      # none, none, a full residual, one that repeats
        if period == 2:
            c["period"] = _log(rng, 1, min(c["rows"], 600))
            c["rows"] = c["rows"] // c["period"] * c["period"]
        else:
            c["period"] = c["rows"] * period
        return {**c, "dtype": rng.choice(["fp16", "bf16"]), "act": rng.choice(["none", "relu", "gelu", "silu"]),
                "bias": rng.random() < 0.7, "train": rng.random() < 0.5}
    if op == "loss":
        c = {"op": op, "fin": _log(rng, 16, 4096), "classes": _log(rng, 2, 128000)}
        if rng.random() < 0.5:
            c["fin"] = (c["fin"] + 15) // 16 * 16
        most = min(_MAX_LOSS // (c["fin"] * c["classes"]), 8192 * 128000 // c["classes"], 280000 * 256 // c["fin"])
        c["rows"] = _log(rng, 1, max(1, min(280000, most)))
        return {**c, "dtype": rng.choice(["fp16", "bf16"]), "smooth": rng.choice([0.0, 0.0, 0.1]), "bias": rng.random() < 0.7,
                "ignored": rng.choice([0.0, 0.05, 0.5]), "reduction": rng.choice(["mean", "sum", "none"]), "train": rng.random() < 0.6}
    dtype = rng.choice(["fp32", "fp16", "bf16"])
    tensors = _log(rng, 1, 600)
    return {"op": op, "tensors": tensors, "elements": _log(rng, max(64, tensors), 350000000), "dtype": dtype,
            "out": rng.choice([dtype, "fp32"]), "clips": rng.random() < 0.7, "packed": rng.random() < 0.5}


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(gen, shape, scale, dtype):
    return (torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32) * scale).to(dtype)


def _parts(case):
    """Element counts of the gradients: a few large ones, many small ones, odd sizes among them."""
    n, total = case["tensors"], case["elements"]
    weights = [1.0 / (1 + (7 * i) % n) for i in range(n)]
    scale = (total - n) / sum(weights)
    counts = [1 + int(w * scale) for w in weights]
    counts[0] += total - sum(counts)
    return counts


def prepare(case, seed):
    gen = _gen(seed)
    s = {"case": case}
    if case["op"] == "clip":
        dt = _TYPES[case["dtype"]]
        s["grads"] = [_normal(gen, (c,), 2e-3, dt) for c in _parts(case)]
        # the results lie in one buffer, as the buckets of a training program do: packed, or each on a boundary of its own
        step = 1 if case["packed"] else 64
        starts = [0]
        for g in s["grads"]:
            starts.append(starts[-1] + (g.numel() + step - 1) // step * step)
        s["flat"] = torch.zeros(starts[-1], dtype=_TYPES[case["out"]], device="cuda")
        s["out"] = [s["flat"][a:a + g.numel()] for a, g in zip(starts, s["grads"])]
        s["inv_scale"] = 1.0 / 64 if case["dtype"] == "fp16" else 1.0
        norm = 2e-3 * s["inv_scale"] * math.sqrt(case["elements"])
        s["max_norm"] = norm * (0.3 if case["clips"] else 3.0)
        return s
    dt = _TYPES[case["dtype"]]
    n, k = case["rows"], case["fin"]
    m = case["fout"] if case["op"] == "linear" else case["classes"]
    s["x"] = _normal(gen, (n, k), 1.0, dt)
    spread = 1.0 if case["op"] == "linear" else 2.0      # scores of a trained head spread wider
    s["w"] = _normal(gen, (m, k), spread / math.sqrt(k), dt)
    s["b"] = _normal(gen, (m,), 0.3, dt) if case["bias"] else None
    if case["op"] == "linear":
        s["r"] = _normal(gen, (case["period"], m), 0.5, dt) if case["period"] else None
        s["dy"] = _normal(gen, (n, m), 1.0, dt) if case["train"] else None
        leaves = ("x", "w", "b", "r")
    else:
        s["labels"] = torch.randint(0, m, (n,), generator=gen, device="cuda", dtype=torch.int32)
        skip = torch.rand((n,), generator=gen, device="cuda") < case["ignored"]
        s["labels"][skip] = _IGNORE
        # the loss scale of 16-bit training; a loss for each row has a gradient for each row
        s["dy"] = None
        if case["train"]:
            s["dy"] = (torch.rand((n,), generator=gen, device="cuda") + 0.5) * 8 if case["reduction"] == "none" else \
                torch.full((), 1024.0 if case["reduction"] == "mean" else 1.0, device="cuda")
        leaves = ("x", "w", "b")
    if case["train"]:
        for name in leaves:
            if s[name] is not None:
                s[name].requires_grad_(True)
    return s


def _act(z, act):
    if act == "relu":
        return z.clamp(min=0)
    if act == "gelu":
        return z * 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
    if act == "silu":
        return z * torch.sigmoid(z)
    return z


def _act_slope(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    if act == "silu":
        g = torch.sigmoid(z)
        return g * (1 + z * (1 - g))
    return torch.ones_like(z)


def _plain_linear(s):
    c = s["case"]
    with torch.no_grad():
        x, w = s["x"].float(), s["w"].float()
        z = x @ w.t()
        if s["b"] is not None:
            z += s["b"].float()
        y = _act(z, c["act"])
        if s["r"] is not None:
            y = (y.view(-1, c["period"], c["fout"]) + s["r"].float()).view(c["rows"], c["fout"])
        dt = s["x"].dtype
        out = {"y": y.to(dt)}
        if c["train"]:
            dy = s["dy"].float()
            dz = dy * _act_slope(z, c["act"])
            out["dx"], out["dw"] = (dz @ w).to(dt), (dz.t() @ x).to(dt)
            if s["b"] is not None:
                out["db"] = dz.sum(0).to(dt)
            if s["r"] is not None:
                out["dr"] = dy.view(-1, c["period"], c["fout"]).sum(0).to(dt)
        return out


def _plain_loss(s):
    c = s["case"]
    with torch.no_grad():
        x, w = s["x"].float(), s["w"].float()
        z = x @ w.t()
        if s["b"] is not None:
            z += s["b"].float()
        labels = s["labels"].long()
        valid = labels != _IGNORE
        at = labels.clamp(min=0)[:, None]
        top = z.max(1, keepdim=True).values
        e = torch.exp(z - top)
        total = e.sum(1, keepdim=True)
        lse = (torch.log(total) + top)[:, 0]
        loss = lse - (1 - c["smooth"]) * z.gather(1, at)[:, 0]
        if c["smooth"]:
            loss -= c["smooth"] / c["classes"] * z.sum(1)
        loss = torch.where(valid, loss, torch.zeros_like(loss))
        count = valid.sum().clamp(min=1)
        out = {"loss": loss if c["reduction"] == "none" else loss.sum() if c["reduction"] == "sum" else loss.sum() / count}
        if c["train"]:
            g = s["dy"] * valid / (count if c["reduction"] == "mean" else 1)
            dz = e.div_(total)
            if c["smooth"]:
                dz -= c["smooth"] / c["classes"]
            dz.scatter_add_(1, at, torch.full_like(at, -(1 - c["smooth"]), dtype=dz.dtype))
            dz *= g[:, None]
            dt = s["x"].dtype
            out["dx"], out["dw"] = (dz @ w).to(dt), (dz.t() @ x).to(dt)
            if s["b"] is not None:
                out["db"] = dz.sum(0).to(dt)
        return out


def _plain_clip(s):
    total = torch.stack([g.float().square().sum(dtype=torch.float64) for g in s["grads"]]).sum()
    norm = (total.sqrt() * s["inv_scale"]).float()
    factor = torch.clamp(s["max_norm"] / (norm + 1e-6), max=1.0) * s["inv_scale"]
    for g, o in zip(s["grads"], s["out"]):
        o.copy_(g.float() * factor)
    return {"norm": norm, "out": s["flat"]}


def _own(s):
    from rocal_b200.plugin import pytorch as P
    c = s["case"]
    if c["op"] == "clip":
        norm = P.clip_grad_norm(s["grads"], s["max_norm"], out=s["out"], inv_scale=s["inv_scale"])
        return {"norm": norm, "out": s["flat"]}
    if c["op"] == "linear":
        y = P.linear(s["x"], s["w"], bias=s["b"], residual=s["r"], activation=c["act"])
        out = {"y": y.detach()}
        names = [n for n in ("x", "w", "b", "r") if s[n] is not None]
    else:
        y = P.linear_cross_entropy(s["x"], s["w"], s["labels"], bias=s["b"], ignore_index=_IGNORE,
                                   label_smoothing=c["smooth"], reduction=c["reduction"])
        out = {"loss": y.detach()}
        names = [n for n in ("x", "w", "b") if s[n] is not None]
    if c["train"]:
        grads = torch.autograd.grad(y, [s[n] for n in names], s["dy"])
        out.update({"d" + n: g for n, g in zip(names, grads)})
    return out


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    return _plain_linear(state) if op == "linear" else _plain_loss(state) if op == "loss" else _plain_clip(state)


def work(case):
    if case["op"] == "clip":
        return {"bytes": case["elements"] * (_SIZE[case["dtype"]] + _SIZE[case["out"]]), "flops": 3 * case["elements"]}
    n, k = case["rows"], case["fin"]
    m = case["fout"] if case["op"] == "linear" else case["classes"]
    size = _SIZE[case["dtype"]]
    flops = 2.0 * n * k * m * (3 if case["train"] else 1)
    values = n * k + m * k + (m if case["bias"] else 0)
    if case["op"] == "linear":
        values += case["period"] * m
        other = n * m * size * (2 if case["train"] else 1)          # y, dy
    else:
        other = n * 4 * 2                                           # labels, losses
    return {"bytes": size * values * (2 if case["train"] else 1) + other, "flops": flops}


# ---- the definitions in 64 bits -----------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "clip":
        with torch.no_grad():
            norm = s["inv_scale"] * math.sqrt(sum(float((p.double() ** 2).sum()) for g in s["grads"] for p in g.split(50000000)))
            factor = s["inv_scale"] * min(1.0, s["max_norm"] / (norm + 1e-6))
            flat = torch.zeros(s["flat"].shape, dtype=torch.float64, device="cuda")
            for g, o in zip(s["grads"], s["out"]):
                at = o.storage_offset()
                flat[at:at + g.numel()] = g.double() * factor
            return {"norm": torch.tensor(norm, dtype=torch.float64), "out": flat}
    wide = {n: None if s[n] is None else s[n].detach().double().requires_grad_(case["train"]) for n in ("x", "w", "b")}
    z = torch.nn.functional.linear(wide["x"], wide["w"], wide["b"])
    if case["op"] == "linear":
        wide["r"] = None if s["r"] is None else s["r"].detach().double().requires_grad_(case["train"])
        f = torch.nn.functional
        y = {"none": lambda v: v, "relu": f.relu, "gelu": f.gelu, "silu": f.silu}[case["act"]](z)
        if wide["r"] is not None:
            y = y + wide["r"].repeat(case["rows"] // case["period"], 1)
        out, top = {"y": y.detach()}, s["dy"] if s["dy"] is None else s["dy"].double()
    else:
        labels = s["labels"].long()
        keep = labels >= 0
        logp = z - torch.logsumexp(z, 1, keepdim=True)
        target = -torch.take_along_dim(logp, labels.clamp(min=0)[:, None], 1)[:, 0]
        rows = (1 - case["smooth"]) * target - case["smooth"] * logp.mean(1)
        rows = rows * keep
        y = rows if case["reduction"] == "none" else rows.sum() / (max(1, int(keep.sum())) if case["reduction"] == "mean" else 1)
        out, top = {"loss": y.detach()}, s["dy"] if s["dy"] is None else s["dy"].double()
    if case["train"]:
        names = [n for n in ("x", "w", "b", "r") if wide.get(n) is not None]
        for n, g in zip(names, torch.autograd.grad(y, [wide[n] for n in names], top)):
            out["d" + n] = g
    return out
