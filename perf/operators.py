"""Operators that hold the memory of a training step down, as cases that can be timed and compared.

``loss``   the cross entropy of a segmentation head with many classes, taken from the features in front of the head (the
           logits are never kept), with its gradients: ``scaffold_b200.ops.head_loss.head_cross_entropy``
``norm``   GroupNorm + ReLU whose backward pass works on an 8-bit copy of its input, forward and backward:
           ``scaffold_b200.ops.group_norm.group_norm_kept8``
``keep``   an activation written to its 8-bit copy and read back: ``scaffold_b200.ops.kept8``

The 8-bit copy: 16 consecutive elements share a power of two 2^e, the smallest (e at least -126) with
max |x| < 126.5 * 2^e, and each is kept as the whole number nearest to x / 2^e (a tie goes to the even one). A block with
an infinity or a NaN is restored as NaN. What would be restored beyond the type's largest number keeps |q| at 63. GroupNorm
keeps its input on its own side of the ReLU: where the nearest whole number would be restored on the other side, the next
one towards x is kept.
"""
import math

import torch

own = False

BLOCK = 16
EPS = 1e-5
IGNORED = -1  # the label of voxels that take no part


def _loss(name, tokens, width, classes, weighted=False, ignored=0.0, train=True):
    return {"name": name, "kind": "loss", "tokens": tokens, "width": width, "classes": classes, "weighted": weighted,
            "ignored": ignored, "train": train}


def _norm(name, batch, voxels, channels, groups, relu=True):
    return {"name": name, "kind": "norm", "batch": batch, "voxels": voxels, "channels": channels, "groups": groups,
            "relu": relu}


def _keep(name, elements, dtype):
    return {"name": name, "kind": "keep", "elements": elements, "dtype": dtype}


def listed():
    return [
        # the smallest step: 16 cubed at base width 16 with 34 classes, where launches and the host path count
        _loss("loss 16^3 w16 c34", 16 ** 3, 16, 34),
        # a batch of the default width with the trainer's class weights and some voxels outside the labelled region
        _loss("loss 64^3 w64 c147 weighted", 64 ** 3, 64, 147, weighted=True, ignored=0.1),
        # the headline batch (2 x 128 cubed, base width 64) with some 250 fractal classes
        _loss("loss 2x128^3 w64 c257", 2 * 128 ** 3, 64, 257),
        # extents that are no powers of two, a narrow network, a thousand classes
        _loss("loss 2x44x60x76 w32 c1001", 2 * 44 * 60 * 76, 32, 1001, weighted=True),
        # a wide feature vector and a vocabulary-sized head with a ragged end
        _loss("loss 8192 w1024 c32771", 8192, 1024, 32771, ignored=0.05),
        # the loss of a single position, without gradients, as a user who scores one answer takes it
        _loss("loss 1 w256 c32768 eval", 1, 256, 32768, train=False),
        # the bottleneck of a 64 cubed volume: 8 cubed at 512 channels, a call bound by its launches
        _norm("norm 1x8^3 c512", 1, 8 ** 3, 512, 8),
        # a decoder level of odd extents
        _norm("norm 2x44x60x76 c32", 2, 44 * 60 * 76, 32, 8),
        # the widest map of the headline batch
        _norm("norm 2x128^3 c64", 2, 128 ** 3, 64, 8),
        # the input of a bottleneck convolution
        _keep("keep 8^3x512 bf16", 8 ** 3 * 512, "bf16"),
        # a length that is no multiple of anything, in 32 bits
        _keep("keep 1000003 fp32", 1000003, "fp32"),
        # the widest map of the headline batch, as a convolution keeps it
        _keep("keep 2x128^3x64 bf16", 2 * 128 ** 3 * 64, "bf16"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choices(("loss", "norm", "keep"), (5, 3, 2))[0]
    if kind == "loss":
        while True:
            tokens, classes, width = _log(rng, 1, 2 ** 22), _log(rng, 33, 50000), 8 * _log(rng, 2, 128)
            if tokens * classes <= 2 ** 30 and tokens * classes * width <= 2 ** 37:
                break
        case = _loss("", tokens, width, classes, rng.random() < 0.5, rng.choice((0.0, 0.0, 0.1, 0.9)), rng.random() < 0.85)
    elif kind == "norm":
        while True:
            channels, groups = 16 * _log(rng, 1, 64), rng.choice((1, 2, 4, 8, 8, 16, 32))
            batch, voxels = rng.choice((1, 1, 2, 3, 4)), _log(rng, 8, 2 ** 21)
            if channels % (8 * groups) == 0 and batch * voxels * channels <= 2 ** 28:
                break
        case = _norm("", batch, voxels, channels, groups, rng.random() < 0.8)
    else:
        case = _keep("", _log(rng, 1, 2 ** 27), rng.choice(("bf16", "bf16", "fp16", "fp32")))
    del case["name"]
    return case


# -- inputs ------------------------------------------------------------------------------------------------------------
_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    normal = lambda *s: torch.randn(*s, generator=gen, device=dev)  # noqa: E731
    if case["kind"] == "loss":
        v, c, k = case["tokens"], case["width"], case["classes"]
        x = torch.relu(normal(v, c)).to(torch.bfloat16)  # the features leave a GroupNorm + ReLU
        w = (normal(k, c) * (2.8 / math.sqrt(c))).to(torch.bfloat16)  # logits of a standard deviation of 2
        b = (normal(k) * 0.5).to(torch.bfloat16)
        y = (torch.rand(v, generator=gen, device=dev) ** 3 * k).long().clamp_(0, k - 1)  # low classes are common
        cw = None
        if case["weighted"]:  # total / background for class 0, total / foreground for the others: the trainer's rule
            bg = (y == 0).sum().clamp(1, max(1, v - 1)).float()
            cw = torch.full((k,), float(v), device=dev) / torch.full((k,), float(v), device=dev).sub(bg).clamp_min(1)
            cw[0] = v / bg
        if case["ignored"]:
            y[torch.rand(v, generator=gen, device=dev) < case["ignored"]] = IGNORED
        y = y.to(torch.int16 if k <= 32767 else torch.int32)
        if case["train"]:
            x, w, b = (t.requires_grad_() for t in (x, w, b))
        return {"case": case, "x": x, "w": w, "b": b, "y": y, "cw": cw}
    if case["kind"] == "norm":
        n, s, c = case["batch"], case["voxels"], case["channels"]
        x = (normal(n, s, 1, 1, c) * (0.5 + torch.rand(c, generator=gen, device=dev)) + 0.3 * normal(c)).to(torch.bfloat16)
        gy = (normal(n, s, 1, 1, c) * 1e-3).to(torch.bfloat16)
        w, b = 1 + 0.2 * normal(c), 0.2 * normal(c)
        x, gy = (t.permute(0, 4, 1, 2, 3) for t in (x, gy))  # NCDHW tensors in channels-last memory
        return {"case": case, "x": x.requires_grad_(), "gy": gy, "w": w.requires_grad_(), "b": b.requires_grad_()}
    n = case["elements"]
    x = normal(n) * torch.exp(normal((n + 255) // 256)).repeat_interleave(256)[:n]  # rows of many sizes
    return {"case": case, "x": x.to(_TYPES[case["dtype"]])}


# -- one pass ----------------------------------------------------------------------------------------------------------
def run(state):
    return {"loss": _run_loss, "norm": _run_norm, "keep": _run_keep}[state["case"]["kind"]](state)


def _run_loss(s):
    if own:
        from scaffold_b200.ops.head_loss import head_cross_entropy
        with torch.set_grad_enabled(s["case"]["train"]):
            loss = head_cross_entropy(s["x"], s["w"], s["b"], s["y"], s["cw"], ignore_label=IGNORED)
        if not s["case"]["train"]:
            return {"loss": loss}
        dx, dw, db = torch.autograd.grad(loss, (s["x"], s["w"], s["b"]))
        return {"loss": loss.detach(), "dx": dx, "dw": dw, "db": db}
    with torch.no_grad():
        x, w, b, y = s["x"].float(), s["w"].float(), s["b"].float(), s["y"].long()
        live = y != IGNORED
        y = torch.where(live, y, 0)
        weight = live.float() if s["cw"] is None else torch.where(live, s["cw"][y], 0.0)
        logits = x @ w.T + b
        at_label = logits.gather(1, y[:, None])[:, 0]
        top = logits.amax(1)
        p = torch.exp(logits - top[:, None])
        total = p.sum(1)
        nll = top + torch.log(total) - at_label
        # the sums over voxels in 64 bits: a long sum of small terms
        num, den = (weight * nll).double().sum(), weight.double().sum().clamp_min(torch.finfo(torch.float32).eps)
        loss = (num / den).float()
        if not s["case"]["train"]:
            return {"loss": loss}
        g = weight / den.float()
        p = p * (g / total)[:, None]
        p.scatter_add_(1, y[:, None], -g[:, None])
        t = torch.bfloat16
        return {"loss": loss, "dx": (p @ w).to(t), "dw": (p.T @ x).to(t), "db": p.sum(0).to(t)}


def _kept(x, limit):
    """(whole numbers, steps, blocks that are not finite), all [blocks, ...], of fp32 x [blocks, 16]."""
    most = x.abs().amax(1, keepdim=True)
    bad = ~torch.isfinite(most)
    m, k = torch.frexp(torch.where(bad, 0.0, most))
    e = torch.where(m * 128 < 126.5, k - 7, k - 6).clamp_min(-126)
    step = ((e + 127).int() << 23).view(torch.float32)  # 2^e by its bits: pow() need not be exact
    cap = torch.where(64.0 * step.double() > limit, 63.0, 127.0)
    q = torch.minimum(torch.maximum(torch.round(torch.where(bad, 0.0, x) / step), -cap), cap)
    return q, step, cap, bad


def _run_keep(s):
    if own:
        from scaffold_b200.ops.kept8 import keep8, restore8
        return {"restored": restore8(keep8(s["x"]))}
    x = s["x"].float()
    n = x.numel()
    pad = torch.zeros((n + BLOCK - 1) // BLOCK * BLOCK, device=x.device)
    pad[:n] = x
    q, step, _, bad = _kept(pad.view(-1, BLOCK), torch.finfo(s["x"].dtype).max)
    back = torch.where(bad, float("nan"), q * step)
    return {"restored": back.reshape(-1)[:n].to(s["x"].dtype)}


def _run_norm(s):
    case = s["case"]
    if own:
        from scaffold_b200.ops.group_norm import group_norm_kept8
        y = group_norm_kept8(s["x"], case["groups"], s["w"], s["b"], EPS, activation="relu" if case["relu"] else None)
        dx, dw, db = torch.autograd.grad(y, (s["x"], s["w"], s["b"]), s["gy"])
        return {"y": y.detach(), "dx": dx, "dw": dw, "db": db}
    with torch.no_grad():
        n, c, g = case["batch"], case["channels"], case["groups"]
        x = s["x"].permute(0, 2, 3, 4, 1).reshape(n, -1, c).float()
        gy = s["gy"].permute(0, 2, 3, 4, 1).reshape(n, -1, c).float()
        count = x.shape[1] * (c // g)
        spread = lambda t: t.repeat_interleave(c // g, 1)[:, None]  # noqa: E731  [n, g] -> [n, 1, c]
        total = lambda t: t.sum(1, dtype=torch.float64).view(n, g, -1).sum(2)  # noqa: E731  [n, s, c] -> [n, g]
        mean = spread((total(x) / count).float())
        rstd = spread(torch.rsqrt(total((x - mean) ** 2) / count + EPS).float())
        a = rstd * s["w"]
        shift = s["b"] - mean * a
        y = x * a + shift
        q, step, cap, bad = _kept(x.reshape(-1, BLOCK), torch.finfo(torch.bfloat16).max)
        if case["relu"]:
            on = y > 0
            other = ((q * step).view(x.shape) * a + shift > 0) != on
            q = q + torch.where(other, torch.where(on == (a > 0), 1.0, -1.0), 0.0).reshape(q.shape)
            q = torch.minimum(torch.maximum(q, -cap), cap)
            y = torch.relu(y)
        kept = torch.where(bad, float("nan"), q * step).view(x.shape)
        if case["relu"]:
            gy = torch.where(kept * a + shift > 0, gy, 0.0)
        xhat = (kept - mean) * rstd
        db, dw = gy.sum((0, 1), dtype=torch.float64).float(), (gy * xhat).sum((0, 1), dtype=torch.float64).float()
        c1 = spread((total(gy * s["w"]) / count).float())
        c2 = spread((total(gy * s["w"] * xhat) / count).float())
        dx = rstd * (gy * s["w"] - c1 - xhat * c2)
        out = lambda t: t.to(torch.bfloat16).view(n, -1, 1, 1, c).permute(0, 4, 1, 2, 3)  # noqa: E731
        return {"y": out(y), "dx": out(dx), "dw": dw, "db": db}


# -- what a pass cannot do without -------------------------------------------------------------------------------------
def work(case):
    if case["kind"] == "loss":
        v, c, k = case["tokens"], case["width"], case["classes"]
        read = 2 * (v * c + k * c + k) + v * (2 if k <= 32767 else 4) + (4 * k if case["weighted"] else 0)
        if not case["train"]:
            return {"bytes": read + 4, "flops": 2 * v * c * k}
        return {"bytes": read + 4 + 2 * (v * c + k * c + k), "flops": 6 * v * c * k}
    if case["kind"] == "norm":
        n = case["batch"] * case["voxels"] * case["channels"]
        # x, gy, y, dx in 16 bits; the 8-bit copy, with a byte for 16 elements, written once and read once
        return {"bytes": 8 * n + 2 * (n + n // BLOCK) + 16 * case["channels"], "flops": 20 * n}
    n, size = case["elements"], 4 if case["dtype"] == "fp32" else 2
    return {"bytes": 2 * size * n + 2 * (n + -(-n // BLOCK)), "flops": 4 * n}


# -- the definitions in 64 bits ----------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"loss": _exact_loss, "norm": _exact_norm, "keep": _exact_keep}[case["kind"]](s)


def _exact_loss(s):
    """The definition, differentiated by autograd."""
    keep = s["y"] != IGNORED
    leaves = [s[n].detach().double().requires_grad_(s["case"]["train"]) for n in ("x", "w", "b")]
    logits = torch.addmm(leaves[2], leaves[0][keep], leaves[1].T)
    y = s["y"][keep].long()
    per_class = torch.ones(s["case"]["classes"], dtype=torch.float64, device=y.device) if s["cw"] is None else s["cw"].double()
    nll = torch.logsumexp(logits, 1) - logits[torch.arange(len(y), device=y.device), y]
    loss = (per_class[y] * nll).sum() / per_class[y].sum().clamp_min(torch.finfo(torch.float32).eps)
    if not s["case"]["train"]:
        return {"loss": loss}
    dx, dw, db = torch.autograd.grad(loss, leaves)
    return {"loss": loss.detach(), "dx": dx, "dw": dw, "db": db}


def _exact_kept(x, limit, side=None):
    """The 8-bit copy's values of 64-bit x [blocks, 16]; ``side`` tells on which side of the ReLU a value is."""
    most = x.abs().max(1).values
    fine = most.isfinite()
    two_to = lambda e: ((e.long() + 1023) << 52).view(torch.float64)  # noqa: E731
    e = torch.full_like(most, -126.0)
    e = torch.where(fine & (most > 0), torch.floor(torch.log2(most.clamp_min(1e-300) / 126.5)) - 1, e).clamp_min(-126)
    for _ in range(3):  # from one or two below to the smallest that holds the block's largest number
        e = torch.where(fine & (most >= 126.5 * two_to(e)), e + 1, e)
    step = two_to(e)[:, None]
    cap = torch.where(64 * step > limit, 63.0, 127.0).double()
    q = torch.round(x.nan_to_num(0, 0, 0) / step).clamp(min=-cap, max=cap)
    if side is not None:
        near = q * step
        q = torch.where(side(near) == side(x), q, q + torch.sign(x - near)).clamp(min=-cap, max=cap)
    return torch.where(fine[:, None], q * step, float("nan"))


def _exact_keep(s):
    n = s["x"].numel()
    x = torch.nn.functional.pad(s["x"].double(), (0, -n % BLOCK)).view(-1, BLOCK)
    return {"restored": _exact_kept(x, torch.finfo(s["x"].dtype).max).reshape(-1)[:n]}


def _exact_norm(s):
    """One sample at a time; the gradients are those of the formula at the kept input, with the statistics of x."""
    case = s["case"]
    c, g, relu = case["channels"], case["groups"], case["relu"]
    w, b = s["w"].detach().double(), s["b"].detach().double()
    ys, dxs, dw, db = [], [], torch.zeros_like(w), torch.zeros_like(b)
    for x, gy in zip(s["x"].detach(), s["gy"]):
        x, gy = (t.reshape(c, -1).T.double() for t in (x, gy))  # [voxels, channels]
        grouped = x.reshape(-1, g, c // g)
        var, mean = torch.var_mean(grouped, (0, 2), unbiased=False)
        mean, rstd = (t.repeat_interleave(c // g) for t in (mean, (var + EPS) ** -0.5))
        pre = lambda t: (t.reshape(x.shape) - mean) * rstd * w + b  # noqa: E731
        y = pre(x)
        side = (lambda t: (pre(t) > 0).reshape(t.shape)) if relu else None
        kept = _exact_kept(x.reshape(-1, BLOCK), torch.finfo(torch.bfloat16).max, side).reshape(x.shape)
        if relu:
            gy = gy * (pre(kept) > 0)
            y = y.clamp_min(0)
        xhat = (kept - mean) * rstd
        db += gy.sum(0)
        dw += (gy * xhat).sum(0)
        means = lambda t: t.reshape(-1, g, c // g).mean((0, 2)).repeat_interleave(c // g)  # noqa: E731
        dxs.append((rstd * (gy * w - means(gy * w) - xhat * means(gy * w * xhat))).T.reshape(c, -1, 1, 1))
        ys.append(y.T.reshape(c, -1, 1, 1))
    return {"y": torch.stack(ys), "dx": torch.stack(dxs), "dw": dw, "db": db}
