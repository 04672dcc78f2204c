"""Cases of the training operators beside the detection losses and the optimizer: what is timed, on what inputs, and what the answers are.

    linear_cross_entropy   softmax cross entropy of a linear classifier over many classes, logits never kept, with its gradients
    clip_grad_norm_        the global norm of many gradient tensors and their scaling
    FusedSGD.step          the same clipping inside the optimizer step over the parameter arena

`own` false: elementary torch operations.  `own` true: the calls a training script makes of yolov6_amd.
"""
import math
import random

import torch

own = False

_TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
_LARGEST_FLOPS = 6 * 8192 * 1024 * 131072
_LARGEST_GRADS = 1 << 27


# ------------------------------------------------------------------------------------------------------------------------ the cases
def _ce(name, rows, width, classes, dtype, **more):
    """`pitch`: elements between feature rows (a channel slice of a wider buffer); `unlabelled`: share of rows with ignore_index;
    `scale`: what the loss is multiplied by before the backward (LossScaler; fp16 gradients of a mean underflow without)."""
    case = {"name": name, "op": "ce", "rows": rows, "width": width, "classes": classes, "dtype": dtype, "train": True, "bias": False,
            "smoothing": 0.0, "reduction": "mean", "unlabelled": 0.0, "pitch": width, "scale": 1.0}
    case.update(more)
    return case


def listed():
    return [
        # one row against a large label set, forward only: the score of a single answer, bound by the classifier's bytes and latency
        _ce("ce_eval_one_row", 1, 1024, 32000, "bf16", train=False, reduction="none"),
        # a validation batch, per-row losses
        _ce("ce_eval_rows", 2048, 512, 21841, "fp16", train=False, reduction="none", bias=True),
        # classification pretraining of YOLOv6-S's backbone: 64 pooled 512-channel features, 1000 classes, label smoothing, loss scale
        _ce("ce_pretrain_b64", 64, 512, 1000, "fp16", bias=True, smoothing=0.1, scale=1024.0),
        # dense labelling: the 8400 anchors of four 640x640 images, 80 classes + background, features a slice of a wider neck buffer,
        # most anchors without a label
        _ce("ce_anchors_4x8400", 33600, 128, 81, "fp16", bias=True, unlabelled=0.7, pitch=256, scale=65536.0),
        # odd in every size
        _ce("ce_odd", 1537, 515, 50021, "bf16", bias=True, unlabelled=0.1),
        # single precision, summed
        _ce("ce_fp32", 1024, 256, 4001, "fp32", bias=True, reduction="sum"),
        # a large vocabulary
        _ce("ce_32k", 4096, 1024, 32000, "bf16"),
        # the largest
        _ce("ce_131k", 8192, 1024, 131072, "bf16", unlabelled=0.02),
        # a handful of small half-precision tensors of odd sizes: latency
        {"name": "clip_small", "op": "clip", "tensors": 40, "least": 1, "most": 5000, "dtype": "fp16", "max_norm": 0.1},
        # as many tensors as YOLOv6-L trains, about as many elements
        {"name": "clip_yolov6l", "op": "clip", "tensors": 489, "least": 64, "most": 590000, "dtype": "fp32", "max_norm": 1.0},
        # a clipped optimizer step at the sizes of YOLOv6-S and of a model of twice its width
        {"name": "sgd_s", "op": "sgd", "width": 0.5, "depth": 0.33, "max_norm": 10.0, "scale": 1024.0},
        {"name": "sgd_l", "op": "sgd", "width": 1.0, "depth": 1.0, "max_norm": 10.0, "scale": 1024.0},
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(("ce", "ce", "ce", "clip", "sgd"))
    if kind == "clip":
        dtype = rng.choice(("fp16", "bf16", "fp32", "mixed"))
        tensors, least = _spread(rng, 1, 600), _spread(rng, 1, 1000)
        most = max(least, min(_spread(rng, 100, 1e7), _LARGEST_GRADS // tensors))
        return {"op": "clip", "tensors": tensors, "least": least, "most": most, "dtype": dtype, "max_norm": 1.0 if dtype == "fp32" else 0.1}
    if kind == "sgd":
        return {"op": "sgd", "width": round(rng.uniform(0.25, 1.0), 3), "depth": round(rng.uniform(0.2, 1.0), 3),
                "max_norm": round(math.exp(rng.uniform(0, 6)), 3), "scale": float(2 ** rng.randrange(0, 13))}
    dtype = rng.choice(("fp16", "bf16", "bf16", "fp32"))
    train = rng.random() < 0.75
    most = _LARGEST_FLOPS / (16 if dtype == "fp32" else 1) / (6 if train else 2)
    while True:
        rows, width, classes = _spread(rng, 1, 16384), _spread(rng, 16, 2048), _spread(rng, 2, 131072)
        if rng.random() < 0.5:
            width = max(16, width // 64 * 64)
        if rows * width * classes <= most:
            break
    reduction = rng.choice(("mean", "sum", "none"))
    scale = float(2 ** int(math.log2(16 * rows))) if dtype == "fp16" and reduction == "mean" else 1.0
    case = _ce("", rows, width, classes, dtype, train=train, bias=rng.random() < 0.5, smoothing=rng.choice((0.0, 0.0, 0.1)), reduction=reduction,
               unlabelled=rng.choice((0.0, 0.0, 0.05, 0.5)), pitch=width + rng.choice((0, 0, 1, 8, 64)), scale=scale)
    del case["name"]
    return case


# ----------------------------------------------------------------------------------------------------------------------- the inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return {"ce": _prepare_ce, "clip": _prepare_clip, "sgd": _prepare_sgd}[case["op"]](case, g)


def _prepare_ce(case, g):
    n, d, v, dtype = case["rows"], case["width"], case["classes"], _TYPES[case["dtype"]]
    weight = torch.randn((v, d), generator=g, device="cuda").mul_(2 / math.sqrt(d))
    # label frequencies fall off as in large label sets; features lean towards their label's row, some rows a lot
    target = torch.rand(n, generator=g, device="cuda", dtype=torch.float64).mul(math.log(v)).exp().long().sub_(1).clamp_(0, v - 1)
    buf = torch.randn((n, case["pitch"]), generator=g, device="cuda")
    buf[:, case["pitch"] - d:] += weight[target] * torch.rand((n, 1), generator=g, device="cuda") * 3
    x = buf.to(dtype)[:, case["pitch"] - d:]
    target[torch.rand(n, generator=g, device="cuda") < case["unlabelled"]] = -100
    bias = torch.randn(v, generator=g, device="cuda").to(dtype) if case["bias"] else None
    state = {"case": dict(case), "x": x.requires_grad_(), "weight": weight.to(dtype).requires_grad_(), "target": target,
             "bias": bias.requires_grad_() if bias is not None else None}
    shape = (n,) if case["reduction"] == "none" else ()
    up = torch.rand(shape, generator=g, device="cuda") + 0.5 if shape else torch.ones((), device="cuda")
    state["upstream"] = up * case["scale"]
    return state


def _sizes(case):
    rng = random.Random(1000 * case["tensors"] + case["least"])
    return [_spread(rng, case["least"], case["most"]) for _ in range(case["tensors"])]


def _prepare_clip(case, g):
    """Gradients as views of flat buffers, each at a 16-byte border, as the parameter arena lays them out."""
    kinds = ["fp32", "bf16", "fp16"] if case["dtype"] == "mixed" else [case["dtype"]]
    sizes = _sizes(case)
    at, place = [0] * len(kinds), []
    for i, s in enumerate(sizes):
        k = i % len(kinds)
        place.append((k, at[k], s))
        at[k] += (s + 7) // 8 * 8
    flats = [torch.zeros(max(a, 8), device="cuda", dtype=_TYPES[k]) for a, k in zip(at, kinds)]
    values = [torch.randn(max(a, 8), generator=g, device="cuda").to(_TYPES[k]) for a, k in zip(at, kinds)]
    grads = [flats[k][o:o + s] for k, o, s in place]
    torch._foreach_copy_(grads, [values[k][o:o + s] for k, o, s in place])
    params = []
    for gr in grads:
        p = torch.nn.Parameter(torch.empty_like(gr))
        p.grad = gr
        params.append(p)
    return {"case": dict(case), "flats": flats, "params": params, "grads": grads}


def _modules(case):
    """Convolutions and BatchNorms of a RepVGG backbone's training form: channels and repeats of EfficientRep scaled by width and depth."""
    channels = [max(8, math.ceil(c * case["width"] / 8) * 8) for c in (64, 128, 256, 512, 1024)]
    repeats = [max(1, round(r * case["depth"])) for r in (1, 6, 12, 18, 6)]
    mods, cin = [], 3
    for c, r in zip(channels, repeats):
        for _ in range(r):
            for k in (3, 1):
                mods += [torch.nn.Conv2d(cin, c, k, bias=False, device="cuda"), torch.nn.BatchNorm2d(c, device="cuda")]
            cin = c
    mods.append(torch.nn.Conv2d(cin, 85, 1, device="cuda"))
    return torch.nn.Sequential(*mods)


def _prepare_sgd(case, g):
    """Parameters in reverse order of registration, each at a 16-byte border of one flat buffer; gradients and momentum alike."""
    model = _modules(case)
    kind = {}
    for m in model:
        if getattr(m, "bias", None) is not None:
            kind[id(m.bias)] = 2
        kind[id(m.weight)] = 0 if isinstance(m, torch.nn.BatchNorm2d) else 1
    params = list(reversed(list(model.parameters())))
    group = torch.cat([torch.nn.functional.pad(torch.full((p.numel(),), kind[id(p)], dtype=torch.uint8, device="cuda"), (0, -p.numel() % 4), value=3)
                       for p in params])
    n = group.numel()
    param, grad, momentum = (torch.randn(n, generator=g, device="cuda") * s for s in (0.05, 0.01 * case["scale"], 0.02))
    state = {"case": dict(case), "scale": torch.full((1,), case["scale"], device="cuda")}
    if own:
        # a training script keeps the arena, the optimizer and the scaler; the values are those of the flat buffers
        from yolov6_amd.solver import FusedSGD, LossScaler
        from yolov6_amd.train_engine import ParamArena
        arena = ParamArena(model)
        opt = FusedSGD(model, arena, lr=0.01, momentum=0.937, weight_decay=5e-4)
        for to, values in ((arena.data, param), (arena.grad, grad), (opt.buf, momentum)):
            to.copy_(values)
        opt.steps = 1
        state.update(model=model, arena=arena, opt=opt, scaler=LossScaler("cuda", init_scale=case["scale"]))
    else:
        state.update(param=param, grad=grad, momentum=momentum, group=group)
    return state


# -------------------------------------------------------------------------------------------------------------------- one pass each
def run(state):
    return {"ce": _run_ce, "clip": _run_clip, "sgd": _run_sgd}[state["case"]["op"]](state)


def _run_ce(state):
    case, x, weight, bias, target = state["case"], state["x"], state["weight"], state["bias"], state["target"]
    if own:
        from yolov6_amd.models.losses.loss_ce import linear_cross_entropy
        options = {"label_smoothing": case["smoothing"], "reduction": case["reduction"]}
        if not case["train"]:
            with torch.no_grad():
                return linear_cross_entropy(x, weight, target, bias, **options)
        loss = linear_cross_entropy(x, weight, target, bias, **options)
        leaves = [x, weight] + ([bias] if bias is not None else [])
        return (loss.detach(), *torch.autograd.grad(loss, leaves, state["upstream"]))
    with torch.no_grad():
        xs, ws = x.float(), weight.float()
        z = xs @ ws.t()
        if bias is not None:
            z = z + bias.float()
        labelled = target != -100
        t = target.clamp_min(0)
        top = z.amax(1, keepdim=True)
        lse = (z - top).exp().sum(1).log() + top[:, 0]
        eps, v = case["smoothing"], case["classes"]
        rows = lse - (1 - eps) * z.gather(1, t[:, None])[:, 0]
        if eps:
            rows = rows - eps * z.mean(1)
        rows = torch.where(labelled, rows, 0.0)
        count = labelled.sum().clamp_min(1) if case["reduction"] == "mean" else 1
        loss = rows if case["reduction"] == "none" else rows.sum() / count
        if not case["train"]:
            return loss
        dz = (z - lse[:, None]).exp()
        if eps:
            dz = dz - eps / v
        dz.scatter_add_(1, t[:, None], torch.full_like(lse, eps - 1)[:, None])
        dz = dz * torch.where(labelled, state["upstream"] / count, 0.0)[:, None]
        grads = [(dz @ ws).to(x.dtype), (dz.t() @ xs).to(x.dtype)]
        if bias is not None:
            grads.append(dz.sum(0).to(x.dtype))
        return (loss, *grads)


def _run_clip(state):
    if own:
        from yolov6_amd.solver import clip_grad_norm_
        return [clip_grad_norm_(state["params"], state["case"]["max_norm"])] + state["flats"]
    with torch.no_grad():
        grads = state["grads"]
        every = torch.cat([gr.float() for gr in grads])
        norm = every.double().square().sum().sqrt()
        share = (state["case"]["max_norm"] / (norm + 1e-6)).clamp_max(1.0).float()
        torch._foreach_copy_(grads, (every * share).split([gr.numel() for gr in grads]))
        return [norm.float()] + state["flats"]


def _run_sgd(state):
    case = state["case"]
    if own:
        norm = state["opt"].step(state["scaler"], max_norm=case["max_norm"])
        return [norm, state["arena"].data, state["opt"].buf]
    p, g, m, group = state["param"], state["grad"], state["momentum"], state["group"]
    norm = g.double().square().sum().sqrt() / state["scale"].double()
    share = ((case["max_norm"] / (norm + 1e-6)).clamp_max(1.0) / state["scale"].double()).float()
    d = g * share + torch.where(group == 1, 5e-4, 0.0) * p
    new = 0.937 * m + d
    live = group < 3
    m.copy_(torch.where(live, new, m))
    p.copy_(torch.where(live, p - 0.01 * (d + 0.937 * new), p))
    return [norm.float().reshape(()), p, m]


# ------------------------------------------------------------------------------------------------------------- bytes and operations
def work(case):
    if case["op"] == "ce":
        n, d, v = case["rows"], case["width"], case["classes"]
        size = 4 if case["dtype"] == "fp32" else 2
        labelled = n * (1 - case["unlabelled"])
        tensors = (labelled * d + v * d + (v if case["bias"] else 0)) * size
        out = 4 * n if case["reduction"] == "none" else 4
        if not case["train"]:
            return {"bytes": tensors + 8 * n + out, "flops": 2 * labelled * d * v}
        return {"bytes": tensors + 8 * n + out + (n * d + v * d + (v if case["bias"] else 0)) * size, "flops": 6 * labelled * d * v}
    if case["op"] == "clip":
        size = {"fp32": 4.0, "mixed": 8 / 3}.get(case["dtype"], 2.0)
        n = sum(_sizes(case))
        return {"bytes": 2 * size * n, "flops": 3 * n}
    channels = [max(8, math.ceil(c * case["width"] / 8) * 8) for c in (64, 128, 256, 512, 1024)]
    repeats = [max(1, round(r * case["depth"])) for r in (1, 6, 12, 18, 6)]
    n, cin = 0, 3
    for c, r in zip(channels, repeats):
        n += 10 * cin * c + 4 * c + (r - 1) * (10 * c * c + 4 * c)
        cin = c
    n += 85 * cin + 85
    return {"bytes": (4 + 8 + 8 + 1) * n, "flops": 10 * n}


# --------------------------------------------------------------------------------------------------------------- answers in 64 bits
def exact(case, seed):
    return {"ce": _exact_ce, "clip": _exact_clip, "sgd": _exact_sgd}[case["op"]](prepare(case, seed))


def _exact_ce(state):
    """Autograd through log-softmax in double precision."""
    case = state["case"]
    leaves = [t.detach().double().requires_grad_(case["train"]) for t in (state["x"], state["weight"], state["bias"]) if t is not None]
    z = torch.nn.functional.linear(*leaves)
    keep = (state["target"] >= 0).nonzero()[:, 0]
    logp = z.index_select(0, keep).log_softmax(1)
    hit = logp[torch.arange(keep.numel(), device=z.device), state["target"][keep]]
    eps = case["smoothing"]
    rows = z.new_zeros(case["rows"]).index_copy(0, keep, -(1 - eps) * hit - (eps * logp.mean(1) if eps else 0.0))
    if case["reduction"] == "none":
        loss = rows
    else:
        loss = rows.sum() / (max(keep.numel(), 1) if case["reduction"] == "mean" else 1)
    if not case["train"]:
        return loss.detach()
    return (loss.detach(), *torch.autograd.grad(loss, leaves, state["upstream"].double()))


def _exact_clip(state):
    parts = [gr.double() for gr in state["grads"]]
    norm = torch.linalg.vector_norm(torch.stack([torch.linalg.vector_norm(p) for p in parts]))
    factor = min(1.0, state["case"]["max_norm"] / (float(norm) + 1e-6))
    flats = [f.double() for f in state["flats"]]
    starts = {f.data_ptr(): k for k, f in enumerate(state["flats"])}
    for gr, p in zip(state["grads"], parts):
        k = starts[gr.untyped_storage().data_ptr()]
        flats[k][gr.storage_offset():gr.storage_offset() + gr.numel()] = p * factor
    return [norm] + flats


def _exact_sgd(state):
    """torch.optim.SGD in double precision on the values of each group."""
    case, group = state["case"], state["group"]
    grad = state["grad"].double() / case["scale"]
    norm = torch.linalg.vector_norm(grad)
    grad *= min(1.0, case["max_norm"] / (float(norm) + 1e-6))
    p, m = state["param"].double(), state["momentum"].double()
    for k, decay in ((0, 0.0), (1, 5e-4), (2, 0.0)):
        at = (group == k).nonzero()[:, 0]
        q = torch.nn.Parameter(p[at])
        q.grad = grad[at]
        opt = torch.optim.SGD([q], lr=0.01, momentum=0.937, weight_decay=decay, nesterov=True)
        opt.state[q]["momentum_buffer"] = m[at]
        opt.step()
        p[at], m[at] = q.detach(), opt.state[q]["momentum_buffer"]
    return [norm, p, m]
