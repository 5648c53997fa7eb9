"""What the operators beside the collectives are measured on: the vocabulary-parallel loss with its gradients, and the
global gradient norm with clipping.

`run` computes a case in its plain form (torch, 32 bits and more), or, where `own` is true, through msccl.executor.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}
IGNORE = -100


def _executor():
    package = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "msccl-tools_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    import msccl.executor
    return msccl.executor


def _loss(name, tokens, hidden, vocab, ranks, dtype, reduction, ignored, grad):
    return {"name": name, "op": "loss", "tokens": tokens, "hidden": hidden, "vocab": vocab, "ranks": ranks, "dtype": dtype,
            "reduction": reduction, "ignored": ignored, "grad": grad}


def _clip(name, tensors, elements, uneven, dtype, out_dtype, norm, clip):
    return {"name": name, "op": "clip", "tensors": tensors, "elements": elements, "uneven": uneven, "dtype": dtype,
            "out_dtype": out_dtype, "norm": norm, "clip": clip}


def listed():
    return [
        # one token scored against the vocabulary of eight ranks, as a server does for each token that it is given: latency
        _loss("score one token", 1, 2048, 32768, 8, "bfloat16", "none", False, False),
        # the loss of a batch of held-out text, no gradient: one long product with a softmax behind it
        _loss("evaluate 4096 tokens", 4096, 4096, 65536, 8, "bfloat16", "mean", True, False),
        # a micro-batch of a small model on two ranks: short in every direction, so launches and the tails of the grid count
        _loss("train 128 tokens", 128, 1024, 8192, 2, "float16", "mean", True, True),
        # an odd number of tokens and a vocabulary that neither the ranks nor any tile divides, weighted row by row
        _loss("train 1021 odd tokens", 1021, 1288, 32003, 5, "float16", "none", True, True),
        # a training micro-batch of ordinary size
        _loss("train 2048 tokens", 2048, 2048, 32768, 8, "bfloat16", "mean", True, True),
        # the largest: a long batch against a large vocabulary
        _loss("train 8192 tokens", 8192, 4096, 131072, 8, "bfloat16", "sum", True, True),
        # the gradients of a small model, a few hundred KiB in many tensors: launches count
        _clip("clip a small model", 74, 300_000, True, "float32", "float32", "l2", True),
        # the 64 ranks' buffers of the small-message ring, 256 KiB each: the largest magnitude, to find an overflow
        _clip("maximum over 64 ranks", 64, 64 * 131072, False, "float16", "float16", "max", False),
        # eight ranks' buffers of 32 MiB
        _clip("norm over 8 ranks", 8, 8 * 8388608, False, "float32", "float32", "l2", False),
        # a model's gradients in tensors of very different sizes, clipped into the optimizer's 32-bit bucket
        _clip("clip 291 uneven tensors", 291, 400_000_003, True, "bfloat16", "float32", "l2", True),
        # the 32 ranks' buffers of the two-level all-reduce, 128 MiB each
        _clip("clip 32 ranks' buckets", 32, 32 * 67108864, False, "bfloat16", "bfloat16", "l2", True),
    ]


def _between(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    if rng.random() < 0.6:
        grad = rng.random() < 0.65
        case = _loss("", _between(rng, 1, 8192), 8 * _between(rng, 64, 512), _between(rng, 2000, 131072), rng.choice([1, 2, 3, 4, 5, 8, 16, 32]),
                     rng.choice(["bfloat16", "float16"]), rng.choice(["none", "sum", "mean"]), rng.random() < 0.7, grad)
    else:
        clip = rng.random() < 0.7
        dtype = rng.choice(["bfloat16", "float16", "float32"])
        tensors = _between(rng, 1, 500)
        case = _clip("", tensors, max(tensors, _between(rng, 10_000, 1_000_000_000)), rng.random() < 0.7, dtype,
                     rng.choice([dtype, "float32"]), rng.choice(["l2", "l2", "max"]), clip)
    del case["name"]
    return case


def _shards(case):
    """Rows of the output matrix on each rank: as even as the vocabulary allows."""
    v, r = case["vocab"], case["ranks"]
    return [v // r + (i < v % r) for i in range(r)]


def _sizes(case):
    """Elements of each tensor: equal, or matrices beside vectors a few hundred times smaller, odd sizes among them."""
    n, total = case["tensors"], case["elements"]
    share = [1 + (i * 7919 % 61) ** 2 * (i % 3 != 1) for i in range(n)] if case["uneven"] else [1] * n
    whole = sum(share)
    sizes = [max(1, total * s // whole) for s in share]
    sizes[0] += max(0, total - sum(sizes))
    return sizes


def _device():
    return "cuda:0" if torch.cuda.is_available() else "cpu"


def _inputs(case, seed):
    dev = _device()
    gen = torch.Generator(device=dev).manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, generator=gen, device=dev)  # noqa: E731
    dtype = DTYPES[case["dtype"]]
    if case["op"] == "loss":
        n, d = case["tokens"], case["hidden"]
        # logits of about 1.5 around zero; every second row leans to its label, as a trained model's does
        weights = [(normal(rows, d) * (1.5 / math.sqrt(d))).to(dtype) for rows in _shards(case)]
        labels = torch.randint(case["vocab"], (n,), generator=gen, device=dev)
        lean = 4.0 * (torch.rand(n, 1, generator=gen, device=dev) < 0.5)
        x = (normal(n, d) + lean * torch.cat(weights)[labels].float()).to(dtype)
        if case["ignored"]:  # a prompt's tokens, and the padding behind a sequence
            labels[torch.rand(n, generator=gen, device=dev) < 0.15] = IGNORE
        upstream = torch.rand(n, generator=gen, device=dev) + 0.5 if case["reduction"] == "none" else torch.rand((), generator=gen, device=dev) + 0.5
        return {"x": x, "weights": weights, "labels": labels, "upstream": upstream}
    # gradients of a few 1e-3 with single large values among them, summed over eight ranks: scale makes their mean
    grads = []
    for size in _sizes(case):
        g = normal(size)
        grads.append((g * (1e-3 + 1e-4 * g * g)).to(dtype))
    return {"grads": grads, "max_norm": 1e-2, "scale": 0.125}


def prepare(case, seed):
    state = dict(_inputs(case, seed), case=case)
    out = DTYPES[case["out_dtype"]] if case["op"] == "clip" else None
    if case["op"] == "clip" and case["clip"]:  # the bucket that the optimizer reads
        state["bucket"] = torch.empty(sum(_sizes(case)), dtype=out, device=_device())
    if own:  # the operator's handle with its workspace; gradients and bucket keep their places from step to step
        if case["op"] == "loss":
            state["handle"] = _executor().VocabLoss(device=_device())
            state["handle"].setup(case["tokens"], case["hidden"], _shards(case), case["dtype"], reduction=case["reduction"], ignore_index=IGNORE,
                                  gradients=case["grad"])
        else:
            state["handle"] = _executor().GradientClip(device=_device())
            state["handle"].setup(_sizes(case), case["dtype"], out_dtype=case["out_dtype"], norm=case["norm"])
            state["handle"].bind(state["grads"], list(state["bucket"].split(_sizes(case))) if case["clip"] else None)
    return state


def run(state):
    case = state["case"]
    if case["op"] == "loss":
        return _run_loss(state, case)
    return _run_clip(state, case)


def _run_loss(state, case):
    x, weights, labels, upstream = state["x"], state["weights"], state["labels"], state["upstream"]
    if own:
        if not case["grad"]:
            loss, lse = state["handle"].forward(x, weights, labels)
            return {"loss": loss, "lse": lse}
        loss, lse, dx, dweights = state["handle"].run(x, weights, labels, upstream)
        return {"loss": loss, "lse": lse, "dx": dx, "dweights": dweights}
    dtype = x.dtype
    x, w = x.float(), torch.cat(weights).float()
    logits = x @ w.t()
    top = logits.amax(1, keepdim=True)
    lse = top + (logits - top).exp().sum(1, keepdim=True).log()
    kept = labels != IGNORE
    target = labels.clamp_min(0).unsqueeze(1)
    rows = torch.where(kept, (lse - logits.gather(1, target))[:, 0], 0.0)
    count = kept.sum().clamp_min(1)
    loss = rows if case["reduction"] == "none" else rows.sum() if case["reduction"] == "sum" else rows.sum() / count
    if not case["grad"]:
        return {"loss": loss, "lse": lse[:, 0]}
    factor = upstream / count if case["reduction"] == "mean" else upstream
    p = (logits - lse).exp()
    p.scatter_add_(1, target, torch.full_like(lse, -1.0))
    p *= (kept * factor).unsqueeze(1)
    return {"loss": loss, "lse": lse[:, 0], "dx": (p @ w).to(dtype), "dweights": [g.to(dtype) for g in (p.t() @ x).split(_shards(case))]}


def _run_clip(state, case):
    if own:
        handle = state["handle"]
        handle.launch(max_norm=state["max_norm"] if case["clip"] else None, scale=state["scale"])
        return {"norm": handle.norm, "bucket": state["bucket"]} if case["clip"] else {"norm": handle.norm}
    flat = torch.cat(state["grads"])
    size = flat.double().square().sum().sqrt() if case["norm"] == "l2" else flat.abs().amax().double()
    norm = size * state["scale"]
    if not case["clip"]:
        return {"norm": norm.float()}
    factor = (state["max_norm"] / (norm + 1e-6)).clamp_max(1.0) * state["scale"]
    state["bucket"].copy_(flat.float() * factor.float())
    return {"norm": norm.float(), "bucket": state["bucket"]}


def work(case):
    if case["op"] == "loss":
        n, d, v = case["tokens"], case["hidden"], case["vocab"]
        moved = 2 * (n * d + v * d) * (2 if case["grad"] else 1) + 8 * n + 8 * n
        return {"bytes": moved, "flops": (6 if case["grad"] else 2) * n * d * v}
    n = sum(_sizes(case))
    size = {"bfloat16": 2, "float16": 2, "float32": 4}
    moved = n * size[case["dtype"]] + (n * size[case["out_dtype"]] if case["clip"] else 0)
    return {"bytes": moved, "flops": (3 if case["clip"] else 2) * n}


def exact(case, seed):
    made = _inputs(case, seed)
    if case["op"] == "clip":
        size = torch.zeros((), dtype=torch.float64, device=_device())
        for g in made["grads"]:
            wide = g.to(torch.float64)
            size = size + (wide * wide).sum() if case["norm"] == "l2" else torch.maximum(size, wide.abs().max())
        norm = (size.sqrt() if case["norm"] == "l2" else size) * made["scale"]
        if not case["clip"]:
            return {"norm": norm}
        factor = min(1.0, made["max_norm"] / (float(norm) + 1e-6)) * made["scale"]
        return {"norm": norm, "bucket": torch.cat([g.to(torch.float64) * factor for g in made["grads"]])}
    # rows in blocks, each against the whole vocabulary; the gradients as sums over the blocks
    n, reduction = case["tokens"], case["reduction"]
    w = torch.cat([s.to(torch.float64) for s in made["weights"]])
    labels, valid = made["labels"], int((made["labels"] != IGNORE).sum())
    losses, lses, dx = [], [], []
    dw = torch.zeros_like(w) if case["grad"] else None
    for at in range(0, n, 2048):
        x, label = made["x"][at:at + 2048].to(torch.float64), labels[at:at + 2048]
        z = torch.matmul(x, w.t())
        lse = torch.logsumexp(z, dim=1)
        keep = (label != IGNORE).to(torch.float64)
        index = torch.where(label == IGNORE, 0, label)
        here = torch.arange(len(label), device=z.device)
        losses.append((lse - z[here, index]) * keep)
        lses.append(lse)
        if not case["grad"]:
            continue
        g = keep * (made["upstream"][at:at + 2048] if reduction == "none" else made["upstream"]).to(torch.float64)
        if reduction == "mean":
            g = g / max(1, valid)
        z.sub_(lse[:, None]).exp_()
        z[here, index] -= 1.0
        z.mul_(g[:, None])
        dx.append(torch.matmul(z, w))
        dw.addmm_(z.t(), x)
    loss = torch.cat(losses)
    loss = loss if reduction == "none" else loss.sum() if reduction == "sum" else loss.sum() / max(1, valid)
    if not case["grad"]:
        return {"loss": loss, "lse": torch.cat(lses)}
    return {"loss": loss, "lse": torch.cat(lses), "dx": torch.cat(dx), "dweights": list(dw.split(_shards(case)))}
