"""Plain 64-bit forms of the vocabulary loss and of clipping, and how far a kernel may be from them.

The bounds count roundings.  u: half a step of the 16-bit type (finfo.eps / 2).  A 32-bit operation is off by 2^-24; 2^-23 per
operation is allowed for the matrix cores, which do not say how they round inside.
"""
import torch

F32 = 2.0 ** -23


def loss_forms(x, weights, labels, reduction, ignore_index, upstream):
    """Everything in 64 bits on the CPU: a dict of values and of elementwise bounds."""
    dtype = x.dtype
    u = torch.finfo(dtype).eps / 2
    x, w = x.cpu().double(), torch.cat([t.cpu() for t in weights]).double()
    labels = labels.cpu().long()
    n, d = x.shape
    v = w.shape[0]
    z = x @ w.t()
    size = x.abs() @ w.abs().t()
    lse = torch.logsumexp(z, 1)
    kept = labels != ignore_index
    target = labels.where(kept, torch.zeros_like(labels))
    y = torch.zeros_like(z)
    if n:
        y[torch.arange(n), target] = 1.0
    rows = torch.where(kept, lse - (z * y).sum(1), torch.zeros_like(lse))
    # a logit is a sum of d exact products; a sum of v exponentials, each off by its argument's rounding, its own and the running sum's
    z_off = (d + 4) * F32 * (size.amax(1) if n else size.sum(1))
    spread = (z.amax(1) - (torch.softmax(z, 1) * z).sum(1)) if n else lse
    lse_off = z_off + F32 * (lse.abs() + 4 * spread + 64)
    row_off = z_off + lse_off + F32 * rows.abs()
    count = max(1, int(kept.sum()))
    g = torch.as_tensor(upstream).cpu().double() * kept
    if reduction == "mean":
        g = g / count
    g = g.expand(n)
    p = torch.exp(z - lse[:, None])
    big = g.abs().max() if n else torch.zeros(())
    G = g[:, None] * (p - y)
    # E and G are rounded to the type; the exponent is off by the logit's and lse's error; fp16 has 2^-25 of its unit 2^15 at the least.
    # bf16 has the exponents of 32 bits, whose hardware exponential gives 0 where the result would be below 2^-126: E = exp(z - m) <= 1 and
    # f = exp(m - lse) <= 1, so a flushed E costs at most 2^-126 f and a flushed f at most 2^-126 E, 2^-126 each.
    least = 2.0 ** -25 / 2.0 ** 15 if dtype == torch.float16 else 2.0 ** -126
    relative = 2 * (z_off + lse_off)[:, None] + F32 * (8 + (z - lse[:, None]).abs())
    G_off = g.abs()[:, None] * (p * (1.1 * u + 1.5 * relative) + (p - y).abs() * 1.1 * u) + 2.2 * least * big * kept[:, None]
    dx, dw = G @ w, G.t() @ x
    dx_size, dw_size = G.abs() @ w.abs(), G.abs().t() @ x.abs()
    tiny = torch.finfo(dtype).tiny * torch.finfo(dtype).eps
    off = lambda value, size, rounded, terms: rounded * 1.01 + (terms + 8) * F32 * size + u * 1.01 * value.abs() + tiny  # noqa: E731
    total = rows if reduction == "none" else rows.sum() / (count if reduction == "mean" else 1)
    total_off = row_off * kept if reduction == "none" else (row_off * kept).sum() / (count if reduction == "mean" else 1) + F32 * total.abs()
    return {"loss": (total, total_off), "lse": (lse, lse_off),
            "dx": (dx, off(dx, dx_size, G_off @ w.abs(), v)), "dw": (dw, off(dw, dw_size, G_off.t() @ x.abs(), n))}


def wide_forms(x, weights, labels, ignore_index, upstream):
    """dx and dw as loss_forms, but with G held in two 16-bit numbers: what the second leaves is half a step of half a step."""
    forms = loss_forms(x, weights, labels, "none", ignore_index, upstream)
    dtype = x.dtype
    u = torch.finfo(dtype).eps / 2
    x, w, labels = x.cpu().double(), torch.cat([t.cpu() for t in weights]).double(), labels.cpu().long()
    lse, lse_off = forms["lse"]
    n = x.shape[0]
    z = x @ w.t()
    y = torch.zeros_like(z)
    kept = labels != ignore_index
    y[torch.arange(n), labels.where(kept, torch.zeros_like(labels))] = 1.0
    g = upstream.cpu().double() * kept
    p = torch.exp(z - lse[:, None])
    G = g[:, None] * (p - y)
    z_off = (x.shape[1] + 4) * F32 * (x.abs() @ w.abs().t()).amax(1)
    relative = 2 * (z_off + lse_off)[:, None] + F32 * (8 + (z - lse[:, None]).abs())
    least = 2.0 ** -25 / 2.0 ** 15 if dtype == torch.float16 else 2.0 ** -126
    G_off = g.abs()[:, None] * (p * 1.5 * relative + (p - y).abs() * (1.1 * u * u + 16 * 2.0 ** -24)) + 2.2 * least * g.abs().max() * kept[:, None]
    tiny = torch.finfo(dtype).tiny * torch.finfo(dtype).eps
    off = lambda value, size, rounded, terms: rounded * 1.01 + (terms + 8) * F32 * size + u * 1.01 * value.abs() + tiny  # noqa: E731
    dx, dw = G @ w, G.t() @ x
    return {"G": G, "dx": (dx, off(dx, G.abs() @ w.abs(), G_off @ w.abs(), 2 * w.shape[0])),
            "dw": (dw, off(dw, G.abs().t() @ x.abs(), G_off.t() @ x.abs(), 2 * n))}


def check(what, got, form):
    """`got` within the bound of form = (value, bound), elementwise; NaN only where the value is NaN."""
    value, bound = form
    got = got.cpu().double()
    assert got.shape == value.shape, (what, got.shape, value.shape)
    assert torch.equal(torch.isnan(got), torch.isnan(value)), f"{what}: NaN elsewhere than in the plain form"
    sure = ~torch.isnan(value)
    far = ((got - value).abs() - bound)[sure & ~(got == value)]
    if far.numel() and not float(far.max()) <= 0:
        worst = ((got - value).abs() / bound).where(sure & ~(got == value), torch.zeros_like(value))
        at = int(worst.argmax())
        raise AssertionError(f"{what}: {int((far > 0).sum())} of {value.numel()} values beyond their bound; worst at {at}: "
                             f"{float(got.flatten()[at])} for {float(value.flatten()[at])}, {float(worst.max()):.2f} bounds off")


def clip_forms(grads, counted, norm, scale, max_norm, out_dtypes):
    """(norm, coefficient, outputs with bounds) in 64 bits."""
    wide = [g.cpu().double() for g in grads]
    taken = torch.cat([g.reshape(-1) for g, c in zip(wide, counted) if c] or [torch.zeros(0, dtype=torch.float64)])
    if norm == "l2":
        size = (taken * taken).sum().sqrt()
    else:
        size = taken.abs().max() if taken.numel() else torch.zeros((), dtype=torch.float64)
    size = size * abs(scale)
    c = torch.ones((), dtype=torch.float64) if max_norm is None else (max_norm / (size + 1e-6))
    c = torch.where(c >= 1, torch.ones_like(c), c)
    outs = []
    for g, t in zip(wide, out_dtypes):
        out = g * (c * scale)
        # the factor, the product and the output are rounded once each
        bound = out.abs() * (torch.finfo(t).eps / 2 * 1.01 + 3 * 2.0 ** -24) + torch.finfo(t).tiny * torch.finfo(t).eps
        outs.append((out, bound))
    return size, c, outs
