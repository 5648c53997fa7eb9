"""A training step's tail as it is used: every data-parallel rank's loss and gradients, the all-reduce that sums the gradients over the
ranks, their norm and clipping -- all on one stream, and once more from a HIP graph."""
import pytest
import torch

from operator_bounds import check, loss_forms

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_loss_all_reduce_norm_and_clip(dtype):
    from msccl.executor import Executor, GradientClip, VocabLoss
    from msccl.programs import catalog
    ranks, tokens, hidden, rows = 4, 96, 64, [70, 58]   # four data-parallel ranks, each with a vocabulary on two tensor-parallel ones
    name = str(dtype).split(".")[1]
    gen = torch.Generator().manual_seed(1)
    weights = [(torch.randn(r, hidden, generator=gen) * 0.2).to(dtype).cuda() for r in rows]
    batches = [((torch.randn(tokens, hidden, generator=gen)).to(dtype).cuda(), torch.randint(sum(rows), (tokens,), generator=gen).cuda()) for _ in range(ranks)]
    # a rank's gradients of both pieces lie one behind the other in its buffer of the collective
    buffers = [torch.zeros(sum(rows) * hidden, dtype=dtype, device="cuda") for _ in range(ranks)]
    views = [[v.view(r, hidden) for v, r in zip(b.split([r * hidden for r in rows]), rows)] for b in buffers]
    loss = VocabLoss()
    loss.setup(tokens, hidden, rows, dtype, reduction="mean")
    reduce = Executor(catalog.ring_allreduce(ranks, channels=1, instances=1))
    reduce.setup(buffers[0].numel() * buffers[0].element_size() // ranks, dtype)
    reduce.bind(buffers, [None] * ranks)
    clip = GradientClip()
    out = [torch.zeros(b.numel(), device="cuda") for b in buffers]
    clip.setup([b.numel() for b in buffers], dtype, out_dtype="float32", counted=[r == 0 for r in range(ranks)])
    clip.bind(buffers, out)
    max_norm = 0.05

    def step():
        losses = []
        for (x, labels), dw in zip(batches, views):
            losses.append(loss.run(x, weights, labels, dweights=dw)[0])
        reduce.launch()
        clip.launch(max_norm=max_norm, scale=1.0 / ranks)
        return losses

    def verify(losses):
        u = torch.finfo(dtype).eps / 2
        forms = [loss_forms(x, weights, labels, "mean", -100, 1.0) for x, labels in batches]
        for got, form in zip(losses, forms):
            check("loss", got, form["loss"])
        # the sum over the ranks: each rank's gradient is off by its bound, and each of the ring's additions rounds once
        total = sum(f["dw"][0] for f in forms)
        off = sum(f["dw"][1] for f in forms) + ranks * 1.01 * u * sum(f["dw"][0].abs() + f["dw"][1] for f in forms) + torch.finfo(dtype).tiny
        for b in buffers:
            check("sum over ranks", b.view(sum(rows), hidden), (total, off))
            assert torch.equal(b, buffers[0])
        # clipping, against the 64-bit form on the very sums that it read
        summed = buffers[0].cpu().double()
        norm = summed.square().sum().sqrt() / ranks
        check("norm", clip.norm, (norm, norm * 2.0 ** -23))
        assert float(norm) > max_norm                     # it clips
        for o in out:
            want = summed * (max_norm / (norm + 1e-6) / ranks)
            check("clipped", o, (want, want.abs() * 2.0 ** -22 + 2.0 ** -149))

    losses = step()
    reduce.wait()
    torch.cuda.synchronize()
    verify(losses)
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        losses = step()
    for seed in (2, 3):
        gen = torch.Generator().manual_seed(seed)
        for x, labels in batches:
            x.copy_(torch.randn(tokens, hidden, generator=gen).to(dtype))
            labels.copy_(torch.randint(sum(rows), (tokens,), generator=gen))
        for t in (*buffers, *out):
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        verify(losses)
