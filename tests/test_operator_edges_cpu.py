"""The operators at the edges of what their documentation allows, without a GPU."""
import os
import subprocess
import sys

import pytest
import torch

from operator_bounds import check, wide_forms
from test_gpu_operator_edges import WIDE
from test_operators_cpu import INVALID, create_loss

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "msccl-tools_amd", "csrc")

WALK = r"""
#include <cstdio>
#include <vector>
#include "step_walk.h"
int main() {
  for (int k = 1; k <= 700; k += k < 140 ? 1 : 8)
    for (int first = 0, steps = (k + 63) / 64; first < steps; ++first) {
      mscclx::StepWalk<64, 128> walk(k, first);
      std::vector<int> seen(steps);
      for (int s = 0; s < steps; ++s) {
        walk.next();
        const int step = (first + s) % steps, there = k - step * 64 < 64 ? k - step * 64 : 64;
        // at the step's bytes, and all of its values are there, none of the next row's
        if (walk.further != step * 128 || (walk.left < 64 ? walk.left : 64) != there || walk.left > k - step * 64) return printf("k %d first %d: turn %d\n", k, first, s), 1;
        ++seen[step];
      }
      for (int n : seen) if (n != 1) return printf("k %d first %d: a step came %d times\n", k, first, n), 1;
      for (int s = 0; s < 8; ++s) {
        walk.next();
        if (walk.left > 0) return printf("k %d first %d: %d values left behind the last step\n", k, first, walk.left), 1;
      }
    }
}
"""


def test_the_steps_of_a_row_come_once_each(tmp_path):
    source, exe = tmp_path / "walk.cpp", str(tmp_path / "walk")
    source.write_text(WALK)
    subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-I", CSRC, str(source), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout + r.stderr


@pytest.mark.parametrize("rows", [(64, (1 << 63) - 1), ((1 << 63) - 1, 64), (1, 1 << 62), (64, (1 << 63) - 64)])
def test_rows_whose_sum_passes_64_bits_are_refused(mscclx_lib, rows):
    rc, handle, _, _ = create_loss(mscclx_lib, rows=rows)
    assert rc == INVALID and not handle.value


@pytest.mark.parametrize("changed", [dict(tokens=(1 << 64) + 5), dict(hidden=(1 << 32) + 64), dict(rank_rows=[(1 << 64) + 100]), dict(piece_bytes=-1), dict(piece_bytes=(1 << 64) + 1),
                                     dict(ignore_index=1 << 63), dict(ignore_index=-(1 << 63) - 1)])
def test_numbers_that_no_argument_of_the_library_holds_are_refused(mscclx_lib, changed):
    """ctypes would cut them off: 2^64 + 5 tokens would be 5."""
    from msccl.executor import GradientClip, VocabLoss
    with pytest.raises(ValueError, match="range"):
        VocabLoss().setup(**{**dict(tokens=8, hidden=64, rank_rows=[100], dtype="bfloat16"), **changed})
    with pytest.raises(ValueError, match="range"):
        GradientClip().setup([3, (1 << 64) + 3], "float32")


def test_workspace_has_no_32_bit_logits_that_no_call_keeps(mscclx_lib):
    """One rank keeps those of at most 32 tokens, eight ranks of 127; what else a token costs is its 16-bit probabilities and their statistics."""
    def size(ranks, tokens, rows=131072):
        rc, handle, nbytes, _ = create_loss(mscclx_lib, rows=(rows // ranks,) * ranks, hidden=8, tokens=tokens)
        assert rc == 0
        mscclx_lib.mscclx_vocab_loss_destroy(handle)
        return nbytes
    per_token = 131072 * 2 + 131072 // 32 * 8
    assert size(1, 128) - size(1, 32) <= 96 * per_token * 1.05
    assert size(8, 127) - size(1, 127) >= 95 * 131072 * 4    # their logits, at least


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens, hidden, rows", WIDE)
def test_the_bound_for_few_tokens_tells_two_numbers_from_one(tokens, hidden, rows, dtype):
    """The bound that the kernel's gradients of few tokens are held to: G in two 16-bit numbers meets it, G rounded once does not."""
    gen = torch.Generator().manual_seed(11)
    weights = [(torch.randn(r, hidden, generator=gen) * 1.5 / hidden ** 0.5).to(dtype) for r in rows]
    x = torch.randn(tokens, hidden, generator=gen).to(dtype)
    labels = torch.randint(sum(rows), (tokens,), generator=gen)
    upstream = torch.rand(tokens, generator=gen) + 0.5
    forms = wide_forms(x, weights, labels, -100, upstream)
    unit = (2.0 ** 15 if dtype == torch.float16 else 1.0) / upstream.max().double()
    G = forms["G"] * unit
    once = G.to(dtype).double()
    both = once + (G - once).to(dtype).double()
    w = torch.cat(weights).double()
    gradients = lambda G: {"dx": (G @ w / unit).to(dtype), "dw": (G.t() @ x.double() / unit).to(dtype)}  # noqa: E731
    for what, got in gradients(both).items():
        check(what, got, forms[what])
    with pytest.raises(AssertionError, match="beyond their bound"):
        for what, got in gradients(once).items():
            check(what, got, forms[what])


COPY = r"""
#include "tile_product.h"
__global__ void copy(const char* const* from, const int* which) {
  __shared__ __attribute__((aligned(1024))) char smem[1024];
  const int lane = threadIdx.x;
  typedef __attribute__((address_space(3))) char* lds_char;
  mscclx::copy_to_lds((unsigned)(uintptr_t)(lds_char)smem, lane * 16, mscclx::resource_at(from[which[lane]]), 0);
}
"""


def test_copies_to_lds_wait_for_a_resource_that_a_vector_instruction_wrote(tmp_path):
    """Five wait states between the write of a scalar register and the load that takes its address from it, in the compiled code."""
    sys.path.insert(0, CSRC)
    import build
    source, listing = tmp_path / "copy.hip", tmp_path / "copy.s"
    source.write_text(COPY)
    subprocess.run([build.hipcc(), "-O3", "-std=c++17", "-I", CSRC, "--offload-arch=gfx950", "--cuda-device-only", "-S", str(source), "-o", str(listing)], check=True)
    lines = [line.split(";")[0].split() for line in listing.read_text().splitlines()]
    lines = [line for line in lines if line and not line[0].startswith(".") and not line[0].endswith(":")]
    load = next(i for i, line in enumerate(lines) if line[0] == "buffer_load_dwordx4")
    write = max(i for i in range(load) if lines[i][0] == "v_readfirstlane_b32")
    states = sum(int(line[1], 0) + 1 if line[0] == "s_nop" else 1 for line in lines[write + 1:load])
    assert states >= 5, lines[write:load + 1]
