"""Opt-in to dynamic shared memory is remembered per device and kernel: the record on the
CPU, and products on a second device where there is one."""

from __future__ import annotations

import shutil
import subprocess
from pathlib import Path

import pytest
import torch

CSRC = Path(__file__).resolve().parents[1] / "ictc_o2_hp_b200" / "csrc"

PROGRAM = r"""
#include "smem_grants.h"
#include <cstdio>
int main() {
  static ictc::SmemGrants g;
  static char kernels[1500];
  int bad = 0;
  const auto expect = [&](bool ok, int line) { if (!ok) { std::printf("line %d\n", line); ++bad; } };
  for (int k = 0; k < 400; ++k) {
    expect(!g.covers(0, kernels + k, 1), __LINE__);
    g.record(0, kernels + k, 1000 + k);
  }
  for (int k = 0; k < 400; ++k) {
    expect(g.covers(0, kernels + k, 1000 + k), __LINE__);
    expect(!g.covers(0, kernels + k, 1001 + k), __LINE__);
    expect(!g.covers(1, kernels + k, 1), __LINE__);      // another device: not granted there
    g.record(1, kernels + k, 10);
    expect(g.covers(1, kernels + k, 10) && !g.covers(1, kernels + k, 11), __LINE__);
    expect(g.covers(0, kernels + k, 1000 + k), __LINE__);
  }
  g.record(0, kernels, 5000);                            // a larger grant replaces the first
  expect(g.covers(0, kernels, 5000), __LINE__);
  for (int d = 0; d < 8; ++d)                            // more than there are slots
    for (int k = 0; k < 1500; ++k) {
      g.record(d, kernels + k, 7 + d);
      expect(!g.covers(d, kernels + k, 8 + d), __LINE__);
    }
  return bad ? 1 : 0;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs a host compiler")
def test_grants_are_kept_per_device_and_kernel(tmp_path):
    source, program = tmp_path / "grants.cpp", tmp_path / "grants"
    source.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", f"-I{CSRC}", str(source),
                    "-o", str(program)], check=True)
    run = subprocess.run([str(program)], capture_output=True, text=True)
    assert run.returncode == 0, run.stdout


@pytest.mark.gpu
def test_second_device(cuda_device):
    if torch.cuda.device_count() < 2:
        pytest.skip("needs two devices")
    from ictc_o2_hp_b200 import dense
    for dtype in (torch.float32, torch.bfloat16):
        for rows, width in ((700, 48), (700, 256)):
            outs = []
            for device in ("cuda:0", "cuda:1"):
                x = torch.linspace(-2, 2, rows * width, dtype=dtype, device=device)
                x = x.reshape(rows, width).requires_grad_(True)
                w = torch.linspace(-1, 1, width * width, dtype=dtype, device=device)
                y = dense.linear(dense.layer_norm(x), w.reshape(width, width), activation="silu")
                outs.append((y.detach().cpu(), torch.autograd.grad(y.sum(), x)[0].cpu()))
            assert all(torch.equal(a, b) for a, b in zip(*outs))
