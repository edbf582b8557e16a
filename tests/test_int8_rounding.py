"""The arithmetic that the 8-bit kernels lean on, over all of its inputs: the
division by multiplication as the header forms it, and the integers of 16-bit
rows against fp32's division for every pair of significands."""

from __future__ import annotations

import re
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

import double_attention as da
from test_int8_ops import HALF, _device

ROWS_HEADER = Path(__file__).resolve().parents[1] / "double-attention_amd" / "csrc" / "int8_rows.h"

_DIVISIONS = """
#include <cstdint>
#include <cstdio>
#define __device__
#define __forceinline__ inline
static uint32_t __umulhi(uint32_t a, uint32_t b) { return static_cast<uint32_t>(static_cast<uint64_t>(a) * b >> 32); }
@DIVISION@
static int wrong(uint32_t d, uint64_t n) {
  if (n >= 1ull << 31 || fast_div(static_cast<uint32_t>(n), make_fast_div(d)) == n / d) return 0;
  std::printf("%llu / %u\\n", static_cast<unsigned long long>(n), d);
  return 1;
}
int main() {
  // Groups of a row: 1 to 65536.  A quotient goes wrong first beside a multiple of d.
  for (uint32_t d = 1; d <= 65536; ++d) {
    const uint64_t most = ((1ull << 31) - 1) / d;
    uint64_t seed = d;
    for (int i = 0; i < 300; ++i) {
      seed = seed * 6364136223846793005ull + 1442695040888963407ull;
      const uint64_t q = i < 20 ? i : i < 60 ? most - (i - 20) % (most + 1) : (seed >> 33) % (most + 1);
      for (int64_t off = -1; off <= 1; ++off)
        if (static_cast<int64_t>(q * d) + off >= 0 && wrong(d, q * d + off)) return 1;
    }
    if (wrong(d, (1ull << 31) - 1)) return 1;
  }
  // All numerators of one divisor.
  const FastDiv f = make_fast_div(12);
  for (uint32_t n = 0; n < 1u << 31; ++n)
    if (fast_div(n, f) != n / 12) return wrong(12, n);
  return 0;
}
"""


def test_fast_division_of_the_header(tmp_path) -> None:
    """``make_fast_div`` and ``fast_div`` as they stand in the header, compiled for the host."""

    compiler = shutil.which("g++")
    if compiler is None:
        pytest.skip("no host compiler")
    text = ROWS_HEADER.read_text()
    code = re.search(r"^struct FastDiv \{.*?^__device__ __forceinline__ uint32_t fast_div\([^\n]*\n", text, re.S | re.M)
    assert code, "the header's division"
    source, program = tmp_path / "divide.cpp", tmp_path / "divide"
    source.write_text(_DIVISIONS.replace("@DIVISION@", code.group(0)))
    subprocess.run([compiler, "-O2", "-std=c++17", "-o", str(program), str(source)], check=True, timeout=120)
    done = subprocess.run([str(program)], capture_output=True, text=True, timeout=120)
    assert done.returncode == 0, done.stdout


@pytest.mark.gpu
@pytest.mark.parametrize("group", [None, 128])
@pytest.mark.parametrize("dtype", HALF)
def test_integers_of_every_pair_of_significands(dtype, group) -> None:
    """``rint(x / scale)``, the quotient rounded to fp32, for every largest
    magnitude and every magnitude down to 2^-11 of it: below, all integers are 0.
    A quotient of fp32 numbers in 64 bits rounds to the one in 32."""

    bits = 8 if dtype == torch.bfloat16 else 11
    significands = torch.arange(1 << (bits - 1), 1 << bits, dtype=torch.float64)
    # fp16: up to 32752, so that no magnitude is below the normal range.
    largest = significands * (1.0 if dtype == torch.bfloat16 else 16.0)
    others = (largest[None, :] * 2.0 ** -torch.arange(12.0, dtype=torch.float64)[:, None]).flatten()
    others = others * torch.where(torch.arange(others.numel()) % 2 == 0, 1.0, -1.0)
    run = others.numel() if group is None else group - 1
    parts = torch.nn.functional.pad(others, (0, -others.numel() % run)).view(-1, run)
    x = torch.zeros(len(largest), len(parts), run + 1, dtype=torch.float64)
    x[..., 0] = largest[:, None]
    x[..., 1:] = torch.where(parts[None].abs() <= largest[:, None, None], parts[None], torch.zeros(()))
    x = x.flatten(1).to(dtype)
    assert torch.equal(x.double().abs().amax(1), largest)
    for kept in [da.quantize_int8_hip(x.to(_device()), group)] + ([da.gelu_int8_hip(x.to(_device()))[1]] if group else []):
        scales = kept.scales.cpu()
        assert torch.equal(scales, (largest.float() * torch.tensor(1 / 127.0, dtype=torch.float32))[:, None].expand_as(scales))
        quotients = (x.double() / scales.double().repeat_interleave(x.shape[1] // scales.shape[1], 1)).float()
        assert torch.equal(kept.values.cpu().float(), torch.round(quotients))
