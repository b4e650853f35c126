"""CPU test of the tree mask's addressing (csrc/fa_kvcache.h, compiled for the host): whatever 32 keys a wave of
the attention kernel asks for, no byte outside the mask of its sequence is read."""
import os
import shutil
import subprocess

import pytest

from conftest import PKG

HOST = r"""
#include "fa_kvcache.h"
#include <cstdio>
#include <initializer_list>
#define CHECK(x) do { if (!(x)) { std::printf("line %d: %s\n", __LINE__, #x); return 1; } } while (0)
int main() {
  const int outside = 0x7ffffff0;
  for (int sq : {1, 2, 13, 64, 4096})
    for (int row : {0, sq, sq + 3, 4 * sq}) {      // 0: one row for all; the last: a slice of a wider mask
      const int bytes = fa::mask_bytes(sq, row);
      CHECK(bytes == (sq - 1) * row + sq);         // up to the last row's last byte, and none behind it
      for (int len = 0; len < 160; ++len) {
        const int total = len + sq;
        for (int t : {0, sq / 2, sq - 1})
          // a step is 128 keys; its waves ask for keys up to its end, behind the last one too
          for (int j = len / 128 * 128; j < (total + 127) / 128 * 128; ++j) {
            const int at = fa::mask_offset(t, j, len, total, row, outside);
            if (j >= len && j < total) CHECK(at == t * row + j - len && at >= 0 && at < bytes);
            else CHECK(at == outside);
          }
      }
    }
  std::puts("ok");
  return 0;
}
"""


def test_mask_addressing_on_the_host(tmp_path):
    hipcc = "/opt/rocm/bin/hipcc"
    if shutil.which(hipcc) is None:
        pytest.skip("no hipcc")
    src, exe = tmp_path / "host.cpp", tmp_path / "host"
    src.write_text(HOST)
    subprocess.run([hipcc, "-x", "hip", "--cuda-host-only", "-std=c++17", "-I", os.path.join(PKG, "csrc"), str(src), "-o",
                    str(exe)], check=True, capture_output=True, text=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout


def test_the_kernel_reads_the_mask_within_its_bytes():
    """The kernel's descriptor has the mask's bytes as its size, and its offsets come from the function above."""
    with open(os.path.join(PKG, "csrc", "fa_kvcache.hip")) as f:
        text = f.read()
    assert "p.mask != nullptr ? mask_bytes(p.sq, (int)p.mask_row) : 0" in text
    loads = [line for line in text.splitlines() if "raw_buffer_load_b8" in line]
    assert len(loads) == 1 and "rmask, mask_offset(t, j, len, total," in loads[0]
