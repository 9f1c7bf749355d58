"""The paged attention's index arithmetic on the CPU: the functions of csrc/attend.cuh that say which heads an item reads,
compiled for the host and run over every split of the heads. (A read past a tensor's end usually finds memory of the same
allocator, and its value is dropped: no comparison of outputs shows it.)"""
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "basal_b200", "csrc")


def host_program(tmp_path, body):
    """Compiles a main() around body with attend.cuh and runs it; body prints a line for each finding."""
    nvcc = shutil.which(os.environ.get("NVCC", "nvcc"))
    if not nvcc:
        pytest.skip("no nvcc")
    src = tmp_path / "index.cu"
    src.write_text('#include <cstdio>\n#include <cuda_bf16.h>\n#include <type_traits>\n#include "common.cuh"\n#include '
                   '"attend.cuh"\nusing namespace b200::paged;\nint main() {\n' + body + '\n  return 0;\n}\n')
    exe = str(tmp_path / "index")
    subprocess.run([nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-O1", "-std=c++17", "--expt-relaxed-constexpr",
                    "-I", CSRC, "-o", exe, str(src)], check=True, capture_output=True)
    return subprocess.run([exe], check=True, capture_output=True, text=True).stdout


def test_every_head_that_an_item_reads_exists(tmp_path):
    """Items of 8 NG heads over 1 to 80 heads a key head: each lane row reads a head of the item's own, whether its head
    exists or not (17 to 24 heads leave the last item with no second eight heads)."""
    assert host_program(tmp_path, """
  for (int ng = 1; ng <= 2; ++ng)
    for (int G = 1; G <= 80; ++G)
      for (int kvh = 0; kvh < 3; ++kvh)
        for (int h0 = 0; h0 < G; h0 += 8 * ng) {
          const int heads = G - h0 < 8 * ng ? G - h0 : 8 * ng, head0 = kvh * G + h0;
          for (int g = 0; g < ng; ++g)
            for (int r = 0; r < 8; ++r) {
              const int h = query_head(head0, heads, g, r);
              if (h < head0 || h >= head0 + heads || (g * 8 + r < heads && h != head0 + g * 8 + r))
                printf("%d heads a key head, NG %d: lane row %d of eight %d reads head %d of %d .. %d\\n", G, ng, r, g, h,
                       head0, head0 + heads - 1);
            }
        }""") == ""


def test_a_wait_that_gave_up_leaves_no_row_as_it_was_allocated(tmp_path):
    """refuse_rows, a warp's 32 lanes one after another: NaN in every value of an output and in every part's maximum, and
    nothing past them. (A wait gives up only when a caller changes the lengths during the call.)"""
    assert host_program(tmp_path, """
  static uint32_t out[1000];
  static float m[100];
  for (int parts : {0, 1, 33, 99})
    for (int pairs : {0, 1, 31, 64, 999}) {
      for (auto& x : out) x = 7;
      for (auto& x : m) x = 7.0f;
      for (int lane = 0; lane < 32; ++lane) refuse_rows(out, pairs, 0x7FFF7FFFu, m, parts, lane, 32);
      for (int i = 0; i < 1000; ++i)
        if (out[i] != (i < pairs ? 0x7FFF7FFFu : 7u)) printf("pair %d of %d\\n", i, pairs);
      for (int i = 0; i < 100; ++i)
        if (i < parts ? m[i] == m[i] : m[i] != 7.0f) printf("part %d of %d\\n", i, parts);
    }""") == ""
