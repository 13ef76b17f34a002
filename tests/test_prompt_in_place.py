"""pa_prompt_attention with its output in an input's place is refused: rows that have to be recomputed
would read what has been written there."""
import os
import shutil
import subprocess

import pytest
import torch

import paged_attn_b200 as pa

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SOURCE = """
#include "mlx-node_b200/csrc/prompt_host.hpp"
int main() {
  alignas(16) static char a[16], b[16], c[16], d[16];
  using pa::check_prompt_in_place;
  bool ok = !check_prompt_in_place(a, b, c, d) && !check_prompt_in_place(a, b, nullptr, nullptr) &&
            !check_prompt_in_place(a, b, c, c) && !check_prompt_in_place(nullptr, nullptr, nullptr, nullptr);
  for (auto e : {check_prompt_in_place(a, a, c, d), check_prompt_in_place(a, b, a, d), check_prompt_in_place(a, b, c, a)})
    ok = ok && e.code == PA_ERR_INVALID_ARG;
  return ok ? 0 : 1;
}
"""


def test_check_on_the_host(tmp_path):
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("no C++ compiler")
    src, exe = tmp_path / "in_place.cpp", str(tmp_path / "in_place")
    src.write_text(SOURCE)
    subprocess.run([cxx, "-std=c++17", "-Wall", "-Wextra", "-Werror", "-I", ROOT, str(src), "-o", exe], check=True)
    assert subprocess.run([exe]).returncode == 0


@pytest.mark.gpu
def test_entry_refuses_and_writes_nothing(cuda_device):
    from test_gpu_prompt_path import Attend
    r = Attend([40, 9], [40, 9], 4, 2, 64, seed=1)
    before = r.q.clone()
    with pytest.raises(pa.PagedAttnError) as e:
        r.run(out=r.q)
    assert e.value.status == 1 and "out may not" in str(e.value)
    torch.cuda.synchronize()
    assert torch.equal(before, r.q)
    r.run()
    r.check()
