"""pa_rope_norm_and_cache in place: with the input's own stride, or not at all."""
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
  alignas(16) static char a[16], b[16], c[16], d[16], e[16];
  auto code = [](void *qo, void *ko, void *q, void *k, void *v, int64_t n, int64_t qs, int64_t qos, int64_t ks, int64_t kos) {
    return pa::check_rotate_in_place(qo, ko, q, k, v, n, qs, qos, ks, kos).code;
  };
  bool ok = true;
  // apart, in place with one stride, one token, no keys kept, no values
  for (int got : {code(d, e, a, b, c, 9, 768, 512, 768, 256), code(a, b, a, b, c, 9, 768, 768, 768, 768),
                  code(a, b, a, b, c, 1, 768, 512, 768, 256), code(a, nullptr, a, b, c, 9, 768, 768, 768, 0),
                  code(a, b, a, b, nullptr, 9, 512, 512, 256, 256), code(d, nullptr, a, b, nullptr, 9, 768, 512, 768, 0)})
    ok = ok && got == PA_OK;
  // another stride; another tensor's place
  for (int got : {code(a, e, a, b, c, 9, 768, 512, 768, 256), code(d, b, a, b, c, 9, 768, 512, 768, 256),
                  code(b, e, a, b, c, 9, 768, 768, 768, 768), code(c, e, a, b, c, 9, 768, 768, 768, 768),
                  code(d, d, a, b, c, 9, 768, 768, 768, 768), code(d, a, a, b, c, 9, 768, 768, 768, 768),
                  code(d, c, a, b, c, 9, 768, 768, 768, 768)})
    ok = ok && got == PA_ERR_INVALID_ARG;
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
def test_entry_refuses_another_stride_and_writes_nothing(cuda_device):
    """The parts of one projection's output rotated in place: the output's stride left to its default, which
    is that of a tensor of its own."""
    from test_gpu_prompt_path import Rotate
    r = Rotate(700, 8, 2, 96, 40, seed=9, write=False)
    before = r.qkv.clone()

    def call(**strides):
        r.cache.rope_norm_and_cache(r.plan, r.q, r.k, r.q, r.k, None, r.qw, r.kw, 1e-6, r.positions, None, r.t, r.hq,
                                    q_stride=r.row, k_stride=r.row, **strides)
    for strides in (dict(), dict(q_out_stride=r.row), dict(k_out_stride=r.row)):
        with pytest.raises(pa.PagedAttnError) as e:
            call(**strides)
        assert e.value.status == 1 and "in place" in str(e.value)
    torch.cuda.synchronize()
    assert torch.equal(before, r.qkv)
    r.run()
    torch.cuda.synchronize()
    call(q_out_stride=r.row, k_out_stride=r.row)
    torch.cuda.synchronize()
    assert torch.equal(r.q, r.q_out[:-1]) and torch.equal(r.k, r.k_out[:-1])
