"""CPU tests of the prompt-path entry points (rotation + cache write, cache read-back, packed
prompt attention): refusals, rotation plans, and the host-only header through a small C++
program."""
import ctypes as C
import math
import os
import shutil
import subprocess

import numpy as np
import pytest

import paged_attn_b200 as pa

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_partition_table_and_argument_checks(tmp_path):
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("no C++ compiler")
    exe = str(tmp_path / "prompt_host_check")
    subprocess.run([cxx, "-std=c++17", "-O1", "-Wall", "-Wextra", "-Werror", "-fsanitize=undefined",
                    "-fno-sanitize-recover", os.path.join(ROOT, "tests", "prompt_host_check.cpp"), "-o", exe],
                   check=True)
    r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr
    assert r.stdout.strip() == "ok"


def test_null_handles_are_refused():
    lib = pa.load_library()
    assert lib.pa_rope_create(None, C.byref(C.c_void_p())) == 1
    assert lib.pa_rope_create(C.byref(pa.PaRopeConfig()), None) == 1
    assert lib.pa_rope_free(None) == 0
    assert lib.pa_rope_frequencies(None, None, None) == 1
    assert lib.pa_prompt_workspace_bytes(None) == 0
    assert lib.pa_rope_norm_and_cache(None, 0, None, None, None, None, None, None, None, None, 0.0, None, None,
                                      1, 1, 1, 1, 1, 1, 1, None) == 1
    assert lib.pa_gather_cache(None, 0, None, None, None, None, None, 1, 1, 1, 1, None) == 1
    assert lib.pa_prompt_attention(None, None, None, None, None, None, None, 1, 1, 1, 1, 1, 1, 1.0, 1.0, None, 0,
                                   None) == 1
    assert pa.last_error() == "cache is null"


@pytest.mark.parametrize("kw", [dict(rope_dims=7), dict(rope_dims=0), dict(rope_dims=300), dict(base=0.0),
                                dict(base=math.inf), dict(scaling="linear", factor=0.0),
                                dict(scaling="bands", factor=2.0), dict(scaling="yarn", factor=2.0),
                                dict(attention_factor=-1.0)])
def test_plan_refusals(kw):
    args = dict(rope_dims=64, base=1e4) | kw
    with pytest.raises(pa.PagedAttnError):
        pa.RopePlan(args.pop("rope_dims"), args.pop("base"), **args)


def test_plan_rejects_an_unknown_scaling():
    with pytest.raises(ValueError):
        pa.RopePlan(64, 1e4, scaling="cubic")


def test_plan_frequencies():
    i = np.arange(32)
    f = 1e4 ** (-i / 32)
    got, gain = pa.RopePlan(64, 1e4).frequencies()
    np.testing.assert_allclose(got, f, rtol=1e-14)
    assert gain == 1.0
    got, gain = pa.RopePlan(64, 1e4, scaling="linear", factor=4.0, attention_factor=0.5).frequencies()
    np.testing.assert_allclose(got, f / 4, rtol=1e-14)
    assert gain == 0.5
    # bands: pairs of under one turn over 2048 positions slowed down, of over four turns kept
    got, gain = pa.RopePlan(64, 1e4, scaling="bands", factor=8.0, original_max_position=2048).frequencies()
    turns = 2048 * f / (2 * math.pi)
    got = np.array(got)
    np.testing.assert_allclose(got[turns > 4], f[turns > 4], rtol=1e-14)
    np.testing.assert_allclose(got[turns < 1], f[turns < 1] / 8, rtol=1e-14)
    mid = (turns > 1) & (turns < 4)
    assert mid.any() and ((got[mid] < f[mid]) & (got[mid] > f[mid] / 8)).all() and gain == 1.0
    # yarn: the first pairs kept, the last slowed down, monotone in between
    got, gain = pa.RopePlan(64, 1e4, scaling="yarn", factor=16.0, original_max_position=4096).frequencies()
    ratio = np.array(got) / f
    assert ratio[0] == 1.0 and abs(ratio[-1] - 1 / 16) < 1e-12 and (np.diff(ratio) <= 1e-15).all()
    assert abs(gain - (0.1 * math.log(16.0) + 1)) < 1e-6
