"""The plans of the 4-bit attention: the planner under sanitizers with random problems (tests/host_fuzz/q4_plan_fuzz.cpp), and its rules from the
outside.  CPU only."""
import os
import shutil
import subprocess

import pytest

from inference_lib_amd import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("seed", [1, 2])
def test_planner_and_validator_under_sanitizers(tmp_path, seed):
    if shutil.which("g++") is None:
        pytest.skip("no g++")
    exe = str(tmp_path / "q4_plan_fuzz")
    cmd = ["g++", "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined", "-fno-sanitize-recover=undefined", "-static-libasan",
           "-I", os.path.join(ROOT, "include"), os.path.join(ROOT, "tests", "host_fuzz", "q4_plan_fuzz.cpp"),
           os.path.join(ROOT, "inference_lib_amd", "csrc", "hogwild_plan.cpp"), "-o", exe]
    subprocess.run(cmd, check=True)
    env = dict(os.environ, ASAN_OPTIONS="detect_leaks=1:abort_on_error=0", UBSAN_OPTIONS="print_stacktrace=1")
    r = subprocess.run([exe, "4000", str(seed)], capture_output=True, text=True, env=env, timeout=300)
    assert r.returncode == 0, r.stdout[-3000:] + r.stderr[-3000:]
    assert " 0 failures" in r.stdout


@pytest.mark.parametrize("D,gq,row_blocks,tiles", [(64, 4, 1, 24), (64, 20, 2, 20), (128, 5, 1, 20), (128, 24, 2, 12), (256, 2, 1, 12), (256, 24, 1, 12)])
def test_short_tables_are_one_workgroup_s(D, gq, row_blocks, tiles):
    def plan(n):
        return _lib.paged_plan(W=4, S=1, Hq=2 * gq, Hkv=2, Ev=D, block_size=32, max_blocks=n, num_cus=256, q4=True)

    for n in range(1, tiles + 1):
        assert plan(n).splits == 1 and plan(n).row_blocks == row_blocks
    assert plan(tiles + 1).splits > 1


@pytest.mark.parametrize("W", [1, 3, 64, 500])
@pytest.mark.parametrize("S,gq", [(1, 1), (1, 5), (4, 8), (33, 1), (7, 5), (16, 1), (17, 1)])
def test_fixed_plans_have_a_workgroup_for_every_row(W, S, gq):
    for D in (64, 128, 256):
        pl = _lib.paged_plan(W=W, S=S, Hq=8 * gq, Hkv=8, Ev=D, block_size=16, max_blocks=300, num_cus=256, q4=True)
        each = 16 * pl.row_blocks
        assert pl.row_groups == W * -(-S * gq // each) and pl.workgroups == 8 * pl.row_groups * pl.splits
