"""Device arrays of a pool's batches (host code, with a stand-in for the device allocator):
what a captured launch reads is neither freed nor mixed with a later batch's arrays when an
upload outgrows it."""
import os
import shutil
import subprocess

import pytest

from nitrorag_amd import _native as N

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIP_INCLUDE = "/opt/rocm/include"


def test_outgrown_batch_arrays_are_kept(tmp_path):
    if shutil.which("g++") is None or not os.path.isdir(HIP_INCLUDE):
        pytest.skip("needs g++ and HIP's headers")
    exe = str(tmp_path / "driver")
    r = subprocess.run(["g++", "-std=c++17", "-O1", "-D__HIP_PLATFORM_AMD__", f"-I{HIP_INCLUDE}",
                        f"-I{ROOT}/nitrorag_amd/csrc", f"{ROOT}/tests/host_driver_batch_arrays.cpp", "-o", exe],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr


def test_reserve_batches_refuses_a_null_pool():
    assert N.lib().nitro_kvpool_reserve_batches(None, 1, 1, 1) == N.INVALID_ARGUMENT
