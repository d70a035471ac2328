"""The library's HOST logic without a GPU: C++ programs that define the HIP runtime's calls themselves (tests/cpp/hip_stub.h) and link the
built library, so that what it queues, on which stream and behind which event, can be read off in order."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ROCM = "/opt/rocm"

pytestmark = pytest.mark.skipif(not os.path.exists(os.path.join(ROCM, "include", "hip", "hip_runtime_api.h")), reason="needs the HIP headers")


def build_and_run(tmp_path, name):
    import fun_ofdm_amd
    lib = fun_ofdm_amd._lib.library_path()
    exe = str(tmp_path / name)
    # (-rdynamic: the library's undefined runtime symbols bind to the program's)
    subprocess.run(["g++", "-O1", "-g", "-std=c++17", "-Wall", "-Wno-unused-function", "-D__HIP_PLATFORM_AMD__", "-isystem", os.path.join(ROCM, "include"),
                    "-I", os.path.join(ROOT, "include"), os.path.join(ROOT, "tests", "cpp", name + ".cpp"), lib, "-rdynamic", "-Wl,--allow-shlib-undefined",
                    "-Wl,-rpath," + os.path.dirname(lib), "-Wl,-rpath," + os.path.join(ROCM, "lib"), "-lpthread", "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, (r.returncode, r.stdout[-4000:], r.stderr[-2000:])
    return r.stdout


def test_a_call_takes_the_registered_events_with_it_whatever_it_returns(tmp_path):
    assert "all checks passed" in build_and_run(tmp_path, "after_events")


def test_every_stream_has_the_default_priority(tmp_path):
    assert "all checks passed" in build_and_run(tmp_path, "stream_priorities")


def test_a_host_decode_copies_its_inputs_behind_the_frames_being_built(tmp_path):
    assert "all checks passed" in build_and_run(tmp_path, "scratch_order")


def test_a_handles_streams_sit_on_queues_of_their_own_whatever_the_host_made(tmp_path):
    assert "all checks passed" in build_and_run(tmp_path, "stream_order")
