"""set_prefill_bits where memory or a launch fails: the model stays as it was, nothing stays
allocated and no error waits for the next launch.  A host program over a stub runtime."""
import os
import subprocess

import pytest

from conftest import ROOT

HIPCC = "/opt/rocm/bin/hipcc"


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="no hipcc")
def test_failures_leave_the_model_as_it_was(tmp_path):
    exe = str(tmp_path / "prefill_bits_alloc")
    # the calls that the stub leaves out are never reached
    subprocess.run([HIPCC, "-x", "hip", "--offload-host-only", "-std=c++17", "-O1", "-w",
                    "-I" + os.path.join(ROOT, "include"),
                    os.path.join(ROOT, "tests", "cxx", "prefill_bits_alloc.cpp"), "-no-hip-rt",
                    "-Wl,--unresolved-symbols=ignore-all", "-o", exe], check=True)
    run = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert run.stdout.strip() == "ok", run
