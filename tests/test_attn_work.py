"""Which rows and keys the 8-bit cache's attention kernels take of a batch, their
arithmetic run on the host (tests/cpp/test_attn_work.cpp): idle requests first, last
and everywhere come to nothing, and no lane reads Q or masks outside its request."""
import os
import subprocess

CPP = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp")


def test_rows_and_keys_of_a_batch():
    subprocess.run(["make", "-s", "-C", CPP, "test_attn_work"], check=True)
    r = subprocess.run([os.path.join(CPP, "test_attn_work")], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout + r.stderr
    assert "attention's work: 0 failure(s)" in r.stdout
