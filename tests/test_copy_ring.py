"""CPU tier: the bookkeeping of a warp's ring of asynchronous copies (csrc/copy_ring.h).

A block whose copies have not all landed may not end: they would write into the shared memory of the next one. After a
wait that gave up, the ring says which copies are still in flight, a full ring included. No GPU run reaches that path, so
tests/cpp/copy_ring_check.cpp gives up at every wait in turn against simulated barriers."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_every_copy_in_flight_is_drained(tmp_path):
    exe = str(tmp_path / "copy_ring_check")
    subprocess.run(["g++", "-std=c++17", "-O2", os.path.join(ROOT, "tests", "cpp", "copy_ring_check.cpp"),
                    "-I", os.path.join(ROOT, "matrixflash_pro_b200", "csrc"), "-o", exe], check=True)
    out = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stdout + out.stderr
    assert " 0 failure(s)" in out.stdout
