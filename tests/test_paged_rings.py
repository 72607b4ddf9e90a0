"""The rings of the two-halved attention kernel, walked on the host; no GPU."""
import shutil
import subprocess
from pathlib import Path


def test_no_half_waits_for_a_fill_it_may_mistake(tmp_path):
    """Random items through rings of two and five slots: before a half waits for a block's values, it knows that the slot's fill before
    has landed."""
    source = Path(__file__).with_name("ring_check.cpp")
    program = tmp_path / "ring_check"
    subprocess.run([shutil.which("g++") or "g++", "-O1", "-std=c++17", "-o", str(program), str(source)], check=True)
    out = subprocess.run([str(program)], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and out.stdout.startswith("ok"), out.stdout
    assert int(out.stdout.split()[1]) > 10000
