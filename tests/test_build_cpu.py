"""csrc/build.sh knows when a built file no longer fits: its sources, its flags, the torch it was compiled against."""
import os
import shutil
import subprocess
import time

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture
def tree(tmp_path):
    """the sources with stand-ins for everything built from them, up to date"""
    src = os.path.join(ROOT, "scpair_amd", "csrc")
    if not os.path.exists(os.path.join(src, "build", "torch")):
        pytest.skip("the library was built elsewhere: its stamps are not here")
    csrc = tmp_path / "scpair_amd" / "csrc"
    csrc.mkdir(parents=True)
    for f in os.listdir(src):
        if f.endswith((".hip", ".h", ".cpp", ".sh")):
            shutil.copy(os.path.join(src, f), csrc)
    shutil.copytree(os.path.join(ROOT, "include"), tmp_path / "include")
    first = stale(tmp_path)
    assert "_trunk.so" in first and "linear8.o" in first                  # nothing is built yet
    later = time.time() + 10
    for name in first:
        f = tmp_path / "scpair_amd" / name if name.endswith(".so") else csrc / "build" / name
        f.write_text("")
        os.utime(f, (later, later))
    for stamp in ("flags", "torch"):
        shutil.copy(os.path.join(src, "build", stamp), csrc / "build")
    return tmp_path


def stale(tree, **extra):
    out = subprocess.run(["bash", str(tree / "scpair_amd" / "csrc" / "build.sh"), "--stale"], capture_output=True, text=True,
                         env={**os.environ, **extra})
    assert out.returncode == 0, out.stderr
    return out.stdout.split()


def test_up_to_date_and_older_than_a_source(tree):
    assert stale(tree) == []
    f = tree / "scpair_amd" / "csrc" / "tiles.hip"
    os.utime(f, (time.time() + 20,) * 2)
    assert stale(tree) == ["tiles.o"]


def test_another_torch_or_other_flags(tree):
    (tree / "scpair_amd" / "csrc" / "build" / "torch").write_text("/usr/lib/torch 2.9.0 /usr/include/python3.10\n")
    assert stale(tree) == ["_trunk.so"]
    assert "linear8.o" in stale(tree, EXTRA_FLAGS="-g")
