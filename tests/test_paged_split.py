"""The rule by which the attention over the multi-sequence cache is split, on the host
alone (hymt2sharp_amd/csrc/paged_split.hpp, tests/c/paged_split.cpp): at every size that
the entry points accept."""
import os
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


def test_sizes(tmp_path):
    cxx = shutil.which("g++")
    if not cxx or os.environ.get("HYMT_SANITIZED_CHILD") == "1":
        pytest.skip("no g++, or the preloaded sanitizer would reach it")
    exe = tmp_path / "paged_split"
    subprocess.run([cxx, "-std=c++17", "-O1", "-Wall", "-Werror", "-o", str(exe),
                    os.path.join(HERE, "c", "paged_split.cpp")], check=True)
    r = subprocess.run([str(exe)], stdout=subprocess.PIPE, text=True)
    assert r.returncode == 0, r.stdout[-2000:]
