"""CPU: the library's build rules.  Nothing is compiled: make only says what it would run."""
import os
import re
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "quantization_amd", "csrc")


@pytest.mark.skipif(shutil.which("make") is None, reason="no make")
def test_a_change_of_the_flags_rebuilds_every_object():
    """The compiler's flags are part of the arithmetic contract: a tree that holds objects of other flags must not link them."""
    out = subprocess.run(["make", "-n", "-W", "Makefile", "libmq.so"], cwd=CSRC, capture_output=True, text=True, check=True).stdout
    link = next(line for line in out.splitlines() if "-shared" in line)
    objects = re.findall(r"\S+\.o\b", link)
    built = set(re.findall(r" -c \S+ -o (\S+\.o)", out))
    assert len(objects) > 20
    assert not [o for o in objects if o not in built]
