"""The Makefile's dependencies: an object is built anew when any header that its source includes has changed."""
import os
import re
import shutil
import subprocess

import pytest

import fhtest

PKG = os.path.join(fhtest.ROOT, "flyhigh-engine_amd")
DIRS = (os.path.join(PKG, "csrc"), os.path.join(fhtest.ROOT, "include"))


def headers(path, seen):
    """The project's headers that a file includes, and theirs."""
    with open(path) as f:
        for name in re.findall(r'^\s*#\s*include\s+"([^"]+)"', f.read(), re.M):
            for d in DIRS:
                at = os.path.join(d, name)
                if os.path.exists(at) and at not in seen:
                    seen.add(at)
                    headers(at, seen)
    return seen


@pytest.mark.skipif(shutil.which("make") is None, reason="no make")
def test_objects_depend_on_the_headers_they_include():
    out = subprocess.run(["make", "-pn", "-C", PKG], capture_output=True, text=True).stdout
    rules = {}
    for target, needs in re.findall(r"^([^\s%]+\.o):(?!=) *(.*)$", out, re.M):
        rules.setdefault(os.path.normpath(target), set()).update(os.path.normpath(n) for n in needs.split())
    lost, sources = [], 0
    for target, needs in rules.items():
        for src in (n for n in needs if n.endswith((".hip", ".cpp"))):
            sources += 1
            lost += [f"{os.path.basename(target)}: {os.path.basename(h)}"
                     for h in sorted(headers(src, set())) if h not in needs]
    assert sources >= 15 and not lost, lost
