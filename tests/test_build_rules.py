"""A change to a header builds everything that includes it: every object's prerequisites hold what its source includes, directly or not."""
import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def included(path, into):
    """The project's own headers that the file includes, in the end."""
    for name in re.findall(r'^\s*#\s*include\s+"([^"]+)"', open(path).read(), re.M):
        for base in (os.path.dirname(path), os.path.join(ROOT, "include")):
            header = os.path.realpath(os.path.join(base, name))
            if os.path.exists(header):
                if header not in into:
                    into.add(header)
                    included(header, into)
                break
    return into


@pytest.mark.parametrize("folder", ["csrc", "drivers"])
def test_objects_depend_on_the_headers_that_they_include(folder):
    where = os.path.join(ROOT, "cutt_amd", folder)
    # (the rules as make has resolved them; nothing is built)
    rules = subprocess.run(["make", "-pn", "-C", where], capture_output=True, text=True, timeout=120).stdout
    seen = 0
    for target, names in re.findall(r"^([\w-]+\.o):(.*)$", rules, re.M):
        needs = {os.path.realpath(os.path.join(where, n)) for n in names.split()}
        source = [n for n in needs if n.endswith((".cpp", ".hip"))]
        if not source:
            continue
        missing = included(source[0], set()) - needs
        assert not missing, (target, sorted(os.path.relpath(m, ROOT) for m in missing))
        seen += 1
    assert seen == len([n for n in os.listdir(where) if n.endswith((".cpp", ".hip"))])
