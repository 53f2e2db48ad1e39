"""CPU: what the build recompiles."""
import glob
import os
import re

from bitcache_b200 import build


def test_every_included_header_makes_objects_stale():
    sources = [f for d in (build.CSRC, build.INCLUDE) for f in glob.glob(os.path.join(d, "*"))]
    known = {os.path.basename(d) for d in build._deps()}
    for path in sources:
        with open(path) as f:
            for name in re.findall(r'^#include "([^"]+)"', f.read(), flags=re.M):
                assert os.path.basename(name) in known, f"{name}, included by {os.path.basename(path)}"
