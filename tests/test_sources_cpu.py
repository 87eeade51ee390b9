"""What the compiler does not check across translation units."""
import collections
import glob
import os
import re

from helpers import ROOT

CSRC = os.path.join(ROOT, "yolo_amd", "csrc")


def test_one_definition_of_every_type():
    """All units share the namespace yolo_amd: two types of one name would be one to the linker."""
    where = collections.defaultdict(set)
    for path in glob.glob(os.path.join(CSRC, "*.hip")) + glob.glob(os.path.join(CSRC, "*.cpp")) + glob.glob(os.path.join(CSRC, "*.h")):
        for name in re.findall(r"^(?:struct|class|union|enum)\s+(\w+)\s*(?::[^;{]*)?\{", open(path).read(), re.M):
            where[name].add(os.path.basename(path))
    assert len(where) > 20
    assert {n: sorted(f) for n, f in where.items() if len(f) > 1} == {}
