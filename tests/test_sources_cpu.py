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


def test_every_load_into_lds_sets_its_own_destination():
    """The destination of a load that goes to LDS is in m0, which the compiler may use between two asm statements: the one
    that loads writes m0 itself."""
    found = 0
    for path in glob.glob(os.path.join(CSRC, "*.hip")) + glob.glob(os.path.join(CSRC, "*.h")):
        for text in re.findall(r"\basm\b(?:\s+volatile)?\s*\(((?:\s*\"[^\"]*\")+)", open(path).read()):
            if re.search(r"_load_lds_|_load_dword\w* [^\"]*\blds\b", text):
                found += 1
                assert "s_mov_b32 m0" in text, (path, text)
    assert found >= 3
