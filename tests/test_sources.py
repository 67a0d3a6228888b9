"""Every source file in leaf_amd/csrc is built or included."""
from __future__ import annotations

import re

from leaf_amd import build

# executables of their own (leaf_amd/build.py)
PROGRAMS = {"main_decoder.cpp", "hbm_copy.hip", "mfma_peak.hip"}


def test_no_source_is_left_out():
    files = {p.name for p in build.CSRC.iterdir() if p.suffix in (".hip", ".cpp", ".h")}
    built = set(build.SOURCES) | PROGRAMS
    included = {name for p in build.CSRC.iterdir() if p.name in files for name in re.findall(r'^#include "([^"/]+)"', p.read_text(), re.M)}
    assert built <= files and files <= built | included
