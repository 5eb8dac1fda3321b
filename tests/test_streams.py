"""The library's streams all have the default priority: work on streams of
different priorities can block for good.  CPU only: the sources are read."""
import glob
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "java-reed-solomon-distributed-file-system_amd", "csrc")
TOOLS = os.path.join(ROOT, "tools")


def test_no_build_makes_a_stream_with_a_priority():
    files = [f for d in (CSRC, TOOLS) for e in ("*.cpp", "*.hpp", "*.hip", "*.py") for f in glob.glob(os.path.join(d, e))]
    assert any(f.endswith("host.cpp") for f in files)
    prioritised = re.compile(r"StreamCreateWithPriority|Stream\([^)]*priority\s*=|is_high_priority_stream\s*=\s*True")
    for f in files:
        with open(f) as h:
            assert not prioritised.search(h.read()), os.path.basename(f)
