"""CPU: kernels that may start while their predecessor drains read what it may have written through L2 (wait_predecessor in
kv8.cuh): no load of the KV caches' kernels may be answered by lines that this SM's L1 has from before."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "-1.7-atlas---apollo_b200", "csrc")
FILES = sorted(os.path.basename(f) for n in ("paged*", "kv8*") for f in glob.glob(os.path.join(CSRC, n)))


@pytest.mark.parametrize("name", FILES)
def test_no_load_may_use_l1(name):
    text = re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, name)).read())
    assert not re.findall(r"__ld(?:cs|g|lu|ca)\(", text)
    assert not re.findall(r"\bld\.global(?!\.cg)[.\w]*", text)
    # the pages' counts and the table by plain subscripts: only written
    assert not re.findall(r"[=(,<>+\-*?:]\s*\w*\.?c?a?\.?(?:refs|table)\[[^\]]*\](?!\s*=[^=])", text)
