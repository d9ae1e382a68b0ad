"""What the packed-prompt calls promise beside their formulas, as far as it shows without a GPU."""
from __future__ import annotations

import os
import re

import pytest

from conftest import ROOT


def source(name: str) -> str:
    with open(os.path.join(ROOT, "rustllm_b200", "csrc", name)) as f:
        return re.sub(r"//[^\n]*", "", f.read())


@pytest.mark.parametrize("name,first,last", [
    ("prompt_linear.cu", "    if (warp == 0) {\n        if (lane == 0) {", "    __syncwarp();\n    if (SPLIT > 1) {"),
    ("prompt_attention.cu", "setmaxnreg.inc", "tcgen05.dealloc")])
def test_roles_of_a_cta_meet_at_no_barrier_without_a_limit(name, first, last):
    """A warp that gave up a wait leaves its loop by itself: a barrier inside the loops would keep
    the other warps for good.  They meet once, behind their loops."""
    text = source(name)
    lo, hi = text.index(first), text.index(last)
    assert lo < hi
    meets = re.findall(r"named_barrier|__syncthreads|bar\.sync|barrier\.cta|cluster_sync_all",
                       text[lo:hi])
    assert meets == (["__syncthreads"] if last == "tcgen05.dealloc" else [])
