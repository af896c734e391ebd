"""What the sources of the paged kernels have to keep to, where no run would show it."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "backburner_b200", "csrc")


@pytest.mark.parametrize("name", ["pa_mask.cuh", "pa_cache.cuh", "pa_decode.cuh", "pa_prefill.cuh", "pa_prefill_pair.cuh"])
def test_paged_kernels_read_their_inputs_with_ordinary_loads(name):
    """The paged kernels start while the stream's earlier kernels run (programmatic launches), so a non-coherent load could
    return what an input held before the kernel that writes it: none, but in an instance that is not paged."""
    with open(os.path.join(CSRC, name)) as f:
        lines = [re.sub(r"//.*", "", line) for line in f]
    for line in lines:
        if re.search(r"__ldg|ld\.global\.nc|__ldcg_nc|__restrict__", line):
            assert re.search(r"PAGED \? \S.* : __ldg", line), line
