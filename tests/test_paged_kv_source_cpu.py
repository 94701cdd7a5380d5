"""Properties of the paged-cache kernels' source that no result shows."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "wush_b200", "csrc")


@pytest.mark.parametrize("name", ["paged_kv.cu", "paged_attention.cu", "paged_kv.cuh"])
def test_early_kernels_do_not_load_through_the_read_only_path(name):
    """ld.global.nc is for data that nobody writes while the kernel is there; a kernel launched early is there while the one
    before it writes its inputs, even though its loads come after griddepcontrol.wait."""
    with open(os.path.join(CSRC, name)) as f:
        code = re.sub(r"//[^\n]*", "", f.read())
    assert not re.findall(r"ld_nc_v4|__ldg|ld\.global\.nc|__restrict__", code)


def test_every_early_kernel_waits():
    """A kernel that is launched through EarlyLaunch waits for the one before it, and one of them for each kernel there is."""
    for name, kernels in (("paged_kv.cu", 4), ("paged_attention.cu", 2)):
        with open(os.path.join(CSRC, name)) as f:
            code = re.sub(r"//[^\n]*", "", f.read())
        bodies = re.split(r"__global__", code)[1:]
        assert len(bodies) == kernels
        for body in bodies:
            assert body.count("griddepcontrol.wait") == 1
