"""Order of two steps that no GPU test may get wrong to show it: a kernel that lets the next one of its
stream start early must have its tensor memory by then. The next one may take all of an SM's tensor
memory and hold it until this grid has ended, which a block that still waits for its own never does."""
import glob
import os
import re

from conftest import PKG_DIR

SOURCES = sorted(glob.glob(os.path.join(PKG_DIR, "csrc", "*.cuh")))


def kernels():
    """(file, body) of each __global__ function of the kernel headers."""
    for path in SOURCES:
        src = re.sub(r"//[^\n]*", "", open(path).read())
        starts = [m.start() for m in re.finditer(r"__global__", src)]
        for a, b in zip(starts, starts[1:] + [len(src)]):
            yield os.path.basename(path), src[a:b]


def test_tensor_memory_is_taken_before_dependents_start():
    both = 0
    for name, body in kernels():
        alloc = [m.end() for m in re.finditer(r"tmem_alloc\w*\(", body)]
        launch = [m.start() for m in re.finditer(r"griddep_launch_dependents\(", body)]
        if alloc and launch:
            both += 1
            assert min(launch) > max(alloc), name
    assert both >= 2  # the offset / mask head, the attention
