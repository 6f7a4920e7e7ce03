"""CPU test: kernels that start before the one in front of them has ended do not read what it writes by the read-only path, which asks that the
data be unchanged for the whole of the reading kernel's life."""
import os
import re

import pytest

from conftest import PKG_DIR

READ_ONLY = re.compile(r"__ldg\s*\(|ld\.global(\.\w+)*\.nc|__restrict__")


def code(name):
    with open(os.path.join(PKG_DIR, "csrc", name)) as f:
        return re.sub(r"//[^\n]*", "", f.read())


@pytest.mark.parametrize("name", ["gg_moe.cuh", "gg_norm.cuh", "gg_i8.cuh", "gg_permute.cuh", "gg_route.cuh"])
def test_no_read_only_loads(name):
    assert not READ_ONLY.search(code(name))


def test_4_bit_products_read_only_their_weights_scales_so():
    """Scales and zeros, which no kernel of the library writes."""
    source = code("gg_w4.cuh")
    queue = re.search(r"struct W4Queue \{.*?\n\};", source, re.S)
    assert queue and READ_ONLY.search(queue.group())
    assert not READ_ONLY.search(source.replace(queue.group(), ""))
