"""Kernels that begin while the kernel ahead of them finishes (those that call wait_for_predecessor), by their source: what they may not do before
or in spite of that wait shows in no result until the timing is bad."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.abspath(__file__)), '..', 'flash-linear-attention_b200', 'csrc')


def source(name):
    with open(os.path.join(CSRC, name)) as f:
        return re.sub(r'//[^\n]*|/\*.*?\*/', '', f.read(), flags=re.S)


# The non-coherent path (__ldg, ld.global.nc, what the compiler makes of a const __restrict__ pointer) is for memory that nothing writes while the
# kernel runs; such a kernel runs from before its predecessor's last write on.
NOT_COHERENT = re.compile(r'__ldg\b|\bld\.global(\.\w+)*\.nc\b|__restrict__')


@pytest.mark.parametrize('name', ['linear.cu'])
def test_what_the_kernel_ahead_writes_is_not_read_by_the_non_coherent_path(name):
    text = source(name)
    assert 'wait_for_predecessor();' in text and not NOT_COHERENT.findall(text)
