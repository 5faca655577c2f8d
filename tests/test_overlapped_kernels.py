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


def overlapped():
    names = [os.path.basename(p) for p in sorted(glob.glob(os.path.join(CSRC, '*.cu')))]
    return [n for n in names if 'wait_for_predecessor();' in source(n)]


@pytest.mark.parametrize('name', overlapped())
def test_what_the_kernel_ahead_writes_is_not_read_by_the_non_coherent_path(name):
    assert not NOT_COHERENT.findall(source(name))


def test_the_sources_are_found():
    assert {'linear.cu', 'scan_bwd.cu', 'rms_norms.cu'} <= set(overlapped())
    for header in glob.glob(os.path.join(CSRC, '*.cuh')):   # what they include
        assert not NOT_COHERENT.findall(source(os.path.basename(header))), header


@pytest.mark.parametrize('name', overlapped())
def test_no_tensor_memory_is_held_while_the_kernel_ahead_is_waited_for(name):
    """That kernel releases its successor's launch before it allocates its own: on one SM each would wait for the other, without an end."""
    for body in source(name).split('__global__')[1:]:
        wait, alloc = body.find('wait_for_predecessor();'), re.search(r'tmem_alloc\(', body)
        assert wait < 0 or alloc is None or wait < alloc.start(), body[:200]
