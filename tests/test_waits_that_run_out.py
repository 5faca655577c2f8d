"""Kernels that load ahead by bulk copies, by their source: a wait that has run out ends the loading, and what is on its way is waited for once more before the CTA
ends (a copy that outlives its CTA lands in another one's shared memory).  No test makes a copy fail to arrive on a GPU."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.abspath(__file__)), '..', 'flash-linear-attention_b200', 'csrc')


@pytest.mark.parametrize('name,load,still,last', [('gated_recurrence.cu', 'tiles.load(', 'patience.ok()', 'tiles.land('), ('rms_norms.cu', 'fill<T>(', 'ring.ok()', 'ring.finish()')])
def test_copies_on_their_way_are_waited_for(name, load, still, last):
    with open(os.path.join(CSRC, name)) as f:
        text = re.sub(r'//[^\n]*', '', f.read())
    kernels = [body for body in text.split('__global__')[1:] if load in body]
    assert len(kernels) == 2   # forward and backward
    for body in kernels:
        loads = [m.start() for m in re.finditer(re.escape(load), body)]
        assert last in body[loads[-1]:]
        loop = body.index('for (int i = 0; i < n;') if name.startswith('gated') else body.index('for (int turn = 0;')
        for at in loads:   # those of the loop (of the lambdas that it calls) ask whether a wait has run out
            if at > loop or 'i + STAGES' in body[at:at + 200]:
                assert still in body[max(0, at - 200):at], body[at - 200:at + 80]
