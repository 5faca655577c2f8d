"""The example that runs norm, mixer, head, log probabilities and distillation together."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu


def test_a_student_learns_from_a_teacher():
    path = os.path.join(os.path.dirname(__file__), '..', 'examples', 'distill_student.py')
    spec = importlib.util.spec_from_file_location('distill_student', path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    losses, scores = example.main(steps=25, vocab=3001, length=128)
    assert losses[-1] < 0.7 * losses[0] and all(x == x for x in losses)
    assert scores.top_ids.shape == (4, 127, 5) and (scores.logprobs <= 0).all() and (scores.entropy >= 0).all()
    assert (scores.top_logprobs.diff(dim=-1) <= 0).all()
