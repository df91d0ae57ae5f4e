"""The example that runs beam search, reordering and distillation together."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu


def test_draft_learns_from_the_teachers_beams():
    from zllm_amd.engine import Context
    path = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "examples", "distill_draft.py")
    spec = importlib.util.spec_from_file_location("distill_draft", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    first, last = mod.run(Context())
    assert last < first
