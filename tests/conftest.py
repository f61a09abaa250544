"""pytest configuration: the `gpu` marker and the repository root on sys.path."""
import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a ROCm GPU (MI355X) and the built HIP library")
    # registers the torch.ops.pragnosia namespace for every test module, whichever subset runs (the library itself
    # loads on the first call)
    import pragnosia_amd.ops  # noqa: F401


# Tests whose expected value is wrong: a distillation loss whose list repeats a word is tau^2 KL(p || q) with the word's
# probability the sum of its entries', and these expect sum_k p_k log p_k over the entries instead (for student logits
# 3, 0, 0, 0 and the first word twice -0.554, a negative divergence, where it is 0.139).
# tests/test_gpu_distill_repeats.py checks the same calls against the words' probabilities.
WRONG_VALUE = ("test_gpu_head.py::test_teacher_edges", "test_gpu_lm_ends.py::test_training_step[True-aspin]",
               "test_gpu_lm_ends.py::test_training_step[True-dspin]")


def pytest_collection_modifyitems(items):
    for item in items:
        if item.nodeid.split("/")[-1] in WRONG_VALUE:
            item.add_marker(pytest.mark.xfail(reason="expects the entropy of a repeated word's entries, not the word's",
                                              raises=AssertionError, strict=True))
