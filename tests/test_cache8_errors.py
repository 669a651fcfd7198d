"""What the 8-bit cache's users are told: the engine's device word, the command line, arguments that no call can take.  No GPU needed."""
from __future__ import annotations

import pytest
import torch

from smoltts_b200._errors import SMOL_ERR_CAPACITY, SMOL_ERR_CUDA, SmolError


class Words:
    """The part of the library that the engine asks for its error word."""

    def __init__(self, at):
        self.at = at

    def smol_lm_error_word(self, handle):
        return self.at


@pytest.mark.parametrize("word,code,text", [(1, SMOL_ERR_CAPACITY, "outside its pools"), (2, SMOL_ERR_CAPACITY, "outside its pools"), (3, SMOL_ERR_CUDA, "ran out")])
def test_the_engine_tells_a_wait_that_ran_out_from_a_bad_page(word, code, text):
    from smoltts_b200.lm import HybridLM

    model = object.__new__(HybridLM)
    model._workspace, model._h = torch.zeros(64, dtype=torch.uint8), None
    model.lib = Words(model._workspace.data_ptr() + 16)
    model.check_device_errors()
    model._workspace[16] = word
    with pytest.raises(SmolError, match=text) as e:
        model.check_device_errors()
    assert e.value.code == code
