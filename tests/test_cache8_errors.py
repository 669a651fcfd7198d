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


class Plain:
    """An engine that knows no 8-bit cache."""

    def __init__(self, config, dtype=None, max_tokens=0, max_seqs=0):
        pass


class Coded:
    def __init__(self, config, dtype=None, max_tokens=0, max_seqs=0, kv_bits=16, first_tokens=0):
        pass


@pytest.mark.parametrize("command", [["generate", "--prompt", "1,2"], ["trace", "--out", "unused", "--max-tokens", "64"]])
def test_the_command_line_says_why_a_design_cannot_have_the_cache(monkeypatch, capsys, command):
    """Both commands end with status 4 and the reason, whether the class does not know the option or its layers are refused; other errors are not taken for one."""
    from smoltts_b200 import __main__ as cli
    from smoltts_b200 import registry
    from smoltts_b200._errors import SMOL_ERR_UNSUPPORTED

    def refuse(code):
        def load(path, **kw):
            assert kw["kv_bits"] == 8 and kw["first_tokens"] == 3
            raise SmolError(code, "8-bit cache: softmax attention over keys and values only")
        return load

    argv = command + ["--model", "somewhere", "--kv-bits", "8", "--first-tokens", "3"]
    monkeypatch.setattr(registry, "design_of", lambda path: "Some")
    monkeypatch.setattr(registry, "model_class", lambda name: Plain)
    monkeypatch.setattr(registry, "load_model", lambda path, **kw: Plain(None, **kw))
    assert cli.main(argv) == 4
    assert "'Some' has no 8-bit cache" in capsys.readouterr().err
    monkeypatch.setattr(registry, "model_class", lambda name: Coded)
    monkeypatch.setattr(registry, "load_model", refuse(SMOL_ERR_UNSUPPORTED))
    assert cli.main(argv) == 4
    said = capsys.readouterr().err
    assert "softmax attention over keys and values only" in said and "explicit-token" not in said
    monkeypatch.setattr(registry, "load_model", refuse(SMOL_ERR_CUDA))
    with pytest.raises(SmolError):
        cli.main(argv)


@pytest.mark.parametrize("first", [-1, 2 ** 31, 2 ** 32 + 4])
def test_first_tokens_outside_32_bits_are_refused(monkeypatch, first):
    """(ctypes would keep the low bits.)"""
    from smoltts_b200.lm import HybridLM

    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    with pytest.raises(ValueError, match="first_tokens"):
        HybridLM(None, kv_bits=8, first_tokens=first)


def test_pages_whose_rows_pass_32_bits_are_refused():
    import ctypes

    from smoltts_b200 import _capi_lm as cl

    lib, p = cl.load(), 1 << 20
    cache = cl.SmolLmCache8(k=p, v=p, k_scale=p, v_scale=p, n_pages=1, page_size=1 << 21, kv_heads=1024, dim=16, vdim=16, err=p)
    batch = cl.SmolLmCache8Batch(n_tokens=1, n_seqs=1, max_pages=1, max_new=1, max_len=40, seq_start=p, seq_pos0=p, block_table=p)
    app = cl.SmolLmCache8Append(dtype=0, k=p, v=p, k_row=128, k_head=64, v_row=96, v_head=48, rot_mult=1.0)
    att = cl.SmolLmCache8Attend(dtype=0, heads=1024, q=p, out=p, q_row=16384, q_head=16, out_row=16384, out_head=16, scale=0.1, out_scale=1.0)
    assert lib.smol_lm_cache8_append(ctypes.byref(cache), ctypes.byref(batch), ctypes.byref(app), None) == -4
    assert lib.smol_lm_cache8_attend(ctypes.byref(cache), ctypes.byref(batch), ctypes.byref(att), None, 0, None) == -4
