"""check_status of the operators, with a module and a device that are not there."""
import types

import pytest
import torch

from unimonomoe_b200 import attention, linear


@pytest.mark.parametrize("operators", [attention, linear])
def test_the_word_is_clean_before_the_fault_is_raised(operators, monkeypatch):
    """What is reported by launches on any stream behind the call is not wiped by it: the device has come to rest with a word of zeros."""
    word = torch.tensor([5, 3], dtype=torch.int32)
    at_rest = []
    monkeypatch.setattr(operators, "_load", lambda: types.SimpleNamespace(status_tensor=lambda index: word))
    monkeypatch.setattr(operators.torch.cuda, "synchronize", lambda index=None: at_rest.append((index, word.tolist())))
    with pytest.raises(RuntimeError, match="code 5, at 3"):
        operators.check_status("cuda:0")
    assert at_rest == [(0, [5, 3]), (0, [0, 0])]
    operators.check_status("cuda:0")
    assert len(at_rest) == 3
