"""A check of the extension that fails raises a Python error, with the values it was given in its message."""
import pytest
import torch


def test_a_refusal_with_values_in_its_message_raises():
    c = pytest.importorskip("arcagi2_flashnext_dots3_b200._C")
    with pytest.raises(ValueError, match="CUDA tensor of 2 dimensions"):
        c.teacher_topk(torch.zeros(2, 3), 1, 1.0)
    with pytest.raises(ValueError, match="of 3 dimensions"):
        c.spec_verify(torch.zeros(2, 3), *[torch.zeros(2)] * 4, None, None)
