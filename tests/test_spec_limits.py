"""Sampled speculative steps take what they took when they verified on the host: any number of drafts, any vocabulary."""
import pytest
import torch

from arcagi2_flashnext_dots3_b200.engine.spec import SpecDecoder
from arcagi2_flashnext_dots3_b200.ops import sampling
from arcagi2_flashnext_dots3_b200.ops.sampling import SamplingParams

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def verify(lg, drafts):
    """The verification of one sequence by an engine step whose model gives the logits lg."""
    class Seq:
        sp, out = SamplingParams(temperature=1.0, seed=5), [1]
    d = SpecDecoder.__new__(SpecDecoder)
    d.k = len(drafts)
    d.llm = type("L", (), {"model": type("M", (), {"vocab_sharded": False, "logits": lambda self, x: lg})()})()
    acc, nxt = d._sample_verify([Seq()], None, [drafts])
    return int(acc[0]), int(nxt[0])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("k,V", [(3, (1 << 20) + 3), (130, 50), (128, 50)])
def test_steps_beyond_the_kernels_limits(k, V, device):
    lg = torch.zeros(k + 1, V, device=device)
    lg[:, V - 1] = 60.0
    assert verify(lg, [V - 1] * k) == (k, V - 1)
    assert verify(lg, [V - 1] * (k - 1) + [2]) == (k - 1, V - 1)


def test_what_the_kernels_take():
    assert sampling.verifies(0, 1) and sampling.verifies(128, 1 << 20)
    assert not sampling.verifies(129, 10) and not sampling.verifies(1, (1 << 20) + 1)
