"""NaN logits: teacher_topk ranks a NaN above every number, lowest id first, and gives NaN log-probabilities, so that a loss
against such a record is NaN."""
import pytest
import torch

from arcagi2_flashnext_dots3_b200.ops import distill

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
NAN, NINF = float("nan"), float("-inf")


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("V", [1, 7, 300, 4099, 70001])
def test_topk_of_rows_with_nan(V, dtype, device):
    g = torch.Generator().manual_seed(V)
    x = torch.randn(8, V, generator=g).to(dtype)
    x[1] = NAN
    x[2, V // 2] = NAN
    x[3, torch.rand(V, generator=g) < 0.2] = NAN
    x[3, V - 1] = NAN
    x[4, V // 3:] = NINF
    x[4, 0] = NAN
    x[5, torch.rand(V, generator=g) < 0.9] = NINF
    x[5, V - 1] = -NAN                                         # the sign of a NaN says nothing
    x[6, V // 2] = float("inf")
    x[6, V - 1] = NAN
    for k in (1, 20, 128):
        ids, lp = distill.teacher_topk(x.to(device), k)
        for i in range(8):
            z = x[i].double()
            order = sorted((j for j in range(V) if not z[j] <= -1e30),
                           key=lambda j: (0, j) if z[j] != z[j] else (1, -float(z[j]), j))[:k]
            assert ids[i].tolist() == order + [-1] * (k - len(order)), i
            got = lp[i].cpu()
            assert bool((got[len(order):] == NINF).all())
            if bool(torch.isnan(z).any()):
                assert bool(torch.isnan(got[:len(order)]).all()), i
            else:
                want = torch.log_softmax(z, 0)[order]
                assert float((got[:len(order)].double() - want).abs().max()) <= 1e-4
