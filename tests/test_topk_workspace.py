"""teacher_topk of many short rows: its workspace is a share of the logits, not a fixed size per row."""
import pytest
import torch

from arcagi2_flashnext_dots3_b200.ops import distill


@pytest.mark.gpu
@pytest.mark.parametrize("V", [3, 37, 260])
def test_workspace_of_short_rows(V):
    """At most 12 bytes for each 16-byte vector that a row can touch (V / 8 + 2 of them) beside the outputs; results as ever."""
    n, k = 1000000, 2
    g = torch.Generator(device="cuda").manual_seed(V)
    x = torch.randn(n, V, generator=g, device="cuda", dtype=torch.bfloat16)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    ids, lp = distill.teacher_topk(x, k)
    torch.cuda.synchronize()
    extra = torch.cuda.max_memory_allocated() - before - 2 * n * k * 4
    assert extra <= 12 * n * (V // 8 + 2) + (4 << 20)
    z, order = torch.sort(x, dim=1, descending=True, stable=True)
    assert torch.equal(ids, order[:, :k].int())
    want = torch.log_softmax(x.float(), 1).gather(1, order[:, :k])
    assert float((lp - want).abs().max()) <= 1e-4
