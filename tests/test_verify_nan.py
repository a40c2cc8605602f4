"""Verification of NaN logits: a position that holds one has no token to give (-1), whatever the temperature, and a speculative
step of the engine raises in place of emitting one."""
import pytest
import torch

from arcagi2_flashnext_dots3_b200.config import EngineConfig, fn_small_config
from arcagi2_flashnext_dots3_b200.engine.llm import LLM
from arcagi2_flashnext_dots3_b200.engine.spec import NgramDrafter, SpecDecoder
from arcagi2_flashnext_dots3_b200.models import fn_weights
from arcagi2_flashnext_dots3_b200.ops import sampling
from arcagi2_flashnext_dots3_b200.ops.sampling import SamplingParams

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
NAN = float("nan")


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("T", [0.0, 1e-10, 0.8])
def test_verification_of_rows_with_nan(T, dtype, device):
    g = torch.Generator().manual_seed(2)
    for V in (2, 300, 40001):
        p = (torch.randn(5, 3, V, generator=g) * 2).to(dtype)
        d = p[:, :2].float().argmax(-1)
        p.scatter_(2, p.float().argmax(-1, keepdim=True), 60.0)    # sure of the drafts
        p[1, 0, V - 1] = NAN
        p[2, 1] = NAN
        p[3, 2, 0] = NAN
        t, s = torch.full((5,), T, device=device), torch.arange(5, device=device)
        acc, nxt = sampling.speculative_verify(p.to(device), d.to(device), t, s, s)
        assert acc.tolist() == [2, 0, 1, 2, 2] and nxt.tolist()[1:4] == [-1, -1, -1]
        best = p[:, 2].float().argmax(-1)
        assert int(nxt[0]) == int(best[0]) and int(nxt[4]) == int(best[4])


@pytest.mark.parametrize("device", DEVICES)
def test_a_draft_row_with_nan_is_no_distribution(device):
    """Its draft is rejected and the next token comes from the target, as without a residual."""
    g = torch.Generator().manual_seed(3)
    for V in (5, 300, 40001):
        p = torch.randn(6, 2, V, generator=g)
        q = p[:, :1] + torch.randn(6, 1, V, generator=g)
        q[::2, 0, V // 2] = NAN
        d = q[:, :, :V // 2].argmax(-1)
        t, s = torch.full((6,), 0.8), torch.arange(6)
        acc, nxt = (x.tolist() for x in sampling.speculative_verify(*(x.to(device) for x in (p, d, t, s, s)),
                                                                    draft_logits=q.to(device)))
        for b in range(0, 6, 2):
            u = torch.from_numpy(sampling.uniform(b, b, torch.arange(V).numpy())).double()
            r = torch.softmax(p[b, 0].double() / 0.8, 0)
            assert acc[b] == 0 and nxt[b] == int((torch.log(r) - torch.log(-torch.log(u))).argmax())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("graph", [True, False])
def test_the_engine_raises_in_place_of_a_token(graph, device):
    if graph and device == "cpu":
        pytest.skip("no CUDA graph on the CPU")
    cfg = fn_small_config(num_layers=2, ple_layers=(0,), indexer_budget=1 << 20)
    W = fn_weights.to_engine(fn_weights.random_dense(cfg, seed=0, symmetric=False), cfg, device)
    llm = LLM(cfg, W, device, EngineConfig(max_seqs=3, max_model_len=128, block_size=16, graph_batch_sizes=(1, 2, 4)))
    logits = llm.model.logits
    sd = SpecDecoder(llm, NgramDrafter(), k=3, use_graph=graph)
    for i in range(2):
        sd.add([5, 9, 11, 40, 7], 16, sp=SamplingParams(temperature=0.8, seed=i))
    llm.model.logits = lambda x: logits(x) * NAN
    with pytest.raises(RuntimeError):
        sd.step()
