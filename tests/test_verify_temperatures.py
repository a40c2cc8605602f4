"""speculative_verify at every temperature that a request can bring: from 1e-38 (nearly greedy) to infinity.

At a small T the largest logit, if it is alone, has all the mass: a distance of one fp32 step between logits of order ten is
1e-6, so from T = 1e-8 down the second has exp(-100) of it, below the smallest uniform's step (2^-24). At a large one (1e20 and
more) all unmasked logits are equal to fp32. Results are compared with equality, so logits are drawn, not fitted."""
import math

import pytest
import torch

from arcagi2_flashnext_dots3_b200.config import EngineConfig, fn_small_config
from arcagi2_flashnext_dots3_b200.engine.llm import LLM
from arcagi2_flashnext_dots3_b200.engine.spec import NgramDrafter, SpecDecoder
from arcagi2_flashnext_dots3_b200.models import fn_weights
from arcagi2_flashnext_dots3_b200.ops import sampling
from arcagi2_flashnext_dots3_b200.ops.sampling import SamplingParams

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
NINF = float("-inf")
SMALL = [1e-38, 1e-30, 1e-20, 1e-12, 1e-10, 1e-9, 4e-9, 5e-9, 1e-8, 1e-7, 1e-6]


def inputs(g, B, k, V, T, device, dtype=torch.float32, alone=True):
    """Rows whose drafts are the best tokens but for one in four."""
    p = (torch.randn(B, k + 1, V, generator=g) * 4).to(dtype)
    if alone and V > 1:                     # no tie at the top: the first of the largest moves up by a quarter
        at = p.float().argmax(-1, keepdim=True)
        p.scatter_(2, at, (p.float().gather(2, at) + 0.25).to(dtype))
    drafts = p[:, :k].float().argmax(-1)
    wrong = torch.rand(B, k, generator=g) < 0.25
    drafts = torch.where(wrong, torch.randint(0, V, (B, k), generator=g), drafts)
    seeds = torch.randint(-(1 << 62), 1 << 62, (B,), generator=g)
    steps = torch.randint(0, 100000, (B,), generator=g)
    return [x.to(device) for x in (p, drafts, torch.full((B,), T), seeds, steps)]


def rule(lg, drafts, T, seed, step, qlg=None):
    """(accepted, next) of one sequence in 64 bits, the largest logit taken off before the division."""
    V = lg.shape[-1]
    ids = torch.arange(V)

    def prob(row):
        z = row.double()
        z = torch.where(z <= -1e30, NINF, z)
        if bool((z == NINF).all()):
            return torch.zeros(V, dtype=torch.float64)
        z = z - z.max()
        return torch.softmax(torch.where(z == 0, 0.0, z / min(T, 1e300)), 0)
    for j in range(len(drafts) + 1):
        p = prob(lg[j])
        r = p
        if j < len(drafts):
            d = drafts[j]
            q = (ids == d).double() if qlg is None else prob(qlg[j])
            if float(sampling.uniform(seed, step + j, [-1 % (1 << 64)])[0]) * float(q[d]) < float(p[d]):
                continue
            r = torch.where(ids == d, 0.0, p) if qlg is None else (p - q).clamp_min(0)
            r = r if bool((r > 0).any()) else p
        if not bool((r > 0).any()):
            return j, -1
        u = torch.from_numpy(sampling.uniform(seed, step + j, ids.numpy())).double()
        return j, int(torch.where(r > 0, torch.log(r) - torch.log(-torch.log(u)), NINF).argmax())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("T", SMALL)
def test_small_temperatures(T, device):
    g = torch.Generator().manual_seed(3)
    for V in (1, 5, 4099, 32768, 151935):
        for dtype in (torch.float32, torch.bfloat16):
            p, drafts, temps, seeds, steps = inputs(g, 4, 2, V, T, device, dtype)
            got = [x.tolist() for x in sampling.speculative_verify(p, drafts, temps, seeds, steps)]
            t = float(temps[0])
            want = [rule(p[b].cpu(), drafts[b].tolist(), t, int(seeds[b]), int(steps[b])) for b in range(4)]
            assert list(zip(*got)) == want, (V, dtype)
            q = (p[:, :2].float() + torch.randn(4, 2, V, generator=g).to(device)).to(dtype)
            acc, nxt = sampling.speculative_verify(p, drafts, temps, seeds, steps, draft_logits=q)
            want = [rule(p[b].cpu(), drafts[b].tolist(), t, int(seeds[b]), int(steps[b]), q[b].cpu()) for b in range(4)]
            assert list(zip(acc.tolist(), nxt.tolist())) == want, (V, dtype)
            if V > 1 and 1e-12 <= T <= 1e-8:      # below, a logit over T leaves fp32; above, the second token may win
                ref = sampling.speculative_accept(p.float().cpu(), drafts.cpu(), temps.tolist(), seeds.tolist(),
                                                  steps.tolist())
                accepted = [[b < a for b in range(2)] for a in ref[0]]
                assert [[b < a for b in range(2)] for a in got[0]] == accepted
                for b, a in enumerate(ref[0]):     # where the draft was the best token, what is left beside it may tie
                    if a == 2 or int(drafts[b, a]) != int(p[b, a].float().argmax()):
                        assert got[1][b] == ref[1][b]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("T", [1e4, 1e20, 1e30, 3e38, math.inf])
def test_large_temperatures_leave_masked_tokens_out(T, device):
    g = torch.Generator().manual_seed(5)
    for V in (6, 4099, 33001):
        for low in (NINF, -1e30, torch.finfo(torch.float32).min):
            p, drafts, temps, seeds, steps = inputs(g, 6, 2, V, T, device)
            hide = torch.rand(p.shape, generator=g).to(device) < 0.5
            hide[..., V // 2] = False
            p = p.masked_fill(hide, low)
            got = sampling.speculative_verify(p, drafts, temps, seeds, steps)
            want = [rule(p[b].cpu(), drafts[b].tolist(), T, int(seeds[b]), int(steps[b])) for b in range(6)]
            assert list(zip(*(x.tolist() for x in got))) == want


@pytest.mark.parametrize("device", DEVICES)
def test_equal_best_tokens_share_the_mass(device):
    """Of m equal largest logits each is drawn with probability 1 / m, however small T is: 4 sqrt(n / 4) from n / 2."""
    n, V = 400, 700
    p = torch.zeros(n, 1, V, device=device)
    p[:, :, 17] = p[:, :, 650] = 2.0
    s = torch.arange(n, device=device)
    for T in (1e-30, 1e-9, 1e-3):
        acc, nxt = sampling.speculative_verify(p, torch.zeros(n, 0, dtype=torch.int64, device=device),
                                               torch.full((n,), T, device=device), s, torch.zeros_like(s))
        assert set(nxt.tolist()) == {17, 650}
        assert abs(int((nxt == 17).sum()) - n / 2) <= 4 * math.sqrt(n / 4)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("graph", [True, False])
def test_the_engine_at_a_nearly_greedy_temperature(graph, device):
    """Speculative decoding at T = 1e-10 emits what it does at T = 0."""
    if graph and device == "cpu":
        pytest.skip("no CUDA graph on the CPU")
    cfg = fn_small_config(num_layers=2, ple_layers=(0,), indexer_budget=1 << 20)
    dense = fn_weights.random_dense(cfg, seed=0, symmetric=False)
    dense["lm_head"] = dense["lm_head"] * 64
    W = fn_weights.to_engine(dense, cfg, device)
    prompts = [[5, 9, 11, 40, 7, 9, 11], [3, 8, 21, 13, 8, 21, 13, 8], [7, 1030, 2]]
    outs = []
    for T in (0.0, 1e-10):
        llm = LLM(cfg, W, device, EngineConfig(max_seqs=3, max_model_len=128, block_size=16, graph_batch_sizes=(1, 2, 4)))
        sd = SpecDecoder(llm, NgramDrafter(), k=3, use_graph=graph)
        seqs = [sd.add(p, 16, sp=SamplingParams(temperature=T, seed=11 + i)) for i, p in enumerate(prompts)]
        while any(not s.done for s in seqs):
            sd.step()
        outs.append([s.out[:16] for s in seqs])
    assert outs[0] == outs[1]
