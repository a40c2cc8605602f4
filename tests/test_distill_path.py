"""The vocabulary-row operators where the framework uses them: the distillation loss over hidden rows, teacher records
from an engine model, the draft head's objective, sampled speculative steps, and the demo that runs them in a row."""
import glob

import numpy as np
import pytest
import torch

from arcagi2_flashnext_dots3_b200.config import EngineConfig, fn_small_config
from arcagi2_flashnext_dots3_b200.engine.llm import LLM
from arcagi2_flashnext_dots3_b200.engine.spec import MTPDrafter, NgramDrafter, SpecDecoder
from arcagi2_flashnext_dots3_b200.models import fn_weights
from arcagi2_flashnext_dots3_b200.models.fn_mtp import MTPHead, random_mtp
from arcagi2_flashnext_dots3_b200.ops.sampling import SamplingParams
from arcagi2_flashnext_dots3_b200.training import kd

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("rows", [1, 4, 100])
@pytest.mark.parametrize("wants", ["h", "W", "hW"])
def test_vocab_kd_equals_autograd(device, rows, wants):
    """VocabKD against autograd of the 64-bit formula. Values are fp32 sums of some tens of terms of order one: 2e-5 of
    the largest value is about 170 roundings."""
    g = torch.Generator().manual_seed(3)
    n, V, H, K = 9, 203, 24, 5
    h = torch.randn(n, H, generator=g)
    W = torch.randn(V, H, generator=g) * 0.5
    ids = torch.stack([torch.randperm(V, generator=g)[:K] for _ in range(n)])
    lp = torch.log_softmax(torch.randn(n, V, generator=g) * 2, -1).gather(1, ids)
    lp, order = lp.sort(-1, descending=True)
    ids = ids.gather(1, order)
    ids[2, 3:] = -1
    ids[5] = -1
    w = torch.rand(n, generator=g)
    hd, Wd = h.double().requires_grad_(), W.double().requires_grad_()
    lq = torch.log_softmax(hd @ Wd.t(), -1)
    on = ids >= 0
    q_k = torch.where(on, lq.gather(1, ids.clamp_min(0)), 0.0)
    p = torch.where(on, lp.double().exp(), 0.0)
    t_t = (1 - p.sum(1)).clamp_min(1e-8)
    t_s = (1 - torch.where(on, q_k.exp(), 0.0).sum(1)).clamp_min(1e-8)
    want = torch.where(on, p * (lp.double() - q_k), 0.0).sum(1) + t_t * (t_t.log() - t_s.log())
    (3.0 * (want * w).sum()).backward()
    a, b = (x.to(device).requires_grad_(y) for x, y in ((h, "h" in wants), (W, "W" in wants)))
    loss, kl, _ = kd.VocabKD.apply(a, b, ids.to(device), lp.to(device), w.to(device), rows)
    (3.0 * loss).backward()

    def close(got, ref):
        assert float((got.cpu().double() - ref).abs().max()) <= 2e-5 * max(1.0, float(ref.abs().max()))
    close(kl, want.detach())
    close(loss.detach(), (want * w).sum().detach())
    if "h" in wants:
        close(a.grad, hd.grad)
    if "W" in wants:
        close(b.grad, Wd.grad)


def test_vocab_kd_matches_the_recomputing_loss():
    """VocabKD and VocabTopK + kl21 are one loss: values, gradients and the top-1 agreement."""
    g = torch.Generator().manual_seed(5)
    h = torch.randn(11, 16, generator=g)
    W = torch.randn(90, 16, generator=g)
    ids = torch.stack([torch.randperm(90, generator=g)[:6] for _ in range(11)])
    lp = torch.log_softmax(torch.randn(11, 90, generator=g), -1).gather(1, ids)
    w = torch.rand(11, generator=g)
    h1, h2 = h.clone().requires_grad_(), h.clone().requires_grad_()
    lp_k = kd.VocabTopK.apply(h1, W, ids, 4)
    want = (kd.kl21(lp_k, ids, lp) * w).sum()
    want.backward()
    loss, _, first = kd.VocabKD.apply(h2, W, ids, lp, w, 4)
    loss.backward()
    torch.testing.assert_close(loss, want.detach(), rtol=1e-5, atol=1e-5)
    torch.testing.assert_close(h2.grad, h1.grad, rtol=1e-4, atol=1e-5)
    assert torch.equal(first, lp_k.detach().argmax(1) == 0)


def _engine(device, max_len=160, seqs=3, sharp=64):
    cfg = fn_small_config(num_layers=2, ple_layers=(0,), indexer_budget=1 << 20)
    dense = fn_weights.random_dense(cfg, seed=0, symmetric=False)
    dense["lm_head"] = dense["lm_head"] * sharp
    W = fn_weights.to_engine(dense, cfg, device)
    ec = EngineConfig(max_seqs=seqs, max_model_len=max_len, block_size=16, graph_batch_sizes=(1, 2, 4))
    return cfg, W, LLM(cfg, W, device, ec)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("chunk", [7, 64])
def test_dump_records(device, chunk, tmp_path):
    """Records hold the top tokens of the engine's own logits at every generated position, for a prompt of one token
    and for a sequence with nothing generated, and load as training records; the slots are free again."""
    cfg, _, llm = _engine(device)
    g = torch.Generator().manual_seed(1)
    seqs = [(torch.randint(2, cfg.vocab_size, (L,), generator=g).tolist(), plen) for L, plen in ((30, 9), (5, 1), (6, 6))]
    free = sorted(llm.free_slots)
    assert kd.dump_records(llm, seqs, tmp_path, k=8, chunk=chunk) == 21 + 4
    assert sorted(llm.free_slots) == free
    files = sorted(glob.glob(str(tmp_path / "*.npz")))
    assert len(files) == 3
    for (ids, plen), f in zip(seqs, files):
        got_ids, pos, tid, tlp = kd.load_record(f)
        assert list(got_ids) == ids and list(pos) == list(range(plen, len(ids)))
        if not len(pos):
            continue
        llm.model.reset_slot(0)
        llm.model.assign_blocks(0, len(ids), llm.alloc)
        one = lambda v: torch.tensor([v], dtype=torch.int32, device=device)  # noqa: E731
        x = llm.model.step(torch.tensor(ids, dtype=torch.int32, device=device), one(0), one(0), len(ids))
        llm.alloc.release(0)
        lp = torch.log_softmax(llm.model.logits(x).double(), -1)[plen - 1:-1].cpu()
        mine = lp.gather(1, torch.from_numpy(np.asarray(tid)).long())
        # a chunk's GEMM shapes round differently from the whole sequence's: values, not the order of near ties
        scale = 5e-2 * float(lp.amax(1).abs().max() + 1)
        assert float((torch.from_numpy(np.asarray(tlp)).double() - mine).abs().max()) <= scale
        assert float((mine - lp.topk(8, -1).values).abs().max()) <= scale


def test_dump_records_refusals(tmp_path):
    _, _, llm = _engine("cpu", max_len=32)
    with pytest.raises(ValueError):
        kd.dump_records(llm, [([1, 2, 3], 0)], tmp_path)
    with pytest.raises(ValueError):
        kd.dump_records(llm, [([1, 2, 3], 4)], tmp_path)
    with pytest.raises(ValueError):
        kd.dump_records(llm, [([1] * 33, 4)], tmp_path)
    llm.free_slots.clear()
    with pytest.raises(RuntimeError):
        kd.dump_records(llm, [([1, 2, 3], 1)], tmp_path)


@pytest.mark.gpu
@pytest.mark.parametrize("drafter", ["ngram", "mtp"])
def test_sampled_spec_graph_equals_the_eager_step(drafter):
    """A sampled speculative step replayed as one CUDA graph emits the tokens of the step run kernel by kernel, a greedy
    row and three sampled ones in one batch."""
    prompts = [[5, 9, 11, 40, 7, 9, 11], [3, 8, 21, 13, 8, 21, 13, 8], [4, 4, 4], [7, 1030, 2]]
    sps = [SamplingParams(temperature=0.8, seed=11), SamplingParams(), SamplingParams(temperature=1.3, seed=(1 << 62) - 1),
           SamplingParams(temperature=1.0, seed=3)]
    outs = []
    for graph in (True, False):
        cfg, W, llm = _engine("cuda", max_len=256, seqs=4)
        d = NgramDrafter() if drafter == "ngram" else MTPDrafter(
            MTPHead(cfg, W, random_mtp(cfg, "cuda"), "cuda", 5, 256, block_size=16))
        sd = SpecDecoder(llm, d, k=3)
        sd.use_graph = graph
        seqs = [sd.add(p, 20, sp=sp) for p, sp in zip(prompts, sps)]
        while any(not s.done for s in seqs):
            sd.step()
        outs.append([s.out[:20] for s in seqs])
        if graph:
            assert any(key[1] for key in sd.graphs)
    # the graph's MTP chain runs over other row counts than the eager one: a near tie may break differently later on
    for a, b in zip(*outs):
        assert a[:4] == b[:4]
        assert sum(x == y for x, y in zip(a, b)) >= 0.8 * len(b)


@pytest.mark.parametrize("device", DEVICES)
def test_demo_runs_the_operators_together(device):
    from arcagi2_flashnext_dots3_b200.launch.distill_demo import run
    log = {(r["stage"], r.get("head")): r for r in run(device, steps=4, draft_steps=10, rollouts=2, tokens=24)}
    assert log["records", None]["positions"] == log["rollouts", None]["tokens"]
    assert log["distillation", None]["kl_last"] < log["distillation", None]["kl_first"]
    assert log["draft head", None]["accepted_last"] > log["draft head", None]["accepted_first"]
    acc = log["acceptance", None]
    # the drawn rate is a mean of `draws` acceptances: five standard deviations of a mean of coin flips
    assert abs(acc["expected"] - acc["drawn"]) <= 5 * 0.5 / acc["draws"] ** 0.5
    assert log["serving", "trained"]["tokens"] == log["serving", "untrained"]["tokens"] == 48
