"""From a teacher's logits to a drafted, sampled answer, on the small FN-shaped model with random weights: the
vocabulary-row operators (:mod:`..ops.distill`, :func:`..ops.sampling.speculative_verify`) as they follow one another.

    python -m arcagi2_flashnext_dots3_b200 distill-demo [--steps N] [--draft-steps N] [--layers N] [--device cuda]

1. rollouts: the teacher engine samples sequences;
2. records: their top-20 teacher tokens (:func:`..training.kd.dump_records`, ``teacher_topk``);
3. distillation: a student whose scales were disturbed trains on them (:func:`..training.kd.seq_kd`, ``kd_topk_grad``);
4. draft head: trains on the teacher's hidden rows (:func:`..training.draft_head.train_draft_head`, ``accept_kl``);
5. acceptance: drafts drawn from the head are verified against the teacher (``speculative_verify`` with the drafts'
   distributions); their rate is an estimate of the mean of sum_v min(q, p) that ``accept_kl`` gives for the same rows;
6. serving: the exported head drafts for the teacher engine, which samples (``speculative_verify`` in the engine's step).

Prints one JSON line per stage and returns them as a list.
"""
from __future__ import annotations

import argparse
import json
import tempfile
from pathlib import Path

import torch


def run(device: str = "cuda", layers: int = 2, steps: int = 8, draft_steps: int = 30, rollouts: int = 4, tokens: int = 48,
        seed: int = 0) -> list:
    from ..config import EngineConfig, fn_small_config
    from ..engine.llm import LLM
    from ..engine.spec import MTPDrafter, SpecDecoder
    from ..models import fn_weights
    from ..models.fn_mtp import MTPHead, mtp_to_engine, random_mtp_dense
    from ..ops import distill, sampling
    from ..ops.sampling import SamplingParams
    from ..training import kd
    from ..training.draft_head import DraftHeadTrain, train_draft_head
    from ..training.student import FNStudent

    dev = torch.device(device)
    log = []

    def report(stage, **kw):
        log.append({"stage": stage, **kw})
        print(json.dumps(log[-1]), flush=True)

    cfg = fn_small_config(num_layers=layers, ple_layers=())
    dense = fn_weights.random_dense(cfg, seed=seed, symmetric=False)
    # random logits are almost flat: a power of two keeps the head on its storage grid and gives it something to say
    dense["lm_head"] = dense["lm_head"] * 64
    weights = fn_weights.to_engine(dense, cfg, dev)
    ec = EngineConfig(max_seqs=rollouts, max_model_len=256, block_size=16, graph_batch_sizes=(rollouts,))
    teacher = LLM(cfg, weights, dev, ec)

    g = torch.Generator().manual_seed(seed)
    prompts = torch.randint(2, cfg.vocab_size, (rollouts, 8), generator=g).tolist()
    outs = [teacher.generate([p], tokens, SamplingParams(temperature=1.0, seed=seed + 100))[0]
            for p in prompts]
    seqs = [(p + o, len(p)) for p, o in zip(prompts, outs)]
    report("rollouts", sequences=len(seqs), tokens=sum(len(o) for o in outs))

    with tempfile.TemporaryDirectory() as tmp:
        report("records", positions=kd.dump_records(teacher, seqs, tmp), k=20)
        files = sorted(Path(tmp).glob("*.npz"))
        student = FNStudent(cfg, dense, dev)
        params = [p for m in student.moe for p in (m.t_gu, m.t_d)]
        with torch.no_grad():
            for p in params:
                p.add_(0.3 * torch.randn(p.shape, generator=g).to(dev))
        opt = torch.optim.Adam(params, lr=3e-2)
        kls = []
        for _ in range(steps):
            opt.zero_grad(set_to_none=True)
            kl, n = 0.0, 0
            for f in files:
                loss, st = kd.seq_kd(student, f)
                (loss / len(files) / tokens).backward()
                kl, n = kl + st["kl"], n + st["n"]
            opt.step()
            kls.append(kl / n)
    report("distillation", kl_first=kls[0], kl_last=kls[-1])

    base = FNStudent(cfg, dense, dev)
    data = []
    with torch.no_grad():
        for ids, _ in seqs:
            ids = torch.tensor(ids)
            h = base.hidden(ids)
            data.append((h, ids, h @ base.lm_head.float().t()))
    mtp = random_mtp_dense(cfg, seed=seed + 9)
    head = DraftHeadTrain(cfg, dense, mtp, dev)
    hist = train_draft_head(head, iter(lambda: data, None), steps=draft_steps, lr_dense=3e-3)
    report("draft head", accepted_first=hist[0][1], accepted_last=hist[-1][1])

    with torch.no_grad():
        q = torch.cat([head.logits(head.step(h[:-1], ids[1:], 0)) for h, ids, _ in data])
        p = torch.cat([t[1:] for _, _, t in data])
        alpha, _ = distill.accept_kl(q, p)
        n = q.shape[0]
        rate = 0.0
        for r in range(8):
            draw = sampling.params_tensors([SamplingParams(temperature=1.0, seed=1000 + r)] * n, list(range(n)), dev)
            drafts, _ = sampling.sample(q, *[x.to(dev) for x in draw], want_lp=False)
            temps, seeds, at = draw[0], draw[3] + 5000, draw[4]
            # every row is one sequence of one draft; the row of the bonus token is not looked at here
            acc, _ = sampling.speculative_verify(p[:, None].expand(n, 2, p.shape[1]), drafts[:, None], temps.to(dev),
                                                 seeds.to(dev), at.to(dev), q[:, None])
            rate += float(acc.float().mean()) / 8
    report("acceptance", expected=float(alpha.mean()), drawn=rate, draws=8 * n)

    for name, weights_mtp in (("untrained", mtp), ("trained", head.export()["dense"])):
        llm = LLM(cfg, weights, dev, ec)
        mh = MTPHead(cfg, weights, mtp_to_engine(weights_mtp, cfg, dense, dev), dev, rollouts + 1, 256, block_size=16)
        sd = SpecDecoder(llm, MTPDrafter(mh), k=3)
        got = sd.generate(prompts, tokens, SamplingParams(temperature=1.0, seed=seed + 100))
        report("serving", head=name, tokens=sum(len(o) for o in got), tokens_per_step=sd.acceptance)
    return log


def main(argv=None):
    ap = argparse.ArgumentParser(prog="distill-demo")
    ap.add_argument("--device", default="cuda" if torch.cuda.is_available() else "cpu")
    ap.add_argument("--layers", type=int, default=2)
    ap.add_argument("--steps", type=int, default=8)
    ap.add_argument("--draft-steps", type=int, default=30)
    ap.add_argument("--rollouts", type=int, default=4)
    ap.add_argument("--tokens", type=int, default=48)
    ap.add_argument("--seed", type=int, default=0)
    a = ap.parse_args(argv)
    run(a.device, a.layers, a.steps, a.draft_steps, a.rollouts, a.tokens, a.seed)


if __name__ == "__main__":
    main()
