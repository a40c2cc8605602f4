"""Timed cases of the vocabulary-row operators: teacher top-k records, top-k distillation loss, acceptance / KL loss of
a draft head, verification of drafted tokens.

``run`` computes a case in elementary torch operations in 32 bits, or with ``own`` through the framework's operators.
``exact`` computes the same from the definitions in 64 bits. Vocabulary sizes are those of the configurations:
151936 (Flash-Next-shaped), 152064 (Dots3-Note-shaped), 32000 (tiny hybrid), 32768 (hot vocabulary of a draft head),
and odd ones next to them.
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
VOCABS = (4096, 4099, 31999, 32000, 32768, 65537, 100003, 151935, 151936, 152064)


def listed():
    return [
        # one decode step of 8 sequences whose teacher distribution is recorded: latency counts
        dict(name="topk_step", op="topk", n=8, vocab=151936, k=20, dtype="fp32", temp=1.0),
        # teacher dump: a prefill chunk of 1024 positions from the engine's fp32 LM head
        dict(name="topk_dump", op="topk", n=1024, vocab=151936, k=20, dtype="fp32", temp=1.0),
        # distillation loss of a few held-out positions, no gradient
        dict(name="kd_eval", op="kd", n=16, vocab=32000, k=20, dtype="fp32", temp=1.0, mode="loss"),
        # the distillation trainer's chunk: 1024 fp32 rows, loss and gradient together
        dict(name="kd_chunk", op="kd", n=1024, vocab=151936, k=20, dtype="fp32", temp=1.0, mode="grad"),
        # a larger half-precision chunk, sharpened teacher
        dict(name="kd_bf16", op="kd", n=4096, vocab=152064, k=20, dtype="bf16", temp=2.0, mode="grad"),
        # autograd form, odd vocabulary (rows that start off every vector boundary), more teacher tokens
        dict(name="kd_odd", op="kd", n=333, vocab=151935, k=50, dtype="bf16", temp=1.0, mode="autograd"),
        # acceptance rate of a draft head on a few positions
        dict(name="accept_eval", op="accept", n=4, vocab=32768, dtype="fp32", temp=1.0, mode="loss"),
        # draft-head training: one unrolled step over 2044 positions of the hot vocabulary
        dict(name="accept_hot", op="accept", n=2044, vocab=32768, dtype="fp32", temp=1.0, mode="autograd"),
        # the same over the full vocabulary in half precision
        dict(name="accept_full", op="accept", n=508, vocab=151936, dtype="bf16", temp=1.0, mode="autograd"),
        # one interactive sequence, three point-mass drafts
        dict(name="verify_one", op="verify", batch=1, k=3, vocab=151936, dtype="fp32", soft=False, ragged=False),
        # a serving batch whose drafts were sampled from the draft head's distribution
        dict(name="verify_soft", op="verify", batch=64, k=3, vocab=151936, dtype="bf16", soft=True, ragged=False),
        # long prompt-lookup drafts of unequal lengths, some sequences greedy
        dict(name="verify_wide", op="verify", batch=32, k=7, vocab=152064, dtype="fp32", soft=False, ragged=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("topk", "kd", "kd", "accept", "accept", "verify", "verify"))
    vocab = rng.choice(VOCABS) if rng.random() < 0.7 else rng.randrange(2000, 152065)
    dtype = rng.choice(("fp32", "bf16", "fp16"))
    temp = rng.choice((1.0, 1.0, 0.7, 2.0))
    rows = 1024 * 151936 // vocab           # at most the elements of the largest listed cases
    if op == "topk":
        return dict(op=op, n=_log_int(rng, 1, min(4096, rows)), vocab=vocab, k=rng.choice((1, 5, 20, 20, 64)),
                    dtype=dtype, temp=temp)
    if op == "kd":
        return dict(op=op, n=_log_int(rng, 1, min(4096, rows)), vocab=vocab, k=rng.choice((1, 7, 20, 20, 64)),
                    dtype=dtype, temp=temp, mode=rng.choice(("loss", "grad", "autograd")))
    if op == "accept":
        return dict(op=op, n=_log_int(rng, 1, min(2048, rows // 2)), vocab=vocab, dtype=dtype, temp=temp,
                    mode=rng.choice(("loss", "autograd")))
    k = rng.randrange(1, 9)
    return dict(op=op, batch=_log_int(rng, 1, max(2, min(128, rows // (2 * k + 1)))), k=k, vocab=vocab, dtype=dtype,
                soft=rng.random() < 0.5, ragged=rng.random() < 0.5)


# --------------------------------------------------------------------------------------------------- inputs
def _rows(g, n, vocab):
    """fp32 next-token logits as a language model gives them: a broad bell of unlikely tokens and, in each row, 32
    plausible ones of widely varying strength."""
    z = torch.randn(n, vocab, generator=g, device="cuda").mul_(1.5)
    at = torch.randint(0, vocab, (n, 32), generator=g, device="cuda")
    up = torch.rand(n, 32, generator=g, device="cuda").mul_(8.0).add_(6.0)
    return z.scatter_(1, at, up)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, dt = case["op"], DTYPES[case["dtype"]]
    s = dict(case)
    if op == "verify":
        B, k, V = case["batch"], case["k"], case["vocab"]
        zp = _rows(g, B * (k + 1), V).view(B, k + 1, V)
        zq = zp[:, :k] + 0.7 * torch.randn(B, k, V, generator=g, device="cuda")
        s["temps"] = torch.full((B,), 0.8, device="cuda")
        if case["ragged"]:
            s["temps"][::5] = 0.0
        s["seeds"] = torch.randint(0, 1 << 62, (B,), generator=g, device="cuda")
        s["steps"] = torch.randint(0, 4096, (B,), generator=g, device="cuda")
        s["n_draft"] = (torch.randint(0, k + 1, (B,), generator=g, device="cuda").to(torch.int32)
                        if case["ragged"] else None)
        drafts = torch.softmax(zq / 0.8, -1).view(B * k, V).multinomial(1, generator=g).view(B, k)
        if not case["soft"]:                # point-mass drafts are the draft head's best tokens
            drafts = zq.argmax(-1)
        s["drafts"] = drafts.to(torch.int32)
        s["logits"] = zp.to(dt)
        s["draft_logits"] = zq.to(dt) if case["soft"] else None
        return s
    n, V = case["n"], case["vocab"]
    z = _rows(g, n, V)
    if op == "topk":
        s["logits"] = z.to(dt)
        return s
    student = z + 0.8 * torch.randn(n, V, generator=g, device="cuda")
    if op == "kd":
        top = torch.log_softmax(z.div_(case["temp"]), -1).topk(case["k"], -1)
        s["t_ids"], s["t_lp"] = top.indices.to(torch.int32), top.values
        s["t_ids"][::17, case["k"] // 2:] = -1          # records with fewer teacher tokens
        s["weight"] = torch.rand(n, generator=g, device="cuda").add_(0.5).div_(n)
        s["logits"] = student.to(dt)
        if case["mode"] == "grad":
            s["out"] = torch.empty_like(s["logits"])
        return s
    s["draft"], s["target"] = student.to(dt), z.to(dt)
    s["g_alpha"] = torch.rand(n, generator=g, device="cuda").neg_().div_(n)
    s["g_kl"] = torch.full((n,), 0.075 / n, device="cuda")
    return s


# --------------------------------------------------------------------------------------------- plain forms
def _plain_topk(logits, k, temp):
    z = logits.float()
    v, ids = torch.sort(z, dim=-1, descending=True, stable=True)
    v, ids = v[:, :k], ids[:, :k]
    m = v[:, :1]
    lse = torch.log(torch.exp((z - m) / temp).sum(-1, keepdim=True))
    return ids.to(torch.int32), (v - m) / temp - lse


def _kd_bins(ids, lp, V):
    """Valid teacher entries (in range, first place of a repeated id), clamped ids, teacher mass per entry."""
    same = (ids[:, :, None] == ids[:, None, :]).tril(-1).any(-1)
    valid = (ids >= 0) & (ids < V) & ~same
    return valid, ids.long().clamp(0, V - 1), torch.where(valid, lp.float().exp(), 0.0)


def _plain_kd(logits, ids, lp, temp, weight):
    n, V = logits.shape
    valid, at, pt = _kd_bins(ids, lp, V)
    z = logits.float() / temp
    e = torch.exp(z - z.max(-1, keepdim=True).values)
    total = e.sum(-1, keepdim=True)
    ek = torch.where(valid, e.gather(1, at), 0.0)
    tail = e.scatter_add(1, at, -ek).sum(-1, keepdim=True) / total
    ps = ek / total
    s = z.gather(1, at) - z.max(-1, keepdim=True).values - total.log()
    tt = (1 - pt.sum(-1, keepdim=True)).clamp_min(1e-8)
    ts = tail.clamp_min(1e-8)
    loss = torch.where(pt > 0, pt * (lp - s), 0.0).sum(-1) + (tt * (tt.log() - ts.log()))[:, 0]
    if weight is None:
        return loss
    c = torch.where(valid, -pt + torch.where(tail >= 1e-8, tt / ts, 0.0) * ps, 0.0)
    d = e.mul_(-c.sum(-1, keepdim=True) / total).scatter_add_(1, at, c)
    return loss, d.mul_(weight[:, None] / temp).to(logits.dtype)


def _plain_accept(draft, target, temp, g_alpha, g_kl):
    zq, zp = draft.float() / temp, target.float() / temp
    lq = zq - zq.max(-1, keepdim=True).values
    lq = lq - torch.exp(lq).sum(-1, keepdim=True).log()
    lp = zp - zp.max(-1, keepdim=True).values
    lp = lp - torch.exp(lp).sum(-1, keepdim=True).log()
    q, p = torch.exp(lq), torch.exp(lp)
    alpha = torch.minimum(q, p).sum(-1)
    kl = torch.where(p > 0, p * (lp - lq), 0.0).sum(-1)
    if g_alpha is None:
        return alpha, kl
    h = (lq < lp).float() + 0.5 * (lq == lp).float()
    a = (q * h).sum(-1, keepdim=True)
    d = g_alpha[:, None] * q * (h - a) + g_kl[:, None] * (q - p)
    return alpha, kl, d.div_(temp).to(draft.dtype)


_C = [c - (1 << 64) for c in (0x9E3779B97F4A7C15, 0xD1B54A32D192ED03, 0x8CB92BA72F3D8DD7, 0xBF58476D1CE4E5B9,
                              0x94D049BB133111EB)]


def _shr(z, n):
    return (z >> n) & ((1 << (64 - n)) - 1)


def _uniform(seeds, steps, index):
    """The sampler's counter hash: uniforms in (0, 1) of (seed, step, index), int64 tensors that broadcast."""
    z = seeds * _C[0] + steps * _C[1] + index * _C[2] + 1
    z = (z ^ _shr(z, 30)) * _C[3]
    z = (z ^ _shr(z, 27)) * _C[4]
    return (_shr(z ^ _shr(z, 31), 41).float() + 0.5) * (1.0 / 8388608.0)


def _lowest_best(x):
    """Index of the largest value of each row, the lowest among equal ones; -1 where every value is -inf."""
    V = x.shape[-1]
    best = x.max(-1, keepdim=True).values
    at = torch.where((x == best) & (best > -math.inf), torch.arange(V, device=x.device), V).min(-1).values
    return torch.where(at == V, -1, at)


def _plain_verify(logits, drafts, temps, seeds, steps, draft_logits, n_draft):
    B, k1, V = logits.shape
    k = k1 - 1
    rows = torch.arange(B, device=logits.device)
    n_draft = torch.full_like(drafts[:, 0], k) if n_draft is None else n_draft
    greedy = temps <= 0
    t = torch.where(greedy, 1.0, temps)[:, None, None]
    z = logits.float() / t
    lp = z - z.max(-1, keepdim=True).values
    lp = lp - torch.exp(lp).sum(-1, keepdim=True).log()
    d = drafts.long()
    lpd = lp[:, :k].gather(2, d[..., None])[..., 0]
    u = _uniform(seeds[:, None], steps[:, None] + torch.arange(k, device=d.device), torch.full_like(d, -1))
    lq = None
    if draft_logits is None:
        ok = u < torch.exp(lpd)
    else:
        zq = draft_logits.float() / t
        lq = zq - zq.max(-1, keepdim=True).values
        lq = lq - torch.exp(lq).sum(-1, keepdim=True).log()
        ok = u * torch.exp(lq.gather(2, d[..., None])[..., 0]) < torch.exp(lpd)
    best = _lowest_best(z)
    ok = torch.where(greedy[:, None], d == best[:, :k], ok)
    ok = ok & (torch.arange(k, device=d.device) < n_draft[:, None])
    acc = torch.cumprod(ok.long(), 1).sum(1)
    p = torch.exp(lp[rows, acc])
    r = p.clone()
    rejected = acc < n_draft
    at = acc.clamp_max(k - 1)
    if lq is None:
        r[rows, d[rows, at]] = torch.where(rejected, 0.0, r[rows, d[rows, at]])
    else:
        r = torch.where(rejected[:, None], (p - torch.exp(lq[rows, at])).clamp_min(0.0), r)
    r = torch.where((r > 0).any(-1, keepdim=True), r, p)
    noise = _uniform(seeds[:, None], (steps + acc)[:, None], torch.arange(V, device=d.device))
    drawn = _lowest_best(torch.log(r) - torch.log(-torch.log(noise)))
    return acc.to(torch.int32), torch.where(greedy, best[rows, acc], drawn).to(torch.int32)


# ------------------------------------------------------------------------------------------- one pass
def run(s):
    op = s["op"]
    if own:
        return _run_own(s)
    if op == "topk":
        return _plain_topk(s["logits"], s["k"], s["temp"])
    if op == "kd":
        return _plain_kd(s["logits"], s["t_ids"], s["t_lp"], s["temp"], None if s["mode"] == "loss" else s["weight"])
    if op == "accept":
        g = (None, None) if s["mode"] == "loss" else (s["g_alpha"], s["g_kl"])
        return _plain_accept(s["draft"], s["target"], s["temp"], *g)
    return _plain_verify(s["logits"], s["drafts"], s["temps"], s["seeds"], s["steps"], s["draft_logits"], s["n_draft"])


def _run_own(s):
    from arcagi2_flashnext_dots3_b200.ops import distill, sampling
    op = s["op"]
    if op == "topk":
        return distill.teacher_topk(s["logits"], s["k"], temperature=s["temp"])
    if op == "kd":
        if s["mode"] == "loss":
            return distill.kd_topk(s["logits"], s["t_ids"], s["t_lp"], temperature=s["temp"])
        if s["mode"] == "grad":
            return distill.kd_topk_grad(s["logits"], s["t_ids"], s["t_lp"], s["weight"], temperature=s["temp"],
                                        out=s["out"])
        z = s["logits"].detach().requires_grad_()
        loss = distill.kd_topk(z, s["t_ids"], s["t_lp"], temperature=s["temp"])
        return loss.detach(), torch.autograd.grad(loss, z, s["weight"])[0]
    if op == "accept":
        if s["mode"] == "loss":
            return distill.accept_kl(s["draft"], s["target"], temperature=s["temp"])
        z = s["draft"].detach().requires_grad_()
        alpha, kl = distill.accept_kl(z, s["target"], temperature=s["temp"])
        d, = torch.autograd.grad((alpha, kl), z, (s["g_alpha"], s["g_kl"]))
        return alpha.detach(), kl.detach(), d
    return sampling.speculative_verify(s["logits"], s["drafts"], s["temps"], s["seeds"], s["steps"],
                                       draft_logits=s["draft_logits"], n_draft=s["n_draft"])


def work(case):
    w = {"fp32": 4, "bf16": 2, "fp16": 2}[case["dtype"]]
    V = case["vocab"]
    if case["op"] == "verify":
        rows = case["batch"] * (case["k"] + 1 + (case["k"] if case["soft"] else 0))
        return {"bytes": rows * V * w + case["batch"] * (4 * case["k"] + 28), "flops": 3 * rows * V}
    n = case["n"]
    if case["op"] == "topk":
        return {"bytes": n * (V * w + 8 * case["k"]), "flops": 4 * n * V}
    if case["op"] == "kd":
        passes = 1 if case["mode"] == "loss" else 2
        return {"bytes": n * (passes * V * w + 8 * case["k"] + 8), "flops": 3 * passes * n * V}
    passes = 2 if case["mode"] == "loss" else 3
    return {"bytes": n * (passes * V * w + 16), "flops": 5 * passes * n * V}


# ------------------------------------------------------------------------------------------- 64-bit results
def _chunks(n, V):
    step = max(1, (1 << 26) // V)
    return [(a, min(n, a + step)) for a in range(0, n, step)]


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "verify":
        got = [_exact_verify(s, b) for b in range(case["batch"])]
        return tuple(torch.tensor(x, dtype=torch.int32, device="cuda") for x in zip(*got))
    T, V = case["temp"], case["vocab"]
    parts = []
    for a, b in _chunks(case["n"], V):
        if op == "topk":
            z = s["logits"][a:b].double()
            order = torch.sort(z, dim=-1, descending=True, stable=True).indices[:, :case["k"]]
            parts.append((order.to(torch.int32), torch.log_softmax(z / T, -1).gather(1, order)))
        elif op == "kd":
            lp = torch.log_softmax(s["logits"][a:b].double() / T, -1)
            parts.append(_exact_kd(lp, s["t_ids"][a:b].long(), s["t_lp"][a:b].double(),
                                   None if case["mode"] == "loss" else s["weight"][a:b].double(), T))
        else:
            lq = torch.log_softmax(s["draft"][a:b].double() / T, -1)
            lp = torch.log_softmax(s["target"][a:b].double() / T, -1)
            alpha, kl = torch.minimum(lq, lp).exp().sum(-1), (lp.exp() * (lp - lq)).sum(-1)
            if case["mode"] == "loss":
                parts.append((alpha, kl))
                continue
            q, h = lq.exp(), torch.where(lq < lp, 1.0, torch.where(lq == lp, 0.5, 0.0)).double()
            ga, gk = s["g_alpha"][a:b, None].double(), s["g_kl"][a:b, None].double()
            parts.append((alpha, kl, (ga * q * (h - (q * h).sum(-1, keepdim=True)) + gk * (q - lp.exp())) / T))
    out = tuple(torch.cat(x) for x in zip(*parts))
    return out[0] if len(out) == 1 else out


def _exact_kd(lp_s, ids, lp_t, weight, T):
    """Per row the K + 1 bins as one distribution each: teacher tokens, then everything else."""
    n, V = lp_s.shape
    at = torch.where(ids >= 0, ids, V)
    mark = torch.zeros(n, V + 1, dtype=torch.bool, device=ids.device).scatter_(1, at, True)[:, :V]
    ls = torch.cat([lp_s, torch.zeros(n, 1, dtype=lp_s.dtype, device=ids.device)], 1).gather(1, at)
    pt = torch.where(ids >= 0, lp_t.exp(), 0.0)
    tt = (1 - pt.sum(-1)).clamp_min(1e-8)
    tail = torch.where(mark, 0.0, lp_s.exp()).sum(-1)
    ts = tail.clamp_min(1e-8)
    loss = torch.where(pt > 0, pt * (lp_t - ls), 0.0).sum(-1) + tt * (tt / ts).log()
    if weight is None:
        return (loss,)
    c = -pt + torch.where(ids >= 0, ls.exp(), 0.0) * torch.where(tail >= 1e-8, tt / ts, 0.0)[:, None]
    d = torch.zeros(n, V + 1, dtype=lp_s.dtype, device=ids.device).scatter_add_(1, at, c)[:, :V]
    return loss, (d - lp_s.exp() * c.sum(-1, keepdim=True)) * (weight / T)[:, None]


def _exact_uniform(seed, step, index):
    """Counter-hash uniforms of a tensor of indices: 64-bit words kept as (high, low) 32-bit halves."""
    start = (seed * 0x9E3779B97F4A7C15 + step * 0xD1B54A32D192ED03 + 1) % (1 << 64)

    def times(hi, lo, c):
        ch, cl = c >> 32, c & 0xFFFFFFFF
        parts = [(lo >> 16) * cl, (lo & 0xFFFF) * cl]           # each below 2^48
        low = (parts[0] << 16) + parts[1]                       # wraps; its low 32 bits count
        top = ((parts[0] >> 16) + (((parts[0] & 0xFFFF) << 16) + parts[1] >> 32))
        cross = ((hi & 0xFFFFFFFF) * (cl & 0xFFFF) + (((hi * (cl >> 16)) & 0xFFFF) << 16)
                 + lo * (ch & 0xFFFF) + (((lo * (ch >> 16)) & 0xFFFF) << 16))
        return (top + cross) & 0xFFFFFFFF, low & 0xFFFFFFFF

    def fold(hi, lo, n):
        return hi ^ (hi >> n), lo ^ (((hi << (32 - n)) | (lo >> n)) & 0xFFFFFFFF)

    hi, lo = times((index >> 32) & 0xFFFFFFFF, index & 0xFFFFFFFF, 0x8CB92BA72F3D8DD7)
    lo = lo + (start & 0xFFFFFFFF)
    hi, lo = (hi + (start >> 32) + (lo >> 32)) & 0xFFFFFFFF, lo & 0xFFFFFFFF
    hi, lo = times(*fold(hi, lo, 30), 0xBF58476D1CE4E5B9)
    hi, lo = times(*fold(hi, lo, 27), 0x94D049BB133111EB)
    hi, lo = fold(hi, lo, 31)
    return ((hi >> 9).double() + 0.5) / 8388608.0


def _exact_verify(s, b):
    """One sequence, draft by draft: (accepted drafts, next token)."""
    T, seed, step = float(s["temps"][b]), int(s["seeds"][b]), int(s["steps"][b])
    z = s["logits"][b].double()
    V = z.shape[-1]
    ids = torch.arange(V, device=z.device)
    n = z.shape[0] - 1 if s["n_draft"] is None else int(s["n_draft"][b])
    j = 0
    while True:
        if T <= 0:
            best = int(ids[z[j] == z[j].max()].min())
            if j == n or int(s["drafts"][b, j]) != best:
                return j, best
        else:
            r = torch.softmax(z[j] / T, -1)
            if j < n:
                d = int(s["drafts"][b, j])
                u = float(_exact_uniform(seed, step + j, torch.full((1,), -1, device=z.device))[0])
                q = None if s["draft_logits"] is None else torch.softmax(s["draft_logits"][b, j].double() / T, -1)
                rejected = u * (1.0 if q is None else float(q[d])) >= float(r[d])
                r = torch.where(ids == d, 0.0, r) if q is None else (r - q).clamp_min(0.0)
            if j == n or rejected:
                race = torch.where(r > 0, -torch.log(_exact_uniform(seed, step + j, ids)) / r, math.inf)
                return j, int(ids[race == race.min()].min())
        j += 1
