"""Vocabulary-row operators (ops/distill.py, ops.sampling.speculative_verify): results and gradients against plain
64-bit statements of the formulas, on the CPU path and on the kernels.

Tolerances. Logits lie within +-64 after the division by the temperature. A log-probability is formed from such
values in fp32 in a handful of operations, so it is off by at most 4 ulp of 64, 4 * 64 * 2^-23 < 3.1e-5 (absolute);
that is also the relative error of a probability. Losses are sums of probabilities (of total at most 1) times such
logs and probabilities times logs of at most 64 + log 2^20: TOL = 1e-4 covers both. A gradient is w (a - b) with a, b
at most one probability each, so it is off by TOL * w * (a + b), plus the rounding to the output type.
"""
import math

import pytest
import torch

from arcagi2_flashnext_dots3_b200.ops import distill, sampling

TOL = 1e-4
EPS = {torch.float32: 2.0 ** -23, torch.float16: 2.0 ** -10, torch.bfloat16: 2.0 ** -7}
NINF = float("-inf")
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


# ------------------------------------------------------------------------------------------------- 64-bit statements
def log_p(row, T):
    """log softmax(row / T) of one row in 64 bits, None when every entry is masked."""
    z = row.detach().cpu().double()
    z = torch.where(z <= -1e30, NINF, z) / T
    return None if bool((z == NINF).all()) else z - torch.logsumexp(z, 0)


def kd_row(row, ids, lp, T):
    """(loss, gradient) of one row."""
    V = row.shape[0]
    ls = log_p(row, T)
    if ls is None:
        return 0.0, torch.zeros(V, dtype=torch.float64)
    seen, entries = set(), []
    for i, t in zip(ids.tolist(), lp.tolist()):
        if 0 <= i < V and i not in seen:
            seen.add(i)
            entries.append((i, t))
    tt = max(1.0 - sum(math.exp(t) for _, t in entries), 1e-8)
    inside = torch.zeros(V, dtype=torch.bool)
    inside[[i for i, _ in entries]] = True
    tail = float(ls[~inside].exp().sum())
    ts = max(tail, 1e-8)
    loss = tt * (math.log(tt) - math.log(ts))
    d = torch.zeros(V, dtype=torch.float64)
    total = 0.0
    for i, t in entries:
        pt, s = math.exp(t), float(ls[i])
        if pt > 0:
            loss += pt * (t - s)
        c = -pt + (tt / ts * math.exp(s) if tail >= 1e-8 else 0.0)
        d[i] += c
        total += c
    return loss, (d - ls.exp() * total) / T


def accept_row(q_row, p_row, T):
    """(alpha, kl, d alpha, d kl) of one row."""
    lq, lp = log_p(q_row, T), log_p(p_row, T)
    V = q_row.shape[0]
    if lq is None or lp is None:
        z = torch.zeros(V, dtype=torch.float64)
        return 0.0, 0.0, z, z
    q, p = lq.exp(), lp.exp()
    h = (lq <= lp).double()
    kl = float(torch.where(p > 0, p * (lp - lq), 0.0).sum())
    return float(torch.minimum(q, p).sum()), kl, q * (h - (q * h).sum()) / T, (q - p) / T


def verify_row(lg, drafts, T, seed, step, qlg=None):
    """(accepted, next) of one sequence, draft by draft."""
    V = lg.shape[-1]
    ids = torch.arange(V)
    for j in range(len(drafts) + 1):
        z = lg[j].detach().cpu().double()
        z = torch.where(z <= -1e30, NINF, z)
        d = drafts[j] if j < len(drafts) else None
        if T <= 0:
            best = -1 if bool((z == NINF).all()) else int(ids[z == z.max()].min())
            if d is not None and d == best and d >= 0:
                continue
            return j, best
        lp = log_p(z, T)
        p = torch.zeros(V, dtype=torch.float64) if lp is None else lp.exp()
        r = p
        if d is not None:
            if qlg is None:
                q = (ids == d).double()
            else:
                lq = log_p(qlg[j], T)
                q = torch.zeros(V, dtype=torch.float64) if lq is None else lq.exp()
            if 0 <= d < V and float(sampling.uniform(seed, step + j, [-1 % (1 << 64)])[0]) * float(q[d]) < float(p[d]):
                continue
            r = torch.where(ids == d, 0.0, p) if qlg is None else (p - q).clamp_min(0)
            if not bool((r > 0).any()):
                r = p
        if not bool((r > 0).any()):
            return j, -1
        u = torch.from_numpy(sampling.uniform(seed, step + j, ids.numpy())).double()
        return j, int(torch.where(r > 0, torch.log(r) - torch.log(-torch.log(u)), NINF).argmax())


def close(got, want):
    got = float(got.detach())
    return got == want or abs(got - want) <= TOL * (1 + abs(want))


# ------------------------------------------------------------------------------------------------------ inputs
def rows(g, n, V, dtype, device, ld=None, offset=0, scale=4.0):
    """[n, V] logits that are a view with row stride ld and a start `offset` elements into its storage."""
    ld = ld or V
    buf = torch.randn(offset + n * ld, generator=g) * scale
    return buf.to(dtype).to(device)[offset:].as_strided((n, V), (ld, 1), offset)


def mask_some(g, x, how):
    """Masks parts of x in place: a third of the row, all but one token, everything."""
    low = NINF if how == "inf" else torch.finfo(torch.float32 if x.dtype == torch.float16 else x.dtype).min
    if x.dtype == torch.float16:
        low = NINF
    V = x.shape[1]
    for i in range(x.shape[0]):
        if i % 4 == 1:
            x[i, torch.rand(V, generator=g).to(x.device) < 0.33] = low
        elif i % 4 == 2:
            keep = int(torch.randint(0, V, (1,), generator=g))
            v = x[i, keep].clone()
            x[i] = low
            x[i, keep] = v
        elif i % 4 == 3:
            x[i] = low
    return x


SHAPES = [(1, 1, None, 0), (4, 2, None, 0), (5, 7, 9, 3), (4, 31, 31, 1), (4, 257, 260, 5), (3, 4099, None, 0),
          (2, 32768, None, 8), (2, 50001, 50007, 2), (1, 151936, None, 0), (2, 151935, None, 0)]
IDS = ["x".join(map(str, s[:2])) for s in SHAPES]


# ------------------------------------------------------------------------------------------------- teacher top-k
def check_topk(x, k, T):
    ids, lp = distill.teacher_topk(x, k, temperature=T)
    assert ids.dtype == torch.int32 and lp.dtype == torch.float32 and ids.shape == lp.shape == (x.shape[0], k)
    for i in range(x.shape[0]):
        ls = log_p(x[i], T)
        if ls is None:
            want = []
        else:
            z = x[i].detach().cpu().double()
            want = [j for j in torch.sort(z, dim=0, descending=True, stable=True).indices[:k].tolist() if ls[j] > NINF]
        assert ids[i].tolist() == want + [-1] * (k - len(want)), i
        for got, j in zip(lp[i].tolist(), want):
            assert abs(got - float(ls[j])) <= TOL
        assert all(v == NINF for v in lp[i, len(want):].tolist())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=IDS)
def test_topk_order_and_log_probabilities(shape, dtype, device):
    n, V, ld, off = shape
    g = torch.Generator().manual_seed(V)
    x = rows(g, n, V, dtype, device, ld, off)
    for k, T in ((1, 1.0), (20, 0.7), (128, 2.0)):
        check_topk(x, k, T)


@pytest.mark.parametrize("device", DEVICES)
def test_topk_ties_masks_and_short_rows(device):
    g = torch.Generator().manual_seed(1)
    for V in (3, 40, 3001, 70000):
        x = torch.randint(0, 3, (6, V), generator=g).float().to(device)      # ties decide nearly every place
        check_topk(x, 20, 1.0)
        x[2] = 1.0                                                            # every token equal
        x[3, ::2] = -0.0
        x[3, 1::2] = 0.0                                                      # both zeros are one value
        check_topk(mask_some(g, x, "low"), 64, 1.0)
    x = torch.full((2, 9000), NINF)
    x[0, 17] = 3.0
    x[1, 8999] = -40.0
    check_topk(x.to(device), 5, 1.0)
    sorted_rows = torch.arange(30000).float().div(1000)[None].repeat(2, 1)
    sorted_rows[1] = sorted_rows[1].flip(0)
    check_topk(sorted_rows.to(device), 128, 1.0)                              # the largest all in one place


# ------------------------------------------------------------------------------------------------- distillation
def teacher(g, x, K, T, device):
    """Teacher records of rows near x: K top tokens with padding, a repeated id and an id out of range."""
    n, V = x.shape
    t = torch.where(x.float().cpu() <= -1e30, 0.0, x.float().cpu()) + torch.randn(n, V, generator=g)
    lp, ids = torch.log_softmax(t / T, -1).topk(min(K, V), -1)
    pad = torch.full((n, K - ids.shape[1]), -1)
    ids, lp = torch.cat([ids, pad], 1), torch.cat([lp, pad.float()], 1)
    if n > 1 and K > 3:
        ids[1, K // 2:] = -1
        ids[0, 2] = ids[0, 0]
        ids[0, 3] = V + 5
        lp[0, 1] = NINF
    return ids.to(device), lp.to(device)


def check_kd(x, ids, lp, T, w):
    n, V = x.shape
    eps = EPS[x.dtype]
    want = [kd_row(x[i], ids[i], lp[i], T) for i in range(n)]
    loss = distill.kd_topk(x, ids, lp, temperature=T)
    loss2, d2 = distill.kd_topk_grad(x, ids, lp, w, temperature=T)
    z = x.detach().requires_grad_()
    loss3 = distill.kd_topk(z, ids, lp, temperature=T)
    d3, = torch.autograd.grad(loss3, z, w)
    assert loss.dtype == torch.float32 and d2.dtype == d3.dtype == x.dtype
    for i, (l, d) in enumerate(want):
        for got in (loss[i], loss2[i], loss3[i]):
            assert close(got, l), (i, got, l)
        wi = float(w[i])
        ls = log_p(x[i], T)
        p = torch.zeros(V, dtype=torch.float64) if ls is None else ls.exp()
        pt = torch.zeros(V, dtype=torch.float64)
        ok = (ids[i].cpu() >= 0) & (ids[i].cpu() < V)
        pt.index_add_(0, ids[i].cpu()[ok].long(), lp[i].cpu()[ok].double().exp())
        scale = float(max(1.0, (1 - pt.sum()).clamp_min(1e-8) / max(1e-8, float(p[pt == 0].sum()))))
        for got in (d2[i], d3[i]):
            err = (got.detach().cpu().double() - wi * d).abs()
            lim = TOL * wi / T * scale * (p + pt) + eps * (wi * d).abs() + 6e-8
            assert bool((err <= lim).all()), (i, float((err - lim).max()))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=IDS)
def test_kd_loss_and_gradient(shape, dtype, device):
    n, V, ld, off = shape
    g = torch.Generator().manual_seed(V + 1)
    for K, T in ((20, 1.0), (1, 0.7), (128, 2.0)):
        x = rows(g, n, V, dtype, device, ld, off)
        ids, lp = teacher(g, x, K, T, device)
        check_kd(x, ids.to(torch.int32) if K == 20 else ids, lp, T, (torch.rand(n, generator=g) + 0.5).to(device))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("how", ["inf", "low"])
def test_kd_masked_rows(how, device):
    g = torch.Generator().manual_seed(7)
    for V in (5, 1000, 40001):
        for dtype in DTYPES:
            x = mask_some(g, rows(g, 8, V, dtype, device), how)
            ids, lp = teacher(g, x, 6, 1.0, device)
            for i in range(8):                 # teacher tokens that the student masks give an infinite loss: keep
                for j in range(6):             # them out of this test (the next one has them)
                    if 0 <= int(ids[i, j]) < V and float(x[i, int(ids[i, j])]) <= -1e30:
                        ids[i, j] = -1
            check_kd(x, ids, lp, 1.0, torch.rand(8, generator=g).to(device))


@pytest.mark.parametrize("device", DEVICES)
def test_kd_infinite_loss_nan_and_floors(device):
    x = torch.randn(5, 300, generator=torch.Generator().manual_seed(3))
    x[0, 10] = NINF
    x[1, 20] = float("nan")
    x[2, 30] = 60.0                                   # the tail of the student is below its floor
    x = x.to(device)
    ids = torch.tensor([[10, 11], [1, 2], [30, 31], [4, 4], [-1, -1]], device=device)
    lp = torch.log(torch.tensor([[0.5, 0.25], [0.5, 0.25], [0.9, 0.05], [0.6, 0.3], [0.5, 0.5]])).to(device)
    loss, d = distill.kd_topk_grad(x, ids, lp, torch.ones(5, device=device))
    assert float(loss[0]) == math.inf and math.isnan(float(loss[1])) and bool(torch.isnan(d[1]).all())
    assert bool(torch.isfinite(d[0]).all()) and abs(float(d[0, 10]) + 0.5) < 1e-6      # -pt of the masked token
    for i in (2, 3, 4):
        l, want = kd_row(x[i], ids[i], lp[i], 1.0)
        assert close(loss[i], l)
        assert float((d[i].cpu().double() - want).abs().max()) <= TOL
    assert abs(float(loss[4])) < 1e-6 and float(d[4].abs().max()) < 1e-6               # no teacher token: one full bin


@pytest.mark.parametrize("device", DEVICES)
def test_kd_in_place_and_strided_output(device):
    g = torch.Generator().manual_seed(5)
    for V in (1000, 4099, 60001):
        for dtype in DTYPES:
            x = rows(g, 3, V, dtype, device, V + 5, 1)
            ids, lp = teacher(g, x, 20, 1.0, device)
            w = torch.rand(3, generator=g).to(device)
            _, want = distill.kd_topk_grad(x, ids, lp, w)
            out = torch.full((3, V + 3), 7.0, dtype=dtype, device=device)
            distill.kd_topk_grad(x, ids, lp, w, out=out[:, 1:V + 1])
            assert torch.equal(out[:, 1:V + 1], want) and bool((out[:, 0] == 7).all()) and bool((out[:, V + 1:] == 7).all())
            buf = x.as_strided((3, V + 5), (V + 5, 1), 0).clone()          # storage around the rows
            y = buf.as_strided((3, V), (V + 5, 1), 1)
            around = buf.clone()
            distill.kd_topk_grad(y, ids, lp, w, out=y)
            assert torch.equal(y, want)
            around.as_strided((3, V), (V + 5, 1), 1).copy_(want)
            assert torch.equal(buf, around)                                # nothing outside the rows was written


def differences(f, x, g, h):
    """d (f(x) . g) / dx by central differences of an fp32 function."""
    d = torch.zeros(x.shape, dtype=torch.float64)
    for i in range(x.numel()):
        e = torch.zeros(x.numel(), device=x.device)
        e[i] = h
        e = e.view(x.shape)
        d.view(-1)[i] = ((f(x + e) - f(x - e)).double() * g.double()).sum().cpu() / (2 * h)
    return d


@pytest.mark.parametrize("device", DEVICES)
def test_gradients_agree_with_differences(device):
    """h = 1/64: truncation h^2 |f'''| / 6 <= 4e-5 for |f'''| <= 1 on losses of unit weight, rounding of a loss below 4
    (2 ulp, 1e-6) over 2 h 3e-5; three of each: 3e-4. min(q, p) has kinks: a change of at most h of one logit moves
    log q - log p by at most h, so rows whose every |log q - log p| exceeds 2 h see none."""
    g = torch.Generator().manual_seed(11)
    x = torch.randn(3, 17, generator=g).to(device)
    ids, lp = teacher(g, x, 4, 1.0, device)
    w = torch.tensor([1.0, 0.5, 0.25], device=device)
    _, d = distill.kd_topk_grad(x, ids, lp, w)
    want = differences(lambda v: distill.kd_topk(v, ids, lp), x, w, 1 / 64)
    assert float((d.cpu().double() - want).abs().max()) <= 3e-4
    y = x + torch.where(torch.rand(3, 17, generator=g).to(device) < 0.5, -0.7, 0.7)
    far = (torch.log_softmax(x, -1) - torch.log_softmax(y, -1)).abs().min()
    assert float(far) > 2 / 64
    z = x.clone().requires_grad_()
    a, k = distill.accept_kl(z, y)
    d, = torch.autograd.grad((a, k), z, (w, -0.5 * w))
    want = differences(lambda v: distill.accept_kl(v, y)[0] - 0.5 * distill.accept_kl(v, y)[1], x, w, 1 / 64)
    assert float((d.cpu().double() - want).abs().max()) <= 3e-4


# ------------------------------------------------------------------------------------------------- acceptance and KL
def check_accept(q, p, T, g):
    n, V = q.shape
    ga, gk = torch.randn(n, generator=g), torch.rand(n, generator=g)
    z = q.detach().requires_grad_()
    alpha, kl = distill.accept_kl(z, p, temperature=T)
    d, = torch.autograd.grad((alpha, kl), z, (ga.to(q.device), gk.to(q.device)))
    a2, k2 = distill.accept_kl(q, p, temperature=T)
    assert torch.equal(a2, alpha.detach()) and torch.equal(k2, kl.detach()) and d.dtype == q.dtype
    for i in range(n):
        a, k, da, dk = accept_row(q[i], p[i], T)
        assert close(alpha[i], a) and close(kl[i], k), (i, alpha[i], a, kl[i], k)
        want = float(ga[i]) * da + float(gk[i]) * dk
        lq, lp = log_p(q[i], T), log_p(p[i], T)
        size = torch.zeros(V, dtype=torch.float64) if lq is None or lp is None else lq.exp() + lp.exp()
        err = (d[i].cpu().double() - want).abs()
        lim = 2 * TOL * (abs(float(ga[i])) + float(gk[i])) / T * size + EPS[q.dtype] * want.abs() + 6e-8
        if lq is not None and lp is not None:      # at a tie within fp32 either subgradient is right
            lim = lim + torch.where((lq - lp).abs() <= TOL, abs(float(ga[i])) / T * lq.exp(), 0.0)
        assert bool((err <= lim).all()), (i, float((err - lim).max()))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=IDS)
def test_accept_and_kl(shape, dtype, device):
    n, V, ld, off = shape
    g = torch.Generator().manual_seed(V + 2)
    for T, off_p in ((1.0, off), (0.7, off + 1), (2.0, 0)):   # rows of draft and target starting on other boundaries
        q = rows(g, n, V, dtype, device, ld, off)
        p = rows(g, n, V, dtype, device, (ld or V) + (2 if off_p != off else 0), off_p)
        check_accept(q, p, T, g)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("how", ["inf", "low"])
def test_accept_masked_equal_and_shared_rows(how, device):
    g = torch.Generator().manual_seed(9)
    for V in (5, 1000, 40001):
        for dtype in DTYPES:
            q, p = rows(g, 8, V, dtype, device), rows(g, 8, V, dtype, device)
            mask_some(g, p, how)
            check_accept(q, p, 1.0, g)                         # the draft gives mass to tokens that the target masks
            q = torch.where(p.float() <= -1e30, p, q)
            check_accept(q, p, 1.0, g)                         # one mask for both
            check_accept(p, p.clone(), 1.0, g)                 # the same distribution: alpha 1, kl 0, no gradient
            check_accept(q, p[:1].expand(8, V), 1.0, g)        # one target row for all
    q, p = torch.zeros(1, 4, device=device), torch.zeros(1, 4, device=device)
    q[0, 1] = NINF
    alpha, kl = distill.accept_kl(q, p)                        # a token of the target that the draft cannot give
    assert abs(float(alpha) - 0.75) < TOL and float(kl) == math.inf
    p[0, 0] = float("nan")
    assert math.isnan(float(distill.accept_kl(q, p)[0])) and math.isnan(float(distill.accept_kl(q, p)[1]))


# ------------------------------------------------------------------------------------------------- verification
def verify_inputs(g, B, k, V, dtype, device, ld=None, temp=0.8):
    p = rows(g, B * (k + 1), V, dtype, device, ld).as_strided((B, k + 1, V), ((k + 1) * (ld or V), ld or V, 1))
    q = (p[:, :k].float() + torch.randn(B, k, V, generator=g).to(device)).to(dtype)
    if k:
        drafts = torch.softmax(q.float() / 0.8, -1).reshape(B * k, V).cpu().multinomial(1, generator=g).view(B, k)
    else:
        drafts = torch.zeros(B, 0, dtype=torch.int64)
    temps = torch.full((B,), temp)
    temps[1::3] = 0.0
    seeds = torch.randint(-(1 << 62), 1 << 62, (B,), generator=g)
    steps = torch.randint(0, 100000, (B,), generator=g)
    return p, q, drafts.to(device), temps.to(device), seeds.to(device), steps.to(device)


def check_verify(p, drafts, temps, seeds, steps, q=None, n_draft=None):
    acc, nxt = sampling.speculative_verify(p, drafts, temps, seeds, steps, draft_logits=q, n_draft=n_draft)
    assert acc.dtype == nxt.dtype == torch.int32
    B, k = drafts.shape
    want = []
    for b in range(B):
        n = k if n_draft is None else min(k, max(0, int(n_draft[b])))
        want.append(verify_row(p[b], drafts[b].tolist()[:n], float(temps[b]), int(seeds[b]), int(steps[b]),
                               None if q is None else q[b]))
    assert list(zip(acc.tolist(), nxt.tolist())) == want
    return acc


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("B,k,V,ld", [(1, 0, 1, None), (3, 1, 2, 5), (7, 3, 31, None), (6, 2, 4099, 4101),
                                      (4, 8, 257, None), (3, 3, 32768, None), (2, 1, 151935, None), (1, 2, 152064, None)])
def test_verify_follows_the_rule(B, k, V, ld, dtype, device):
    g = torch.Generator().manual_seed(V + k)
    for rep in range(3):
        p, q, drafts, temps, seeds, steps = verify_inputs(g, B, k, V, dtype, device, ld)
        n = torch.randint(0, k + 1, (B,), generator=g).to(torch.int32).to(device)
        check_verify(p, drafts, temps, seeds, steps)
        check_verify(p, drafts.to(torch.int32), temps, seeds, steps, n_draft=n)
        check_verify(p, drafts, temps, seeds, steps, q)
        check_verify(p, drafts, temps, seeds, steps, q, n)


@pytest.mark.parametrize("device", DEVICES)
def test_verify_masks_bad_drafts_and_empty_residuals(device):
    g = torch.Generator().manual_seed(4)
    for V in (6, 3000, 33001):
        for how in ("inf", "low"):
            p, q, drafts, temps, seeds, steps = verify_inputs(g, 9, 2, V, torch.float32, device)
            p, q = p.contiguous(), q.contiguous()
            mask_some(g, p.view(27, V), how)
            mask_some(g, q.view(18, V), how)
            drafts[0, 0], drafts[1, 0], drafts[2, 1], drafts[3, 0] = -1, V, V + (1 << 33), -(1 << 40)
            check_verify(p, drafts, temps, seeds, steps)
            check_verify(p, drafts, temps, seeds, steps, q)
    p = torch.zeros(2, 2, 5, device=device)
    q = torch.zeros(2, 1, 5, device=device)
    p[:, 0] = NINF
    p[:, 0, 3] = 1.0
    q[0, 0, 0] = 50.0                               # a draft that the target masks: rejected, token 3 is all that is left
    d = torch.tensor([[0], [3]], device=device)
    t, s = torch.ones(2, device=device), torch.arange(2, device=device)
    acc, nxt = sampling.speculative_verify(p, d, t, s, s, draft_logits=q)
    assert acc.tolist() == [0, 1] and int(nxt[0]) == 3
    acc, nxt = sampling.speculative_verify(p, d, t, s, s)
    assert acc.tolist() == [0, 1] and int(nxt[0]) == 3
    p[:, 0] = NINF
    acc, nxt = sampling.speculative_verify(p, d, t, s, s)
    assert acc.tolist() == [0, 0] and nxt.tolist() == [-1, -1]
    acc, nxt = sampling.speculative_verify(p, d, 0 * t, s, s)
    assert acc.tolist() == [0, 0] and nxt.tolist() == [-1, -1]


@pytest.mark.parametrize("device", DEVICES)
def test_verify_equals_speculative_accept_for_point_mass_drafts(device):
    g = torch.Generator().manual_seed(6)
    p, _, drafts, temps, seeds, steps = verify_inputs(g, 12, 3, 500, torch.float32, device)
    want = sampling.speculative_accept(p.cpu(), drafts.cpu(), temps.tolist(), seeds.tolist(), steps.tolist())
    acc, nxt = sampling.speculative_verify(p, drafts, temps, seeds, steps)
    assert (acc.tolist(), nxt.tolist()) == want


@pytest.mark.parametrize("device", DEVICES)
def test_verify_preserves_the_target_distribution(device):
    """Drafts drawn from q, verified against p: the first emitted token is distributed as p. The total variation of n
    draws over V = 6 tokens is about 0.5 sum_v sqrt(2 p_v (1 - p_v) / (pi n)) <= 0.9 / sqrt(n); four times that."""
    n = 3000 if device == "cpu" else 40000
    V, T = 6, 0.8
    lp = torch.tensor([1.0, 0.2, -0.5, 2.0, 0.0, 1.5])
    lq = torch.tensor([0.0, 1.2, 0.5, 1.0, 1.0, -1.5])
    g = torch.Generator().manual_seed(8)
    drafts = torch.softmax(lq / T, 0).multinomial(n, replacement=True, generator=g)[:, None].to(device)
    p = torch.stack([lp, torch.zeros(V)])[None].expand(n, 2, V).to(device)
    q = lq[None, None].expand(n, 1, V).to(device)
    threads = torch.get_num_threads()
    torch.set_num_threads(1)
    try:
        acc, nxt = sampling.speculative_verify(p, drafts, torch.full((n,), T, device=device),
                                               torch.arange(n, device=device), torch.zeros_like(drafts[:, 0]),
                                               draft_logits=q)
    finally:
        torch.set_num_threads(threads)
    first = torch.where(acc == 1, drafts[:, 0], nxt)
    tv = 0.5 * (torch.bincount(first.cpu(), minlength=V) / n - torch.softmax(lp / T, 0)).abs().sum()
    assert float(tv) < 3.6 / math.sqrt(n)


# ------------------------------------------------------------------------------------------------- refusals, edges
def raises(f, *a, **kw):
    with pytest.raises((ValueError, RuntimeError)):
        f(*a, **kw)


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    x = torch.zeros(2, 10, device=device)
    ids, lp = torch.zeros(2, 3, dtype=torch.int64, device=device), torch.zeros(2, 3, device=device)
    w = torch.ones(2, device=device)
    raises(distill.teacher_topk, x, 0)
    raises(distill.teacher_topk, x, 129)
    raises(distill.teacher_topk, x[0], 3)
    raises(distill.teacher_topk, x.double(), 3)
    raises(distill.teacher_topk, x.long(), 3)
    raises(distill.teacher_topk, x, 3, temperature=0.0)
    raises(distill.teacher_topk, x, 3, temperature=float("nan"))
    raises(distill.teacher_topk, x[:, :0], 3)
    raises(distill.kd_topk, x, ids[:1], lp)
    raises(distill.kd_topk, x, ids, lp[:, :2])
    raises(distill.kd_topk, x, ids.float(), lp)
    raises(distill.kd_topk, x, ids[:, :0], lp[:, :0])
    raises(distill.kd_topk, x, ids.repeat(1, 50), lp.repeat(1, 50))
    raises(distill.kd_topk, x, ids, lp, temperature=-1.0)
    raises(distill.kd_topk_grad, x, ids, lp, w[:1])
    raises(distill.kd_topk_grad, x, ids, lp, w, out=x.half())
    raises(distill.kd_topk_grad, x, ids, lp, w, out=x[:1])
    raises(distill.kd_topk_grad, x, ids, lp, w, out=torch.zeros(10, 2, device=device).t())
    raises(distill.accept_kl, x, x[:1])
    raises(distill.accept_kl, x, x.half())
    raises(distill.accept_kl, x, x, temperature=1e7)
    lg = torch.zeros(2, 3, 10, device=device)
    d, s = torch.zeros(2, 2, dtype=torch.int64, device=device), torch.zeros(2, dtype=torch.int64, device=device)
    v = sampling.speculative_verify
    raises(v, lg[0], d, w, s, s)
    raises(v, lg, d[:, :1], w, s, s)
    raises(v, lg, d.float(), w, s, s)
    raises(v, lg, d, w.double(), s, s)
    raises(v, lg, d, w, s.int(), s)
    raises(v, lg, d, w, s, s[:1])
    raises(v, lg, d, w, s, s, draft_logits=lg)
    raises(v, lg, d, w, s, s, draft_logits=lg[:, :2].half())
    raises(v, lg, d, w, s, s, n_draft=s)


@pytest.mark.gpu
def test_refuses_tensors_of_another_device():
    x = torch.zeros(2, 10, device="cuda")
    raises(distill.kd_topk, x, torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2, 3))
    raises(distill.kd_topk_grad, x, torch.zeros(2, 3, dtype=torch.int64, device="cuda"), torch.zeros(2, 3, device="cuda"),
           torch.ones(2))
    raises(distill.accept_kl, x, x.cpu())
    lg, d = torch.zeros(2, 3, 10, device="cuda"), torch.zeros(2, 2, dtype=torch.int64)
    raises(sampling.speculative_verify, lg, d, torch.ones(2), d[:, 0], d[:, 0])


@pytest.mark.parametrize("device", DEVICES)
def test_no_rows_and_other_strides(device):
    e = torch.zeros(0, 10, device=device)
    none = torch.zeros(0, device=device)
    assert distill.teacher_topk(e, 3)[0].shape == (0, 3)
    ids, lp = torch.zeros(0, 3, dtype=torch.int64, device=device), torch.zeros(0, 3, device=device)
    assert distill.kd_topk(e, ids, lp).shape == (0,)
    assert distill.kd_topk_grad(e, ids, lp, none)[1].shape == (0, 10)
    assert distill.accept_kl(e, e)[1].shape == (0,)
    z = e[:, 0].long()
    acc, nxt = sampling.speculative_verify(torch.zeros(0, 3, 10, device=device), torch.zeros(0, 2, device=device).long(),
                                           none, z, z)
    assert acc.shape == nxt.shape == (0,)
    g = torch.Generator().manual_seed(2)
    x = rows(g, 700, 6, torch.float32, device).t()               # columns a row apart
    check_topk(x, 5, 1.0)
    ids, lp = teacher(g, x, 5, 1.0, device)
    check_kd(x, ids, lp, 1.0, torch.ones(6, device=device))
    check_accept(x, x.flip(0), 1.0, g)
    t = torch.ones(2, device=device)
    s = torch.arange(2, device=device)
    check_verify(rows(g, 60, 4, torch.float32, device).t().reshape(2, 2, 60).transpose(0, 1),
                 torch.zeros(2, 1, dtype=torch.int64, device=device), t, s, s)


@pytest.mark.gpu
def test_rows_past_32_bit_offsets():
    V, ld = 5000, (1 << 31) + 8
    buf = torch.empty(ld + V, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator().manual_seed(3)
    x = buf.as_strided((2, V), (ld, 1))
    x.copy_(rows(g, 2, V, torch.bfloat16, "cuda"))
    check_topk(x, 20, 1.0)
    ids, lp = teacher(g, x, 20, 1.0, "cuda")
    w = torch.rand(2, generator=g).cuda()
    check_kd(x, ids, lp, 1.0, w)
    check_accept(x, x.flip(0), 1.0, g)
    check_accept(x.flip(0).contiguous(), x, 1.0, g)
    _, want = distill.kd_topk_grad(x, ids, lp, w)
    y = x.unsqueeze(0)                                           # one sequence, its second position far away
    check_verify(y, torch.tensor([[int(x[0].float().argmax())]], device="cuda"), torch.ones(1, device="cuda"),
                 torch.tensor([5], device="cuda"), torch.tensor([7], device="cuda"))
    distill.kd_topk_grad(x, ids, lp, w, out=x)
    assert torch.equal(x, want)


@pytest.mark.gpu
def test_streams_and_graph_capture():
    """Calls run on the current stream and can be captured; a replay follows new inputs."""
    g = torch.Generator().manual_seed(12)
    x, y = rows(g, 40, 30001, torch.float32, "cuda"), rows(g, 40, 30001, torch.float32, "cuda")
    ids, lp = teacher(g, x, 20, 1.0, "cuda")
    w = torch.rand(40, generator=g).cuda()
    p, q, drafts, temps, seeds, steps = verify_inputs(g, 8, 3, 30001, torch.float32, "cuda")

    def everything():
        return [*distill.teacher_topk(x, 20), distill.kd_topk(x, ids, lp), *distill.kd_topk_grad(x, ids, lp, w),
                *distill.accept_kl(x, y), *sampling.speculative_verify(p, drafts, temps, seeds, steps),
                *sampling.speculative_verify(p, drafts, temps, seeds, steps, draft_logits=q)]

    want = everything()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        on_side = everything()
    torch.cuda.current_stream().wait_stream(s)
    for a, b in zip(want, on_side):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = everything()
    x2, p2 = x.roll(1, 0), p.roll(1, 0).contiguous()
    x.copy_(x2)
    p.copy_(p2)
    want = everything()
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert torch.equal(a, b)
