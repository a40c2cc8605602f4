"""Vocabulary-row operators where their kernels take another course: the distillation gradient of more logits than L2
holds (rows over one block, over clusters, with shares that fit into shared memory and that do not), draws from a residual
of little mass, and long runs of equal logits.

Tolerances are those of the small cases (test_vocab_ops.py): TOL for values, and for a gradient w (a - b) with a and b at
most one probability each TOL * w / T * (a + b), scaled where the student's tail is below the teacher's, plus the rounding
to the output type."""
import pytest
import torch

from arcagi2_flashnext_dots3_b200.ops import distill, sampling

TOL = 1e-4
EPS = {torch.float32: 2.0 ** -23, torch.float16: 2.0 ** -10, torch.bfloat16: 2.0 ** -7}
NINF = float("-inf")


def kd_rows(x, ids, lp, T):
    """The 64-bit statement for a block of rows: loss, gradient, probabilities, teacher mass and scale per row."""
    n, V = x.shape
    z = x.double()
    z = torch.where(z <= -1e30, NINF, z) / T
    empty = (z == NINF).all(1)
    ls = torch.where(empty[:, None], NINF, z - torch.logsumexp(torch.where(empty[:, None], 0.0, z), 1, keepdim=True))
    same = (ids[:, :, None] == ids[:, None, :]).tril(-1).any(-1)
    ok = (ids >= 0) & (ids < V) & ~same
    at = ids.long().clamp(0, V - 1)
    pt = torch.where(ok, lp.double().exp(), 0.0)
    s = ls.gather(1, at)
    p = ls.exp()
    mass = torch.zeros(n, V, dtype=torch.float64, device=x.device).scatter_add_(1, at, pt)
    inside = torch.zeros(n, V, dtype=torch.float64, device=x.device).scatter_add_(1, at, ok.double()) > 0
    tail = torch.where(inside, 0.0, p).sum(1)
    tt, ts = (1 - pt.sum(1)).clamp_min(1e-8), tail.clamp_min(1e-8)
    loss = tt * (tt.log() - ts.log()) + torch.where(pt > 0, pt * (lp.double() - s), 0.0).sum(1)
    c = torch.where(ok, -pt + torch.where(tail >= 1e-8, tt / ts, 0.0)[:, None] * s.exp(), 0.0)
    d = (-p * c.sum(1, keepdim=True)).scatter_add_(1, at, c) / T
    return torch.where(empty, 0.0, loss), torch.where(empty[:, None], 0.0, d), p, mass, (tt / ts).clamp_min(1.0)


CASES = [(270, 151935, 5, 3, torch.float32, 20, 1.0), (500, 152064, 0, 0, torch.bfloat16, 20, 2.0),
         (40, 1 << 20, 0, 0, torch.float32, 128, 1.0), (2000000, 37, 0, 1, torch.bfloat16, 3, 1.0),
         (66000, 1001, 6, 1, torch.bfloat16, 7, 0.7), (2100, 32000, 0, 0, torch.float16, 50, 1.0),
         (150, 303871, 1, 2, torch.bfloat16, 20, 1.0), (300, 151936, 0, 0, torch.float32, 20, 1.0)]


@pytest.mark.gpu
@pytest.mark.parametrize("n,V,pad,off,dtype,K,T", CASES, ids=lambda v: str(v))
def test_gradient_of_more_logits_than_l2(n, V, pad, off, dtype, K, T):
    g = torch.Generator(device="cuda").manual_seed(V)
    if n * V * torch.tensor([], dtype=dtype).element_size() <= torch.cuda.get_device_properties(0).L2_cache_size:
        n = torch.cuda.get_device_properties(0).L2_cache_size // (V * torch.tensor([], dtype=dtype).element_size()) + 1
    buf = torch.empty(off + n * (V + pad), dtype=dtype, device="cuda")
    x = buf.as_strided((n, V), (V + pad, 1), off)
    for i in range(0, n, 4096):
        x[i:i + 4096] = (torch.randn(min(4096, n - i), V, generator=g, device="cuda") * 4).to(dtype)
    at = torch.randint(0, V, (n, K), generator=g, device="cuda")
    lp = torch.log_softmax(torch.randn(n, K + 1, generator=g, device="cuda") * 2, -1)[:, :K].contiguous()
    at[::5, K // 2:] = -1                                            # fewer teacher tokens
    if K > 2:
        at[1::7, 2] = at[1::7, 0]                                    # repeated
        at[2::9, 1] = V + 3                                          # outside
    x[3::11, : V // 3] = NINF
    hidden = torch.gather(x, 1, at.clamp(0, V - 1)) == NINF
    at[hidden] = -1                                                  # an infinite loss is another test's
    x[n // 2] = NINF                                                 # nothing left
    at[n // 2] = -1
    w = torch.rand(n, generator=g, device="cuda") + 0.5
    loss, d = distill.kd_topk_grad(x, at, lp, w, temperature=T)
    step = max(1, (1 << 24) // V)
    for i in range(0, n, step):
        e = slice(i, min(n, i + step))
        want, grad, p, mass, scale = kd_rows(x[e], at[e], lp[e], T)
        assert bool(((loss[e].double() - want).abs() <= TOL * (1 + want.abs())).all()), i
        we = w[e].double()[:, None]
        lim = TOL * we / T * scale[:, None] * (p + mass) + EPS[dtype] * (we * grad).abs() + 6e-8
        assert bool(((d[e].double() - we * grad).abs() <= lim).all()), i
    around = buf.clone()
    loss2, same = distill.kd_topk_grad(x, at, lp, w, temperature=T, out=x)
    assert same.data_ptr() == x.data_ptr() and torch.equal(loss2, loss) and torch.equal(x, d)
    around.as_strided((n, V), (V + pad, 1), off).copy_(d)
    assert torch.equal(buf.view(torch.uint8), around.view(torch.uint8))      # nothing outside the rows was written


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("V", [50, 3001, 152064])
@pytest.mark.parametrize("moved", [1e-1, 1e-3, 2e-5])
def test_draw_from_a_residual_of_little_mass(V, moved, device):
    """Target and draft agree but for one token's mass `moved`, which the target gives to two others in equal parts. That
    token is drafted, and always rejected; the next one must be one of the two: the one that the race picks, where the two
    times differ by more than what rounding of the probabilities can do. Half of `moved` as a difference of probabilities
    of 0.25 is off by at most 2 * 2^-24 * 8 / moved of itself, under 5% for 2e-5. Rounding may leave the other tokens a
    residual of some 2^-24 of their mass, a share of the residual of 8 * 2^-24 / moved: 2.4%, or 2 draws of 64, allowed 8."""
    B, d, a, b = 64, 3, V - 7, V // 2
    q = torch.full((V,), 0.5 / (V - 3), dtype=torch.float64)
    q[a] = q[b] = 0.25 - moved / 2
    q[d] = moved
    p = q.clone()
    p[d] = 0
    p[a] = p[b] = 0.25
    zp = p.log().float()[None, None].repeat(B, 2, 1).to(device)
    zq = q.log().float()[None, None].repeat(B, 1, 1).to(device)
    seeds = torch.arange(B) * 7919 + 13
    steps = torch.arange(B) * 3
    acc, nxt = sampling.speculative_verify(zp, torch.full((B, 1), d).to(device), torch.ones(B, device=device),
                                           seeds.to(device), steps.to(device), draft_logits=zq)
    assert acc.tolist() == [0] * B
    compared = right = 0
    for i in range(B):
        u = torch.from_numpy(sampling.uniform(int(seeds[i]), int(steps[i]), [a, b])).double()
        ta, tb = (-torch.log(u)).tolist()
        if abs(ta - tb) <= 0.1 * max(ta, tb):
            continue
        compared += 1
        right += int(nxt[i]) == (a if ta < tb else b)
    assert compared >= 40 and right >= compared - 8
    if moved > 1e-2:
        assert right >= compared - 1


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_top_tokens_among_many_equal_logits(dtype):
    """More tokens at the bound than a block lists, over one unit of a row and over many: lowest ids first."""
    for V in (1000, 20000, 151936):
        x = torch.zeros(3, V, device="cuda", dtype=dtype)
        x[1, V // 2:] = 1.0
        x[1, 5] = 2.0
        x[2, ::2] = NINF
        for k in (1, 20, 128):
            ids, lp = distill.teacher_topk(x, k)
            assert ids[0].tolist() == list(range(k))
            assert ids[1].tolist() == ([5] + list(range(V // 2, V // 2 + k)))[:k]
            assert ids[2].tolist() == list(range(1, 2 * k, 2))
            want = torch.log_softmax(x.double(), -1).gather(1, ids.long())
            assert float((lp.double() - want).abs().max()) <= TOL


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_autograd_edges(device):
    """Strided logits, an unused output, mixed precision of the incoming gradient, no graph under no_grad, and an error in
    place of a second derivative."""
    g = torch.Generator().manual_seed(8)
    base = torch.randn(40, 6, generator=g).to(device).requires_grad_()
    x = base.t()                                                         # [6, 40], not unit stride
    ids = torch.randint(0, 40, (6, 4), generator=g).to(device)
    lp = torch.log_softmax(torch.randn(6, 5, generator=g), -1)[:, :4].to(device)
    y = torch.randn(6, 40, generator=g).to(device)
    _, want = distill.kd_topk_grad(x, ids, lp, torch.ones(6, device=device))
    got, = torch.autograd.grad(distill.kd_topk(x, ids, lp).sum(), base)
    assert float((got.t() - want).abs().max()) <= 1e-6
    both, = torch.autograd.grad(sum(t.sum() for t in distill.accept_kl(x, y)), base)
    one, = torch.autograd.grad(distill.accept_kl(x, y)[0].sum(), base)
    other, = torch.autograd.grad(distill.accept_kl(x, y)[1].sum(), base)
    assert float((both - one - other).abs().max()) <= 1e-6
    h = x.detach().to(torch.bfloat16).requires_grad_()
    (distill.kd_topk(h, ids, lp).double() * 2).sum().backward()
    assert h.grad.dtype == torch.bfloat16 and bool(torch.isfinite(h.grad).all())
    with torch.no_grad():
        assert not distill.kd_topk(x, ids, lp).requires_grad and not distill.accept_kl(x, y)[0].requires_grad
    assert not distill.kd_topk(x.detach(), ids, lp).requires_grad
    for loss in (distill.kd_topk(x, ids, lp).sum(), distill.accept_kl(x, y)[1].sum()):
        d, = torch.autograd.grad(loss, base, create_graph=True)
        with pytest.raises(RuntimeError):
            d.square().sum().backward()
    z = y.clone().requires_grad_()
    t = z * 1.0
    loss = distill.accept_kl(t, y)[1].sum()
    with torch.no_grad():
        t.add_(1.0)                                                      # what backward reads was overwritten
    with pytest.raises(RuntimeError):
        loss.backward()


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_a_gradient_written_over_saved_logits_is_noticed(device):
    """kd_topk_grad over logits that another function has saved for its backward: that backward raises."""
    g = torch.Generator().manual_seed(9)
    x = torch.randn(3, 50, generator=g).to(device).requires_grad_()
    z = x * 2.0
    ids = torch.randint(0, 50, (3, 4), generator=g).to(device)
    lp = torch.full((3, 4), -2.0, device=device)
    loss = distill.accept_kl(z, z.detach().flip(0))[0].sum()
    with torch.no_grad():
        distill.kd_topk_grad(z, ids, lp, torch.ones(3, device=device), out=z.detach())
    with pytest.raises(RuntimeError):
        loss.backward()
