"""The gradient of accept_kl where one token has nearly all the mass of both sides, and where both sides agree: A = sum q h
must count a token as its own h does, or the surest tokens get a gradient of full size.

Tolerance of d alpha / d z_v = g q_v (h_v - A) / T. A probability is off by 3.1e-5 of itself (test_vocab_ops.py), so q_v (h_v -
A) by 3.1e-5 q_v (1 - q_v) from q_v itself and as much again from A's other terms: TOL = 1e-4 times q_v (1 - q_v) covers both.
A is a sum of at most 2^18 terms of total at most 1, added over a tree whose longest chain is below 2^10 additions of partial
sums: 2^-16 would be its worst case, and rounding errors of random sign keep it below sqrt(2^10) 2^-24 < 2^-18: 2^-18 q_v. Where
log q and log p lie closer than fp32 forms them (within 2^-17 of each other: 64 in fp32 is 2^-18 coarse, each side), a token may
be taken on either side of q = p, or at it, but by h and A alike. That moves its own gradient by at most q (1 - q), since
h - A without its own term lies in [0, 1 - q] or [-(1 - q), 0], and that of any other token v by at most q_v q."""
import pytest
import torch

from arcagi2_flashnext_dots3_b200.ops import distill

TOL = 1e-4
SUM = 2.0 ** -18
TIE = 2.0 ** -17
EPS = {torch.float32: 2.0 ** -23, torch.float16: 2.0 ** -10, torch.bfloat16: 2.0 ** -7}
NINF = float("-inf")
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def alpha_gradient(q, p, T):
    """(q, log q - log p, d alpha) of all rows in 64 bits, equal tokens counted half."""
    z = [torch.where(x.cpu().double() <= -1e30, NINF, x.cpu().double()) / T for x in (q, p)]
    lq, lp = (torch.log_softmax(x, -1) for x in z)
    gap = torch.where((lq == NINF) & (lp == NINF), 0.0, lq - lp)
    h = (gap < 0).double() + 0.5 * (gap == 0).double()
    m = lq.exp()
    return m, gap, m * (h - (m * h).sum(-1, keepdim=True)) / T


def gradient(q, p, T, g):
    z = q.detach().requires_grad_()
    alpha, _ = distill.accept_kl(z, p, temperature=T)
    return torch.autograd.grad(alpha, z, g.to(q.device))[0].cpu().double()


def check(q, p, T, g, ties=True):
    d = gradient(q, p, T, g)
    m, gap, want = alpha_gradient(q, p, T)
    a = g.double()[:, None] / T
    near = torch.where((gap.abs() <= TIE) & (m > 0), m, 0.0) if ties else torch.zeros_like(m)
    moved = near * (1 - m) + m * (near.sum(-1, keepdim=True) - near)
    want = want * T * a
    lim = a.abs() * (TOL * m * (1 - m) + SUM * m + moved) + EPS[q.dtype] * want.abs() + 6e-8
    assert bool(((d - want).abs() <= lim).all()), float(((d - want).abs() - lim).max())
    # a softmax's gradient sums to 0; each element is rounded to its type
    off = d.sum(-1).abs()
    assert bool((off <= a[:, 0].abs() * SUM * 2 + (EPS[q.dtype] * d.abs() + 6e-8).sum(-1)).all()), float(off.max())


def sure(g, n, V, miss, top):
    """fp32 rows whose token `top` has probability about 1 - miss at T = 1."""
    z = torch.randn(n, V, generator=g)
    rest = z.scatter(1, top[:, None], NINF).logsumexp(1)
    return z.scatter(1, top[:, None], (rest + torch.log1p(-miss.double()).float() - miss.log())[:, None])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("V", [2, 257, 32768, 50001])
def test_rows_where_both_sides_are_sure(V, dtype, device):
    g = torch.Generator().manual_seed(V)
    for T in (1.0, 0.7):
        for lo in (1e-4, 2e-5, 1e-6, 1e-7, 6e-9, 1e-9):
            n = 24
            top = torch.randint(0, V, (n,), generator=g)
            miss = lo * torch.exp(torch.rand(2, n, generator=g) - 0.5)
            miss[1, ::3] = miss[0, ::3]                       # equally sure, of other tokens beside it
            miss[1, 1::3] *= 30                               # the target less sure
            q, p = (sure(g, n, V, miss[i], top).mul(T).to(dtype).to(device) for i in (0, 1))
            check(q, p, T, torch.randn(n, generator=g))
            check(p, q, T, torch.randn(n, generator=g))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_equal_rows_have_no_gradient(dtype, device):
    """Equal sides are equal in every step of fp32 too, so nothing is allowed for ties."""
    g = torch.Generator().manual_seed(2)
    for V in (1, 2, 31, 4099, 32768, 151935):
        for T in (1.0, 0.7, 2.0):
            x = (torch.randn(3, V, generator=g) * 4).to(dtype).to(device)
            if V > 2:
                x[1, ::2] = NINF
                x[2] = NINF
                x[2, V // 2] = 1.5
            check(x, x.clone(), T, torch.ones(3), ties=False)
            if V > 1:                                          # rows on another 16-byte boundary, cut into the same units
                y = torch.zeros(3, V + 1, dtype=dtype, device=device)
                y[:, 1:] = x
                check(x, y[:, 1:], T, torch.ones(3), ties=False)
    one = torch.tensor([[3.3]], dtype=dtype, device=device)
    check(one, one - 0.6, 1.0, torch.ones(1), ties=False)      # one token: probability 1 on both sides


@pytest.mark.parametrize("device", DEVICES)
def test_equal_tokens_beside_others(device):
    """Two tokens change places, the others are equal: both sums are the same, so the others are ties and count half."""
    q = torch.tensor([[1.0, 2.0, 0.5, -0.25], [0.0, 9.0, 9.0, 9.0], [7.0, 0.0, 12.0, 0.0]], device=device)
    p = q[:, [1, 0, 2, 3]].contiguous()
    for T in (1.0, 0.7):
        check(q, p, T, torch.ones(3), ties=False)
        d = gradient(q, p, T, torch.ones(3))
        m, _, _ = alpha_gradient(q, p, T)
        # token 1 of the first row lies above the target, token 0 below it
        a = m[0, 0] + 0.5 * (m[0, 2] + m[0, 3])
        assert abs(float(d[0, 0] - m[0, 0] * (1 - a) / T)) <= TOL and abs(float(d[0, 1] + m[0, 1] * a / T)) <= TOL


@pytest.mark.gpu
def test_training_and_evaluation_give_one_alpha():
    """The forward with the backward's statistics and the one without return the same bits."""
    g = torch.Generator().manual_seed(4)
    for V in (1000, 32768, 151936):
        q, p = ((torch.randn(5, V, generator=g) * 4).cuda() for _ in range(2))
        a, k = distill.accept_kl(q, p)
        b, l = distill.accept_kl(q.clone().requires_grad_(), p)
        assert torch.equal(a, b.detach()) and torch.equal(k, l.detach())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("shift", [0.0, 100.0, -1000.0])
def test_alpha_keeps_its_digits(shift, device):
    """alpha of sure and of flat rows, whatever constant the logits carry: each probability is an exponential of z - max, so
    alpha is off by the rounding of the exponentials' arguments, at most 2^-20 for arguments below 16, of the instruction (2
    ulp) and of the sums: 2^-18 of itself covers them. (Smaller probabilities have a larger relative error and no weight.)"""
    g = torch.Generator().manual_seed(6)
    for V in (2, 300, 32768, 50001):
        n = 60
        top = torch.randint(0, V, (n,), generator=g)
        miss = torch.exp(torch.rand(2, n, generator=g) * -18)
        q, p = (sure(g, n, V, miss[i].clamp_max(0.9), top) + shift for i in (0, 1))
        q[::4] = torch.randn(15, V, generator=g) + shift
        p[::4] = q[::4] + 0.5 * torch.randn(15, V, generator=g)
        q[1::4] = p[1::4] + 0.001 * torch.randn(15, V, generator=g)
        a, _ = distill.accept_kl(q.to(device), p.to(device))
        want = torch.minimum(torch.log_softmax(q.double(), -1), torch.log_softmax(p.double(), -1)).exp().sum(-1)
        assert float((a.cpu().double() - want).abs().div(want).max()) <= 2.0 ** -18
