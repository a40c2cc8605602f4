"""The distillation gradient of students that are sure of a teacher's token: at a teacher's token it is w / T ((tt + sum pt) ps -
pt), without the ratio of the tails that the chain of its derivation goes through (w / T (ps sum pt - pt) where the student's
tail is below its floor), and must not carry that ratio's rounding.

Tolerance. Probabilities are off by 3.1e-5 of themselves (test_vocab_ops.py): TOL w / T (ps + pt) at a teacher's token, and
TOL w / T p_v (1 + tt / ts) at the others, whose gradient is w / T p_v (tt + sum pt - tt / ts)."""
import pytest
import torch

from arcagi2_flashnext_dots3_b200.ops import distill

TOL = 1e-4
EPS = {torch.float32: 2.0 ** -23, torch.float16: 2.0 ** -10, torch.bfloat16: 2.0 ** -7}
NINF = float("-inf")
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def students(g, n, V, K, tail, T, dtype):
    """Rows with about `tail` of their mass outside the K teacher tokens, and nearly all the rest on one or two of them."""
    z = torch.randn(n, V, generator=g)
    ids = torch.stack([torch.randperm(V, generator=g)[:K] for _ in range(n)])
    z.scatter_(1, ids, NINF)
    out = z.logsumexp(1)
    inside = torch.randn(n, K, generator=g) - 8.0
    inside[:, 0] = 2.0
    inside[::2, 1] = 1.0
    inside = inside - inside.logsumexp(1, keepdim=True) + (out + torch.log1p(-tail).float() - tail.log().float())[:, None]
    return z.scatter(1, ids, inside).mul(T).to(dtype), ids


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("n,V", [(12, 40), (12, 4099), (6, 32768), (400, 151935)])
def test_gradient_of_a_sure_student(n, V, dtype, device):
    """400 x 151935 holds more than L2 in fp32: the form whose clusters look twice."""
    if device == "cpu" and n > 100:
        n = 4
    g = torch.Generator().manual_seed(V)
    for K, T in ((5, 1.0), (20, 0.7)):
        tail = torch.tensor([1e-3, 1e-5, 1e-6, 1e-7, 1e-9, 1e-11], dtype=torch.float64)[torch.arange(n) % 6]
        if T != 1.0:
            tail = tail.clamp_min(1e-7)
        x, ids = students(g, n, V, K, tail, T, dtype)
        lp = torch.log_softmax(torch.randn(n, K + 1, generator=g), -1)[:, :K].contiguous()
        w = torch.rand(n, generator=g) + 0.5
        x, ids, lp, w = (t.to(device) for t in (x, ids, lp, w))
        z = torch.nn.Parameter(x.clone())
        first = distill.kd_topk_grad(x, ids, lp, w, temperature=T)[1]
        second, = torch.autograd.grad(distill.kd_topk(z, ids, lp, temperature=T), z, w)
        for i in range(0, n, 50):
            e = slice(i, i + 50)
            ls = torch.log_softmax(x[e].double() / T, -1)
            ps, pt = ls.gather(1, ids[e]).exp(), lp[e].double().exp()
            p = ls.exp().scatter(1, ids[e], 0.0)
            ts, mass = p.sum(1, keepdim=True), pt.sum(1, keepdim=True)
            tt = (1 - mass).clamp_min(1e-8)
            assert bool(((ts - 1e-8).abs() > 2e-9).all())        # a tail at its floor's edge may fall on either side
            on = ts >= 1e-8
            a = (w[e].double() / T)[:, None]
            ratio = torch.where(on, tt / ts, 0.0)
            want = a * (torch.where(on, tt, 0.0) + mass - ratio) * p
            want = want.scatter(1, ids[e], a * ((torch.where(on, tt, 0.0) + mass) * ps - pt))
            lim = (TOL * a * (1 + ratio) * p).scatter(1, ids[e], TOL * a * (ps + pt)) + EPS[dtype] * want.abs() + 6e-8
            for got in (first[e], second[e]):
                assert bool(((got.double() - want).abs() <= lim).all()), (K, i, float(((got.double() - want).abs() - lim).max()))
