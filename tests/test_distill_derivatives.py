"""The training objectives where their callers want more than one gradient: second derivatives, forward-mode derivatives and vmap,
gradients of the target, more teacher tokens or a larger vocabulary than the kernels list, other shapes. The torch forms
gave all of these, and the results are compared with those."""
import pytest
import torch

from arcagi2_flashnext_dots3_b200.ops import distill
from arcagi2_flashnext_dots3_b200.training import draft_head
from arcagi2_flashnext_dots3_b200.training.d3_student import kd_topk_loss

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def torch_kd(z, ids, lp):
    ls = torch.log_softmax(z.float(), -1)
    ps, pt = ls.gather(1, ids.long()), lp.float().exp()
    tail_t = (1 - pt.sum(-1)).clamp_min(1e-8)
    tail_s = (1 - ps.exp().sum(-1)).clamp_min(1e-8)
    return ((pt * (lp.float() - ps)).sum(-1) + tail_t * (tail_t.log() - tail_s.log())).mean()


def torch_accept(q, p):
    lq, lp = torch.log_softmax(q, -1), torch.log_softmax(p, -1)
    return torch.minimum(lq.exp(), lp.exp()).sum(-1), (lp.exp() * (lp - lq)).sum(-1)


def inputs(device, n=5, V=40, K=4):
    g = torch.Generator().manual_seed(3)
    z = torch.randn(n, V, generator=g)
    lp, ids = torch.log_softmax(torch.randn(n, V, generator=g), -1).topk(K, -1)
    return z.to(device), ids.to(device), lp.to(device), torch.randn(n, V, generator=g).to(device)


def same(a, b):
    # fp32 sums of some tens of terms of order one
    assert float((a - b).detach().abs().max()) <= 2e-5 * max(1.0, float(b.detach().abs().max()))


@pytest.mark.parametrize("device", DEVICES)
def test_second_derivatives_of_the_distillation_loss(device):
    z, ids, lp, v = inputs(device)
    out = []
    for f in (kd_topk_loss, torch_kd):
        x = z.clone().requires_grad_()
        d, = torch.autograd.grad(f(x, ids, lp), x, create_graph=True)
        out.append((d, torch.autograd.grad((d * v).sum(), x)[0]))
        same(d, torch.autograd.grad(f(x, ids, lp), x)[0])
    same(out[0][0], out[1][0])
    same(out[0][1], out[1][1])
    x = z.clone().requires_grad_()                       # one graph walked twice
    loss = kd_topk_loss(x, ids, lp)
    a, = torch.autograd.grad(loss, x, retain_graph=True)
    b, = torch.autograd.grad(loss, x)
    assert torch.equal(a, b)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(loss, x)
    assert not kd_topk_loss(z, ids, lp).requires_grad
    with torch.no_grad():
        assert not kd_topk_loss(x, ids, lp).requires_grad


@pytest.mark.parametrize("device", DEVICES)
def test_forward_mode_and_vmap_of_the_distillation_loss(device):
    z, ids, lp, v = inputs(device)
    got = torch.func.jvp(lambda x: kd_topk_loss(x, ids, lp), (z,), (v,))
    want = torch.func.jvp(lambda x: torch_kd(x, ids, lp), (z,), (v,))
    for a, b in zip(got, want):
        same(a, b)
    import torch.autograd.forward_ad as fwd
    with fwd.dual_level():
        t = fwd.unpack_dual(kd_topk_loss(fwd.make_dual(z, v), ids, lp)).tangent
    same(t, want[1])
    zz = torch.stack([z, v])
    same(torch.func.vmap(lambda x: kd_topk_loss(x, ids, lp))(zz), torch.stack([torch_kd(x, ids, lp) for x in zz]))
    same(torch.func.grad(lambda x: kd_topk_loss(x, ids, lp))(z), torch.func.grad(lambda x: torch_kd(x, ids, lp))(z))


@pytest.mark.parametrize("device", DEVICES)
def test_shapes_of_the_distillation_loss(device):
    z, ids, lp, _ = inputs(device, V=200, K=150)              # more teacher tokens than the kernels list
    same(kd_topk_loss(z, ids, lp), torch_kd(z, ids, lp))
    z, ids, lp, _ = inputs(device)
    same(kd_topk_loss(z, ids[:3], lp[:3]), torch_kd(z, ids[:3], lp[:3]))
    same(kd_topk_loss(z, ids, lp[:1]), torch_kd(z, ids, lp[:1]))
    same(kd_topk_loss(z, ids[:, :0], lp[:, :0]), torch_kd(z, ids[:, :0], lp[:, :0]))
    wide = torch.zeros(1, distill.MAX_V + 8, device=device)
    wide[0, 5] = 3.0
    x = wide.requires_grad_()
    one = torch.tensor([[5]], device=device), torch.tensor([[-0.1]], device=device)
    loss = kd_topk_loss(x, *one)
    same(loss, torch_kd(x, *one))
    assert bool(torch.isfinite(torch.autograd.grad(loss, x)[0]).all())
    t = lp.clone().requires_grad_()
    u = lp.clone().requires_grad_()
    kd_topk_loss(z, ids, t).backward()
    torch_kd(z, ids, u).backward()
    same(t.grad, u.grad)


class Head(torch.nn.Module):
    """What draft_objective asks of a draft head."""

    def __init__(self, W, device):
        super().__init__()
        self.W, self.device, self.hot = W, torch.device(device), None

    def step(self, x, ids, pos):
        return torch.tanh(x + 0.1 * ids[:, None].float() + pos)

    def logits(self, x):
        return x @ self.W


@pytest.mark.parametrize("device", DEVICES)
def test_derivatives_of_the_draft_objective(device):
    """First and second derivatives in the head, and the gradient of target logits that want one."""
    g = torch.Generator().manual_seed(7)
    h, W = torch.randn(9, 6, generator=g).to(device), torch.randn(6, 30, generator=g).to(device)
    tl, ids = torch.randn(9, 30, generator=g).to(device), torch.randint(0, 5, (9,), generator=g)
    v = torch.randn(6, 30, generator=g).to(device)

    def plain(head, tl):
        prod, E, kl, x = 1.0, 0.0, 0.0, h[:6]
        for k in range(1, 4):
            x = head.step(x, ids.to(device)[k:k + 6], k - 1)
            a, l = torch_accept(head.logits(x), tl[k:k + 6])
            prod = prod * a
            E, kl = E + prod, kl + l.mean()
        return -E.mean() + 0.3 * kl / 3
    out = []
    for f in (lambda m, t: draft_head.draft_objective(m, h, ids, t, K=3)[0], plain):
        w = W.clone().requires_grad_()
        d, = torch.autograd.grad(f(Head(w, device), tl), w, create_graph=True)
        e, = torch.autograd.grad((d * v).sum(), w)
        same(d, torch.autograd.grad(f(Head(w, device), tl), w)[0])
        t = tl.clone().requires_grad_()
        out.append((d, e, torch.autograd.grad(f(Head(w, device), t), t)[0],
                    torch.func.jvp(lambda w: f(Head(w, device), tl), (W,), (v,))[1]))
    for a, b in zip(*out):
        same(a, b)
