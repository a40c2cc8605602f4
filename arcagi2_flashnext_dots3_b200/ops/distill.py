"""Vocabulary-row operators of distillation: the teacher's top tokens, the loss against them, and the acceptance / KL
objective of a draft head. CUDA tensors go to the `_C` kernels (csrc/k_vocab.cu), CPU tensors to torch code with the
same math. The recipe is the reference's (flashnext/training/kd/train_kd.py `kl21`,
flashnext/training/draft_head/train.py); its code works in torch on whole [rows, vocab] tensors.

* :func:`teacher_topk` - the k most likely tokens of each row and their log-probabilities;
* :func:`kd_topk` / :func:`kd_topk_grad` - KL(teacher || student) over the teacher's K tokens plus one bin for all
  others, differentiable, or with the gradient in the same pass when the rows' weights are known;
* :func:`accept_kl` - sum min(q, p) and KL(p || q) of a draft distribution q against a target p, differentiable in
  the draft.

Logits are [rows, vocab] in fp32, fp16 or bf16 (vocab up to 2^20; rows may be strided). A logit at or below -1e30
(-inf, the lowest fp32 / bf16 value) is masked and has probability 0; a row with nothing left gives loss 0, gradient
0 and id -1. A NaN makes its row's results NaN. Temperatures are 1e-6 to 1e6, and logits on the GPU at most 2^30 T.
Results per row are fp32, gradients have the logits' type. Nothing here reads from the host, so every call can be
captured in a CUDA graph.
"""
from __future__ import annotations

import torch
import torch.autograd.forward_ad

from . import native

MASKED = -1e30       # csrc/k_vocab.cu kFloor is the float above it
TAIL_FLOOR = 1e-8    # csrc/k_vocab.cu kTailFloor
MAX_K = 128          # csrc/vocab.h kMaxK
MAX_V = 1 << 20      # csrc/vocab.h kMaxV
DTYPES = (torch.float32, torch.float16, torch.bfloat16)


def _rows(x: torch.Tensor, name: str) -> torch.Tensor:
    if x.dim() != 2 or x.shape[1] < 1:
        raise ValueError(f"{name}: expected [rows, vocab], got {tuple(x.shape)}")
    if x.dtype not in DTYPES:
        raise ValueError(f"{name}: fp32, fp16 or bf16 logits, got {x.dtype}")
    return x if x.shape[1] == 1 or x.stride(1) == 1 else x.contiguous()


def _teacher(logits, t_ids, t_lp):
    if t_ids.dim() != 2 or t_ids.shape != t_lp.shape or t_ids.shape[0] != logits.shape[0]:
        raise ValueError(f"teacher ids and log-probabilities: expected two [{logits.shape[0]}, K], got "
                         f"{tuple(t_ids.shape)} and {tuple(t_lp.shape)}")
    if not 1 <= t_ids.shape[1] <= MAX_K:
        raise ValueError(f"1 to {MAX_K} teacher tokens per row, got {t_ids.shape[1]}")
    if t_ids.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"teacher ids: int32 or int64, got {t_ids.dtype}")
    if t_ids.device != logits.device or t_lp.device != logits.device:
        raise ValueError("logits, teacher ids and teacher log-probabilities must be on one device")
    return t_ids.contiguous(), t_lp.detach().float().contiguous()


def _temperature(t: float) -> float:
    t = float(t)
    if not 1e-6 <= t <= 1e6:
        raise ValueError(f"temperature must be in [1e-6, 1e6], got {t}")
    return t


def _log_softmax(x: torch.Tensor, t: float, dtype=torch.float32) -> torch.Tensor:
    """log softmax(x / t) with masked logits at -inf; a row with nothing left is -inf throughout."""
    z = x.to(dtype)
    z = z.masked_fill(z <= MASKED, float("-inf")) / t
    nothing = (z == float("-inf")).all(-1, keepdim=True)
    return torch.log_softmax(z.masked_fill(nothing, 0.0), -1).masked_fill(nothing, float("-inf"))


def transformed() -> bool:
    """Whether the caller runs under forward-mode differentiation or a torch.func transform, which the operators here do
    not take part in."""
    return torch._C._are_functorch_transforms_active() or torch.autograd.forward_ad._current_level >= 0


class _Twice(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, fast, plain):
        ctx.fast, ctx.plain = fast, plain
        ctx.save_for_backward(x)
        ctx.inner = _Twice.run(fast, x)
        return tuple(o.detach() for o in ctx.inner[1])

    @staticmethod
    def run(f, x):
        with torch.enable_grad():
            z = x.detach().requires_grad_()
            return z, f(z)

    @staticmethod
    def backward(ctx, *g):
        x, = ctx.saved_tensors
        if torch.is_grad_enabled():
            return torch.autograd.grad(ctx.plain(x), x, g, create_graph=True)[0], None, None
        z, out = ctx.inner or _Twice.run(ctx.fast, x)       # the graph that forward left is walked once
        ctx.inner = None
        return torch.autograd.grad(out, z, g)[0], None, None


def twice(x: torch.Tensor, fast, plain) -> tuple:
    """fast(x), a tuple of tensors, for callers that may differentiate its gradient again: a backward pass that is itself recorded
    goes through plain(x), the same in torch operations."""
    if not (x.requires_grad and torch.is_grad_enabled()):
        return fast(x)
    return _Twice.apply(x, fast, plain)


# ------------------------------------------------------------------------------------------------ teacher top-k
def teacher_topk(logits: torch.Tensor, k: int, temperature: float = 1.0):
    """(ids int32 [rows, k], log-probabilities fp32 [rows, k]) of the k largest logits of each row, best first (ties:
    lowest id), under softmax(logits / temperature). Rows with fewer than k unmasked tokens are padded with id -1 and
    log-probability -inf, the padding of the distillation records. A NaN ranks above every number and makes the row's
    log-probabilities NaN. k <= 128."""
    if logits.is_cuda:
        return native.C().teacher_topk(logits, k, temperature)
    logits = _rows(logits.detach(), "logits")
    t = _temperature(temperature)
    if not 1 <= k <= MAX_K:
        raise ValueError(f"k must be in [1, {MAX_K}], got {k}")
    n, V = logits.shape
    ls = _log_softmax(logits, t)
    z = logits.float()
    z, order = torch.sort(z.masked_fill(z <= MASKED, float("-inf")), dim=-1, descending=True, stable=True)
    z, order = z[:, :k], order[:, :k]
    lp = ls.gather(1, order).masked_fill(z == float("-inf"), float("-inf"))
    ids = order.to(torch.int32).masked_fill(z == float("-inf"), -1)
    if k > V:
        ids = torch.cat([ids, ids.new_full((n, k - V), -1)], 1)
        lp = torch.cat([lp, lp.new_full((n, k - V), float("-inf"))], 1)
    return ids, lp


# ------------------------------------------------------------------------------------------------ distillation
def _kd_cpu(logits, t_ids, t_lp, t, weight=None):
    """Per-row loss, or with weights (loss, d sum(weight * loss) / d logits)."""
    n, V = logits.shape
    ls = _log_softmax(logits, t)
    nothing = (ls == float("-inf")).all(-1)
    ids = t_ids.long()
    same = (ids[:, :, None] == ids[:, None, :]).tril(-1).any(-1)
    valid = (ids >= 0) & (ids < V) & ~same
    at = torch.where(valid, ids, V)                                  # column V collects what is left out
    p = torch.cat([ls.exp(), ls.new_zeros(n, 1)], 1)
    s = torch.cat([ls, ls.new_zeros(n, 1)], 1).gather(1, at)
    pt = torch.where(valid, t_lp.exp(), 0.0)
    tt = (1 - pt.double().sum(-1)).clamp_min(TAIL_FLOOR).float()
    tail = p.scatter(1, at, 0.0).sum(-1)
    ts = tail.clamp_min(TAIL_FLOOR)
    loss = torch.where(pt > 0, pt * (t_lp - s), 0.0).sum(-1) + tt * (tt.log() - ts.log())
    loss = torch.where(nothing, 0.0, loss)
    if weight is None:
        return loss
    on, mass, ps = tail >= TAIL_FLOOR, pt.sum(-1), torch.where(valid, s.exp(), 0.0)
    csum = torch.where(on, tt / ts, 0.0) * ps.sum(-1) - mass
    pull = torch.where(on, tt, 0.0) + mass            # tt / ts - csum, which would lose a sure student's tail as a difference
    d = (-csum[:, None] * p).scatter(1, at, pull[:, None] * ps - pt)[:, :V] * (weight / t)[:, None]
    return loss, torch.where(nothing[:, None], 0.0, d).to(logits.dtype)


class _KDTopK(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, t_ids, t_lp, t):
        ctx.t = t
        ctx.save_for_backward(logits, t_ids, t_lp)
        return _kd_cpu(logits, t_ids, t_lp, t)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        return _kd_cpu(*ctx.saved_tensors, ctx.t, g.float())[1], None, None, None


def kd_topk(logits: torch.Tensor, t_ids: torch.Tensor, t_lp: torch.Tensor, temperature: float = 1.0) -> torch.Tensor:
    """KL(teacher || student) per row over the teacher's K tokens and a tail bin, fp32 [rows], differentiable in the
    logits. ``t_ids`` int32 / int64 [rows, K] with K <= 128, ``t_lp`` the teacher's log-probabilities at them (at the
    same temperature). Ids outside the vocabulary (the -1 of padded records) are left out and their mass falls to the
    tail; a repeated id counts once, at its first place. Both tail masses have a floor of 1e-8."""
    if logits.is_cuda:
        return native.C().kd_topk(logits, t_ids, t_lp, temperature)
    logits = _rows(logits, "logits")
    t_ids, t_lp = _teacher(logits, t_ids, t_lp)
    return _KDTopK.apply(logits, t_ids, t_lp, _temperature(temperature))


def kd_topk_grad(logits: torch.Tensor, t_ids: torch.Tensor, t_lp: torch.Tensor, weight: torch.Tensor,
                 temperature: float = 1.0, out: torch.Tensor = None):
    """(loss [rows], d sum(weight * loss) / d logits in the logits' type) of :func:`kd_topk` in one pass over the
    logits, for callers that know the rows' weights (fp32 [rows]). ``out``: where the gradient goes; it may be the
    logits themselves, which are then overwritten."""
    if logits.is_cuda:
        return native.C().kd_topk_grad(logits, t_ids, t_lp, weight, temperature, out)
    logits = _rows(logits.detach(), "logits")
    t_ids, t_lp = _teacher(logits, t_ids, t_lp)
    t = _temperature(temperature)
    n = logits.shape[0]
    if weight.shape != (n,) or weight.device != logits.device:
        raise ValueError(f"weight: expected [{n}] on the logits' device, got {tuple(weight.shape)}")
    weight = weight.detach().float().contiguous()
    if out is None:
        out = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    elif out.shape != logits.shape or out.dtype != logits.dtype or out.device != logits.device or \
            (out.shape[1] > 1 and out.stride(1) != 1):
        raise ValueError("out must have the logits' shape, type and device and unit stride along the vocabulary")
    loss, g = _kd_cpu(logits, t_ids, t_lp, t, weight)
    return loss, out.copy_(g)


# ------------------------------------------------------------------------------------------------ acceptance and KL
def _accept_cpu(draft, target, t, g_alpha=None, g_kl=None):
    """(alpha, kl) per row, or with their gradients the gradient of the draft."""
    ninf = float("-inf")
    lq, lp = (_log_softmax(x, t, torch.float64) for x in (draft, target))
    nothing = (lq == ninf).all(-1) | (lp == ninf).all(-1)
    q, p = lq.exp(), lp.exp()
    if g_alpha is None:
        kl = torch.where(p > 0, p * (lp - lq), 0.0)
        kl = torch.where(torch.isnan(p), p, kl).sum(-1)
        return torch.where(nothing, 0.0, torch.minimum(q, p).sum(-1)).float(), torch.where(nothing, 0.0, kl).float()
    # h - A of a token from the masses of the other sides: a sure token's 1 - A is lost in a difference
    below, even, above = ((q * on).sum(-1, keepdim=True) for on in (lq < lp, lq == lp, lq > lp))
    h_a = torch.where(lq < lp, above + 0.5 * even, torch.where(lq == lp, 0.5 * (above - below), -(below + 0.5 * even)))
    d = (g_alpha / t)[:, None] * q * h_a + (g_kl / t)[:, None] * (q - p)
    return torch.where(nothing[:, None], 0.0, d).to(draft.dtype)


class _AcceptKL(torch.autograd.Function):
    @staticmethod
    def forward(ctx, draft, target, t):
        ctx.t = t
        ctx.save_for_backward(draft, target)
        return _accept_cpu(draft, target, t)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g_alpha, g_kl):
        return _accept_cpu(*ctx.saved_tensors, ctx.t, g_alpha.float(), g_kl.float()), None, None


def accept_kl(draft: torch.Tensor, target: torch.Tensor, temperature: float = 1.0):
    """(alpha, kl) fp32 [rows] of draft logits against target logits of the same shape and type: alpha = sum_v
    min(q_v, p_v), the probability that speculative verification accepts a token drawn from q, and kl = KL(p || q),
    with q, p the softmaxes at `temperature`. Differentiable in the draft; the target is taken as given. Where q_v =
    p_v (for the kernels: to within a few fp32 roundings) the gradient of alpha is the mean of its two sides. A row in
    which either side has no token left gives zeros."""
    if draft.is_cuda:
        return native.C().accept_kl(draft, target, temperature)
    draft = _rows(draft, "draft logits")
    target = _rows(target.detach(), "target logits")
    if draft.shape != target.shape or draft.dtype != target.dtype or draft.device != target.device:
        raise ValueError(f"draft and target logits must agree in shape, type and device: {tuple(draft.shape)} "
                         f"{draft.dtype} {draft.device} and {tuple(target.shape)} {target.dtype} {target.device}")
    return _AcceptKL.apply(draft, target, _temperature(temperature))
