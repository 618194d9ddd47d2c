"""Plain 64-bit forms of the token-policy operators, for the tests: written from the formulas, on whatever device the
inputs are on, differentiable with torch's autograd where a gradient is asked for."""
import math

import torch


def logprobs(logits, actions, temperature=1.0, ignore=-100):
    """(log p, entropy) in f64; an ignored token and the entropy of a row without a legal action are 0."""
    z = logits.double() / temperature
    empty = (z == -math.inf).all(-1)
    z = torch.where(empty.unsqueeze(-1), torch.zeros_like(z), z)
    z = z - z.amax(-1, keepdim=True)                     # in rows at the type's lowest value even 64 bits lose ln A otherwise
    lp = z - torch.logsumexp(z, -1, keepdim=True)
    safe = torch.where(lp == -math.inf, torch.zeros_like(lp), lp)
    p = torch.where(lp == -math.inf, torch.zeros_like(lp), torch.exp(safe))
    h = -(p * safe).sum(-1)
    dead = actions == ignore
    lp_a = lp.gather(-1, torch.where(dead, 0, actions).long().unsqueeze(-1)).squeeze(-1)
    lp_a = torch.where(empty, torch.full_like(lp_a, -math.inf), lp_a)
    return torch.where(dead, torch.zeros_like(lp_a), lp_a), torch.where(dead | empty, torch.zeros_like(h), h)


def logprobs_grad(logits, actions, g_logp, g_entropy, temperature=1.0, ignore=-100):
    """(gradient of sum g_logp log p + g_entropy H, sum of the magnitudes of its terms), from the formula."""
    z = logits.double() / temperature
    empty = (z == -math.inf).all(-1, keepdim=True)
    z = torch.where(empty, torch.zeros_like(z), z)
    z = z - z.amax(-1, keepdim=True)                     # in rows at the type's lowest value even 64 bits lose ln A otherwise
    lp = z - torch.logsumexp(z, -1, keepdim=True)
    safe = torch.where(lp == -math.inf, torch.zeros_like(lp), lp)
    p = torch.where(lp == -math.inf, torch.zeros_like(lp), torch.exp(safe))
    h = -(p * safe).sum(-1, keepdim=True)
    dead = (actions == ignore).unsqueeze(-1)
    hot = torch.zeros_like(p).scatter_(-1, torch.where(dead.squeeze(-1), 0, actions).long().unsqueeze(-1), 1.0)
    live = (~dead & ~empty).double() / temperature
    gl = g_logp.double().unsqueeze(-1) * live
    gh = (g_entropy.double().unsqueeze(-1) if g_entropy is not None else torch.zeros_like(gl)) * live
    return gl * (hot - p) - gh * p * (safe + h), gl.abs() * (hot + p) + gh.abs() * p * (safe.abs() + h)


def _weights(mask, reduction):
    n = mask.sum(1, keepdim=True)
    if reduction == "token":
        return mask / n.sum().clamp(min=1)
    return mask / n.clamp(min=1) / (n > 0).sum().clamp(min=1)


def policy(new, old, adv, mask=None, ref=None, lo=0.2, hi=0.2, coef=0.0, kl="k3", reduction="token"):
    """[loss, policy, kl, clip fraction, drift, tokens] in f64, differentiable in `new`."""
    mask = torch.ones_like(new, dtype=torch.bool) if mask is None else mask != 0
    clean = lambda t: torch.where(mask, t.double(), torch.zeros((), dtype=torch.float64, device=t.device))  # noqa: E731
    x, o = clean(new), clean(old)
    a = clean(adv.unsqueeze(1).expand_as(new) if adv.dim() == 1 else adv)
    w = _weights(mask.double(), reduction)
    d = x - o
    r = torch.exp(d)
    term = -torch.minimum(r * a, torch.clamp(r, 1 - lo, 1 + hi) * a)
    k = torch.zeros_like(x)
    if ref is not None:
        e = x - clean(ref)
        k = {"k1": e, "k2": 0.5 * e * e, "k3": torch.exp(-e) - 1 + e}[kl]
    pg, klm = (w * term).sum(), (w * k).sum()
    out = ((d > math.log1p(hi)) | (d < math.log1p(-lo))).double()
    return torch.stack([pg + coef * klm, pg, klm, (w * out).sum(), (w * (r - 1 - d)).sum(), mask.double().sum()]), w, a, r, k


def preference(chosen, rejected, ref_c=None, ref_r=None, mask_c=None, mask_r=None, beta=0.1, kind="sigmoid", smoothing=0.0, average=False):
    """(mean loss, accuracy, rewards) in f64, differentiable in the two log-probs."""
    sums = []
    for lp, ref, mask in ((chosen, ref_c, mask_c), (rejected, ref_r, mask_r)):
        m = torch.ones_like(lp, dtype=torch.bool) if mask is None else mask != 0
        v = lp.double() if ref is None else lp.double() - ref.double()
        s = torch.where(m, v, torch.zeros_like(v)).sum(1)
        sums.append(s / m.sum(1).clamp(min=1) if average else s)
    z = beta * (sums[0] - sums[1])
    sp = torch.nn.functional.softplus
    if kind == "sigmoid":
        loss = (1 - smoothing) * sp(-z) + smoothing * sp(z)
    elif kind == "hinge":
        loss = torch.clamp(1 - z, min=0)
    else:
        loss = (z / beta - 0.5 / beta) ** 2
    return loss.mean(), (z > 0).double().mean(), torch.stack([beta * sums[0], beta * sums[1]], 1)


def linear(x, weight, bias=None, activation="none", residual=None):
    """act(x W^T + b) + residual in f64."""
    z = x.double() @ weight.double().t()
    if bias is not None:
        z = z + bias.double()
    f = torch.nn.functional
    gelu = lambda v: v * 0.5 * torch.erfc(v * -math.sqrt(0.5))  # noqa: E731  (1 + erf loses its left tail even in 64 bits)
    y = {"none": lambda v: v, "tanh": torch.tanh, "relu": f.relu, "gelu": gelu, "silu": f.silu}[activation](z)
    return y if residual is None else y + residual.double()
