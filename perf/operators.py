"""The token-policy operators as a training or scoring program meets them: log-probabilities and entropy of
actions under wide categorical heads, the clipped policy loss with a KL term, the preference loss on paired log
ratios, and the linear layer with bias, activation and residual -- each in a plain form of elementary torch
operations, from its definition in 64 bits, and as the call into ppo_amd.ops.

    listed()             the cases                     run(state)          one pass
    draw(rng)            one more of the same ranges   work(case)          bytes and operations it cannot do without
    prepare(case, seed)  inputs on the GPU             exact(case, seed)   the outputs in 64 bits
"""
import math

import torch

own = False      # False: the plain forms; True: the calls into ppo_amd.ops

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
IGNORE = -100


# ------------------------------------------------------------------------------------------------- cases
def _logprobs(name, batch, length, actions, dtype, train, ignored=0.0, masked=False, temperature=1.0, shifted=False):
    """[batch, length] tokens (length - 1 of them with `shifted`: the view logits[:, :-1]) over `actions` actions;
    `ignored`: share of tokens that carry the ignored label; `masked`: 30 % of the actions of a row at -inf, and
    every action of one row where there is more than one."""
    return {"name": name, "op": "logprobs", "batch": batch, "length": length, "actions": actions, "dtype": dtype,
            "train": train, "ignored": ignored, "masked": masked, "temperature": temperature, "shifted": shifted}


def _policy(name, batch, length, mask, ref, kl, reduction, per_sequence, clip_low=0.2, clip_high=0.2, kl_coef=0.05):
    """mask: "none", "ragged" (sequences of unequal length, one of them empty) or "random"."""
    return {"name": name, "op": "policy", "batch": batch, "length": length, "mask": mask, "ref": ref, "kl": kl,
            "reduction": reduction, "per_sequence": per_sequence, "clip_low": clip_low, "clip_high": clip_high,
            "kl_coef": kl_coef}


def _preference(name, pairs, chosen, rejected, mask, ref, kind, beta=0.1, smoothing=0.0, average=False):
    return {"name": name, "op": "preference", "pairs": pairs, "chosen": chosen, "rejected": rejected, "mask": mask,
            "ref": ref, "kind": kind, "beta": beta, "smoothing": smoothing, "average": average}


def _linear(name, rows, inputs, outputs, dtype, activation, bias, residual, train):
    return {"name": name, "op": "linear", "rows": rows, "inputs": inputs, "outputs": outputs, "dtype": dtype,
            "activation": activation, "bias": bias, "residual": residual, "train": train}


def listed():
    return [
        # one decoding step of eight sequences, whose chosen tokens are scored: latency of a long row
        _logprobs("score one step", 8, 1, 32768, "bf16", False),
        # a minibatch of a Discrete head with more actions than the fused PPO head takes, some of them illegal
        _logprobs("wide action head", 64, 4096, 18, "f32", True, masked=True),
        # next-token training on padded sequences: the shifted view of the logits, an odd vocabulary
        _logprobs("token batch, shifted", 8, 1025, 50001, "bf16", True, ignored=0.2, shifted=True),
        # the largest: a long batch over a large vocabulary, sampled at another temperature
        _logprobs("large vocabulary", 4, 2048, 131072, "f16", True, temperature=0.7),
        # the policy loss of a handful of short answers: launch latency
        _policy("a few short answers", 4, 17, "ragged", True, "k3", "token", True),
        # a full rollout of long answers, advantages per token, KL to the reference policy
        _policy("long answers", 4096, 8192, "ragged", True, "k3", "token", False),
        # two pairs of very long documents of odd lengths: few rows, long sums
        _preference("two long pairs", 2, 131071, 99999, "ragged", True, "sigmoid", smoothing=0.1),
        # a large batch of preference pairs, length-normalised
        _preference("many pairs", 2048, 4096, 4000, "ragged", True, "ipo", average=True),
        # serving: one token through a wide layer, the weights read once
        _linear("one token", 1, 4096, 16384, "bf16", "gelu", True, False, False),
        # the sizes of the Atari agents' trunk, Linear(3136, 512), on a minibatch, in 32 bits as those agents train
        _linear("feature trunk", 16384, 3136, 512, "f32", "tanh", True, False, True),
        # a layer of odd sizes with its residual
        _linear("odd residual layer", 2047, 1000, 3001, "f16", "silu", True, True, True),
        # the largest: a wide layer over a long batch, forward and backward
        _linear("wide layer", 8192, 4096, 16384, "bf16", "gelu", True, False, True),
    ]


def _spread(rng, low, high):
    """A whole number of [low, high], its logarithm uniform."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["logprobs", "policy", "preference", "linear"])
    coin = lambda: rng.random() < 0.5  # noqa: E731
    if op == "logprobs":
        actions = _spread(rng, 2, 131072)
        tokens = _spread(rng, 1, max(1, min(1 << 18, (1 << 29) // actions)))
        batch = _spread(rng, 1, min(tokens, 64))
        shifted = coin()
        return _logprobs("", batch, tokens // batch + shifted, actions, rng.choice(["f32", "bf16", "f16"]), coin(),
                         rng.choice([0.0, 0.2]), coin(), rng.choice([1.0, 0.7, 1.5]), shifted)
    if op == "policy":
        length = _spread(rng, 1, 8192)
        batch = _spread(rng, 1, min(4096, (1 << 24) // length))
        return _policy("", batch, length, rng.choice(["none", "ragged", "random"]), coin(), rng.choice(["k1", "k2", "k3"]),
                       rng.choice(["token", "sequence"]), coin(), rng.choice([0.1, 0.2]), rng.choice([0.2, 0.28]),
                       rng.choice([0.0, 0.05, 0.2]))
    if op == "preference":
        chosen, rejected = _spread(rng, 1, 131072), _spread(rng, 1, 131072)
        pairs = _spread(rng, 1, min(2048, max(1, (1 << 23) // (chosen + rejected))))
        kind = rng.choice(["sigmoid", "hinge", "ipo"])
        return _preference("", pairs, chosen, rejected, rng.choice(["none", "ragged", "random"]), coin(), kind,
                           rng.choice([0.05, 0.1, 0.5]), rng.choice([0.0, 0.1]) if kind == "sigmoid" else 0.0, coin())
    inputs, outputs = _spread(rng, 16, 8192), _spread(rng, 16, 16384)
    rows = _spread(rng, 1, max(1, min(16384, (1 << 37) // (inputs * outputs))))
    dtype, train = rng.choice(["f32", "bf16", "f16"]), coin()
    # relu's derivative jumps at 0, where two sums in 32 bits differ in sign: with f32 gradients that is all one would see
    smooth = ["none", "tanh", "gelu", "silu"]
    return _linear("", rows, inputs, outputs, dtype, rng.choice(smooth if train and dtype == "f32" else smooth + ["relu"]),
                   coin(), coin(), train)


# ------------------------------------------------------------------------------------------------- inputs
def _mask(gen, kind, rows, length):
    """[rows, length] truth values on the GPU, or None."""
    if kind == "none":
        return None
    if kind == "random":
        return torch.rand(rows, length, device="cuda", generator=gen) < 0.7
    lengths = torch.randint(1, length + 1, (rows, 1), device="cuda", generator=gen)
    if rows > 2:
        lengths[rows // 2] = 0
    return torch.arange(length, device="cuda") < lengths


def prepare(case, seed):
    gen = torch.Generator("cuda")
    gen.manual_seed(seed)
    randn = lambda *shape, dtype=torch.float32: torch.randn(*shape, dtype=dtype, device="cuda", generator=gen)  # noqa: E731
    s = {"case": case}
    if case["op"] == "logprobs":
        dtype, B, L, A = DTYPES[case["dtype"]], case["batch"], case["length"], case["actions"]
        logits = randn(B, L, A, dtype=dtype).mul_(3.0)
        T = L - case["shifted"]
        actions = torch.randint(0, A, (B, T), device="cuda", generator=gen)
        if case["masked"]:
            off = torch.rand(B, L, A, device="cuda", generator=gen) < 0.3
            off[:, :T].scatter_(2, actions.unsqueeze(2), False)
            off[B // 2, T // 2] |= B * T > 1
            logits.masked_fill_(off, -math.inf)
        if case["ignored"]:
            actions[torch.rand(B, T, device="cuda", generator=gen) < case["ignored"]] = IGNORE
        s["logits"], s["actions"] = (logits[:, :-1] if case["shifted"] else logits), actions
        if case["train"]:      # what a loss sends back: a mean over the tokens, and an entropy bonus
            s["g_logp"] = randn(B, T) / (B * T)
            s["g_entropy"] = torch.full((B, T), -0.01 / (B * T), device="cuda")
    elif case["op"] == "policy":
        B, L = case["batch"], case["length"]
        s["old"] = -randn(B, L).abs()
        s["new"] = s["old"] + 0.15 * randn(B, L)
        s["ref"] = s["old"] + 0.3 * randn(B, L) if case["ref"] else None
        s["adv"] = randn(B) if case["per_sequence"] else randn(B, L)
        s["mask"] = _mask(gen, case["mask"], B, L)
    elif case["op"] == "preference":
        B = case["pairs"]
        for side in ("chosen", "rejected"):
            L = case[side]
            s[side] = -randn(B, L).abs()
            s["ref_" + side] = s[side] + 0.05 * randn(B, L) if case["ref"] else None
            s["mask_" + side] = _mask(gen, case["mask"], B, L)
    else:
        dtype, M, K, N = DTYPES[case["dtype"]], case["rows"], case["inputs"], case["outputs"]
        s["x"] = randn(M, K, dtype=dtype)
        s["weight"] = randn(N, K, dtype=dtype).mul_(K ** -0.5)
        s["bias"] = randn(N, dtype=dtype).mul_(0.1) if case["bias"] else None
        s["residual"] = randn(M, N, dtype=dtype) if case["residual"] else None
        if case["train"]:
            s["g"] = randn(M, N, dtype=dtype).mul_(0.1)
    return s


# ------------------------------------------------------------------------------------------------- plain forms
def _plain_logprobs(s, c):
    """z = logits / temperature; log p_a = z_a - lse(z); H = -sum p log p.  An ignored token gives 0 and no gradient,
    a row without a legal action log p = -inf, H = 0 and no gradient."""
    logits, actions = s["logits"], s["actions"]
    z = logits.float() * (1.0 / c["temperature"])
    top = z.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    ex = torch.exp(z - top)
    total = ex.sum(-1, keepdim=True)
    lp = z - (top + torch.log(total))
    p = ex / torch.where(total == 0, torch.ones_like(total), total)
    plogp = torch.where(p > 0, p * lp, torch.zeros_like(p))
    entropy = -plogp.sum(-1)
    ignored, empty = actions == IGNORE, (total == 0).squeeze(-1)
    index = torch.where(ignored, torch.zeros_like(actions), actions)
    logp = lp.gather(-1, index.unsqueeze(-1)).squeeze(-1)
    logp = torch.where(empty, torch.full_like(logp, -math.inf), logp)
    zero = torch.zeros_like(logp)
    out = [torch.where(ignored, zero, logp), torch.where(ignored, zero, entropy)]
    if c["train"]:
        dead = ignored | empty
        g_lp = torch.where(dead, zero, s["g_logp"]).unsqueeze(-1)
        g_h = torch.where(dead, zero, s["g_entropy"]).unsqueeze(-1)
        g = -g_lp * p - g_h * (plogp + p * entropy.unsqueeze(-1))
        g.scatter_add_(-1, index.unsqueeze(-1), g_lp)
        out.append((g * (1.0 / c["temperature"])).to(logits.dtype))
    return out


def _plain_policy(s, c):
    """A token's loss: -min(r A, clip(r) A) + kl_coef k(new - ref), r = exp(new - old); the mean over the tokens, or over
    the sequences of their tokens' means.  Sums, the clip's border and the third estimator in 64 bits."""
    new, old, ref, adv = s["new"], s["old"], s["ref"], s["adv"]
    adv = adv.unsqueeze(1) if c["per_sequence"] else adv
    mask = s["mask"] if s["mask"] is not None else torch.ones_like(new, dtype=torch.bool)
    d = new.double() - old.double()
    above, below = d > math.log1p(c["clip_high"]), d < math.log1p(-c["clip_low"])
    ratio = torch.exp(new - old)
    cut = torch.where(adv >= 0, above, below)
    bound = torch.where(adv >= 0, adv * (1 + c["clip_high"]), adv * (1 - c["clip_low"]))
    pg = -torch.where(cut, bound.expand_as(new), ratio * adv)
    g = -torch.where(cut, torch.zeros_like(new), ratio * adv)
    kl = torch.zeros_like(d)
    if ref is not None:
        e = new - ref
        if c["kl"] == "k1":
            kl, g_kl = e.double(), torch.ones_like(e)
        elif c["kl"] == "k2":
            kl, g_kl = (0.5 * e * e).double(), e
        else:
            kl, g_kl = torch.expm1(-e.double()) + e.double(), -torch.expm1(-e)
        g = g + c["kl_coef"] * g_kl
    count = mask.sum(1, keepdim=True).double()
    if c["reduction"] == "token":
        weight = 1.0 / count.sum().clamp(min=1).expand_as(count)
    else:
        weight = 1.0 / (count.clamp(min=1) * (count > 0).sum().clamp(min=1))
    mean = lambda v: (torch.where(mask, v.double(), 0.0).sum(1, keepdim=True) * weight).sum()  # noqa: E731
    policy, kl_mean = mean(pg), mean(kl)
    drift = mean(torch.expm1(d) - d)
    out = torch.stack([policy + c["kl_coef"] * kl_mean, policy, kl_mean, mean(above | below), drift, count.sum()]).float()
    return [out, torch.where(mask, g * weight.float(), torch.zeros_like(g))]


def _plain_preference(s, c):
    """D = sum(chosen - ref) - sum(rejected - ref) over the unmasked tokens (their means with `average`); loss of a pair:
    -(1 - e) log s(bD) - e log s(-bD), max(0, 1 - bD), or (D - 1 / 2b)^2; the mean over the pairs.  Sums in 64 bits."""
    beta, eps, pairs = c["beta"], c["smoothing"], c["pairs"]

    def side(name):
        v = s[name].double() if s["ref_" + name] is None else s[name].double() - s["ref_" + name].double()
        mask = s["mask_" + name] if s["mask_" + name] is not None else torch.ones_like(s[name], dtype=torch.bool)
        scale = 1.0 / mask.sum(1).clamp(min=1).double() if c["average"] else torch.ones(pairs, dtype=torch.float64, device="cuda")
        return torch.where(mask, v, 0.0).sum(1) * scale, mask, scale

    (dc, mask_c, scale_c), (dr, mask_r, scale_r) = side("chosen"), side("rejected")
    delta = dc - dr
    z = beta * delta
    softplus = lambda v: torch.clamp(v, min=0) + torch.log1p(torch.exp(-v.abs()))  # noqa: E731
    if c["kind"] == "sigmoid":
        loss = (1 - eps) * softplus(-z) + eps * softplus(z)
        g = -beta * ((1 - eps) / (1 + torch.exp(z)) - eps / (1 + torch.exp(-z)))
    elif c["kind"] == "hinge":
        loss, g = torch.clamp(1 - z, min=0), torch.where(z < 1, -beta, 0.0).double()
    else:
        off = delta - 0.5 / beta
        loss, g = off * off, 2 * off
    g = g / pairs
    zero = torch.zeros((), device="cuda")
    g_c = torch.where(mask_c, (g * scale_c).float().unsqueeze(1), zero)
    g_r = torch.where(mask_r, (-g * scale_r).float().unsqueeze(1), zero)
    out = torch.stack([loss.mean(), (z > 0).double().mean()]).float()
    return [out, torch.stack([beta * dc, beta * dr], 1).float(), g_c, g_r]


def _act(z, name):
    """(activation, its derivative)"""
    if name == "tanh":
        t = torch.tanh(z)
        return t, 1 - t * t
    if name == "relu":
        return torch.clamp(z, min=0), (z > 0).to(z.dtype)
    if name == "gelu":
        phi = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
        return z * phi, phi + z * torch.exp(-0.5 * z * z) * (0.5 / math.pi) ** 0.5
    if name == "silu":
        sig = 1 / (1 + torch.exp(-z))
        return z * sig, sig * (1 + z * (1 - sig))
    return z, torch.ones_like(z)


def _plain_linear(s, c):
    """y = act(x W^T + b) + residual, and for a gradient g of y:  u = g act'(.), g_x = u W, g_W = u^T x, g_b = sum u."""
    x, w, dtype = s["x"].float(), s["weight"].float(), s["x"].dtype
    z = x @ w.t()
    if s["bias"] is not None:
        z = z + s["bias"].float()
    y, d = _act(z, c["activation"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    out = [y.to(dtype)]
    if c["train"]:
        u = s["g"].float() * d
        out += [(u @ w).to(dtype), (u.t() @ x).to(dtype)]
        if s["bias"] is not None:
            out.append(u.sum(0).to(dtype))
    return out


# ------------------------------------------------------------------------------------------------- the framework's calls
def _own_logprobs(s, c):
    from ppo_amd import ops
    logp, entropy, lse = ops.token_logprobs_fwd(s["logits"], s["actions"], temperature=c["temperature"], ignore_index=IGNORE)
    if not c["train"]:
        return [logp, entropy]
    g = ops.token_logprobs_bwd(s["logits"], s["actions"], lse, entropy, s["g_logp"], s["g_entropy"],
                               temperature=c["temperature"], ignore_index=IGNORE)
    return [logp, entropy, g]


def _own_policy(s, c):
    from ppo_amd import ops
    out, g = ops.policy_kl_loss_fwd_bwd(s["new"], s["old"], s["adv"], mask=s["mask"], ref_lp=s["ref"], clip_low=c["clip_low"],
                                        clip_high=c["clip_high"], kl_coef=c["kl_coef"], kl=c["kl"], reduction=c["reduction"])
    return [out, g]


def _own_preference(s, c):
    from ppo_amd import ops
    return list(ops.preference_loss_fwd_bwd(
        s["chosen"], s["rejected"], s["ref_chosen"], s["ref_rejected"], s["mask_chosen"], s["mask_rejected"], beta=c["beta"],
        kind=c["kind"], label_smoothing=c["smoothing"], average=c["average"]))


def _own_linear(s, c):
    from ppo_amd import ops
    y, deriv = ops.linear_act_fwd(s["x"], s["weight"], s["bias"], c["activation"], s["residual"], want_deriv=c["train"])
    if not c["train"]:
        return [y]
    g_x, g_w, g_b = ops.linear_act_bwd(s["g"], s["x"], s["weight"], deriv, want_bias=s["bias"] is not None)
    return [y, g_x, g_w] + ([g_b] if g_b is not None else [])


def run(state):
    c = state["case"]
    if own:
        f = {"logprobs": _own_logprobs, "policy": _own_policy, "preference": _own_preference, "linear": _own_linear}[c["op"]]
    else:
        f = {"logprobs": _plain_logprobs, "policy": _plain_policy, "preference": _plain_preference, "linear": _plain_linear}[c["op"]]
    return f(state, c)


# ------------------------------------------------------------------------------------------------- work
def work(case):
    c = case
    if c["op"] == "logprobs":
        rows = c["batch"] * (c["length"] - c["shifted"])
        row = c["actions"] * SIZE[c["dtype"]]
        # forward: a logit is read, exp'd and summed twice; backward: its gradient is written, and the logits, which no
        # cache holds from the forward pass, are read once more
        per = 3 if c["train"] else 1
        return {"bytes": rows * (per * row + (8 + 8 + (8 if c["train"] else 0))), "flops": rows * c["actions"] * (14.0 if c["train"] else 6.0)}
    if c["op"] == "policy":
        n = c["batch"] * c["length"]
        adv = c["batch"] if c["per_sequence"] else n
        return {"bytes": n * (12 + (4 if c["ref"] else 0) + (c["mask"] != "none")) + 4 * adv + 24, "flops": n * 25.0}
    if c["op"] == "preference":
        n = c["pairs"] * (c["chosen"] + c["rejected"])
        return {"bytes": n * (8 + (4 if c["ref"] else 0) + (c["mask"] != "none")) + 8 * c["pairs"] + 8, "flops": n * 3.0}
    M, K, N, e = c["rows"], c["inputs"], c["outputs"], SIZE[c["dtype"]]
    forward = M * K + N * K + M * N * (1 + c["residual"]) + N * c["bias"]
    if not c["train"]:
        return {"bytes": e * forward, "flops": 2.0 * M * K * N}
    # backward: g, x and the weights once more, g_x, g_W and g_b
    return {"bytes": e * (forward + M * N + 2 * (M * K + N * K) + N * c["bias"]), "flops": 6.0 * M * K * N}


# ------------------------------------------------------------------------------------------------- exact
def _exact_logprobs(s, c):
    """Row by row in 64 bits, from the definition by softmax."""
    logits = s["logits"]
    A, t = c["actions"], c["temperature"]
    flat, act = logits.reshape(-1, A), s["actions"].reshape(-1)
    rows = act.numel()
    logp, entropy = (torch.zeros(rows, dtype=torch.float64, device="cuda") for _ in range(2))
    grads = []
    step = max(1, (1 << 28) // A)
    for at in range(0, rows, step):
        z = flat[at:at + step].double() / t
        a = act[at:at + step]
        live = a != IGNORE
        empty = (z == -math.inf).all(1)
        lp = torch.log_softmax(torch.where(empty.unsqueeze(1), 0.0, z), 1)
        p = lp.exp()
        finite = torch.where(lp == -math.inf, 0.0, lp)
        h = -(p * finite).sum(1)
        one = torch.where(live, a, 0)
        rows_here = torch.arange(a.numel(), device="cuda")
        value = torch.where(empty, -math.inf, lp[rows_here, one])
        logp[at:at + step] = torch.where(live, value, 0.0)
        entropy[at:at + step] = torch.where(live & ~empty, h, 0.0)
        if c["train"]:
            use = (live & ~empty).double()
            glp = (s["g_logp"].reshape(-1)[at:at + step].double() * use).unsqueeze(1)
            gh = (s["g_entropy"].reshape(-1)[at:at + step].double() * use).unsqueeze(1)
            g = -p * (glp + gh * (finite + h.unsqueeze(1)))
            g[rows_here, one] += glp.squeeze(1)
            grads.append((g / t).to(torch.float32 if c["dtype"] != "f32" else torch.float64))
    shape = s["actions"].shape
    out = [logp.reshape(shape), entropy.reshape(shape)]
    return out + ([torch.cat(grads).reshape(*shape, A)] if c["train"] else [])


def _exact_policy(s, c):
    new, old = s["new"].double(), s["old"].double()
    adv = s["adv"].double()
    adv = adv[:, None].expand_as(new) if adv.dim() == 1 else adv
    mask = torch.ones_like(new) if s["mask"] is None else s["mask"].double()
    leaf = new.clone().requires_grad_(True)
    r = torch.exp(leaf - old)
    lo, hi = 1 - c["clip_low"], 1 + c["clip_high"]
    pg = -torch.minimum(r * adv, torch.clamp(r, lo, hi) * adv)
    kl = torch.zeros_like(new)
    if s["ref"] is not None:
        q = s["ref"].double() - leaf
        kl = {"k1": -q, "k2": q * q / 2, "k3": torch.exp(q) - q - 1}[c["kl"]]
    per_row = mask.sum(1)
    if c["reduction"] == "token":
        w = mask / mask.sum().clamp(min=1)
    else:
        w = mask / per_row.clamp(min=1)[:, None] / (per_row > 0).sum().clamp(min=1)
    total = (w * (pg + c["kl_coef"] * kl)).sum()
    grad, = torch.autograd.grad(total, leaf)
    with torch.no_grad():
        out = [total, (w * pg).sum(), (w * kl).sum(), (w * ((r < lo) | (r > hi))).sum(), (w * (r - 1 - (leaf - old))).sum(), mask.sum()]
    return [torch.stack([v.detach() for v in out]), grad]


def _exact_preference(s, c):
    b, e = c["beta"], c["smoothing"]
    leaves, sums = [], []
    for name in ("chosen", "rejected"):
        lp = s[name].double().requires_grad_(True)
        mask = torch.ones_like(lp) if s["mask_" + name] is None else s["mask_" + name].double()
        ratio = lp if s["ref_" + name] is None else lp - s["ref_" + name].double()
        total = (ratio * mask).sum(1)
        sums.append(total / mask.sum(1).clamp(min=1) if c["average"] else total)
        leaves.append(lp)
    z = b * (sums[0] - sums[1])
    if c["kind"] == "sigmoid":
        loss = -(1 - e) * torch.nn.functional.logsigmoid(z) - e * torch.nn.functional.logsigmoid(-z)
    elif c["kind"] == "hinge":
        loss = torch.relu(1 - z)
    else:
        loss = (z / b - 1 / (2 * b)) ** 2
    g = torch.autograd.grad(loss.mean(), leaves)
    out = torch.stack([loss.mean(), (z > 0).double().mean()]).detach()
    return [out, torch.stack([b * sums[0], b * sums[1]], 1).detach(), g[0], g[1]]


def _exact_linear(s, c):
    x, w = s["x"].double().requires_grad_(True), s["weight"].double().requires_grad_(True)
    b = None if s["bias"] is None else s["bias"].double().requires_grad_(True)
    z = torch.nn.functional.linear(x, w, b)
    f = torch.nn.functional
    y = {"none": lambda v: v, "tanh": torch.tanh, "relu": f.relu, "gelu": f.gelu, "silu": f.silu}[c["activation"]](z)
    y = y if s["residual"] is None else y + s["residual"].double()
    out = [y.detach()]
    if c["train"]:
        out += list(torch.autograd.grad(y, [x, w] + ([b] if b is not None else []), s["g"].double()))
    return out


def exact(case, seed):
    s = prepare(case, seed)
    f = {"logprobs": _exact_logprobs, "policy": _exact_policy, "preference": _exact_preference, "linear": _exact_linear}
    return f[case["op"]](s, case)
