"""GPU: token_logprobs, policy_kl_loss and preference_loss against plain 64-bit forms.

Tolerances.  e = 2^-24 is half a step of f32.  A log-probability is (x - max) / t - ln s: three roundings of the first
term; s is a sum of at most 32 terms in a chunk, 16 chunks and 10 joins of lanes (3 roundings each), every term an exp2
(one step) of an argument with 3 roundings, |t| 2^t < 0.54: below 90 e in all, so 90 e + 4 e |log p|.  The entropy is
ln s - u / s with both of them that exact relative to 1 + ln A: 180 e (1 + ln A).  A gradient's terms carry the same
relative error (90 e, and 4 e |ln p| of the exponent), and the result is rounded to its type once."""
import math

import pytest
import torch

import token_reference as ref

pytestmark = pytest.mark.gpu
E = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
SMALLEST = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25}   # half a step of a subnormal (f16), flush (others)


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(gen, *shape, dtype=torch.float32):
    return torch.randn(tuple(shape), device="cuda", generator=gen).to(dtype)


def _check_logprobs(logits, actions, temperature=1.0, ignore=-100, seed=0):
    from ppo_amd import ops
    A = logits.shape[-1]
    logp, H, stats = ops.token_logprobs_fwd(logits, actions, temperature, ignore)
    want_lp, want_h = ref.logprobs(logits, actions, temperature, ignore)
    assert logp.dtype == H.dtype == torch.float32 and logp.shape == H.shape == actions.shape
    fin = torch.isfinite(want_lp)
    assert torch.equal(torch.isfinite(logp), fin) and torch.equal(logp[~fin].double(), want_lp[~fin])
    assert bool(((logp.double() - want_lp).abs()[fin] <= (90 * E + 4 * E * want_lp.abs())[fin]).all())
    assert bool(((H.double() - want_h).abs() <= 180 * E * (1 + math.log(A))).all())
    gen = _gen(seed + 1)
    gl, gh = _randn(gen, *actions.shape), _randn(gen, *actions.shape)
    for glp, gent in ((gl, gh), (gl, None), (None, gh)):
        g = ops.token_logprobs_bwd(logits, actions, stats, H, glp, gent, temperature, ignore)
        assert g.dtype == logits.dtype and g.shape == logits.shape and g.is_contiguous()
        want, size = ref.logprobs_grad(logits, actions, glp if glp is not None else torch.zeros_like(gh), gent, temperature, ignore)
        half = torch.finfo(logits.dtype).eps / 2
        lnp = 10 * (1 + math.log(A))                     # |ln p| where p is not negligible beside what the bound leaves
        tol = half * want.abs() + (100 + 4 * lnp) * E * size * 2 + SMALLEST[logits.dtype]
        assert bool(((g.double() - want).abs() <= tol).all()), float(((g.double() - want).abs() / tol).max())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("A", [1, 2, 3, 8, 9, 18, 31, 32, 33, 63, 64, 65, 255, 256, 257, 1000, 1024, 1025, 2048, 4095, 4096, 4097, 8192, 8195, 50001])
def test_logprobs_sizes(A, dtype):
    gen = _gen(A)
    for shape in ((), (1,), (37,), (3, 5)):
        logits = _randn(gen, *shape, A, dtype=dtype) * 3
        actions = torch.randint(0, A, shape, device="cuda", generator=gen)
        _check_logprobs(logits, actions.int() if len(shape) == 1 else actions, temperature=1.0 if len(shape) < 2 else 0.7)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,A", [(1500, 4100), (1030, 9001)])
def test_logprobs_many_rows(rows, A, dtype):
    """The kernels of a workgroup a row."""
    gen = _gen(rows)
    _check_logprobs(_randn(gen, rows, A, dtype=dtype) * 2, torch.randint(0, A, (rows,), device="cuda", generator=gen))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("A", [18, 200, 3000, 5001])
def test_logprobs_masks_and_ignored(A, dtype):
    gen = _gen(A + 1)
    B, T = 5, 9
    logits = _randn(gen, B, T, A, dtype=dtype) * 4
    actions = torch.randint(0, A, (B, T), device="cuda", generator=gen)
    off = torch.rand(B, T, A, device="cuda", generator=gen) < 0.5
    logits[off] = -math.inf                                # chosen actions among them: log p = -inf
    logits[1, 2] = -math.inf                               # a row without a legal action
    logits[2, 3] = -math.inf
    logits[2, 3, actions[2, 3]] = 7.0                      # one legal action: log p 0, entropy 0
    logits[3, 4] = torch.finfo(dtype).min                  # the lowest value throughout: uniform
    logits[3, 5, : A // 2] = torch.finfo(dtype).min        # ... and as a mask
    logits[3, 5, A // 2:] = 1.0
    logits[4, 0] = 3000.0                                  # a large common offset
    actions[0, 1] = -100
    logits[0, 1, 0] = math.nan                             # an ignored row is not used
    want_nan = logits.clone()
    want_nan[0, 1, 0] = 0.0
    from ppo_amd import ops
    logp, H, stats = ops.token_logprobs_fwd(logits, actions)
    assert float(logp[0, 1]) == 0.0 and float(H[0, 1]) == 0.0
    assert float(logp[1, 2]) == -math.inf and float(H[1, 2]) == 0.0
    assert float(logp[2, 3]) == 0.0 and float(H[2, 3]) == 0.0
    g = ops.token_logprobs_bwd(logits, actions, stats, H, torch.ones_like(logp), torch.ones_like(logp))
    assert float(g[0, 1].abs().max()) == 0.0 and float(g[1, 2].abs().max()) == 0.0 and bool(torch.isfinite(g).all())
    a = ops.token_logprobs_fwd(logits, actions)
    b = ops.token_logprobs_fwd(want_nan, actions)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    _check_logprobs(want_nan, actions)
    # the lowest value at a temperature that would overflow it
    low = torch.full((2, A), torch.finfo(dtype).min, dtype=dtype, device="cuda")
    logp = ops.token_logprobs_fwd(low, torch.zeros(2, dtype=torch.int64, device="cuda"), temperature=0.5)[0]
    assert float((logp + math.log(A)).abs().max()) <= 90 * E + 4 * E * math.log(A)


@pytest.mark.parametrize("A", [18, 100, 3000, 9000])
def test_logprobs_nan_inf_and_bad_actions(A):
    from ppo_amd import ops
    logits = _randn(_gen(5), 6, A)
    actions = torch.tensor([0, 1, A, -1, 5, 2], device="cuda")
    logits[0, 3] = math.nan
    logits[1, 4] = math.inf
    logits[4] = math.nan
    logp, H, stats = ops.token_logprobs_fwd(logits, actions)
    assert bool(torch.isnan(logp[:5]).all()) and bool(torch.isnan(H[:5]).all()) and bool(torch.isfinite(logp[5]))
    one = torch.ones_like(logp)
    g = ops.token_logprobs_bwd(logits, actions, stats, H, one, one)
    assert bool(torch.isnan(g[:5]).all()) and bool(torch.isfinite(g[5]).all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_logprobs_strided_views(dtype):
    """Shifted, sliced, transposed, expanded and unaligned logits are read as they lie and equal their contiguous copies."""
    from ppo_amd import ops
    gen = _gen(11)
    A = 5003
    base = _randn(gen, 4, 7, A + 3, dtype=dtype)
    views = [base[:, :-1, :A], base[:, 1:, 1:A + 1], base.transpose(0, 1)[..., 3:], base[:1, :, :A].expand(3, 7, A),
             base[0, 0, 2:A], base[:, 2, 1:], base.unsqueeze(1)[..., :A], base[..., : 2 * 900: 2]]
    for v in views:
        actions = torch.randint(0, v.shape[-1], v.shape[:-1], device="cuda", generator=gen)
        got = ops.token_logprobs_fwd(v, actions)
        want = ops.token_logprobs_fwd(v.contiguous(), actions)
        assert all(torch.equal(x, y) for x, y in zip(got, want))
        gl = _randn(gen, *actions.shape)
        assert torch.equal(ops.token_logprobs_bwd(v, actions, got[2], got[1], gl, gl), ops.token_logprobs_bwd(v.contiguous(), actions, got[2], got[1], gl, gl))
    none = base[:0, :, :A]
    logp, H, stats = ops.token_logprobs_fwd(none, torch.zeros(0, 7, dtype=torch.int64, device="cuda"))
    assert logp.shape == (0, 7) and ops.token_logprobs_bwd(none, torch.zeros(0, 7, dtype=torch.int64, device="cuda"), stats, H, logp).shape == none.shape


def test_logprobs_autograd_and_differences():
    from ppo_amd import ops
    gen = _gen(21)
    logits = (_randn(gen, 6, 10, 301) * 2).requires_grad_(True)
    actions = torch.randint(0, 301, (6, 10), device="cuda", generator=gen)
    cl, ch = _randn(gen, 6, 10), _randn(gen, 6, 10)
    logp, H = ops.token_logprobs(logits, actions, temperature=1.3)
    (g,) = torch.autograd.grad((cl * logp + ch * H).sum(), logits)
    lv = logits.detach().double().requires_grad_(True)
    wl, wh = ref.logprobs(lv, actions, 1.3)
    (want,) = torch.autograd.grad((cl * wl + ch * wh).sum(), lv)
    size = ref.logprobs_grad(logits.detach(), actions, cl, ch, 1.3)[1]
    assert bool(((g.double() - want).abs() <= E * want.abs() + 400 * E * size).all())
    # a difference of the 64-bit form along a random direction: truncation h^2, cancellation 1e-16 / h
    v, h = _randn(gen, 6, 10, 301).double(), 1e-5
    f = lambda x: float(sum((c.double() * t).sum() for c, t in zip((cl, ch), ref.logprobs(x, actions, 1.3))))  # noqa: E731
    diff = (f(lv.detach() + h * v) - f(lv.detach() - h * v)) / (2 * h)
    assert abs(diff - float((g.double() * v).sum())) <= 1e-5 * float((g.double() * v).abs().sum())
    # one output only, and no gradient at all
    (g1,) = torch.autograd.grad(ops.token_logprobs(logits, actions)[1].sum(), logits)
    (w1,) = torch.autograd.grad(ref.logprobs(lv, actions)[1].sum(), lv)
    assert float((g1.double() - w1).abs().max()) <= 1e-5
    assert not ops.token_logprobs(logits.detach(), actions)[0].requires_grad


# ------------------------------------------------------------------------------------------------- policy loss
def _policy_case(gen, B, L, mask_kind, per_sequence=False):
    old = -_randn(gen, B, L).abs()
    new = old + 0.2 * _randn(gen, B, L)
    refp = old + 0.4 * _randn(gen, B, L)
    adv = _randn(gen, B) if per_sequence else _randn(gen, B, L)
    mask = None
    if mask_kind == "ragged":
        n = torch.randint(0, L + 1, (B, 1), device="cuda", generator=gen)
        n[:1] = 0
        mask = torch.arange(L, device="cuda") < n
    elif mask_kind == "random":
        mask = (torch.rand(B, L, device="cuda", generator=gen) < 0.5).to(torch.uint8) * 3
    elif mask_kind == "nothing":
        mask = torch.zeros(B, L, dtype=torch.bool, device="cuda")
    return new, old, adv, mask, refp


def _check_policy(new, old, adv, mask, refp, kl, reduction, coef=0.3, lo=0.2, hi=0.28):
    """A term is a product of an exponential (two steps, one rounding of its argument, |d| < 2) and an advantage: 8 e; the
    KL's estimators have at most 8 roundings of |e| + k; the weights, the final sum and product 4 more."""
    from ppo_amd import ops
    out, g = ops.policy_kl_loss_fwd_bwd(new, old, adv, mask, refp, lo, hi, coef, kl, reduction)
    x = new.double().requires_grad_(True)
    want, w, a, r, k = ref.policy(x, old, adv, mask, refp, lo, hi, coef, kl, reduction)
    (wg,) = torch.autograd.grad(want[0], x)
    wg = torch.nan_to_num(wg)
    live = w > 0
    dist = torch.where(live, (new.double() - refp.double()).abs(), torch.zeros_like(w)) if refp is not None else torch.zeros_like(w)
    size = w * ((r * a).abs() + abs(coef) * (dist + k.abs() + 1) * (refp is not None))
    assert bool(((g.double() - wg).abs() <= 16 * E * size + 1e-38).all())
    assert bool((g[~live] == 0).all())
    bounds = [size.sum(), (w * (r * a).abs() * (1 + hi)).sum() + (w * a.abs()).sum() * (1 + hi), (w * (k.abs() + dist)).sum(), torch.ones(()), (w * (r + 1)).sum(), want[5]]
    for i in range(6):
        assert abs(float(out[i]) - float(want[i].detach())) <= 16 * E * float(bounds[i]) + (16 * E * float(bounds[1]) if i == 0 else 0.0), i


@pytest.mark.parametrize("mask_kind", ["none", "ragged", "random", "nothing"])
@pytest.mark.parametrize("B,L", [(1, 1), (1, 3), (3, 4), (4, 17), (7, 129), (64, 64), (300, 5), (33, 1000), (2, 20001), (1000, 33), (5000, 256), (3000, 257), (70000, 3)])
def test_policy_loss(B, L, mask_kind):
    for i, (kl, reduction) in enumerate((("k1", "token"), ("k2", "sequence"), ("k3", "token"), ("k3", "sequence"))):
        new, old, adv, mask, refp = _policy_case(_gen(B * L + i), B, L, mask_kind, per_sequence=i % 2 == 1)
        _check_policy(new, old, adv, mask, refp, kl, reduction)
        _check_policy(new, old, adv, mask, None, kl, reduction, coef=0.0, lo=0.0, hi=0.0)


def test_policy_loss_masked_tokens_are_not_used():
    from ppo_amd import ops
    for B, L in ((5, 37), (40, 700)):
        new, old, adv, mask, refp = _policy_case(_gen(3), B, L, "random")
        want = ops.policy_kl_loss_fwd_bwd(new, old, adv, mask, refp, kl_coef=0.1, reduction="sequence")
        off = mask == 0
        for t, bad in ((new, math.nan), (old, math.inf), (adv, math.nan), (refp, -math.inf)):
            t[off] = bad
        got = ops.policy_kl_loss_fwd_bwd(new, old, adv, mask, refp, kl_coef=0.1, reduction="sequence")
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert bool((got[1][off] == 0).all())


def test_policy_loss_strided_rows_and_repeats():
    """Rows of larger buffers at any offset, column-major and expanded inputs; the same call twice gives the same bits."""
    from ppo_amd import ops
    gen = _gen(8)
    for B, L in ((6, 50), (70, 301)):
        wide = [-_randn(gen, B, L + 9).abs() for _ in range(4)]
        new, old, adv, refp = (w[:, k:k + L] for k, w in enumerate(wide))
        mask = (torch.rand(B, L + 5, device="cuda", generator=gen) < 0.6)[:, 3:L + 3]
        got = ops.policy_kl_loss_fwd_bwd(new, old, adv, mask, refp, kl_coef=0.1)
        want = ops.policy_kl_loss_fwd_bwd(*(t.contiguous() for t in (new, old, adv, mask, refp)), kl_coef=0.1)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        cols = new.t().contiguous().t()
        got = ops.policy_kl_loss_fwd_bwd(cols, old, adv[:1].expand(B, L), mask, refp, kl_coef=0.1)
        want = ops.policy_kl_loss_fwd_bwd(new, old, adv[:1].repeat(B, 1), mask, refp, kl_coef=0.1)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_policy_loss_zero_sizes_and_autograd():
    from ppo_amd import ops
    for shape in ((0, 5), (5, 0), (0, 0)):
        z = torch.zeros(shape, device="cuda")
        out, g = ops.policy_kl_loss_fwd_bwd(z, z, z)
        assert g.shape == shape and float(out.abs().max()) == 0.0
    new, old, adv, mask, refp = _policy_case(_gen(4), 9, 77, "ragged")
    new.requires_grad_(True)
    loss, pl, kl, cf, drift = ops.policy_kl_loss(new, old, adv, mask, refp, kl_coef=0.2, reduction="sequence")
    (g,) = torch.autograd.grad(3.0 * loss, new)
    x = new.detach().double().requires_grad_(True)
    (want,) = torch.autograd.grad(3.0 * ref.policy(x, old, adv, mask, refp, coef=0.2, reduction="sequence")[0][0], x)
    assert float((g.double() - want).abs().max()) <= 1e-6 and not pl.requires_grad
    # along a random direction, away from the clip's kinks (none is within 1e-6 of these tokens' ratios)
    v, h = _randn(_gen(5), 9, 77).double(), 1e-7
    f = lambda t: float(ref.policy(t, old, adv, mask, refp, coef=0.2, reduction="sequence")[0][0])  # noqa: E731
    diff = (f(x.detach() + h * v) - f(x.detach() - h * v)) / (2 * h)
    assert abs(3 * diff - float((g.double() * v).sum())) <= 1e-5 * float((g.double() * v).abs().sum())


# ------------------------------------------------------------------------------------------------- preference loss
def _pairs(gen, B, Lc, Lr, mask_kind):
    out = []
    for L in (Lc, Lr):
        lp = -_randn(gen, B, L).abs()
        m = None
        if mask_kind == "ragged":
            n = torch.randint(0, L + 1, (B, 1), device="cuda", generator=gen)
            n[:1] = 0
            m = torch.arange(L, device="cuda") < n
        elif mask_kind == "random":
            m = (torch.rand(B, L, device="cuda", generator=gen) < 0.5).to(torch.uint8)
        out += [lp, lp + 0.1 * _randn(gen, B, L), m]
    return out


@pytest.mark.parametrize("mask_kind", ["none", "ragged", "random"])
@pytest.mark.parametrize("B,Lc,Lr", [(1, 1, 1), (1, 5, 0), (0, 3, 4), (4, 33, 40), (300, 7, 130), (20000, 3, 5), (70, 600, 5), (3, 9001, 8193), (2, 50001, 17), (17, 1000, 1001)])
def test_preference_loss(B, Lc, Lr, mask_kind):
    """Sums and the pair's loss are f64: what is left are a rounding of the loss, of a reward and of a gradient to f32."""
    from ppo_amd import ops
    for i, (kind, eps, average, with_ref) in enumerate((("sigmoid", 0.0, False, True), ("sigmoid", 0.2, True, True), ("hinge", 0.0, False, False),
                                                        ("ipo", 0.0, True, True))):
        c, rc, mc, r, rr, mr = _pairs(_gen(B + Lc + i), B, Lc, Lr, mask_kind)
        if not with_ref:
            rc = rr = None
        out, rewards, gc, gr = ops.preference_loss_fwd_bwd(c, r, rc, rr, mc, mr, 0.3, kind, eps, average)
        if B == 0:
            assert float(out.abs().max()) == 0.0 and rewards.shape == (0, 2) and gc.shape == (0, Lc)
            continue
        x, y = c.double().requires_grad_(True), r.double().requires_grad_(True)
        loss, acc, want = ref.preference(x, y, rc, rr, mc, mr, 0.3, kind, eps, average)
        wc, wr = torch.autograd.grad(loss, (x, y), allow_unused=True)
        assert abs(float(out[0]) - float(loss)) <= 2 * E * abs(float(loss)) + 1e-12 and abs(float(out[1]) - float(acc)) <= 2 * E
        assert bool(((rewards.double() - want).abs() <= 2 * E * want.abs() + 1e-12).all())
        for got, w, m in ((gc, wc, mc), (gr, wr, mr)):
            if got.numel():
                assert bool(((got.double() - w).abs() <= 2 * E * w.abs() + 1e-12).all())
                assert m is None or bool((got[m == 0] == 0).all())


def test_preference_loss_masked_views_halves_and_autograd():
    from ppo_amd import ops
    gen = _gen(31)
    for B, L in ((6, 45), (3, 9000)):
        both = -_randn(gen, 2 * B, L + 3).abs()
        refs = both + 0.1 * _randn(gen, 2 * B, L + 3)
        mask = torch.rand(2 * B, L + 3, device="cuda", generator=gen) < 0.7
        args = [t[k * B:(k + 1) * B, 1:L + 1] for t in (both, refs, mask) for k in (0, 1)]     # views: chosen, rejected rows
        want = ops.preference_loss_fwd_bwd(*(t.contiguous() for t in args), beta=0.2)
        both[~mask] = math.nan
        refs[~mask] = math.inf
        got = ops.preference_loss_fwd_bwd(*args, beta=0.2)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        c, r = args[0].clone().requires_grad_(True), args[1].clone().requires_grad_(True)
        loss, acc, rewards = ops.preference_loss(c, r, *args[2:], beta=0.2)
        gc, gr = torch.autograd.grad(2.0 * loss, (c, r))
        assert torch.equal(gc, 2.0 * got[2]) and torch.equal(gr, 2.0 * got[3]) and torch.equal(rewards, got[1])
        (only,) = torch.autograd.grad(ops.preference_loss(c.detach(), r, *args[2:], beta=0.2)[0], r)
        assert torch.equal(only, got[3])


def test_preference_loss_extremes():
    """Margins whose exponential overflows, the hinge at its corner, a difference of the loss."""
    from ppo_amd import ops
    for d, beta in ((2000.0, 1.0), (-2000.0, 1.0), (0.0, 0.5), (1.0, 1.0)):
        c, r = torch.full((1, 1), d, device="cuda"), torch.zeros(1, 1, device="cuda")
        for kind in ("sigmoid", "hinge", "ipo"):
            out, _, gc, gr = ops.preference_loss_fwd_bwd(c, r, beta=beta, kind=kind)
            x = c.double().requires_grad_(True)
            loss = ref.preference(x, r.double(), beta=beta, kind=kind)[0]
            assert abs(float(out[0]) - float(loss)) <= 2 * E * abs(float(loss)) and float(gc) == -float(gr)
            if kind != "hinge" or beta * d != 1.0:       # torch's clamp takes the other side of the corner
                (w,) = torch.autograd.grad(loss, x)
                assert abs(float(gc) - float(w)) <= 2 * E * abs(float(w)) + 1e-38
    gen = _gen(32)
    c, rc, mc, r, rr, mr = _pairs(gen, 5, 40, 50, "random")
    _, _, gc, gr = ops.preference_loss_fwd_bwd(c, r, rc, rr, mc, mr, beta=0.4, label_smoothing=0.1)
    v, u, h = _randn(gen, 5, 40).double(), _randn(gen, 5, 50).double(), 1e-6
    f = lambda s: float(ref.preference(c.double() + s * v, r.double() + s * u, rc, rr, mc, mr, 0.4, "sigmoid", 0.1)[0])  # noqa: E731
    want = float((gc.double() * v).sum() + (gr.double() * u).sum())
    assert abs((f(h) - f(-h)) / (2 * h) - want) <= 1e-6 * float((gc.double() * v).abs().sum() + (gr.double() * u).abs().sum()) + 1e-9


# ------------------------------------------------------------------------------------------------- streams, graphs
def _step(x):
    from ppo_amd import ops
    logits, actions, old, adv, mask = x
    logp, H, stats = ops.token_logprobs_fwd(logits, actions)
    out, g = ops.policy_kl_loss_fwd_bwd(logp, old, adv, mask, ref_lp=old, kl_coef=0.1, reduction="sequence")
    grad = ops.token_logprobs_bwd(logits, actions, stats, H, g, None)
    half = logp.shape[0] // 2
    pref = ops.preference_loss_fwd_bwd(logp[:half], logp[half:], old[:half], old[half:], mask[:half], mask[half:])
    return [logp, H, out, g, grad, *pref]


def _inputs(seed, B=6, L=40, A=700):
    gen = _gen(seed)
    logits = _randn(gen, B, L, A, dtype=torch.bfloat16)
    return [logits, torch.randint(0, A, (B, L), device="cuda", generator=gen), -6 - _randn(gen, B, L).abs(), _randn(gen, B, L),
            torch.rand(B, L, device="cuda", generator=gen) < 0.8]


@pytest.mark.parametrize("B,L", [(6, 40), (4, 5000)])
def test_captured_steps_replay(B, L):
    """Two captured graphs, replayed in turn with eager calls between them, give the eager results each time."""
    static = [_inputs(1, B, L), _inputs(2, B, L)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for s in static:
            _step(s)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for s in static:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_step(s))
        graphs.append(g)
    for turn in range(4):
        for k in (0, 1):
            fresh = _inputs(10 + 2 * turn + k, B, L)
            want = [t.clone() for t in _step(fresh)]
            for dst, src in zip(static[k], fresh):
                dst.copy_(src)
            graphs[k].replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(outs[k], want))


def test_another_stream_and_two_at_once():
    x = [_inputs(3), _inputs(4)]
    want = [[t.clone() for t in _step(s)] for s in x]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [None, None]
    for _ in range(3):
        for k in (0, 1):
            with torch.cuda.stream(streams[k]):
                got[k] = _step(x[k])
    torch.cuda.synchronize()
    for k in (0, 1):
        assert all(torch.equal(a, b) for a, b in zip(got[k], want[k]))
