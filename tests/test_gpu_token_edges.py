"""GPU: token_logprobs, policy_kl_loss and preference_loss where a call needs more than one launch, and with infinite log-probs.

Row counts: a launch of the head's kernels holds 2^31 threads, i.e. 2^28, 2^25 and 2^23 rows at 8, 64 and 256 threads each.
Tolerances are those of test_gpu_token_losses.py."""
import math

import pytest
import torch

import token_reference as ref

pytestmark = pytest.mark.gpu
E = 2.0 ** -24


@pytest.mark.parametrize("rows,A", [(2 ** 28 + 37, 2), (2 ** 25 + 5, 40), (2 ** 23 + 3, 1030)])
def test_logprobs_rows_of_more_than_one_launch(rows, A):
    from ppo_amd import ops
    logits = torch.empty(rows, A, device="cuda", dtype=torch.bfloat16).normal_(generator=torch.Generator("cuda").manual_seed(A))
    actions = torch.randint(0, A, (rows,), device="cuda", dtype=torch.int32, generator=torch.Generator("cuda").manual_seed(rows))
    logp, H, stats = ops.token_logprobs_fwd(logits, actions)
    ones = torch.ones(1, device="cuda").expand(rows).contiguous()
    g = ops.token_logprobs_bwd(logits, actions, stats, None, ones)
    assert bool(torch.isfinite(logp).all()) and bool((logp < 0).all()) and bool((H > 0).all())
    most = 2 ** 31 // (8 if A <= 32 else 64 if A <= 1024 else 256)
    for at in (slice(0, 200), slice(most - 100, most + 3), slice(rows - 64, rows)):
        lp, h = ref.logprobs(logits[at], actions[at])
        assert bool(((logp[at].double() - lp).abs() <= 90 * E + 4 * E * lp.abs()).all())
        assert bool(((H[at].double() - h).abs() <= 180 * E * (1 + math.log(A))).all())
        want, size = ref.logprobs_grad(logits[at], actions[at], ones[at], None)
        tol = 2.0 ** -8 * want.abs() + (100 + 40 * (1 + math.log(A))) * E * size * 2 + 2.0 ** -126
        assert bool(((g[at].double() - want).abs() <= tol).all())


def test_preference_pairs_of_more_than_one_round():
    from ppo_amd import ops
    pairs = 2 ** 20 + 7
    gen = torch.Generator("cuda").manual_seed(3)
    c, r = (-torch.rand(pairs, n, device="cuda", generator=gen) for n in (3, 2))
    out, rewards, gc, gr = ops.preference_loss_fwd_bwd(c, r, beta=0.3)
    x, y = c.double().requires_grad_(True), r.double().requires_grad_(True)
    loss, acc, want = ref.preference(x, y, beta=0.3)
    wc, wr = torch.autograd.grad(loss, (x, y))
    loss = loss.detach()
    assert abs(float(out[0]) - float(loss)) <= 2 * E * float(loss) and abs(float(out[1]) - float(acc)) <= 2 * E
    assert bool(((rewards.double() - want).abs() <= 2 * E * want.abs() + 1e-12).all())
    for got, w in ((gc, wc), (gr, wr)):
        assert bool(((got.double() - w).abs() <= 2 * E * w.abs()).all())


@pytest.mark.parametrize("shape", [(1, 4), (300, 4), (2, 20000)])
def test_preference_of_an_impossible_rejected_answer(shape):
    """A rejected token of log-prob -inf: the margin is infinite, -ln s of it 0 and so is the gradient; the other way round inf."""
    from ppo_amd import ops
    c, r = torch.full(shape, -0.5, device="cuda"), torch.full(shape, -0.5, device="cuda")
    r[:, 1] = -math.inf
    out, _, gc, gr = ops.preference_loss_fwd_bwd(c, r)
    assert float(out[0]) == 0.0 and float(out[1]) == 1.0 and float(gc.abs().max()) == 0.0 and float(gr.abs().max()) == 0.0
    out, _, gc, gr = ops.preference_loss_fwd_bwd(c, r, kind="hinge")
    assert float(out[0]) == 0.0 and float(gc.abs().max()) == 0.0
    out, _, gc, gr = ops.preference_loss_fwd_bwd(r, c)
    pairs = shape[0]
    assert float(out[0]) == math.inf and float(out[1]) == 0.0
    assert bool(((gc + 0.1 / pairs).abs() <= 2 * E * 0.1 / pairs).all()) and torch.equal(gr, -gc)


@pytest.mark.parametrize("kl", ["k1", "k2", "k3"])
@pytest.mark.parametrize("B,L", [(2, 9), (300, 70)])
def test_policy_loss_with_a_reported_kl_only(B, L, kl):
    """kl_coef 0: an infinite estimate is reported and changes neither the loss nor its gradient."""
    from ppo_amd import ops
    gen = torch.Generator("cuda").manual_seed(B)
    new = -torch.rand(B, L, device="cuda", generator=gen)
    adv = torch.randn(B, L, device="cuda", generator=gen)
    old, refp = new - 0.1, new.clone()
    refp[1, 3] = -math.inf
    plain, g0 = ops.policy_kl_loss_fwd_bwd(new, old, adv)
    out, g = ops.policy_kl_loss_fwd_bwd(new, old, adv, ref_lp=refp, kl=kl)
    assert torch.equal(out[:2], plain[:2]) and torch.equal(out[3:], plain[3:]) and torch.equal(g, g0)
    assert float(out[2]) == math.inf


def test_logits_of_four_axes_and_no_tokens():
    from ppo_amd import ops
    for shape in ((2, 3, 0), (0, 3, 4), (2, 0, 4)):
        logits = torch.zeros(*shape, 7, device="cuda", requires_grad=True)
        logp, H = ops.token_logprobs(logits, torch.zeros(shape, dtype=torch.int64, device="cuda"))
        assert logp.shape == H.shape == shape
        (g,) = torch.autograd.grad(logp.sum() + H.sum(), logits)
        assert g.shape == logits.shape


@pytest.mark.parametrize("pairs", [3, 80, 81, 70000])
def test_preference_of_pairs_without_tokens(pairs):
    """D = 0 of every pair: ln 2, no pair preferred, rewards 0."""
    from ppo_amd import ops
    none = torch.zeros(pairs, 0, device="cuda")
    out, rewards, gc, gr = ops.preference_loss_fwd_bwd(none, none)
    assert abs(float(out[0]) - math.log(2.0)) <= 2 * E * math.log(2.0) and float(out[1]) == 0.0
    assert float(rewards.abs().max()) == 0.0 and gc.shape == gr.shape == (pairs, 0)


@pytest.mark.parametrize("kl,slope", [("k1", 1.0), ("k2", math.inf), ("k3", 1.0)])
@pytest.mark.parametrize("B,L", [(2, 9), (300, 70)])
def test_policy_loss_of_a_token_the_reference_excludes(B, L, kl, slope):
    """A reference log-prob of -inf, and one that is 2^26 lower: the estimate is infinite or 2^26 (its square), its derivative
    1 - e^-e = 1 (e for k2), and the other tokens' gradients are those without it.  A gradient is w (surrogate + c dk): three
    roundings of its terms."""
    from ppo_amd import ops
    gen = torch.Generator("cuda").manual_seed(B + 1)
    new = -torch.rand(B, L, device="cuda", generator=gen)
    adv = torch.randn(B, L, device="cuda", generator=gen)
    old, refp = new - 0.1, new - 0.2
    coef, far = 0.25, 2.0 ** 26
    want, g0 = ops.policy_kl_loss_fwd_bwd(new, old, adv, ref_lp=refp, kl_coef=coef, kl=kl)
    _, plain = ops.policy_kl_loss_fwd_bwd(new, old, adv)
    for low, dk in ((-math.inf, slope), (-far, {"k1": 1.0, "k2": far, "k3": 1.0}[kl])):
        refp[1, 3] = low
        out, g = ops.policy_kl_loss_fwd_bwd(new, old, adv, ref_lp=refp, kl_coef=coef, kl=kl)
        others = torch.ones_like(new, dtype=torch.bool)
        others[1, 3] = False
        assert torch.equal(g[others], g0[others])
        at = float(plain[1, 3]) + coef * dk / (B * L)
        if math.isinf(dk):
            assert float(g[1, 3]) == math.inf
        else:
            assert abs(float(g[1, 3]) - at) <= 4 * E * (abs(float(plain[1, 3])) + coef * dk / (B * L))
        if math.isinf(low):
            assert float(out[0]) == float(out[2]) == math.inf
        assert torch.equal(out[[1, 3, 4, 5]], want[[1, 3, 4, 5]])


@pytest.mark.parametrize("g_entropy,temperature", [(600.0, 1e-6), (65536.0, 1e-4), (1e28, 1e-6), (-3e9, 1.0)])
@pytest.mark.parametrize("A", [18, 300, 3000, 9000])
def test_masked_actions_under_large_entropy_gradients(A, g_entropy, temperature):
    """The gradient of an illegal action is 0, however large its factors: g_entropy / temperature up to 1e34.  Logits whose
    differences are of the temperature's size; tolerances as in test_gpu_token_losses.py."""
    from ppo_amd import ops
    gen = torch.Generator("cuda").manual_seed(A)
    logits = torch.randn(5, A, device="cuda", generator=gen) * temperature
    off = torch.rand(5, A, device="cuda", generator=gen) < 0.4
    off[:, 0] = False
    logits[off] = -math.inf
    logits[3, 1] = torch.finfo(torch.float32).min              # masked by the type's lowest value
    actions = torch.zeros(5, dtype=torch.int64, device="cuda")
    logp, H, stats = ops.token_logprobs_fwd(logits, actions, temperature)
    gh = torch.full_like(logp, g_entropy)
    g = ops.token_logprobs_bwd(logits, actions, stats, H, None, gh, temperature)
    want, size = ref.logprobs_grad(logits, actions, torch.zeros_like(gh), gh, temperature)
    assert bool((g[off] == 0).all()) and float(g[3, 1]) == 0.0
    tol = E * want.abs() + (100 + 40 * (1 + math.log(A))) * E * size * 2
    assert bool(((g.double() - want).abs() <= tol).all())


@pytest.mark.parametrize("rows,A,most_fwd,most_bwd", [(2 ** 27 + 5, 129, 2 ** 27, 2 ** 27), (2 ** 26 + 9, 257, 2 ** 26, None), (2 ** 25 + 5, 513, 2 ** 25, 2 ** 25),
                                                      (2 ** 23 + 3, 4097, 2 ** 23, 2 ** 23), (2 ** 22 + 3, 8193, None, 2 ** 22)])
def test_logprobs_rows_of_more_than_one_launch_each_kernel(rows, A, most_fwd, most_bwd):
    """bf16 rows just beyond what one launch of 2^31 threads holds (None: it holds them all): 129 actions have 16 lanes a row in both
    directions, 257 have 32 forward, 513 a wave in both, 4097 a workgroup of 256 in both, 8193 two workgroups backward.  Rows on both
    sides of the border, the first and the last, at the tolerances of test_gpu_token_losses.py."""
    from ppo_amd import ops
    torch.cuda.empty_cache()
    logits = torch.empty(rows, A, device="cuda", dtype=torch.bfloat16).normal_(generator=torch.Generator("cuda").manual_seed(A))
    actions = torch.randint(0, A, (rows,), device="cuda", dtype=torch.int32, generator=torch.Generator("cuda").manual_seed(rows))
    logp, H, stats = ops.token_logprobs_fwd(logits, actions)
    ones = torch.ones(1, device="cuda").expand(rows).contiguous()
    g = ops.token_logprobs_bwd(logits, actions, stats, None, ones)
    assert bool(torch.isfinite(logp).all()) and bool((logp < 0).all()) and bool((H > 0).all())
    slices = [slice(0, 64), slice(rows - 64, rows)] + [slice(m - 64, min(m + 64, rows)) for m in {most_fwd, most_bwd} - {None}]
    for at in slices:
        lp, h = ref.logprobs(logits[at], actions[at])
        assert bool(((logp[at].double() - lp).abs() <= 90 * E + 4 * E * lp.abs()).all())
        assert bool(((H[at].double() - h).abs() <= 180 * E * (1 + math.log(A))).all())
        want, size = ref.logprobs_grad(logits[at], actions[at], ones[at], None)
        tol = 2.0 ** -8 * want.abs() + (100 + 40 * (1 + math.log(A))) * E * size * 2 + 2.0 ** -126
        assert bool(((g[at].double() - want).abs() <= tol).all())
    # every row's gradient sums to 0: p_a - 1 against the rest, each rounded to bf16
    del logits
    step = max(1, 2 ** 31 // A)
    for at in range(0, rows, step):
        part = g[at:at + step]
        assert bool((part.sum(-1, dtype=torch.float32).abs() <= 2.0 ** -8 * part.abs().sum(-1, dtype=torch.float32) + 1e-3).all())
    del part, g
    torch.cuda.empty_cache()


@pytest.mark.parametrize("B,L,A", [(1, 1, 1), (3, 5, 18), (7, 33, 129), (2, 9, 513), (5, 3, 4099), (3, 20001, 3), (300, 71, 2)])
def test_nothing_beside_the_outputs_is_written(B, L, A):
    """The C entries with every output and workspace between guards, odd sizes, outputs at their least alignment: the bits of the
    wrappers' results, and the guards are as they were."""
    from ppo_amd import _lib, ops
    from test_gpu_linear_edges import _Guarded
    lib, gen, guard = _lib.load(), torch.Generator("cuda").manual_seed(B + L + A), _Guarded()
    stream = torch.cuda.current_stream().cuda_stream
    f32 = lambda view, *shape: view.clone().view(torch.float32).view(shape)  # noqa: E731
    actions = torch.randint(0, A, (B, L), device="cuda", generator=gen)
    for dt, dtype in ((0, torch.float32), (1, torch.bfloat16), (2, torch.float16)):
        logits = torch.randn(B, L, A, device="cuda", generator=gen).to(dtype)
        (pl, lp), (ph, h), (ps, st) = guard.of(B * L * 4, 4), guard.of(B * L * 4, 4), guard.of(B * L * 8, 8)
        (pg, g) = guard.of(logits.numel() * logits.element_size(), logits.element_size())
        assert lib.ppo_token_logprobs_fwd(logits.data_ptr(), dt, B, L, A, L * A, A, actions.data_ptr(), 8, 0.8, -100, pl, ph, ps, stream) == 0
        want = ops.token_logprobs_fwd(logits, actions, 0.8)
        assert lib.ppo_token_logprobs_bwd(logits.data_ptr(), dt, B, L, A, L * A, A, actions.data_ptr(), 8, ps, ph, pl, ph, 0.8, -100, pg, stream) == 0
        guard.check()
        assert torch.equal(f32(lp, B, L), want[0]) and torch.equal(f32(h, B, L), want[1]) and torch.equal(f32(st, B, L, 2), want[2])
        assert torch.equal(g.clone().view(dtype).view(B, L, A), ops.token_logprobs_bwd(logits, actions, want[2], want[1], want[0], want[1], 0.8))
    new, old, adv, refp = (-torch.rand(B, L, device="cuda", generator=gen) for _ in range(4))
    mask = torch.rand(B, L, device="cuda", generator=gen) < 0.7
    n = lib.ppo_policy_kl_loss_workspace_bytes(B, L)
    (po, out), (pg, g), (pw, _) = guard.of(24, 4), guard.of(B * L * 4, 4), guard.of(n, 8)
    assert lib.ppo_policy_kl_loss(new.data_ptr(), L, old.data_ptr(), L, adv.data_ptr(), L, 0, refp.data_ptr(), L, mask.data_ptr(), L, B, L, 0.2, 0.2, 0.1, 3, 1,
                                  po, pg, pw, n, stream) == 0
    guard.check()
    want = ops.policy_kl_loss_fwd_bwd(new, old, adv, mask, refp, kl_coef=0.1, reduction="sequence")
    assert torch.equal(f32(out, 6), want[0]) and torch.equal(f32(g, B, L), want[1])
    m = L // 2                                               # the rejected answers are shorter, none at all with one token
    n = lib.ppo_preference_loss_workspace_bytes(B, L, m)
    (po, out), (pr, rew), (pc, gc), (pj, gr), (pw, _) = guard.of(8, 4), guard.of(B * 8, 4), guard.of(B * L * 4, 4), guard.of(B * m * 4, 4), guard.of(n, 8)
    assert lib.ppo_preference_loss(new.data_ptr(), L, refp.data_ptr(), L, mask.data_ptr(), L, L, old.data_ptr(), L, adv.data_ptr(), L, mask.data_ptr(), L, m, B, 0,
                                   0.1, 0.0, 0, po, pr, pc, pj, pw, n, stream) == 0
    guard.check()
    want = ops.preference_loss_fwd_bwd(new, old[:, :m], refp, adv[:, :m], mask, mask[:, :m])
    for got, w in zip((out, rew, gc, gr), want):
        assert torch.equal(f32(got, *w.shape), w)
