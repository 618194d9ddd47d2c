"""CPU: how the token-policy operators may be called, seen from what they refuse before anything is launched."""
import ctypes

import pytest
import torch

from ppo_amd import _lib, ops

BAD = _lib.PpoAmdError


def z(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


CALLS = [
    (ops.token_logprobs_fwd, {"logits": z(2, 3, 4), "actions": z(2, 3, dtype=torch.int64)}),
    (ops.token_logprobs_bwd, {"logits": z(2, 3, 4), "actions": z(2, 3, dtype=torch.int64), "stats": z(2, 3, 2), "entropy": z(2, 3), "g_logp": z(2, 3)}),
    (ops.policy_kl_loss_fwd_bwd, {"new_lp": z(3, 5), "old_lp": z(3, 5), "adv": z(3)}),
    (ops.preference_loss_fwd_bwd, {"chosen_lp": z(3, 5), "rejected_lp": z(3, 4)}),
    (ops.linear_act_fwd, {"x": z(3, 5), "weight": z(4, 5)}),
    (ops.linear_act_bwd, {"g": z(3, 4), "x": z(3, 5), "weight": z(4, 5)}),
    (ops.token_logprobs, {"logits": z(2, 3, 4), "actions": z(2, 3, dtype=torch.int64)}),
    (ops.policy_kl_loss, {"new_lp": z(3, 5), "old_lp": z(3, 5), "adv": z(3)}),
    (ops.preference_loss, {"chosen_lp": z(3, 5), "rejected_lp": z(3, 4)}),
    (ops.linear_act, {"x": z(3, 5), "weight": z(4, 5)}),
]


@pytest.mark.parametrize("fn,args", CALLS, ids=[c[0].__name__ for c in CALLS])
def test_every_argument_may_be_named(fn, args):
    """Host tensors: the refusal that comes after all checks of shapes and types, however the call is written."""
    with pytest.raises(BAD, match="HIP device tensors"):
        fn(**args)
    with pytest.raises(BAD, match="HIP device tensors"):
        fn(*args.values())
    with pytest.raises(TypeError):
        fn()


@pytest.mark.parametrize("fn,args", CALLS, ids=[c[0].__name__ for c in CALLS])
def test_forward_mode_inputs_are_refused(fn, args):
    """A tangent (torch.autograd.forward_ad) on any of the inputs would be lost: an error, also where a gradient is recorded."""
    for key, t in args.items():
        if not t.is_floating_point():
            continue
        for grad in (False, True):
            with torch.autograd.forward_ad.dual_level():
                dual = torch.autograd.forward_ad.make_dual(t.clone().requires_grad_(grad), torch.ones_like(t))
                with pytest.raises(BAD, match="forward-mode"):
                    fn(**{**args, key: dual})
                with torch.no_grad(), pytest.raises(BAD, match="forward-mode"):
                    fn(**{**args, key: dual})
                with pytest.raises(BAD, match="HIP device tensors"):       # inside the level, but without tangents
                    fn(**args)


def _on_the_host(monkeypatch):
    """policy_kl_loss and preference_loss with a loss sum x^2 in the kernels' place: what their autograd nodes do needs no GPU."""
    monkeypatch.setattr(ops, "policy_kl_loss_fwd_bwd", lambda new, *a, **k: (torch.full((6,), float((new * new).sum())), 2 * new))
    monkeypatch.setattr(ops, "preference_loss_fwd_bwd", lambda c, r, *a, **k: (torch.full((2,), float((c * c).sum() + (r * r).sum())), z(2, 2), 2 * c, 2 * r))


@pytest.mark.parametrize("which", ["policy", "preference"])
def test_second_derivatives_of_the_losses_raise(which, monkeypatch):
    """The gradients come from the kernels as constants: a second derivative would leave out the loss's own curvature."""
    _on_the_host(monkeypatch)
    x = torch.arange(6.0).reshape(2, 3).requires_grad_(True)
    loss = ops.policy_kl_loss(x, x, x)[0] if which == "policy" else ops.preference_loss(x, z(2, 3))[0]
    (g,) = torch.autograd.grad(loss * loss, x, create_graph=True)
    assert torch.equal(g, 2 * loss.detach() * 2 * x.detach())
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()


def test_pairs_without_tokens_are_shared_out():
    """Both sides of length 0: as soon as there are more pairs than one workgroup takes in a few turns the others have work, and a
    workspace for its results, as with one token a side."""
    lib = _lib.load()
    for pairs in (1, 8, 80, 81, 5000, 1 << 20):
        one, none = (lib.ppo_preference_loss_workspace_bytes(pairs, n, 0) for n in (1, 0))
        assert one == none and (none > 0) == (pairs > 80), pairs


@pytest.mark.parametrize("kl_coef", [float("inf"), -float("inf"), 1e31, 1e300])
def test_kl_coefficients_that_f32_does_not_hold_are_refused(kl_coef):
    """As infinity they made a token whose estimate is 0 NaN."""
    x = z(3, 5)
    for fn in (ops.policy_kl_loss, ops.policy_kl_loss_fwd_bwd):
        with pytest.raises(BAD, match="kl_coef"):
            fn(x, x, x, ref_lp=x, kl_coef=kl_coef)
    buf = (ctypes.c_char * 4096)()
    p = (ctypes.addressof(buf) + 63) // 64 * 64
    assert _lib.load().ppo_policy_kl_loss(p, 4, p, 4, p, 4, 0, p, 4, p, 4, 2, 4, 0.2, 0.2, kl_coef, 3, 0, p, p, None, 0, None) == 1


def test_preparing_more_than_2_36_elements_is_refused():
    """u of 2^22 - 128 rows and 16500 outputs, and an input of as many odd columns: no launch holds their tiles of 64 x 64."""
    lib = _lib.load()
    buf = (ctypes.c_char * 4096)()
    p = (ctypes.addressof(buf) + 63) // 64 * 64
    rows, wide = (1 << 22) - 128, 16501
    for outputs, inputs in ((wide, 8), (8, wide)):
        n = max(lib.ppo_linear_act_fwd_workspace_bytes(rows, inputs, outputs, 1), lib.ppo_linear_act_bwd_workspace_bytes(rows, inputs, outputs, 1))
        assert n > 1 << 36
        if inputs == wide:
            assert lib.ppo_linear_act_fwd(p, inputs, p, inputs, None, None, 0, 1, rows, inputs, outputs, 0, p, None, p, n, None) == 1
        else:
            assert lib.ppo_linear_act_bwd(p, outputs, p, inputs, p, inputs, p, 1, rows, inputs, outputs, p, p, p, p, n, None) == 1
