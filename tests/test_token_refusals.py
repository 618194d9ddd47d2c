"""CPU: what the token-policy operators refuse -- shapes, types, ranges and host tensors in the wrappers, pointers, sizes
and strides at the C entries -- before anything is launched."""
import ctypes

import pytest
import torch

from ppo_amd import _lib, ops

BAD = _lib.PpoAmdError
INVALID = 1


def z(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


def test_logprobs_wrapper_refuses():
    a = z(2, 3, dtype=torch.int64)
    for logits, actions, kw in (
            (z(2, 3, 4, dtype=torch.float64), a, {}), (z(2, 3, 0), a, {}), (z(2, 3, 4), a.float(), {}), (z(2, 3, 4), a[:, :2], {}),
            (z(2, 3, 4), a.to(torch.int16), {}), (z(2, 3, 4), a, {"temperature": 0.0}), (z(2, 3, 4), a, {"temperature": -1.0}),
            (z(2, 3, 4), a, {"temperature": float("nan")}), (z(2, 3, 4), a, {"temperature": 1e7}), (z(2, 3, 4), None, {}), (None, a, {}),
            (z(2, 3, 4), a, {})):                         # the last one: host tensors
        with pytest.raises(BAD):
            ops.token_logprobs_fwd(logits, actions, **kw)
        with pytest.raises((BAD, AttributeError)):
            ops.token_logprobs(logits, actions, **kw)
    with pytest.raises(BAD):
        ops.token_logprobs_bwd(z(2, 3, 4), a, z(2, 3, 2), z(2, 3), None, None)


def test_policy_wrapper_refuses():
    x = z(3, 5)
    for args, kw in (
            ((z(5), z(5), z(5)), {}), ((x, z(3, 4), x), {}), ((x, x.double(), x), {}), ((x, x, z(4)), {}), ((x, x, None), {}), ((x, None, x), {}),
            ((x, x, x), {"mask": z(3, 5)}), ((x, x, x), {"mask": z(5, 3, dtype=torch.bool)}), ((x, x, x), {"ref_lp": x.half()}),
            ((x, x, x), {"kl": "k4"}), ((x, x, x), {"reduction": "sum"}), ((x, x, x), {"clip_low": 1.0}), ((x, x, x), {"clip_low": -0.1}),
            ((x, x, x), {"clip_high": -0.1}), ((x, x, x), {"clip_high": float("nan")}), ((x, x, x), {"kl_coef": float("nan")}), ((x, x, x), {})):
        with pytest.raises(BAD):
            ops.policy_kl_loss_fwd_bwd(*args, **kw)


def test_preference_wrapper_refuses():
    x, y = z(3, 5), z(3, 7)
    for args, kw in (
            ((z(5), y), {}), ((x, z(4, 7)), {}), ((x, y.half()), {}), ((x, y), {"ref_chosen_lp": y}), ((x, y), {"chosen_mask": z(3, 7, dtype=torch.bool)}),
            ((x, y), {"rejected_mask": z(3, 7)}), ((x, y), {"beta": 0.0}), ((x, y), {"beta": float("nan")}), ((x, y), {"kind": "none"}),
            ((x, y), {"label_smoothing": 0.5}), ((x, y), {"label_smoothing": -0.1}), ((x, None), {}), ((x, y), {})):
        with pytest.raises(BAD):
            ops.preference_loss_fwd_bwd(*args, **kw)


def test_c_entries_refuse():
    lib = _lib.load()
    buf = (ctypes.c_char * 4096)()
    p = (ctypes.addressof(buf) + 63) // 64 * 64
    fwd = lambda logits=p, dtype=0, b=1, n=1, A=4, bs=4, ts=4, act=p, ab=8, t=1.0, logp=p, H=p, st=p: lib.ppo_token_logprobs_fwd(  # noqa: E731
        logits, dtype, b, n, A, bs, ts, act, ab, t, -100, logp, H, st, None)
    assert fwd(b=0) == 0 and fwd(n=0) == 0
    for kw in ({"logits": None}, {"logits": p + 2}, {"dtype": 3}, {"b": -1}, {"n": -1}, {"A": 0}, {"bs": -1}, {"ts": -4}, {"act": None}, {"ab": 2},
               {"act": p + 4}, {"t": 0.0}, {"t": float("nan")}, {"t": float("inf")}, {"logp": None}, {"st": None}, {"st": p + 4}, {"b": 1 << 20, "n": 1 << 20},
               {"b": 1 << 20, "bs": 1 << 50}, {"A": 1 << 41}):
        assert fwd(**kw) == INVALID, kw
    bwd = lambda st=p, H=p, gl=p, gh=p, g=p, A=4, b=1, t=1.0: lib.ppo_token_logprobs_bwd(p, 0, b, 1, A, 4, 4, p, 8, st, H, gl, gh, t, -100, g, None)  # noqa: E731
    assert bwd(b=0) == 0
    for kw in ({"st": None}, {"H": None}, {"gl": None, "gh": None}, {"g": None}, {"g": p + 2}, {"A": 0}, {"t": -1.0}, {"A": 1 << 40, "b": 1 << 20}):
        assert bwd(**kw) == INVALID, kw
    assert lib.ppo_policy_kl_loss_workspace_bytes(2, 4) == 0
    n = lib.ppo_policy_kl_loss_workspace_bytes(2, 1 << 16)
    pol = lambda lp=p, s=1 << 16, adv=p, mask=p, b=2, n_=1 << 16, lo=0.2, hi=0.2, c=0.1, kl=3, out=p, g=p, ws=p, nws=n: lib.ppo_policy_kl_loss(  # noqa: E731
        lp, s, p, 4, adv, 4, 0, p, 4, mask, 4, b, n_, lo, hi, c, kl, 0, out, g, ws, nws, None)
    for kw in ({"lp": None}, {"lp": p + 2}, {"s": -1}, {"adv": None}, {"b": 0}, {"n_": 0}, {"b": 1 << 32}, {"n_": 1 << 31}, {"lo": 1.0}, {"lo": -0.5}, {"hi": -1.0},
               {"hi": float("inf")}, {"c": float("nan")}, {"kl": 0}, {"kl": 4}, {"out": None}, {"g": p + 1}, {"ws": None}, {"nws": n - 1}, {"ws": p + 4}):
        assert pol(**kw) == INVALID, kw
    assert lib.ppo_preference_loss_workspace_bytes(2, 4, 4) == 0
    n = lib.ppo_preference_loss_workspace_bytes(2, 1 << 16, 1 << 16)
    pref = lambda c=p, s=1 << 16, L=1 << 16, b=2, kind=0, beta=0.1, eps=0.0, out=p, rew=p, ws=p, nws=n: lib.ppo_preference_loss(  # noqa: E731
        c, s, p, 4, p, 4, L, p, 4, p, 4, p, 4, 1 << 16, b, kind, beta, eps, 0, out, rew, p, p, ws, nws, None)
    for kw in ({"c": None}, {"c": p + 2}, {"s": -1}, {"L": -1}, {"b": 0}, {"b": 1 << 29}, {"kind": 3}, {"beta": 0.0}, {"beta": float("nan")}, {"eps": 0.5},
               {"out": None}, {"rew": None}, {"ws": None}, {"nws": n - 1}):
        assert pref(**kw) == INVALID, kw


def test_linear_wrapper_refuses():
    x, w = z(3, 5), z(7, 5)
    for args, kw in (
            ((x, z(7, 4)), {}), ((x, z(7)), {}), ((x, None), {}), ((x.double(), w.double()), {}), ((x, w.half()), {}), ((x, w, z(5)), {}), ((x, w, z(7).half()), {}),
            ((x, w, None, "gelu2"), {}), ((x, w, None, "none", z(3, 5)), {}), ((x, w, None, "none", z(3, 7).half()), {}), ((x, z(0, 5)), {}), ((z(3, 0), z(7, 0)), {}),
            ((z(1, 1).expand(1 << 22, 1), z(1, 1)), {}), ((x, w), {})):
        with pytest.raises(BAD):
            ops.linear_act_fwd(*args, **kw)
    y = z(3, 7)
    for args, kw in (((z(3, 6), x, w), {}), ((y, x, w, z(3, 6)), {}), ((y.half(), x, w), {}), ((y, x, w, y.half()), {}), ((y, x, z(7)), {}), ((y, None, w), {}),
                     ((y, x, w), {})):
        with pytest.raises(BAD):
            ops.linear_act_bwd(*args, **kw)
    h = torch.bfloat16
    with pytest.raises(BAD, match="deriv is torch.float16"):
        ops.linear_act_bwd(z(3, 7, dtype=h), z(3, 5, dtype=h), z(7, 5, dtype=h), z(3, 7, dtype=h))


def test_linear_c_entries_refuse():
    lib = _lib.load()
    buf = (ctypes.c_char * 4096)()
    p = (ctypes.addressof(buf) + 63) // 64 * 64
    n = lib.ppo_linear_act_fwd_workspace_bytes(64, 8, 8, 1)
    assert lib.ppo_linear_act_fwd_workspace_bytes(8, 8, 8, 0) == 0 and n > 0
    fwd = lambda x=p, xs=8, w=p, ws_=8, b=p, r=p, rs=8, dt=1, M=64, K=8, N=8, act=1, y=p, d=p, ws=p, nws=n: lib.ppo_linear_act_fwd(  # noqa: E731
        x, xs, w, ws_, b, r, rs, dt, M, K, N, act, y, d, ws, nws, None)
    assert fwd(M=0) == 0
    for kw in ({"x": None}, {"x": p + 1}, {"xs": 7}, {"w": None}, {"ws_": 7}, {"w": p + 1}, {"b": p + 1}, {"r": p + 1}, {"rs": 7}, {"dt": 3}, {"dt": -1}, {"M": -1},
               {"K": 0}, {"N": 0}, {"M": 1 << 22}, {"K": 1 << 22, "xs": 1 << 22, "ws_": 1 << 22}, {"N": 1 << 22}, {"act": 5}, {"act": -1}, {"y": None}, {"y": p + 1},
               {"d": p + 1}, {"ws": None}, {"xs": 1 << 22}, {"ws_": 1 << 22}, {"ws": p + 8}, {"nws": n - 1}):
        assert fwd(**kw) == INVALID, kw
    n = lib.ppo_linear_act_bwd_workspace_bytes(16, 8, 8, 0)
    bwd = lambda g=p, gs=8, x=p, xs=8, w=p, ws_=8, d=p, dt=0, M=16, K=8, N=8, gx=p, gw=p, gb=p, ws=p, nws=n: lib.ppo_linear_act_bwd(  # noqa: E731
        g, gs, x, xs, w, ws_, d, dt, M, K, N, gx, gw, gb, ws, nws, None)
    for kw in ({"g": None}, {"g": p + 2}, {"gs": 7}, {"x": None}, {"xs": 7}, {"w": None}, {"ws_": 7}, {"d": p + 2}, {"dt": 3}, {"M": 0}, {"K": 0}, {"N": 0}, {"M": 1 << 22},
               {"gx": p + 2}, {"gw": p + 1}, {"gb": p + 2}, {"ws": None}, {"ws": p + 8}, {"nws": n - 1}):
        assert bwd(**kw) == INVALID, kw
    assert bwd(gx=None, gw=None, gb=None) == 0
