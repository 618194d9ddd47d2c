"""GPU: linear_act forward and backward against 64-bit forms.

Tolerances.  h = half a step of the type relative to the value (2^-8 bf16, 2^-11 f16, 2^-24 f32), e = 2^-24.
A product of K terms: f32 accumulation of 16-bit inputs adds at most K e of sum |a b| in the worst case; f32 inputs add the
split's 2^-23 to that.  The matrix cores add in blocks and the errors are random: (8 + 4 sqrt(K)) e sum |a b| covers both with a
margin (a random walk of K steps of e / 2 stays below it by far more than six standard deviations).
y: h |y| + the product's error times the largest slope of the activation (1.13, gelu) + 32 e (|y| + 1) for its own evaluation.
g_x, g_W: u = g d is rounded to the type, d beforehand to f16 (bf16 layers) or f32: every term is off by (h + hd), all with
the same sign at worst; then h of the result.  z's own error reaches d by act'' <= 1.  Bounds are per element."""
import math

import pytest
import torch

import token_reference as ref

pytestmark = pytest.mark.gpu
E = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
ACTS = ["none", "tanh", "relu", "gelu", "silu"]


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _make(seed, M, K, N, dtype, bias=True, residual=True):
    g = _gen(seed)
    r = lambda *s: torch.randn(s, device="cuda", generator=g)  # noqa: E731
    x, w = r(M, K).to(dtype), (r(N, K) * K ** -0.5).to(dtype)
    return x, w, r(N).to(dtype) if bias else None, r(M, N).to(dtype) if residual else None, r(M, N).to(dtype)


def _product_error(K):
    return (8 + 4 * math.sqrt(K)) * E


def _check(x, w, b, r, g, act):
    from ppo_amd import ops
    dtype, K = x.dtype, x.shape[-1]
    h = torch.finfo(dtype).eps / 2
    hd = {torch.bfloat16: 2.0 ** -11, torch.float16: E, torch.float32: E}[dtype]
    tiny = 2.0 ** -24 if dtype != torch.float32 else 1e-37          # f16's subnormals, in d and in the outputs
    y, d = ops.linear_act_fwd(x, w, b, act, r, want_deriv=True)
    assert y.dtype == dtype and y.is_contiguous() and (d is None) == (act == "none")
    assert torch.equal(y, ops.linear_act_fwd(x, w, b, act, r)[0])    # the derivative changes nothing, and the same bits again
    leaves = [t.double().requires_grad_(True) for t in (x, w) + ((b,) if b is not None else ())]
    want = ref.linear(leaves[0], leaves[1], leaves[2] if b is not None else None, act, r)
    # error of z
    size = x.double().abs() @ w.double().abs().t()
    ez = _product_error(K) * size + 2 * E * ((b.double().abs() if b is not None else 0.0) + size)
    tol = h * want.abs() + 1.2 * ez + 32 * E * (want.abs() + 1 + (r.double().abs() if r is not None else 0.0)) + tiny
    assert bool(((y.double() - want).abs() <= tol).all()), float(((y.double() - want).abs() / tol).max())
    got = ops.linear_act_bwd(g, x, w, d, want_bias=b is not None)
    grads = torch.autograd.grad(want, leaves, g.double())
    # u and its error: d off by its rounding, by z's error (act'' <= 1; relu's jump where z is within its error of 0)
    z = ref.linear(x, w, b)
    zz = z.detach().requires_grad_(True)
    (dz,) = torch.autograd.grad(ref.linear(zz, torch.eye(zz.shape[1], device="cuda"), None, act).sum(), zz)
    jump = (z.abs() <= ez).double() if act == "relu" else torch.zeros_like(z)
    gd = g.double().abs()
    u = (g.double() * dz).abs()
    eu = gd * (hd * dz.abs() + ez + 32 * E + jump + tiny) * (act != "none") + tiny
    er = eu + h * u                                                   # after the rounding to the type
    M, N = g.shape
    for name, a, c, s, err, k in (("g_x", got[0], grads[0], u @ w.double().abs(), er @ w.double().abs(), N),
                                  ("g_w", got[1], grads[1], u.t() @ x.double().abs(), er.t() @ x.double().abs(), M),
                                  ("g_b", got[2], grads[2] if b is not None else None, u.sum(0), eu.sum(0), M)):
        if a is None:
            continue
        assert a.dtype == dtype and a.shape == c.shape and a.is_contiguous()
        tol = h * c.abs() + err + _product_error(k) * s + tiny
        assert bool(((a.double() - c).abs() <= tol).all()), (name, float(((a.double() - c).abs() / tol).max()))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K,N", [(1, 1, 1), (1, 7, 5), (1, 64, 16), (1, 1000, 333), (2, 513, 17), (4, 100, 33), (5, 64, 64), (8, 4096, 100), (9, 1, 1),
                                   (9, 33, 15), (16, 128, 17), (100, 64, 130), (127, 65, 129), (128, 128, 128), (129, 127, 257), (255, 192, 64), (256, 256, 256),
                                   (1000, 96, 40), (40, 2049, 300), (300, 1000, 31), (2047, 129, 65),
                                   (40, 1, 33), (33, 2, 70), (200, 3, 5), (100, 50, 1), (65, 4000, 2), (500, 31, 513)])
def test_sizes(M, K, N, dtype):
    for i, act in enumerate(ACTS if M * N < 40000 else ["none", "gelu"]):
        x, w, b, r, g = _make(M + K + N + i, M, K, N, dtype, bias=i != 1, residual=i != 2)
        _check(x, w, b, r, g, act)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K,N", [(4000, 130, 3100), (3584, 100, 3600)])
def test_large_tiles(M, K, N, dtype):
    """The tiles of 256 x 256, whole and cut, forward and in one of the gradients."""
    x, w, b, r, g = _make(M, M, K, N, dtype)
    _check(x, w, b, r, g, "silu")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K,N", [(20000, 64, 40), (20001, 63, 64), (9001, 18, 65), (64, 8001, 128), (50, 130, 9000), (35, 4999, 64), (66, 6000, 3),
                                   (70000, 33, 18)])
def test_narrow_sizes(M, K, N, dtype):
    """At most 64 of one dimension and, in one of the three products, many of k: tiles of their own and up to hundreds of sums a result."""
    _check(*_make(M + K + N, M, K, N, dtype), "tanh")


def test_the_most_rows_and_offsets_beyond_32_bits():
    """2^22 - 128 rows, and results of more than 2^31 elements: the last rows, and a sum over all of them."""
    from ppo_amd import ops
    M = 2 ** 22 - 128
    _check(*_make(5, M, 33, 18, torch.bfloat16, residual=False), "silu")
    g = _gen(6)
    x, w = torch.randn(M, 32, device="cuda", generator=g).bfloat16(), (torch.randn(640, 32, device="cuda", generator=g) / 6).bfloat16()
    y, d = ops.linear_act_fwd(x, w, None, "tanh", want_deriv=True)
    got = ops.linear_act_bwd(y, x, w, d)
    h = 2.0 ** -8
    for at in (slice(0, 70), slice(M - 300, M)):
        xs = x[at].double().requires_grad_(True)
        want = torch.tanh(xs @ w.double().t())
        ez = _product_error(32) * (xs.detach().abs() @ w.double().abs().t())
        assert bool(((y[at].double() - want).abs() <= h * want.abs() + 1.2 * ez + 32 * E).all())
        (gx,) = torch.autograd.grad(want, xs, y[at].double())
        u = (y[at].double() * (1 - want * want)).abs()
        err = (y[at].double().abs() * (2.0 ** -11 + ez + 32 * E) + h * u) @ w.double().abs()
        assert bool(((got[0][at].double() - gx).abs() <= h * gx.abs() + err + _product_error(640) * (u @ w.double().abs())).all())
    # g_b sums f32 products of the y and d that the backward pass was given
    want = sum((a.double() * b.double()).sum(0) for a, b in zip(y.split(1 << 18), d.split(1 << 18)))
    size = sum((a.double() * b.double()).abs().sum(0) for a, b in zip(y.split(1 << 18), d.split(1 << 18)))
    assert bool(((got[2].double() - want).abs() <= h * want.abs() + _product_error(M) * size).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [4, 5, 10, 11, 12, 13, 32, 33])
def test_few_rows_of_large_weights(rows, dtype):
    """Both sides of each border between the vector units and the matrix cores, weights in place and not (4.2 and 8.4 MB)."""
    for K in (1024, 1025):
        x, w, b, r, g = _make(rows, rows, K, 2100, dtype)
        _check(x, w, b, r, g, "gelu")


@pytest.mark.parametrize("dtype", DTYPES)
def test_long_sums(dtype):
    """Long inner dimensions: splits and their joining."""
    for M, K, N in ((130, 20000, 70), (20011, 40, 33), (12, 9000, 16)):
        x, w, b, r, g = _make(K, M, K, N, dtype)
        _check(x, w, b, r, g, "tanh")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M", [1, 7, 150])
def test_views_and_leading_axes(M, dtype):
    """Row-strided, unaligned, transposed and expanded inputs give the bits of their contiguous copies."""
    from ppo_amd import ops
    g = _gen(M)
    K, N = 192, 129
    big = torch.randn((M, 2 * K + 9), device="cuda", generator=g).to(dtype)
    wbig = torch.randn((N + 1, K + 5), device="cuda", generator=g).to(dtype)
    rbig = torch.randn((M, N + 3), device="cuda", generator=g).to(dtype)
    xs = [big[:, :K], big[:, 1:K + 1], big[:, 8:K + 8], big[:, : 2 * K: 2], big[:, :K].t().contiguous().t(), big[:1, :K].expand(M, K)]
    ws = [wbig[:N, :K], wbig[1:, 3:K + 3], wbig[:N, :K].t().contiguous().t()]
    b = torch.randn(2 * N, device="cuda", generator=g).to(dtype)[::2]
    for i, x in enumerate(xs):
        w = ws[i % len(ws)]
        r = rbig[:, i % 3:N + i % 3]
        y, d = ops.linear_act_fwd(x, w, b, "gelu", r, want_deriv=True)
        assert torch.equal(y, ops.linear_act_fwd(x.contiguous(), w.contiguous(), b.contiguous(), "gelu", r.contiguous())[0])
        got = ops.linear_act_bwd(r, x, w, d)
        want = ops.linear_act_bwd(r.contiguous(), x.contiguous(), w.contiguous(), d)
        assert all(torch.equal(p, q) for p, q in zip(got, want))
    x3 = torch.randn((3, M, K), device="cuda", generator=g).to(dtype)
    y3, d3 = ops.linear_act_fwd(x3, ws[0], b, "tanh", want_deriv=True)
    y2, _ = ops.linear_act_fwd(x3.view(-1, K), ws[0], b, "tanh")
    assert y3.shape == (3, M, N) and torch.equal(y3.view(-1, N), y2)
    assert ops.linear_act_bwd(y3, x3, ws[0], d3)[0].shape == x3.shape
    y1 = ops.linear_act_fwd(x3[0, 0], ws[0])[0]
    assert y1.shape == (N,)
    empty = x3[:, :0]
    y0, d0 = ops.linear_act_fwd(empty, ws[0], b, "tanh", want_deriv=True)
    gx, gw, gb = ops.linear_act_bwd(y0, empty, ws[0], d0)
    assert y0.shape == (3, 0, N) and gx.shape == empty.shape and float(gw.abs().max()) == 0.0 and float(gb.abs().max()) == 0.0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K,N", [(3, 70, 40), (150, 37, 130), (150, 70, 130), (260, 100, 301), (300, 1031, 70)])
def test_what_lies_beside_the_operands_is_not_used(M, K, N, dtype):
    """Operands cut out of buffers that hold NaN everywhere else, at even and odd strides and offsets."""
    from ppo_amd import ops
    x, w, b, r, g = _make(M, M, K, N, dtype)

    def inside(t, left, right):
        if t.dim() == 1:
            return inside(t.unsqueeze(0), left, right)[0]
        big = torch.full((t.shape[0] + 2, t.shape[1] + left + right), math.nan, dtype=t.dtype, device="cuda")
        big[1:-1, left:left + t.shape[1]] = t
        return big[1:-1, left:left + t.shape[1]]

    for left, right in ((2, 4), (1, 2), (0, 3), (8, 8)):
        X, W, B, R, G = (inside(t, left, right) for t in (x, w, b, r, g))
        y, d = ops.linear_act_fwd(X, W, B, "tanh", R, want_deriv=True)
        want, dw = ops.linear_act_fwd(x, w, b, "tanh", r, want_deriv=True)
        assert torch.allclose(y, want, rtol=8 * torch.finfo(dtype).eps, atol=8 * torch.finfo(dtype).eps)
        got = ops.linear_act_bwd(G, X, W, d)
        for p, q in zip(got, ops.linear_act_bwd(g, x, w, dw)):
            assert bool(torch.isfinite(p).all())
            assert float((p - q).float().abs().max()) <= 8 * torch.finfo(dtype).eps * float(q.float().abs().max())
        # without an activation the gradient itself is read in place
        for p, q in zip(ops.linear_act_bwd(G, X, W), ops.linear_act_bwd(g, x, w)):
            assert bool(torch.isfinite(p).all())
            assert float((p - q).float().abs().max()) <= 8 * torch.finfo(dtype).eps * float(q.float().abs().max())


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_do_not_reach_each_other(dtype):
    """A NaN or an infinity in a row of x stays in that row of y; one in a row of W in that column; nothing behind the
    outputs is written."""
    from ppo_amd import ops
    for M, K, N in ((3, 70, 40), (200, 70, 300), (300, 1000, 270)):
        x, w, b, r, _ = _make(M, M, K, N, dtype)
        x[1, 3] = math.nan
        w[5, 2] = math.inf
        y = ops.linear_act_fwd(x, w, b, "none", r)[0]
        bad = torch.zeros(M, N, dtype=torch.bool, device="cuda")
        bad[1] = True
        bad[:, 5] = True
        assert torch.equal(~torch.isfinite(y), bad)


def test_activation_extremes():
    """Inputs whose exponentials overflow, and infinities, at one row and on the matrix cores."""
    from ppo_amd import ops
    vals = [0.0, 1e-30, -1e-30, 1e-4, -1e-4, 0.05, -0.05, 3.0, -3.0, 9.0, -9.0, 40.0, -40.0, 200.0, -200.0, 1e30, -1e30]
    for dtype, M in ((torch.float32, 1), (torch.float32, 20), (torch.bfloat16, 20)):
        z = torch.tensor(vals, device="cuda").to(dtype)
        n = z.numel()
        x = torch.zeros(M, n, dtype=dtype, device="cuda")
        for act in ACTS:
            y, d = ops.linear_act_fwd(x, torch.eye(n, dtype=dtype, device="cuda"), z, act, want_deriv=True)
            zz = z.double().requires_grad_(True)
            want = ref.linear(zz.unsqueeze(0), torch.eye(n, device="cuda", dtype=torch.float64), None, act)[0]
            (dw,) = torch.autograd.grad(want.sum(), zz)
            h = torch.finfo(dtype).eps / 2
            assert bool(((y[-1].double() - want).abs() <= h * want.abs() + 32 * E * (want.abs() + want.abs().clamp(max=1)) + 1e-37).all()), act
            if d is not None:
                # f32: 40 e of the value plus what 40 e of the terms that cancel leaves; f16: its half step
                tol = (2.0 ** -11 if dtype == torch.bfloat16 else 0.0) * dw.abs() + 64 * E * (dw.abs() + 1e-3 + (zz.abs() < 30).double()) + 1e-37
                assert bool(((d[-1].double() - dw).abs() <= tol).all()), act


@pytest.mark.parametrize("dtype", DTYPES)
def test_autograd_and_differences(dtype):
    from ppo_amd import ops
    x, w, b, r, g = _make(77, 90, 150, 70, dtype)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b, r)]
    y = ops.linear_act(leaves[0].view(9, 10, 150), leaves[1], leaves[2], "gelu", leaves[3].view(9, 10, 70))
    got = torch.autograd.grad(y, leaves, g.view(9, 10, 70))
    _, d = ops.linear_act_fwd(x, w, b, "gelu", r, want_deriv=True)
    want = ops.linear_act_bwd(g, x, w, d)
    assert all(torch.equal(p, q) for p, q in zip(got, (*want, g)))
    # some of the leaves
    only = torch.autograd.grad(ops.linear_act(x, leaves[1], None, "silu"), leaves[1], g)[0]
    assert only.shape == w.shape
    assert not ops.linear_act(x, w, b).requires_grad
    # a difference of the 64-bit form along random directions; the gradients' own roundings are what is allowed
    gen = _gen(5)
    vs = [torch.randn(t.shape, device="cuda", generator=gen, dtype=torch.float64) for t in (x, w, b)]
    h = 1e-5
    f = lambda s: float((ref.linear(x.double() + s * vs[0], w.double() + s * vs[1], b.double() + s * vs[2], "gelu", r) * g.double()).sum())  # noqa: E731
    diff = (f(h) - f(-h)) / (2 * h)
    mine = sum(float((p.double() * v).sum()) for p, v in zip(got, vs))
    size = sum(float((p.double() * v).abs().sum()) for p, v in zip(got, vs))
    assert abs(diff - mine) <= (4 * torch.finfo(dtype).eps + 1e-6) * size


@pytest.mark.parametrize("M", [4, 300])
def test_captured_layers_replay(M):
    """Two captured forward and backward passes replay to the eager bits, eager calls between."""
    from ppo_amd import ops

    def step(s):
        x, w, b, r, g = s
        y, d = ops.linear_act_fwd(x, w, b, "gelu", r, want_deriv=True)
        return [y, *ops.linear_act_bwd(g, x, w, d)]

    statics = [list(_make(k, M, 500, 120, torch.bfloat16)) for k in (1, 2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for s in statics:
            step(s)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for s in statics:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(s))
        graphs.append(g)
    for turn in range(3):
        for k in (0, 1):
            fresh = _make(10 + 2 * turn + k, M, 500, 120, torch.bfloat16)
            want = [t.clone() for t in step(fresh)]
            for dst, src in zip(statics[k], fresh):
                dst.copy_(src)
            graphs[k].replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, c) for a, c in zip(outs[k], want))


def test_two_streams_at_once():
    from ppo_amd import ops
    sets = [_make(k, 700, 600, 500, torch.float32) for k in (3, 4)]

    def step(s):
        x, w, b, r, g = s
        y, d = ops.linear_act_fwd(x, w, b, "tanh", r, want_deriv=True)
        return [y, *ops.linear_act_bwd(g, x, w, d)]

    want = [step(s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [None, None]
    for _ in range(3):
        for k in (0, 1):
            with torch.cuda.stream(streams[k]):
                got[k] = step(sets[k])
    torch.cuda.synchronize()
    for k in (0, 1):
        assert all(torch.equal(a, c) for a, c in zip(got[k], want[k]))


@pytest.mark.parametrize("loss", ["policy", "preference"])
def test_token_policy_end_to_end(loss):
    """The operators as they are used together: a residual trunk and a wide head, log-probs and entropy of the actions
    taken, a masked loss -- every parameter's gradient against the same net in 64 bits.  All of it is f32, so that what
    separates the two is rounding: 1e-4 of the largest element of a gradient, where its relative error in f32 is a few 1e-6."""
    from ppo_amd import ops
    gen = _gen(9)
    r = lambda *s: torch.randn(s, device="cuda", generator=gen)  # noqa: E731
    B, L, H, A = 6, 33, 96, 515
    obs = r(B, L, H)
    params = [r(128, H) / H ** 0.5, 0.1 * r(128), r(H, 128) / 128 ** 0.5, 0.1 * r(H), r(A, H) / H ** 0.5, 0.1 * r(A)]
    actions = torch.randint(0, A, (B, L), device="cuda", generator=gen)
    mask = torch.arange(L, device="cuda") < torch.tensor([[33], [1], [0], [20], [7], [32]], device="cuda")
    actions[~mask] = -100
    old = -6 - 0.3 * r(B, L).abs()
    refp, adv = old + 0.1 * r(B, L), r(B)

    def net(ps, lin, logprobs):
        h = lin(obs.to(ps[0].dtype), ps[0], ps[1], "gelu", None)
        h = lin(h, ps[2], ps[3], "none", obs.to(ps[0].dtype))
        return logprobs(lin(h, ps[4], ps[5], "none", None), actions)

    mine = [p.clone().requires_grad_(True) for p in params]
    logp, ent = net(mine, ops.linear_act, ops.token_logprobs)
    theirs = [p.double().requires_grad_(True) for p in params]
    flat = lambda x, w, b, a, q: ref.linear(x.reshape(-1, x.shape[-1]), w, b, a, None if q is None else q.reshape(-1, q.shape[-1])).view(*x.shape[:-1], -1)  # noqa: E731
    wlogp, went = net(theirs, flat, ref.logprobs)
    if loss == "policy":
        a = ops.policy_kl_loss(logp, old, adv, mask, refp, kl_coef=0.1)[0] - 0.01 * (ent * mask).sum() / mask.sum()
        b = ref.policy(wlogp, old, adv, mask, refp, coef=0.1)[0][0] - 0.01 * (went * mask).sum() / mask.sum()
    else:
        a = ops.preference_loss(logp[:3], logp[3:], refp[:3], refp[3:], mask[:3], mask[3:])[0]
        b = ref.preference(wlogp[:3], wlogp[3:], refp[:3], refp[3:], mask[:3], mask[3:])[0]
    assert abs(float(a.detach()) - float(b.detach())) <= 1e-5 * abs(float(b.detach())) + 1e-6
    for p, q in zip(torch.autograd.grad(a, mine), torch.autograd.grad(b, theirs)):
        assert float((p.double() - q).abs().max()) <= 1e-4 * float(q.abs().max())
