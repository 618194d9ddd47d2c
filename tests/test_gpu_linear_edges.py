"""GPU: linear_act's activations in f32 over fine grids and at infinite arguments, and its products where operands are infinite.

e = 2^-24, half a step of f32."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
E = 2.0 ** -24


def _of_bias(z, act, rows=1):
    """(y, d) of a layer whose products are 0: act(z) and act'(z) of its bias z, on the vector units (1 row) or the matrix cores"""
    from ppo_amd import ops
    x, w = torch.zeros(rows, 2, device="cuda", dtype=z.dtype), torch.zeros(z.numel(), 2, device="cuda", dtype=z.dtype)
    y, d = ops.linear_act_fwd(x, w, z, act, want_deriv=True)
    return y[-1], d[-1]


@pytest.mark.parametrize("low,high", [(-12.0, 12.0), (-80.0, 80.0)])
def test_silu_derivative_keeps_its_digits(low, high):
    """d = s (1 + z r), s = s(z), r = s(-z).  e^-|z| is good to 4 half steps (an exp2 of 2, its correction, a product), 1 / (1 + e) to 3,
    their product to 8.  z >= 0: s 3, z r <= 0.28 to 9, the sum 1, the product 1: below 8 d.  z < 0: s 8 of d (and 1 for the product),
    r 3 and z r 1 more of s |z| <= 0.28, the sum 1 of s max(1, |1 + z r|): below 9 d + 2.  Bound: e (9 |d| + 2)."""
    z = torch.linspace(low, high, 1 << 20, device="cuda")
    x = z.double()
    s, r = torch.sigmoid(x), torch.sigmoid(-x)
    want = s * (1 + x * r)
    for rows in (1, 40):
        d = _of_bias(z[:: 1 if rows == 1 else 64].contiguous(), "silu", rows)[1].double()
        w = want[:: 1 if rows == 1 else 64]
        assert bool(((d - w).abs() <= E * (9 * w.abs() + 2) + 1e-37).all()), float(((d - w).abs() / (9 * w.abs() + 2)).max() / E)


LIMITS = {  # act(z), act'(z) for z = inf and -inf
    "none": (math.inf, -math.inf, None, None), "tanh": (1.0, -1.0, 0.0, 0.0), "relu": (math.inf, 0.0, 1.0, 0.0),
    "gelu": (math.inf, 0.0, 1.0, 0.0), "silu": (math.inf, 0.0, 1.0, 0.0)}


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act", list(LIMITS))
@pytest.mark.parametrize("M,K,N", [(1, 70, 40), (8, 2, 3), (300, 70, 270), (60, 4000, 50)])
def test_infinite_arguments_of_activations(M, K, N, act, dtype):
    """z = inf and -inf, by the bias and by an operand, at one row, a few and on the matrix cores, with and without splits of k: the
    limits of the activation and of its derivative; everything else is as without them, bit for bit."""
    from ppo_amd import ops
    g = torch.Generator("cuda").manual_seed(M + K)
    x, w, b, r = (torch.randn(s, device="cuda", generator=g).to(dtype) for s in ((M, K), (N, K), (N,), (M, N)))
    want, dwant = ops.linear_act_fwd(x, w, b, act, r, want_deriv=True)
    up, down, d_up, d_down = LIMITS[act]
    want[:, 1], want[:, 2] = (up + r[:, 1].float()).to(dtype), (down + r[:, 2].float()).to(dtype)
    if dwant is not None:
        dwant[:, 1], dwant[:, 2] = d_up, d_down
    bias = b.clone()
    bias[1], bias[2] = math.inf, -math.inf
    y, d = ops.linear_act_fwd(x, w, bias, act, r, want_deriv=True)
    assert torch.equal(y, want) and (d is None or torch.equal(d, dwant))
    # the same by rows of the weights, against an input that is 1 there
    x = x.clone()
    x[:, K // 2] = 1.0
    want, dwant = ops.linear_act_fwd(x, w, b, act, r, want_deriv=True)
    want[:, 1], want[:, 2] = (up + r[:, 1].float()).to(dtype), (down + r[:, 2].float()).to(dtype)
    if dwant is not None:
        dwant[:, 1], dwant[:, 2] = d_up, d_down
    weight = w.clone()
    weight[1, K // 2], weight[2, K // 2] = math.inf, -math.inf
    y, d = ops.linear_act_fwd(x, weight, b, act, r, want_deriv=True)
    assert torch.equal(y, want) and (d is None or torch.equal(d, dwant))


HUGE = 3.4e38                                               # above the largest bf16 value


@pytest.mark.parametrize("M,K,N", [(3, 70, 40), (40, 70, 300), (300, 70, 301), (300, 1000, 270), (60, 4000, 50), (20001, 64, 40), (3585, 700, 3601), (3700, 3601, 700)])
def test_infinite_and_huge_operands_of_f32_layers(M, K, N):
    """The three products, f32, with infinities, a NaN and values that bf16 rounds to infinity: what 64 bits give rounded to f32, at any
    number of rows (a few, and each tile, with splits and without), and the other rows and columns keep their bits.  A finite sum
    is off by (8 + 4 sqrt K) e of its terms' magnitudes (test_gpu_linear_act.py)."""
    from ppo_amd import ops
    gen = torch.Generator("cuda").manual_seed(M + K + N)
    r = lambda *s: torch.randn(s, device="cuda", generator=gen)  # noqa: E731

    def check(call, a, b, k):
        """call(a, b) = a b^T over k, both with rows along k here; specials into rows 1, 2 of a and row 5 of b"""
        a, b = a.clamp(-2, 2), b.clamp(-2, 2)
        clean = call(a, b)
        a2, b2 = a.clone(), b.clone()
        a2[1, k // 3], a2[1, k // 2] = math.inf, 1.5
        a2[2, k - 1] = HUGE
        a2[0, 0] = math.nan
        b2[5, k // 2], b2[5, k - 1] = -math.inf, 0.25
        b[:, k - 1] *= 0.25                                 # HUGE times these stays finite
        b2[:, k - 1] *= 0.25
        clean = call(a, b)
        got, want = call(a2, b2), (a2.double() @ b2.double().t())
        want32 = want.float()
        assert torch.equal(torch.isnan(got), torch.isnan(want32)) and torch.equal(got == math.inf, want32 == math.inf)
        assert torch.equal(got == -math.inf, want32 == -math.inf)
        assert bool(torch.isinf(got[1]).any()) and bool(torch.isfinite(got[2, 6:]).all())
        size = a2.double().abs() @ b2.double().abs().t()
        fin = torch.isfinite(want32)
        assert bool(((got.double() - want).abs()[fin] <= ((8 + 4 * math.sqrt(k)) * E * size)[fin]).all())
        rows, cols = torch.ones(a.shape[0], dtype=torch.bool), torch.ones(b.shape[0], dtype=torch.bool)
        rows[:3] = False
        cols[5] = False
        if rows.any():
            assert torch.equal(got[rows][:, cols], clean[rows][:, cols])

    check(lambda a, b: ops.linear_act_fwd(a, b)[0], r(M, K), r(N, K), K)
    x, w = r(M, K), r(N, K)
    check(lambda a, b: ops.linear_act_bwd(a, x, b.t().contiguous(), want_weight=False, want_bias=False)[0], r(M, N), r(K, N), N)
    check(lambda a, b: ops.linear_act_bwd(a.t().contiguous(), b.t().contiguous(), w, want_input=False, want_bias=False)[1], r(N, M), r(K, M), M)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,K,N", [(3600, 3500, 3700), (3601, 3501, 3703), (1500, 8192, 3000), (1501, 3001, 8191), (8191, 2999, 1500), (2048, 16385, 3000)])
def test_large_tiles_in_every_product(M, K, N, dtype):
    """The tile of 256 x 256 forward and in both gradients, whole and cut, operands in place and copied, through many stages of its
    ring; the last four have splits of k in it: forward (3 in 16 bits), g_x (3), g_W (3) and forward again (2)."""
    from test_gpu_linear_act import _check, _make
    _check(*_make(M + K + N, M, K, N, dtype), "silu")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_small_magnitudes(dtype):
    """Inputs of 2^-100 in f32 and bf16 (f32's third bf16 piece ends at 2^-126), 2^-10 in f16: as exact, relative to the terms, as others."""
    from ppo_amd import ops
    gen = torch.Generator("cuda").manual_seed(7)
    x, w = (torch.randn(s, device="cuda", generator=gen).to(dtype) for s in ((200, 300), (150, 300)))
    x *= 2.0 ** (-10 if dtype == torch.float16 else -100)
    y = ops.linear_act_fwd(x, w)[0].double()
    want, size = x.double() @ w.double().t(), x.double().abs() @ w.double().abs().t()
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    assert bool(((y - want).abs() <= torch.finfo(dtype).eps / 2 * want.abs() + (8 + 4 * math.sqrt(300)) * E * size + tiny).all())


class _Guarded:
    """Buffers on the GPU inside one that is full of 0xab, and whether what is around them still is."""

    def __init__(self):
        self.raw, self.used = [], []

    def of(self, nbytes, align):
        raw = torch.full((nbytes + 4096,), 0xAB, dtype=torch.uint8, device="cuda")
        at = 1024 + align                                   # torch's own blocks begin at multiples of 512
        self.raw.append(raw)
        self.used.append((at, nbytes))
        return raw.data_ptr() + at, raw[at:at + nbytes]

    def check(self):
        for raw, (at, n) in zip(self.raw, self.used):
            assert bool((raw[:at] == 0xAB).all()) and bool((raw[at + n:] == 0xAB).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,K,N", [(1, 7, 5), (3, 70, 41), (9, 33, 15), (40, 2049, 301), (129, 127, 257), (300, 1031, 71), (20001, 63, 41), (61, 8001, 127),
                                   (3601, 701, 3603), (3701, 3601, 701), (701, 3601, 3585)])
def test_nothing_beside_the_outputs_is_written(M, K, N, dtype):
    """The C entries with every output and the workspace between guards: odd sizes at the outputs' least alignment, each tile."""
    from ppo_amd import _lib, ops
    lib = _lib.load()
    gen = torch.Generator("cuda").manual_seed(M * N)
    x, w, b, r, g = (torch.randn(s, device="cuda", generator=gen).to(dtype) for s in ((M, K), (N, K), (N,), (M, N), (M, N)))
    e, dt = x.element_size(), {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}[dtype]
    de, ddt = (2, torch.float16) if dtype == torch.bfloat16 else (4, torch.float32)
    guard = _Guarded()
    nws = lib.ppo_linear_act_fwd_workspace_bytes(M, K, N, dt)
    (py, y), (pd, d), (pw, _) = guard.of(M * N * e, e), guard.of(M * N * de, de), guard.of(nws, 16)
    stream = torch.cuda.current_stream().cuda_stream
    assert lib.ppo_linear_act_fwd(x.data_ptr(), K, w.data_ptr(), K, b.data_ptr(), r.data_ptr(), N, dt, M, K, N, 2, py, pd, pw, nws, stream) == 0
    guard.check()
    want, dwant = ops.linear_act_fwd(x, w, b, "relu", r, want_deriv=True)
    y, d = y.clone().view(dtype).view(M, N), d.clone().view(ddt).view(M, N)
    assert torch.equal(y, want) and torch.equal(d, dwant)
    nws = lib.ppo_linear_act_bwd_workspace_bytes(M, K, N, dt)
    (px, gx), (pgw, gw), (pb, gb), (pw, _) = guard.of(M * K * e, e), guard.of(N * K * e, e), guard.of(N * e, e), guard.of(nws, 16)
    assert lib.ppo_linear_act_bwd(g.data_ptr(), N, x.data_ptr(), K, w.data_ptr(), K, dwant.data_ptr(), dt, M, K, N, px, pgw, pb, pw, nws, stream) == 0
    guard.check()
    for got, q in zip((gx, gw, gb), ops.linear_act_bwd(g, x, w, dwant)):
        assert torch.equal(got.clone().view(dtype).view(q.shape), q)


@pytest.mark.parametrize("M,K,N", [(3, 2, 40), (300, 2, 301), (40, 8000, 300), (60, 4000, 50)])
def test_f32_products_below_the_largest_value(M, K, N):
    """1.9901 2^127 times 1.0041 is finite (1.9983 2^127) although the product of their first bf16 pieces is not; twice that is infinite."""
    from ppo_amd import ops
    x, w = torch.zeros(M, K, device="cuda"), torch.zeros(N, K, device="cuda")
    x[:, 1], w[:, 1] = 1.9901 * 2.0 ** 127, 1.0041
    w[1::2, 1] *= -1.0
    w[2] *= 2.0
    x[1, 0], w[:, 0] = 1.0, torch.arange(N, device="cuda").float()
    want = x.double() @ w.double().t()
    got = ops.linear_act_fwd(x, w)[0]
    assert torch.equal(torch.isinf(got), torch.isinf(want.float())) and bool(torch.isinf(got[:, 2]).all())
    fin = torch.isfinite(want.float())
    assert bool(((got.double() - want).abs()[fin] <= 4 * E * want.abs()[fin]).all())
