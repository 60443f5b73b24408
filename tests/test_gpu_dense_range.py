"""-m gpu: the dense feed-forward's activations over the range of their arguments, value by value against the definition in 64 bits:
far tails, every constant of SiTU; offsets beyond 32 bits in every operand, and a dense layer's features.

A pre-activation is put in exactly: x has one value that is not 0, a weight row one that meets it. Bounds count roundings (see
dense_oracle); an exponential's argument v is itself rounded, by at most 2^-22 |v| for each function here, which moves the value by
that much of itself."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

import dense_oracle as ref  # noqa: E402
from vkernels_b200 import torch_ops as ops  # noqa: E402

DEV = "cuda:0"


@pytest.fixture(params=["tcgen05", "simt"])
def impl(request):
    ops.set_impl(request.param)
    yield request.param
    torch.cuda.synchronize()
    ops.kernel_status()
    ops.set_impl("tcgen05")


def situ64(g, u, beta, linear_beta):
    """(value, dh/dg, dh/du) from accurate parts: nothing cancels for gates far below 0."""
    p, a = torch.sigmoid(g), torch.tanh(g / beta)
    b = torch.tanh(u / linear_beta) if linear_beta > 0 else None
    up = u if b is None else linear_beta * b
    return beta * a * p * up


@pytest.mark.parametrize("beta,linear_beta", [(4.0, 25.0), (1.5, 6.0), (30.0, 100.0), (4.0, 0.0)])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("T", [1, 600])
def test_situ_far_from_zero(T, dtype, beta, linear_beta, impl):
    """Gates from where the product is tiny to where the sigmoid is 1, up values from tiny to several hundred."""
    dt = ref.TYPES[dtype]
    gates = [-200.0, -110.0, -100.0, -92.0, -86.5, -80.0, -73.0, -70.0, -68.0, -60.0, -40.0, -12.0, -1.0, -0.01, 0.0, 0.02, 3.0, 50.0, 300.0]
    ups = [-1000.0, -300.0, -260.0, -100.0, -3.0, -0.001, 0.0, 0.5, 40.0, 100.0, 260.0, 300.0, 1000.0]
    pairs = torch.tensor([(g, u) for g in gates for u in ups], dtype=torch.float64, device=DEV).to(dt)
    N = len(pairs)
    w13 = torch.zeros(2 * N, 8, dtype=dt, device=DEV)
    w13[:N, 0], w13[N:, 0] = pairs[:, 0], pairs[:, 1]
    x = torch.zeros(T, 8, dtype=dt, device=DEV)
    x[:, 0] = 1.0
    got = ops.gated_linear(x, w13, activation=ops.SITU, beta=beta, linear_beta=linear_beta)
    g, u = pairs[:, 0].double(), pairs[:, 1].double()
    value = situ64(g, u, beta, linear_beta)
    error = (ref.APPROX + 2.0 ** -22 * g.abs()) * value.abs()
    bound = error + ref.half_step(dt) * (value.abs() + error) + ref.tiny(dt)
    ref.assert_within(got, value.expand(T, N), bound.expand(T, N), "h")


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("T", [1, 600])
def test_gelu_tail_is_good_relatively(T, dtype, impl):
    """Value and slope of gelu (erf) for negative arguments, down to where the value leaves the type's range: within a rounding of
    their own size, not of z's."""
    dt = ref.TYPES[dtype]
    z = -torch.linspace(0.0, 13.0 if dtype == "bf16" else 6.0, 1601, dtype=torch.float64, device=DEV).to(dt).unique()
    N = z.numel()
    w = torch.zeros(N, 8, dtype=dt, device=DEV)
    w[:, 0] = z
    x = torch.zeros(T, 8, dtype=dt, device=DEV)
    x[:, 0] = 1.0
    y, preact = ops.fused_linear(x, w, activation="gelu", return_preact=True)
    z = z.double()
    assert torch.equal(preact, z.float().expand(T, N))
    cdf, density = 0.5 * torch.special.erfc(-z / math.sqrt(2)), torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    h, rel = ref.half_step(dt), ref.APPROX + 2.0 ** -22 * z * z
    value = z * cdf
    error = rel * value.abs()
    bound = error + h * (value.abs() + error) + ref.tiny(dt)
    ref.assert_within(y, value.expand(T, N), bound.expand(T, N), "y")
    # the gradient of the bias of one token is the slope itself, rounded once
    _, _, db = ops.fused_linear_backward(torch.ones(1, N, dtype=dt, device=DEV), x[:1], w, preact[:1], activation="gelu", bias_grad=True,
                                         x_grad=False, w_grad=False)
    slope = cdf + z * density
    error = rel * (cdf + z.abs() * density)
    ref.assert_within(db, slope, error + h * (slope.abs() + error) + ref.tiny(dt), "slope")


@pytest.mark.parametrize("beta,linear_beta", [(1.5, 6.0), (4.0, 0.0), (0.5, -1.0), (30.0, 100.0)])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("T,K,N", [(1, 256, 72), (17, 640, 130), (129, 192, 64), (300, 320, 257), (600, 136, 96)])
def test_situ_with_other_constants(T, K, N, dtype, beta, linear_beta, impl):
    """Forward and backward of SiTU with constants that are not the defaults, up left unbent among them."""
    dt = ref.TYPES[dtype]
    g = torch.Generator(device=DEV)
    g.manual_seed(T + 7 * K + 13 * N)
    r = lambda *s: torch.randn(s, generator=g, device=DEV)  # noqa: E731
    x, w, b, dh = r(T, K).to(dt), (r(2 * N, K) * (1.5 / K ** 0.5)).to(dt), (0.3 * r(2 * N)).to(dt), r(T, N).to(dt)
    kw = dict(activation=ops.SITU, beta=beta, linear_beta=linear_beta)
    h, preact = ops.gated_linear(x, w, b, return_preact=True, **kw)
    assert torch.equal(h, ops.gated_linear(x, w, b, **kw))
    z, mags = ref.project(x, w, b)
    value, _, _, made_of, _, _ = ref.gated(z, "situ", 0.0, beta, linear_beta)
    # |dh/dg| <= |up| (1.2 + beta / 4): (1 - a^2) p <= 1, |a| p (1 - p) <= 1 / 4; |dh/du| <= |gate| <= min(|g|, beta)
    zb = z.abs() + ref.sum_error(K, impl) * mags
    up = zb[:, N:].clamp(max=linear_beta) if linear_beta > 0 else zb[:, N:]
    dz = ref.sum_error(K, impl) * mags
    error = up * (1.2 + beta / 4) * dz[:, :N] + zb[:, :N].clamp(max=beta) * dz[:, N:] + ref.APPROX * made_of
    ref.assert_within(h, value, error + ref.half_step(dt) * (value.abs() + error) + ref.tiny(dt), "h")
    got = ops.gated_linear_backward(dh, x, w, preact, bias_grad=True, **kw)
    _, dg, du, _, mg, mu = ref.gated(preact.double(), "situ", 0.0, beta, linear_beta)
    d = dh.double()
    dz = torch.cat([d * dg, d * du], 1)
    error = ref.APPROX * torch.cat([d.abs() * mg, d.abs() * mu], 1)
    for name, t, (v, bound) in zip(("dx", "dw13", "db13"), got, ref.gradients(dz, error, x, w, dt, impl)):
        ref.assert_within(t, v, bound, name)


def test_offsets_beyond_32_bits_in_the_backward_pass():
    """More than 2^31 pre-activations: kept by the forward call, read by the gradient's kernel, whose result and both products then
    pass 2^31 elements too. Rows and columns at the ends and in the middle against the definition."""
    T, K, N, act = 266000, 64, 8256, "silu"
    g = torch.Generator(device=DEV)
    g.manual_seed(7)
    r = lambda *s: torch.randn(s, generator=g, device=DEV)  # noqa: E731
    dt = torch.bfloat16
    x, w, b = r(T, K).to(dt), (r(N, K) * (1.5 / K ** 0.5)).to(dt), (0.3 * r(N)).to(dt)
    y, preact = ops.fused_linear(x, w, b, activation=act, return_preact=True)
    assert preact.numel() > 2 ** 31
    rows = torch.tensor([0, 1, T // 2 + 5, 260111, 260112, T - 3, T - 1], device=DEV)   # 260112 * 8256 is just above 2^31
    z, mags = ref.project(x[rows], w, b)
    dz = ref.sum_error(K) * mags
    ref.assert_within(preact[rows], z, dz + 2.0 ** -23 * z.abs() + 1e-37, "preact")
    value, _ = ref.linear_act(z, act)
    error = 1.2 * dz + ref.APPROX * z.abs()
    ref.assert_within(y[rows], value, error + ref.half_step(dt) * (value.abs() + error) + ref.tiny(dt), "y")
    dy = y                                        # any values do as the result's gradient: its own memory is the forward call's
    dx, dw, db = ops.fused_linear_backward(dy, x, w, preact, activation=act, bias_grad=True)
    cols = torch.tensor([0, 1, N // 2 + 1, N - 8, N - 1], device=DEV)

    def operand(of_dy, of_z):
        d, zz = of_dy.double(), of_z.double()
        return d * ref.linear_act(zz, act)[1], ref.APPROX * d.abs() * (1 + zz.abs())
    grad, error = operand(dy[rows], preact[rows])
    ref.assert_within(dx[rows], *ref.gradients(grad, error, x[rows], w, dt)[0], "dx")
    grad, error = operand(dy[:, cols], preact[:, cols])
    _, (dw64, dw_bound), (db64, db_bound) = ref.gradients(grad, error, x, w[cols], dt)
    ref.assert_within(dw[cols], dw64, dw_bound, "dw")
    ref.assert_within(db[cols], db64, db_bound, "db")
    torch.cuda.synchronize()
    ops.kernel_status()


def test_strided_operand_beyond_32_bits_in_the_backward_pass():
    """x as the last columns of a matrix of more than 2^31 elements: both gradients are those of a copy of it."""
    T, K, N = 266000, 64, 32
    g = torch.Generator(device=DEV)
    g.manual_seed(8)
    dt = torch.bfloat16
    wide = torch.zeros(T, 8256, dtype=dt, device=DEV)
    wide[:, -K:] = torch.randn(T, K, generator=g, device=DEV)
    x = wide[:, -K:]
    w13 = (torch.randn(2 * N, K, generator=g, device=DEV) * (1.5 / K ** 0.5)).to(dt)
    dh = torch.randn(T, N, generator=g, device=DEV).to(dt)
    h, preact = ops.gated_linear(x, w13, return_preact=True)
    dx, dw, db = ops.gated_linear_backward(dh, x, w13, preact, bias_grad=True)
    near = x.contiguous()
    h2, preact2 = ops.gated_linear(near, w13, return_preact=True)
    assert torch.equal(h, h2) and torch.equal(preact, preact2)
    _, dg, du, _, mg, mu = ref.gated(preact.double(), "swiglu", 0.0)
    d = dh.double()
    grad, error = torch.cat([d * dg, d * du], 1), ref.APPROX * torch.cat([d.abs() * mg, d.abs() * mu], 1)
    for name, t, (v, bound) in zip(("dx", "dw13", "db13"), (dx, dw, db), ref.gradients(grad, error, near, w13, dt)):
        ref.assert_within(t, v, bound, name)
    torch.cuda.synchronize()
    ops.kernel_status()


@pytest.mark.parametrize("T", [1, 70, 300])
def test_features_of_a_wide_dense_layer(T):
    """7168 -> 2 x 18432 gated and 18432 -> 7168, forward and backward."""
    H, ispp, dt = 7168, 18432, torch.bfloat16
    g = torch.Generator(device=DEV)
    g.manual_seed(T)
    r = lambda *s: torch.randn(s, generator=g, device=DEV)  # noqa: E731
    x, w13, w2, dh, dy = r(T, H).to(dt), (r(2 * ispp, H) * (1.5 / H ** 0.5)).to(dt), (r(H, ispp) / ispp ** 0.5).to(dt), r(T, ispp).to(dt), r(T, H).to(dt)
    h, preact = ops.gated_linear(x, w13, swiglu_limit=7.0, return_preact=True)
    half = ref.half_step(dt)
    z, mags = ref.project(x, w13)
    dz = ref.sum_error(H) * mags
    ref.assert_within(preact, z, dz + 2.0 ** -23 * z.abs() + 1e-37, "preact")
    value, _, _, made_of, _, _ = ref.gated(z, "swiglu", 7.0)
    sg, su = ref.gated_slopes_bound(z, "swiglu", 7.0)
    error = sg * dz[:, :ispp] + su * dz[:, ispp:] + ref.APPROX * made_of
    ref.assert_within(h, value, error + half * (value.abs() + error) + ref.tiny(dt), "h")
    y, (z2, mags2) = ops.fused_linear(h, w2, residual=x), ref.project(h, w2)
    value = z2 + x.double()
    error = ref.sum_error(ispp) * mags2 + 2.0 ** -23 * value.abs()
    ref.assert_within(y, value, error + half * (value.abs() + error) + ref.tiny(dt), "y")
    _, dg, du, _, mg, mu = ref.gated(preact.double(), "swiglu", 7.0)
    d = dh.double()
    grad, error = torch.cat([d * dg, d * du], 1), ref.APPROX * torch.cat([d.abs() * mg, d.abs() * mu], 1)
    got = ops.gated_linear_backward(dh, x, w13, preact, swiglu_limit=7.0, bias_grad=True)
    for name, t, (v, bound) in zip(("dx", "dw13", "db13"), got, ref.gradients(grad, error, x, w13, dt)):
        ref.assert_within(t, v, bound, name)
    got = ops.fused_linear_backward(dy, h, w2, bias_grad=True)
    for name, t, (v, bound) in zip(("dh", "dw2", "db2"), got, ref.gradients(dy.double(), torch.zeros_like(z2), h, w2, dt)):
        ref.assert_within(t, v, bound, name)
    torch.cuda.synchronize()
    ops.kernel_status()


@pytest.mark.parametrize("T,K,N", [(2 ** 27, 8, 8), (2, 2 ** 27, 8), (2, 8, 2 ** 27)])
def test_largest_sizes(T, K, N):
    """The documented limits, 2^27 tokens, inputs or weight rows. Operands of -1 and 1: every sum is a whole number that fp32 holds in
    any order (below 2^24; these are random walks of at most 2^27 steps, 12000 wide), so results are those numbers, rounded once."""
    g = torch.Generator(device=DEV)
    g.manual_seed(5)
    sign = lambda *s: torch.randint(0, 2, s, generator=g, device=DEV, dtype=torch.int8).mul_(2).sub_(1).to(torch.bfloat16)  # noqa: E731
    x, w, dy = sign(T, K), sign(N, K), sign(T, N)

    def product(a, b):
        """a b^T, exactly, a long sum in pieces"""
        total = torch.zeros(a.shape[0], b.shape[0], dtype=torch.float64, device=DEV)
        for i in range(0, a.shape[1], 2 ** 24):
            total += a[:, i:i + 2 ** 24].double() @ b[:, i:i + 2 ** 24].double().T
        return total

    def check(got, a, b, what):
        """Rows and columns at both ends where a or b is long, all of them where both are short."""
        rows, cols = (torch.arange(n, device=DEV) if n <= 64 else torch.tensor([0, 1, 2, n // 2 + 3, n - 2, n - 1], device=DEV) for n in got.shape)
        want = product(a[rows], b[cols])
        assert torch.equal(got[rows][:, cols], want.to(got.dtype)), what
        assert bool(got.isfinite().all()), what
    check(ops.fused_linear(x, w), x, w, "y")
    dx, dw, db = ops.fused_linear_backward(dy, x, w, bias_grad=True)
    check(dx, dy, w.T, "dx")
    check(dw, dy.T, x.T, "dw")
    check(db[:, None], dy.T, torch.ones(1, T, dtype=dy.dtype, device=DEV), "db")
    torch.cuda.synchronize()
    ops.kernel_status()
