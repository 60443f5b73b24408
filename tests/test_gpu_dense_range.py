"""-m gpu: the dense feed-forward's activations over the range of their arguments, value by value against the definition in 64 bits:
far tails.

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
