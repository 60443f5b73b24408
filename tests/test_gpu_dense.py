"""-m gpu: the dense feed-forward operators against their definition in 64 bits, value by value, at bounds that count the
roundings (dense_oracle), on both kernels sets; refusals; strides, alignments, streams, graphs."""
import pytest
import torch

pytestmark = pytest.mark.gpu

import dense_oracle as ref  # noqa: E402
from vkernels_b200 import torch_ops as ops  # noqa: E402

DEV = "cuda:0"
KIND = {"swiglu": ops.SWIGLU, "situ": ops.SITU}
# tokens, in, out: single tokens, tile borders (64, 128, 256) and one beside them, sizes that are multiples of nothing
SIZES = [(1, 64, 64), (1, 2880, 360), (2, 72, 8), (7, 64, 192), (16, 512, 256), (17, 640, 130), (33, 1, 1), (63, 1000, 90), (64, 256, 2880),
         (65, 511, 257), (127, 33, 129), (128, 128, 128), (129, 192, 64), (200, 320, 513), (255, 65, 200), (256, 64, 256), (257, 264, 255),
         (300, 2048, 96), (513, 96, 384), (1000, 136, 72)]


@pytest.fixture(params=["tcgen05", "simt"])
def impl(request):
    ops.set_impl(request.param)
    yield request.param
    torch.cuda.synchronize()
    ops.kernel_status()
    ops.set_impl("tcgen05")


def tensors(T, K, rows, dtype, seed=0, bias=True, gap=0, std=1.5):
    g = torch.Generator(device=DEV)
    g.manual_seed(1000 * seed + T + 7 * K + 13 * rows)
    r = lambda *s: torch.randn(s, generator=g, device=DEV)  # noqa: E731
    dt = ref.TYPES[dtype]
    x = r(T, K + gap).to(dt)[:, :K]
    w = (r(rows, K + gap) * (std / K ** 0.5)).to(dt)[:, :K]
    return x, w, ((0.3 * r(rows)).to(dt) if bias else None), lambda n: r(T, n).to(dt)


def check_gated(got, preact, z, mags, K, dtype, impl, kind, limit):
    h = ref.half_step(dtype)
    dz = ref.sum_error(K, impl) * mags
    value, _, _, made_of, _, _ = ref.gated(z, kind, limit)
    sg, su = ref.gated_slopes_bound(z, kind, limit)
    n = got.shape[1]
    error = sg * dz[:, :n] + su * dz[:, n:] + ref.APPROX * made_of
    ref.assert_within(got, value, error + h * (value.abs() + error) + ref.tiny(dtype), "h")
    if preact is not None:
        ref.assert_within(preact, z, dz + 2.0 ** -23 * z.abs() + 1e-37, "preact")


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("T,K,N", SIZES)
def test_gated_linear(T, K, N, dtype, impl):
    for kind, limit, bias, gap in (("swiglu", 0.0, False, 0), ("swiglu", 2.0, True, 8), ("situ", 0.0, True, 3)):
        x, w, b, _ = tensors(T, K, 2 * N, dtype, bias=bias, gap=gap)
        z, mags = ref.project(x, w, b)
        h = ops.gated_linear(x, w, b, activation=KIND[kind], swiglu_limit=limit)
        h2, preact = ops.gated_linear(x, w, b, activation=KIND[kind], swiglu_limit=limit, return_preact=True)
        assert torch.equal(h, h2) and h.dtype == x.dtype and h.shape == (T, N)
        check_gated(h, preact, z, mags, K, x.dtype, impl, kind, limit)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("T,K,N", SIZES)
def test_fused_linear(T, K, N, dtype, impl):
    for act, bias, res, gap in ((None, False, False, 0), (None, True, True, 8), ("silu", True, False, 3), ("gelu", False, True, 0),
                                ("gelu_tanh", True, True, 1)):
        x, w, b, more = tensors(T, K, N, dtype, bias=bias, gap=gap)
        r = more(N + gap)[:, :N] if res else None
        z, mags = ref.project(x, w, b)
        y, preact = ops.fused_linear(x, w, b, activation=act, residual=r, return_preact=True)
        assert torch.equal(y, ops.fused_linear(x, w, b, activation=act, residual=r)) and y.shape == (T, N)
        dz, h = ref.sum_error(K, impl) * mags, ref.half_step(x.dtype)
        value, _ = ref.linear_act(z, act)
        error = 1.2 * dz + ref.APPROX * z.abs()      # no slope of the activations exceeds 1.13
        if r is not None:
            value = value + r.double()
            error = error + 2.0 ** -23 * value.abs()
        ref.assert_within(y, value, error + h * (value.abs() + error) + ref.tiny(x.dtype), f"y {act}")
        assert (preact is None) == (act is None)
        if act:
            ref.assert_within(preact, z, dz + 2.0 ** -23 * z.abs() + 1e-37, "preact")


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("T,K,N", SIZES)
def test_gated_linear_backward(T, K, N, dtype, impl):
    for kind, limit, gap in (("swiglu", 0.0, 0), ("swiglu", 2.0, 8), ("situ", 0.0, 3)):
        x, w, b, more = tensors(T, K, 2 * N, dtype, gap=gap)
        dh = more(N + gap)[:, :N]
        _, preact = ops.gated_linear(x, w, b, activation=KIND[kind], swiglu_limit=limit, return_preact=True)
        got = ops.gated_linear_backward(dh, x, w, preact, activation=KIND[kind], swiglu_limit=limit, bias_grad=True)
        _, dg, du, _, mg, mu = ref.gated(preact.double(), kind, limit)
        d = dh.double()
        dz = torch.cat([d * dg, d * du], 1)
        error = ref.APPROX * torch.cat([d.abs() * mg, d.abs() * mu], 1)
        for name, t, (value, bound) in zip(("dx", "dw13", "db13"), got, ref.gradients(dz, error, x, w, x.dtype, impl)):
            ref.assert_within(t, value, bound, f"{name} {kind}")


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("T,K,N", SIZES)
def test_fused_linear_backward(T, K, N, dtype, impl):
    for act, gap in ((None, 0), (None, 3), ("silu", 8), ("gelu", 0), ("gelu_tanh", 1)):
        x, w, b, more = tensors(T, K, N, dtype, gap=gap)
        dy = more(N + gap)[:, :N]
        _, preact = ops.fused_linear(x, w, b, activation=act, return_preact=True)
        got = ops.fused_linear_backward(dy, x, w, preact, activation=act, bias_grad=True)
        d = dy.double()
        if act is None:
            dz, error = d, torch.zeros_like(d)
        else:
            z = preact.double()
            _, slope = ref.linear_act(z, act)
            dz, error = d * slope, ref.APPROX * d.abs() * (1 + z.abs())
        for name, t, (value, bound) in zip(("dx", "dw", "db"), got, ref.gradients(dz, error, x, w, x.dtype, impl)):
            ref.assert_within(t, value, bound, f"{name} {act}")
