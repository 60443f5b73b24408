"""Dense feed-forward operators, the part that needs no GPU: refusals of the Python operators and of the C entries (host checks
run before any CUDA call), and the 64-bit definition's gradients against differences of it."""
import numpy as np
import pytest
import torch

import dense_oracle as ref
from vkernels_b200 import native_runtime as nr
from vkernels_b200 import torch_ops as ops

BF = torch.bfloat16


def t(*shape, dtype=BF):
    return torch.zeros(shape, dtype=dtype)


def test_cpu_tensors_are_refused():
    with pytest.raises(ops.OpNotEligible, match="CUDA"):
        ops.gated_linear(t(2, 8), t(16, 8))
    with pytest.raises(ops.OpNotEligible, match="CUDA"):
        ops.fused_linear(t(2, 8), t(16, 8))
    with pytest.raises(ops.OpNotEligible, match="CUDA"):
        ops.gated_linear_backward(t(2, 8), t(2, 8), t(16, 8), t(2, 16, dtype=torch.float32))
    with pytest.raises(ops.OpNotEligible, match="CUDA"):
        ops.fused_linear_backward(t(2, 16), t(2, 8), t(16, 8))
    with pytest.raises(ops.OpNotEligible, match="CUDA"):
        ops.fused_linear(t(2, 8).requires_grad_(), t(16, 8))


@pytest.mark.parametrize("match,call", [
    ("bfloat16 or float16", lambda: ops.gated_linear(t(2, 8, dtype=torch.float32), t(16, 8, dtype=torch.float32))),
    ("like the other", lambda: ops.gated_linear(t(2, 8), t(16, 8, dtype=torch.float16))),
    ("like the other", lambda: ops.gated_linear(t(2, 8), t(16, 8), t(16, dtype=torch.float32))),
    ("even row count", lambda: ops.gated_linear(t(2, 8), t(15, 8))),
    ("expected", lambda: ops.gated_linear(t(2, 8), t(16, 9))),
    ("expected", lambda: ops.fused_linear(t(2, 8), t(2, 16, 8))),
    ("positive", lambda: ops.fused_linear(t(2, 0), t(16, 0))),
    ("positive", lambda: ops.fused_linear(t(2, 8), t(0, 8))),
    ("SWIGLU or SITU", lambda: ops.gated_linear(t(2, 8), t(16, 8), activation=2)),
    ("negative", lambda: ops.gated_linear(t(2, 8), t(16, 8), swiglu_limit=-1.0)),
    ("negative", lambda: ops.gated_linear(t(2, 8), t(16, 8), swiglu_limit=float("nan"))),
    ("positive beta", lambda: ops.gated_linear(t(2, 8), t(16, 8), activation=ops.SITU, beta=0.0)),
    ("activation", lambda: ops.fused_linear(t(2, 8), t(16, 8), activation="relu")),
    ("activation", lambda: ops.fused_linear(t(2, 8), t(16, 8), activation=1)),
    ("bias", lambda: ops.fused_linear(t(2, 8), t(16, 8), t(15))),
    ("bias", lambda: ops.fused_linear(t(2, 8), t(16, 8), t(32)[::2])),
    ("residual", lambda: ops.fused_linear(t(2, 8), t(16, 8), residual=t(16))),
    ("residual", lambda: ops.fused_linear(t(2, 8), t(16, 8), residual=t(1, 16))),
    ("overlap", lambda: ops.fused_linear(t(2, 8), t(16, 8), residual=t(1, 16).expand(2, 16))),
    ("neighbours", lambda: ops.fused_linear(t(2, 8), t(16, 8), residual=t(16, 2).T)),
    ("out", lambda: ops.fused_linear(t(2, 8), t(16, 8), out=t(2, 15))),
    ("like the other", lambda: ops.fused_linear(t(2, 8), t(16, 8), out=t(2, 16, dtype=torch.float16))),
    ("neighbours", lambda: ops.fused_linear(t(2, 8), t(16, 8), out=t(16, 2).T)),
    ("overlap", lambda: ops.fused_linear(t(2, 8), t(16, 8), out=t(1, 16).expand(2, 16))),
    ("gradient must be", lambda: ops.gated_linear_backward(t(2, 16), t(2, 8), t(16, 8), t(2, 16, dtype=torch.float32))),
    ("preact must be", lambda: ops.gated_linear_backward(t(2, 8), t(2, 8), t(16, 8), t(2, 8, dtype=torch.float32))),
    ("preact must be", lambda: ops.gated_linear_backward(t(2, 8), t(2, 8), t(16, 8), t(2, 16))),
    ("pre-activations", lambda: ops.gated_linear_backward(t(2, 8), t(2, 8), t(16, 8), None)),
    ("pre-activations", lambda: ops.fused_linear_backward(t(2, 16), t(2, 8), t(16, 8), activation="silu")),
    ("overlap", lambda: ops.fused_linear_backward(t(1, 16).expand(2, 16), t(2, 8), t(16, 8))),
])
def test_python_refusals(match, call):
    with pytest.raises(ops.OpNotEligible, match=match):
        call()


def test_out_must_not_overlap_the_inputs():
    a = t(4, 16)
    with pytest.raises(ops.OpNotEligible, match="overlap x"):
        ops.fused_linear(a[:2], t(16, 16), out=a[1:3])
    w = t(16, 16)
    with pytest.raises(ops.OpNotEligible, match="overlap w"):
        ops.fused_linear(a, w, out=w[:4])
    with pytest.raises(ops.OpNotEligible, match="residual"):
        ops.fused_linear(t(2, 16), w, residual=a[:2], out=a[1:3])
    wide = t(4, 40)
    for x, out, match in ((wide[:, 24:], wide[:, :16], "CUDA"), (wide[:, :16], wide[:, 16:32], "CUDA"),     # beside one another
                          (wide[:, 24:], wide[:, 9:25], "overlap x"), (wide[:, :16], wide[:, 15:31], "overlap x"),
                          (wide[:3, 24:], wide[1:, :16], "CUDA"), (wide[:3, 24:], wide[1:, 20:36], "overlap x")):
        with pytest.raises(ops.OpNotEligible, match=match):
            ops.fused_linear(x, w, out=out)
    one = t(1, 16).as_strided((1, 16), (0, 1))               # a single row, of any pitch
    with pytest.raises(ops.OpNotEligible, match="overlap x"):
        ops.fused_linear(one, w, out=one.as_strided((1, 16), (0, 1)))
    with pytest.raises(ops.OpNotEligible, match="CUDA"):     # the residual itself is a place for the result
        ops.fused_linear(t(2, 16), w, residual=a[:2], out=a[:2])
    with pytest.raises(ops.OpNotEligible, match="overlap w13"):
        ops.gated_linear(t(2, 16), w, out=w[:1].view(2, 8))


P = 1 << 20      # an aligned address that is never followed: every call below is refused on the host


def linear_args(**k):
    a = dict(x=P, ldx=64, w=P, ldw=64, bias=None, residual=None, ldr=0, y=P, ldy=64, preact=None, ldp=0, dtype=0, T=4, n_in=64,
             n_out=64, act=0, work=None, nbytes=0, stream=None)
    assert not set(k) - set(a)
    return list({**a, **k}.values())


def gated_args(**k):
    a = dict(x=P, ldx=64, w=P, ldw=64, bias=None, h=P, ldh=64, preact=None, ldp=0, dtype=0, T=4, n_in=64, ispp=64, act=0, limit=0.0,
             beta=4.0, lbeta=25.0, work=None, nbytes=0, stream=None)
    assert not set(k) - set(a)
    return list({**a, **k}.values())


def linear_back_args(**k):
    a = dict(dy=P, lddy=64, x=P, ldx=64, w=P, ldw=64, preact=P, ldp=64, dx=P, lddx=64, dw=P, lddw=64, db=P, dtype=0, T=4, n_in=64,
             n_out=64, act=1, work=P, nbytes=1 << 20, stream=None)
    assert not set(k) - set(a)
    return list({**a, **k}.values())


@pytest.mark.parametrize("bad,word", [
    (dict(dtype=2), b"dtype"), (dict(T=-1), b"T"), (dict(n_in=0), b"positive"), (dict(n_out=0), b"positive"), (dict(x=None), b"null"),
    (dict(w=None), b"null"), (dict(x=P + 1), b"odd"), (dict(x=P + 2), b"workspace"), (dict(w=P + 8), b"workspace"),
    (dict(ldx=68), b"workspace"), (dict(x=P + 2, work=P, nbytes=511), b"workspace"), (dict(ldw=66, work=P + 8, nbytes=1 << 20), b"workspace"),
    (dict(ldw=56), b"pitch"), (dict(y=None), b"null"), (dict(y=P + 1), b"odd"), (dict(ldy=63), b"pitch"), (dict(bias=P + 1), b"bias"),
    (dict(residual=P + 1, ldr=64), b"odd"), (dict(residual=P, ldr=63), b"pitch"), (dict(preact=P, ldp=63), b"pitch"), (dict(preact=P + 2, ldp=64), b"preact"),
    (dict(act=4), b"activation"), (dict(act=-1), b"activation"), (dict(n_in=(1 << 27) + 1, ldx=1 << 28, ldw=1 << 28), b"sizes"), (dict(T=(1 << 27) + 1), b"sizes")])
def test_linear_entry_refuses(bad, word):
    lib = nr.load_library()
    assert lib.vk_cuda_fused_linear(*linear_args(**bad)) == 1 and word in lib.vk_last_error(), lib.vk_last_error()


@pytest.mark.parametrize("bad,word", [
    (dict(dtype=-1), b"dtype"), (dict(act=2), b"SwiGLU"), (dict(limit=-1.0), b"limit"), (dict(limit=float("nan")), b"limit"),
    (dict(act=1, beta=0.0), b"beta"), (dict(preact=P, ldp=127), b"pitch"), (dict(ldh=63), b"pitch"), (dict(x=P + 4), b"workspace")])
def test_gated_entry_refuses(bad, word):
    lib = nr.load_library()
    assert lib.vk_cuda_gated_linear(*gated_args(**bad)) == 1 and word in lib.vk_last_error(), lib.vk_last_error()


@pytest.mark.parametrize("bad,word", [
    (dict(preact=None), b"pre-activations"), (dict(dy=None), b"null"), (dict(lddy=63), b"pitch"), (dict(dx=P + 1), b"odd"),
    (dict(lddw=63), b"pitch"), (dict(db=P + 1), b"odd"), (dict(work=None), b"workspace"), (dict(work=P + 8), b"workspace"),
    (dict(nbytes=16), b"workspace"), (dict(x=P + 1), b"odd"), (dict(w=P + 1), b"odd"), (dict(x=None), b"null"),
    (dict(preact=P + 2), b"preact")])
def test_linear_backward_entry_refuses(bad, word):
    lib = nr.load_library()
    assert lib.vk_cuda_fused_linear_backward(*linear_back_args(**bad)) == 1 and word in lib.vk_last_error(), lib.vk_last_error()


def test_no_tokens_and_nothing_asked_are_no_work():
    lib = nr.load_library()
    assert lib.vk_cuda_fused_linear(*linear_args(T=0, x=None, y=None)) == 0
    assert lib.vk_cuda_gated_linear(*gated_args(T=0, x=None, h=None)) == 0
    assert lib.vk_cuda_fused_linear_backward(*linear_back_args(dx=None, dw=None, db=None, work=None)) == 0
    assert lib.vk_cuda_fused_linear_backward(*linear_back_args(T=0, dw=None, db=None)) == 0


def test_workspace_sizes():
    lib = nr.load_library()
    fwd, back = lib.vk_cuda_dense_forward_workspace_bytes, lib.vk_cuda_dense_backward_workspace_bytes
    assert fwd(P, 64, P, 64, 4, 64, 64) == 0 and fwd(P + 2, 64, P, 64, 0, 64, 64) == 0
    assert fwd(P + 2, 64, P, 64, 4, 64, 64) == 4 * 64 * 2 and fwd(P, 64, P, 70, 4, 60, 3) == 512   # 3 rows of 64, in whole 256 bytes
    assert back(P, 64, P, 64, 100, 64, 13, 1) >= 100 * 32 * 2 + 26 * 4
    assert back(P + 2, 64, P, 64, 100, 64, 13, 1) >= back(P, 64, P, 64, 100, 64, 13, 1) + 100 * 64 * 2
    # one of 74 tiles' worth of parts for each gradient with a long sum: 5000 tokens of 64 x 64, 9 parts of [64, 64] fp32
    assert back(P, 64, P, 64, 5000, 64, 64, 0) >= back(P, 64, P, 64, 100, 64, 64, 0) + 9 * 64 * 64 * 4
    for most in (2 ** 27 + 1, 2 ** 30, 2 ** 31 - 1):
        for sizes in ((most, 64, 64), (100, most, 64), (100, 64, most)):
            for gated in (0, 1):
                lib.vk_set_last_error(0, b"")
                assert back(P, 64, P, 64, *sizes, gated) == 0 and b"2^27" in lib.vk_last_error()
            lib.vk_set_last_error(0, b"")
            assert fwd(P, 64, P, 64, *sizes) == 0 and b"2^27" in lib.vk_last_error()
    lib.vk_set_last_error(0, b"")
    assert fwd(P, 64, P, 64, -1, 64, 64) == 0 and lib.vk_last_error_code() == 1
    lib.vk_set_last_error(0, b"")
    assert back(P, 64, P, 64, -1, 64, 8, 0) == 0 and lib.vk_last_error_code() == 1


@pytest.mark.parametrize("kind,limit,linear_beta", [("swiglu", 0.0, 25.0), ("swiglu", 1.0, 25.0), ("situ", 0.0, 25.0), ("situ", 0.0, 0.0)])
def test_gated_slopes_against_differences(kind, limit, linear_beta):
    rng = np.random.default_rng(3)
    z = torch.from_numpy(rng.normal(size=(40, 24)) * 1.5)
    eps, n = 1e-6, 12
    near = (z.abs() - limit).abs() < 1e-4 if limit else torch.zeros_like(z, dtype=torch.bool)
    assert not near.any()
    value = lambda v: ref.gated(v, kind, limit, linear_beta=linear_beta)[0]  # noqa: E731
    _, dg, du, *_ = ref.gated(z, kind, limit, linear_beta=linear_beta)
    for slope, cols in ((dg, slice(0, n)), (du, slice(n, 2 * n))):
        step = torch.zeros_like(z)
        step[:, cols] = eps
        # central difference: error eps^2 / 6 times the third derivative, and cancellation 2^-52 / eps
        assert torch.allclose(slope, (value(z + step) - value(z - step)) / (2 * eps), rtol=0, atol=1e-8)


@pytest.mark.parametrize("act", [None, "silu", "gelu", "gelu_tanh"])
def test_linear_slopes_against_differences(act):
    z, eps = torch.linspace(-9, 9, 501, dtype=torch.float64), 1e-6
    value, slope = ref.linear_act(z, act)
    diff = (ref.linear_act(z + eps, act)[0] - ref.linear_act(z - eps, act)[0]) / (2 * eps)
    assert torch.allclose(slope, diff, rtol=0, atol=1e-8)
    if act:
        named = {"silu": torch.nn.functional.silu(z), "gelu": torch.nn.functional.gelu(z),
                 "gelu_tanh": torch.nn.functional.gelu(z, approximate="tanh")}[act]
        assert torch.allclose(value, named, rtol=1e-12, atol=1e-15)


def test_feed_forward_checks_its_weights():
    from vkernels_b200.dist import CudaBackend
    from vkernels_b200.feedforward import DenseFeedForward

    DenseFeedForward(t(32, 8), t(8, 16), b13=t(32), b2=t(8))
    for bad in ((t(32, 8), t(8, 15)), (t(32, 8), t(9, 16)), (t(31, 8), t(8, 16)), (t(32, 8), t(8, 16, dtype=torch.float16))):
        with pytest.raises(ops.OpNotEligible):
            DenseFeedForward(*bad)
    with pytest.raises(ops.OpNotEligible, match="b2"):
        DenseFeedForward(t(32, 8), t(8, 16), b2=t(8, dtype=torch.float32))

    class Layer:
        shared_ffn = DenseFeedForward(t(32, 8), t(8, 16))
    with pytest.raises(ValueError, match="routed experts only"):
        CudaBackend(Layer(), "cpu")
