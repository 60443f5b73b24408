"""Dense feed-forward, calls that are refused before anything reaches the GPU: places for results that lie in what is still read,
arguments that are no tensors, forward-mode differentiation."""
import pytest
import torch

from vkernels_b200 import torch_ops as ops

BF = torch.bfloat16


def t(*shape, dtype=BF):
    return torch.zeros(shape, dtype=dtype)


def test_feed_forward_places_must_not_overlap_what_is_read_later():
    """The product is written before the residual and the second projection are read; the result after the first one's weights, which
    the next call needs."""
    from vkernels_b200.feedforward import DenseFeedForward

    H, ispp = 16, 8
    w13, w2, room, x, res = t(2 * ispp, H), t(H, ispp), t(256), t(4, H), t(4, H)
    b13, b2 = room[64:64 + 2 * ispp], room[192:192 + H]
    ffn = DenseFeedForward(w13, w2, b13=b13, b2=b2)
    for kw, match in ((dict(product=res[:2].view(4, ispp)), "product must not overlap the residual"),
                      (dict(product=res[:, 4:12]), "product must not overlap the residual"),
                      (dict(product=w2[4:8]), "product must not overlap w2"),
                      (dict(product=room[200:200 + 4 * ispp].view(4, ispp)), "product must not overlap b2"),
                      (dict(out=w13[:4]), "out must not overlap w13"),
                      (dict(out=room[72:72 + 4 * H].view(4, H)), "out must not overlap b13"),
                      (dict(product=[0.0]), "tensor"), (dict(out=[0.0]), "tensor")):
        with pytest.raises(ops.OpNotEligible, match=match):
            ffn(x, res, **kw)
    wide = t(4, H + ispp)
    for r, kw in ((res, dict(product=t(4, ispp))), (wide[:, :H], dict(product=wide[:, H:])), (res, dict(out=res)), (res, dict(out=x)), (None, dict(out=x))):
        with pytest.raises(ops.OpNotEligible, match="CUDA"):      # not in the way of one another: on to the operators
            ffn(x, r, **kw)


def test_tangents_are_refused():
    """Forward-mode differentiation is not offered; what carries a tangent is refused by name, under no_grad too."""
    import torch.autograd.forward_ad as fwd

    x, w, b, res, dy, preact = t(2, 8), t(16, 8), t(16), t(2, 16), t(2, 16), t(2, 16, dtype=torch.float32)
    with fwd.dual_level():
        dual = lambda v: fwd.make_dual(v, torch.ones_like(v))  # noqa: E731
        for call in (lambda: ops.gated_linear(dual(x), w), lambda: ops.gated_linear(x, w, dual(b)), lambda: ops.gated_linear(x, w, out=dual(t(2, 8))),
                     lambda: ops.fused_linear(x, dual(w)), lambda: ops.fused_linear(x, w, residual=dual(res)),
                     lambda: ops.fused_linear_backward(dual(dy), x, w), lambda: ops.gated_linear_backward(t(2, 8), x, w, dual(preact))):
            with pytest.raises(ops.OpNotEligible, match="forward-mode"):
                call()
            with torch.no_grad(), pytest.raises(ops.OpNotEligible, match="forward-mode"):
                call()
        with pytest.raises(ops.OpNotEligible, match="CUDA"):      # a level alone changes nothing
            ops.fused_linear(x, w, b)
    with pytest.raises(ops.OpNotEligible, match="CUDA"):
        ops.fused_linear(x, w, b)


def test_layer_that_cannot_record_refuses_before_it_starts():
    """A layer whose always-on expert holds parameters: refused before any of its buffers is touched, unless gradients are off."""
    from vkernels_b200.experts import FusedMoEMxfp4
    from vkernels_b200.feedforward import DenseFeedForward

    for which in range(4):
        parts = [t(32, 8), t(8, 16), t(32), t(8)]
        parts[which].requires_grad_()
        layer = FusedMoEMxfp4.__new__(FusedMoEMxfp4)
        layer.shared_ffn = DenseFeedForward(parts[0], parts[1], b13=parts[2], b2=parts[3])
        layer.hidden = 8
        layer._buffers = lambda T: {}
        with pytest.raises(ops.OpNotEligible, match="records no gradient"):
            layer.forward(t(4, 8))
        with torch.no_grad():
            assert not layer.shared_ffn.records(t(4, 8))
    ffn = DenseFeedForward(t(32, 8), t(8, 16))
    assert not ffn.records(t(4, 8), None) and ffn.records(t(4, 8).requires_grad_())


def test_a_place_that_is_no_tensor_is_refused_beside_a_residual():
    for out in ([0.0], 1.0, "y"):
        with pytest.raises(ops.OpNotEligible, match="out must be a tensor"):
            ops.fused_linear(t(2, 8), t(16, 8), residual=t(2, 16), out=out)
        with pytest.raises(ops.OpNotEligible, match="out must be a tensor"):
            ops.fused_linear(t(2, 8), t(16, 8), out=out)
        with pytest.raises(ops.OpNotEligible, match="out must be a tensor"):
            ops.gated_linear(t(2, 8), t(16, 8), out=out)


def test_no_rows_have_any_stride():
    """Of a batch of no tokens an expanded gradient is one number's strides: there is nothing to refuse in it."""
    none = torch.ones((), dtype=BF).expand(0, 16)
    for call in (lambda: ops.fused_linear_backward(none, t(0, 8), t(16, 8)), lambda: ops.fused_linear(t(8, 0).T, t(16, 8), residual=none)):
        with pytest.raises(ops.OpNotEligible, match="CUDA"):
            call()
