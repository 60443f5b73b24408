"""-m gpu: the dense feed-forward where its tensors lie in one another's memory, and calls that must not go through."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from vkernels_b200 import torch_ops as ops  # noqa: E402

DEV = "cuda:0"


def layers(T, grad=False):
    """A small routed layer with and one without a bf16 always-on expert, that expert, and activations for them."""
    from gpu_common import make_case
    from vkernels_b200 import synthetic as syn
    from vkernels_b200.experts import layer_from_config
    from vkernels_b200.feedforward import DenseFeedForward

    cfg = syn.scaled(syn.CONFIGS["c0"], H=512, I=256, E=8, top_k=2)
    w, A, r = make_case(cfg, T, backend="torch")
    g = torch.Generator(device=DEV)
    g.manual_seed(3)
    ispp = 192
    w13 = (torch.randn(2 * ispp, cfg.H, generator=g, device=DEV) / cfg.H ** 0.5).to(torch.bfloat16).requires_grad_(grad)
    w2 = (torch.randn(cfg.H, ispp, generator=g, device=DEV) / ispp ** 0.5).to(torch.bfloat16).requires_grad_(grad)
    ffn = DenseFeedForward(w13, w2)
    return layer_from_config(cfg, w, r, max_tokens=T), layer_from_config(cfg, w, r, max_tokens=T, shared_ffn=ffn), ffn, A


def same(got, want, T):
    """Bit by bit, but for batches whose routed part adds with atomics."""
    return torch.equal(got, want) or T > 256 and torch.allclose(got.float(), want.float(), atol=2e-2, rtol=2.0 ** -7)


@pytest.mark.parametrize("T", [1, 40, 600])
def test_layer_result_where_its_activations_lie(T):
    """The always-on expert sees the activations although the result takes their place: given as out_bf16, overlapping by a row
    less, and in the layer's own result buffer, when one call's result is the next one's input."""
    routed, layer, ffn, A = layers(T)
    want = ffn(A, routed(A))
    assert not same(ffn(routed(A).clone(), routed(A)), want, T)      # what the expert would add for the routed result
    x = A.clone()
    got = layer(x, out_bf16=x)
    assert got is x and same(x, want, T)
    room = torch.empty(T + 1, A.shape[1], dtype=A.dtype, device=DEV)
    room[1:] = A
    assert same(layer(room[1:], out_bf16=room[:T]), want, T)
    first = layer(A)
    keep = first.clone()
    want = ffn(keep, routed(keep))
    assert same(layer(first), want, T)
    torch.cuda.synchronize()
    ops.kernel_status()


def test_dual_tensors_are_refused():
    """Forward-mode differentiation is not offered: a tangent is refused, not dropped, on the direct path and behind it."""
    import torch.autograd.forward_ad as fwd

    g = torch.Generator(device=DEV)
    g.manual_seed(1)
    r = lambda *s: torch.randn(s, generator=g, device=DEV).to(torch.bfloat16)  # noqa: E731
    x, w, b, res, dy = r(8, 64), r(32, 64), r(32), r(8, 32), r(8, 32)
    _, preact = ops.fused_linear(x, w, b, activation="silu", return_preact=True)
    plain = ops.fused_linear(x, w, b, residual=res)
    with fwd.dual_level():
        dual = lambda t: fwd.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in (lambda: ops.gated_linear(dual(x), w), lambda: ops.gated_linear(x, dual(w), b), lambda: ops.gated_linear(x, w, dual(b)),
                     lambda: ops.fused_linear(dual(x), w), lambda: ops.fused_linear(x, dual(w)), lambda: ops.fused_linear(x, w, dual(b)),
                     lambda: ops.fused_linear(x, w, residual=dual(res)), lambda: ops.fused_linear(x.view(2, 4, 64), dual(w)),
                     lambda: ops.fused_linear(x, w, residual=res, out=dual(res)),
                     lambda: ops.fused_linear_backward(dual(dy), x, w, preact, activation="silu"),
                     lambda: ops.fused_linear_backward(dy, x, w, dual(preact), activation="silu"),
                     lambda: ops.gated_linear_backward(dual(dy)[:, :16], x, w, preact)):
            with pytest.raises(ops.OpNotEligible, match="forward-mode"):
                call()
            with torch.no_grad(), pytest.raises(ops.OpNotEligible, match="forward-mode"):
                call()
        assert torch.equal(ops.fused_linear(x, w, b, residual=res), plain)      # a level alone changes nothing


def test_layer_records_nothing_and_says_so_before_any_work():
    """The routed experts record no gradient: with a feed-forward of parameters, or activations, that require one the layer is called
    under no_grad; elsewhere it refuses before it writes anything."""
    routed, layer, ffn, A = layers(40, grad=True)
    with torch.no_grad():
        want = ffn(A, routed(A)).clone()
        assert torch.equal(layer(A), want)
        graph, y = layer.capture(A)
        graph.replay()
        assert torch.equal(y, want)
    out = torch.full_like(A, 7.0)
    with pytest.raises(ops.OpNotEligible, match="records no gradient"):
        layer(A, out_bf16=out)
    frozen_routed, frozen, _, A = layers(40)
    with pytest.raises(ops.OpNotEligible, match="records no gradient"):
        frozen(A.clone().requires_grad_(), out_bf16=out)
    torch.cuda.synchronize()
    assert bool((out == 7).all())
    with torch.inference_mode():
        assert torch.equal(layer(A), want)


def test_forked_capture():
    """Calls on two streams of one capture, forked and joined: each result is that of its own inputs on every replay."""
    g = torch.Generator(device=DEV)
    g.manual_seed(2)
    r = lambda *s: torch.randn(s, generator=g, device=DEV)  # noqa: E731
    for T in (3, 300):
        x = r(T, 256).to(torch.bfloat16)
        w13, wa, wb, wc = ((r(n, k) / k ** 0.5).to(torch.bfloat16) for n, k in ((512, 256), (256, 256), (256, 256), (256, 256)))

        def step(side=None):
            h, preact = ops.gated_linear(x, w13, return_preact=True)
            main = torch.cuda.current_stream()
            if side is not None:
                side.wait_stream(main)
            with torch.cuda.stream(side or main):
                a = ops.fused_linear(h, wa, activation="silu")
                da, dwa, _ = ops.fused_linear_backward(a, h, wa)
            b = ops.fused_linear(h, wb, activation="gelu")
            dx, dw13, db = ops.gated_linear_backward(h, x, w13, preact, bias_grad=True)
            if side is not None:
                main.wait_stream(side)
            return [a, b, da, dwa, dx, dw13, db, ops.fused_linear(a, wc, residual=b), ops.fused_linear(da, wc, residual=dx)]
        step()
        torch.cuda.synchronize()
        graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(graph):
            got = step(side)
        for _ in range(5):
            x.mul_(-0.75)
            graph.replay()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(got, step()))
    ops.kernel_status()


def test_calls_from_two_threads():
    """Two threads, a stream each, call at once: every result has its own inputs' bits."""
    import threading

    g = torch.Generator(device=DEV)
    g.manual_seed(4)
    r = lambda *s: torch.randn(s, generator=g, device=DEV).to(torch.bfloat16)  # noqa: E731
    jobs = [(r(T, 264), r(2 * 72, 264), r(T, 72)) for T in (5, 90, 700)]

    def step(x, w13, dh):
        h, preact = ops.gated_linear(x, w13, return_preact=True)
        return (h, *ops.gated_linear_backward(dh, x, w13, preact, bias_grad=True))
    want = [step(*j) for j in jobs]
    torch.cuda.synchronize()
    wrong = []

    def work(first):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for i in range(60):
                    k = (first + i) % len(jobs)
                    got = step(*jobs[k])
                    if not all(torch.equal(p, q) for p, q in zip(got, want[k])):
                        wrong.append(k)
        except Exception as e:  # noqa: BLE001
            wrong.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
    ops.kernel_status()


@pytest.mark.parametrize("T", [1, 20, 600])
def test_feed_forward_in_place_of_its_input(T):
    """x as the residual and as the place for the result, and the product beside it in one buffer."""
    from vkernels_b200.feedforward import DenseFeedForward

    g = torch.Generator(device=DEV)
    g.manual_seed(T)
    r = lambda *s: torch.randn(s, generator=g, device=DEV).to(torch.bfloat16)  # noqa: E731
    x, w13, w2 = r(T, 128), r(2 * 96, 128) * 0.1, r(128, 96) * 0.1
    ffn = DenseFeedForward(w13, w2, swiglu_limit=5.0)
    want = ffn(x, x)
    wide = r(T, 128 + 96)
    wide[:, :128] = x
    assert torch.equal(ffn(wide[:, :128], wide[:, :128], out=wide[:, :128], product=wide[:, 128:]), want)
    assert torch.equal(wide[:, :128], want) and torch.equal(wide[:, 128:], ffn.product(x))
    assert ffn(x, x, out=x) is x and torch.equal(x, want)


def test_recorded_gradients_of_no_tokens():
    g = torch.Generator(device=DEV)
    g.manual_seed(1)
    w13, w, b = (torch.randn(s, generator=g, device=DEV).to(torch.bfloat16).requires_grad_() for s in ((32, 64), (64, 16), (64,)))
    x = torch.empty(0, 64, dtype=torch.bfloat16, device=DEV, requires_grad=True)
    y = ops.fused_linear(ops.gated_linear(x, w13), w, b, activation="gelu", residual=x)
    grads = torch.autograd.grad(y.sum(), [x, w13, w, b])
    assert [tuple(t.shape) for t in grads] == [(0, 64), (32, 64), (64, 16), (64,)] and not any(bool(t.any()) for t in grads)
