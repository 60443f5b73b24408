"""-m gpu: the dense feed-forward operators against their definition in 64 bits, value by value, at bounds that count the
roundings (dense_oracle), on both kernels sets; refusals; strides, alignments, streams, graphs."""
import pytest
import torch

pytestmark = pytest.mark.gpu

import dense_oracle as ref  # noqa: E402
from vkernels_b200 import native_runtime as nr  # noqa: E402
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


# One gradient with few tiles and a long sum (many tokens of few features, or a few features behind many), beside another or alone.
LONG = [(4100, 128, 96), (9001, 70, 300), (100, 64, 4500), (300, 33, 2300), (2600, 250, 2500), (16384, 64, 64), (1, 40, 5000)]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("T,K,N", LONG)
def test_gradients_of_long_sums(T, K, N, dtype):
    for gated, gap in ((False, 0), (False, 3), (True, 0)):
        x, w, b, more = tensors(T, K, 2 * N if gated else N, dtype, gap=gap)
        dy = more(N + gap)[:, :N]
        d = dy.double()
        if gated:
            _, preact = ops.gated_linear(x, w, b, return_preact=True)
            _, dg, du, _, mg, mu = ref.gated(preact.double(), "swiglu", 0.0)
            dz, error = torch.cat([d * dg, d * du], 1), ref.APPROX * torch.cat([d.abs() * mg, d.abs() * mu], 1)
            call = lambda **kw: ops.gated_linear_backward(dy, x, w, preact, **kw)  # noqa: E731
        else:
            dz, error = d, torch.zeros_like(d)
            call = lambda **kw: ops.fused_linear_backward(dy, x, w, **kw)  # noqa: E731
        wanted = ref.gradients(dz, error, x, w, x.dtype, "tcgen05")
        both = call(bias_grad=True)
        for name, t, (value, bound) in zip(("dx", "dw", "db"), both, wanted):
            ref.assert_within(t, value, bound, f"{name} {gated} {gap}")
        ref.assert_within(call(w_grad=False)[0], *wanted[0], "dx alone")
        ref.assert_within(call(x_grad=False)[1], *wanted[1], "dw alone")
        assert all(torch.equal(p, q) for p, q in zip(call(bias_grad=True), both))
        assert torch.equal(call(x_grad=False, w_grad=False, bias_grad=True)[2], both[2])
    torch.cuda.synchronize()
    ops.kernel_status()


def test_parts_of_long_sums_in_a_workspace_on_16_bytes():
    """The sums' parts lie behind one another from the workspace's start on, which need not be a 32-byte one; nothing behind its end
    is written, nor beside the gradients."""
    T, K, N = 5000, 100, 90
    x, w, _, more = tensors(T, K, N, "bf16", bias=False, gap=4)   # pitches of 104
    dy = more(N + 6)[:, :N]                                       # 96
    wanted = ops.fused_linear_backward(dy, x, w)[1]
    lib = nr.load_library()
    nbytes = lib.vk_cuda_dense_backward_workspace_bytes(x.data_ptr(), 104, w.data_ptr(), 104, T, K, N, 0)
    room = torch.full((nbytes + 64,), 7, dtype=torch.uint8, device=DEV)
    assert room.data_ptr() % 256 == 0
    dw = torch.full((N, 107), 3.0, dtype=torch.bfloat16, device=DEV)
    torch.cuda.synchronize()
    rc = lib.vk_cuda_fused_linear_backward(dy.data_ptr(), 96, x.data_ptr(), 104, w.data_ptr(), 104, None, 0, None, K, dw.data_ptr(), 107,
                                           None, 0, T, K, N, 0, room.data_ptr() + 16, nbytes, torch.cuda.current_stream().cuda_stream)
    assert rc == 0, lib.vk_last_error()
    torch.cuda.synchronize()
    assert torch.equal(dw[:, :K], wanted) and bool((dw[:, K:] == 3).all())
    assert bool((room[:16] == 7).all()) and bool((room[16 + nbytes:] == 7).all())
    assert lib.vk_cuda_fused_linear_backward(dy.data_ptr(), 96, x.data_ptr(), 104, w.data_ptr(), 104, None, 0, None, K, dw.data_ptr(), 107,
                                             None, 0, T, K, N, 0, room.data_ptr(), 4096, torch.cuda.current_stream().cuda_stream) == 1
    lib.vk_set_last_error(0, b"")


# ---------------------------------------------------------------------------
# how the operators are called
# ---------------------------------------------------------------------------

def both(x, w13, w, r=None, **kw):
    return ops.gated_linear(x, w13), ops.fused_linear(x, w, residual=r, activation="silu")


def test_strides_and_leading_dimensions():
    """Rows of any pitch and start, in x, weights, residual and out; three dimensions; a transposed view is refused."""
    g = torch.Generator(device=DEV)
    g.manual_seed(1)
    T, K, N = 70, 136, 72
    r = lambda *s: torch.randn(s, generator=g, device=DEV).to(torch.bfloat16)  # noqa: E731
    x, w13, w, res = r(T, K), r(2 * N, K) * 0.1, r(N, K) * 0.1, r(T, N)
    want = both(x, w13, w, res)
    for pad, off in ((8, 0), (3, 0), (64, 5), (1, 1)):
        def loose(t):
            wide = torch.full((t.shape[0], t.shape[1] + pad + off), float("nan"), dtype=t.dtype, device=DEV)
            wide[:, off:off + t.shape[1]] = t
            return wide[:, off:off + t.shape[1]]
        got = both(loose(x), loose(w13), loose(w), loose(res))
        assert all(torch.equal(a, b) for a, b in zip(got, want)), (pad, off)
        out = torch.full((T, N + pad + off), 7.0, dtype=x.dtype, device=DEV)
        y = ops.fused_linear(x, w, residual=res, activation="silu", out=out[:, off:off + N])
        assert torch.equal(y, want[1]) and torch.equal(out[:, off:off + N], want[1])
        assert bool((out[:, :off] == 7).all()) and bool((out[:, off + N:] == 7).all())   # what lies beside the rows stays
    x3 = x.view(7, 10, K)
    assert torch.equal(ops.gated_linear(x3, w13).view(T, N), want[0]) and ops.gated_linear(x3, w13).shape == (7, 10, N)
    assert torch.equal(ops.fused_linear(x3, w, residual=res.view(7, 10, N), activation="silu").view(T, N), want[1])
    assert torch.equal(ops.gated_linear(x3[:, :4], w13), ops.gated_linear(x3[:, :4].contiguous(), w13))
    assert torch.equal(ops.gated_linear(x[5], w13), ops.gated_linear(x[5:6], w13)[0])
    in_place = res.clone()
    assert ops.fused_linear(x, w, residual=in_place, activation="silu", out=in_place) is in_place and torch.equal(in_place, want[1])
    with pytest.raises(ops.OpNotEligible, match="neighbours"):
        ops.fused_linear(x, r(K, N).T)
    with pytest.raises(ops.OpNotEligible, match="overlap"):
        ops.fused_linear(x, w, out=x[:, :N])


def test_results_do_not_depend_on_what_lies_behind_the_tensors():
    """Memory behind x, weights and results that holds NaN changes nothing and is not written."""
    for T, K, N in ((1, 72, 40), (5, 200, 24), (130, 72, 40), (300, 200, 136)):
        def inside(t):
            room = torch.full((t.numel() + 4096,), float("nan"), dtype=t.dtype, device=DEV)
            room[2048:2048 + t.numel()] = t.reshape(-1)
            return room, room[2048:2048 + t.numel()].view(t.shape)
        x, w13, b, more = tensors(T, K, 2 * N, "bf16")
        rooms, (x2, w2, b2) = zip(*[inside(t.contiguous()) for t in (x, w13, b)])
        out_room, out = inside(torch.zeros(T, N, dtype=x.dtype, device=DEV))
        assert torch.equal(ops.gated_linear(x2, w2, b2, out=out), ops.gated_linear(x, w13, b))
        assert bool(out_room[:2048].isnan().all()) and bool(out_room[2048 + T * N:].isnan().all())
        assert not bool(out.isnan().any())


@pytest.mark.parametrize("T", [0, 1, 3])
def test_smallest_batches(T):
    x, w13, b, more = tensors(T, 64, 32, "bf16")
    h, preact = ops.gated_linear(x, w13, b, return_preact=True)
    dx, dw, db = ops.gated_linear_backward(torch.ones_like(h), x, w13, preact, bias_grad=True)
    assert h.shape == (T, 16) and preact.shape == (T, 32) and dx.shape == x.shape and dw.shape == w13.shape and db.shape == (32,)
    if T == 0:
        assert not dw.any() and not db.any()      # sums over no tokens
        assert ops.fused_linear(x.view(0, 2, 32), w13[:, :32]).shape == (0, 2, 32)
        assert ops.fused_linear_backward(torch.empty(0, 32, dtype=x.dtype, device=DEV), x, w13)[0].shape == (0, 64)


def test_special_values():
    """inf and NaN come out where the definition has them, in their own rows only; the clamp keeps a NaN."""
    for T in (4, 200):
        x, w13, _, _ = tensors(T, 64, 64, "bf16")
        w13 = w13.abs() + 0.01        # an infinite input then meets no opposite one
        x[1, 3] = float("inf")
        x[2, 5] = float("-inf")
        x[3, 7] = float("nan")
        z, _ = ref.project(x, w13)
        for kind, limit in (("swiglu", 0.0), ("swiglu", 2.0), ("situ", 0.0)):
            got = ops.gated_linear(x, w13, activation=KIND[kind], swiglu_limit=limit).double()
            want = ref.gated(z, kind, limit)[0]
            assert torch.equal(got.isnan(), want.isnan()), (kind, limit)
            assert torch.equal(got.isinf(), want.isinf()) and torch.equal(got[want.isinf()], want[want.isinf()])
        for act in (None, "silu", "gelu", "gelu_tanh"):
            got, want = ops.fused_linear(x, w13, activation=act).double(), ref.linear_act(z, act)[0]
            assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got[want.isinf()], want[want.isinf()]), act
    big = torch.full((2, 8), 200.0, dtype=torch.float16, device=DEV)
    assert bool(ops.fused_linear(big, big).isinf().all())       # beyond fp16's range: 320000
    w = big.repeat(2, 1)[:4]
    y, preact = ops.fused_linear(big, w, activation="silu", return_preact=True)
    dx, dw, db = ops.fused_linear_backward(torch.full_like(y, 1e-3), big, w, preact, activation="silu", bias_grad=True)
    assert bool((preact == 320000).all()) and bool(db.isfinite().all()) and bool(dx.isfinite().all())   # the slope there is 1


def test_the_clamp_decides_on_unrounded_sums():
    """A pre-activation just above the limit, that would round to it, has no gradient; one just below has."""
    x = torch.ones(1, 8, dtype=torch.bfloat16, device=DEV)
    w13 = torch.zeros(4, 8, dtype=torch.bfloat16, device=DEV)
    w13[0, 0], w13[0, 1] = 7.0, 2.0 ** -9          # gate 7.002: above 7, nearest bf16 value 7
    w13[1, 0], w13[1, 1] = 7.0, -(2.0 ** -9)
    w13[2:, 0] = 1.0
    h, preact = ops.gated_linear(x, w13, swiglu_limit=7.0, return_preact=True)
    _, dw, _ = ops.gated_linear_backward(torch.ones_like(h), x, w13, preact, swiglu_limit=7.0)
    assert not dw[0].any() and bool((dw[1] != 0).all())


def test_same_bits_every_time_and_on_every_stream():
    x, w13, b, more = tensors(333, 640, 512, "bf16")
    dh = more(256)
    h, preact = ops.gated_linear(x, w13, b, return_preact=True)
    first = (h, preact, *ops.gated_linear_backward(dh, x, w13, preact, bias_grad=True))
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = []
    for i in range(12):
        with torch.cuda.stream(streams[i % 3]):
            h, preact = ops.gated_linear(x, w13, b, return_preact=True)
            got.append((h, preact, *ops.gated_linear_backward(dh, x, w13, preact, bias_grad=True)))
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, first))


@pytest.mark.parametrize("T", [1, 48, 300, 4100])
def test_captured_graphs_share_nothing(T):
    """Two graphs of forward and backward, captured on one stream and replayed on two at once, on new inputs."""
    cases = []
    capture = torch.cuda.Stream()
    for seed in (1, 2):
        x, w13, b, more = tensors(T, 264, 2 * 136, "bf16", seed=seed)
        dh = more(136)

        def step(x=x, w13=w13, b=b, dh=dh):
            h, preact = ops.gated_linear(x, w13, b, swiglu_limit=1.5, return_preact=True)
            return (h, *ops.gated_linear_backward(dh, x, w13, preact, swiglu_limit=1.5, bias_grad=True))
        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=capture):
            out = step()
        cases.append((graph, out, step, x, dh))
    side = [torch.cuda.Stream() for _ in cases]
    for round_ in range(3):
        for graph, out, step, x, dh in cases:
            x.mul_(0.75)
            dh.mul_(-1.25)
        torch.cuda.synchronize()
        for _ in range(4):
            for s, (graph, *_) in zip(side, cases):
                with torch.cuda.stream(s):
                    graph.replay()
        torch.cuda.synchronize()
        for graph, out, step, x, dh in cases:
            assert all(torch.equal(a, b) for a, b in zip(out, step())), round_
    ops.kernel_status()


def test_kernels_that_follow_one_another_see_each_others_results():
    """Calls may start before the ones ahead of them have ended: every result still is that of its own inputs, through chains of
    small calls that feed each other and buffers that are written again."""
    x, w, _, _ = tensors(3, 256, 256, "bf16", std=1.0)
    want = x
    for _ in range(20):
        want = ops.fused_linear(want, w, activation="silu")
        torch.cuda.synchronize()
    a, b = torch.empty_like(x), torch.empty_like(x)
    for _ in range(5):
        a.copy_(x)
        for _ in range(10):
            ops.fused_linear(a, w, activation="silu", out=b)
            ops.fused_linear(b, w, activation="silu", out=a)
        assert torch.equal(a, want)


# ---------------------------------------------------------------------------
# recorded gradients
# ---------------------------------------------------------------------------

def test_recorded_gradients_are_the_backward_operators():
    x, w13, b, more = tensors(50, 136, 2 * 72, "bf16")
    x, w13 = x.clone(), w13.clone()
    dh = more(72)
    h, preact = ops.gated_linear(x, w13, b, swiglu_limit=2.0, return_preact=True)
    want = ops.gated_linear_backward(dh, x, w13, preact, swiglu_limit=2.0, bias_grad=True)
    leaves = [t.requires_grad_() for t in (x, w13, b)]
    got = ops.gated_linear(*leaves, swiglu_limit=2.0)
    assert torch.equal(got, h) and got.requires_grad
    grads = torch.autograd.grad(got, leaves, dh)
    assert all(torch.equal(p, q) for p, q in zip(grads, want))
    # a part of the leaves; a sum, whose gradient is one expanded number; the same weight twice
    dx, = torch.autograd.grad(ops.gated_linear(x, w13.detach(), b.detach(), swiglu_limit=2.0), [x], dh)
    assert torch.equal(dx, want[0])
    w = w13.detach()[:, :72].clone().requires_grad_()            # [144, 72]
    res = more(144).requires_grad_()
    y = ops.fused_linear(h.detach(), w, residual=res, activation="gelu")
    gw, gr = torch.autograd.grad(y.sum(), [w, res])
    one = torch.ones(50, 144, dtype=torch.bfloat16, device=DEV)
    _, preact = ops.fused_linear(h, w.detach(), activation="gelu", return_preact=True)
    assert torch.equal(gw, ops.fused_linear_backward(one, h, w.detach(), preact, activation="gelu")[1]) and torch.equal(gr, one)
    sq = torch.randn(72, 72, device=DEV).to(torch.bfloat16).requires_grad_()
    h2 = h.detach()
    once = [ops.fused_linear_backward(d, v, sq.detach())[:2] for d, v in ((dh, ops.fused_linear(h2, sq.detach())),)]
    twice, = torch.autograd.grad(ops.fused_linear(ops.fused_linear(h2, sq), sq), [sq], dh)
    inner = ops.fused_linear_backward(once[0][0], h2, sq.detach())[1]
    assert torch.equal(twice, once[0][1] + inner)
    x3 = x.detach().view(5, 10, 136).requires_grad_()
    g3, = torch.autograd.grad(ops.gated_linear(x3, w13.detach(), b.detach(), swiglu_limit=2.0), [x3], dh.view(5, 10, 72))
    assert torch.equal(g3.view(50, 136), want[0])


def test_recording_refuses_what_it_cannot_do():
    x, w13, b, more = tensors(8, 64, 32, "bf16")
    w13 = w13.clone().requires_grad_()
    with pytest.raises(ops.OpNotEligible, match="no gradient"):
        ops.gated_linear(x, w13, out=torch.empty(8, 16, dtype=x.dtype, device=DEV))
    with pytest.raises(ops.OpNotEligible, match="no gradient"):
        ops.fused_linear(x, w13, return_preact=True)
    with torch.no_grad():
        ops.fused_linear(x, w13, return_preact=True)
    y = ops.fused_linear(x.clone().requires_grad_(), w13)
    g, = torch.autograd.grad(y, [w13], torch.ones_like(y), create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable|does not require grad"):
        torch.autograd.grad(g.sum(), [w13])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(ops.OpNotEligible, match="captured"):
        with torch.cuda.graph(graph):
            ops.fused_linear(x, w13)
    torch.cuda.synchronize()
    changed = w13.detach().clone().requires_grad_()
    y = ops.fused_linear(x, changed)
    with torch.no_grad():
        ops.fused_linear(x, w13, out=changed[:8, :32])          # writes a saved weight: backward must notice
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward(torch.ones_like(y))


def test_what_is_not_a_tensor_is_refused():
    x, w13, b, more = tensors(8, 64, 32, "bf16")
    dy = more(32)
    for call in (lambda: ops.gated_linear(x, w13, [0.0] * 32), lambda: ops.fused_linear(x, w13, [0.0] * 32), lambda: ops.fused_linear(x, w13, residual=1.0),
                 lambda: ops.fused_linear_backward(dy, x, w13, 1.0, activation="silu"), lambda: ops.fused_linear_backward(None, x, w13),
                 lambda: ops.gated_linear_backward(dy[:, :16], x, w13, "none"), lambda: ops.fused_linear(x.cpu(), w13), lambda: ops.fused_linear(x, w13.cpu())):
        with pytest.raises(ops.OpNotEligible):
            call()


def test_directional_differences():
    """The recorded gradients against differences of the forward operator itself, along the gradient: fp16 results are good to
    2^-11 of themselves each, the step moves the loss by a tenth."""
    x, w13, b, more = tensors(24, 96, 2 * 40, "fp16", std=1.0)
    leaves = [t.clone().requires_grad_() for t in (x, w13, b)]
    c = more(40).double()
    loss = lambda *t: (ops.gated_linear(*t, swiglu_limit=3.0).double() * c).sum()  # noqa: E731
    grads = torch.autograd.grad(loss(*leaves), leaves)
    with torch.no_grad():
        for i, g in enumerate(grads):
            def moved(step):
                t = [v.detach() for v in leaves]
                t[i] = (t[i].double() + step * g.double()).to(x.dtype)
                return t
            step = 0.02 / float(g.double().norm())
            up, down = moved(step), moved(-step)
            change = float(loss(*up) - loss(*down))
            expected = float((g.double() * (up[i].double() - down[i].double())).sum())
            # results: h of each value at either end, independent: the 2-norm; curvature along the step: a thousandth
            noise = 2 * ref.half_step(torch.float16) * float((ops.gated_linear(*leaves, swiglu_limit=3.0).double() * c).norm())
            assert abs(change - expected) <= 4 * noise + 0.02 * abs(expected), (i, change, expected)


# ---------------------------------------------------------------------------
# the layer, and beside the routed experts
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("T", [1, 37, 300])
def test_feed_forward_runs_both_projections(T, dtype):
    from vkernels_b200.feedforward import DenseFeedForward

    H, ispp = 192, 136
    x, w13, b13, more = tensors(T, H, 2 * ispp, dtype)
    g = torch.Generator(device=DEV)
    g.manual_seed(5)
    w2 = (torch.randn(H, ispp, generator=g, device=DEV) / ispp ** 0.5).to(x.dtype)
    b2 = torch.randn(H, generator=g, device=DEV).to(x.dtype)
    res, dy = more(H), more(H)
    params = [t.clone().requires_grad_() for t in (x, w13, b13, w2, b2, res)]
    px, p13, pb13, p2, pb2, pres = params
    y = DenseFeedForward(p13, p2, b13=pb13, b2=pb2, swiglu_limit=3.0)(px, pres)
    grads = torch.autograd.grad(y, params, dy)
    plain = DenseFeedForward(w13, w2, b13=b13, b2=b2, swiglu_limit=3.0)
    keep = res.clone()
    assert torch.equal(plain(x, keep, out=keep, product=torch.empty(T, ispp, dtype=x.dtype, device=DEV)), y)
    # 64 bits from end to end; h: the product and its gradient are rounded between the projections, each once
    d = [t.detach().double().requires_grad_() for t in params]
    z, mags = ref.project(d[0], d[1], d[2])
    hid = ref.gated(z, "swiglu", 3.0)[0]
    want = hid @ d[3].T + d[4] + d[5]
    h = ref.half_step(x.dtype)
    rel = lambda a, b: float((a.double() - b).norm() / b.norm())  # noqa: E731
    assert rel(y, want) <= 2 * h
    for name, a, b_ in zip(("x", "w13", "b13", "w2", "b2", "residual"), grads, torch.autograd.grad(want, d, dy.double())):
        assert rel(a, b_) <= 4 * h, name      # at most four roundings of half a step each on the way


@pytest.mark.parametrize("T", [1, 40, 600])
def test_shared_expert_beside_the_routed_ones(T):
    """FusedMoEMxfp4 with a bf16 always-on expert: the routed layer's own result plus the feed-forward, eager and replayed."""
    from gpu_common import make_case
    from vkernels_b200 import synthetic as syn
    from vkernels_b200.experts import layer_from_config
    from vkernels_b200.feedforward import DenseFeedForward

    cfg = syn.scaled(syn.CONFIGS["c0"], H=512, I=256, E=8, top_k=2)
    w, A, r = make_case(cfg, T, backend="torch")
    g = torch.Generator(device=DEV)
    g.manual_seed(3)
    ispp = 192
    w13 = (torch.randn(2 * ispp, cfg.H, generator=g, device=DEV) / cfg.H ** 0.5).to(torch.bfloat16)
    w2 = (torch.randn(cfg.H, ispp, generator=g, device=DEV) / ispp ** 0.5).to(torch.bfloat16)
    ffn = DenseFeedForward(w13, w2)
    routed = layer_from_config(cfg, w, r, max_tokens=T)
    layer = layer_from_config(cfg, w, r, max_tokens=T, shared_ffn=ffn)
    base = routed(A).clone()
    want = ffn(A, base)
    got = layer(A)
    assert torch.equal(got, want) or T > 256 and torch.allclose(got.float(), want.float(), atol=2e-2, rtol=2.0 ** -7)
    assert not torch.equal(want, base)
    graph, y = layer.capture(A)
    first = layer(A).clone()
    for scale in (1.0, 0.5):
        A.mul_(scale)
        graph.replay()
        torch.cuda.synchronize()
        want = ffn(A, routed(A))
        assert torch.equal(y, want) or T > 256 and torch.allclose(y.float(), want.float(), atol=2e-2, rtol=2.0 ** -7)
    assert first.shape == y.shape
    ops.kernel_status()


def test_columns_of_one_buffer():
    """x, residual and result as columns of one wider buffer: read and written where they lie."""
    x, w, b, more = tensors(70, 72, 40, "bf16")
    wide = more(200)
    wide[:, 8:80] = x
    want = ops.fused_linear(x, w, b, residual=wide[:, 80:120].clone())
    keep = wide.clone()
    got = ops.fused_linear(wide[:, 8:80], w, b, residual=wide[:, 80:120], out=wide[:, 120:160])
    assert torch.equal(got, want)
    keep[:, 120:160] = want
    assert torch.equal(wide, keep)


def test_offsets_beyond_32_bits():
    """More than 2^31 elements in the result, the residual, x (as columns of that result) and the pre-activations."""
    T, K, N = 266000, 64, 8256
    x, w, b, more = tensors(T, K, N, "bf16")
    y = ops.fused_linear(x, w, b)
    assert y.numel() > 2 ** 31
    some = torch.tensor([0, 1, T // 2 + 5, T - 3, T - 1], device=DEV)
    z, mags = ref.project(x[some], w, b)
    bound = ref.sum_error(K) * mags
    ref.assert_within(y[some], z, bound + ref.half_step(y.dtype) * (z.abs() + bound), "y")
    tail = y[:, N - 64:]                       # the last 64 columns: rows 16512 bytes apart
    w13 = w[:64, :64]
    h, preact = ops.gated_linear(tail, w13, return_preact=True)
    assert torch.equal(h, ops.gated_linear(tail.contiguous(), w13))
    dx, dw, _ = ops.gated_linear_backward(more(32), tail, w13, preact)
    assert dx.shape == (T, 64) and bool(dx[some].isfinite().all())
    before = y[some].clone()
    del h, preact, dx, dw
    again = ops.fused_linear(x, w, b, residual=y, out=y)         # in place: residual and result far beyond 2^31
    value = z + before.double()
    ref.assert_within(again[some], value, bound + 2.0 ** -23 * value.abs() + ref.half_step(y.dtype) * (value.abs() + bound), "y + y")
    ops.kernel_status()


_FIRST_CALL = """
import sys
sys.path.insert(0, {root!r})
import torch
from vkernels_b200 import torch_ops as ops
for T in (4, 400):
    x = torch.randn(T, 128, device="cuda").to(torch.bfloat16)
    w = torch.randn(192, 128, device="cuda").to(torch.bfloat16)
    dy = torch.randn(T, 96, device="cuda").to(torch.bfloat16)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        h, preact = ops.gated_linear(x, w, return_preact=True)
        grads = ops.gated_linear_backward(dy, x, w, preact, bias_grad=True)
    g.replay()
    torch.cuda.synchronize()
    want = ops.gated_linear(x, w)
    assert torch.equal(h, want)
    assert all(torch.equal(a, b) for a, b in zip(grads, ops.gated_linear_backward(dy, x, w, preact, bias_grad=True)))
print("replayed")
# a backward pass of a graph recorded before the capture: refused with an exception, and the process lives on
x = torch.randn(8, 64, device="cuda").to(torch.bfloat16).requires_grad_()
w = torch.randn(32, 64, device="cuda").to(torch.bfloat16).requires_grad_()
y = ops.gated_linear(x, w)
torch.cuda.synchronize()
try:
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        torch.autograd.grad(y, [x, w], torch.ones_like(y))
except Exception as e:
    print("refused", type(e).__name__)
torch.cuda.synchronize()
y = ops.gated_linear(x, w)
y.sum().backward()
print("alive", bool(x.grad.isfinite().all()))
"""


def test_first_call_of_a_process_inside_a_capture():
    import os
    import subprocess
    import sys

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", _FIRST_CALL.format(root=root)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "replayed" in r.stdout and "refused" in r.stdout and "alive True" in r.stdout, (r.stdout, r.stderr[-2000:])


@pytest.mark.parametrize("T,N,gap", [(1, 512, 0), (40, 333, 0), (300, 512, 0), (700, 1000, 8), (600, 333, 0), (520, 770, 3)])
def test_result_in_place_of_the_residual(T, N, gap):
    """Every tile reads its part of the residual before it writes it, whichever kernel runs and however the rows lie."""
    x, w, b, more = tensors(T, 200, N, "bf16")
    room = more(N + gap)
    res = room[:, :N]
    want = ops.fused_linear(x, w, b, activation="gelu", residual=res.clone())
    beside = room[:, N:].clone()
    assert torch.equal(ops.fused_linear(x, w, b, activation="gelu", residual=res, out=res), want)
    assert torch.equal(room[:, N:], beside)
