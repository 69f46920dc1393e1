"""Calls of the matrix and token operators that their documentation allows and that are easy to get wrong: weights with several uses
in one pass, forward-mode derivatives, ties and NaN beyond a list's room, sizes past what an index holds."""
import math

import pytest
import torch
import torch.nn as tnn

from distributed_deep_learning_amd import nn as dnn
from distributed_deep_learning_amd.nn import functional as F
from distributed_deep_learning_amd.ops import kernels as K
from distributed_deep_learning_amd.ops import streams
from distributed_deep_learning_amd.parallel import ParamArena

gpu = pytest.mark.gpu
B8, H24 = 2.0 ** -8, 2.0 ** -24
BF = torch.bfloat16


def _randn(seed, *shape, scale=1.0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale


def _arena(*weights, device="cpu"):
    net = tnn.ParameterList([tnn.Parameter(w.float().to(device)) for w in weights])
    return net, ParamArena(net.named_parameters())


# ================================================================================================= gradients in an arena
class _Direct(torch.autograd.Function):
    """A layer that adds its weight's gradient to the arena by itself, as the kernels do."""

    @staticmethod
    def forward(ctx, x, w, log):
        ctx.log = log
        return x * 1.0

    @staticmethod
    def backward(ctx, g):
        ctx.log.append("direct")
        return g, None, None


def test_autograd_adds_to_an_arena_weight_behind_the_side_stream(monkeypatch):
    """A penalty on a weight beside a layer that adds to its gradient directly: autograd's addition is ordered behind the side stream, once,
    after every use, and not asked for where autograd adds nothing."""
    (w,), _ = net, arena = _arena(_randn(1, 6, 8))
    log = []
    monkeypatch.setattr(streams, "order", lambda device: log.append(w.grad.clone()), raising=False)
    x = torch.ones(3, requires_grad=True)
    for loss in (lambda: _Direct.apply(x, w, log).sum() + w.pow(2).sum(), lambda: w.pow(2).sum() + _Direct.apply(x, w, log).sum()):
        arena.zero_grad()
        log.clear()
        loss().backward()
        assert len(log) == 2 and log[0] == "direct" and torch.equal(log[1], torch.zeros_like(w))
        assert torch.equal(w.grad, 2 * w.detach())
    log.clear()
    _Direct.apply(x, w, log).sum().backward()
    assert log == ["direct"]


@gpu
def test_penalty_beside_a_direct_gradient_loses_nothing():
    """Linear and the gated block add to their weights' gradients on the side stream while autograd adds a penalty's."""
    T, D, H = 4096, 512, 1024
    x, dy = _randn(2, T, D).to(BF).cuda(), _randn(3, T, D, scale=0.1).to(BF).cuda()
    torch.manual_seed(0)
    net = tnn.ModuleList([dnn.GatedMLP(D, H), dnn.Linear(D, D)]).cuda()
    arena = ParamArena(net.named_parameters())
    run = lambda: net[1](net[0](x))                                                  # noqa: E731
    run().backward(dy)
    torch.cuda.synchronize()
    plain = {n: p.grad.clone() for n, p in net.named_parameters()}
    for _ in range(5):
        arena.zero_grad()
        pen = sum((100.0 * p).sum() for p in net.parameters())                       # its gradient is exactly 100
        torch.autograd.backward([run(), pen], [dy, torch.ones((), device="cuda")])
        for n, p in net.named_parameters():
            # 100 + g rounds once per addition; Linear's parts meet in any order
            tol = 4 * 2 * H24 * (100 + plain[n].abs()) + (1e-5 * plain[n].abs().max() if n.startswith("1") else 0.0)
            assert float(((p.grad - 100.0 - plain[n]).abs() - tol).max()) <= 0.0, n


def _spy_dw(monkeypatch):
    """What the gated block's weight gradients are computed into: one list of three truth values a launch, and whether it adds."""
    seen, real = [], K.gated_dw

    def dw(x, dy, kept, dgu, out, M, D, F_, accumulate=False):
        seen.append(([t is not None for t in out], accumulate))
        return real(x, dy, kept, dgu, out, M, D, F_, accumulate)

    monkeypatch.setattr(K, "gated_dw", dw)
    return seen


@gpu
@pytest.mark.parametrize("twice_first", [True, False])
def test_gated_mlp_arena_weight_alone_in_one_call_and_twice_in_another(monkeypatch, twice_first):
    """One arena weight, once as gate beside another (added by the kernel) and once as gate and up (left to autograd), in one pass: nothing is
    lost.  The parts are the same fp32 values everywhere; only up to four additions of them round."""
    T, D, H = 2048, 256, 1032
    x, dy = _randn(11, T, D).to(BF).cuda(), _randn(12, T, D, scale=0.1).to(BF).cuda()
    w = [_randn(13, H, D, scale=D ** -0.5).to(BF), _randn(14, H, D, scale=D ** -0.5).to(BF), _randn(15, D, H, scale=H ** -0.5).to(BF)]
    leaves = [t.float().cuda().requires_grad_() for t in w]
    g0, u1, d2 = torch.autograd.grad(F.gated_mlp(x, *leaves), leaves, dy)
    twin = [leaves[0], leaves[0].detach().clone().requires_grad_(), leaves[2]]
    ga, gb, gd = torch.autograd.grad(F.gated_mlp(x, *twin), twin, dy)
    net, arena = _arena(*w, device="cuda")
    seen = _spy_dw(monkeypatch)
    calls = [lambda: F.gated_mlp(x, net[0], net[0], net[2]), lambda: F.gated_mlp(x, net[0], net[1], net[2])]
    for _ in range(3):
        arena.zero_grad()
        seen.clear()
        ys = [f() for f in (calls if twice_first else calls[::-1])]
        torch.autograd.backward(ys, [dy, dy])
        assert sorted(seen) == sorted([([False, False, True], True), ([True, True, False], False), ([True, True, True], True)])
        for p, terms in zip(net, ((g0, ga, gb), (u1,), (d2, gd))):
            assert arena.grad_is_arena_view(p)
            tol = 4 * H24 * sum(t.abs() for t in terms)
            assert float(((p.grad - sum(terms)).abs() - tol).max()) <= 0.0


@gpu
def test_gated_mlp_gate_outside_the_arena_beside_weights_in_it(monkeypatch):
    """A gate derived from something else (an adapter merged into it): the other weights' gradients still go straight to the arena."""
    T, D, H = 300, 64, 264
    x, dy = _randn(21, T, D).to(BF).cuda(), _randn(22, T, D, scale=0.1).to(BF).cuda()
    w = [_randn(23, H, D, scale=D ** -0.5).to(BF), _randn(24, H, D, scale=D ** -0.5).to(BF), _randn(25, D, H, scale=H ** -0.5).to(BF)]
    leaves = [t.float().cuda().requires_grad_() for t in w]
    ref = torch.autograd.grad(F.gated_mlp(x, *leaves), leaves, dy)
    net, arena = _arena(*w[1:], device="cuda")
    base = w[0].float().cuda().requires_grad_()
    seen = _spy_dw(monkeypatch)
    for dtype in (torch.float32, BF):
        arena.zero_grad()
        seen.clear()
        base.grad = None
        F.gated_mlp(x, (base * 1.0).to(dtype), net[0], net[1]).backward(dy)
        assert seen == [([False, True, True], True), ([True, False, False], False)]
        assert torch.equal(net[0].grad, ref[1]) and torch.equal(net[1].grad, ref[2])
        assert torch.equal(base.grad, ref[0].to(dtype).float())


@gpu
def test_reducer_hears_of_a_shared_gated_weight_behind_its_last_use():
    """Two blocks with the same weights: when the first signal of a tensor arrives (the one the reducer counts), its gradient is whole."""
    T, D, H = 700, 128, 520
    x, dy = _randn(31, T, D).to(BF).cuda(), _randn(32, T, D, scale=0.1).to(BF).cuda()
    block = dnn.GatedMLP(D, H).cuda()
    arena = ParamArena(block.named_parameters())
    snaps = {}

    def ready(seg):
        if seg not in snaps:
            s = arena.segments[seg]
            with streams.comm_context(arena.grad):                                    # as a collective would be enqueued
                snaps[seg] = arena.grad[s.offset:s.offset + s.numel].clone()

    arena.on_grad_ready = ready
    for p in arena.params:
        p.register_post_accumulate_grad_hook(lambda p: ready(p._ddl_segment))
    block(block(x)).backward(dy)
    torch.cuda.synchronize()
    assert sorted(snaps) == [0, 1, 2]
    for seg, snap in snaps.items():
        s = arena.segments[seg]
        assert float(snap.abs().sum()) > 0.0 and torch.equal(snap, arena.grad[s.offset:s.offset + s.numel])


# ================================================================================================= token log probabilities
@gpu
@pytest.mark.parametrize("dtype", [torch.float32, BF])
@pytest.mark.parametrize("N,V,top", [(520, 5003, 5), (1, 4099, 3), (2, 4096, 64), (1, 70_000, 64), (1, 900, 20)])
def test_token_logprobs_list_of_rows_of_nothing_but_nan(N, V, top, dtype):
    """More elements tie at the top than a list holds, the first of them at index 0: in one part, in several, and where the parts are joined."""
    z = torch.full((N, V), float("nan"), dtype=dtype)
    z[N // 2, 1:] = 2.0                                                              # and one NaN at index 0 above a long tie
    tok = torch.zeros(N, dtype=torch.int64)
    out, cpu = F.token_logprobs(z.cuda(), tok.cuda(), top), F.token_logprobs(z, tok, top)
    for o in (out, cpu):
        assert torch.isnan(o[2]).all() and torch.equal(o[3].cpu(), torch.arange(top).expand(N, top))


# ================================================================================================= derivatives
@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_forward_mode_derivatives_are_right_or_refused(device):
    """Never a result without its tangent."""
    import torch.autograd.forward_ad as fw
    z, t = _randn(41, 4, 30).to(device), _randn(42, 4, 30).to(device)
    tok = torch.tensor([1, 2, 3, 29]).to(device)
    x, dx, w, wd = (_randn(43 + i, *s).to(device) for i, s in enumerate(((4, 16), (4, 16), (24, 16), (16, 24))))
    calls = [lambda f: F.token_logprobs(f(z, t), tok, 2)[0], lambda f: F.gated_mlp(f(x, dx), w, w, wd), lambda f: F.gated_mlp(x, w, f(w, 0.5 * w), wd)]
    for grad in (True, False):
        for call in calls:
            with torch.set_grad_enabled(grad), fw.dual_level():
                if device == "cuda":
                    with pytest.raises(NotImplementedError, match="forward-mode"):
                        call(fw.make_dual)
                else:
                    assert fw.unpack_dual(call(fw.make_dual)).tangent is not None
                assert call(lambda p, _: p) is not None                              # inside a level, without a tangent
    logq = torch.log_softmax(z.cpu().double(), 1)
    ref = (t.cpu().double() - (logq.exp() * t.cpu()).sum(1, keepdim=True)).gather(1, tok.cpu()[:, None])[:, 0]
    if device == "cpu":
        with fw.dual_level():
            assert torch.allclose(fw.unpack_dual(calls[0](fw.make_dual)).tangent.double(), ref, atol=1e-5)


@gpu
def test_orthogonalize_is_detached_from_a_weight_that_requires_a_gradient():
    w = _randn(51, 40, 70).cuda().requires_grad_()
    out = K.orthogonalize(w)
    assert not out.requires_grad and torch.equal(out, K.orthogonalize(w.detach()))


# ================================================================================================= sizes
def test_gated_mlp_sizes_past_32_bit_offsets_are_refused():
    """128 rows of more than 2^24 16-bit elements span 4 GiB: a lane's offset would wrap and read another row."""
    most = 1 << 24
    K.check_gated_sizes(K.GATED_MAX_TOKENS, most, most)
    for sizes in ((1, most + 1, 8), (1, 8, most + 1), (K.GATED_MAX_TOKENS + 1, 8, 8), (2 ** 32 + 5, 8, 8), (8, 2 ** 32 + 8, 8)):
        with pytest.raises(ValueError):
            K.check_gated_sizes(*sizes)
    if K._lib.available():
        work = K._lib.require().ddl_gated_workspace
        assert work(200, 256, most, 0) > 0
        for sizes in ((200, most + 1, 256), (200, 256, most + 1), (-1, 8, 8), (0x7fffff01, 8, 8)):
            assert all(work(*sizes, p) == -1 for p in (0, 1, 2))


@gpu
def test_gated_mlp_refuses_long_rows_before_it_reads_them():
    one = torch.zeros(1, dtype=BF, device="cuda")
    for T, D, H in ((1, (1 << 24) + 8, 8), (1, 8, (1 << 24) + 8), (2 ** 32 + 5, 8, 8)):
        with pytest.raises(ValueError, match="at most"):
            F.gated_mlp(one.expand(T, D), one.expand(H, D), one.expand(H, D), one.expand(D, H))


@gpu
@pytest.mark.parametrize("T", [3, 130])
def test_gated_mlp_of_the_widest_rows(T):
    """Rows of 2^24 elements: the last rows and columns count.  All operands are powers of two with few bits, so every product and sum is exact
    up to the rounding of h and of the results."""
    D, H = 1 << 24, 136
    x = torch.zeros(T, D, dtype=BF, device="cuda")
    wg, wu = torch.zeros(2, H, D, dtype=BF, device="cuda")
    wd = torch.zeros(D, H, dtype=BF, device="cuda")
    k = torch.tensor([0, 1, D // 2 + 3, D - 2, D - 1], device="cuda")
    r = lambda i, *s: (torch.randint(1, 5, s, generator=torch.Generator().manual_seed(i)).float() / 4).to(BF).cuda()      # noqa: E731
    x[:, k], wg[:, k], wu[:, k], wd[k] = r(1, T, 5), r(2, H, 5), r(3, H, 5), r(4, 5, H)
    with torch.no_grad():
        y = F.gated_mlp(x, wg, wu, wd, activation="relu")
    g, u = (x[:, k].double() @ w[:, k].double().T for w in (wg, wu))
    h = g.relu() * u
    ref = h @ wd[k].double().T
    tol = (B8 * (h @ wd[k].double().T.abs()) + B8 * ref.abs()) * 1.01
    assert float(((y[:, k].double() - ref).abs() - tol).max()) <= 0.0
    y[:, k] = 0
    assert float(y.abs().max()) == 0.0


def test_orthogonalize_sizes_past_32_bit_offsets_are_refused():
    """128 split rows of more than 2^23 elements span 4 GiB of hi and lo values: a lane's offset would wrap and read another row."""
    if not K._lib.available():
        pytest.skip("kernel library not built")
    plan, f32 = K.orthogonalize_plan, torch.float32
    for ok in ((1, 128, 1 << 23, f32), (1, 1 << 26, 128, f32), (1, 2, 1 << 25, f32), (1, 1, (1 << 30) - 64, BF), (1, 200, 1 << 24, BF), (1 << 30, 4, 4, f32)):
        assert plan(*ok)[1] >= 0
    for bad in ((1, 128, (1 << 23) + (1 << 17), f32), (1, 64, 1 << 25, f32), (1, 200, (1 << 24) + (1 << 18), BF), (1, 2 ** 32 + 5, 4, f32), (1, 4, 2 ** 32 + 5, BF),
                (2 ** 32 + 3, 4, 4, f32), (1, 1, 1 << 30, f32)):
        with pytest.raises(ValueError, match="too large"):
            plan(*bad)
    if torch.cuda.is_available():
        with pytest.raises(ValueError, match="too large"):
            K.orthogonalize(torch.zeros(1, device="cuda").expand(128, 1 << 24))


@gpu
@pytest.mark.parametrize("shape", [(3, 1 << 22), (1 << 22, 3)])
def test_orthogonalize_of_long_rows(shape):
    """Rows far longer than a tile, against 64 bits: as in the small cases, with sums of 2^22 products, sqrt(2^22) 2^-24 each, in one product of three."""
    g = torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(5), device="cuda")
    x = g.double() / (g.double().norm() + 1e-7)
    x = x.t() if shape[0] > shape[1] else x
    a, b, c = K.NS_COEFFICIENTS
    for _ in range(5):
        s = x.contiguous() @ x.t().contiguous()
        x = a * x + (b * s + c * s @ s) @ x
    ref = x.t() if shape[0] > shape[1] else x
    tol = 30 * 2.0 ** -22 + 5 * 2048 * H24
    assert float((K.orthogonalize(g).double() - ref).norm()) <= tol * float(ref.norm())


@gpu
def test_token_logprobs_refuses_vocabularies_past_31_bits():
    one = torch.zeros(1, dtype=BF, device="cuda")
    for V in (2 ** 31, 2 ** 32 + 5):
        with pytest.raises(ValueError, match="vocabulary"):
            F.token_logprobs(one.expand(1, V), torch.zeros(1, dtype=torch.int64, device="cuda"))


@gpu
def test_token_logprobs_of_more_rows_than_a_launch_has_blocks():
    """2^24 rows and some: forward, list and gradient of rows on both sides of the cut equal those of the rows alone."""
    N, V = (1 << 24) + 1000, 8
    z = torch.randn(N, V, generator=torch.Generator(device="cuda").manual_seed(6), device="cuda", dtype=BF).requires_grad_()
    tok = torch.arange(N, device="cuda") % (V + 1)                                   # every ninth row is padding
    pick = torch.cat([torch.arange(300), torch.arange((1 << 24) - 300, (1 << 24) + 300), torch.arange(N - 300, N)]).cuda()
    out = F.token_logprobs(z, tok, 3)
    heads = [out[0].sum(), out[1].sum(), out[2].square().sum()]
    (dz,) = torch.autograd.grad(sum(heads), z)
    few = z.detach()[pick].requires_grad_()
    ref = F.token_logprobs(few, tok[pick], 3)
    (dr,) = torch.autograd.grad(ref[0].sum() + ref[1].sum() + ref[2].square().sum(), few)
    assert all(torch.equal(o[pick], r) for o, r in zip(out, ref)) and torch.equal(dz[pick], dr)
    for i in range(0, N, 1 << 22):                                                   # gradients of a softmax add up to zero in every row, but for their rounding
        d = dz[i:i + (1 << 22)].float()
        size = d.abs().sum(1)
        assert float((d.sum(1).abs() - 1.01 * B8 * size).max()) <= 1e-3 and float(size.min()) > 0.0


@gpu
@pytest.mark.parametrize("batch,rows,cols,cut", [((1 << 23) + 77, 2, 3, 1 << 23), ((1 << 22) + 5, 1, 257, (1 << 23) // 3)])
def test_orthogonalize_of_more_matrices_than_a_launch_has_blocks(batch, rows, cols, cut):
    """Matrices on both sides of the cut equal those of a small call (in one block a matrix, and in the shared launches, three blocks a matrix)."""
    g = torch.randn(batch, rows, cols, generator=torch.Generator(device="cuda").manual_seed(7), device="cuda", dtype=BF)
    out = K.orthogonalize(g)
    for at in (0, cut - 40, batch - 50):
        assert torch.equal(out[at:at + 50], K.orthogonalize(g[at:at + 50].clone()))
    for i in range(0, batch, 1 << 21):
        assert bool((out[i:i + (1 << 21)].float().abs().amax((1, 2)) > 0.04).all())


@gpu
@pytest.mark.parametrize("steps,coef", [(2, (2.0, -0.5, 0.1)), (3, (1.33, 0.0, 0.0)), (5, (1.5, -0.5, 0.0)), (2, (1.0, 0.25, 0.0))])
def test_orthogonalize_chains_of_polynomials_that_let_singular_values_grow(steps, coef):
    """Steps on the small side, whose factors are multiplied in fp16 at a scale: singular values that start at one and end above two are in range.
    A step's operands are rounded to 2^-22 relative; its factor is below 2.5 and what one step leaves grows by the next ones' slopes, 2.5 at most
    over the whole chain, so 30 2^-22 and the sums as in the other cases, four times."""
    K.check_newton_schulz(steps, coef)
    g = (_randn(61, 1024, 1) @ _randn(62, 1, 4096) + 0.05 * _randn(63, 1024, 4096)).cuda()
    a, b, c = coef
    x = g.double() / (g.double().norm() + 1e-7)
    for _ in range(steps):
        s = x @ x.t().contiguous()
        x = a * x + (b * s + c * s @ s) @ x
    out = K.orthogonalize(g, steps=steps, coefficients=coef).double()
    assert torch.isfinite(out).all()
    assert float((out - x).norm()) <= 4 * (30 * 2.0 ** -22 + 15 * 71 * H24) * float(x.norm())


# ================================================================================================= errors that only a rounding of the result may leave
# Rounding v in [2^e, 2^(e+1)) to bf16 is off by at most 2^(e-8), evenly spread: sqrt(1/3) 2^(e-8) <= 2^-8 |v| / sqrt(3) in the mean square, so the
# norm of n roundings is below 2^-8 / sqrt(3) = 0.00226 of the result's norm, up to about 1 / sqrt(n) of that by chance (three times that is allowed).
def _rounding_alone(out, ref, what, extra):
    ref = ref.to(out.device)
    tol = B8 / math.sqrt(3) * (1 + 3 / math.sqrt(ref.numel())) + extra
    err = float((out.double() - ref).norm() / ref.norm())
    assert err <= tol, (what, err, tol)


@gpu
@pytest.mark.parametrize("shape", [(64, 147), (20, 200), (200, 100), (128, 512), (100, 2000)])
def test_orthogonalize_of_small_bf16_matrices_rounds_its_result_only(shape):
    """Up to 128 rows or columns the products take 22-bit operands: 30 2^-22 and the sums of up to 2000 products, 15 sqrt(2000) 2^-24."""
    g = (_randn(sum(shape), *shape) * 1e-3).to(BF).cuda()
    a, b, c = K.NS_COEFFICIENTS
    x = g.double() / (g.double().norm() + 1e-7)
    for _ in range(5):
        s = x @ x.t().contiguous()
        x = a * x + (b * s + c * s @ s) @ x
    _rounding_alone(K.orthogonalize(g), x, "orthogonalize", 30 * 2.0 ** -22 + 15 * 45 * H24)


@gpu
@pytest.mark.parametrize("T,D,H", [(64, 512, 1032), (16, 1024, 520), (5, 2048, 512)])
def test_gated_mlp_of_few_tokens_rounds_results_only_in_the_mean(T, D, H):
    """h, dg and du as pairs (2^-16 of them is left), factors in 24 bits (2^-17), act' to 1e-5: 1e-4 covers them and the sums."""
    x, dy = _randn(71, T, D).to(BF).cuda(), _randn(72, T, D, scale=0.1).to(BF).cuda()
    w = [_randn(73, H, D, scale=D ** -0.5).to(BF).cuda(), _randn(74, H, D, scale=D ** -0.5).to(BF).cuda(), _randn(75, D, H, scale=H ** -0.5).to(BF).cuda()]
    leaves = [t.requires_grad_() for t in (x, *w)]
    y = F.gated_mlp(*leaves)
    got = (y.detach(), *torch.autograd.grad(y, leaves, dy))
    exact = [t.detach().double().requires_grad_() for t in leaves]
    silu = lambda v: v * torch.sigmoid(v)                                            # noqa: E731
    ye = (silu(exact[0] @ exact[1].t()) * (exact[0] @ exact[2].t())) @ exact[3].t()
    want = (ye.detach(), *torch.autograd.grad(ye, exact, dy.double()))
    for what, o, r in zip(("y", "dx", "dwg", "dwu", "dwd"), got, want):
        if what != "y" or T <= 32:
            _rounding_alone(o, r, what, 1e-4)


@gpu
@pytest.mark.parametrize("T,D,H", [(1, 1, 1), (3, 1, 5), (70, 2, 1), (65, 1, 9), (129, 7, 3), (64, 15, 17)])
def test_gated_mlp_of_tiny_widths_and_expanded_gradients(T, D, H):
    """The smallest widths, from strided operands, with the gradient of a sum (one element, expanded) arriving at the block."""
    x = _randn(81, T, 2 * D + 1)[:, 1:2 * D:2].to(BF)
    w = [_randn(82, H, D).to(BF), _randn(83, D, H).to(BF).t(), _randn(84, D, H).to(BF)]
    net, arena = _arena(*w, device="cuda")
    xs = torch.zeros(T, 2 * D + 1, dtype=BF, device="cuda")
    xs[:, 1:2 * D:2] = x.cuda()
    xs = xs[:, 1:2 * D:2].detach().requires_grad_()
    F.gated_mlp(xs, *net).sum().backward()
    exact = [t.detach().double().clone().requires_grad_() for t in (x, *w)]
    (torch.nn.functional.silu(exact[0] @ exact[1].t()) * (exact[0] @ exact[2].t()) @ exact[3].t()).sum().backward()
    size = [float(t.grad.abs().max()) for t in exact]
    for p, e, s in zip((xs, *net), exact, size):
        # at most three roundings to bf16 (h or dg and du, the result) of terms whose sum of magnitudes is within T + H + D times the largest gradient
        assert float((p.grad.cpu().double() - e.grad).abs().max()) <= 3 * B8 * (T + H + D) * s


@gpu
@pytest.mark.parametrize("T", [1, 9, 32, 50, 64, 65])
def test_gated_mlp_infinite_hidden_values_stay_infinite(T):
    """One hidden value overflows: results are infinities of the right sign whatever the number of tokens, not NaN (the pair of bf16 values that few
    tokens keep must not hold inf - inf)."""
    D, H = 8, 16
    x = torch.ones(T, D, dtype=BF, device="cuda")
    wg, wu = torch.zeros(2, H, D, dtype=BF, device="cuda")
    wg[3], wu[3] = 1e30, 1e30
    sign = torch.tensor([1.0, -1.0] * (D // 2), device="cuda")
    wd = torch.zeros(D, H, dtype=BF, device="cuda")
    wd[:, 3] = sign
    leaves = [t.requires_grad_() for t in (x, wg, wu, wd)]
    y = F.gated_mlp(*leaves)
    assert torch.equal(y, (sign * float("inf")).to(BF).expand(T, D))
    with torch.no_grad():
        assert torch.equal(F.gated_mlp(*leaves), y)
    dy = torch.zeros(T, D, dtype=BF, device="cuda")
    dy[:, 0] = 1e10                                                                  # dg = du = 1e10 * 8e30: infinite
    dx, dwg, dwu, _ = torch.autograd.grad(y, leaves, dy)
    assert bool((dx == float("inf")).all()) and bool((dwg[3] == float("inf")).all()) and bool((dwu[3] == float("inf")).all())
    assert float(dwg[:3].abs().max()) == 0.0


@gpu
def test_token_logprobs_of_sliced_logits_strided_tokens_and_no_rows_with_gradients():
    base = _randn(91, 6, 520).cuda().requires_grad_()
    pairs = torch.randint(0, 500, (6, 2), generator=torch.Generator().manual_seed(92)).cuda()
    g = _randn(93, 6).cuda()
    out = F.token_logprobs(base[:, 3:503], pairs[:, 1], 2)
    (dz,) = torch.autograd.grad([out[0], out[2].sum(1)], base, [g, g])
    z = base.detach()[:, 3:503].clone().requires_grad_()
    ref = F.token_logprobs(z, pairs[:, 1].clone(), 2)
    (dr,) = torch.autograd.grad([ref[0], ref[2].sum(1)], z, [g, g])
    assert all(torch.equal(a, b) for a, b in zip(out, ref)) and torch.equal(dz[:, 3:503], dr) and float(dz[:, :3].abs().sum() + dz[:, 503:].abs().sum()) == 0.0
    turned = _randn(94, 500, 6).cuda().t().requires_grad_()                           # stored column by column
    (dt,) = torch.autograd.grad(F.token_logprobs(turned, pairs[:, 0])[0], turned, g)
    straight = turned.detach().contiguous().requires_grad_()
    assert torch.equal(dt, torch.autograd.grad(F.token_logprobs(straight, pairs[:, 0])[0], straight, g)[0])
    none = torch.zeros(0, 9, device="cuda", requires_grad=True)
    out = F.token_logprobs(none, torch.zeros(0, dtype=torch.int64, device="cuda"), 2)
    assert torch.autograd.grad([out[0].sum() + out[1].sum() + out[2].sum()], none)[0].shape == (0, 9)


@gpu
def test_captured_forward_and_backward_of_block_and_loss_replay():
    """One graph: block, token loss with a list, gradients of everything; replays with eager work between them equal eager runs to the bit."""
    T, D, H, V = 96, 64, 136, 1000
    x = _randn(95, T, D).to(BF).cuda()
    head = _randn(96, V, D, scale=D ** -0.5).to(BF).cuda()
    tok = torch.randint(0, V, (T,), generator=torch.Generator().manual_seed(97)).cuda()
    w = [_randn(98, H, D, scale=D ** -0.5).to(BF).cuda(), _randn(99, H, D, scale=D ** -0.5).to(BF).cuda(), _randn(100, D, H, scale=H ** -0.5).to(BF).cuda()]
    g = torch.full((T,), -1.0 / T, device="cuda")

    def step():
        leaves = [t.detach().requires_grad_() for t in (x, *w)]
        y = F.gated_mlp(*leaves)
        logits = (y.detach().float() @ head.float().t()).requires_grad_()
        out = F.token_logprobs(logits, tok, 3)
        (dz,) = torch.autograd.grad([out[0], out[1], out[2]], logits, [g, 0.01 * g, g[:, None].expand(T, 3)])
        return [*out, dz, *torch.autograd.grad(y, leaves, (dz @ head.float()).to(BF))]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for k in range(4):
        x.copy_(_randn(200 + k, T, D).to(BF))
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), k


# ================================================================================================= data parallel
def _muon_worker(rank, world):
    from distributed_deep_learning_amd.optim import Muon
    from distributed_deep_learning_amd.parallel import DistributedDataParallel
    torch.manual_seed(11 + rank)                                                     # the broadcast makes them equal
    block = dnn.GatedMLP(12, 40)
    ddp = DistributedDataParallel(block, bucket_mb=1e-3)
    opt = Muon(ddp.arena, lr=0.05, weight_decay=0.01)
    start = ddp.arena.master.clone()
    for s in range(3):
        ddp(_randn(10 * s + rank, 6, 12)).pow(2).mean().backward()
        ddp.step(opt)
    return {"start": start, "end": ddp.arena.master.clone(), "buckets": len(ddp.arena.buckets)}


def test_muon_in_data_parallel_equals_one_process_on_the_mean_gradient():
    from _dist_util import run_ranks
    from distributed_deep_learning_amd.optim import Muon
    a, b = run_ranks(_muon_worker, 2)
    assert a["buckets"] > 1 and torch.equal(a["end"], b["end"]) and torch.equal(a["start"], b["start"])
    torch.manual_seed(11)
    block = dnn.GatedMLP(12, 40)
    arena = ParamArena(block.named_parameters(), bucket_bytes=int(1e-3 * 2 ** 20))         # laid out as the reducer lays it out
    opt = Muon(arena, lr=0.05, weight_decay=0.01)
    for s in range(3):
        sum(block(_randn(10 * s + r, 6, 12)).pow(2).mean() for r in range(2)).backward()
        arena.grad.mul_(0.5)
        opt.step()
    for p, s in zip(arena.params, arena.segments):
        # three steps of lr times an orthogonal factor in fp32 (1e-5 of it), from the same start
        assert float((p.detach().reshape(-1) - a["end"][s.offset:s.offset + s.numel]).abs().max()) <= 1e-4


@gpu
def test_shared_gated_weights_under_the_reducer_are_whole_when_their_bucket_goes():
    """Two blocks with the same weights, beside a Linear, with the collectives of one rank: what a bucket holds when its collective is enqueued
    is what it holds at the end of the pass, and every bucket goes inside the pass."""
    import os
    import torch.distributed as td
    from distributed_deep_learning_amd.optim import Muon
    from distributed_deep_learning_amd.parallel import DistributedDataParallel
    from distributed_deep_learning_amd.utils import GradLedger
    dev = torch.device("cuda:0")
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT="29653", HSA_ENABLE_IPC_MODE_LEGACY="0")
    td.init_process_group("nccl", rank=0, world_size=1, device_id=dev)
    try:
        torch.manual_seed(12)

        class Net(tnn.Module):
            def __init__(self):
                super().__init__()
                self.inp, self.ff, self.out = dnn.Linear(64, 128), dnn.GatedMLP(128, 520), dnn.Linear(128, 64)

            def forward(self, x):
                h = self.inp(x)
                h = h + self.ff(h)
                return self.out(h + self.ff(h))

        net = Net().to(dev)
        d = DistributedDataParallel(net, bucket_mb=0.1, force_collectives=True)
        assert len(d.arena.buckets) > 2
        ledger = GradLedger(d, snapshot=True)
        opt = Muon(d.arena, lr=0.01)
        x = _randn(13, 512, 64).to(dev)
        for _ in range(3):
            d(x).float().pow(2).mean().backward()
            assert d._next_bucket == -1
            d.step(opt)
        assert ledger.verified == 3 * len(d.arena.buckets) and not ledger.violations
    finally:
        td.destroy_process_group()


@gpu
def test_captured_data_parallel_step_with_a_gated_block_follows_the_eager_one():
    """Block, Linear and Muon with native collectives (one rank) in one graph: the buckets of the block's weights go from autograd's hooks there too."""
    import os
    import torch.distributed as td
    from distributed_deep_learning_amd.optim import Muon
    from distributed_deep_learning_amd.parallel import DistributedDataParallel
    from distributed_deep_learning_amd.utils import GraphedTrainStep
    dev = torch.device("cuda:0")
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT="29655", HSA_ENABLE_IPC_MODE_LEGACY="0")
    td.init_process_group("nccl", rank=0, world_size=1, device_id=dev)
    try:
        x, y = _randn(14, 256, 64).to(dev), torch.randint(0, 40, (256,), generator=torch.Generator().manual_seed(15)).to(dev)

        def make():
            torch.manual_seed(16)
            net = tnn.Sequential(dnn.Linear(64, 128), dnn.GatedMLP(128, 520), dnn.Linear(128, 40)).to(dev)
            d = DistributedDataParallel(net, bucket_mb=0.1, force_collectives=True, comm="native")
            opt = Muon(d.arena, lr=0.01)
            d.attach(opt)
            return net, d, opt, dnn.SoftmaxCrossEntropyLoss()

        net, d, opt, crit = make()
        for _ in range(6):
            crit(d(x), y).backward()
            d.step(opt)
        net2, d2, opt2, crit2 = make()
        step = GraphedTrainStep(net2, crit2, opt2, x, y, warmup=2, ddp=d2)
        for _ in range(4):
            step(x, y)
        torch.cuda.synchronize()
        a, b = d.arena.master, d2.arena.master
        assert float((a - b).norm()) <= 1e-3 * float(a.norm())                       # sums of the Linear layers may differ in order
    finally:
        td.destroy_process_group()
