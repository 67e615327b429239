"""Cross entropy of a linear head without its logits: the piecewise reference (CPU) and the tensor-core kernels (GPU) against the
definition in 64 bits, gradients against differences, refusals, the model path, strides, streams and captured graphs."""
import math

import pytest
import torch

from nanotron_b200 import ops
from nanotron_b200.ops import native_ce
from nanotron_b200.ops import reference as ref
from nanotron_b200.parallel.tensor_parallel.functional import linear_cross_entropy, linear_cross_entropy_with_z_loss, sharded_cross_entropy

gpu = pytest.mark.gpu
DEV = "cuda"


def definition(x, w, y, g, gz=None, z=0.0):
    """loss, z term, d, dx, dw in 64 bits; targets outside the vocabulary are a class of score 0."""
    x, w, g = x.double(), w.double(), g.double()
    scores = x @ w.t()
    logz = torch.logsumexp(scores, -1)
    inside = (y >= 0) & (y < w.shape[0])
    picked = torch.where(inside, scores.gather(1, y.clamp(0, w.shape[0] - 1)[:, None])[:, 0], torch.zeros_like(logz))
    coef = g + (2 * z * logz * gz.double() if gz is not None else 0)
    p = torch.exp(scores - logz[:, None]) * coef[:, None]
    d = p.clone()
    d[torch.arange(len(y))[inside.cpu()], y[inside]] -= g[inside]
    return logz - picked, z * logz**2, p, d, d @ w, d.t() @ x


def inputs(T, H, V, device, dtype, seed=0, spread=1.5):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(T, H, generator=gen).to(device, dtype)
    w = (torch.randn(V, H, generator=gen) * spread / math.sqrt(H)).to(device, dtype)
    y = torch.randint(0, V, (T,), generator=gen).to(device)
    g = torch.rand(T, generator=gen).to(device)
    g[T // 2] = 0  # a masked token
    return x, w, y, g


# ------------------------------------------------------------------------------------------------ CPU
@pytest.mark.parametrize("T,H,V,piece", [(1, 3, 1, 4), (7, 16, 50, 8), (5, 8, 33, 33), (4, 5, 20, 7)])
def test_reference_pieces_match_the_definition(T, H, V, piece):
    x, w, y, g = inputs(T, H, V, "cpu", torch.float64)
    loss, _, _, _, dx, dw = definition(x, w, y, g)
    m, s, t = ref.linear_ce_partials(x, w, y, 0, piece=piece)
    logz = m + s.log()
    torch.testing.assert_close(logz - t, loss, rtol=1e-12, atol=1e-12)
    dx2, dw2 = ref.linear_ce_backward(x, w, y, logz, g, None, 0.0, 0, piece=piece)
    torch.testing.assert_close(dx2, dx, rtol=1e-12, atol=1e-12)
    torch.testing.assert_close(dw2, dw, rtol=1e-12, atol=1e-12)


def test_gradients_against_differences():
    x, w, y, _ = inputs(4, 6, 11, "cpu", torch.float64)
    y[1], y[2] = -100, 11  # outside: a class of score 0 without gradient
    x.requires_grad_(), w.requires_grad_()

    def f(x, w):
        loss, z = linear_cross_entropy_with_z_loss(x.view(2, 2, 6), w, y.view(2, 2), z_loss_coef=0.3)
        return loss, z

    assert torch.autograd.gradcheck(f, (x, w), eps=1e-6, atol=1e-8, rtol=1e-6)


def test_same_as_logits_and_sharded_cross_entropy():
    x, w, y, g = inputs(9, 32, 70, "cpu", torch.float32)
    a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
    c, d = x.clone().requires_grad_(), w.clone().requires_grad_()
    l1, l2 = linear_cross_entropy(a, b, y.int()), sharded_cross_entropy(c @ d.t(), y, group=None)
    torch.testing.assert_close(l1, l2, rtol=1e-5, atol=1e-5)
    (l1 * g).sum().backward(), (l2 * g).sum().backward()
    torch.testing.assert_close(a.grad, c.grad, rtol=1e-4, atol=1e-6)
    torch.testing.assert_close(b.grad, d.grad, rtol=1e-4, atol=1e-6)


def test_no_tokens_frozen_operands_and_main_grad():
    x, w, y, g = inputs(6, 8, 20, "cpu", torch.float32)
    e, v = x[:0].clone().requires_grad_(), w.clone().requires_grad_()
    loss = linear_cross_entropy(e, v, y[:0])
    loss.sum().backward()
    assert loss.shape == (0,) and e.grad.shape == (0, 8) and not v.grad.any()
    a = x.clone().requires_grad_()
    (linear_cross_entropy(a, w, y) * g).sum().backward()  # frozen head
    v = w.clone().requires_grad_()
    (linear_cross_entropy(x, v, y) * g).sum().backward()  # frozen body
    p = torch.nn.Parameter(w.clone())
    p.main_grad = torch.ones_like(w)
    (linear_cross_entropy(x, p, y) * g).sum().backward()
    assert p.grad is None
    torch.testing.assert_close(p.main_grad, 1 + v.grad)
    with torch.no_grad():
        assert not linear_cross_entropy(a, p, y).requires_grad
    loss, z = linear_cross_entropy_with_z_loss(x, w, y, z_loss_coef=0.0)
    assert z is None and loss.shape == (6,)


def test_one_token_and_leading_dimensions():
    x, w, y, _ = inputs(6, 8, 20, "cpu", torch.float32)
    want = linear_cross_entropy(x, w, y)
    assert torch.equal(linear_cross_entropy(x.view(2, 3, 8), w, y.view(2, 3)), want.view(2, 3))
    one = x[4].clone().requires_grad_()
    loss = linear_cross_entropy(one, w, y[4])
    loss.backward()
    assert loss.shape == () and one.grad.shape == (8,)
    torch.testing.assert_close(loss, want[4])


def test_refusals():
    x, w, y, _ = inputs(6, 8, 20, "cpu", torch.float32)
    for bad in [(x[:, :7], w, y), (x, w[0], y), (x, w.double(), y), (x, w, y[:5]), (x, w, y.float()), (x, w[:0], y), (x.long(), w.long(), y)]:
        with pytest.raises(ValueError):
            linear_cross_entropy(*bad)
    with pytest.raises(ValueError):
        linear_cross_entropy_with_z_loss(x, w, y, z_loss_coef=-1.0)
    a = x.clone().requires_grad_()
    (dx,) = torch.autograd.grad(linear_cross_entropy(a, w, y).sum(), a, create_graph=True)
    with pytest.raises(RuntimeError):  # one level of differentiation
        dx.sum().backward()
    # what the kernels refuse is decided on the host
    bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)  # noqa: E731
    native_ce.check_operands(bf(3, 64), bf(5, 64), y)
    for bad in [(bf(3, 96), bf(5, 96)), (bf(3, 64).float(), bf(5, 64)), (bf(3, 64), bf(5, 64).half()), (bf(3, 0), bf(5, 0)), (bf(3, 64), bf(5, 64).to("meta"))]:
        with pytest.raises(ValueError):
            native_ce.check_operands(*bad, y)


@pytest.mark.parametrize("T,V", [(1, 1), (1, 128256), (333, 50257), (8192, 128256), (16384, 151936), (1 << 20, 128256), (40000, 4097)])
def test_pieces_cover_the_vocabulary_and_stay_in_their_budget(T, V):
    width = native_ce.piece_width(T, V)
    assert width % 256 == 0 and width > 0
    n = -(-V // width)
    assert width * (n - 1) < V <= width * n
    assert min(width, V) * T <= max(native_ce.PIECE_ELEMENTS, native_ce.PIECE_MIN * T) + 256 * T


def test_rows_are_read_in_place_or_copied():
    t = torch.zeros(8, 128, dtype=torch.bfloat16)
    assert native_ce._rows(t) is t
    assert native_ce._rows(t[:, :64]).data_ptr() == t.data_ptr()
    odd = torch.zeros(8 * 128 + 1, dtype=torch.bfloat16)[1:].view(8, 128)  # contiguous, but off by one element
    for bad in (t[:, 1:65], t.t(), t[:1].expand(8, 128), odd):
        assert native_ce._rows(bad).is_contiguous() and native_ce._rows(bad).data_ptr() % 16 == 0 and native_ce._rows(bad).data_ptr() != bad.data_ptr()


# ------------------------------------------------------------------------------------------------ GPU
def bounds(x, w, p, d, dx, dw, loss):
    """Error bounds of the kernels (elementwise), in 64 bits.
    * a score: bf16 products are exact in fp32; the sum of H of them is off by at most 2^-23 of sum |x||w| per accumulation step
      (H / 16 steps, one more for the alignment inside a step);
    * exp / log of the statistics: a few fp32 units, 2^-20 in all;
    * d: the scores' errors times p, and one rounding to bf16 (2^-8 of |d|); the products of d with bf16 operands sum those, plus the
      accumulation error of their own length; the result is rounded once more (2^-8)."""
    xa, wa = x.double().abs(), w.double().abs()
    H, (T, V) = x.shape[1], d.shape
    ds = (xa @ wa.t()).amax(dim=1) * (H / 16 + 2) * 2.0**-23 + 2.0**-20  # one per token
    e = 2 * ds[:, None] * p.abs() + 2.0**-8 * d.abs() + 2.0**-20 * d.abs()
    acc = lambda k: (k / 16 + 2) * 2.0**-23  # noqa: E731
    bx = (e + d.abs() * acc(V)) @ wa + 2.0**-8 * dx.abs() + 1e-30
    bw = (e + d.abs() * acc(T)).t() @ xa + 2.0**-8 * dw.abs() + 1e-30
    return 2 * ds + 2.0**-20 * loss.abs(), bx, bw


def within(got, want, bound, what):
    off = (got.double() - want).abs()
    assert torch.isfinite(got).all(), what
    worst = (off / bound).max().item() if off.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst:.3g} of the bound"


def check(x, w, y, g, z=0.0, main_grad=None):
    a, b = x.detach().requires_grad_(), (torch.nn.Parameter(w) if main_grad is not None else w.detach().requires_grad_())
    gz = 0.5 * g.flip(0) if z else None
    loss64, z64, p, d, dx, dw = definition(x, w, y, g, gz, z)
    bl, bx, bw = bounds(x, w, p, d, dx, dw, loss64)
    if main_grad is not None:
        b.main_grad = main_grad.clone()
    loss, zt = linear_cross_entropy_with_z_loss(a, b, y, z_loss_coef=z)
    within(loss, loss64, bl, "loss")
    if z:
        within(zt, z64, 2 * z * (loss64.abs() + 100) * bl + 2.0**-20 * z64, "z")
    torch.autograd.backward((loss,) + ((zt,) if z else ()), (g,) + ((gz,) if z else ()))
    within(a.grad, dx, bx, "dx")
    if main_grad is not None:
        assert b.grad is None
        within(b.main_grad, dw + main_grad.double(), bw + 2.0**-22 * (dw.abs() + main_grad.abs()), "main_grad")
    else:
        within(b.grad, dw, bw, "dw")


SHAPES = [(1, 64, 1), (1, 64, 257), (3, 128, 255), (2, 192, 64), (257, 64, 1000), (128, 448, 4096), (130, 4096, 513), (515, 576, 9001), (64, 1024, 20011), (2049, 128, 777), (300, 1088, 1000), (257, 4096, 700), (40, 2112, 3000)]
# up to 8 tokens take their own kernel: odd block counts, last rows, and the sizes just past it
SHAPES += [(1, 2048, 5003), (8, 8192, 300), (9, 4096, 1000), (16, 4160, 129), (17, 64, 16), (31, 576, 2400), (32, 2048, 4111), (33, 64, 100), (7, 64, 40000), (1, 8256, 33)]
# GEMM kernel with operands of fewer rows than a load takes otherwise
SHAPES += [(24, 4096, 600), (113, 320, 1500), (121, 1152, 260), (127, 64, 70000), (129, 1088, 300)]
# the product turned around: its tile widths, several token tiles, fewer vocabulary tiles than CTA pairs, and the sizes past it
SHAPES += [(60, 64, 1), (65, 2048, 9000), (192, 128, 70000), (200, 64, 70), (255, 1088, 300), (333, 256, 5000), (450, 2048, 129), (520, 192, 3001), (1000, 2112, 1300), (1024, 2048, 257), (1025, 2048, 257)]


@gpu
@pytest.mark.parametrize("T,H,V", SHAPES)
@pytest.mark.parametrize("z", [0.0, 1e-2])
def test_kernels_match_the_definition(T, H, V, z):
    check(*inputs(T, H, V, DEV, torch.bfloat16), z=z)


@gpu
@pytest.mark.parametrize("T", [3, 40, 100, 130, 300, 1100])
def test_masked_vocabulary_and_tokens_that_are_not_finite(T):
    """Rows of the weight whose scores are -inf or the lowest numbers take no part; a token that is not finite spoils its own loss alone."""
    x, w, y, _ = inputs(T, 128, 700, DEV, torch.bfloat16, seed=5)
    x = x.abs() + 0.25  # positive: a weight row of -inf scores -inf, without 0 * inf
    w[17], w[600] = float("-inf"), -1e36
    y[(y == 17) | (y == 600)] = 5
    bad = [1, T - 1]
    x[1, 7], x[T - 1, 100] = float("nan"), float("inf")
    loss = linear_cross_entropy(x, w, y)
    assert loss[bad].isnan().all()
    good = [t for t in range(T) if t not in bad]
    scores = x[good].double() @ w.double().t()
    want = torch.logsumexp(scores, 1) - scores.gather(1, y[good][:, None])[:, 0]
    kept = [v for v in range(700) if v not in (17, 600)]
    ds = (x[good].double() @ w[kept].double().abs().t()).amax(dim=1) * (128 / 16 + 2) * 2.0**-23 + 2.0**-20
    within(loss[good], want, 2 * ds + 2.0**-20 * want.abs(), "loss")


@gpu
@pytest.mark.parametrize("T,H,V", [(300, 128, 5000), (513, 320, 2817), (20, 64, 1300)])
def test_several_pieces(T, H, V, monkeypatch):
    monkeypatch.setattr(native_ce, "PIECE_MIN", 256)
    monkeypatch.setattr(native_ce, "PIECE_ELEMENTS", 1)
    x, w, y, g = inputs(T, H, V, DEV, torch.bfloat16, seed=3)
    assert native_ce.piece_width(T, V) == 256
    check(x, w, y, g, z=1e-3)
    check(x, w, y, g, main_grad=torch.randn(V, H, device=DEV))


@gpu
def test_main_grad_takes_the_gradient_in_one_piece():
    x, w, y, g = inputs(200, 128, 999, DEV, torch.bfloat16)
    check(x, w, y, g, main_grad=torch.randn(999, 128, device=DEV))


@gpu
@pytest.mark.parametrize("T", [5, 300])
def test_frozen_operands_get_no_gradient_and_cost_none(T):
    x, w, y, g = inputs(T, 128, 999, DEV, torch.bfloat16)
    _, _, p, d, dx, dw = definition(x, w, y, g)
    bl, bx, bw = bounds(x, w, p, d, dx, dw, torch.zeros(T, device=DEV))
    a = x.detach().requires_grad_()
    (linear_cross_entropy(a, w, y) * g).sum().backward()
    within(a.grad, dx, bx, "dx")
    b = w.detach().requires_grad_()
    n0 = ops.native_launches()
    (linear_cross_entropy(x, b, y) * g).sum().backward()
    assert ops.native_launches() - n0 == 2 + 3  # statistics, join; coefficients, gradient of the scores, dw
    within(b.grad, dw, bw, "dw")


@gpu
def test_peaked_and_masked_rows():
    """Certain tokens (one score far above the rest), targets outside the vocabulary, masked rows, all rows masked, tiny upstream."""
    x, w, y, g = inputs(70, 64, 600, DEV, torch.bfloat16, spread=1.0)
    x[:8] = (w[y[:8]].float() * 40).to(torch.bfloat16)
    y[3], y[9], y[10] = -100, 600, 1 << 40
    check(x, w, y, g)
    check(x, w, y, torch.zeros_like(g))
    check(x, w, y, g * 2.0**-60)


@gpu
def test_strided_hidden_states_and_broadcast_upstream():
    x, w, y, _ = inputs(64, 128, 300, DEV, torch.bfloat16)
    wide = torch.zeros(64, 3 * 128, dtype=torch.bfloat16, device=DEV)
    wide[:, 128:256] = x
    odd = torch.zeros(64 * 128 + 1, dtype=torch.bfloat16, device=DEV)
    odd[1:] = x.flatten()
    want = None
    for view in (x, wide[:, 128:256], x.t().contiguous().t(), odd[1:].view(64, 128)):
        a, b = view.detach().requires_grad_(), w.detach().requires_grad_()
        loss = linear_cross_entropy(a.view(64, 128) if view.is_contiguous() else a, b, y)
        loss.mean().backward()  # the upstream gradient is one number, expanded
        got = (loss.detach(), a.grad, b.grad)
        want = want or got
        assert all(torch.equal(p, q) for p, q in zip(got, want))


@gpu
def test_repeats_are_bit_equal_and_streams_are_followed():
    x, w, y, g = inputs(700, 256, 6000, DEV, torch.bfloat16)
    def step():
        a, b = x.detach().requires_grad_(), w.detach().requires_grad_()
        loss = linear_cross_entropy(a, b, y)
        return (loss.detach(),) + torch.autograd.grad(loss, (a, b), g)
    first = step()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s1):
        one = step()
    with torch.cuda.stream(s2):
        two = step()
    torch.cuda.synchronize()
    for other in (one, two):
        assert all(torch.equal(p, q) for p, q in zip(first, other))


@gpu
def test_captured_step_replays_on_new_inputs():
    x, w, y, g = inputs(130, 128, 700, DEV, torch.bfloat16)
    linear_cross_entropy(x, w, y)  # first call outside the capture
    torch.cuda.synchronize()

    def step(x, w, y):
        a, b = x.detach().requires_grad_(), w.detach().requires_grad_()
        loss = linear_cross_entropy(a, b, y)
        return (loss.detach(),) + torch.autograd.grad(loss, (a, b), g)

    graphs = []
    for _ in range(2):  # two graphs of the same call share no scratch that is alive between their launches
        sx, sw, sy = x.clone(), w.clone(), y.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(sx, sw, sy)
        graphs.append((graph, sx, sw, sy, out))
    x2, w2, y2, _ = inputs(130, 128, 700, DEV, torch.bfloat16, seed=9)
    for graph, sx, sw, sy, _ in graphs:
        sx.copy_(x2), sw.copy_(w2), sy.copy_(y2)
    for graph, *_ in graphs:
        graph.replay()
    want = step(x2, w2, y2)
    torch.cuda.synchronize()
    for *_, out in graphs:
        assert all(torch.equal(p, q) for p, q in zip(out, want))


@gpu
def test_backward_can_be_repeated():
    x, w, y, g = inputs(70, 128, 900, DEV, torch.bfloat16)
    a, b = x.requires_grad_(), w.requires_grad_()
    loss, z = linear_cross_entropy_with_z_loss(a, b, y, z_loss_coef=1e-3)
    first = torch.autograd.grad((loss, z), (a, b), (g, g), retain_graph=True)
    second = torch.autograd.grad((loss, z), (a, b), (g, g))
    assert all(torch.equal(p, q) for p, q in zip(first, second))
    only_z = torch.autograd.grad(linear_cross_entropy_with_z_loss(a, b, y, z_loss_coef=1e-3)[1], a, g)  # the loss itself unused
    assert only_z[0].isfinite().all()


FRESH = """
import sys
sys.path[:0] = [{root!r}, {root!r} + "/tests"]
import torch
from nanotron_b200.parallel.tensor_parallel.functional import linear_cross_entropy
from test_linear_cross_entropy import inputs
x, w, y, g = inputs(20, 64, 300, "cuda", torch.bfloat16)
linear_cross_entropy(x, w, y)
torch.cuda.synchronize()
def step():
    a, b = x.detach().requires_grad_(), w.detach().requires_grad_()
    loss = linear_cross_entropy(a, b, y)
    return (loss.detach(),) + torch.autograd.grad(loss, (a, b), g)
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = step()
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(p, q) for p, q in zip(out, step()))
print("captured")
"""


@gpu
def test_first_backward_of_a_process_inside_a_capture():
    """The autograd thread meets the library for the first time while the stream is being captured."""
    import os
    import subprocess
    import sys

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", FRESH.format(root=root)], capture_output=True, text=True, timeout=200)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


@gpu
def test_first_call_inside_a_capture_is_refused():
    from nanotron_b200.ops import native, native_gemm

    x, w, y, _ = inputs(20, 64, 300, DEV, torch.bfloat16)
    linear_cross_entropy(x, w, y)
    known = native_gemm._STATUS.pop(str(x.device))
    try:
        with pytest.raises(native.NativeKernelError, match="captured"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                linear_cross_entropy(x, w, y)
    finally:
        native_gemm._STATUS[str(x.device)] = known
    torch.cuda.synchronize()
    linear_cross_entropy(x, w, y)


@gpu
def test_gpu_refusals():
    x, w, y, _ = inputs(8, 64, 100, DEV, torch.bfloat16)
    for bad in [(x.float(), w.float(), y), (x.half(), w.half(), y), (x[:, :32], w[:, :32], y), (x, w.cpu(), y), (x, w, y.cpu())]:
        with pytest.raises(ValueError):
            linear_cross_entropy(*bad)
    with ops.mode("torch"):  # the oracle takes any type and size
        linear_cross_entropy(x[:, :32].float(), w[:, :32].float(), y)
