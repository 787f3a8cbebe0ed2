"""GroupNorm (+ ReLU) whose backward pass works on an 8-bit copy of its input, against the definition in 64 bits."""
import pytest
import torch

from scaffold_b200.ops import gn_kernels as gk
from scaffold_b200.ops._lib import NativeError
from scaffold_b200.ops.group_norm import GroupNorm, group_norm_kept8
from scaffold_b200.ops.kept8 import Kept8, block_steps, restore8


def _inputs(shape, seed, dev="cuda"):
    g = torch.Generator(device=dev).manual_seed(seed)
    n, d, h, w, c = shape
    r = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    x = (r(n, d, h, w, c) * (0.3 + torch.rand(c, generator=g, device=dev)) + 0.5 * r(c)).to(torch.bfloat16)
    gy = r(n, d, h, w, c).to(torch.bfloat16)
    return x, gy, 1 + 0.3 * r(c), 0.3 * r(c)


def _vm(kept, like):
    return restore8(Kept8(kept, tuple(like.shape), like.stride(), torch.bfloat16))


def _reference(x, xk, gy, w, b, groups, eps, relu):
    """(y, dx, dw, db) in 64 bits: y of x, the gradients at the kept values xk with the statistics and the mask of x."""
    n, c = x.shape[0], x.shape[-1]
    x, xk, gy = (t.double().reshape(n, -1, c) for t in (x, xk, gy))
    w, b = w.double(), b.double()
    grp = lambda t: t.reshape(n, -1, groups, c // groups)  # noqa: E731
    up = lambda t: t.reshape(n, 1, groups, 1).expand(n, 1, groups, c // groups).reshape(n, 1, c)  # noqa: E731
    mean, var = up(grp(x).mean((1, 3))), up(grp(x).var((1, 3), unbiased=False))
    rstd = (var + eps) ** -0.5
    pre = (x - mean) * rstd * w + b
    if relu:
        gy = gy * (pre > 0)
    xhat = (xk - mean) * rstd
    dw, db = (gy * xhat).sum((0, 1)), gy.sum((0, 1))
    c1, c2 = up(grp(gy * w).mean((1, 3))), up(grp(gy * w * xhat).mean((1, 3)))
    return pre.clamp_min(0) if relu else pre, rstd * (gy * w - c1 - xhat * c2), dw, db, pre


SHAPES = [((1, 1, 1, 1, 16), 1), ((2, 1, 1, 1, 16), 2), ((1, 3, 5, 7, 16), 8), ((2, 3, 5, 7, 32), 8),
          ((3, 4, 4, 5, 48), 3), ((1, 5, 9, 11, 80), 10), ((2, 8, 8, 8, 512), 8), ((1, 2, 3, 4, 2048), 16),
          ((2, 16, 17, 19, 64), 8), ((5, 2, 2, 2, 64), 32)]


@pytest.mark.gpu
@pytest.mark.parametrize("relu", [True, False])
@pytest.mark.parametrize("shape,groups", SHAPES, ids=str)
def test_forward_and_gradients(shape, groups, relu):
    x, gy, w, b = _inputs(shape, sum(shape))
    eps = 1e-5
    y, kept, stats = gk.gn8_forward(x, w, b, groups, eps, relu)
    mean, rstd = stats
    ordinary = gk.gn_forward(x, w, b, groups, eps, relu)
    # statistics and result: those of the ordinary kernels, to the bit
    assert torch.equal(y, ordinary[0]) and torch.equal(mean, ordinary[1]) and torch.equal(rstd, ordinary[2])
    xk = _vm(kept, x)
    ry, rdx, rdw, rdb, pre = _reference(x, xk, gy, w, b, groups, eps, relu)
    # the copy: nearest whole number of steps, or the next one on the value's own side of the ReLU
    _, step, cap = block_steps(x.float().reshape(-1, 16).cpu(), torch.bfloat16)
    off = ((xk - x.float()).abs().reshape(-1, 16).cpu() / step[:, None])
    assert (off <= (1.0 if relu else 0.5)).all()
    if relu:
        a = rstd.repeat_interleave(shape[-1] // groups, 1).view(shape[0], 1, 1, 1, -1) * w
        shift = b - mean.repeat_interleave(shape[-1] // groups, 1).view(shape[0], 1, 1, 1, -1) * a
        side = lambda t: torch.addcmul(shift.double(), t.double(), a.double()) > 0  # noqa: E731
        near = (pre.abs() < 1e-5).view(x.shape)  # where fp32 and 64 bits may see another sign
        assert (side(xk) == side(x))[~near].all()
    # bf16 result: half a step, 2^-8 of the value, with the fp32 error of statistics and affine (a few 2^-24 of values below 50)
    assert ((y.double().reshape(ry.shape) - ry).abs() <= 2 ** -8 * ry.abs() + 1e-4 * (rstd.max() + 1)).all()
    dx, dw, db = gk.gn8_backward(gy, kept, w, b, stats, groups, relu)
    # dx: half a step of bf16 (2^-8 of the value), and terms of the size of rstd * max|gy w| in fp32 with the errors of
    # mean and rstd (fp32 sums in a tree: 1e-5 of the terms is far above them); a value nearer to the ReLU's border
    # than fp32 resolves may take the other mask
    size = float(rdx.abs().max() + (rstd.max() * (gy.abs().max() * w.abs().max())))
    bad = (dx.double().reshape(rdx.shape) - rdx).abs() > 2 ** -8 * rdx.abs() + 2e-5 * size
    assert not (bad & ~(pre.abs() < 1e-5)).any()
    # sums over up to 10^4 values: per-thread chains of at most some hundred additions, 1e-5 of the sum of magnitudes
    mag = gy.double().abs().sum((0, 1, 2, 3))
    assert ((db.double() - rdb).abs() <= 1e-5 * mag + 1e-30).all()
    assert ((dw.double() - rdw).abs() <= 2e-5 * mag * (1 + float((xk.float().abs().max() + mean.abs().max()) * rstd.max()))).all()


@pytest.mark.gpu
def test_the_gradient_is_that_of_the_function_to_the_step_of_the_copy():
    """Against differences of the loss along random directions (64 bits): dx follows the formula at x itself up to the
    copy's step, 1/126 of a block's largest value."""
    shape, groups = (2, 4, 6, 5, 32), 8
    x, gy, w, b = _inputs(shape, 3)
    y, kept, stats = gk.gn8_forward(x, w, b, groups, 1e-5, False)
    dx, dw, db = gk.gn8_backward(gy, kept, w, b, stats, groups, False)

    def loss(xx, ww, bb):
        n, c = shape[0], shape[-1]
        t = xx.reshape(n, -1, groups, c // groups)
        t = (t - t.mean((1, 3), keepdim=True)) / (t.var((1, 3), unbiased=False, keepdim=True) + 1e-5).sqrt()
        return ((t.reshape(n, -1, c) * ww + bb) * gy.double().reshape(n, -1, c)).sum()

    g = torch.Generator(device="cuda").manual_seed(9)
    for grad, at in ((dx, 0), (dw, 1), (db, 2)):
        args = [x.double(), w.double(), b.double()]
        v = torch.randn(args[at].shape, generator=g, device="cuda", dtype=torch.float64)
        h = 1e-5
        hi, lo = list(args), list(args)
        hi[at], lo[at] = args[at] + h * v, args[at] - h * v
        slope = (loss(*hi) - loss(*lo)) / (2 * h)
        got = (grad.double() * v).sum()
        assert abs(got - slope) <= 0.02 * grad.double().norm() * 3  # steps and bf16 roundings are random along v


@pytest.mark.gpu
def test_statistics_of_nothing_but_equal_values_and_values_that_are_not_finite():
    shape = (2, 2, 4, 4, 32)
    x, gy, w, b = _inputs(shape, 1)
    x[0] = 1.5
    y, kept, stats = gk.gn8_forward(x, w, b, 8, 1e-5, True)
    assert torch.equal(y, gk.gn_forward(x, w, b, 8, 1e-5, True)[0])
    dx, dw, db = gk.gn8_backward(gy, kept, w, b, stats, 8, True)
    assert dx.isfinite().all() and dw.isfinite().all() and db.isfinite().all()
    x[1, 0, 0, 0, 5] = float("inf")  # group 1 of sample 1
    y, kept, stats = gk.gn8_forward(x, w, b, 8, 1e-5, True)
    want = gk.gn_forward(x, w, b, 8, 1e-5, True)
    assert torch.equal(y.nan_to_num(), want[0].nan_to_num()) and torch.equal(y.isnan(), want[0].isnan())
    dx, *_ = gk.gn8_backward(gy, kept, w, b, stats, 8, True)
    assert dx[1, ..., 4:8].isnan().all()
    # the block of 16 channels around the infinity is NaN, the rest of the sample and the other sample are not
    assert dx[0].isfinite().all() and dx[1, ..., 16:].isfinite().all()


@pytest.mark.gpu
def test_module_and_function_agree_and_direct_gradients_are_added():
    x, gy, w, b = _inputs((2, 4, 5, 6, 64), 4)
    x, gy = (t.permute(0, 4, 1, 2, 3) for t in (x, gy))
    m = GroupNorm(8, 64, activation="relu").cuda()
    with torch.no_grad():
        m.weight.copy_(w)
        m.bias.copy_(b)
    m.keep_bits = 8
    a = x.clone(memory_format=torch.preserve_format).requires_grad_()
    c = x.clone(memory_format=torch.preserve_format).requires_grad_()
    y = m(a)
    y.backward(gy)
    wf, bf = w.clone().requires_grad_(), b.clone().requires_grad_()
    z = group_norm_kept8(c, 8, wf, bf, activation="relu")
    z.backward(gy)
    assert torch.equal(y, z) and torch.equal(a.grad, c.grad)
    assert torch.equal(m.weight.grad, wf.grad) and torch.equal(m.bias.grad, bf.grad)
    assert y.stride() == x.stride() and a.grad.stride() == x.stride()
    m.keep_bits = 16
    with torch.no_grad():
        assert torch.equal(m(x), y)  # without a backward pass to come, and ordinary: the same result
    # twice: gradients accumulate
    group_norm_kept8(c, 8, wf, bf, activation="relu").backward(gy)
    assert torch.equal(wf.grad, 2 * m.weight.grad)


@pytest.mark.gpu
def test_less_memory_is_kept():
    x, gy, w, b = _inputs((1, 16, 32, 32, 64), 5)
    x = x.permute(0, 4, 1, 2, 3)
    # bytes that the graph holds on to (not the allocator's figure: it does not split a block for less than 1 MiB)
    saved = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: (saved.append(t.numel() * t.element_size()), t)[1], lambda t: t):
        group_norm_kept8(x, 8, w.requires_grad_(), b)
    assert sum(saved) <= 1.0625 * x.numel() + 4 * (2 * 64 + 2 * 8)


@pytest.mark.gpu
def test_a_captured_pass_is_replayed_on_new_values():
    x, gy, w, b = _inputs((2, 4, 5, 6, 32), 6)
    xs, gs = (t.permute(0, 4, 1, 2, 3) for t in (x, gy))
    leaf = xs.detach().requires_grad_()
    wf, bf = w.requires_grad_(), b.requires_grad_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(group_norm_kept8(leaf, 8, wf, bf, activation="relu"), (leaf, wf, bf), gs)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = group_norm_kept8(leaf, 8, wf, bf, activation="relu")
        grads = torch.autograd.grad(y, (leaf, wf, bf), gs)
    for seed in (7, 8):
        nx, ng, _, _ = _inputs((2, 4, 5, 6, 32), seed)
        with torch.no_grad():
            x.copy_(nx)
            gy.copy_(ng)
        graph.replay()
        ey, kept, stats = gk.gn8_forward(nx, w.detach(), b.detach(), 8, 1e-5, True)
        want = gk.gn8_backward(ng, kept, w.detach(), b.detach(), stats, 8, True)
        assert torch.equal(y.permute(0, 2, 3, 4, 1), ey) and torch.equal(grads[0].permute(0, 2, 3, 4, 1), want[0])
        assert torch.equal(grads[1], want[1]) and torch.equal(grads[2], want[2])


@pytest.mark.gpu
def test_inputs_and_gradients_may_start_anywhere():
    x, gy, w, b = _inputs((2, 3, 4, 5, 32), 11)

    def off(t, by):
        buf = torch.empty(t.numel() + by, dtype=t.dtype, device="cuda")
        return buf[by:].view(t.shape).copy_(t).permute(0, 4, 1, 2, 3)

    results = []
    for by in (0, 1, 4):
        leaf = off(x, by).requires_grad_()
        y = group_norm_kept8(leaf, 8, w, b, activation="relu")
        # (a gradient that is a piece of a larger one: what a concatenation hands back)
        (dx,) = torch.autograd.grad(y, leaf, off(gy, by))
        flat = torch.cat([w.new_zeros(by, dtype=torch.bfloat16), group_norm_kept8(leaf, 8, w, b, activation="relu")
                          .permute(0, 2, 3, 4, 1).reshape(-1)])
        (dz,) = torch.autograd.grad(flat, leaf, torch.cat([flat.new_zeros(by), gy.reshape(-1)]))
        results.append((y.detach(), dx, dz))
    for other in results[1:]:
        assert all(torch.equal(p, q) for p, q in zip(results[0], other))
    assert torch.equal(results[0][1], results[0][2])


def test_refusals():
    w, b = torch.ones(32), torch.zeros(32)
    x = torch.zeros(1, 32, 2, 2, 2, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        group_norm_kept8(x, 8, w, b)
    with pytest.raises(ValueError, match="activation"):
        group_norm_kept8(x, 8, w, b, activation="gelu")
    assert not gk.supported_kept8(24, 3) and not gk.supported_kept8(16, 16) and gk.supported_kept8(48, 6)


@pytest.mark.gpu
def test_refusals_on_the_device():
    w, b = torch.ones(32, device="cuda"), torch.zeros(32, device="cuda")
    x = torch.zeros(1, 32, 2, 2, 2, dtype=torch.bfloat16, device="cuda")
    for args in ((x.float(), 8, w, b), (x[0], 8, w, b), (x, 7, w, b), (x, 8, w[:16], b), (x, 8, w.cpu(), b),
                 (x[:, :24], 3, w[:24], b[:24]), (x[:0], 8, w, b)):
        with pytest.raises(ValueError):
            group_norm_kept8(*args)


def test_the_scratch_of_sizes_outside_the_range():
    for n, s in ((65536, 1), (0, 8), (1, 0)):
        with pytest.raises(NativeError, match="samples"):
            gk._scratch8(0, n, s, 16, 1)


@pytest.mark.gpu
def test_more_samples_than_a_grid_has():
    w, b = torch.ones(16, device="cuda"), torch.zeros(16, device="cuda")
    x = torch.zeros(65536, 16, 1, 1, 1, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="65535"):
        group_norm_kept8(x, 1, w, b)
    assert group_norm_kept8(x[:65535], 1, w, b).shape == x[:65535].shape
