"""The cross entropy of a head with many classes, taken from its features: against the definition in 64 bits."""
import math
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from scaffold_b200.ops import _lib
from scaffold_b200.ops import head_loss as H
from scaffold_b200.ops.head_loss import head_cross_entropy

IGNORED = -1


def _inputs(v, c, k, seed=0, ignored=0.0, weighted=False, bias=True, w_type=torch.bfloat16, dev="cuda", scale=2.8):
    g = torch.Generator(device=dev).manual_seed(seed + 1000 * v + k)
    r = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    x = torch.relu(r(v, c)).to(torch.bfloat16)
    w = (r(k, c) * (scale / math.sqrt(c))).to(torch.bfloat16).to(w_type)
    b = (r(k) * 0.5).to(torch.bfloat16).to(w_type) if bias else None
    y = (torch.rand(v, generator=g, device=dev) ** 3 * k).long().clamp_(0, k - 1)
    if ignored:
        y[torch.rand(v, generator=g, device=dev) < ignored] = IGNORED
    cw = torch.rand(k, generator=g, device=dev) + 0.5 if weighted else None
    return x, w, b, y, cw


def _definition(x, w, b, y, cw, ignore=IGNORED, scale=1.0):
    """(loss, dx, dw, db) in 64 bits, the gradients by the formula; also the voxels' weights g and the matrix D."""
    x, w = x.double(), w.double().reshape(w.shape[0], -1)
    s = x @ w.T + (0 if b is None else b.double())
    live = (y >= 0) & (y < w.shape[0]) & (y != ignore)
    yy = torch.where(live, y, 0)
    u = live.double() if cw is None else torch.where(live, cw.double()[yy], 0.0)
    den = u.sum().clamp_min(torch.finfo(torch.float32).eps)
    lse = torch.logsumexp(s, 1)
    nll = lse - s.gather(1, yy[:, None])[:, 0]
    loss = torch.where(live, u * nll, 0.0).sum() / den
    p = torch.exp(s - lse[:, None])
    d = p.scatter_add(1, yy[:, None], torch.full_like(yy[:, None], -1, dtype=torch.float64)) * (u / den * scale)[:, None]
    return loss, d @ w, d.T @ x, d.sum(0), d, s


def _check(x, w, b, y, cw, ignore=IGNORED, scale=1.0, label_type=torch.int32):
    x, w = x.clone().requires_grad_(), w.clone().requires_grad_()
    b = None if b is None else b.clone().requires_grad_()
    loss = head_cross_entropy(x, w, b, y.to(label_type), cw, ignore_label=ignore)
    (loss * scale).backward()
    _lib.check_status()
    w16 = w.detach().to(torch.bfloat16)
    rl, rdx, rdw, rdb, d, s = _definition(x.detach(), w16, None if b is None else b.detach(), y, cw, ignore, scale)
    n = x.shape[1]
    # a logit: products are exact, C of them added in fp32 (2^-24 each, 2^-23 where the sum is cut off instead of rounded);
    # the logarithm's argument a sum of rounded exponentials (2^-22 each)
    e_logit = n * 2 ** -23 * (x.detach().double().abs() @ w16.double().abs().T).amax() if len(x) else 0.0
    e_term = float(e_logit) + 2 ** -21 * (1 + float(s.abs().amax()) * 2)
    assert loss.dtype == torch.float32 and abs(float(loss) - float(rl)) <= e_term * 2 + 2 ** -23 * abs(float(rl))
    # D's entries are rounded to bf16 (2^-8 of the value at most, 2^-8 of one for the target is covered by its value),
    # after errors of e_term relative to p; then the products' fp32 sums and the result's own rounding
    rel = 2 ** -8 + 4 * e_term
    # D = g (p - [j = y]): p is off by e_term p at most, the one by nothing, so fp32 leaves errors of e_term g, however
    # small p - 1 itself is (one class: exactly 0); g is the voxel's weight over their sum
    live = (y >= 0) & (y < w16.shape[0]) & (y != ignore)
    u = live.double() if cw is None else torch.where(live, cw.double()[torch.where(live, y, 0)], 0.0)
    g = (u / u.sum().clamp_min(torch.finfo(torch.float32).eps) * scale)[:, None].abs()
    slack = 4 * e_term * g
    ex = (d.abs() * rel + slack) @ w16.double().abs()
    ew = (d.abs() * rel + slack).T @ x.detach().double().abs()
    round_w = 2 ** -8 if w.dtype == torch.bfloat16 else 2 ** -23
    assert x.grad.dtype == torch.bfloat16 and w.grad.dtype == w.dtype
    assert ((x.grad.double() - rdx).abs() <= ex + 2 ** -8 * rdx.abs()).all()
    assert ((w.grad.double().reshape(rdw.shape) - rdw).abs() <= ew + round_w * rdw.abs()).all()
    if b is not None:
        eb = (d.abs() * 4 * e_term + slack).sum(0) + d.abs().sum(0) * 2 ** -17  # chains of fp32 additions
        assert ((b.grad.double() - rdb).abs() <= eb + round_w * rdb.abs()).all()
    # and as a whole the errors do not line up: a few 2^-9
    for got, want in ((x.grad, rdx), (w.grad.reshape(rdw.shape), rdw)):
        if float(want.norm()) > 1e-12 and len(x) >= 64:
            assert float((got.double() - want).norm()) <= 4e-3 * float(want.norm())
    return loss, x.grad, w.grad, None if b is None else b.grad


NARROW = [(128, 64, 128), (1, 64, 34), (1, 8, 1), (2, 16, 2), (127, 24, 33), (129, 40, 129), (300, 64, 147), (777, 128, 300),
          (1000, 32, 1001), (500, 200, 500), (513, 256, 1025), (260, 136, 64), (3, 256, 5000), (20000, 16, 257),
          (6000, 64, 65)]
WIDE = [(1, 264, 40), (256, 512, 256), (300, 320, 300), (257, 264, 513), (1000, 1024, 1001), (20, 2048, 70), (700, 640, 2)]


@pytest.mark.gpu
@pytest.mark.parametrize("v,c,k", NARROW + WIDE)
def test_loss_and_gradients(v, c, k):
    _check(*_inputs(v, c, k))


# both gradients in one kernel: one to four tiles of classes, one and more voxel tiles a CTA, its limits and just behind,
# several launches
BOTH = [(129, 8, 1), (200, 64, 32), (256, 16, 33), (19000, 64, 128), (38100, 24, 40), (57000, 64, 257), (40000, 32, 500),
        (40000, 128, 100), (19073, 128, 128), (1000, 128, 129), (300, 64, 384), (300, 64, 385), (500, 48, 512),
        (500, 32, 513), (38017, 40, 130), (20000, 32, 1001), (300, 64, 769), (2000, 16, 1537),
        (76000, 32, 1001), (80001, 16, 1537), (90000, 24, 513), (76543, 32, 800)]


@pytest.mark.gpu
@pytest.mark.parametrize("v,c,k", BOTH)
def test_both_gradients_at_once(v, c, k):
    x, w, b, y, _ = _inputs(v, c, k, ignored=0.1)
    cw = torch.rand(k, device="cuda") + 0.5
    cw[::3] = 0.0 if k > 2 else 2.0
    _check(x, w, b, y, cw)
    _, dx, dw, db = _check(x, w, b, y, None)
    # and each of them alone, where one is asked for: the same sums from other kernels
    one = [t.clone().requires_grad_() for t in (x, w, b)]
    dx1, = torch.autograd.grad(head_cross_entropy(one[0], w, b, y, ignore_label=IGNORED), one[:1])
    dw1, db1 = torch.autograd.grad(head_cross_entropy(x, *one[1:], y, ignore_label=IGNORED), one[1:])
    # each side is within 4e-3 of the truth by its roundings to bf16 (_check), and within what fp32 leaves of D: e_term
    # of p and of the target's one, so twice e_term / V a voxel at most, along rows of W, rows of X and ones
    logits = x.double() @ w.double().T + b.double()
    e = 4 * 2 * 2 ** -21 * (1 + 2 * float(logits.abs().amax())) / int((y != IGNORED).sum())
    for got, want, size in ((dx1, dx, v ** 0.5 * float(w.double().norm(dim=1).max())),
                            (dw1, dw, float(x.double().norm(dim=1).sum())), (db1, db, v)):
        assert float((got.double() - want.double()).norm()) <= 8e-3 * float(want.double().norm()) + 2 * e * size


FIRST = """
import torch
from scaffold_b200.ops.head_loss import head_cross_entropy
x, w = (torch.randn(n, %d, device="cuda").bfloat16().requires_grad_() for n in (4096, %d))
y = torch.zeros(4096, dtype=torch.int32, device="cuda")
dx, dw = torch.autograd.grad(head_cross_entropy(x, w, None, y), (x, w))
assert torch.isfinite(dx.float()).all() and dw.abs().sum() > 0
"""


@pytest.mark.gpu
@pytest.mark.parametrize("c,k", [(16, 34), (64, 1000), (320, 40)])
def test_the_first_backward_pass_of_a_process(c, k):
    """autograd's thread has used the device for nothing yet: the first call there is the one under test."""
    root = Path(__file__).resolve().parents[1]
    run = subprocess.run([sys.executable, "-c", FIRST % (c, k)], cwd=root, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stderr[-2000:]


@pytest.mark.gpu
def test_both_gradients_are_the_same_each_time():
    x, w, b, y, _ = _inputs(30000, 64, 257)
    runs = []
    for _ in range(3):
        ps = [t.clone().requires_grad_() for t in (x, w, b)]
        runs.append(torch.autograd.grad(head_cross_entropy(*ps, y), ps))
    for other in runs[1:]:
        assert all(torch.equal(p, q) for p, q in zip(runs[0], other))


@pytest.mark.gpu
@pytest.mark.parametrize("v,c,k", [(300, 64, 147), (513, 256, 300), (400, 320, 300)])
@pytest.mark.parametrize("label_type", [torch.int16, torch.int32, torch.int64])
def test_class_weights_ignored_voxels_and_label_types(v, c, k, label_type):
    _check(*_inputs(v, c, k, ignored=0.3, weighted=True), label_type=label_type, scale=3.0)


@pytest.mark.gpu
@pytest.mark.parametrize("c", [64, 512])
def test_without_a_bias_and_with_an_fp32_weight(c):
    _check(*_inputs(400, c, 200, bias=False))
    _check(*_inputs(400, c, 200, w_type=torch.float32, weighted=True))


@pytest.mark.gpu
@pytest.mark.parametrize("v,c,k", [(20000, 264, 3000), (40000, 512, 700), (300, 320, 120000),
                                   (24000, 264, 3500), (600, 320, 120000), (20000, 264, 5000)])
def test_the_wide_gradient_in_several_pieces(v, c, k):
    """More classes, more voxels, more of both than one piece of the gradient's matrix holds: against fp32 products of
    the formula."""
    x, w, b, y, cw = _inputs(v, c, k, weighted=True)
    x, w, b = (t.requires_grad_() for t in (x, w, b))
    loss = head_cross_entropy(x, w, b, y.int(), cw)
    loss.backward()
    with torch.no_grad():
        s = (x.float() @ w.float().T + b.float())
        u = cw[y] / cw[y].sum()
        p = torch.softmax(s, 1)
        ref = (torch.logsumexp(s, 1) - s.gather(1, y[:, None])[:, 0]).mul(u).sum()
        p.scatter_add_(1, y[:, None], -torch.ones_like(y[:, None], dtype=torch.float32))
        p *= u[:, None]
        # roundings of D and of the result at random, 2^-9 / sqrt(3) each and once more for a target that stands alone
        for got, want in ((x.grad, p @ w.float()), (w.grad, p.T @ x.float()), (b.grad, p.sum(0))):
            assert float((got.float() - want).norm()) <= 4e-3 * float(want.norm())
            assert float((got.float() - want).abs().max()) <= 2e-2 * float(want.abs().max())
        assert abs(float(loss) - float(ref)) <= 1e-5 * float(ref)


@pytest.mark.gpu
@pytest.mark.parametrize("c", [32, 320])
def test_confident_voxels_keep_the_gradient_of_their_target(c):
    """p of the target near one: p - 1 is taken before anything is rounded to bf16."""
    x, w, b, y, _ = _inputs(600, c, 300, seed=3)
    w = (w.float() * 8).to(torch.bfloat16)
    y = (x.double() @ w.double().T + b.double()).argmax(1)
    rl, rdx, _, _, d, _ = _definition(x, w, b, y, None)
    assert float(d.gather(1, y[:, None]).abs().median()) < 0.1 / 600  # the inputs are what they are for
    xg = x.clone().requires_grad_()
    head_cross_entropy(xg, w, b, y).backward()
    size = rdx.norm(dim=1)
    # voxels whose own 1 - p is well above fp32's resolution of one
    some = d.gather(1, y[:, None])[:, 0].abs() * 600 > 1e-3
    assert some.sum() > 20
    assert ((xg.grad.double() - rdx).norm(dim=1)[some] <= 0.01 * size[some]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("c", [64, 320])
def test_voxels_that_take_no_part(c):
    x, w, b, y, _ = _inputs(500, c, 100, ignored=0.5)
    _, dx, dw, db = _check(x, w, b, y, None)
    assert not dx[y == IGNORED].any()
    # all of them
    xs, ws, bs = (t.clone().requires_grad_() for t in (x, w, b))
    loss = head_cross_entropy(xs, ws, bs, torch.full_like(y, IGNORED), None, ignore_label=IGNORED)
    loss.backward()
    assert float(loss) == 0 and not xs.grad.any() and not ws.grad.any() and not bs.grad.any()
    # a class of weight zero takes no part either
    cw = torch.ones(100, device="cuda")
    cw[y[y >= 0][0]] = 0
    _check(x, w, b, y, cw)
    # no voxels at all
    none = x[:0].requires_grad_()
    loss = head_cross_entropy(none, w, b, y[:0])
    loss_grad = torch.autograd.grad(loss, none)[0]
    assert float(loss) == 0 and loss_grad.shape == (0, c)


@pytest.mark.gpu
@pytest.mark.parametrize("c", [64, 320])
def test_labels_outside_the_classes_are_reported_and_take_no_part(c):
    x, w, b, y, _ = _inputs(300, c, 40)
    y[7], y[200] = 40, -100
    xg = x.clone().requires_grad_()
    loss = head_cross_entropy(xg, w, b, y)
    with pytest.raises(_lib.DeviceArgumentError, match="head loss"):
        _lib.check_status()
    rl, rdx, *_ = _definition(x, w, b, y, None)
    assert abs(float(loss) - float(rl)) <= 1e-5 * float(rl)
    loss.backward()
    assert not xg.grad[7].any() and not xg.grad[200].any()
    assert float((xg.grad.double() - rdx).norm()) <= 4e-3 * float(rdx.norm())
    loss = head_cross_entropy(x, w, b, torch.where(y == 40, 3, y), ignore_label=-100)
    _lib.check_status()


@pytest.mark.gpu
@pytest.mark.parametrize("c", [64, 320])
def test_infinite_logits(c):
    """A class switched off by a bias of -inf has probability zero; NaN features of a voxel show in the loss."""
    x, w, b, y, _ = _inputs(300, c, 70)
    b[5], b[64] = float("-inf"), float("-inf")
    y[(y == 5) | (y == 64)] = 6
    xs, ws, bs = (t.clone().requires_grad_() for t in (x, w, b))
    loss = head_cross_entropy(xs, ws, bs, y)
    loss.backward()
    rl, rdx, rdw, rdb, *_ = _definition(x, w, b, y, None)
    assert abs(float(loss) - float(rl)) <= 1e-5 * float(rl)
    assert not ws.grad[5].any() and not bs.grad[64].any()
    for got, want in ((xs.grad, rdx), (ws.grad, rdw), (bs.grad, rdb)):
        assert got.isfinite().all() and float((got.double() - want).norm()) <= 4e-3 * float(want.norm())
    x[3, 1] = float("nan")
    xs = x.clone().requires_grad_()
    loss = head_cross_entropy(xs, w, b, y)
    loss.backward()
    assert loss.isnan() and xs.grad[3].isnan().all()
    y[3] = IGNORED  # a voxel that takes no part leaves the loss and the others' gradients alone
    xs = x.clone().requires_grad_()
    loss = head_cross_entropy(xs, w, b, y, ignore_label=IGNORED)
    loss.backward()
    assert loss.isfinite() and xs.grad[:3].isfinite().all() and xs.grad[4:].isfinite().all()


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("v,c,k", [(300, 64, 70), (5000, 16, 34), (400, 128, 300), (7, 256, 3000), (300, 320, 70), (5, 320, 3000)])
def test_a_label_on_a_class_that_is_off(v, c, k, dev):
    """Its bias is -inf: the loss is +inf. The type's lowest number: as large, not the stand-in that the kernels multiply
    with. A class weight of zero takes the voxel out."""
    x, w, b, y, _ = _inputs(v, c, k, dev=dev)
    y[y == 5] = 6
    fine = float(head_cross_entropy(x, w, b, y))
    assert math.isfinite(fine)
    y[v // 2] = 5
    b[5] = float("-inf")
    xs, ws, bs = (t.clone().requires_grad_() for t in (x, w, b))
    loss = head_cross_entropy(xs, ws, bs, y)
    assert float(loss.detach()) == math.inf
    if dev == "cuda":  # (in 32 bits the formula's gradients are those of inf - inf)
        loss.backward()
        for got, want in zip((xs.grad, ws.grad, bs.grad), _definition(x, w, b, y, None)[1:4]):
            assert got.isfinite().all() and float((got.double() - want).norm()) <= 4e-3 * float(want.norm())
    cw = torch.ones(k, device=dev)
    cw[5] = 0
    keep = torch.where(y == 5, IGNORED, y)
    assert float(head_cross_entropy(x, w, b, y, cw)) == float(head_cross_entropy(x, w, b, keep, torch.ones_like(cw),
                                                                                 ignore_label=IGNORED))
    b = b.float()
    for low in (torch.finfo(torch.bfloat16).min, torch.finfo(torch.float32).min, -1e31):
        b[5] = low
        got = float(head_cross_entropy(x, w, b, y))
        # one term of the size of -low among v: fp32's roundings of the logit and of the result
        assert abs(got - -float(b[5]) / v) <= 2 ** -22 * -float(b[5]) / v, (got, low)


@pytest.mark.gpu
@pytest.mark.parametrize("low", [float("-inf"), torch.finfo(torch.bfloat16).min, -1e30, -1e20, -1e10, -3e9, -1e9, -1e6, -1e4])
@pytest.mark.parametrize("v,c,k", [(300, 64, 147), (5000, 16, 129), (63, 48, 385), (1575, 40, 129), (70000, 24, 100),
                                   (300, 200, 300), (7, 256, 3000), (300, 320, 300)])
def test_runs_of_classes_that_are_off(v, c, k, low):
    """A mask of the classes at the front, at the end and in between, as a bias far below the others: whole runs of columns
    have nothing else, and their probabilities are zero."""
    x, w, b, y, _ = _inputs(v, c, k, w_type=torch.float32, scale=4.0)
    w = w.to(torch.bfloat16)
    b = b.float()
    y = y % 5 + 70  # the classes that stay are 64 to 95
    for off in (slice(0, 64), slice(128, None), slice(0, 1), slice(96, None)):
        b[off] = low
        leaves = [t.clone().requires_grad_() for t in (x, w, b)]
        loss = head_cross_entropy(*leaves, y)
        grads = torch.autograd.grad(loss, leaves)
        rl, *want, _, s = _definition(x, w, b, y, None)
        error = c * 2 ** -23 * float((x.double().abs() @ w.double().abs().T).amax()) + 2 ** -20 * (1 + float(s[:, 64:96].abs().amax()))
        assert abs(float(loss.detach()) - float(rl)) <= 2 * error + 2 ** -23 * float(rl)
        for got, ref in zip(grads, want):
            assert got.isfinite().all()
            assert float((got.double() - ref).norm()) <= 4e-3 * float(ref.norm()) + 4 * error * float(ref.abs().amax()) * ref.numel() ** 0.5
        assert ((H.head_predict(x, w, b) >= 64) & (H.head_predict(x, w, b) < 128)).all() or off.start == 0


@pytest.mark.gpu
def test_shapes_views_and_evaluation():
    x, w, b, y, cw = _inputs(2 * 3 * 4 * 5, 48, 50, weighted=True)
    ref = head_cross_entropy(x, w, b, y, cw)
    vol, lab = x.view(2, 3, 4, 5, 48), y.view(2, 3, 4, 5)
    conv = w.view(50, 48, 1, 1, 1)
    assert torch.equal(head_cross_entropy(vol, conv, b, lab, cw), ref)
    padded = torch.zeros(2, 3, 4, 5, 64, dtype=torch.bfloat16, device="cuda")
    padded[..., 8:56] = vol
    assert torch.equal(head_cross_entropy(padded[..., 8:56], conv, b, lab, cw), ref)  # a strided view
    shifted = torch.empty(x.numel() + 1, dtype=torch.bfloat16, device="cuda")[1:].view_as(x).copy_(x)  # off 16 bytes
    assert torch.equal(head_cross_entropy(shifted, w, b, y, cw), ref)
    assert torch.equal(head_cross_entropy(x, w.T.contiguous().T, b, y, cw), ref)
    assert torch.equal(head_cross_entropy(x.t().contiguous().t(), w, b, y, cw), ref)
    one = head_cross_entropy(x[0], w, b, y[0], cw)
    assert abs(float(one) - float(_definition(x[:1], w, b, y[:1], cw)[0])) <= 1e-5 * max(1.0, float(one))
    with torch.autocast("cuda", dtype=torch.bfloat16):
        assert torch.equal(head_cross_entropy(x.float(), w.float(), b.float(), y, cw), ref)
    # only what is asked for
    wg = w.clone().requires_grad_()
    head_cross_entropy(x, wg, b, y, cw).backward()
    xg, wh, bg = (t.clone().requires_grad_() for t in (x, w, b))
    head_cross_entropy(xg, wh, bg, y, cw).backward()
    assert torch.equal(wg.grad, wh.grad)
    bo = b.clone().requires_grad_()
    head_cross_entropy(x, w, bo, y, cw).backward()
    assert torch.equal(bo.grad, bg.grad)
    xo = vol.clone().requires_grad_()
    head_cross_entropy(xo, conv, b, lab, cw).backward()
    assert torch.equal(xo.grad.view_as(x), xg.grad)


@pytest.mark.gpu
@pytest.mark.parametrize("v,c,k", [(5000, 64, 300), (900, 512, 700)])
def test_the_same_call_gives_the_same_bits(v, c, k):
    x, w, b, y, cw = _inputs(v, c, k, weighted=True)
    first = None
    for _ in range(3):
        xs, ws, bs = (t.clone().requires_grad_() for t in (x, w, b))
        loss = head_cross_entropy(xs, ws, bs, y, cw)
        loss.backward()
        got = loss.detach(), xs.grad, ws.grad, bs.grad
        first = first or got
        assert all(torch.equal(p, q) for p, q in zip(first, got))


@pytest.mark.gpu
@pytest.mark.parametrize("c", [64, 320])
def test_two_calls_in_one_graph_of_gradients_and_two_streams(c):
    x, w, b, y, _ = _inputs(400, c, 90)
    xs, ws, bs = (t.clone().requires_grad_() for t in (x, w, b))
    first = head_cross_entropy(xs, ws, bs, y)
    second = head_cross_entropy(xs, ws, bs, (y + 1) % 90)
    (first + 2 * second).backward()
    want = _definition(x, w, b, y, None)[1] + 2 * _definition(x, w, b, (y + 1) % 90, None)[1]
    assert float((xs.grad.double() - want).norm()) <= 6e-3 * float(want.norm())
    streams = [torch.cuda.Stream() for _ in range(2)]
    out = []
    torch.cuda.synchronize()
    for s in streams:
        with torch.cuda.stream(s):
            a = x.clone().requires_grad_()
            head_cross_entropy(a, w, b, y).backward()
            out.append(a)
    torch.cuda.synchronize()
    assert torch.equal(out[0].grad, out[1].grad)


@pytest.mark.gpu
@pytest.mark.parametrize("c", [64, 320])
def test_a_captured_pass_is_replayed_on_new_values(c):
    x, w, b, y, _ = _inputs(700, c, 150)
    xs, ws, bs = (t.requires_grad_() for t in (x, w, b))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(head_cross_entropy(xs, ws, bs, y), (xs, ws, bs))
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):  # two graphs: neither shares anything with the other
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            loss = head_cross_entropy(xs, ws, bs, y)
            outs.append((loss, *torch.autograd.grad(loss, (xs, ws, bs))))
        graphs.append(graph)
    nx, nw, nb, ny, _ = _inputs(700, c, 150, seed=5)
    with torch.no_grad():
        for t, n in ((xs, nx), (ws, nw), (bs, nb), (y, ny)):
            t.copy_(n)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for s, graph in zip(streams, graphs):
        with torch.cuda.stream(s):
            graph.replay()
    torch.cuda.synchronize()
    loss = head_cross_entropy(xs, ws, bs, y)
    want = (loss, *torch.autograd.grad(loss, (xs, ws, bs)))
    for got in outs:
        assert all(torch.equal(p, q) for p, q in zip(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize("v,c,k", [(130, 24, 35), (300, 320, 70)])
def test_nothing_is_written_beside_the_gradients(v, c, k):
    """The neighbours in memory of gradients, state and scratch: each in the middle of a larger buffer."""
    x, w, b, y, cw = _inputs(v, c, k, weighted=True)
    dev, margin = x.device, 4096
    L, st, status = _lib.lib(), _lib.stream_ptr(), _lib.status_tensor(x.device).data_ptr()
    y = y.int()

    def guarded(n, t=torch.uint8):
        buf = torch.full((n + 2 * margin,), 77, dtype=t, device=dev)
        return buf, buf[margin:].data_ptr()

    bufs = [guarded(n) for n in H._bytes(v, k, c, True)]
    loss, dx, dw, db = guarded(1, torch.float32), *(guarded(n, torch.bfloat16) for n in (v * c, k * c, k))
    _lib.check(L.sb_head_forward(x.data_ptr(), w.data_ptr(), b.data_ptr(), 0, y.data_ptr(), 4, 0, 0, cw.data_ptr(), v, k, c,
                                 bufs[0][1], bufs[1][1], loss[1], status, st), "sb_head_forward")
    one = torch.ones(1, device=dev)
    _lib.check(L.sb_head_backward(x.data_ptr(), w.data_ptr(), cw.data_ptr(), v, k, c, bufs[0][1], bufs[2][1], one.data_ptr(),
                                  dx[1], dw[1], 0, db[1], 0, status, st), "sb_head_backward")
    torch.cuda.synchronize()
    _lib.check_status()
    for t, _ in (*bufs, loss, dx, dw, db):
        assert (t[:margin] == 77).all() and (t[-margin:] == 77).all()
    xs, ws, bs = (t.clone().requires_grad_() for t in (x, w, b))
    head_cross_entropy(xs, ws, bs, y, cw).backward()
    assert torch.equal(dx[0][margin:-margin].view(v, c), xs.grad) and torch.equal(dw[0][margin:-margin].view(k, c), ws.grad)
    assert torch.equal(db[0][margin:-margin], bs.grad)


@pytest.mark.gpu
@pytest.mark.parametrize("v,c,k,weighted", [(130, 24, 35, False), (300, 64, 257, False), (5000, 64, 147, True),
                                            (76001, 24, 1001, False), (4100, 8, 33, True), (300, 320, 70, True)])
def test_nothing_is_written_beside_both_gradients(v, c, k, weighted):
    """As above where both gradients come from one kernel, also in several launches: dX leaves it by TMA."""
    x, w, b, y, cw = _inputs(v, c, k, ignored=0.1, weighted=weighted)
    dev, margin = x.device, 4096
    L, st, status = _lib.lib(), _lib.stream_ptr(), _lib.status_tensor(x.device).data_ptr()
    y = y.int()

    def guarded(n, t=torch.uint8):
        buf = torch.full((n + 2 * margin,), 77, dtype=t, device=dev)
        return buf, buf[margin:].data_ptr()

    n_state, n_fwd, _, n_both = H._bytes(v, k, c, weighted)
    bufs = [guarded(n) for n in (n_state, n_fwd, n_both)]
    loss, dx, dw, db = guarded(1, torch.float32), *(guarded(n, torch.bfloat16) for n in (v * c, k * c, k))
    _lib.check(L.sb_head_forward(x.data_ptr(), w.data_ptr(), b.data_ptr(), 0, y.data_ptr(), 4, 1, IGNORED, _lib.ptr(cw), v, k,
                                 c, bufs[0][1], bufs[1][1], loss[1], status, st), "sb_head_forward")
    one = torch.ones(1, device=dev)
    _lib.check(L.sb_head_backward(x.data_ptr(), w.data_ptr(), _lib.ptr(cw), v, k, c, bufs[0][1], bufs[2][1], one.data_ptr(),
                                  dx[1], dw[1], 0, db[1], 0, status, st), "sb_head_backward")
    torch.cuda.synchronize()
    _lib.check_status()
    for t, _ in (*bufs, loss, dx, dw, db):
        assert (t[:margin] == 77).all() and (t[-margin:] == 77).all()
    xs, ws, bs = (t.clone().requires_grad_() for t in (x, w, b))
    head_cross_entropy(xs, ws, bs, y, cw, ignore_label=IGNORED).backward()
    assert torch.equal(dx[0][margin:-margin].view(v, c), xs.grad) and torch.equal(dw[0][margin:-margin].view(k, c), ws.grad)
    assert torch.equal(db[0][margin:-margin], bs.grad)


@pytest.mark.gpu
@pytest.mark.parametrize("v,c,k", [(1, 8, 1), (1, 64, 5000), (300, 64, 147), (1000, 16, 33), (129, 256, 1000), (257, 320, 513),
                                   (30, 1024, 3000), (70000, 32, 34)])
def test_the_predicted_class(v, c, k):
    """Whole numbers make every logit exact: the class is torch's, with many ties (the lowest wins)."""
    g = torch.Generator(device="cuda").manual_seed(v + k)
    x = torch.randint(-1, 2, (v, c), generator=g, device="cuda").to(torch.bfloat16)
    w = torch.randint(-1, 2, (k, c), generator=g, device="cuda").to(torch.bfloat16)
    b = torch.randint(-2, 3, (k,), generator=g, device="cuda").to(torch.bfloat16)
    logits = x.double() @ w.double().T + b.double()
    got = H.head_predict(x, w, b)
    assert got.dtype == torch.int64 and torch.equal(got, logits.argmax(1))
    assert torch.equal(H.head_predict(x.view(1, v, 1, c), w.view(k, c, 1, 1, 1)), (x.double() @ w.double().T).argmax(1).view(1, v, 1))
    if k > 2:
        b[1] = float("inf")
        b[0] = float("-inf")
        assert (H.head_predict(x, w, b) == 1).all()
        x[0, 0] = float("nan")  # every logit of the voxel: the first one
        assert int(H.head_predict(x, w)[0]) == 0
    assert H.head_predict(x[:0], w).shape == (0,)


@pytest.mark.gpu
@pytest.mark.parametrize("v,c,k", [(1, 8, 1), (5, 64, 33), (40, 64, 147), (600, 16, 1001), (129, 256, 1025), (9, 320, 40),
                                   (300, 320, 513)])
def test_the_predicted_class_is_a_class_whatever_the_features_hold(v, c, k):
    """Infinite features make every logit infinite or NaN, and NaN of the zeros behind the last class."""
    g = torch.Generator(device="cuda").manual_seed(v + k)
    sign = lambda *s: (torch.randint(0, 2, s, generator=g, device="cuda") * 2 - 1).to(torch.bfloat16)  # noqa: E731
    x, w = sign(v, c), sign(k, c)
    w[:, 1] = -1
    x[::3, 0] = float("inf")   # logits of +inf and -inf: the first class of +inf
    x[1::3, 1] = float("inf")  # -inf in every class: the first one
    got = H.head_predict(x, w)
    want = (x.float() @ w.float().T).argmax(1)
    assert torch.equal(got, want) and int(want[1::3].max() if v > 1 else 0) == 0
    # large finite logits of one sign are smaller than the zeros behind the last class
    big = torch.full((3, c), 1e36, dtype=torch.bfloat16, device="cuda")
    assert torch.equal(H.head_predict(big, -w.abs()), torch.zeros(3, dtype=torch.int64, device="cuda"))


def test_the_predicted_class_on_the_cpu():
    x, w, b, *_ = _inputs(50, 16, 9, dev="cpu")
    assert torch.equal(H.head_predict(x, w, b), (x.float() @ w.float().T + b.float()).argmax(1))
    with pytest.raises(ValueError, match="weight"):
        H.head_predict(x, w[:, :8], b)


def test_the_formula_on_the_cpu_and_its_gradients():
    x, w, b, y, cw = _inputs(60, 24, 40, ignored=0.2, weighted=True, dev="cpu")
    xs, ws, bs = (t.double().requires_grad_() for t in (x, w, b))
    loss = head_cross_entropy(xs, ws, bs, y, cw, ignore_label=IGNORED)
    loss.backward()
    rl, rdx, rdw, rdb, *_ = _definition(x, w, b, y, cw)
    assert torch.allclose(loss.detach(), rl) and torch.allclose(xs.grad, rdx) and torch.allclose(ws.grad, rdw)
    assert torch.allclose(bs.grad, rdb)
    low = head_cross_entropy(x, w, b, y.to(torch.int16), cw, ignore_label=IGNORED)
    assert low.dtype == torch.float32 and abs(float(low) - float(rl)) < 1e-5


@pytest.mark.parametrize("bias", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_autocast_leaves_the_formula_in_32_bits(dtype, bias):
    x, w, b, y, cw = _inputs(700, 24, 40, weighted=True, bias=bias, w_type=torch.float32, dev="cpu")
    want, pred = head_cross_entropy(x, w, b, y, cw), H.head_predict(x, w, b)
    with torch.autocast("cpu", dtype=dtype):
        loss = head_cross_entropy(x, w, b, y, cw)
        assert loss.dtype == torch.float32 and torch.equal(loss, want)
        assert torch.equal(H.head_predict(x, w, b), pred)


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_class_weights_have_no_gradient(dev):
    x, w, b, y, cw = _inputs(60, 24, 40, weighted=True, dev=dev)
    x.requires_grad_()
    loss = head_cross_entropy(x, w, b, y, cw.requires_grad_())
    assert torch.equal(loss, head_cross_entropy(x, w, b, y, cw.detach()))
    dx, none = torch.autograd.grad(loss, (x, cw), allow_unused=True)
    assert none is None and dx.any()


def test_the_gradient_against_differences():
    x, w, b, y, cw = _inputs(7, 8, 12, weighted=True, dev="cpu")
    leaves = [t.double().requires_grad_() for t in (x, w, b)]
    assert torch.autograd.gradcheck(lambda *t: head_cross_entropy(*t, y, cw), leaves)


def test_refusals():
    x, w, b, y, cw = _inputs(10, 16, 5, weighted=True, dev="cpu")
    with pytest.raises(ValueError, match="labels"):
        head_cross_entropy(x, w, b, y[:9])
    with pytest.raises(ValueError, match="weight"):
        head_cross_entropy(x, w[:, :8], b, y)
    with pytest.raises(ValueError, match="weight"):
        head_cross_entropy(x, w.reshape(5, 4, 4), b, y)
    with pytest.raises(ValueError, match="bias"):
        head_cross_entropy(x, w, b[:4], y)
    with pytest.raises(ValueError, match="class_weights"):
        head_cross_entropy(x, w, b, y, cw[:4])
    with pytest.raises(TypeError, match="labels"):
        head_cross_entropy(x, w, b, y.float())
    with pytest.raises(ValueError, match="ignore_label"):
        head_cross_entropy(x, w, b, y, ignore_label=2 ** 63)
    assert H.head_supported(8) and H.head_supported(1024) and not H.head_supported(12) and not H.head_supported(4)


@pytest.mark.gpu
def test_refusals_on_the_device():
    x, w, b, y, cw = _inputs(10, 16, 5, weighted=True)
    with pytest.raises(ValueError, match="multiples of 8"):
        head_cross_entropy(x[:, :12], w[:, :12], b, y)
    with pytest.raises(ValueError, match="labels is on"):
        head_cross_entropy(x, w, b, y.cpu())
    with pytest.raises(TypeError, match="bf16 or fp32"):
        head_cross_entropy(x, w.half(), b, y)
    xs = x.requires_grad_()
    loss = head_cross_entropy(xs, w, b, y)
    (g,) = torch.autograd.grad(loss, xs, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
