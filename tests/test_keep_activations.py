"""Training with 8-bit activations and with the logit-free loss, through the model, the engine and the configuration."""
import pytest
import torch

from helpers.launch import ROOT, results, torchrun_gloo
from scaffold_b200.models.unet import UNet
from scaffold_b200.ops import _lib, loss as L
from scaffold_b200.ops.conv3d import Conv3d, ConvTranspose3d
from scaffold_b200.ops.head_loss import head_cross_entropy, head_predict
from scaffold_b200.ops.optim import FusedClipAdam
from scaffold_b200.train.engine import TrainEngine


def _model(n_classes=6, width=32, layers=2, dev="cuda", seed=0):
    torch.manual_seed(seed)
    return UNet(3, n_classes, layers=layers, base_width=width).to(dev, memory_format=torch.channels_last_3d)


def _batch(n_classes, dims=(32, 32, 32), batch=2, dev="cuda", seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    x = torch.rand(batch, 3, *dims, generator=g, device=dev)
    y = (torch.rand(batch, *dims, generator=g, device=dev) ** 3 * n_classes).to(torch.int16)
    return x, y


def _gradients(model, x, y, n_classes, saved=None):
    model.zero_grad(set_to_none=True)
    weights = {p.data_ptr() for p in model.parameters()}  # saved too, and nobody's activations

    def pack(t):
        if saved is not None and t.data_ptr() not in weights:
            saved[t.data_ptr()] = t.numel() * t.element_size()
        return t
    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
        with torch.autocast("cuda", dtype=torch.bfloat16):
            logits = model.forward_padded_logits(x)
        loss, *_ = L.segmentation_loss_fused(logits, y, n_classes)
    loss.backward()
    return loss.detach(), {n: p.grad.clone() for n, p in model.named_parameters()}


@pytest.mark.gpu
@pytest.mark.parametrize("dims,width", [((32, 32, 32), 32), ((20, 28, 36), 16), ((16, 16, 16), 64)])
def test_eight_bits_change_the_gradients_by_the_copies_steps_only(dims, width):
    model = _model(width=width)
    x, y = _batch(6, dims)
    plain, kept = {}, {}
    loss, want = _gradients(model, x, y, 6, plain)
    model.keep_activations(8)
    loss8, got = _gradients(model, x, y, 6, kept)
    assert torch.equal(loss, loss8)  # the forward pass is the same
    # A step is at most 1/63 of a block's largest value, its rounding uniform: 1/63/sqrt(12) = 0.5 % of it in the root mean
    # square, at random, per layer; the deepest path has some twenty layers: below 0.005 * sqrt(20) * 2 of a gradient
    for n, g in want.items():
        assert float((got[n] - g).norm()) <= 0.05 * float(g.norm()) + 1e-12, n
    assert sum(kept.values()) <= 0.66 * sum(plain.values())
    model.keep_activations(16)
    again = _gradients(model, x, y, 6)[1]
    assert all(torch.equal(again[n], want[n]) for n in want)


@pytest.mark.gpu
def test_a_few_steps_run_with_captured_passes_and_recomputation():
    for recompute in (False, True):
        model = _model(width=16)
        model.keep_activations(8)
        if recompute:
            model.use_checkpointing()
        engine = TrainEngine(model, FusedClipAdam(model.parameters(), lr=1e-3), 6, "cuda")
        x, y = _batch(6, (16, 16, 16))
        losses = [float(engine.step(x, y)) for _ in range(6)]
        assert all(v == v for v in losses)
        _lib.check_status()
    model.keep_activations(16)  # a setting of the modules: the captured passes with the other one are not replayed
    assert float(engine.step(x, y)) == float(engine.last_ce + 1 - engine.last_dice)


@pytest.mark.gpu
def test_a_captured_step_is_the_ordinary_step():
    x, y = _batch(6, (16, 16, 16))
    results = []
    for captured in (True, False):
        model = _model(width=16)
        model.keep_activations(8)
        engine = TrainEngine(model, FusedClipAdam(model.parameters(), lr=1e-3), 6, "cuda")
        if not captured:
            engine._graphs._usable = lambda *a: False
        results.append([float(engine.step(x, y)) for _ in range(5)])
    assert results[0] == results[1]


@pytest.mark.gpu
def test_a_pass_without_gradients_makes_no_copies():
    model = _model(width=16)
    x, y = _batch(6, (16, 20, 16))
    engine = TrainEngine(model, torch.optim.SGD(model.parameters(), lr=0.0), 6, "cuda")
    counts, losses = [], []
    for bits in (16, 8):
        model.keep_activations(bits)
        engine.eval_step(x, y)  # operand copies are made
        before = _lib.launch_count()
        losses.append(engine.eval_step(x, y)[0])
        counts.append(_lib.launch_count() - before)
    assert counts[0] == counts[1] > 0 and torch.equal(*losses)


@pytest.mark.gpu
def test_passes_that_were_captured_with_other_bits_are_not_replayed():
    """Results of the forward pass are the same with 8 and 16 bits, gradients are not: those tell what ran."""
    x, y = _batch(6, (16, 16, 16))
    grads = {}
    for name, bits, captured in (("8", 8, True), ("8 ordinary", 8, False), ("16 ordinary", 16, False)):
        model = _model(width=16)
        engine = TrainEngine(model, FusedClipAdam(model.parameters(), lr=0.0), 6, "cuda")
        if not captured:
            engine._graphs._usable = lambda *a: False
        model.keep_activations(bits)
        for _ in range(4):
            engine.step(x, y)
        grads[name] = engine.flat.grad.clone()
        if captured:
            (old,) = engine._graphs._passes.values()
            assert type(old).__name__ == "_Pass" and old.fingerprint.holds(engine)
            model.keep_activations(16)
            assert not old.fingerprint.holds(engine)
            for _ in range(4):
                engine.step(x, y)
            (new,) = engine._graphs._passes.values()
            assert new is not old and type(new).__name__ == "_Pass"
            grads["16"] = engine.flat.grad.clone()
    assert torch.equal(grads["8"], grads["8 ordinary"]) and torch.equal(grads["16"], grads["16 ordinary"])
    assert not torch.equal(grads["8"], grads["16"])


class _Halo:
    """A spatial context of two shards along the depth whose neighbours are outside of the volume."""

    size, dims, lead_swap, halo_channel = 2, [2], None, None

    @staticmethod
    def halo_pad(x, halo):
        return torch.nn.functional.pad(x, (0, 0, 0, 0, halo, halo))


@pytest.mark.gpu
@pytest.mark.parametrize("kernel,kept", [(3, False), (1, True)])
def test_a_convolution_that_exchanges_with_other_shards_keeps_16_bits(kernel, kept):
    torch.manual_seed(0)
    conv = Conv3d(32, 32, kernel, padding=kernel // 2, bias=False).cuda()
    x = torch.randn(1, 32, 8, 12, 16, device="cuda").to(memory_format=torch.channels_last_3d).requires_grad_()
    grads = []
    for bits, spatial in ((16, None), (16, _Halo), (8, _Halo)):
        conv.keep_bits = bits
        conv.set_spatial(spatial)
        saved = []
        with torch.autograd.graph.saved_tensors_hooks(lambda t: (saved.append(t.dtype), t)[1], lambda t: t):
            with torch.autocast("cuda", dtype=torch.bfloat16):
                y = conv(x)
        grads.append(torch.autograd.grad(y, (x, conv.weight), torch.ones_like(y)))
        assert (torch.uint8 in saved) == (kept and bits == 8)
    _lib.check_status()
    if not kept:
        assert all(torch.equal(a, b) for a, b in zip(grads[1], grads[2]))
    # (a padded volume is cut into other parts: the same products in another order)
    for a, b in zip(grads[0], grads[1]):
        assert float((a - b).norm()) <= 1e-3 * float(a.norm())


def test_the_setting_on_the_cpu():
    model = _model(dev="cpu", width=8, layers=1)
    x, y = _batch(6, (8, 8, 8), 1, "cpu")
    grads = []
    for bits in (16, 8):
        model.keep_activations(bits)
        model.zero_grad()
        model(x).sum().backward()
        grads.append([p.grad.clone() for p in model.parameters()])
    assert all(torch.equal(a, b) for a, b in zip(*grads))  # the kernel path alone keeps copies
    with pytest.raises(ValueError, match="8 or 16"):
        model.keep_activations(4)


# -- the loss without logits -------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("n_classes,weighted", [(40, False), (150, True), (6, True)])
def test_the_cross_entropy_of_a_wide_head_trains_through_the_engine(n_classes, weighted):
    x, y = _batch(n_classes, (16, 24, 20))
    cw = torch.linspace(0.5, 2.0, n_classes, device="cuda") if weighted else None
    model = _model(n_classes)
    engine = TrainEngine(model, torch.optim.SGD(model.parameters(), lr=0.0), n_classes, "cuda", class_weights=cw,
                         loss="ce", max_norm=1e9)
    loss = engine.step(x, y)
    _lib.check_status()
    got = {n: p.grad.clone() for n, p in model.named_parameters()}
    model.zero_grad(set_to_none=True)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        features = model.features(x)
    head = model.up_list[-1].conv
    logits = torch.einsum("ncdhw,kc->nkdhw", features.float(), head.weight.flatten(1).to(torch.bfloat16).float())
    logits = logits + head.bias[:, None, None, None]
    want = L.sharded_cross_entropy(torch.log_softmax(logits, 1), y, cw)
    want.backward()
    assert engine.last_dice.isnan() and torch.equal(loss, engine.last_ce)
    # the formula keeps the softmax's entries in fp32, the kernels round them to bf16 (2^-8 at most, at random); the
    # gradient of the features is rounded to bf16 on both sides and goes through the same backward pass
    assert abs(float(loss.detach()) - float(want.detach())) <= 1e-5 * float(want.detach())
    for n, p in model.named_parameters():
        assert float((got[n] - p.grad).norm()) <= 0.02 * float(p.grad.norm()) + 1e-12, n


@pytest.mark.gpu
def test_copies_and_the_loss_without_logits_together():
    """The set as it is used: 8-bit copies in every layer, a head of 200 classes, the flat optimizer, validation."""
    n_classes = 200
    x, y = _batch(n_classes, (32, 32, 32), 1)
    model = _model(n_classes)
    model.keep_activations(8)
    engine = TrainEngine(model, FusedClipAdam(model.parameters(), lr=1e-3), n_classes, "cuda", loss="ce")
    losses = [float(engine.step(x, y)) for _ in range(4)]
    val, dice = engine.eval_step(x, y)
    _lib.check_status()
    assert all(v == v for v in losses) and float(val) == float(val) and dice.shape == (1, n_classes)
    head = model.up_list[-1].conv
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16):
        features = model.features(x)
    with torch.no_grad():
        logits = torch.einsum("ncdhw,kc->nkdhw", features.double(), head.weight.flatten(1).to(torch.bfloat16).double())
        logits = logits + head.bias.double()[:, None, None, None]
        want = L.sharded_cross_entropy(torch.log_softmax(logits, 1), y)
        pred = head_predict(features.permute(0, 2, 3, 4, 1), head.weight, head.bias)
    assert abs(float(val) - float(want)) <= 1e-5 * float(want)
    # the predicted class has the largest logit up to fp32's error of a sum of 32 products
    top = logits.amax(1)
    assert (top - logits.gather(1, pred[:, None])[:, 0] <= 1e-4).all()
    ref = L.hard_dice_reference(torch.nn.functional.one_hot(pred, n_classes).permute(0, 4, 1, 2, 3).float(), y, n_classes)
    torch.testing.assert_close(dice, ref, rtol=2e-7, atol=0)


@pytest.mark.gpu
def test_another_loss_ends_the_replays():
    x, y = _batch(6, (16, 16, 16))
    model = _model(width=16)
    engine = TrainEngine(model, FusedClipAdam(model.parameters(), lr=0.0), 6, "cuda")
    for _ in range(4):
        engine.step(x, y)
    for _ in range(4):
        both = engine.eval_step(x, y)
    assert all(type(p).__name__ == "_Pass" for p in engine._graphs._passes.values()) and len(engine._graphs._passes) == 2
    ce = engine.last_ce.clone()
    assert not engine.last_dice.isnan()
    engine.loss = "ce"
    loss = engine.step(x, y)
    # the head's logits are rounded to bf16 in front of the other loss
    assert engine.last_dice.isnan() and torch.equal(loss, engine.last_ce) and abs(float(loss - ce)) <= 2 ** -8 * float(ce)
    assert float(engine.eval_step(x, y)[0]) == float(loss) != float(both[0])
    engine.loss = "ce_dice"
    engine.step(x, y)
    assert torch.equal(engine.last_ce, ce)


@pytest.mark.parametrize("amp", [True, False])
def test_the_engine_on_the_cpu(amp):
    x, y = _batch(40, (8, 8, 8), 1, "cpu")
    model = _model(40, 8, 1, "cpu")
    engine = TrainEngine(model, torch.optim.SGD(model.parameters(), lr=0.1), 40, "cpu", loss="ce", amp=amp)
    first = float(engine.step(x, y))
    for _ in range(3):
        last = float(engine.step(x, y))
    assert last == last and engine.last_dice.isnan()
    val, dice = engine.eval_step(x, y.to(torch.uint8))
    assert dice.shape == (1, 40) and float(val) == float(val) and first > 0
    with pytest.raises(ValueError, match="loss"):
        TrainEngine(model, torch.optim.SGD(model.parameters(), lr=0.1), 40, "cpu", loss="dice")


class _Exchanged:
    """A spatial context of one shard whose volume is processed with H (or W) exchanged with the depth."""

    size, dims, halo_channel = 1, [2], None

    def __init__(self, lead_swap):
        self.lead_swap = lead_swap

    def to_kernel_space(self, t, first_spatial=2):
        return t.transpose(first_spatial, first_spatial + self.lead_swap - 2)


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("axis", [3, 4])
def test_the_loss_of_a_volume_whose_axes_are_exchanged(axis, dev):
    n_classes = 40
    x, y = _batch(n_classes, (8, 16, 24) if dev == "cpu" else (16, 32, 24), 1, dev)
    results = []
    for spatial in (None, _Exchanged(axis)):
        model = _model(n_classes, 16, 1, dev)
        model.set_spatial(spatial)
        for m in model.modules():
            if isinstance(m, (Conv3d, ConvTranspose3d)):
                m.set_spatial(spatial)
        engine = TrainEngine(model, torch.optim.SGD(model.parameters(), lr=0.0), n_classes, dev, spatial=spatial,
                             class_weights=torch.linspace(0.5, 2.0, n_classes, device=dev), amp=dev == "cuda", loss="ce",
                             max_norm=1e9)
        loss = engine.step(x, y)
        grads = [p.grad.clone() for p in model.parameters()]
        val, dice = engine.eval_step(x, y)
        results.append((loss, grads, val, dice))
    (loss, grads, val, dice), (loss2, grads2, val2, dice2) = results
    # the exchanged volume's features against labels that were exchanged by hand: the same calls, to the bit
    labels = y.transpose(1, axis - 1).contiguous()
    head = model.up_list[-1].conv
    with torch.autocast(dev, dtype=torch.bfloat16, enabled=dev == "cuda"):
        features = model.features(x).permute(0, 2, 3, 4, 1)
        want = head_cross_entropy(features, head.weight, head.bias, labels, engine.class_weights)
        pred = head_predict(features, head.weight, head.bias)
    assert torch.equal(loss2, want)
    for p, g in zip(model.parameters(), torch.autograd.grad(want, list(model.parameters()))):
        assert torch.equal(p.grad, g)
    assert torch.equal(dice2, L.hard_dice_of_prediction(pred, labels, n_classes))
    if dev == "cpu":  # and in 32 bits the volume as it is gives the same
        assert abs(float(loss - loss2)) <= 1e-5 * float(loss) and abs(float(val - val2)) <= 1e-5 * float(val)
        for a, b in zip(grads, grads2):
            assert float((a - b).norm()) <= 1e-3 * float(a.norm()) + 1e-7


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_the_dice_of_a_prediction_over_shards(dev):
    _, labels = _batch(7, (6, 10, 8), 2, dev)
    labels[0, 0, 0, :3] = 9  # outside the classes
    pred = torch.where(torch.rand(labels.shape, device=dev) < 0.5, labels, 2).clamp(max=6)
    want = L.hard_dice_of_prediction(pred, labels, 7)
    cut = [slice(0, 4), slice(4, 10)]

    class Shard:
        size, lead_swap = 2, None

        def __init__(self, others=None):
            self.others = others

        def all_reduce_sum(self, t):
            self.sent = t.clone()
            if self.others is not None:
                t += self.others

    sent = []
    for c in cut:
        shard = Shard()
        L.hard_dice_of_prediction(pred[:, :, c], labels[:, :, c], 7, shard)
        sent.append(shard.sent)
    for c, others in zip(cut, reversed(sent)):
        assert torch.equal(L.hard_dice_of_prediction(pred[:, :, c], labels[:, :, c], 7, Shard(others)), want)


@pytest.mark.slow
def test_the_trainer_with_both_options_on_one_rank_and_on_two_shards(tmp_path):
    script = ROOT / "tests" / "helpers" / "rank_scripts" / "benchmark_tiny.py"
    runs = []
    for ranks in (1, 2):
        proc = torchrun_gloo(script, ranks, [str(tmp_path), str(ranks), "2", "{loss: ce, activation_bits: 8}"])
        assert proc.returncode == 0, proc.stdout[-3000:] + proc.stderr[-3000:]
        runs.append(results(proc.stdout))
    for key in ("epoch1", "epoch2"):
        a, b = ([float(v) for v in r[key][0].split()] for r in runs)
        # fp32-level agreement of the losses; hard Dice: a few argmax near-ties may flip
        assert abs(a[0] - b[0]) <= 5e-4 * a[0] and abs(a[1] - b[1]) <= 5e-4 * a[1] and abs(a[2] - b[2]) <= 5e-3, (key, a, b)


def test_configuration_keys(tmp_path):
    import yaml
    from scaffold_b200 import config as C

    def config(**kw):
        d = yaml.safe_load(C.default_config_path().read_text())
        d.update(base_run_dir=str(tmp_path), dataset_dir=str(tmp_path), fract_base_dir=str(tmp_path), **kw)
        return C.Config(d)

    assert config().activation_bits == 16 and config().loss == "ce_dice"
    cfg = config(activation_bits=8, loss="ce")
    assert cfg.activation_bits == 8 and cfg.loss == "ce"
    for bad in (dict(activation_bits=4), dict(activation_bits=True), dict(activation_bits="8"), dict(loss="dice")):
        with pytest.raises(ValueError):
            config(**bad)
