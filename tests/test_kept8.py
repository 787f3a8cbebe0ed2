"""The 8-bit copy of an activation: its format (CPU formula and CUDA kernel give the same bytes), its error and its
refusals."""
import math

import pytest
import torch

from scaffold_b200.ops import kept8 as k8
from scaffold_b200.ops.kept8 import Kept8, keep8, restore8

TYPES = [torch.bfloat16, torch.float16, torch.float32]
ON = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _values(n, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, generator=g) * torch.exp(2 * torch.randn((n + 99) // 100, generator=g)).repeat_interleave(100)[:n]
    return x.to(dtype)


def _oracle(x):
    """What the copy restores, element by element in exact arithmetic (Python integers and floats)."""
    out = []
    flat = x.double().reshape(-1).tolist()
    limit = torch.finfo(x.dtype).max
    for i in range(0, len(flat), 16):
        block = flat[i:i + 16]
        if not all(math.isfinite(v) for v in block):
            out += [math.nan] * len(block)
            continue
        most = max(abs(v) for v in block)
        e = -126
        while most >= math.ldexp(126.5, e):
            e += 1
        cap = 63 if math.ldexp(64, e) > limit else 127
        for v in block:
            q = round(math.ldexp(v, -e))  # Python rounds ties to even
            out.append(math.ldexp(max(-cap, min(cap, q)), e))
    return torch.tensor(out, dtype=torch.float64).view(x.shape)


@pytest.mark.parametrize("dev", ON)
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("n", [1, 15, 16, 17, 31, 4099, 40000])
def test_restored_values_are_the_definition(n, dtype, dev):
    x = _values(n, dtype, n)
    got = restore8(keep8(x.to(dev))).cpu()
    assert got.dtype == dtype and torch.equal(got.double(), _oracle(x))


@pytest.mark.parametrize("dev", ON)
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_borders_of_the_range(dtype, dev):
    """Zeros, ties, a block at the significand where the step doubles, the largest and the smallest numbers."""
    top, tiny = torch.finfo(dtype).max, torch.finfo(dtype).tiny
    rows = [[0.0] * 16, [-0.0] * 16, [126.0, 0.5, 1.5, 2.5, -0.5, -1.5], [126.5, 1.0, 3.0], [127.0, 1.0], [253.0, 1.0, 3.0],
            [top, -top, top / 2, top / 128, 1.0], [top * 0.49, 1.0], [tiny, -tiny], [tiny * 130, tiny, -tiny * 3],
            [1.0, 1e-6, -1e-3]]
    x = torch.zeros(len(rows), 16, dtype=torch.float64)
    for r, row in enumerate(rows):
        x[r, :len(row)] = torch.tensor(row, dtype=torch.float64)
    x = x.to(dtype)
    got = restore8(keep8(x.to(dev))).cpu()
    assert torch.isfinite(got).all() and torch.equal(got.double(), _oracle(x))


@pytest.mark.parametrize("dev", ON)
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_a_block_that_is_not_finite_comes_back_as_nan(bad, dtype, dev):
    x = _values(100, dtype)
    x[37] = bad
    got = restore8(keep8(x.to(dev))).cpu()
    want = _oracle(x)
    assert torch.equal(got.isnan(), want.isnan()) and got.isnan().sum() == 16 and got[32:48].isnan().all()
    assert torch.equal(got.double().nan_to_num(), want.nan_to_num())


@pytest.mark.parametrize("dev", ON)
def test_every_bf16_number_as_the_largest_of_its_block(dev):
    """The step is the smallest that holds the block, for each of the 65280 finite bf16 numbers."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16)
    most = bits.view(torch.bfloat16)
    most = most[most.isfinite()]
    x = torch.zeros(len(most), 16, dtype=torch.bfloat16)
    x[:, 3] = most
    x[:, 9] = most / 3
    got = restore8(keep8(x.to(dev))).cpu().double()
    big = most.double().abs()
    m, k = torch.frexp(big)
    e = torch.where(m * 128 < 126.5, k - 7, k - 6).clamp_min(-126)
    step = torch.ldexp(torch.ones_like(big), e)
    half = torch.where(64 * step > torch.finfo(torch.bfloat16).max, 0.75, 0.5) * step  # the top keeps 63 steps
    assert ((got[:, 3] - most.double()).abs() <= half).all()
    assert ((got[:, 9] - x[:, 9].double()).abs() <= half).all()
    assert got.isfinite().all()


@pytest.mark.parametrize("dev", ON)
def test_shapes_strides_and_views(dev):
    base = _values(2 * 3 * 4 * 5 * 16, torch.bfloat16).to(dev)
    plain = base.view(2, 3, 4, 5, 16)
    last = plain.permute(0, 4, 1, 2, 3)  # NCDHW over channels-last memory
    kept = keep8(last)
    assert kept.shape == last.shape and kept.numel() == last.numel() and kept.device == last.device
    got = restore8(kept)
    assert got.shape == last.shape and got.stride() == last.stride()
    assert torch.equal(got.permute(0, 2, 3, 4, 1), restore8(keep8(plain)))  # blocks follow the memory
    for view in (plain[:, :, 1:3], plain[..., 3:11], plain[:1].expand(4, -1, -1, -1, -1), base[1:], base[3:18]):
        assert torch.equal(restore8(keep8(view)), restore8(keep8(view.contiguous().clone())))
    assert restore8(keep8(base[:0])).shape == (0,)
    assert restore8(keep8(base[5])).shape == ()


def test_refusals():
    for bad in (torch.zeros(4, dtype=torch.float64), torch.zeros(4, dtype=torch.int8), torch.zeros(4, dtype=torch.complex64)):
        with pytest.raises(TypeError):
            keep8(bad)
    kept = keep8(torch.ones(40))
    with pytest.raises(TypeError):
        restore8(kept._replace(dtype=torch.float64))
    with pytest.raises(ValueError):
        restore8(kept._replace(shape=(64,)))
    with pytest.raises(ValueError):
        restore8(Kept8(kept.data.float(), (40,), (1,), torch.float32))
    with pytest.raises(ValueError):
        restore8(kept._replace(shape=(4, 10), stride=(1, 1)))


def test_no_gradient_flows_through_the_copy():
    x = torch.ones(20, requires_grad=True)
    assert not restore8(keep8(x)).requires_grad


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_the_kernels_write_what_the_formula_writes(dtype):
    x = _values(100003, dtype, 5)
    x[500], x[9000] = math.inf, math.nan
    a, b = keep8(x), keep8(x.cuda())
    assert torch.equal(a.data, b.data.cpu())


@pytest.mark.gpu
def test_nothing_is_written_beside_the_copy():
    from scaffold_b200.ops import _lib
    n = 1003
    x = _values(n, torch.bfloat16).cuda()
    buf = torch.full((k8.kept_bytes(n) + 512,), 0xA5, dtype=torch.uint8, device="cuda")
    _lib.check(_lib.lib().sb_keep8(x.data_ptr(), 0, n, buf.data_ptr() + 256, _lib.stream_ptr()), "sb_keep8")
    out = torch.full((n + 256,), -7.0, dtype=torch.bfloat16, device="cuda")
    _lib.check(_lib.lib().sb_restore8(buf.data_ptr() + 256, 0, n, out.data_ptr() + 256, _lib.stream_ptr()), "sb_restore8")
    assert (buf[:256] == 0xA5).all() and (buf[-256:] == 0xA5).all()
    assert (out[:128] == -7).all() and (out[128 + n:] == -7).all()
    assert torch.equal(out[128:128 + n], restore8(keep8(x)))


@pytest.mark.gpu
def test_streams_and_graphs():
    """A copy made on another stream, and made and read inside a graph that is replayed on new values."""
    x = _values(5000, torch.bfloat16, 1).cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = restore8(keep8(x))
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, restore8(keep8(x)))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = restore8(keep8(x))
    for seed in (2, 3):
        x.copy_(_values(5000, torch.bfloat16, seed))
        graph.replay()
        assert torch.equal(out, restore8(keep8(x)))
