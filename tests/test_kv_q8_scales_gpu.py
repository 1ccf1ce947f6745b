"""8-bit pages whose stored scales are no power of two (a pool that another program filled),
and pages whose stored scale is no scale at all."""
import math

import pytest
import torch

from custom_inference_engine_b200 import native
from oracle import kv_q8 as ref

pytestmark = pytest.mark.gpu
PAGE, D, HKV = 16, 64, 2
SCALES = [0.75, 2.0 ** -30, 3.0, 1.0 / 3, 2.0 ** -24, 0.1, 700.0, 1.1 * 2.0 ** -20, 1e-39, 5e4]


@pytest.fixture(autouse=True)
def _no_device_errors(cuda_device):
    native.device_errors(0, clear=True)
    yield
    assert native.device_errors(0, clear=True) == 0


@pytest.fixture(scope="module")
def ops(cuda_device):
    native.load_ops()
    return torch.ops.inference


def _pool(dev, seed, scales=SCALES):
    """A slot for every scale; its page holds ten rows under that scale."""
    g = torch.Generator().manual_seed(seed)
    n = len(scales)
    k, v = (torch.randint(-127, 128, (n + 1, HKV, PAGE, D), generator=g, dtype=torch.int8)
            for _ in range(2))
    s = torch.ones(n + 1, 2, HKV)
    s[1:, 0] = torch.tensor(scales)[:, None]
    s[1:, 1] = torch.tensor(scales).roll(3)[:, None]
    bt = torch.zeros(n + 1, n + 1, dtype=torch.long)
    bt[:, 0] = torch.arange(n + 1)
    lens = torch.full((n + 1,), 10)
    slots = torch.arange(1, n + 1)
    return [t.to(dev) for t in (k, v, s, lens, slots, bt)], g


@pytest.mark.parametrize("mixed", [False, True])
@pytest.mark.parametrize("size", [1e-4, 1.0, 90.0, 2000.0])
def test_update_keeps_the_larger_of_the_two_scales(ops, cuda_device, size, mixed):
    """max(stored scale, 2^e): the stored scale stays as it is where the new rows fit it, and
    the older codes then stay too; else they are rounded once to the new power of two."""
    (k, v, s, lens, slots, bt), g = _pool(cuda_device, 1)
    n = slots.shape[0]
    new = (torch.randn(2, 1, n, HKV, D, generator=g) * size).half()
    want = [t.cpu().clone() for t in (k, v, s)]
    ref.update(*want, [(i + 1, 10, i, 1) for i in range(n)], bt.cpu(), new[0, 0], new[1, 0])
    rows = [t.to(cuda_device) for t in new]
    if mixed:
        cu = torch.arange(n + 1, device=cuda_device)
        ops.kv_q8_mixed_update(k, v, s, cu, lens[1:].contiguous(), slots, bt, *rows)
    else:
        ops.kv_q8_decode_update(k, v, s, lens, slots, bt, *rows)
    for got, w in zip((s, k, v), (want[2], want[0], want[1])):
        assert torch.equal(got.cpu(), w)


def test_codes_at_the_borders_of_rounding(ops, cuda_device):
    """x / scale is rounded to the nearest whole number by its exact value, ties to even,
    also where its fp32 quotient lies on a tie that the exact one misses."""
    dev = cuda_device
    scales = [0.75, 1.0 / 3, 0.1, 3.0, 0.7, 1.3]
    (k, v, s, lens, slots, bt), _ = _pool(dev, 2, scales)
    s[1:, 1] = s[1:, 0]
    n = len(scales)
    half = torch.arange(D).double() + 0.5                    # the ties 0.5 .. 63.5
    x = (half[None] * s[1:, 0, 0].double().cpu()[:, None]).half()
    new = x[None, :, None].expand(1, n, HKV, D).contiguous()
    want = [t.cpu().clone() for t in (k, v, s)]
    ref.update(*want, [(i + 1, 10, i, 1) for i in range(n)], bt.cpu(), new[0], new[0])
    ops.kv_q8_decode_update(k, v, s, lens, slots, bt, new.to(dev), new.to(dev))
    for got, w in zip((s, k, v), (want[2], want[0], want[1])):
        assert torch.equal(got.cpu(), w)


def test_read_and_attend(ops, cuda_device):
    scales = [x for x in SCALES if 127 * x < 65504]          # (read back holds fp16)
    (k, v, s, _, slots, bt), g = _pool(cuda_device, 3, scales)
    lens = torch.tensor([1 + i for i in range(len(scales))], device=cuda_device)
    out = [torch.full(k.shape, 7.5, device=cuda_device).half() for _ in range(2)]
    want = [t.cpu().clone() for t in out]
    ref.read(k.cpu(), v.cpu(), s.cpu(), torch.zeros_like(lens), lens, slots, bt.cpu(), *want)
    ops.kv_q8_read(k, v, s, None, lens, slots, bt, *out)
    for a, b in zip(out, want):
        assert torch.equal(a.cpu(), b)
    s[:, 0].clamp_(max=0.75)                                 # scores of a size that varies
    q = (torch.randn(1, len(scales), 14, D, generator=g) / 16).half().to(cuda_device)
    args = (q, k, v, s, lens, slots, bt)
    o, tol = ref.decode_attention(*args)
    assert ((ops.gqa_decode_attention_q8(*args).double() - o).abs() <= tol).all()


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf, -0.5])
def test_a_stored_scale_that_is_none(ops, cuda_device, bad):
    """The rows under it hold no values: they become 0, and an error bit says so. A first row
    of a page does not look at the scale, and a scale of 0 (a new pool's) is no error."""
    dev = cuda_device
    (k, v, s, lens, slots, bt), g = _pool(dev, 4, [0.5, 0.5, 0.0, 0.5])
    s[1], s[2], s[3] = bad, bad, 0.0
    lens[2] = 0
    new = torch.randn(1, 4, HKV, D, generator=g).half()
    before = [t.cpu().clone() for t in (k, v, s)]
    ops.kv_q8_decode_update(k, v, s, lens, slots, bt, new.to(dev), new.to(dev))
    assert native.device_errors(0, clear=True) == 1 << 7  # CIE_DEVERR_BAD_SCALE
    before[2][1], before[2][2] = 0.0, 0.0
    ref.update(*before, [(i + 1, int(lens[i + 1]), i, 1) for i in range(4)], bt.cpu(), new[0],
               new[0])
    assert k[1, :, :10].eq(0).all() and k[3, :, :10].eq(0).all()
    for got, w in zip((s, k, v), (before[2], before[0], before[1])):
        assert torch.equal(got.cpu(), w)
    lens[2] = 11
    ops.kv_q8_decode_update(k, v, s, lens, slots, bt, new.to(dev), new.to(dev))
    assert native.device_errors(0, clear=True) == 0
