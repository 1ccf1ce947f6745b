"""Lengths that change between decode calls without a kernel in between (a copy from pinned
memory): the split and the merge kernel of a call cut every sequence alike."""
import pytest
import torch

from custom_inference_engine_b200 import native

pytestmark = pytest.mark.gpu
PAGE, D, B, HKV = 16, 64, 16, 2
# per step: all pages in one split, a page more or less per split, many splits
STEPS = [40, 1500, 63, 64, 511, 512, 2900, 1023, 1024, 15, 16, 2047]


@pytest.mark.parametrize("bits", [8, 16])
def test_lengths_copied_between_calls(cuda_device, bits):
    native.load_ops()
    ops, dev = torch.ops.inference, cuda_device
    g = torch.Generator().manual_seed(bits)
    pages = -(-(max(STEPS) + 2 * B) // PAGE)
    n_pages = B * pages + 1
    bt = torch.zeros(B + 1, n_pages, dtype=torch.long)
    bt[1:, :pages] = (torch.randperm(n_pages - 1, generator=g) + 1).view(B, pages)
    bt, slots = bt.to(dev), torch.arange(1, B + 1, device=dev)
    shape = (n_pages, HKV, PAGE, D)
    if bits == 8:
        pool = [torch.randint(-127, 128, shape, generator=g, dtype=torch.int8) for _ in range(2)]
        pool.append(torch.full((n_pages, 2, HKV), 2.0 ** -6))
    else:
        pool = [torch.randn(shape, generator=g).half() for _ in range(2)]
    x = torch.randn(1, B, 18 * D, generator=g).half().to(dev)
    angle = torch.rand(1, B, D, generator=g)
    cos, sin = angle.cos().half().to(dev), angle.sin().half().to(dev)
    host = [torch.tensor([0] + [n + i for i in range(B)]).pin_memory() for n in STEPS]
    lens = torch.zeros(B + 1, dtype=torch.long, device=dev)
    one, update, attend = (
        (ops.rope_kv_q8_decode_attention, ops.rope_kv_q8_decode_update, ops.gqa_decode_attention_q8)
        if bits == 8 else
        (ops.rope_kv_decode_attention, ops.rope_kv_decode_update, ops.gqa_decode_attention))
    a, b = [t.to(dev) for t in pool], [t.to(dev) for t in pool]
    got = []
    for n in host * 8:
        lens.copy_(n, non_blocking=True)
        got.append(one(x, cos, sin, *a, lens, slots, bt))
    for i, n in enumerate(host * 8):
        lens.copy_(n)
        torch.cuda.synchronize()
        q = update(x, cos, sin, *b, lens, slots, bt)
        assert torch.equal(got[i], attend(q, *b, lens[slots] + 1, slots, bt)), (i, n[1])
    for s, t in zip(a, b):
        assert torch.equal(s, t)
