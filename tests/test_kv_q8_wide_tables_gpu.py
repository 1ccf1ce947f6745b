"""Block tables that are columns of a wider table: a length beyond a row's pages is refused,
and does not run on into the neighbouring columns."""
import pytest
import torch

from custom_inference_engine_b200 import native

pytestmark = pytest.mark.gpu
PAGE, D, HKV, N = 16, 64, 2, 6


@pytest.mark.parametrize("dtype", [torch.int64, torch.int32])
@pytest.mark.parametrize("left", [True, False])
def test_columns_of_a_wider_table(cuda_device, dtype, left):
    native.load_ops()
    ops, dev = torch.ops.inference, cuda_device
    g = torch.Generator().manual_seed(3)
    wide = torch.randint(1, N, (3, 2 * N), generator=g).to(dev, dtype)
    bt = wide[:, :N] if left else wide[:, N:]
    bt[1, :3], bt[2, :3] = (torch.tensor(x, device=dev, dtype=dtype) for x in ([1, 2, 3], [4, 5, 0]))
    k, v = (torch.randint(-127, 128, (N, HKV, PAGE, D), generator=g, dtype=torch.int8).to(dev)
            for _ in range(2))
    s = torch.full((N, 2, HKV), 0.25, device=dev)
    slots = torch.tensor([1, 2], device=dev)
    t = lambda *x: torch.tensor(x, device=dev)
    q = torch.randn(1, 2, 14, D, generator=g).half().to(dev)
    new = torch.randn(1, 2, HKV, D, generator=g).half().to(dev)
    qkv = torch.randn(1, 2, 18 * D, generator=g).half().to(dev)
    cos = torch.ones(1, 2, D, device=dev).half()
    native.device_errors(0, clear=True)
    # good lengths: the results of a table of its own
    own = bt.contiguous()
    lens, per_slot = t(40, 20), t(0, 40, 20)
    results = []
    for table in (bt, own):
        a, b, c = (x.clone() for x in (k, v, s))
        out = [torch.zeros(a.shape, device=dev).half() for _ in range(2)]
        o = [ops.gqa_decode_attention_q8(q, a, b, c, lens, slots, table),
             ops.rope_kv_q8_decode_attention(qkv, cos, cos, a, b, c, per_slot, slots, table)]
        ops.kv_q8_mixed_update(a, b, c, t(0, 1, 2), t(41, 21), slots, table, new, new)
        ops.kv_q8_read(a, b, c, None, t(42, 22), slots, table, *out)
        results.append(o + [a, b, c] + out)
    for x, y in zip(*results):
        assert torch.equal(x, y)
    assert native.device_errors(0, clear=True) == 0
    # one row more than the pages of a row hold
    before = [x.clone() for x in (k, v, s)]
    full, per_slot = t(N * PAGE, N * PAGE), t(0, N * PAGE, N * PAGE)
    out = [torch.zeros(k.shape, device=dev).half() for _ in range(2)]
    for call in (lambda: ops.kv_q8_decode_update(k, v, s, per_slot, slots, bt, new, new),
                 lambda: ops.kv_q8_mixed_update(k, v, s, t(0, 1, 2), full, slots, bt, new, new),
                 lambda: ops.rope_kv_q8_decode_attention(qkv, cos, cos, k, v, s, per_slot, slots, bt),
                 lambda: ops.gqa_decode_attention_q8(q, k, v, s, full + 1, slots, bt),
                 lambda: ops.kv_q8_read(k, v, s, None, full + 1, slots, bt, *out)):
        call()
        assert native.device_errors(0, clear=True) == 1 << 1  # CIE_DEVERR_BAD_LENGTH
    for x, y in zip((k, v, s), before):
        assert torch.equal(x, y)
    whole = ops.gqa_decode_attention_q8(q, k, v, s, full, slots, bt)
    assert native.device_errors(0, clear=True) == 0
    # a refused length counts as a full row, however large it is
    for n in (N * PAGE + 1, 2 ** 40, 2 ** 63 - 1):
        assert torch.equal(ops.gqa_decode_attention_q8(q, k, v, s, t(n, n), slots, bt), whole)
        assert native.device_errors(0, clear=True) == 1 << 1
