"""The 8-bit KV pool (quantised writes, read back, decode attention) against its
definition in float64 (``oracle/kv_q8.py``).

Codes and scales are exact: a scale is a power of two, so x / scale is exact and
its rounding has one answer. With the rotary embedding the same holds for the rows
rotated in fp32 operation by operation. Attention is held to a bound derived from
the kernel's roundings in ``oracle.kv_q8.decode_attention``.
"""
import math

import pytest
import torch

from custom_inference_engine_b200 import cabi, native
from oracle import kv_q8 as ref

pytestmark = pytest.mark.gpu
PAGE, D = 16, 64


@pytest.fixture(autouse=True)
def _no_device_errors(cuda_device):
    native.device_errors(0, clear=True)
    yield
    assert native.device_errors(0, clear=True) == 0


@pytest.fixture(scope="module")
def ops(cuda_device):
    native.load_ops()
    return torch.ops.inference


def _pool(lens, hkv, seed, dev, table=torch.int64, extra=3):
    """Pools of codes already there, scales that are powers of two, scattered pages."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // PAGE) for n in lens]
    n_pages = sum(need) + 1 + extra
    perm = torch.randperm(n_pages - 1, generator=g) + 1
    bt = torch.zeros(len(lens) + 1, n_pages, dtype=table)
    at = 0
    for s, n in enumerate(need):
        bt[s + 1, :n] = perm[at:at + n]
        at += n
    k = torch.randint(-127, 128, (n_pages, hkv, PAGE, D), generator=g, dtype=torch.int8)
    v = torch.randint(-127, 128, (n_pages, hkv, PAGE, D), generator=g, dtype=torch.int8)
    scales = torch.exp2(torch.randint(-8, -2, (n_pages, 2, hkv), generator=g).float())
    return [t.to(dev) for t in (k, v, scales, bt)], g


def _rows(T, hq, hkv, g, dev, big=1.0):
    """A fused projection with rows of very different size."""
    x = torch.randn(1, T, hq + 2 * hkv, D, generator=g) * big
    x = x * torch.exp2(torch.randint(-6, 5, (1, T, 1, 1), generator=g).float())
    x[..., 5] *= 8
    return x.half().to(dev)


def _rotary(pos, dev):
    inv = 1.0 / (1e6 ** (torch.arange(0, D, 2, dtype=torch.float64) / D))
    a = pos.double()[:, None] * inv
    a = torch.cat((a, a), -1)
    return a.cos().half()[None].to(dev), a.sin().half()[None].to(dev)


def _check_pools(got, want, name):
    for a, b, what in zip(got, want, ("k codes", "v codes", "scales")):
        assert torch.equal(a.cpu(), b), (name, what)


@pytest.mark.parametrize("hkv", [1, 2, 3, 4])
@pytest.mark.parametrize("table", [torch.int64, torch.int32])
@pytest.mark.parametrize("rope", [False, True])
def test_decode_update(ops, cuda_device, hkv, table, rope):
    dev = cuda_device
    hist = [0, 1, 15, 16, 17, 31, 40, 100, 5, 2000]
    B = len(hist)
    (k, v, s, bt), g = _pool([h + 1 for h in hist], hkv, 3 + hkv, dev, table)
    lens = torch.tensor([7] + hist, device=dev)
    slots = torch.arange(1, B + 1, device=dev).flip(0).contiguous()
    x = _rows(B, 7 * hkv, hkv, g, dev)
    qkv = x.reshape(1, B, -1)
    pos = lens[slots].cpu()
    cos, sin = _rotary(pos, dev)
    kn, vn = x[:, :, 7 * hkv:8 * hkv], x[:, :, 8 * hkv:]
    want = [t.cpu().clone() for t in (k, v, s)]
    rows_k = ref.rope_fp32(kn.cpu(), cos.cpu(), sin.cpu())[0] if rope else kn[0].cpu()
    chunks = [(int(slots[i]), int(pos[i]), i, 1) for i in range(B)]
    ref.update(*want, chunks, bt.cpu(), rows_k, vn[0].cpu())
    if rope:
        q = ops.rope_kv_q8_decode_update(qkv, cos, sin, k, v, s, lens, slots, bt)
        q32 = ref.rope_fp32(x[:, :, :7 * hkv].cpu(), cos.cpu(), sin.cpu())
        assert torch.equal(q.cpu(), q32.half())
    else:
        ops.kv_q8_decode_update(k, v, s, lens, slots, bt, kn, vn)
    _check_pools((k, v, s), want, "op")
    # a second write of the same rows changes nothing (their page already holds them)
    if not rope:
        cabi.kv_q8_decode_update(k, v, s, lens, slots, bt, kn, vn)
        _check_pools((k, v, s), want, "again")


CHUNKS = {
    "one token": ([0], [1], 0),
    "page borders": ([0, 15, 16, 1, 8, 0, 31], [16, 1, 1, 15, 9, 33, 2], 0),
    "ragged, decode rows, empty, padding": ([5, 0, 16, 1000, 77, 3], [1, 40, 0, 300, 1, 17], 21),
    "long": ([0, 513], [700, 65], 3),
}


@pytest.mark.parametrize("name", CHUNKS)
@pytest.mark.parametrize("hkv,table", [(2, torch.int64), (1, torch.int32), (4, torch.int64)])
@pytest.mark.parametrize("rope", [False, True])
def test_mixed_update(ops, cuda_device, name, hkv, table, rope):
    dev = cuda_device
    hist, n, pad = CHUNKS[name]
    B, T = len(hist), sum(n) + pad
    (k, v, s, bt), g = _pool([h + c for h, c in zip(hist, n)], hkv, len(name) + hkv, dev, table)
    cu = [0]
    for c in n:
        cu.append(cu[-1] + c)
    # two absent sequences on the padding slot, as a captured pass has them
    cu_t = torch.tensor(cu + [cu[-1]] * 2, device=dev)
    kv_lens = torch.tensor(hist + [0, 0], device=dev)
    slots = torch.tensor(list(range(1, B + 1)) + [0, 0], device=dev)
    x = _rows(T, 7 * hkv, hkv, g, dev)
    pos = torch.cat([torch.arange(h, h + c) for h, c in zip(hist, n)] + [torch.zeros(pad)])
    cos, sin = _rotary(pos, dev)
    kn, vn = x[:, :, 7 * hkv:8 * hkv], x[:, :, 8 * hkv:]
    want = [t.cpu().clone() for t in (k, v, s)]
    rows_k = ref.rope_fp32(kn.cpu(), cos.cpu(), sin.cpu())[0] if rope else kn[0].cpu()
    ref.update(*want, [(b + 1, hist[b], cu[b], n[b]) for b in range(B)], bt.cpu(), rows_k,
               vn[0].cpu())
    if rope:
        q = ops.rope_kv_q8_mixed_update(x.reshape(1, T, -1), cos, sin, k, v, s, cu_t, kv_lens,
                                        slots, bt)
        q32 = ref.rope_fp32(x[:, :, :7 * hkv].cpu(), cos.cpu(), sin.cpu())
        assert torch.equal(q.cpu(), q32.half())
    else:
        ops.kv_q8_mixed_update(k, v, s, cu_t, kv_lens, slots, bt, kn, vn)
    _check_pools((k, v, s), want, name)


def test_rotated_q_against_64_bits(ops, cuda_device):
    """q is rotated in fp32 (three roundings of at most 2^-24) and rounded to fp16 once."""
    dev = cuda_device
    (k, v, s, bt), g = _pool([40000], 2, 1, dev)
    x = _rows(4, 14, 2, g, dev)
    pos = torch.tensor([39996, 39997, 39998, 39999])
    cos, sin = _rotary(pos, dev)
    q = ops.rope_kv_q8_mixed_update(x.reshape(1, 4, -1), cos, sin, k, v, s,
                                    torch.tensor([0, 4], device=dev),
                                    torch.tensor([39996], device=dev),
                                    torch.tensor([1], device=dev), bt)
    y, c, sn = x[:, :, :14].double(), cos.double().unsqueeze(2), sin.double().unsqueeze(2)
    rot = torch.cat((-y[..., 32:], y[..., :32]), -1)
    exact = y * c + rot * sn
    tol = 2.0 ** -11 * exact.abs() + 3 * 2.0 ** -24 * ((y * c).abs() + (rot * sn).abs()) + 2.0 ** -25
    assert ((q.double() - exact).abs() <= tol).all()


@pytest.mark.parametrize("offset,stride", [(0, 0), (1, 3), (4, 2)])
def test_rows_at_any_alignment(ops, cuda_device, offset, stride):
    """New rows as views that start anywhere and lie any distance apart."""
    dev = cuda_device
    (k, v, s, bt), g = _pool([60], 2, 9, dev)
    buf = torch.randn(50 * (4 * D + stride) + offset + 8, generator=g).half().to(dev)
    row = 4 * D + stride
    kn = buf[offset:].as_strided((1, 50, 2, D), (0, row, D, 1))
    vn = buf[offset + 2 * D:].as_strided((1, 50, 2, D), (0, row, D, 1))
    want = [t.cpu().clone() for t in (k, v, s)]
    ref.update(*want, [(1, 7, 0, 50)], bt.cpu(), kn[0].cpu(), vn[0].cpu())
    ops.kv_q8_mixed_update(k, v, s, torch.tensor([0, 50], device=dev),
                           torch.tensor([7], device=dev), torch.tensor([1], device=dev), bt,
                           kn, vn)
    _check_pools((k, v, s), want, "strided")


def test_combined_pool(ops, cuda_device):
    """K and V of a page side by side in one allocation (strided views), as the fp16
    entry points allow."""
    dev = cuda_device
    (k, v, s, bt), g = _pool([33, 47], 2, 21, dev)
    both = torch.zeros(k.shape[0], 2, 2, PAGE, D, dtype=torch.int8, device=dev)
    both[:, 0], both[:, 1] = k, v
    kn = torch.randn(1, 2, 2, D, generator=g).half().to(dev)
    vn = torch.randn(1, 2, 2, D, generator=g).half().to(dev)
    args = (torch.tensor([0, 32, 46], device=dev), torch.tensor([1, 2], device=dev), bt, kn, vn)
    s2 = s.clone()
    ops.kv_q8_decode_update(both[:, 0], both[:, 1], s2, *args)
    ops.kv_q8_decode_update(k, v, s, *args)
    assert torch.equal(both[:, 0], k) and torch.equal(both[:, 1], v) and torch.equal(s, s2)
    lens = torch.tensor([33, 47], device=dev)
    q = torch.randn(1, 2, 14, D, generator=g).half().to(dev)
    a = ops.gqa_decode_attention_q8(q, both[:, 0], both[:, 1], s, lens, args[1], bt)
    assert torch.equal(a, ops.gqa_decode_attention_q8(q, k, v, s, lens, args[1], bt))


def test_growing_page_stays_within_one_step(ops, cuda_device):
    """A page filled row by row, every row larger than the last: the error of every
    value is at most one step of the final scale (half a step when written at once),
    and the scale does not depend on how the page was filled."""
    dev = cuda_device
    g = torch.Generator().manual_seed(2)
    x = torch.randn(1, PAGE, 2, D, generator=g)
    x = (x * torch.exp2(torch.arange(PAGE).float() / 2 - 4).view(1, -1, 1, 1)).half().to(dev)
    bt = torch.tensor([[0, 0], [1, 0]], device=dev)
    slot = torch.tensor([1], device=dev)
    pools = []
    for at_once in (False, True):
        k = torch.full((2, 2, PAGE, D), 77, dtype=torch.int8, device=dev)
        v, s = k.clone(), torch.full((2, 2, 2), 32.0, device=dev)
        if at_once:
            ops.kv_q8_mixed_update(k, v, s, torch.tensor([0, PAGE], device=dev),
                                   torch.tensor([0], device=dev), slot, bt, x, x)
        else:
            for i in range(PAGE):
                ops.kv_q8_decode_update(k, v, s, torch.tensor([0, i], device=dev), slot, bt,
                                        x[:, i:i + 1], x[:, i:i + 1])
        assert torch.equal(k[1], v[1]) and k[0].eq(77).all() and s[0].eq(32).all()
        err = (k[1].double() * s[1, 0].double().view(2, 1, 1) - x[0].transpose(0, 1).double()).abs()
        steps = err / s[1, 0].double().view(2, 1, 1)
        assert steps.max().item() <= (0.5 if at_once else 1.0)
        pools.append(s[1].clone())
    assert torch.equal(*pools)


def test_the_last_of_several_rows_for_one_slot_wins(ops, cuda_device):
    """Padding rows of a decode batch share slot 0; what its page holds afterwards is
    the last row's, and every other page is untouched by them."""
    dev = cuda_device
    (k, v, s, bt), g = _pool([20, 5], 2, 4, dev)
    slots = torch.tensor([0, 1, 0, 2, 0, 0], device=dev)
    lens = torch.tensor([0, 19, 4], device=dev)
    kn = torch.randn(1, 6, 2, D, generator=g).half().to(dev)
    vn = torch.randn(1, 6, 2, D, generator=g).half().to(dev)
    want = [t.cpu().clone() for t in (k, v, s)]
    ref.update(*want, [(0, 0, 5, 1), (1, 19, 1, 1), (2, 4, 3, 1)], bt.cpu(), kn[0].cpu(),
               vn[0].cpu())
    ops.kv_q8_decode_update(k, v, s, lens, slots, bt, kn, vn)
    _check_pools((k, v, s), want, "decode")
    # the same of a mixed pass: sequence 2 repeats sequence 0's slot, sequence 3 is empty
    slots = torch.tensor([1, 2, 1, 1], device=dev)
    cu = torch.tensor([0, 3, 4, 6, 6], device=dev)
    kvl = torch.tensor([16, 4, 17, 0], device=dev)
    ref.update(*want, [(2, 4, 3, 1), (1, 17, 4, 2)], bt.cpu(), kn[0].cpu(), vn[0].cpu())
    ops.kv_q8_mixed_update(k, v, s, cu, kvl, slots, bt, kn, vn)
    _check_pools((k, v, s), want, "mixed")


def test_extreme_and_non_finite_values(ops, cuda_device):
    dev = cuda_device
    k = torch.zeros(2, 1, PAGE, D, dtype=torch.int8, device=dev)
    v, s = k.clone(), torch.zeros(2, 2, 1, device=dev)
    bt = torch.tensor([[0, 0], [1, 0]], device=dev)
    args = (torch.tensor([0, 3], device=dev), torch.tensor([0], device=dev),
            torch.tensor([1], device=dev), bt)
    x = torch.zeros(1, 3, 1, D).half()
    x[0, 0, 0, :4] = torch.tensor([65504.0, -65504.0, 2.0 ** -24, 65024.0])
    ops.kv_q8_mixed_update(k, v, s, *args, x.to(dev), torch.zeros_like(x).to(dev))
    assert s[1, 0, 0] == 512 and s[1, 1, 0] == 2.0 ** -24
    assert k[1, 0, 0, :4].tolist() == [127, -127, 0, 127] and v.eq(0).all()
    x[0, 1, 0, :3] = torch.tensor([math.inf, -math.inf, math.nan])
    x[0, 0, 0, 0] = math.nan
    ops.kv_q8_mixed_update(k, v, s, *args, x.to(dev), torch.zeros_like(x).to(dev))
    assert native.device_errors(0, clear=True) == 1 << 6  # CIE_DEVERR_NONFINITE
    assert k[1, 0, 1, :3].tolist() == [127, -127, 0] and k[1, 0, 0, 0] == 0
    # all of a page's rows the smallest subnormal: exact
    x = torch.full((1, 3, 1, D), 2.0 ** -24).half().to(dev)
    ops.kv_q8_mixed_update(k, v, s, *args, x, x)
    out = [torch.zeros(2, 1, PAGE, D, device=dev).half() for _ in range(2)]
    ops.kv_q8_read(k, v, s, None, torch.tensor([3], device=dev), torch.tensor([1], device=dev),
                   bt, *out)
    assert torch.equal(out[0][1, :, :3], x[0].transpose(0, 1))


@pytest.mark.parametrize("hkv,table", [(1, torch.int32), (2, torch.int64), (3, torch.int64),
                                       (4, torch.int32)])
def test_read(ops, cuda_device, hkv, table):
    """Positions [starts, lens): whole pages, parts of a page, nothing; all other
    values of the output pool stay."""
    dev = cuda_device
    lens = [0, 1, 16, 17, 333, 40, 64, 100]
    starts = [0, 0, 0, 16, 18, 39, 64, 0]
    (k, v, s, bt), _ = _pool(lens, hkv, hkv, dev, table)
    t = lambda x: torch.tensor(x, device=dev)
    slots = torch.arange(1, len(lens) + 1, device=dev)
    out = [torch.full(k.shape, 7.5, device=dev).half() for _ in range(2)]
    want = [x.cpu().clone() for x in out]
    ref.read(k.cpu(), v.cpu(), s.cpu(), t(starts), t(lens), slots, bt.cpu(), *want)
    ops.kv_q8_read(k, v, s, t(starts), t(lens), slots, bt, *out)
    for a, b in zip(out, want):
        assert torch.equal(a.cpu(), b)
    # into a combined fp16 pool, from the start
    both = torch.full((k.shape[0], 2, *k.shape[1:]), 7.5, device=dev).half()
    ref.read(k.cpu(), v.cpu(), s.cpu(), t([0] * 8), t(lens), slots, bt.cpu(), *want)
    cabi.kv_q8_read(k, v, s, None, t(lens), slots, bt, both[:, 0], both[:, 1])
    assert torch.equal(both[:, 0].cpu(), want[0]) and torch.equal(both[:, 1].cpu(), want[1])


def _attend(dev, lens, hkv, group, seed, table=torch.int64):
    (k, v, s, bt), g = _pool(lens, hkv, seed, dev, table)
    q = torch.randn(1, len(lens), hkv * group, D, generator=g).half().to(dev)
    return q, k, v, s, torch.tensor(lens, device=dev), torch.arange(1, len(lens) + 1, device=dev), bt


def _near(o, args):
    want, tol = ref.decode_attention(*args)
    err = (o.double() - want).abs()
    assert (err <= tol).all(), (err / tol.clamp_min(1e-30)).max().item()


@pytest.mark.parametrize("lens", [[1], [0], [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65],
                                  [511], [4096, 5, 0, 1000], [777] * 40, [20000]],
                         ids=lambda x: f"{len(x)}x{max(x)}")
@pytest.mark.parametrize("hkv,group", [(2, 7), (1, 8), (4, 1), (4, 8), (2, 3)])
def test_decode_attention(ops, cuda_device, lens, hkv, group):
    args = _attend(cuda_device, lens, hkv, group, len(lens) + hkv,
                   torch.int32 if group == 3 else torch.int64)
    _near(ops.gqa_decode_attention_q8(*args), args)


@pytest.mark.parametrize("splits", [1, 2, 7, 8, 9, 64, 300])
def test_decode_attention_any_split_count(cuda_device, splits):
    args = _attend(cuda_device, [1, 0, 100, 1023, 4097, 64], 2, 7, splits)
    _near(cabi.decode_attention_q8(*args, num_splits=splits), args)


def test_decode_attention_wide_range_of_scales(ops, cuda_device):
    """Page scales from 2^-24 to 2^9 next to one another: no page's share is lost in
    the range of fp16."""
    args = list(_attend(cuda_device, [1600, 90], 2, 7, 77))
    s = args[3]
    g = torch.Generator().manual_seed(5)
    s[:, 1] = torch.exp2(torch.randint(-24, 10, s[:, 1].shape, generator=g).float()).to(s.device)
    s[:, 0] = torch.exp2(torch.randint(-24, -4, s[:, 0].shape, generator=g).float()).to(s.device)
    _near(ops.gqa_decode_attention_q8(*args), args)
    s[:, 1] = 2.0 ** -24
    _near(ops.gqa_decode_attention_q8(*args), args)


def test_rows_behind_the_end_do_not_matter(ops, cuda_device):
    """Codes behind a sequence's last row, and pages of no sequence with any scale."""
    args = list(_attend(cuda_device, [5, 33, 100], 2, 7, 8))
    want = ops.gqa_decode_attention_q8(*args)
    q, k, v, s, lens, slots, bt = args
    for b, n in enumerate(lens.tolist()):
        page = int(bt[b + 1, (n - 1) // PAGE])
        k[page, :, n % PAGE:] = 127
        v[page, :, n % PAGE:] = -128
    used = torch.zeros(k.shape[0], dtype=torch.bool)
    for b, n in enumerate(lens.tolist()):
        used[bt[b + 1, :-(-n // PAGE)].long().cpu()] = True
    s[~used.to(s.device)] = math.nan
    assert torch.equal(ops.gqa_decode_attention_q8(*args), want)


def test_bad_slots_pages_and_lengths_set_error_bits(ops, cuda_device):
    """Out-of-range ids and lengths are refused on the device, never followed."""
    dev = cuda_device
    (k, v, s, bt), g = _pool([40, 40], 2, 1, dev)
    q = torch.randn(1, 2, 14, D, generator=g).half().to(dev)
    new = torch.randn(1, 2, 2, D, generator=g).half().to(dev)
    t = lambda *x: torch.tensor(x, device=dev)
    out = [torch.zeros_like(k, dtype=torch.half) for _ in range(2)]
    before = [x.clone() for x in (k, v, s)]
    good_bt, n_pages = bt.clone(), k.shape[0]

    def calls(slots, lens, table):
        per_slot = torch.zeros(3, dtype=torch.long, device=dev)
        per_slot[1:] = lens
        yield lambda: ops.gqa_decode_attention_q8(q, k, v, s, lens, slots, table)
        yield lambda: ops.kv_q8_read(k, v, s, None, lens, slots, table, *out)
        yield lambda: ops.kv_q8_decode_update(k, v, s, per_slot, slots, table, new, new)
        yield lambda: ops.kv_q8_mixed_update(k, v, s, t(0, 1, 2), lens, slots, table, new, new)

    bad_bt = bt.clone()
    bad_bt[1:] = n_pages
    neg_bt = bt.clone()
    neg_bt[1:] = -1
    for bit, slots, lens, table in (
            (1 << 0, t(3, -1), t(20, 20), good_bt),
            (1 << 1, t(1, 2), t(16 * n_pages + 1, 16 * n_pages + 1), good_bt),
            (1 << 2, t(1, 2), t(20, 20), bad_bt), (1 << 2, t(1, 2), t(20, 20), neg_bt)):
        for i, call in enumerate(calls(slots, lens, table)):
            call()
            got = native.device_errors(0, clear=True)
            assert got & bit, (bit, i, got)
    for a, b in zip((k, v, s), before):
        assert torch.equal(a, b)
    ops.kv_q8_mixed_update(k, v, s, t(0, 5, 2), t(0, 0), t(1, 2), bt, new, new)
    assert native.device_errors(0, clear=True) & (1 << 5)


def test_captured_replayed_and_on_a_side_stream(ops, cuda_device):
    """Write, attend and read back in a CUDA graph, replayed with other lengths and
    rows; two graphs of the same pool."""
    dev = cuda_device
    hist = [40, 0, 100, 15]
    (k, v, s, bt), g = _pool([h + 8 for h in hist], 2, 6, dev)
    lens = torch.tensor([0] + hist, device=dev)
    slots = torch.arange(1, 5, device=dev)
    x = _rows(4, 14, 2, g, dev).reshape(1, 4, -1)
    cos, sin = _rotary(torch.tensor(hist), dev)
    out = [torch.zeros(k.shape, device=dev).half() for _ in range(2)]

    def step():
        q = ops.rope_kv_q8_decode_update(x, cos, sin, k, v, s, lens, slots, bt)
        now = lens[slots] + 1
        o = ops.gqa_decode_attention_q8(q, k, v, s, now, slots, bt)
        ops.kv_q8_read(k, v, s, None, now, slots, bt, *out)
        return o

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager = step()
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step())
        graphs.append(graph)
    graphs[0].replay()
    assert torch.equal(outs[0], eager)
    for i in range(4):
        lens[1:] += 1
        x.normal_()
        graphs[i % 2].replay()
        codes = [t.clone() for t in (k, v, s)]
        assert torch.equal(step(), outs[i % 2])
        for a, b in zip((k, v, s), codes):
            assert torch.equal(a, b)


def test_a_pass_without_sequences_rotates_its_rows(ops, cuda_device):
    dev = cuda_device
    (k, v, s, bt), g = _pool([20], 2, 3, dev)
    x = _rows(5, 14, 2, g, dev)
    cos, sin = _rotary(torch.arange(5), dev)
    none = torch.zeros(0, dtype=torch.long, device=dev)
    before = [t.clone() for t in (k, v, s)]
    q = ops.rope_kv_q8_mixed_update(x.reshape(1, 5, -1), cos, sin, k, v, s,
                                    torch.zeros(1, dtype=torch.long, device=dev), none, none, bt)
    assert torch.equal(q.cpu(), ref.rope_fp32(x[:, :, :14].cpu(), cos.cpu(), sin.cpu()).half())
    for a, b in zip((k, v, s), before):
        assert torch.equal(a, b)


def test_pools_beyond_32_bit_offsets(ops, cuda_device):
    """The last pages of pools of more than 2^31 bytes (and 2^31 fp16 values read back)."""
    dev, n_pages, n = cuda_device, 1_100_000, 200
    k, v = (torch.zeros(n_pages, 2, PAGE, D, dtype=torch.int8, device=dev) for _ in range(2))
    s = torch.zeros(n_pages, 2, 2, device=dev)
    out = [torch.zeros(k.shape, dtype=torch.half, device=dev) for _ in range(2)]
    used = -(-n // PAGE)
    bt = torch.zeros(2, n_pages, dtype=torch.int32, device=dev)
    bt[1, :used] = torch.arange(n_pages - used, n_pages, dtype=torch.int32, device=dev)
    g = torch.Generator().manual_seed(1)
    rows = torch.randn(2, 1, n, 2, D, generator=g).half()
    t = lambda *x: torch.tensor(x, device=dev)
    ops.kv_q8_mixed_update(k, v, s, t(0, n), t(0), t(1), bt, rows[0].to(dev), rows[1].to(dev))
    small = [torch.zeros(used, 2, PAGE, D, dtype=torch.int8) for _ in range(2)]
    scales = torch.zeros(used, 2, 2)
    near = torch.stack([torch.zeros(used), torch.arange(used)]).long()
    ref.update(*small, scales, [(1, 0, 0, n)], near, rows[0, 0], rows[1, 0])
    assert torch.equal(k[-used:].cpu(), small[0]) and torch.equal(v[-used:].cpu(), small[1])
    assert torch.equal(s[-used:].cpu(), scales) and not k[:1000].any()
    ops.kv_q8_read(k, v, s, None, t(n), t(1), bt, *out)
    back = (small[0].float() * scales[:, 0, :, None, None]).half()
    assert torch.equal(out[0][n_pages - used:-1].cpu(), back[:-1]) and not out[0][:1000].any()
    args = (torch.randn(1, 1, 14, D, generator=g).half().to(dev), k, v, s, t(n), t(1), bt)
    _near(ops.gqa_decode_attention_q8(*args), args)


def test_op_refusals(ops, cuda_device):
    dev = cuda_device
    q, k, v, s, lens, slots, bt = _attend(dev, [20, 40], 2, 7, 1)
    new = torch.zeros(1, 2, 2, D, device=dev).half()
    att = lambda **kw: ops.gqa_decode_attention_q8(**{**dict(
        q=q, k=k, v=v, kv_scales=s, lens=lens, slot_ids=slots, block_table=bt), **kw})
    dec = lambda **kw: ops.kv_q8_decode_update(**{**dict(
        k_cache=k, v_cache=v, kv_scales=s, lens=lens, slot_ids=slots, block_table=bt,
        k_new=new, v_new=new), **kw})
    out = torch.zeros_like(k, dtype=torch.half)
    rd = lambda **kw: ops.kv_q8_read(**{**dict(
        k_cache=k, v_cache=v, kv_scales=s, starts=None, lens=lens, slot_ids=slots,
        block_table=bt, k_out=out, v_out=out), **kw})
    for call, kw in ((att, dict(q=q.float())), (att, dict(k=k.half())), (att, dict(kv_scales=s.half())),
                     (att, dict(kv_scales=s[:-1])), (att, dict(lens=lens.int())),
                     (att, dict(block_table=bt[:, :-1])), (att, dict(q=q.transpose(2, 3))),
                     (att, dict(q=q.repeat(1, 1, 2, 1))), (att, dict(lens=lens.cpu())),
                     (att, dict(block_table=bt.float())), (att, dict(v=v[:, :1])),
                     (dec, dict(k_new=new.float())), (dec, dict(slot_ids=slots[:1])),
                     (dec, dict(k_new=new[..., :32], v_new=new[..., :32])),
                     (dec, dict(kv_scales=s.cpu())), (rd, dict(k_out=out.float())),
                     (rd, dict(starts=lens[:1])), (rd, dict(k_out=out[:-1], v_out=out[:-1]))):
        with pytest.raises(RuntimeError):
            call(**kw)
    empty = torch.zeros(0, dtype=torch.long, device=dev)
    assert att(q=q[:, :0], lens=empty, slot_ids=empty).shape == (1, 0, 14, D)
    dec(slot_ids=empty, k_new=new[:, :0], v_new=new[:, :0])
    rd(lens=empty, slot_ids=empty)
