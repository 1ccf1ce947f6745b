"""The decode pass over 8-bit pages in one call (``rope_kv_q8_decode_attention``) against
the update and the attention op in sequence: the same bits in every output and pool."""
import pytest
import torch

from custom_inference_engine_b200 import cabi, native
from oracle import kv_q8 as ref

pytestmark = pytest.mark.gpu
PAGE, D = 16, 64


@pytest.fixture(scope="module")
def ops(cuda_device):
    native.load_ops()
    return torch.ops.inference


@pytest.fixture(autouse=True)
def _no_device_errors(cuda_device):
    native.device_errors(0, clear=True)
    yield
    assert native.device_errors(0, clear=True) == 0


def _case(hist, hkv, group, seed, dev, table=torch.int64, room=1):
    """Slots 1.. with ``hist`` rows and pages for ``room`` more, slot 0 with one page."""
    g = torch.Generator().manual_seed(seed)
    need = [1] + [-(-(h + room) // PAGE) for h in hist]
    n_pages = sum(need) + 2
    perm = torch.randperm(n_pages - 1, generator=g) + 1
    bt = torch.zeros(len(need), n_pages, dtype=table)
    at = 0
    for s, n in enumerate(need):
        bt[s, :n] = perm[at:at + n]
        at += n
    k, v = (torch.randint(-127, 128, (n_pages, hkv, PAGE, D), generator=g, dtype=torch.int8)
            for _ in range(2))
    scales = torch.exp2(torch.randint(-8, -2, (n_pages, 2, hkv), generator=g).float())
    lens = torch.tensor([3] + list(hist))
    return [t.to(dev) for t in (k, v, scales, lens, bt)], g


def _token(B, hkv, group, pos, g, dev, big=1.0):
    x = torch.randn(1, B, (group + 2) * hkv, D, generator=g) * big
    x = x * torch.exp2(torch.randint(-6, 5, (1, B, 1, 1), generator=g).float())
    inv = 1.0 / (1e6 ** (torch.arange(0, D, 2, dtype=torch.float64) / D))
    a = pos.double().cpu()[:, None] * inv
    a = torch.cat((a, a), -1)
    return x.half().reshape(1, B, -1).to(dev), a.cos().half()[None].to(dev), a.sin().half()[None].to(dev)


def _in_sequence(ops, x, cos, sin, k, v, s, lens, slots, bt):
    q = ops.rope_kv_q8_decode_update(x, cos, sin, k, v, s, lens, slots, bt)
    return ops.gqa_decode_attention_q8(q, k, v, s, lens[slots] + 1, slots, bt)


HIST = {
    "one": [0],
    "page borders": [0, 1, 14, 15, 16, 17, 30, 31, 32, 33, 47, 48, 63, 64, 127, 128, 129, 255],
    "long and short": [5000, 0, 15, 16, 700, 9000, 2047, 2048],
    "one split": [40 * i + 7 for i in range(256)],
    "few": [513, 4095, 4096],
}


@pytest.mark.parametrize("name", HIST)
@pytest.mark.parametrize("hkv,group,table", [(2, 7, torch.int64), (1, 8, torch.int32),
                                             (4, 3, torch.int64), (2, 1, torch.int32)])
def test_the_same_bits_as_in_sequence(ops, cuda_device, name, hkv, group, table):
    dev, hist = cuda_device, HIST[name]
    (k, v, s, lens, bt), g = _case(hist, hkv, group, len(name) + hkv, dev, table)
    slots = torch.arange(1, len(hist) + 1, device=dev).flip(0).contiguous()
    args = _token(len(hist), hkv, group, lens[slots], g, dev, big=4.0)
    mine, c = [t.clone() for t in (k, v, s)], [t.clone() for t in (k, v, s)]
    want = _in_sequence(ops, *args, k, v, s, lens, slots, bt)
    got = ops.rope_kv_q8_decode_attention(*args, *mine, lens, slots, bt)
    assert torch.equal(got, want)
    for a, b in zip(mine, (k, v, s)):
        assert torch.equal(a, b)
    got = cabi.rope_kv_q8_decode_attention(*args, *c, lens, slots, bt)
    assert torch.equal(got, want) and torch.equal(c[2], s)
    # and the definition, over the pages as they now are
    q = ref.rope_fp32(args[0].reshape(1, len(hist), -1, D)[:, :, :group * hkv].cpu(),
                      args[1].cpu(), args[2].cpu()).half()
    o, bound = ref.decode_attention(q.to(dev), k, v, s, lens[slots] + 1, slots, bt)
    assert (got.double() - o).abs().le(bound).all()


@pytest.mark.parametrize("splits", [1, 2, 5, 64, 300])
def test_any_split_count(cuda_device, splits, ops):
    dev, hist = cuda_device, [3000, 15, 16, 257, 1023]
    (k, v, s, lens, bt), g = _case(hist, 2, 7, splits, dev)
    slots = torch.arange(1, 6, device=dev)
    args = _token(5, 2, 7, lens[slots], g, dev)
    mine = [t.clone() for t in (k, v, s)]
    q = ops.rope_kv_q8_decode_update(*args, k, v, s, lens, slots, bt)
    want = cabi.decode_attention_q8(q, k, v, s, lens[slots] + 1, slots, bt, num_splits=splits)
    got = cabi.rope_kv_q8_decode_attention(*args, *mine, lens, slots, bt, num_splits=splits)
    assert torch.equal(got, want)


def test_padding_rows_and_slots_that_come_twice(ops, cuda_device):
    """Rows of slot 0 share its page: the last one is written, the other slots' rows are
    those of a call without them."""
    dev, hist = cuda_device, [100, 15, 2000]
    (k, v, s, lens, bt), g = _case(hist, 2, 7, 5, dev)
    slots = torch.tensor([1, 0, 2, 0, 3, 0, 0], device=dev)
    x, cos, sin = _token(7, 2, 7, lens[slots], g, dev)
    mine = [t.clone() for t in (k, v, s)]
    want = _in_sequence(ops, x, cos, sin, k, v, s, lens, slots, bt)
    got = ops.rope_kv_q8_decode_attention(x, cos, sin, *mine, lens, slots, bt)
    for a, b in zip(mine, (k, v, s)):
        assert torch.equal(a, b)
    for i in (0, 2, 4):
        assert torch.equal(got[:, i], want[:, i])


def test_layers_in_a_captured_step(ops, cuda_device):
    """A step of several layers over pools of their own, captured once and replayed while the
    slots grow over page borders and the pages' scales grow with the rows."""
    dev, hist, layers, steps = cuda_device, [0, 5, 15, 31, 300, 1000, 4000], 6, 20
    B = len(hist)
    (k, v, s, lens, bt), g = _case(hist, 2, 7, 9, dev, room=steps)
    slots = torch.arange(1, B + 1, device=dev)
    pools = [[t.clone() for t in (k, v, s)] for _ in range(layers)]
    other = [[t.clone() for t in p] for p in pools]
    x = torch.zeros(1, B, 18 * D, device=dev).half()
    cos, sin = (torch.zeros(1, B, D, device=dev).half() for _ in range(2))
    now = lens.clone()

    def step(pools, op):
        h, out = x, []
        for p in pools:
            o = op(h, cos, sin, *p, now, slots, bt)
            h = x + torch.nn.functional.pad(o.reshape(1, B, -1), (0, 4 * D)) * 0.01
            out.append(o)
        return out

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step([[t.clone() for t in p] for p in pools], ops.rope_kv_q8_decode_attention)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(pools, ops.rope_kv_q8_decode_attention)
    sequence = lambda *a: _in_sequence(ops, *a)
    for i in range(steps):
        a, b, c = _token(B, 2, 7, now[slots], g, dev, big=0.5 * (1 + i))
        x.copy_(a), cos.copy_(b), sin.copy_(c)
        graph.replay()
        for got, want in zip(captured, step(other, sequence)):
            assert torch.equal(got, want), i
        now[1:] += 1
    for p, q in zip(pools, other):
        for a, b in zip(p, q):
            assert torch.equal(a, b)


def test_two_streams_at_once(ops, cuda_device):
    """Decode passes and sampled tokens of two models on streams of their own."""
    dev, steps = cuda_device, 30
    sides = []
    for seed, hist in ((1, [700, 15, 3000, 31]), (2, [16, 900, 63, 2048, 5])):
        (k, v, s, lens, bt), g = _case(hist, 2, 7, seed, dev, room=steps)
        slots = torch.arange(1, len(hist) + 1, device=dev)
        tokens = []
        at = lens.clone()
        for _ in range(steps):
            tokens.append(_token(len(hist), 2, 7, at[slots], g, dev, big=2.0))
            at[1:] += 1
        logits = (torch.randn(len(hist), 60000, generator=g) * 3).half().to(dev)
        u = torch.rand(steps, len(hist), generator=g).to(dev)
        sides.append((k, v, s, lens, bt, slots, tokens, logits, u, torch.ones(len(hist), device=dev)))

    def step(side, pools, at, i, op):
        _, _, _, _, bt, slots, tokens, logits, u, t = side
        return op(*tokens[i], *pools, at, slots, bt), ops.sample_rows(logits, u[i], t)

    want = []
    for side in sides:
        pools, at = [x.clone() for x in side[:3]], side[3].clone()
        for i in range(steps):
            want.append(step(side, pools, at, i, lambda *a: _in_sequence(ops, *a)))
            at[1:] += 1
    streams = [torch.cuda.Stream() for _ in sides]
    state = [([x.clone() for x in side[:3]], side[3].clone()) for side in sides]
    torch.cuda.synchronize()
    got = [[], []]
    for i in range(steps):
        for n, (side, (pools, at), stream) in enumerate(zip(sides, state, streams)):
            with torch.cuda.stream(stream):
                got[n].append(step(side, pools, at, i, ops.rope_kv_q8_decode_attention))
                at[1:] += 1
    torch.cuda.synchronize()
    for (a, b), (c, d) in zip(got[0] + got[1], want):
        assert torch.equal(a, c) and torch.equal(b, d)


def test_a_refused_call_writes_nothing(ops, cuda_device):
    dev = cuda_device
    (k, v, s, lens, bt), g = _case([20, 40], 2, 7, 1, dev)
    slots = torch.tensor([1, 2], device=dev)
    x, cos, sin = _token(2, 2, 7, lens[slots], g, dev)
    before = [t.clone() for t in (k, v, s)]
    call = lambda **kw: ops.rope_kv_q8_decode_attention(**{**dict(
        qkv=x, cos=cos, sin=sin, k_cache=k, v_cache=v, kv_scales=s, lens=lens, slot_ids=slots,
        block_table=bt), **kw})
    nine = torch.zeros(1, 2, 22 * D, device=dev).half()  # nine query heads a kv head
    odd = torch.zeros(1, 2, 18 * D + 3, device=dev).half()[:, :, :18 * D]
    for kw in (dict(qkv=x.float()), dict(cos=cos[:, :1]), dict(slot_ids=slots[:1]), dict(qkv=nine),
               dict(lens=lens.int()), dict(kv_scales=s[:-1]), dict(block_table=bt[:, :-1]),
               dict(qkv=odd), dict(sin=sin.cpu()), dict(k_cache=k.half())):
        with pytest.raises(RuntimeError):
            call(**kw)
    for kw in (dict(workspace=torch.empty(16, dtype=torch.uint8, device=dev)),
               dict(num_splits=5000)):
        with pytest.raises(RuntimeError):
            cabi.rope_kv_q8_decode_attention(x, cos, sin, k, v, s, lens, slots, bt, **kw)
    torch.cuda.synchronize()
    for a, b in zip(before, (k, v, s)):
        assert torch.equal(a, b)
    none = torch.zeros(0, dtype=torch.long, device=dev)
    assert call(qkv=x[:, :0], cos=cos[:, :0], sin=sin[:, :0], slot_ids=none).shape == (1, 0, 14, D)
