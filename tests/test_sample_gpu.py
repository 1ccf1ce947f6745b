"""Sampled tokens (``inference::sample_rows``) against the definition in float64, one
row at a time (``oracle/sampling.py``). Tokens are compared for equality: a row
whose cumulative mass comes within rounding of its random number would be the
only exception, at odds of about 1e-12 per row with these fixed seeds."""
import math

import pytest
import torch

from custom_inference_engine_b200 import cabi, native
from oracle.sampling import sample_row

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(cuda_device):
    native.load_ops()
    return torch.ops.inference


def _want(logits, u, t, k=None, p=None, m=None):
    n = logits.shape[0]
    at = lambda x, d: [d] * n if x is None else x.tolist()
    x = logits.float().cpu().numpy()
    return [sample_row(x[i], uu, tt, kk, pp, mm) for i, (uu, tt, kk, pp, mm) in enumerate(
        zip(u.tolist(), t.tolist(), at(k, 0), at(p, 1.0), at(m, 0.0)))]


def _logits(n, v, seed, dev, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(n, v, generator=g) * spread).half().to(dev), g


@pytest.mark.parametrize("vocab", [1, 2, 7, 8, 9, 255, 1000, 4096, 32003, 65528, 65529, 151936,
                                   262113, 524224])
@pytest.mark.parametrize("rows", [1, 5, 70])
def test_filters(ops, cuda_device, rows, vocab):
    if rows * vocab > 20_000_000:
        rows = 9
    x, g = _logits(rows, vocab, rows + vocab, cuda_device)
    r = lambda: torch.rand(rows, generator=g)
    u, t = r(), r() * 1.5 + 0.05
    k = torch.randint(-1, min(vocab, 300) + 3, (rows,), generator=g)
    p = torch.where(r() < 0.3, torch.ones(rows), r())
    m = torch.where(r() < 0.5, torch.zeros(rows), r() * 0.3)
    want = lambda *a: _want(x, *a)
    dev = [a.to(cuda_device) for a in (u, t, k, p, m)]
    assert ops.sample_rows(x, *dev).tolist() == want(u, t, k, p, m)
    assert ops.sample_rows(x, dev[0], dev[1]).tolist() == want(u, t)
    assert ops.sample_rows(x, dev[0], dev[1], dev[2]).tolist() == want(u, t, k)
    assert ops.sample_rows(x, dev[0], dev[1], top_p=dev[3]).tolist() == want(u, t, None, p)
    assert ops.sample_rows(x, dev[0], dev[1], min_p=dev[4]).tolist() == want(u, t, None, None, m)


@pytest.mark.parametrize("u", [0.0, 1e-9, 0.25, 0.5, 0.999, 1 - 2.0 ** -24, 1.0, 7.0, -1.0])
def test_numbers_at_the_ends(ops, cuda_device, u):
    x, g = _logits(4, 5000, 3, cuda_device)
    t = torch.tensor([0.1, 0.7, 1.0, 50.0])
    k = torch.tensor([0, 40, 0, 3])
    uu = torch.full((4,), u)
    got = ops.sample_rows(x, uu.to(cuda_device), t.to(cuda_device), k.to(cuda_device))
    assert got.tolist() == _want(x, uu, t, k)


def test_ties_go_to_the_lowest_index(ops, cuda_device):
    """Equal logits, signed zeros among them: the order is the vocabulary's, and a
    top-k that ends among equals keeps the first of them."""
    dev = cuda_device
    x = torch.zeros(8, 6000).half()
    x[:, ::2] = -0.0
    x[:, 4000:4100] = 2.0
    x = x.to(dev)
    u = torch.arange(8) / 8 + 0.01
    t = torch.full((8,), 0.05)  # the hundred maxima hold the mass
    got = ops.sample_rows(x, u.to(dev), t.to(dev)).tolist()
    assert got == _want(x, u, t)
    assert got == [4000 + int(a * 100) for a in u.tolist()]  # u as held in fp32
    k = torch.full((8,), 150)
    t = torch.full((8,), 1e6)   # flat: 150 kept, the hundred and the first fifty others
    got = ops.sample_rows(x, u.to(dev), t.to(dev), k.to(dev)).tolist()
    assert got == _want(x, u, t, k)
    assert max(g for g in got if g < 4000) < 50


def test_greedy_rows(ops, cuda_device):
    """temperature <= 0 or NaN: argmax_rows' token, whatever the other columns say."""
    dev = cuda_device
    x, g = _logits(6, 151936, 11, dev)
    x[2, 70000] = x[2, 3] = 60.0
    x[3] = -math.inf
    x[4, 500:700] = math.nan
    x[5, 9] = math.inf
    t = torch.tensor([0.0, -1.0, math.nan, 0.0, 0.0, 0.0], device=dev)
    u = torch.full((6,), 0.9, device=dev)
    k = torch.full((6,), 5, device=dev)
    got = ops.sample_rows(x, u, t, k, top_p=u, min_p=u)
    assert torch.equal(got, ops.argmax_rows(x))


def test_infinities_nan_and_banned_tokens(ops, cuda_device):
    dev = cuda_device
    x, g = _logits(7, 3000, 12, dev)
    x[0] = -math.inf                      # nothing left
    x[1, :2999] = -math.inf               # one token left
    x[2, 100:] = -math.inf
    x[3, 7] = x[3, 2000] = math.inf       # two tokens hold everything
    x[4, 1234] = math.nan
    x[5, ::2] = -math.inf
    x[6] = 65504.0
    x[6, 1] = -65504.0
    for u in (0.0, 0.3, 0.6, 0.99):
        for t in (0.2, 1.0, 1e4, math.inf):
            uu, tt = torch.full((7,), u), torch.full((7,), t)
            got = ops.sample_rows(x, uu.to(dev), tt.to(dev)).tolist()
            assert got == _want(x, uu, tt), (u, t)
            assert got[0] == 0 and got[1] == 2999 and got[2] < 100 and got[4] == 1234


def test_extreme_filters(ops, cuda_device):
    dev = cuda_device
    x, g = _logits(8, 2000, 13, dev)
    u = torch.rand(8, generator=g)
    t = torch.ones(8)
    top = x.float().argmax(-1).tolist()
    f = lambda v: torch.full((8,), v)
    for kw in (dict(top_p=f(0.0)), dict(top_p=f(1e-30)), dict(top_p=f(-1.0)),
               dict(top_k=torch.ones(8, dtype=torch.long)), dict(min_p=f(2.0)),
               dict(min_p=f(math.nan))):
        got = ops.sample_rows(x, u.to(dev), t.to(dev), **{a: b.to(dev) for a, b in kw.items()})
        assert got.tolist() == top, kw
    got = ops.sample_rows(x, u.to(dev), t.to(dev), min_p=f(1.0).to(dev))  # every maximum
    assert got.tolist() == _want(x, u, t, None, None, f(1.0))
    plain = ops.sample_rows(x, u.to(dev), t.to(dev)).tolist()
    for kw in (dict(top_p=f(1.0)), dict(top_p=f(9.0)), dict(min_p=f(0.0)), dict(min_p=f(-1.0)),
               dict(top_k=f(0).long()), dict(top_k=f(-5).long()), dict(top_k=f(2000).long()),
               dict(top_k=torch.full((8,), 1 << 40))):
        got = ops.sample_rows(x, u.to(dev), t.to(dev), **{a: b.to(dev) for a, b in kw.items()})
        assert got.tolist() == plain, kw


def test_rows_at_any_alignment_and_stride(ops, cuda_device):
    dev = cuda_device
    buf, g = _logits(6, 70001, 14, dev)
    u, t = torch.rand(6, generator=g), torch.full((6,), 0.8)
    for view in (buf[:, 1:], buf[:, 3:66000], buf[:, 8:40], buf[::2, :], buf[:, :70000]):
        n = view.shape[0]
        got = ops.sample_rows(view, u[:n].to(dev), t[:n].to(dev))
        assert got.tolist() == _want(view, u[:n], t[:n])
    three = buf[:, :70000].reshape(2, 3, 70000)
    got = ops.sample_rows(three, u.to(dev).view(2, 3), t.to(dev))
    assert got.shape == (2, 3) and got.view(-1).tolist() == _want(buf[:, :70000], u, t)
    assert cabi.sample_rows(buf, u.to(dev), t.to(dev)).tolist() == _want(buf, u, t)


def test_a_row_alone_and_rows_that_coincide(ops, cuda_device):
    dev = cuda_device
    x, g = _logits(1, 4000, 19, dev)
    u, t = torch.rand(1, generator=g).to(dev), torch.ones(1, device=dev)
    got = ops.sample_rows(x[0], u, t)
    assert got.shape == () and [got.item()] == _want(x, u.cpu(), t.cpu())
    with pytest.raises(RuntimeError):  # rows may not overlap
        ops.sample_rows(x.expand(3, 4000), u.repeat(3), t.repeat(3))


def test_constant_rows(ops, cuda_device):
    """Every token the same: the counters hold a whole part of a row, and the cumulative
    mass meets its random number exactly."""
    dev = cuda_device
    for vocab in (4, 65528, 131056, 262144, 524224):
        x = torch.full((5, vocab), 3.25, device=dev).half()
        u = torch.tensor([0.0, 0.25, 0.5, 0.75, 1 - 2.0 ** -24])
        t = torch.full((5,), 0.7, device=dev)
        got = ops.sample_rows(x, u.to(dev), t)
        assert got.tolist() == [min(int(a * vocab), vocab - 1) for a in u.tolist()], vocab
        k = torch.full((5,), vocab // 2, device=dev)
        got = ops.sample_rows(x, u.to(dev), t, k, top_p=torch.full((5,), 0.5, device=dev))
        n = vocab // 4
        assert got.tolist() == [min(int(a * n), n - 1) for a in u.tolist()], vocab


@pytest.mark.parametrize("rows,vocab", [(76, 98296), (76, 98289), (40, 151936), (40, 196592),
                                        (20, 390001)])
def test_parts_of_more_than_two_to_the_16_tokens(ops, cuda_device, rows, vocab):
    """One token value fills most of a part: counted apart when it is found early, and found
    by a second count when 32 evenly spread tokens of the part are others."""
    dev, g = cuda_device, torch.Generator().manual_seed(vocab)
    rand = lambda *n: torch.rand(*n, generator=g)
    parts = next(c for c in (1, 2, 4, 8) if -(-vocab // (8 * c)) * 8 <= 98296)
    part = -(-vocab // (8 * parts)) * 8
    fill = [0.25, 0.25024414, -0.0, 0.0, -65504.0, -math.inf]  # (keys of either parity)
    x = torch.empty(rows, vocab).half()
    for i, value in enumerate(fill):
        x[i] = torch.randn(vocab, generator=g) * 2.5
        where = rand(vocab) < 0.9
        if i % 2:  # the sampled tokens stay as they are, each twice
            for lo in range(0, vocab, part):
                n = min(part, vocab - lo)
                at = torch.tensor([lo + (n * l >> 5) for l in range(32)])
                where[at] = False
                x[i, at] = x[i, at[:16]].repeat(2)
        x[i, where] = value
        if value == 0:  # zeros of both signs, fewer than 2^16 of each
            x[i, where.nonzero()[::2, 0]] = -value
    # exactly 65535, 65536 and 65537 tokens of one value in the first part
    for i, n in enumerate((65535, 65536, 65537)):
        x[6 + i] = (torch.randn(vocab, generator=g) * 2.5).half()
        x[6 + i, torch.randperm(min(part, vocab), generator=g)[:n]] = 1.5 + i / 1024
    x[9:] = x[8]
    u, t = rand(rows), torch.ones(rows)
    t[4] = 1e5  # (the lowest value keeps half of its weight)
    k = torch.full((rows,), vocab // 2)
    p, m = rand(rows), torch.full((rows,), 0.01)
    for args in ((u, t), (u, t, k), (u, t, k, p, m)):
        got = ops.sample_rows(x.to(dev), *(a.to(dev) for a in args))
        assert got[:9].tolist() == _want(x[:9], *(a[:9] for a in args))
        again = ops.sample_rows(x.to(dev), *(a.to(dev) for a in args))
        assert torch.equal(got, again)


def test_follows_the_distribution(ops, cuda_device):
    """Evenly spaced numbers over one row: the tokens' counts are their probabilities
    to within one."""
    dev = cuda_device
    n, v = 4096, 40
    x, g = _logits(1, v, 15, dev, spread=1.0)
    u = ((torch.arange(n) + 0.5) / n).to(dev)
    t = torch.full((n,), 0.9, device=dev)
    got = ops.sample_rows(x.expand(n, v).contiguous(), u, t)
    count = torch.bincount(got, minlength=v).double().cpu()
    prob = torch.softmax(x[0].double().cpu() / float(torch.tensor(0.9)), -1)
    assert (count - prob * n).abs().max() <= 1.0


def test_captured_and_replayed(ops, cuda_device):
    dev = cuda_device
    x, g = _logits(3, 151936, 16, dev)
    u, t = torch.rand(3, device=dev), torch.ones(3, device=dev)
    ops.sample_rows(x, u, t)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.sample_rows(x, u, t)
    for _ in range(3):
        x.normal_(0, 3)
        u.uniform_()
        graph.replay()
        assert out.tolist() == _want(x, u.cpu(), t.cpu())


def test_refusals(ops, cuda_device):
    dev = cuda_device
    x, _ = _logits(4, 100, 17, dev)
    u = torch.rand(4, device=dev)
    for bad in (lambda: ops.sample_rows(x.float(), u, u), lambda: ops.sample_rows(x, u[:3], u),
                lambda: ops.sample_rows(x, u.double(), u), lambda: ops.sample_rows(x, u, u.half()),
                lambda: ops.sample_rows(x, u, u, top_k=u), lambda: ops.sample_rows(x, u.cpu(), u),
                lambda: ops.sample_rows(x.T, u, u), lambda: ops.sample_rows(x[:, :0], u, u),
                lambda: ops.sample_rows(x, u, u, top_p=u[:1]),
                lambda: ops.sample_rows(torch.zeros(1, 524225, device=dev).half(), u[:1], u[:1])):
        with pytest.raises(RuntimeError):
            bad()
    assert ops.sample_rows(x[:0], u[:0], u[:0]).shape == (0,)
