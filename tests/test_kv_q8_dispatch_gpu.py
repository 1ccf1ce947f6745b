"""The forms of the 8-bit update, decode pass and sampling that only some sizes, settings or
default types reach."""
import numpy as np
import pytest
import torch

from custom_inference_engine_b200 import model_runner as MR
from custom_inference_engine_b200 import native
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


def _rotary(pos):
    inv = 1.0 / (1e6 ** (torch.arange(0, D, 2, dtype=torch.float64) / D))
    a = pos.double()[:, None] * inv
    a = torch.cat((a, a), -1)
    return a.cos().half()[None], a.sin().half()[None]


@pytest.mark.parametrize("batch", [510, 511, 512, 513, 700])
@pytest.mark.parametrize("rope", [False, True])
def test_mixed_updates_of_many_sequences(ops, cuda_device, batch, rope):
    """cu_seqlens is searched in shared memory up to 511 sequences and in place beyond: empty
    sequences, one that spans pages, a slot that comes twice, rows behind the last."""
    dev, hkv = cuda_device, 2
    g = torch.Generator().manual_seed(batch)
    n = torch.randint(0, 4, (batch,), generator=g).tolist()
    n[batch // 2], n[-1] = 37, 2
    hist = torch.randint(0, 20, (batch,), generator=g).tolist()
    slots = list(range(1, batch + 1))
    n[7], n[-3], slots[-3], hist[-3] = 3, 2, slots[7], hist[7]   # (the later one is written)
    T = sum(n) + 5
    cu = [0] + np.cumsum(n).tolist()
    need = [-(-(h + c) // PAGE) for h, c in zip(hist, n)]
    n_pages = sum(need) + 2
    bt = torch.zeros(batch + 1, n_pages, dtype=torch.int32)
    perm, at = torch.randperm(n_pages - 1, generator=g).int() + 1, 0
    for s in range(1, batch + 1):
        c = need[s - 1]
        bt[s, :c] = perm[at:at + c]
        at += c
    k, v = (torch.randint(-127, 128, (n_pages, hkv, PAGE, D), generator=g, dtype=torch.int8)
            for _ in range(2))
    s = torch.exp2(torch.randint(-8, -2, (n_pages, 2, hkv), generator=g).float())
    x = torch.randn(1, T, 9 * hkv, D, generator=g).half()
    pos = torch.cat([torch.arange(h, h + c) for h, c in zip(hist, n)] + [torch.zeros(5)])
    cos, sin = _rotary(pos)
    kn, vn = x[:, :, 7 * hkv:8 * hkv], x[:, :, 8 * hkv:]
    rows_k = ref.rope_fp32(kn, cos, sin)[0] if rope else kn[0]
    got = [t.to(dev) for t in (k, v, s)]
    ref.update(k, v, s, [(slots[b], hist[b], cu[b], n[b]) for b in range(batch) if b != 7], bt,
               rows_k, vn[0])
    at = [torch.tensor(t, device=dev) for t in (cu, hist, slots)] + [bt.to(dev)]
    if rope:
        q = ops.rope_kv_q8_mixed_update(x.reshape(1, T, -1).to(dev), cos.to(dev), sin.to(dev),
                                        *got, *at)
        assert torch.equal(q.cpu(), ref.rope_fp32(x[:, :, :7 * hkv], cos, sin).half())
    else:
        ops.kv_q8_mixed_update(*got, *at, kn.to(dev), vn.to(dev))
    for a, b in zip(got, (k, v, s)):
        assert torch.equal(a.cpu(), b)


def _runner(dev, **kw):
    cfg = MR.qwen2_config(num_hidden_layers=2, vocab_size=4096, intermediate_size=2048)
    model = MR.random_qwen2(cfg, seed=0, device=dev)
    return MR.PagedRunner(model, max_cache_len=2048, n_slots=5, token_budget=64,
                          kv_cache_dtype=torch.int8, **kw)


def test_update_and_attention_apart_match_the_one_call_pass(cuda_device):
    """Decode steps with fuse_decode_attention off: the bits of the one-call pass."""
    runs = []
    for fused in (True, False):
        r = _runner(cuda_device, fused_lm_head=False)
        for layer in r.model.model.layers:
            layer.self_attn.fuse_decode_attention = fused
        prompts = [list(range(1, n + 1)) for n in (5, 31, 100)]
        for s, p in zip((1, 2, 3), prompts):
            r.admit(s, len(p) + 20)
        d = r.decode_graph([1, 2, 3], r.prefill([1, 2, 3], prompts).first_tokens)
        steps = []
        for _ in range(12):
            d.step()
            steps.append(d.logits.clone())
        runs.append(steps + [t[1:].clone() for t in r.kv.pool(1)])
    for a, b in zip(*runs):
        assert torch.equal(a, b)


def test_sampled_steps_under_another_default_type(cuda_device):
    """The random numbers are fp32 whatever torch's default type is."""
    sampling, tokens = MR.Sampling(0.9, 20), []
    for dtype in (torch.float32, torch.float16):
        r = _runner(cuda_device)
        torch.set_default_dtype(dtype)
        try:
            r.admit(1, 40)
            pre = r.prefill([1], [[5, 6, 7]], sampling)
            d = r.decode_graph([1], pre.first_tokens, sampling=sampling)
            tokens.append([pre.first_tokens, d.step().tolist(), d.step(torch.rand(1) * 0 + 0.25).tolist()])
        finally:
            torch.set_default_dtype(torch.float32)
    assert tokens[0] == tokens[1]


@pytest.mark.parametrize("lens,hkv,group", [([511], 2, 7), ([0, 1, 700, 4096], 2, 7),
                                            ([3000] * 70, 2, 7), ([9001, 20], 4, 3)])
def test_attention_repeats_itself(ops, cuda_device, lens, hkv, group):
    """The same bits from every call: partials are merged in a fixed order."""
    dev, B = cuda_device, len(lens)
    g = torch.Generator().manual_seed(B)
    pages = -(-max(lens) // PAGE)
    bt = torch.zeros(B + 1, B * pages + 1, dtype=torch.long)
    bt[1:, :pages] = (torch.randperm(B * pages, generator=g) + 1).view(B, pages)
    k, v = (torch.randint(-127, 128, (B * pages + 1, hkv, PAGE, D), generator=g, dtype=torch.int8)
            for _ in range(2))
    s = torch.exp2(torch.randint(-8, -2, (B * pages + 1, 2, hkv), generator=g).float())
    q = torch.randn(1, B, hkv * group, D, generator=g).half()
    args = [t.to(dev) for t in (q, k, v, s, torch.tensor(lens), torch.arange(1, B + 1), bt)]
    first = ops.gqa_decode_attention_q8(*args)
    noise = torch.empty(1 << 26, device=dev)
    for _ in range(10):
        noise.normal_()  # other workspace contents, cold caches
        assert torch.equal(ops.gqa_decode_attention_q8(*args), first)
