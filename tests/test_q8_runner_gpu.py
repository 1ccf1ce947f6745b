"""The 8-bit KV pages and the sampled tokens as they are used together: through the
attention module and QuantizedKVStorage, the paged runner's eager and captured
passes, and the serving loop."""
import numpy as np
import pytest
import torch

from custom_inference_engine_b200 import model_runner as MR
from custom_inference_engine_b200 import native
from custom_inference_engine_b200 import serving as SV
from oracle import kv_q8 as ref
from oracle.sampling import sample_row

pytestmark = pytest.mark.gpu
SAMPLING = MR.Sampling(temperature=0.8, top_k=50, top_p=0.9, min_p=0.01)


@pytest.fixture(autouse=True)
def _no_device_errors(cuda_device):
    native.device_errors(0, clear=True)
    yield
    assert native.device_errors(0, clear=True) == 0


def _model(dev, layers=2):
    cfg = MR.qwen2_config(num_hidden_layers=layers, vocab_size=4096, intermediate_size=2048)
    return MR.random_qwen2(cfg, seed=0, device=dev)


def _runner(dev, **kw):
    kw = {**dict(max_cache_len=4096, n_slots=8, token_budget=64, kv_cache_dtype=torch.int8), **kw}
    return MR.PagedRunner(_model(dev), **kw)


def _prompts():
    rng = np.random.default_rng(7)
    return [rng.integers(0, 4096, size=n).tolist() for n in (5, 40, 17, 130, 1)]


def _start(runner, sampling=None, new=16):
    prompts = _prompts()
    slots = list(range(1, len(prompts) + 1))
    for s, p in zip(slots, prompts):
        runner.admit(s, len(p) + new)
    return slots, runner.prefill(slots, prompts, sampling)


@pytest.mark.parametrize("fuse_rope", [True, False])
def test_attention_module_over_8_bit_pages(cuda_device, fuse_rope):
    """Two prefill chunks of two slots and three decode steps through one attention
    module: the pages are the oracle's after every pass, and every output row is the
    float64 attention over them within the kernels' roundings."""
    from custom_inference_engine_b200.attn import core
    from custom_inference_engine_b200.attn.metadata import AttentionMetadata
    from custom_inference_engine_b200.kv_cache.storage import QuantizedKVStorage

    dev = cuda_device
    model = _model(dev, 1)
    core.use_cuda_attention(model)
    attn = model.model.layers[0].self_attn
    attn.fuse_rope = fuse_rope
    kv = QuantizedKVStorage(model.config, 20 * 16, 16, 4, dev, torch.float16)
    kv.block_table[1, :5] = torch.tensor([7, 3, 11, 5, 9], device=dev)
    kv.block_table[2, :4] = torch.tensor([2, 12, 6, 14], device=dev)
    want = [t.cpu().clone() for t in kv.pool(0)]
    rotary = model.model.rotary_emb
    lens = {1: 0, 2: 0}
    g = torch.Generator(device=dev).manual_seed(1)
    captured = {}
    attn.original.o_proj.register_forward_pre_hook(lambda m, x: captured.update(o=x[0]))

    def run(chunks, decode):
        slots, n = list(chunks), list(chunks.values())
        T = sum(n)
        x = torch.randn(1, T, 896, generator=g, device=dev).half()
        pos = torch.cat([torch.arange(lens[s], lens[s] + c) for s, c in chunks.items()]).to(dev)
        cos, sin = rotary(x, pos.view(1, -1))
        md = AttentionMetadata(token_count=T, full_decode=decode, device=dev)
        md.prepare_full_graph(len(slots))
        md.write_slot_ids(slots)
        cu = np.concatenate([[0], np.cumsum(n)])
        md.write_cu_seqlens(cu)
        with torch.inference_mode():
            attn(x, (cos, sin), kv_manager=kv, metadata=md)
            qkv = torch.nn.functional.linear(x, attn.qkv_weight, attn.qkv_bias)
            q, k, v = attn._rotated(qkv, cos, sin)
        split = qkv.view(1, T, 18, 64).cpu()
        if fuse_rope:  # the kernels rotate in fp32
            rows_k = ref.rope_fp32(split[:, :, 14:16], cos.cpu(), sin.cpu())[0]
            q = ref.rope_fp32(split[:, :, :14], cos.cpu(), sin.cpu()).half().to(dev)
        else:
            rows_k = k[0].cpu()
        ref.update(*want, [(s, lens[s], int(cu[i]), n[i]) for i, s in enumerate(slots)],
                   kv.block_table.cpu(), rows_k, v[0].cpu())
        for a, b in zip(kv.pool(0), want):
            assert torch.equal(a.cpu(), b)
        # every row attends to its slot up to itself
        rows = [(s, lens[s] + j + 1) for s, c in chunks.items() for j in range(c)]
        o, tol = ref.decode_attention(q, *kv.pool(0), torch.tensor([r[1] for r in rows]),
                                      torch.tensor([r[0] for r in rows]), kv.block_table)
        got = captured["o"].view(1, T, 14, 64).double()
        assert ((got - o).abs() <= tol).all()
        for s, c in chunks.items():
            lens[s] += c
            kv.lens[s] += c

    run({1: 20, 2: 3}, False)
    run({2: 30, 1: 17}, False)
    for _ in range(3):
        run({1: 1, 2: 1}, True)


def test_captured_passes_match_eager_ones(cuda_device):
    """Prefill through captured mixed passes and decode through a captured step give the
    bits of the eager passes."""
    logits = []
    for capture in (False, True):
        r = _runner(cuda_device, mixed_graphs=capture, fused_lm_head=False)
        slots, pre = _start(r)
        d = r.decode_graph(slots, pre.first_tokens, capture=capture)
        steps = [pre.last_logits.half()]
        for _ in range(10):
            d.step()
            steps.append(d.logits.clone())
        logits.append(steps)
    for a, b in zip(*logits):
        assert torch.equal(a, b)


def test_any_chunking_of_a_prompt_keeps_the_page_scales(cuda_device):
    """Layer 0's K and V rows do not depend on how a prompt is cut into passes, so its
    page scales do not either, and its codes differ by at most one step."""
    pools = []
    for budget in (64, 24):
        r = _runner(cuda_device, token_budget=budget)
        slots, _ = _start(r)
        pools.append([t.clone() for t in r.kv.pool(0)])
    (ka, va, sa), (kb, vb, sb) = pools
    assert torch.equal(sa[1:], sb[1:])
    for a, b in ((ka, kb), (va, vb)):
        assert (a[1:].int() - b[1:].int()).abs().max() <= 1


@pytest.mark.parametrize("kv_cache_dtype", [None, torch.int8])
@pytest.mark.parametrize("capture", [False, True])
def test_sampled_decoding(cuda_device, kv_cache_dtype, capture):
    """Every sampled step's tokens are the definition's for the step's logits and random
    numbers; two captured steps of other parameters share a pool."""
    r = _runner(cuda_device, kv_cache_dtype=kv_cache_dtype)
    slots, pre = _start(r, SAMPLING)
    per_row = MR.Sampling(temperature=[0.0, 0.5, 1.0, 1.5, 0.7], top_k=[0, 3, 0, 100, 0],
                          top_p=[1.0, 1.0, 0.8, 0.95, 1.0], min_p=[0.0, 0.0, 0.0, 0.1, 0.02])
    graphs = [r.decode_graph(slots, pre.first_tokens, capture=capture, sampling=s)
              for s in (SAMPLING, per_row)]
    tokens = torch.tensor(pre.first_tokens, device=cuda_device)
    seen = set()
    for i in range(8):
        d = graphs[i % 2]
        d.tokens.copy_(tokens)
        given = torch.rand(5) if i < 4 else None
        tokens = d.step(given).clone()
        u = d.uniform.tolist()
        if given is not None:
            assert u == given.tolist()
        cols = [c.tolist() for c in d.columns]
        x = d.logits.float().cpu().numpy()
        assert tokens.tolist() == [sample_row(x[b], u[b], *(c[b] for c in cols))
                                   for b in range(5)]
        seen.add(tuple(u))
    assert len(seen) == 8  # every step has numbers of its own


def test_capturing_a_step_leaves_the_pages_alone(cuda_device):
    r = _runner(cuda_device)
    slots, pre = _start(r)
    before = [t.clone() for layer in range(2) for t in r.kv.pool(layer)]
    r.decode_graph(slots, [4095] * 5)
    after = [t for layer in range(2) for t in r.kv.pool(layer)]
    for a, b in zip(after, before):
        assert torch.equal(a[1:], b[1:])  # page 0 is padding


def test_temperature_zero_is_greedy(cuda_device):
    runs = []
    for sampling in (None, MR.Sampling(temperature=0.0)):
        r = _runner(cuda_device, fused_lm_head=False)
        slots, pre = _start(r, sampling)
        d = r.decode_graph(slots, pre.first_tokens, sampling=sampling)
        runs.append([pre.first_tokens] + [d.step().tolist() for _ in range(6)])
    assert runs[0] == runs[1]


def test_served_requests_with_8_bit_pages_and_sampling(cuda_device):
    """The serving loop over 8-bit pages with sampled tokens finishes every request, and
    the same seed serves the same tokens (requests all there from the start)."""
    served = []
    for _ in range(2):
        r = _runner(cuda_device, n_slots=5, sample_seed=3)
        reqs = SV.poisson_requests(6, rate=1e9, seed=5, vocab=4096, median_prompt=60,
                                   max_prompt=200, min_new=4, max_new=10)
        engine = SV.RunnerEngine(r, 5, sampling=SAMPLING)
        clock = iter(range(10**6))
        out, steps = SV.serve(engine, reqs, n_slots=5, token_budget=64,
                              clock=lambda: float(next(clock)))
        assert steps["mixed"] > 0 and steps["decode"] > 0
        assert all(len(q.new_tokens) == q.max_new for q in out)
        assert len(r.free_pages) == r.kv.n_pages - 1
        served.append([q.new_tokens for q in out])
    assert served[0] == served[1]


def test_refusals(cuda_device):
    from custom_inference_engine_b200.kv_cache.storage import QuantizedKVStorage

    r = _runner(cuda_device)
    with pytest.raises(RuntimeError, match="by sequence"):
        r.kv.mixed_update(0, None, None, None, None)
    with pytest.raises(ValueError):
        QuantizedKVStorage(r.model.config, 64, 16, 2, cuda_device, torch.bfloat16)
    with pytest.raises(ValueError):
        QuantizedKVStorage(r.model.config, 64, 32, 2, cuda_device, torch.float16)
    with pytest.raises(ValueError):
        MR.PagedRunner(r.model, 64, 2, kv_cache_dtype=torch.float8_e4m3fn)
