"""The forms of the 8-bit update, decode pass and sampling that only some sizes, settings or
default types reach."""
import pytest
import torch

from custom_inference_engine_b200 import model_runner as MR
from custom_inference_engine_b200 import native

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _no_device_errors(cuda_device):
    native.device_errors(0, clear=True)
    yield
    assert native.device_errors(0, clear=True) == 0


def _runner(dev, **kw):
    cfg = MR.qwen2_config(num_hidden_layers=2, vocab_size=4096, intermediate_size=2048)
    model = MR.random_qwen2(cfg, seed=0, device=dev)
    return MR.PagedRunner(model, max_cache_len=2048, n_slots=5, token_budget=64,
                          kv_cache_dtype=torch.int8, **kw)


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
