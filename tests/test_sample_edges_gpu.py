"""Sampling calls at the edges of their definition: a NaN top_p, and rows without tokens."""
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


@pytest.mark.parametrize("rows,vocab", [(3, 17), (5, 9000), (2, 151936), (80, 32003)])
@pytest.mark.parametrize("with_k", [False, True])
def test_a_nan_top_p_keeps_the_first_token(ops, cuda_device, rows, vocab, with_k):
    """No mass reaches a NaN: as a NaN min_p does, it keeps the order's first token."""
    g = torch.Generator().manual_seed(vocab)
    x = (torch.randn(rows, vocab, generator=g) * 3).half()
    x[0, 5], x[0, 9] = 20.0, 20.0
    u = torch.rand(rows, generator=g) * 0.5 + 0.4
    t = torch.full((rows,), 1.3)
    p = torch.full((rows,), math.nan)
    p[1] = 0.9
    k = torch.full((rows,), 7) if with_k else None
    got = ops.sample_rows(*(None if a is None else a.to(cuda_device) for a in (x, u, t, k, p)))
    want = [sample_row(x[i].float().numpy(), float(u[i]), float(t[i]), 7 if with_k else 0,
                       float(p[i])) for i in range(rows)]
    assert got.tolist() == want
    assert want[0] == 5 and want[2:] == x[2:].float().argmax(-1).tolist()


def test_rows_without_tokens_are_refused(ops, cuda_device):
    """There is no token to give: no output is left unwritten."""
    none = torch.zeros(0, device=cuda_device)
    for shape in ((4, 0), (0,), (2, 3, 0)):
        x = torch.zeros(shape, device=cuda_device).half()
        with pytest.raises(RuntimeError, match="empty row"):
            ops.sample_rows(x, none, none)
    with pytest.raises(RuntimeError):
        cabi.sample_rows(torch.zeros(4, 0, device=cuda_device).half(), none, none)
    empty = torch.zeros(0, 10, device=cuda_device).half()
    assert ops.sample_rows(empty, none, none).shape == (0,)
