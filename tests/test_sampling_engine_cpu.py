"""What the serving engine and the decode step refuse of a Sampling, on the host."""
import pytest
import torch

from custom_inference_engine_b200 import model_runner as MR
from custom_inference_engine_b200 import serving as SV


@pytest.mark.parametrize("kw", [dict(temperature=[0.7, 1.0]), dict(top_k=(1, 2, 3)),
                                dict(top_p=torch.tensor([0.9])), dict(min_p=[0.0] * 4)])
def test_the_engine_takes_one_value_for_all_requests(kw):
    """Which row a request gets changes from step to step, so that a value per row belongs to
    no request."""
    for make in (lambda s: SV.RunnerEngine(None, 5, sampling=s),
                 lambda s: SV.DecodeBuckets(None, 4, sampling=s)):
        with pytest.raises(ValueError, match="one value"):
            make(MR.Sampling(**kw))


def test_one_value_is_no_list():
    MR.Sampling(0.7, 50, 0.9, 0.01).check_scalar()
    MR.Sampling(torch.tensor(0.7), torch.tensor(5)).check_scalar()


def test_a_greedy_step_refuses_random_numbers():
    d = MR.DecodeGraph.__new__(MR.DecodeGraph)
    d.uniform = d.graph = None
    d.slots, d.tokens = [], torch.zeros(2, dtype=torch.long)
    d._step = lambda: None
    assert torch.equal(d.step(), d.tokens)
    with pytest.raises(ValueError, match="greedy"):
        d.step(torch.rand(2))
