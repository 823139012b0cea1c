"""The example policy on the high-low game: games played through the step calls, trained
through the calls over whole games."""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu
PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "high_low_policy.py")


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("high_low_policy", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_moves_and_whole_games_agree(example):
    # Both forms keep float32 throughout; a log probability is a sum of four, each of a few
    # hundred float32 roundings of values of order 1 to 10: within 1e-3 by a wide margin.
    assert example.main(["--envs", "48", "--players", "5", "--rounds", "6", "--updates", "2"]) < 1e-3


def test_gradients_reach_every_parameter(example):
    torch.manual_seed(3)
    policy = example.Policy(20, 6, 2, D=32, blocks=2, H=2, P=16, N=16).cuda()
    obs = torch.randn(7, 9, 20, device="cuda")
    choice = torch.randint(0, 3, (7, 9, 4), device="cuda")
    (-example.log_prob(policy(obs), choice).mean()).backward()
    for name, p in policy.named_parameters():
        assert p.grad is not None and bool(torch.isfinite(p.grad).all()) and float(p.grad.abs().max()) > 0, name
