"""Tests that draw from torch's default generators draw the same numbers each time (conftest.default_generators)."""
import pytest
import torch


@pytest.mark.parametrize("run", [0, 1])
def test_the_default_generator_starts_anew(run):
    first = torch.randn(5)
    torch.manual_seed(20)
    assert torch.equal(first, torch.randn(5))


@pytest.mark.gpu
@pytest.mark.parametrize("run", [0, 1])
def test_the_devices_default_generator_starts_anew(run):
    first = torch.randn(5, device="cuda", dtype=torch.float64)
    torch.manual_seed(20)
    assert torch.equal(first, torch.randn(5, device="cuda", dtype=torch.float64))
