"""The policy loss on both sides of the size from which on it takes two launches."""
import pytest
import torch

from tests.test_policy_loss_gpu import compare, cut, inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens", [4095, 4096, 4097, 6000])
@pytest.mark.parametrize("seqs", [None, 1, 9, 2048, 2049])
def test_both_sides(tokens, seqs):
    compare(inputs(tokens), None if seqs is None else cut(tokens, seqs), kl_weight=0.1)
