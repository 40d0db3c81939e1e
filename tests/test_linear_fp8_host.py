"""CPU: the 8-bit linear module beside nn.Linear"""
import pickle

import torch

from multiagentperception_amd import train_ops


def test_a_module_that_was_pickled_before_it_knew_fast():
    m = train_ops.LinearFp8(6, 4)
    del m.__dict__["fast"]
    old = pickle.loads(pickle.dumps(m))
    x = torch.randn(3, 6)
    assert old.fast is False and torch.equal(old(x), m(x))


def test_arguments_of_nn_linear_keep_their_places():
    m = train_ops.LinearFp8(6, 4, False, None, torch.bfloat16)
    assert m.bias is None and m.weight.dtype == torch.bfloat16 and not m.fast and train_ops.LinearFp8(6, 4, fast=True).fast
