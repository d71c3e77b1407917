"""Calls of the row operators that are refused before a device is touched, besides those of test_row_operators_host.py."""
import ctypes as C

import pytest
import torch

from cellerator_b200 import capi
from test_row_operators_host import ADDRESS, norm


@pytest.mark.parametrize("apart", [0, 1, 7, -1, -7])
def test_gradients_of_parameters_that_overlap(apart):
    """dgamma and dbeta of eight columns, so many elements from one another: what both write would be the one that ends last."""
    n = norm(dgamma=9 * ADDRESS, dbeta=9 * ADDRESS + 4 * apart)
    assert capi.lib().cb200_layer_norm_backward(C.byref(n), None) == capi.INVALID_ARGUMENT


@pytest.mark.parametrize("apart", [8, -8])
def test_gradients_of_parameters_side_by_side(apart):
    if torch.cuda.is_available():
        pytest.skip("a CUDA device is present")                 # what is not refused would run
    n = norm(dgamma=9 * ADDRESS, dbeta=9 * ADDRESS + 4 * apart)
    assert capi.lib().cb200_layer_norm_backward(C.byref(n), None) == capi.CUDA_ERROR
