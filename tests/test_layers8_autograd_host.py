"""What the differentiable 8-bit layers and norms refuse before anything touches a GPU: tangents of forward mode, for which they have no formula."""
import pytest
import torch
from torch.autograd import forward_ad

import tab_amd
from tab_amd import nn as tab_nn


def test_tangents_are_refused_and_not_dropped():
    def dual(*shape):
        return forward_ad.make_dual(torch.ones(shape), torch.ones(shape))

    x, w = torch.zeros(4, 128), torch.zeros(8, 128)
    q, s = torch.zeros(8, 128).to(torch.float8_e4m3fn), torch.zeros(1, 1, dtype=torch.uint8).view(torch.float8_e8m0fnu)
    with forward_ad.dual_level():
        for a, b in ((dual(4, 128), w), (x, dual(8, 128)), (dual(4, 128).requires_grad_(), w)):
            with pytest.raises(RuntimeError, match="forward mode"):
                tab_nn.linear8(a, b)
        with pytest.raises(RuntimeError, match="forward mode"):
            tab_nn.Linear8(q, s, 128, 8)(dual(4, 128))
        v = torch.zeros(128)
        for args in ((dual(4, 128), x), (x, dual(4, 128)), (x, x, dual(1, 128)), (x, x, None, dual(128)), (x, x, None, v, dual(128)), (dual(4, 128),)):
            for output in (tab_amd.NORM_PLAIN, tab_amd.NORM_8BIT):
                with pytest.raises(RuntimeError, match="forward mode"):
                    tab_nn.norm_residual(*args, output=output)
        with pytest.raises(RuntimeError, match="CUDA tensor"):  # a level alone changes nothing
            tab_nn.linear8(x, w)
        with forward_ad._set_fwd_grad_enabled(False), pytest.raises(RuntimeError, match="CUDA tensor"):
            tab_nn.linear8(dual(4, 128), w)


def test_gates_that_would_have_to_be_repeated_are_refused():
    """A row of the gate holds for consecutive rows: a gate for each position, repeated over the sequences, would be taken for something else."""
    x = torch.zeros(2, 3, 4, 8)
    for sizes in ((1, 3, 4, 8), (1, 3, 1, 8), (2, 1, 4, 8), (1, 1, 4, 8), (3, 1, 1, 8)):
        with pytest.raises(RuntimeError, match="consecutive rows"):
            tab_nn.norm_residual(x, x, torch.zeros(sizes))
    for sizes in ((1, 1, 1, 8), (2, 1, 1, 8), (2, 3, 1, 8), (2, 3, 4, 8), (6, 8), (1, 8), (8,)):
        with pytest.raises(RuntimeError, match="CUDA tensor"):  # as far as that
            tab_nn.norm_residual(x, x, torch.zeros(sizes))


def test_a_stack_refuses_such_gates_too():
    stack = tab_nn.ResidualStack([torch.nn.Identity()], 8)
    x = torch.zeros(2, 4, 8)
    with pytest.raises(RuntimeError, match="consecutive rows"):
        stack(x, [torch.zeros(1, 4, 8)])
    for sizes in ((2, 1, 8), (1, 1, 8), (2, 8), (8, 8)):
        with pytest.raises(RuntimeError, match="CUDA tensor"):
            stack(x, [torch.zeros(sizes)])
    with pytest.raises(TypeError):
        stack(x, [0.5])
    with pytest.raises(RuntimeError, match="CUDA tensor"):  # one tensor for all blocks
        stack(x, torch.zeros(1, 2, 8))
