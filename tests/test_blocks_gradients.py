"""Gradients of block_linear: those that a backward pass asks for, and no others."""
import pytest
import torch

from tab_b200 import nn as tab_nn


@pytest.mark.gpu
@pytest.mark.parametrize("M, N, wanted", [(8192, 128, 1), (128, 8192, 0)])
def test_only_the_gradient_that_is_asked_for_is_formed(cuda, M, N, wanted):
    """Both leaves want gradients, a pass asks for one: the other, many times larger, is not formed.  Values as of a pass for both."""
    K = 8192
    x, w = torch.randn(M, K, device=cuda, requires_grad=True), torch.randn(N, K, device=cuda, requires_grad=True)
    g = torch.randn(M, N, device=cuda)
    both = torch.autograd.grad(tab_nn.block_linear(x, w), (x, w), g)
    want, other = both[wanted].clone(), 4 * (x, w)[1 - wanted].numel()
    del both
    y = tab_nn.block_linear(x, w)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    got, = torch.autograd.grad(y, (x, w)[wanted], g)
    assert torch.equal(got, want) and torch.cuda.max_memory_allocated() - before < other / 4


@pytest.mark.gpu
def test_leaves_that_take_turns(cuda):
    """One graph, several passes: for the one leaf, the other, both, and into .grad."""
    x, w = torch.randn(70, 256, device=cuda, requires_grad=True), torch.randn(96, 256, device=cuda, requires_grad=True)
    y, g = tab_nn.block_linear(x, w), torch.randn(70, 96, device=cuda)
    dx, dw = torch.autograd.grad(y, (x, w), g, retain_graph=True)
    assert torch.equal(torch.autograd.grad(y, w, g, retain_graph=True)[0], dw) and torch.equal(torch.autograd.grad(y, x, g, retain_graph=True)[0], dx)
    y.backward(g, inputs=[w], retain_graph=True)
    assert x.grad is None and torch.equal(w.grad, dw)
    y.backward(g)
    assert torch.equal(x.grad, dx) and torch.equal(w.grad, 2 * dw)
