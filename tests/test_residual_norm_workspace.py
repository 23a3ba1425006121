"""The backward pass's workspace: what the kernels write stays within the size that is asked for, and that size near what they write."""
import pytest
import torch

import tab_b200 as TAB
from tab_b200 import _cabi, nn as tab_nn


@pytest.mark.parametrize("C", [1, 100, 256, 257, 512, 1001, 1024, 2048, 4096, 4100, 8192, 8193, 16384])
@pytest.mark.parametrize("M", [1, 7, 148, 777, 8192, 1 << 20])
def test_workspace_is_a_few_rows_an_sm(M, C):
    """Five sums for each part of the rows; parts: what the device holds at once (16 CTAs an SM of the narrowest rows, one of the widest), no more than rows."""
    parts = min(4 * -(-M // 4), 148 * max(1, min(16, 8192 // C)))
    assert 5 * 4 * C <= _cabi.lib().tab_residual_norm_workspace_bytes(M, C) <= 5 * 4 * C * parts


class Watched:
    """The library, with a workspace of the test's own around which a pattern shows what was written."""
    PATTERN = 12345.678

    def __init__(self, real):
        self.real, self.guards, self.used = real, [], []

    def __getattr__(self, name):
        return getattr(self.real, name)

    def tab_residual_norm_backward_launch(self, args, stream):
        b = args._obj
        n = self.real.tab_residual_norm_workspace_bytes(b.f.M, b.f.C) // 4
        room = torch.full((n + 4 * 5 * b.f.C * 148,), self.PATTERN, device="cuda")
        b.partial = room.data_ptr()
        rc = self.real.tab_residual_norm_backward_launch(args, stream)
        self.guards.append(bool((room[n:] == self.PATTERN).all()))
        self.used.append(float((room[:n] != self.PATTERN).float().mean()))
        return rc


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("type", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M", [1, 150, 700, 4000])
@pytest.mark.parametrize("C", [64, 100, 264, 512, 1001, 1024, 1608, 2048, 4096, 5000, 8192, 9000, 16384])
def test_workspace_holds_what_the_kernels_write(cuda, monkeypatch, C, M, type, kind):
    watched = Watched(_cabi.lib())
    monkeypatch.setattr(_cabi, "lib", lambda: watched)
    monkeypatch.setattr(TAB.ops, "_native", False)
    y, x = (torch.randn(M, C, device=cuda).to(type) for _ in range(2))
    w = [torch.rand(C, device=cuda, requires_grad=True) for _ in range(5)]
    bias = dict(pre_bias=w[3], post_bias=w[4]) if kind == "layer" else {}
    out = tab_nn.residual_norm(y, x, pre_weight=w[0], post_weight=w[1], gate=w[2], kind=kind, **bias)
    torch.autograd.grad(out, w[:5 if bias else 3], [torch.ones_like(t) for t in out])
    # a centred norm's five sums are what is asked for; three of them, and fp32 rows of which an SM holds half as many, are the least of it
    assert watched.guards == [True] and watched.used[0] >= (0.5 if kind == "layer" and type == torch.bfloat16 else 0.25)
