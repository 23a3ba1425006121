"""Layouts of the tensors that the 8-bit block operators and the residual stream are given: broadcast dimensions, far sizes, what hooks hand back."""
import itertools
import types

import pytest
import torch

import tab_b200 as TAB
from tab_b200 import nn as tab_nn


def layouts():
    """Views of one buffer with every mix of broadcast, single, packed and spaced dimensions before a row of 1 or 8."""
    buffer = torch.zeros(1 << 14)
    for K, sizes in itertools.product((1, 8), itertools.product((1, 2, 3), repeat=3)):
        for strides in itertools.product((0, 1, K, 3 * K, 9 * K, 64), repeat=3):
            yield buffer.as_strided((*sizes, K), (*strides, 1))


def test_both_bodies_take_the_same_rows():
    """Which tensors are evenly spaced rows, and what their pitch is: the native bodies and those behind them agree, and what they say holds for every row."""
    host = TAB.ops._host()
    assert host, "the native bodies are not built"
    taken = 0
    for t in layouts():
        try:
            want = TAB.ops._rows(t, "t")
        except RuntimeError:
            want = None
        assert host.row_layout(t) == want, (tuple(t.shape), t.stride())
        if want is not None:
            M, K, pitch = want
            offsets = sorted(sum(i * s for i, s in zip(at, t.stride())) for at in itertools.product(*(range(n) for n in t.shape[:-1])))
            assert offsets == [i * pitch for i in range(M)]
            taken += 1
    assert taken > 100


@pytest.mark.parametrize("view", [lambda t: t[:, None].expand(4, 256, 512), lambda t: t[:, None, :1].expand(4, 256, 1), lambda t: t[:, None, None].expand(4, 3, 5, 512)])
def test_broadcast_rows_are_no_even_rows(view):
    t = view(torch.zeros(4, 512))
    assert TAB.ops._host().row_layout(t) is None and TAB.ops._host().row_layout(t.contiguous()) is not None
    with pytest.raises(RuntimeError, match="rows"):
        TAB.ops._rows(t, "t")


def test_both_bodies_take_the_same_scales(monkeypatch):
    """Scales of any even strides, those of broadcast rows among them: the native body and the one behind it agree, and what they say holds for every scale."""
    monkeypatch.setattr(TAB.ops, "_on_device", lambda *_: None)
    buffer, taken, shared = torch.zeros(4096, dtype=torch.uint8).view(torch.float8_e8m0fnu), 0, 0
    for KB, sizes, wide in itertools.product((1, 2), itertools.product((1, 2, 3), repeat=2), (False, True)):
        lead = (128 * sizes[0] * sizes[1] - 1,) if wide else sizes         # values: a row for each scale, or 128 rows
        q = torch.zeros(*lead, 128 * KB, dtype=torch.uint8).view(torch.float8_e4m3fn)
        for strides in itertools.product((0, 1, 2, 3, 4, 8, 12), (0, 1, 2, 4), (0, 1, 16)):
            s = buffer.as_strided((*sizes, KB), strides)
            try:
                want = TAB.ops._operand(q, s, "a", None)[0][4:]
            except RuntimeError:
                want = None
            got = TAB.ops._host().scale_layout(q, s)
            assert (got is None) == (want is None), (tuple(s.shape), s.stride())
            if got is None:
                continue
            flat = [sum(i * n for i, n in zip(at, strides)) for at in itertools.product(range(sizes[0]), range(sizes[1]))]
            for share, sr, sk in (got, want):
                assert share == (1 if q.numel() // (128 * KB) == len(flat) else 128) and (KB == 1 or sk == strides[2])
                assert len(flat) == 1 or flat == [i * sr for i in range(len(flat))], (tuple(s.shape), s.stride())
            taken += 1
            shared += share == 128
    assert taken > 100 and shared > 20


def test_scales_broadcast_along_one_of_two_dimensions():
    q, s = torch.zeros(5, 64, 256, dtype=torch.uint8).view(torch.float8_e4m3fn), torch.zeros(5, 1, 2, dtype=torch.uint8)
    layout = TAB.ops._host().scale_layout
    assert layout(q, s.expand(5, 64, 2)) is None and layout(q, s.expand(5, 64, 2).contiguous()) == (1, 2, 1)
    assert layout(q, s[:1, :, :1].expand(5, 64, 2)) == (1, 0, 0)


FAR = 1 << 32                                                              # what 32 bits take for 0


@pytest.mark.parametrize("shape", [(1 << 31,), (FAR,), (FAR + 5,), (1, FAR + 5), (FAR, 1), (FAR + 5, 1), (1 << 16, 1 << 16, 2)])
def test_rows_beyond_32_bits_are_refused(monkeypatch, shape):
    """Before a size meets a 32-bit parameter: neither rows nor elements of a row may be 2^31 or more.  (Meta tensors: shapes without memory.)"""
    monkeypatch.setattr(TAB.ops, "_on_device", lambda *_: None)
    x, q = torch.empty(shape, dtype=torch.bfloat16, device="meta"), torch.empty(shape, dtype=torch.float8_e4m3fn, device="meta")
    s = torch.empty((*shape[:-1], -(-shape[-1] // 128)), dtype=torch.float8_e8m0fnu, device="meta")
    few = torch.empty((1, shape[-1]), dtype=torch.float8_e4m3fn, device="meta"), torch.empty((1, s.shape[-1]), dtype=torch.float8_e8m0fnu, device="meta")
    two = (lambda t: t) if len(shape) == 2 else (lambda t: t.view(-1, t.shape[-1]))
    w = torch.empty(shape[-1], device="meta")
    for call in (lambda: TAB.ops._rows(x, "x"), lambda: TAB.quantize_blocks(x), lambda: TAB.quantize_blocks2d(two(x)), lambda: TAB.matmul_blocks(q, s, *few), lambda: TAB.matmul_blocks(*few, two(q), two(s)),
                 lambda: TAB.residual_norm(x, pre_weight=w), lambda: TAB.ops._norm_args(x, None, w, None, None, None, None, 1.0, "rms", 1e-6)):
        with pytest.raises(RuntimeError, match="2\\^31"):
            call()


def test_empty_sums_of_many_rows_are_refused(monkeypatch):
    """An empty sum is a result of zeros, however many rows the operands have; results of no rows stay what they are."""
    monkeypatch.setattr(TAB.ops, "_on_device", lambda *_: None)
    blocks = lambda *shape: (torch.empty(shape, dtype=torch.float8_e4m3fn, device="meta"), torch.empty((*shape[:-1], -(-shape[-1] // 128)), dtype=torch.float8_e8m0fnu, device="meta"))
    for a, b in ((blocks(FAR, 0), blocks(3, 0)), (blocks(3, 0), blocks(FAR, 0)), (blocks(1 << 16, 1 << 16, 0), blocks(3, 0)), (blocks(FAR + 7, 0), blocks(1, 0))):
        with pytest.raises(RuntimeError, match="2\\^31"):
            TAB.matmul_blocks(*a, *b)
    assert TAB.ops._rows(torch.empty(0, FAR, device="meta"), "t") == (0, FAR, FAR)


def test_an_older_extension_is_named(monkeypatch):
    """A native body that is not there: the extension is older than the sources, and the slow body behind it does not stand in without a word."""
    monkeypatch.setattr(TAB.ops, "_native", types.SimpleNamespace(quantize=lambda *_: None))
    assert TAB.ops._try("quantize") is None
    with pytest.raises(RuntimeError, match="older"):
        TAB.quantize_blocks(torch.zeros(2, 128))


@pytest.mark.gpu
@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("dim", [0, 1, (0, 1)])
def test_gradients_of_sums_over_tokens(cuda, monkeypatch, native, dim):
    """Autograd hands such a gradient over with broadcast dimensions: the same as from a contiguous one."""
    if not native:
        monkeypatch.setattr(TAB.ops, "_native", False)
    x, w, p = torch.randn(3, 40, 256, device=cuda, requires_grad=True), torch.randn(96, 256, device=cuda, requires_grad=True), torch.rand(256, device=cuda, requires_grad=True)
    for of, result in (((x, w), lambda: tab_nn.block_linear(x, w)), ((x, p), lambda: tab_nn.residual_norm(x, pre_weight=p)[1]), ((x,), lambda: tab_nn.residual_norm(x, x)[0])):
        g = torch.randn_like(result().sum(dim))
        y = result()
        got = torch.autograd.grad(y.sum(dim), of, g)
        full = g.expand_as(y) if dim != 1 else g[:, None].expand_as(y)
        want = torch.autograd.grad(result(), of, full.contiguous())
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize("native", [True, False])
def test_tensors_broadcast_over_tokens(cuda, monkeypatch, native):
    """One row (or one number) of each sequence for all of its tokens: refused where the kernels would need rows of their own, laid out in the
    differentiable forms, which say the same as for contiguous tensors."""
    if not native:
        monkeypatch.setattr(TAB.ops, "_native", False)
    B, S, C = 3, 40, 256
    y, p, w = torch.randn(B, S, C, device=cuda), torch.rand(C, device=cuda), torch.randn(64, C, device=cuda)
    one, number = torch.randn(B, 1, C, device=cuda), torch.randn(B, 1, 1, device=cuda)
    wide, narrow = one.expand(B, S, C), number.expand(B, S, 1)
    for call in (lambda: TAB.quantize_blocks(wide), lambda: TAB.residual_norm(wide, pre_weight=p), lambda: TAB.residual_norm(y, wide, pre_weight=p),
                 lambda: TAB.residual_norm(y, gate=wide), lambda: TAB.residual_norm(y, gate=narrow)):
        with pytest.raises(RuntimeError, match="rows"):
            call()
    for make in (lambda t: t, torch.Tensor.contiguous):
        leaves = [t.clone().requires_grad_() for t in (y, one, number, w)]
        full, token = make(leaves[1].expand(B, S, C)), make(leaves[2].expand(B, S, 1))
        out = [tab_nn.block_linear(full, leaves[3]), tab_nn.residual_norm(full, leaves[0], pre_weight=p)[1], *tab_nn.residual_norm(leaves[0], full, pre_weight=p, gate=full),
               tab_nn.residual_norm(leaves[0], full, gate=token)[0]]
        grads = torch.autograd.grad(out, leaves, [torch.ones_like(t) for t in out])
        if make is torch.Tensor.contiguous:
            assert all(torch.equal(a, b) for a, b in zip(kept, [*out, *grads]))
        kept = [*out, *grads]


@pytest.mark.gpu
@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("B, S", [(2, 3), (5, 64), (9, 128)])
def test_products_with_broadcast_scales(cuda, monkeypatch, native, B, S):
    """One row of scales for a sequence: refused, since its rows are not evenly spaced; one for everything is taken.  (The product as of laid-out scales.)"""
    if not native:
        monkeypatch.setattr(TAB.ops, "_native", False)
    a, b = TAB.quantize_blocks(torch.randn(B, S, 256, device=cuda)), TAB.quantize_blocks(torch.randn(70, 256, device=cuda))
    one = a[1][:, :1].expand(B, S, 2)
    with pytest.raises(RuntimeError, match="rows"):
        TAB.matmul_blocks(a[0], one, *b)
    for same in (a[1][:1, :1].expand(B, S, 2), a[1][:1, :1, :1].expand(B, S, 2)):
        assert torch.equal(TAB.matmul_blocks(a[0], same, *b), TAB.matmul_blocks(a[0], same.contiguous(), *b))


@pytest.mark.gpu
@pytest.mark.parametrize("n", [FAR, FAR + 300])
def test_a_flat_tensor_beyond_32_bits(cuda, n):
    """A flat vector of 2^32 elements and more has no place in 32-bit sizes and is refused; the same memory as rows is taken."""
    x = torch.zeros(n, dtype=torch.float8_e4m3fn, device=cuda)
    s = torch.full((-(-n // 128),), 127, dtype=torch.uint8, device=cuda).view(torch.float8_e8m0fnu)
    with pytest.raises(RuntimeError, match="2\\^31"):
        TAB.matmul_blocks(x, s, x[None], s[None])
    column, one = x[:, None], s.new_empty(0).set_(s.untyped_storage(), 0, (n, 1), (0, 1))
    with pytest.raises(RuntimeError, match="2\\^31"):
        TAB.matmul_blocks(TAB.ops._new_blocks((2, 1), 2, 1, x.dtype, cuda), s[:2, None], column, one)
    with pytest.raises(RuntimeError, match="2\\^31"):
        TAB.quantize_blocks(torch.empty(n, dtype=torch.bfloat16, device=cuda), columns=True)


def wider(t):
    """The same values, rows farther apart."""
    if t.dim() < 2:
        return t
    return torch.cat([t, torch.full_like(t, 7)], -1)[..., :t.shape[-1]]


def turned(t):
    """The same values, the last two dimensions the other way round in memory."""
    return t if t.dim() < 2 else t.transpose(-1, -2).contiguous().transpose(-1, -2)


@pytest.mark.gpu
@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("unpack", [wider, turned])
@pytest.mark.parametrize("shape", [(37, 100), (400, 1032), (2, 3, 64)])
def test_kept_tensors_that_come_back_with_other_strides(cuda, monkeypatch, native, unpack, shape):
    if not native:
        monkeypatch.setattr(TAB.ops, "_native", False)
    x, y = (torch.randn(*shape, device=cuda, requires_grad=True) for _ in range(2))
    p, g = torch.rand(shape[-1], device=cuda, requires_grad=True), torch.rand(shape[-1], device=cuda, requires_grad=True)
    grads = []
    for hook in (None, unpack):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, hook or (lambda t: t)):
            out = [*tab_nn.residual_norm(y, x, pre_weight=p, post_weight=p, gate=g), tab_nn.residual_norm(y, pre_weight=p)[1], tab_nn.residual_norm(y, gate=x)[0]]
        grads.append(torch.autograd.grad(out, (x, y, p, g), [torch.ones_like(t) * i for i, t in enumerate(out, 1)]))
    # rows farther apart may be worked by another kernel than packed ones: up to fp32 roundings of sums of a row, and over the rows
    for a, b in zip(*grads):
        assert float((a - b).abs().max()) <= (float(b.abs().max()) + 30) * (96 + 4 * b.numel() ** 0.5) * 2.0 ** -24


@pytest.mark.gpu
@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("unpack", [lambda t: t.half(), lambda t: t.half() if t.dim() == 2 and t.shape[-1] > 4 else t, lambda t: t.cpu(), lambda t: t[..., :-1] if t.dim() == 2 else t,
                                    lambda t: t.double() if t.shape[-1:] == (4,) else t, lambda t: t[:5] if t.dim() == 2 else t])
def test_kept_tensors_that_come_back_as_others_are_refused(cuda, monkeypatch, native, unpack):
    if not native:
        monkeypatch.setattr(TAB.ops, "_native", False)
    x, y, p = torch.randn(37, 96, device=cuda, requires_grad=True), torch.randn(37, 96, device=cuda), torch.rand(96, device=cuda)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
        out = tab_nn.residual_norm(y, x, pre_weight=p)
        plain = tab_nn.residual_norm(x, pre_weight=p)[1]
    for result in (out[0].sum() + out[1].sum(), plain.sum()):
        with pytest.raises(RuntimeError):
            result.backward()
    torch.cuda.synchronize()
