"""The residual stream between two blocks: refusals (no GPU), results and gradients against 64-bit references."""
import ctypes

import numpy as np
import pytest
import torch

import blocks_ref as ref
import tab_b200 as TAB
from tab_b200 import _cabi, nn as tab_nn

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BASE = 1 << 20
NAMES = ("y", "residual", "pre_weight", "pre_bias", "post_weight", "post_bias", "gate")


def forward_args(**over):
    a = dict(y=BASE, x=BASE, w1=BASE, w2=BASE, gate=BASE, ldy=64, ldx=64, ldg=64, type=1, ptype=0, gtype=0, gkind=2, layer=0, alpha=1.0, eps=1e-6, C=64, M=4,
             r=BASE, h=BASE, ldr=64, ldh=64)
    a.update(over)
    return _cabi.NormArgs(**a)


@pytest.mark.parametrize("over, code", [
    (dict(type=3), -1), (dict(ptype=-1), -1), (dict(gtype=7), -1), (dict(gkind=4), -1), (dict(layer=2), -1), (dict(M=-1), -1), (dict(C=-1), -1), (dict(b1=BASE), -1),
    (dict(b2=BASE), -1), (dict(M=0), 0), (dict(C=0), 0), (dict(y=None), -2), (dict(gate=None), -2), (dict(w2=None), -2), (dict(q=BASE, ldq=64), -2),
    (dict(q=BASE, s=BASE, ldq=64, lds=16, format=5), -1), (dict(q=BASE, s=BASE, ldq=256, lds=3, C=256, ldy=256, ldx=256, ldr=256, ldh=256), -1), (dict(ldy=63), -1), (dict(ldx=1), -1), (dict(ldr=0), -1), (dict(ldh=63), -1), (dict(gkind=3, ldg=63), -1),
    (dict(gkind=1, ldg=-1), -1), (dict(q=BASE, s=BASE, ldq=63), -1), (dict(y=BASE + 1), -6), (dict(w1=BASE + 2), -6), (dict(gate=BASE + 1), -6), (dict(stats=BASE + 8), -6),
    (dict(C=16385), -5), (dict(M=1 << 31), -5),
])
def test_residual_norm_refuses(over, code):
    assert _cabi.lib().tab_residual_norm_launch(ctypes.byref(forward_args(**over)), None) == code


@pytest.mark.parametrize("over, f, code", [
    ({}, dict(stats=None), -2), ({}, dict(y=None), -2), ({}, dict(r=None), -2), ({}, dict(gate=None), -2), (dict(partial=None), {}, -3), (dict(partial=BASE + 16), {}, -3),
    (dict(db1=BASE), {}, -1), (dict(ldgr=1), {}, -1), (dict(ldgh=63), {}, -1), (dict(lddy=63), {}, -1), (dict(lddx=63), {}, -1), (dict(dy=BASE + 1), {}, -6),
    (dict(dw1=BASE + 2), {}, -6), ({}, dict(C=20000), -5), ({}, dict(C=0), 0),
])
def test_residual_norm_backward_refuses(over, f, code):
    b = _cabi.NormBackwardArgs(f=forward_args(**{"stats": BASE, **f}))
    for k, v in {**dict(gr=BASE, gh=BASE, dy=BASE, dx=BASE, dgate=BASE, dw1=BASE, dw2=BASE, ldgr=64, ldgh=64, lddy=64, lddx=64, partial=BASE), **over}.items():
        setattr(b, k, v)
    assert _cabi.lib().tab_residual_norm_backward_launch(ctypes.byref(b), None) == code


def test_learned_factor_of_the_residual_is_refused():
    x = torch.zeros(2, 128)
    with pytest.raises(RuntimeError, match="residual_scale"):
        tab_nn.residual_norm(x, x, pre_weight=x[0], residual_scale=torch.ones((), requires_grad=True))


def test_workspace_and_host_tensors():
    l = _cabi.lib()
    assert l.tab_residual_norm_workspace_bytes(0, 5) == 0 and l.tab_residual_norm_workspace_bytes(5, 16385) == 0
    assert l.tab_residual_norm_workspace_bytes(1, 4096) == 5 * 4096 * 4 and l.tab_residual_norm_workspace_bytes(3, 100) == 4 * 5 * 100 * 4
    assert l.tab_residual_norm_launch(None, None) == -2 and l.tab_residual_norm_backward_launch(None, None) == -2
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        TAB.residual_norm(torch.zeros(2, 8))
    with pytest.raises(RuntimeError, match="kind"):
        TAB.residual_norm(torch.zeros(2, 8), kind="group")


def make(seed, shape, type, ptype, kind, gate, post, pre, residual, shift=0.0):
    gen = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64)
    C, dt, pt = shape[-1], TYPES[type], TYPES[ptype]
    bias = kind == "layer"
    gshape = {None: None, "channel": (C,), "token": (*shape[:-1], 1), "full": shape}[gate]
    t = dict(y=(n(*shape) + shift).to(dt), residual=(2 * n(*shape)).to(dt) if residual else None,
             pre_weight=(1 + 0.3 * n(C)).to(pt) if pre else None, pre_bias=(0.3 * n(C)).to(pt) if pre and bias else None,
             post_weight=(1 + 0.3 * n(C)).to(pt) if post else None, post_bias=(0.3 * n(C)).to(pt) if post and bias else None,
             gate=None if gate is None else n(*gshape).to(pt))
    return t, n(*shape).to(dt), n(*shape).to(dt)


def close(got, want, type, terms, scale=None, extra=0.0):
    """Half a step of the type for the last rounding; before it `terms` fp32 roundings (2^-24 each) of values of size `scale`."""
    want = want.detach().double()
    got = got.detach().double().cpu()
    scale = want.abs().max() if scale is None else scale
    bound = want.abs() * torch.finfo(TYPES[type]).eps / 2 * 1.01 + scale * terms * 2.0 ** -24 + extra + (2.0 ** -25 if type == "fp16" else 0)
    assert got.shape == want.shape and bool(((got - want).abs() <= bound).all()), float(((got - want).abs() - bound).max())


CASES = [
    # shape, type, weights, kind, gate, post, pre, residual, alpha
    ((1, 1), "fp32", "fp32", "rms", None, True, True, True, 1.0),
    ((1, 4096), "bf16", "fp32", "rms", "channel", True, True, True, 1.25),
    ((3, 7), "bf16", "bf16", "layer", "token", True, True, True, 1.0),
    ((2, 5, 100), "fp16", "fp32", "rms", "token", False, True, True, 0.5),
    ((130, 129), "fp32", "fp32", "layer", "channel", True, True, True, 2.0),
    ((600, 256), "bf16", "fp32", "rms", None, False, True, False, 1.0),
    ((64, 264), "bf16", "bf16", "rms", "full", True, True, True, 1.0),
    ((777, 1001), "fp32", "fp32", "layer", "token", True, True, True, 1.0),
    ((10, 1024), "bf16", "fp32", "layer", "full", True, True, False, 1.0),
    ((9, 2048), "fp16", "fp16", "rms", "channel", True, False, True, 1.0),
    ((300, 3000), "bf16", "fp32", "rms", "channel", True, True, True, 1.0),
    ((5, 5000), "fp32", "fp32", "layer", "channel", True, True, True, 1.0),
    ((7, 8192), "bf16", "bf16", "layer", None, True, True, True, 1.0),
    ((4, 16384), "bf16", "fp32", "rms", "channel", True, True, True, 1.0),
    ((3, 12345), "fp32", "fp32", "layer", "full", True, True, True, 1.0),
    ((2000, 64), "bf16", "fp32", "rms", "token", True, True, True, 1.0),
    # many rows
    ((1300, 264), "fp32", "fp32", "layer", "token", True, True, True, 1.0),
    ((2500, 512), "bf16", "bf16", "rms", "channel", True, True, True, 1.5),
    ((1300, 1032), "bf16", "fp32", "rms", "token", True, True, True, 1.0),
    ((700, 2048), "fp16", "fp32", "layer", "channel", True, True, True, 1.0),
    ((700, 4096), "bf16", "fp32", "rms", "channel", True, True, True, 1.25),
    ((333, 4000), "fp32", "fp32", "layer", "full", True, True, True, 1.0),
    ((640, 3064), "bf16", "bf16", "rms", None, False, True, True, 1.0),
    ((600, 2056), "bf16", "fp32", "rms", "full", True, False, False, 1.0),
    ((400, 8192), "bf16", "fp32", "layer", "channel", True, True, True, 1.0),
    ((310, 5008), "fp16", "fp32", "rms", "token", False, True, True, 1.0),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=lambda c: "x".join(map(str, c[0])) + "-" + "-".join(map(str, c[1:])))
def test_residual_norm(cuda, case):
    """Results, then every gradient.  Roundings before the last one, counted generously: a mean over the row of sums of at most 16 terms a
    thread and 10 of the tree (26), and some 14 operations on an element: 64 for results, of values of the size of the largest."""
    shape, type, ptype, kind, gate, post, pre, residual, alpha = case
    t, gr, gh = make(len(shape) + shape[-1], shape, type, ptype, kind, gate, post, pre, residual)
    leaf = {k: None if v is None else v.double().requires_grad_() for k, v in t.items()}
    r, h = ref.norm_forward(leaf, kind, 1e-5, alpha, TYPES[type])
    dev = {k: None if v is None else v.to(cuda).requires_grad_() for k, v in t.items()}
    args = dict(residual_scale=alpha, kind=kind, eps=1e-5)
    with torch.no_grad():
        plain_r, plain_h = TAB.residual_norm(**dev, **args)
    gr_, gh_ = tab_nn.residual_norm(**dev, **args)
    assert torch.equal(gr_, plain_r) and (not pre or torch.equal(gh_, plain_h))
    # an fp32 difference of 64 units of the sum may round r the other way; where r is wider than that it is at most one step of the type
    step = torch.finfo(TYPES[type]).eps if type != "fp32" else 0
    close(gr_, r, type, 64, extra=r.detach().abs() * step * 0.51)
    # the norms' outputs and gradients follow such a step of r
    if pre:
        close(gh_, h, type, 64, extra=(h.detach().abs() + leaf["pre_weight"].detach().abs()) * step * 1.1)
    wanted = [k for k in NAMES if t[k] is not None]
    grads = torch.autograd.grad((r, h) if pre else (r,), [leaf[k] for k in wanted], (gr.double(), gh.double()) if pre else (gr.double(),))
    got = torch.autograd.grad((gr_, gh_) if pre else (gr_,), [dev[k] for k in wanted], (gr.to(cuda), gh.to(cuda)) if pre else (gr.to(cuda),))
    rows = int(np.prod(shape[:-1]))
    for k, a, b in zip(wanted, got, grads):
        ty = type if k in ("y", "residual") else ptype
        summed = shape[-1] if k == "gate" and gate == "token" else rows if k not in ("y", "residual") and not (k == "gate" and gate == "full") else 1
        # a sum of n terms: sizes of terms are taken as at most 30 (deviations of products of normal variables), and 96 roundings go into a term
        size = max(float(b.detach().abs().max()), 30.0 * (1 if summed == 1 else summed ** 0.5))
        assert a.dtype == TYPES[ty]
        close(a, b, ty, 96 + summed ** 0.5 * 4, scale=size, extra=size * step * 1.1 * (0.5 if k == "residual" else 1))


@pytest.mark.gpu
@pytest.mark.parametrize("format", ["e4m3", "e5m2"])
@pytest.mark.parametrize("shape, type, kind", [((1, 4096), "bf16", "rms"), ((33, 100), "fp32", "layer"), ((2, 9, 1411), "bf16", "rms"), ((3, 9000), "fp16", "layer"), ((260, 128), "bf16", "rms"),
                                               ((700, 4096), "bf16", "rms"), ((310, 8192), "bf16", "layer"), ((600, 1416), "fp32", "rms")])
def test_residual_norm_quantized(cuda, shape, type, kind, format):
    """h as blocks: what the stored r gives in 64 bits, up to the roundings of fp32 (64 units of 2^-24 of the largest of the block) and then
    half a step of the format under the block's scale."""
    t, _, _ = make(shape[-1], shape, type, "fp32", kind, "channel", True, True, True)
    dev = {k: None if v is None else v.to(cuda) for k, v in t.items()}
    f8, largest, _, digits, bias = ref.FORMATS[format]
    r, q, s = TAB.residual_norm(**dev, kind=kind, quantize=f8)
    r0, h0 = TAB.residual_norm(**dev, kind=kind)
    assert torch.equal(r, r0) and q.dtype == f8 and q.shape == r.shape and tuple(s.shape) == (*shape[:-1], -(-shape[-1] // 128))
    C = shape[-1]
    only = {**{k: None for k in NAMES}, "y": r.double().cpu(), "pre_weight": t["pre_weight"].double(), "pre_bias": None if t["pre_bias"] is None else t["pre_bias"].double()}
    h = ref.norm_forward(only, kind, 1e-6, 1.0, torch.float64)[1].reshape(-1, C).numpy()
    qb, sb = np_flat(q, C), np_flat(s, -(-C // 128))
    v = ref.values(qb, sb, format)
    top = np.repeat(np.array([[np.abs(row[j:j + 128]).max() for j in range(0, C, 128)] for row in h]), 128, axis=1)[:, :C]
    scale = np.repeat(2.0 ** (sb.astype(float) - 127), 128, axis=1)[:, :C]
    # the scale is the least that holds the block (up to a rounding at the border)
    assert np.all(top <= largest * scale * (1 + 2.0 ** -17)) and np.all(top > largest * scale / 2 * (1 - 2.0 ** -17))
    half = np.maximum(np.abs(h) * 2.0 ** -(digits + 1), scale * 2.0 ** (1 - bias - digits) / 2)
    assert np.all(np.abs(v - h) <= half * 1.01 + top * 64 * 2.0 ** -24)


def np_flat(t, n):
    return t.contiguous().view(torch.uint8).cpu().numpy().reshape(-1, n)


@pytest.mark.gpu
def test_residual_norm_differences(cuda):
    """Gradients against differences of the fp32 function itself: (f(x + d) - f(x - d)) / 2 along random directions.  |d| = 1e-2 of unit vectors:
    cubic terms below 1e-4 of the function's size, rounding 2^-24 * size / 1e-2."""
    t, gr, gh = make(5, (6, 40), "fp32", "fp32", "layer", "channel", True, True, True)
    dev = {k: v.to(cuda) for k, v in t.items()}
    gr, gh = gr.to(cuda), gh.to(cuda)
    f = lambda d: sum(float((a.double() * g.double()).sum()) for a, g in zip(TAB.residual_norm(**d, kind="layer", eps=1e-2, residual_scale=1.5), (gr, gh)))
    leaves = {k: v.clone().requires_grad_() for k, v in dev.items()}
    grads = dict(zip(NAMES, torch.autograd.grad(tab_nn.residual_norm(**leaves, kind="layer", eps=1e-2, residual_scale=1.5), [leaves[k] for k in NAMES], (gr, gh))))
    size = float(gr.double().abs().sum() + gh.double().abs().sum())
    for k in NAMES:
        d = torch.randn(dev[k].shape, generator=torch.Generator().manual_seed(1)).to(cuda)
        d = d / d.norm() * 1e-2
        slope = (f({**dev, k: dev[k] + d}) - f({**dev, k: dev[k] - d})) / 2
        assert abs(slope - float((grads[k].double() * d.double()).sum())) <= 1e-2 * 1e-4 * size + size * 2.0 ** -24 * 4, k


@pytest.mark.gpu
def test_residual_norm_rows_apart(cuda):
    """Pitches, misaligned starts, NaN and infinities that stay in their row, rows of equal values, and an offset that a one-pass variance loses."""
    big = torch.randn(50, 700, device=cuda)
    w = torch.rand(301, device=cuda) + 0.5
    y, x = big[3:40, 5:306], big[4:41, 350:651]
    r, h = TAB.residual_norm(y, x, pre_weight=w, post_weight=w, kind="layer")
    r0, h0 = TAB.residual_norm(y.contiguous(), x.contiguous(), pre_weight=w, post_weight=w, kind="layer")
    assert torch.equal(r, r0) and torch.equal(h, h0)
    y = y.contiguous()
    y[3, 7], y[5, 0], y[9] = float("nan"), float("inf"), 2.5
    r1, h1 = TAB.residual_norm(y, x, pre_weight=w, post_weight=w, kind="layer")
    keep = [i for i in range(37) if i not in (3, 5, 9)]
    assert torch.equal(r1[keep], r0[keep]) and torch.equal(h1[keep], h0[keep])
    assert r1[3].isnan().all() and h1[3].isnan().all() and r1[5].isnan().any() and torch.equal(r1[9], x[9])
    far = torch.randn(8, 512, device=cuda, dtype=torch.float64) + 10000
    got = TAB.residual_norm(far.float(), pre_weight=torch.ones(512, device=cuda), kind="layer")[1].double()
    f = far.float().double()
    want = (f - f.mean(1, keepdim=True)) / (f.var(1, unbiased=False, keepdim=True) + 1e-6).sqrt()
    assert float((got - want).abs().max()) <= 4 * 10000 * 2.0 ** -24 * 2          # the mean is off by half a step of 10000 or so


@pytest.mark.gpu
def test_residual_norm_forms(cuda):
    """What is absent: no norms, no residual; gradients of one output only; empty batches; the same bits twice; argument errors."""
    y, x, w = (torch.randn(5, 96, device=cuda, requires_grad=True) for _ in range(2)), None, torch.rand(96, device=cuda, requires_grad=True)
    y, x = y
    r, h = TAB.residual_norm(y.detach())
    assert r.data_ptr() == y.data_ptr() and h is None
    r, h = TAB.residual_norm(y.detach(), x.detach(), residual_scale=2.0)
    assert torch.equal(r, torch.addcmul(y.detach(), x.detach(), torch.tensor(2.0, device=cuda))) and h is None
    r, h = tab_nn.residual_norm(y, pre_weight=w)
    assert r is y
    g = torch.randn(5, 96, device=cuda)
    both = torch.autograd.grad((r * 1.0, h), (y, w), (g, g))
    only_h = torch.autograd.grad(tab_nn.residual_norm(y, pre_weight=w)[1], (y, w), g)
    assert torch.equal(both[1], only_h[1]) and torch.allclose(both[0], only_h[0] + g, atol=1e-6)
    r, h = tab_nn.residual_norm(y, x, pre_weight=w)
    dy, dw = torch.autograd.grad(r, (y, w), g, allow_unused=True)
    assert torch.equal(dy, g) and (dw is None or not dw.any())
    empty = torch.zeros(0, 96, device=cuda, requires_grad=True)
    r, h = tab_nn.residual_norm(empty, empty, pre_weight=w, post_weight=w)
    assert r.shape == h.shape == (0, 96) and not torch.autograd.grad(h, w, h.detach())[0].any()
    big = torch.randn(3000, 512, device=cuda, requires_grad=True)
    wb = torch.rand(512, device=cuda, requires_grad=True)
    runs = [torch.autograd.grad(tab_nn.residual_norm(big, big, pre_weight=wb, post_weight=wb, gate=wb), (big, wb), (big.detach(), big.detach())) for _ in range(2)]
    assert all(torch.equal(a, b) for a, b in zip(*runs))
    z = torch.zeros(4, 96, device=cuda)
    for kw, words in [(dict(residual=z[:2]), "shape of y"), (dict(residual=z.half()), "residual must be"), (dict(pre_weight=w[:5]), "vector of 96"), (dict(pre_weight=w.double()), "pre_weight"),
                      (dict(pre_bias=w), "comes with"), (dict(pre_weight=w, pre_bias=w), "no bias"), (dict(gate=z[:3]), "gate must be"), (dict(quantize=torch.float8_e4m3fn), "needs pre_weight"),
                      (dict(quantize=torch.int8, pre_weight=w), "float8")]:
        with pytest.raises(RuntimeError, match=words):
            TAB.residual_norm(z, **kw)
    with pytest.raises(_cabi.TabError, match="exceeds"):
        TAB.residual_norm(torch.zeros(1, 16385, device=cuda), pre_weight=torch.ones(16385, device=cuda))


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(9, 100), (700, 1032)])
@pytest.mark.parametrize("only", NAMES)
def test_one_gradient_alone(cuda, shape, only):
    """A single gradient asked for is that of all of them: other kernels may form it, so up to fp32 roundings (as counted above)."""
    t, gr, gh = make(8, shape, "fp32", "fp32", "layer", "channel", True, True, True)
    dev = {k: v.to(cuda) for k, v in t.items()}
    grads = []
    for names in (NAMES, (only,)):
        leaves = {k: v.clone().requires_grad_(k in names) for k, v in dev.items()}
        out = tab_nn.residual_norm(**leaves, kind="layer")
        grads.append(torch.autograd.grad(out, leaves[only], (gr.to(cuda), gh.to(cuda)))[0])
    size = float(grads[0].abs().max()) + 30 * (1 if only in ("y", "residual") else shape[0] ** 0.5)
    assert float((grads[0] - grads[1]).abs().max()) <= size * (96 + 4 * shape[0] ** 0.5) * 2.0 ** -24


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(9, 100), (700, 1032), (500, 4096), (350, 8192)])
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("gate", [None, "token", "channel"])
def test_one_output_alone(cuda, shape, kind, gate):
    """Gradients of r alone and of h alone add up to those of both (fp32 roundings as counted above, for each of the three)."""
    t, gr, gh = make(9, shape, "fp32", "fp32", kind, gate, True, True, True)
    dev = {k: None if v is None else v.to(cuda).requires_grad_() for k, v in t.items() if not k.endswith("bias")}      # (centred norms without shifts, too)
    leaves = [v for v in dev.values() if v is not None]
    out = tab_nn.residual_norm(**dev, kind=kind)
    gr, gh = gr.to(cuda), gh.to(cuda)
    parts = [torch.autograd.grad(o, leaves, g, retain_graph=True, allow_unused=True) for o, g in zip(out, (gr, gh))]
    both = torch.autograd.grad(out, leaves, (gr, gh))
    for a, b, c, leaf in zip(*parts, both, leaves):
        total = sum(v for v in (a, b) if v is not None)
        size = float(c.abs().max()) + 30 * (1 if leaf.shape == c.new_empty(shape).shape else max(shape[0], shape[1] if leaf.shape[-1] == 1 else 1) ** 0.5)
        assert float((total - c).abs().max()) <= 3 * size * (96 + 4 * max(shape) ** 0.5) * 2.0 ** -24


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(6, 200), (6, 1032), (400, 4096)])
@pytest.mark.parametrize("format", ["e4m3", "e5m2"])
def test_residual_norm_quantized_non_finite(cuda, shape, format):
    """A NaN voids its row; an infinite weight makes its column infinite (NaN in e4m3) and leaves the other values of the block as they are."""
    y, w = torch.randn(*shape, device=cuda), torch.rand(shape[1], device=cuda) + 0.5
    f8 = ref.FORMATS[format][0]
    _, q0, s0 = TAB.residual_norm(y, pre_weight=w, quantize=f8)
    bad = y.clone()
    bad[2, 3] = float("nan")
    _, q, s = TAB.residual_norm(bad, pre_weight=w, quantize=f8)
    keep = [i for i in range(shape[0]) if i != 2]
    bytes_of = lambda t: t.contiguous().view(torch.uint8)
    assert q[2].float().isnan().all() and torch.equal(bytes_of(q[keep]), bytes_of(q0[keep])) and torch.equal(bytes_of(s[keep]), bytes_of(s0[keep]))
    w[5] = 0
    _, q0, s0 = TAB.residual_norm(y, pre_weight=w, quantize=f8)
    w[5] = float("inf")
    _, q, s = TAB.residual_norm(y, pre_weight=w, quantize=f8)
    column = q[:, 5].float()
    assert (column.isnan() if format == "e4m3" else column.isinf()).all()
    others = [i for i in range(shape[1]) if i != 5]
    assert torch.equal(bytes_of(s), bytes_of(s0)) and torch.equal(bytes_of(q)[:, others], bytes_of(q0)[:, others])
