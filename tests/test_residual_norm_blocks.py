"""The residual stream's results as blocks beside the same results as values: NaN and infinities in any place of a block."""
import pytest
import torch

import blocks_ref as ref
import tab_b200 as TAB

NAN, INF = float("nan"), float("inf")
bytes_of = lambda t: t.contiguous().view(torch.uint8)


def same_blocks(got, want, format):
    """Equal scales and bytes, any NaN standing for any other."""
    (q, s), (wq, ws) = ([bytes_of(t).cpu().numpy() for t in pair] for pair in (got, want))
    return bool((s == ws).all()) and ref.same_bytes(q, wq, format)


# single rows, unaligned rows, and widths on either side of every choice of threads
SHAPES = [(6, 200), (6, 203), (5, 256), (1, 512), (7, 1032), (333, 1024), (40, 2048), (300, 4096), (5, 4100), (3, 8192), (2, 8200), (2, 16384)]


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("format", ["e4m3", "e5m2"])
@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_blocks_are_those_of_the_values(cuda, shape, format, kind):
    """In fp32, where h as values is not rounded: h as blocks is what quantize_blocks makes of it, NaN, infinities and voided rows included."""
    f8, C = ref.FORMATS[format][0], shape[1]
    gen = torch.Generator(device=cuda).manual_seed(C)
    y, w = torch.randn(*shape, device=cuda, generator=gen), torch.rand(C, device=cuda, generator=gen) + 0.5
    for odd in ([], [(slice(8, 16), NAN)], [(slice(0, 8), NAN), (slice(C - 8, C), NAN)], [(slice(128, 192), NAN), (3, INF)], [(slice(24, 32), NAN), (35, -INF), (slice(64, 65), NAN)]):
        v = w.clone()
        for at, value in odd:
            v[at] = value
        for bad in (None, NAN, INF):
            x = y.clone()
            if bad is not None:
                x[shape[0] // 2, C // 3] = bad
            h = TAB.residual_norm(x, pre_weight=v, kind=kind)[1]
            q, s = TAB.residual_norm(x, pre_weight=v, kind=kind, quantize=f8)[1:]
            assert same_blocks((q, s), TAB.quantize_blocks(h, f8), format), (odd, bad)


@pytest.mark.gpu
@pytest.mark.parametrize("type", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("format", ["e4m3", "e5m2"])
def test_nan_leaves_the_other_values_of_its_block(cuda, shape, format, type):
    """Weights of NaN void their columns and nothing else: the scales are those of the other values (as with weights of zero), a voided row's those of zeros."""
    f8, C, row = ref.FORMATS[format][0], shape[1], shape[0] // 2
    gen = torch.Generator(device=cuda).manual_seed(C + 1)
    y, x = (torch.randn(*shape, device=cuda, generator=gen).to(type) for _ in range(2))
    w, p, gate = (torch.rand(C, device=cuda, generator=gen) + 0.5 for _ in range(3))
    for at in (slice(8, 16), slice(0, 64), slice(96, 128), slice(C - 8, C)):
        void, zero = w.clone(), w.clone()
        void[at], zero[at] = NAN, 0
        (r, q, s), (r0, q0, s0) = (TAB.residual_norm(y, x, pre_weight=v, post_weight=p, gate=gate, quantize=f8) for v in (void, zero))
        kept = torch.ones(C, dtype=torch.bool, device=cuda)
        kept[at] = False
        assert torch.equal(r, r0) and torch.equal(bytes_of(s), bytes_of(s0)) and torch.equal(bytes_of(q)[:, kept], bytes_of(q0)[:, kept]) and q[:, at].float().isnan().all()
    bad = y.clone()
    bad[row, C // 2] = NAN
    _, q, s = TAB.residual_norm(bad, x, pre_weight=w, post_weight=p, gate=gate, quantize=f8)
    assert q[row].float().isnan().all() and bool((bytes_of(s)[row] == 127).all())
