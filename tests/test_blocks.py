"""8-bit block quantisers and the block-scaled product: what is refused (no GPU), and the results against 64-bit references."""
import contextlib
import copy

import numpy as np
import pytest
import torch

import blocks_ref as ref
import tab_b200 as TAB
from tab_b200 import _cabi, nn as tab_nn

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
F8 = {f: v[0] for f, v in ref.FORMATS.items()}
BASE = 1 << 20                                                      # a made-up, aligned address: nothing follows it


def np_bytes(t):
    return t.contiguous().view(torch.uint8).cpu().numpy()


# ---- refusals, on the CPU ---------------------------------------------------------------------------------------------

def quantize_args(**over):
    a = dict(x=BASE, type=1, ldx=256, M=4, K=256, format=0, square=0, q=BASE, ldq=256, s=BASE, lds=16, qt=None, ldqt=0, st=None, ldst=0)
    a.update(over)
    return [*a.values(), None]


@pytest.mark.parametrize("over, code", [
    (dict(type=3), -1), (dict(type=-1), -1), (dict(format=2), -1), (dict(square=2), -1), (dict(M=-1), -1), (dict(K=-1), -1),
    (dict(M=0), 0), (dict(K=0), 0), (dict(x=None), -2), (dict(q=None), -2), (dict(s=None), -2), (dict(qt=BASE, ldqt=16, ldst=256), -2),
    (dict(square=1, q=None, s=None), -2), (dict(ldx=255), -1), (dict(ldq=255), -1), (dict(qt=BASE, st=BASE, ldqt=3, ldst=256), -1), (dict(lds=3), -1), (dict(qt=BASE, st=BASE, ldqt=16, M=129, ldst=255, lds=256), -1), (dict(square=1, M=129, lds=1), -1),
    (dict(square=1, qt=BASE, st=BASE, ldqt=16, lds=2, ldst=0), -1), (dict(lds=1 << 40), -5),
    (dict(x=BASE + 1), -6), (dict(type=0, x=BASE + 2), -6), (dict(M=1 << 31, lds=1 << 31), -5), (dict(ldx=1 << 40), -5),
])
def test_quantize_blocks_refuses(over, code):
    assert _cabi.lib().tab_quantize_blocks_launch(*quantize_args(**over)) == code


def matmul_args(**over):
    a = dict(a=BASE, af=0, lda=256, as_=BASE, ash=1, ar=2, ab=1, b=BASE, bf=0, ldb=256, bs=BASE, bsh=128, br=2, bb=1, y=BASE, type=1, ldy=64, M=4, N=64, K=256)
    a.update(over)
    return [*a.values(), None]


@pytest.mark.parametrize("over, code", [
    (dict(af=2), -1), (dict(bf=-1), -1), (dict(type=4), -1), (dict(ash=2), -1), (dict(bsh=0), -1), (dict(M=-1), -1), (dict(N=-1), -1), (dict(K=-1), -1),
    (dict(M=0), 0), (dict(N=0), 0), (dict(lda=255), -1), (dict(ldb=128), -1), (dict(ldy=63), -1), (dict(a=None), -2), (dict(b=None), -2), (dict(as_=None), -2),
    (dict(bs=None), -2), (dict(y=None), -2), (dict(a=BASE + 8), -6), (dict(b=BASE + 1), -6), (dict(lda=264), -6), (dict(ldb=257), -6), (dict(y=BASE + 1), -6),
    (dict(type=0, y=BASE + 2), -6), (dict(ldy=1 << 40), -5), (dict(lda=1 << 40), -5), (dict(K=2 ** 31 - 1, lda=1 << 32, ldb=1 << 32), -5),
])
def test_matmul_blocks_refuses(over, code):
    assert _cabi.lib().tab_matmul_blocks_launch(*matmul_args(**over)) == code


@pytest.mark.parametrize("K", [2 ** 31 - 1, 2 ** 31 - 255])
@pytest.mark.parametrize("square", [0, 1])
def test_quantize_blocks_refuses_rows_beyond_its_indexes(K, square):
    """Columns are counted in 32 bits, two blocks at a time."""
    over = dict(K=K, M=1, lds=1 << 25, square=square)
    assert _cabi.lib().tab_quantize_blocks_launch(*quantize_args(**over)) == -5
    assert _cabi.lib().tab_quantize_blocks_launch(*quantize_args(**over, qt=BASE, st=BASE, ldqt=16, ldst=1 << 31)) == -5


@pytest.mark.parametrize("x, w", [((2 ** 24 + 1, 2), (3, 2)), ((4096, 4097, 2), (3, 2)), ((3, 2), (2 ** 24 + 1, 2)), ((1, 2 ** 24 + 1), (1, 2 ** 24 + 1))])
def test_block_linear_refuses_longer_sums(x, w):
    """Before the forward pass, not in the backward pass that would need them."""
    with pytest.raises(RuntimeError, match="2\\^24"):
        tab_nn.block_linear(torch.zeros(1).expand(x), torch.zeros(1).expand(w))


def test_block_linear_refuses_types_before_the_backward_pass():
    x = torch.zeros(2, 128)
    for over in (dict(grad_dtype=torch.float8_e4m3fnuz), dict(grad_dtype=torch.bfloat16), dict(out_dtype=torch.float64)):
        with pytest.raises(RuntimeError, match="grad_dtype must be"):
            tab_nn.block_linear(x, x, **over)


def test_operators_refuse_host_tensors():
    x = torch.zeros(2, 128)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        TAB.quantize_blocks(x)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        TAB.quantize_blocks2d(x)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        TAB.matmul_blocks(x, x, x, x)
    with pytest.raises(RuntimeError, match="float8"):
        TAB.quantize_blocks(x, torch.int8)
    with pytest.raises(ValueError, match="Wq"):
        tab_nn.BlockLinear(torch.zeros(2, 128), torch.zeros(1, 2))


def test_row_layouts():
    """What counts as evenly spaced rows (the arithmetic that hands pitches to the kernels)."""
    rows = TAB.ops._rows
    t = torch.zeros(6, 5, 40)
    assert rows(t, "t") == (30, 40, 40)
    assert rows(t[:, 0], "t") == (6, 40, 200)
    assert rows(t[..., :7], "t") == (30, 7, 40)
    assert rows(t[0, 0], "t") == (1, 40, 40)
    assert rows(t[:0], "t")[0] == 0 and rows(t[..., :0], "t")[1] == 0
    assert rows(torch.zeros(0, 0), "t")[:2] == (0, 0)
    for bad in (t[:, :3], t[..., ::2], t.transpose(0, 1), t[:1, :1].expand(3, 1, 40), torch.zeros(())):
        with pytest.raises(RuntimeError):
            rows(bad, "t")
    for shape in ((3, 7), (2, 3, 7), (7,), (3, 32), (2, 2, 32), (0, 7), (4, 0)):
        q = TAB.ops._new_blocks(shape, int(np.prod(shape[:-1])), shape[-1], torch.float8_e4m3fn, "cpu")
        assert tuple(q.shape) == shape and (q.numel() == 0 or q.dim() == 1 or rows(q, "q")[2] % 16 == 0)


# ---- quantisers -------------------------------------------------------------------------------------------------------

def spread(seed, M, K, dtype):
    """Values over many magnitudes: blocks of large, small, subnormal and zero values, ties between neighbours, the types' ends."""
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((M, K)) * 2.0 ** rng.integers(-20, 8, (M, 1)) * 2.0 ** rng.integers(-6, 7, (1, K))
    x[rng.random((M, K)) < 0.1] = 0
    t = torch.from_numpy(x).to(dtype)
    if M > 3 and K > 3:
        t[1, :] = 0
        t[2, :min(K, 128)] = torch.linspace(-448, 448, min(K, 128)).to(dtype)
        t[3, ::3] = torch.finfo(dtype).max
        t[M - 1, :] = torch.finfo(dtype).tiny / 4
        t[0, K // 2] = -0.0
    return t


@pytest.mark.gpu
@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("format", F8)
@pytest.mark.parametrize("M, K", [(1, 1), (1, 128), (3, 127), (16, 129), (128, 128), (130, 300), (257, 64), (5, 2100), (300, 1000)])
def test_quantize_blocks(cuda, type, format, M, K):
    x = spread(M * 1000 + K, M, K, TYPES[type])
    v = x.double().numpy()
    want, ws = ref.quantize(v, format)
    want_t, wst = ref.quantize(v.T.copy(), format)
    xd = x.to(cuda)
    q, s = TAB.quantize_blocks(xd, F8[format])
    assert q.shape == (M, K) and s.shape == (M, -(-K // 128)) and (M == 1 or q.stride(0) % 16 == 0)
    assert np.array_equal(np_bytes(s), ws) and ref.same_bytes(np_bytes(q), want, format)
    q, s, qt, st = TAB.quantize_blocks(xd, F8[format], columns=True)
    assert np.array_equal(np_bytes(s), ws) and ref.same_bytes(np_bytes(q), want, format)
    assert np.array_equal(np_bytes(st), wst) and ref.same_bytes(np_bytes(qt), want_t, format)
    want, ws = ref.quantize(v, format, square=True)
    q, s, qt, st = TAB.quantize_blocks2d(xd, F8[format], transposed=True)
    assert np.array_equal(np_bytes(s), ws) and ref.same_bytes(np_bytes(q), want, format)
    assert np.array_equal(np_bytes(st), ws.T) and ref.same_bytes(np_bytes(qt), want.T, format)
    q, s = TAB.quantize_blocks2d(xd, F8[format])
    assert np.array_equal(np_bytes(s), ws) and ref.same_bytes(np_bytes(q), want, format)


@pytest.mark.gpu
@pytest.mark.parametrize("format", F8)
@pytest.mark.parametrize("type", TYPES)
def test_quantize_blocks_non_finite(cuda, type, format):
    x = spread(5, 40, 260, TYPES[type])
    x[4, 7], x[4, 200], x[5, :] = float("nan"), float("inf"), float("-inf")
    x[6, 130:256] = float("nan")
    v = x.double().numpy()
    q, s, qt, st = TAB.quantize_blocks(x.to(cuda), F8[format], columns=True)
    for got, gs, want in ((q, s, v), (qt, st, v.T.copy())):
        wq, ws = ref.quantize(want, format)
        assert np.array_equal(np_bytes(gs), ws) and ref.same_bytes(np_bytes(got), wq, format)


@pytest.mark.gpu
def test_quantize_blocks_strided_and_bounded(cuda):
    """Slices with a row pitch and odd starts; bytes behind the rows and behind the last row stay as they are."""
    big = spread(9, 70, 700, torch.bfloat16).to(cuda)
    for cut in (big[3:60, 5:402], big[::2, 16:272], big.view(10, 7, 700)[:, 2]):
        q, s = TAB.quantize_blocks(cut)
        wq, ws = ref.quantize(cut.double().cpu().numpy(), "e4m3")
        assert np.array_equal(np_bytes(s), ws) and ref.same_bytes(np_bytes(q), wq, "e4m3")
    l, x = _cabi.lib(), big[:9, :200].contiguous()
    for qt in (None, torch.full((202, 16), 0xAA, dtype=torch.uint8, device=cuda)):
        q, s, st = (torch.full(z, 0xAA, dtype=torch.uint8, device=cuda) for z in ((11, 208), (3, 13), (2, 207)))
        assert l.tab_quantize_blocks_launch(x.data_ptr(), 1, 200, 9, 200, 0, 0, q.data_ptr(), 208, s.data_ptr(), 13, qt.data_ptr() if qt is not None else None, 16,
                                            st.data_ptr(), 207, torch.cuda.current_stream().cuda_stream) == 0
        wq, ws = ref.quantize(x.double().cpu().numpy(), "e4m3")
        assert np.array_equal(q[:9, :200].cpu().numpy(), wq) and np.array_equal(s[:2, :9].cpu().numpy(), ws.T)
        assert bool((q[:, 200:] == 0xAA).all()) and bool((q[9:] == 0xAA).all()) and bool((s[:, 9:] == 0xAA).all()) and bool((s[2:] == 0xAA).all())
        if qt is not None:
            assert bool((qt[:, 9:] == 0xAA).all()) and bool((qt[200:] == 0xAA).all()) and bool((st[:, 200:] == 0xAA).all()) and bool((st[1:] == 0xAA).all())


# ---- product ----------------------------------------------------------------------------------------------------------

def random_blocks(rng, rows, K, format, squares, whole):
    """Bytes and scale bytes; whole: small whole numbers under scales 1, 2, 4, whose products and sums fp32 holds exactly."""
    R, KB = (-(-rows // 128) if squares else rows), -(-K // 128)
    if whole:
        table = ref.decode(format)
        numbers = np.array([int(np.flatnonzero(table == v)[0]) for v in (-3.0, -2.0, -1.0, 0.0, 1.0, 2.0, 3.0, 4.0)], np.uint8)
        return numbers[rng.integers(0, 8, (rows, K))], (127 + rng.integers(0, 3, (R, KB))).astype(np.uint8)
    q = rng.integers(0, 256, (rows, K)).astype(np.uint8)
    bad = ~np.isfinite(ref.decode(format))[q]
    q[bad] = 0x31
    return q, (127 + rng.integers(-9, 10, (R, KB))).astype(np.uint8)


def device_blocks(cuda, q, s, format):
    rows, K = q.shape
    held = torch.full((rows, -(-K // 16) * 16), 0x55, dtype=torch.uint8, device=cuda)        # what lies behind the rows must not count
    held[:, :K] = torch.from_numpy(q).to(cuda)
    return held.view(F8[format])[:, :K], torch.from_numpy(s).to(cuda).view(torch.float8_e8m0fnu)


SIZES = [(1, 1, 1), (1, 128, 128), (1, 256, 1024), (2, 130, 96), (5, 512, 4096), (16, 100, 640), (17, 1000, 1040), (33, 64, 513), (64, 384, 256), (100, 129, 300),
         (128, 128, 127), (129, 257, 1000), (200, 2048, 512), (256, 256, 2048), (300, 300, 100), (513, 777, 1411), (1024, 512, 384), (40, 1024, 6000), (257, 1, 4100), (1, 5, 30000),
         (2304, 1300, 700), (2600, 2900, 300), (1030, 10000, 513), (5000, 4100, 130),
         (8, 72, 4500), (9, 1000, 4224), (16, 129, 16500), (24, 4000, 4096), (33, 9000, 8200), (64, 20000, 520), (65, 64, 9000), (140, 4100, 5000), (1000, 2100, 384), (1024, 16, 4096), (1500, 1500, 640)]


@pytest.mark.gpu
@pytest.mark.parametrize("squares, turned", [((False, True), False), ((False, False), False), ((True, True), False), ((False, False), True)])
@pytest.mark.parametrize("M, N, K", SIZES)
def test_matmul_blocks_exact(cuda, M, N, K, squares, turned):
    """Whole numbers: |product| <= 4 * 4 * 4 * 4, sums of 30000 of them stay below 2^24, so every order of additions gives the same."""
    rng = np.random.default_rng(M + 3 * N + 7 * K)
    fa, fb = ("e4m3", "e5m2") if K % 2 else ("e4m3", "e4m3")
    a, b = random_blocks(rng, M, K, fa, squares[0], True), random_blocks(rng, N, K, fb, squares[1], True)
    want = ref.values(*a, fa) @ ref.values(*b, fb).T
    (qa, sa), (qb, sb) = device_blocks(cuda, *a, fa), device_blocks(cuda, *b, fb)
    if turned:                                                      # as quantize_blocks lays them out: block by block
        sa, sb = (TAB.ops._new_scales(tuple(s.shape), *s.shape, cuda).copy_(s) for s in (sa, sb))
    y = TAB.matmul_blocks(qa, sa, qb, sb, out_dtype=torch.float32)
    assert y.shape == (M, N) and np.array_equal(y.cpu().numpy(), want)
    assert _cabi.lib().tab_device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("formats", [("e4m3", "e4m3"), ("e5m2", "e4m3"), ("e4m3", "e5m2"), ("e5m2", "e5m2")])
@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("M, N, K", [(1, 300, 1000), (31, 129, 640), (150, 260, 1411), (300, 520, 2048)])
def test_matmul_blocks(cuda, M, N, K, type, formats):
    """Any bytes and scales.  Products are exact in fp32; K additions, each off by at most 2^-23 of the running sum of magnitudes, then
    one rounding to the result's type (half its eps of the result; fp16 below 2^-14 in steps of 2^-24)."""
    rng = np.random.default_rng(M + N + K)
    fa, fb = formats
    a, b = random_blocks(rng, M, K, fa, False, False), random_blocks(rng, N, K, fb, True, False)
    va, vb = ref.values(*a, fa), ref.values(*b, fb)
    if type == "fp16":                                              # keep within the type: scale rows of a down by a power of two
        shift = int(np.ceil(np.log2(np.abs(va) @ np.abs(vb).T).max())) - 15
        a = (a[0], (a[1].astype(int) - max(shift, 0)).astype(np.uint8))
        va = ref.values(*a, fa)
    want, size = va @ vb.T, np.abs(va) @ np.abs(vb).T
    y = TAB.matmul_blocks(*device_blocks(cuda, *a, fa), *device_blocks(cuda, *b, fb), out_dtype=TYPES[type]).double().cpu().numpy()
    eps = torch.finfo(TYPES[type]).eps / 2
    bound = size * K * 2.0 ** -23 * (1 + eps) + np.abs(want) * eps + (2.0 ** -25 if type == "fp16" else 0)
    assert np.all(np.abs(y - want) <= bound)


@pytest.mark.gpu
def test_matmul_blocks_non_finite(cuda):
    """A NaN or an infinity reaches the results of its own row and column only."""
    rng = np.random.default_rng(3)
    a, b = random_blocks(rng, 140, 300, "e5m2", False, True), random_blocks(rng, 200, 300, "e4m3", True, True)
    want = ref.values(*a, "e5m2") @ ref.values(*b, "e4m3").T
    a[0][7, 200], a[0][139, 0], b[0][150, 299] = 0x7F, 0x7E, 0x7F
    y = TAB.matmul_blocks(*device_blocks(cuda, *a, "e5m2"), *device_blocks(cuda, *b, "e4m3"), out_dtype=torch.float32).cpu().numpy()
    hit = np.zeros_like(want, bool)
    hit[7], hit[139], hit[:, 150] = True, True, True
    assert np.isnan(y[hit]).all() and np.array_equal(y[~hit], want[~hit])


@pytest.mark.gpu
@pytest.mark.parametrize("M, N", [(3, 200), (40, 200), (200, 300), (2304, 1300)])
def test_matmul_blocks_nan_scales(cuda, M, N):
    """A scale of NaN (the byte 255) voids the results of its row, or of its square's rows, and no others; whole kernels apart."""
    rng = np.random.default_rng(M)
    a, b = random_blocks(rng, M, 520, "e4m3", False, True), random_blocks(rng, N, 520, "e4m3", True, True)
    want = ref.values(*a, "e4m3") @ ref.values(*b, "e4m3").T
    a[1][M - 1, 2], b[1][1, 4] = 255, 255
    y = TAB.matmul_blocks(*device_blocks(cuda, *a, "e4m3"), *device_blocks(cuda, *b, "e4m3"), out_dtype=torch.float32).cpu().numpy()
    hit = np.zeros_like(want, bool)
    hit[M - 1], hit[:, 128:256] = True, True
    assert np.isnan(y[hit]).all() and np.array_equal(y[~hit], want[~hit])


@pytest.mark.gpu
@pytest.mark.parametrize("M, N", [(2, 100), (40, 200), (200, 300), (2304, 1300)])
def test_matmul_blocks_far_scales(cuda, M, N):
    """Scales at the ends of their range whose products are not: 2^-120 against 2^100."""
    rng = np.random.default_rng(N)
    a, b = random_blocks(rng, M, 300, "e4m3", False, True), random_blocks(rng, N, 300, "e4m3", False, True)
    want = ref.values(*a, "e4m3") @ ref.values(*b, "e4m3").T
    far = lambda o, e: (o[0], (o[1].astype(int) + e).astype(np.uint8))
    y = TAB.matmul_blocks(*device_blocks(cuda, *far(a, -120), "e4m3"), *device_blocks(cuda, *far(b, 100), "e4m3"), out_dtype=torch.float32).cpu().numpy()
    assert np.array_equal(y.astype(np.float64) * 2.0 ** 20, want)


@pytest.mark.gpu
def test_blocks_beyond_32_bits(cuda):
    """More than 2^31 values: quantised along both axes and multiplied; rows near the ends against the reference."""
    M, K, N = 66000, 32768 + 128, 16
    rows = [0, 1, 31337, 65279, M - 2, M - 1]
    x = torch.empty(M, K, dtype=torch.bfloat16, device=cuda)
    gen = torch.Generator(device=cuda).manual_seed(1)
    for i in range(0, M, 6000):
        x[i:i + 6000].normal_(generator=gen)
    q, s, qt, st = TAB.quantize_blocks(x, columns=True)
    v = x[rows].double().cpu().numpy()
    wq, ws = ref.quantize(v, "e4m3")
    assert ref.same_bytes(np_bytes(q[rows]), wq, "e4m3") and np.array_equal(np_bytes(s[rows]), ws)
    cols = [0, 127, 20000, K - 1]
    wq, ws = ref.quantize(x[:, cols].t().contiguous().double().cpu().numpy(), "e4m3")
    assert ref.same_bytes(np_bytes(qt[cols]), wq, "e4m3") and np.array_equal(np_bytes(st[cols]), ws)
    del qt, st, x
    b = random_blocks(np.random.default_rng(2), N, K, "e4m3", True, True)
    y = TAB.matmul_blocks(q, s, *device_blocks(cuda, *b, "e4m3"), out_dtype=torch.float32)
    qa, sa = np_bytes(q[rows]), np_bytes(s[rows])
    va, vb = ref.values(qa, sa, "e4m3"), ref.values(*b, "e4m3")
    assert np.all(np.abs(y[rows].double().cpu().numpy() - va @ vb.T) <= np.abs(va) @ np.abs(vb).T * K * 2.0 ** -23)
    assert _cabi.lib().tab_device_status() == 0


@pytest.mark.gpu
def test_matmul_blocks_layouts(cuda):
    """Leading dimensions, scales of any strides, slices of operands, an empty sum, empty results, bytes behind the result."""
    rng = np.random.default_rng(4)
    a, b = random_blocks(rng, 60, 512, "e4m3", False, True), random_blocks(rng, 300, 512, "e4m3", True, True)
    want = ref.values(*a, "e4m3") @ ref.values(*b, "e4m3").T
    (qa, sa), (qb, sb) = device_blocks(cuda, *a, "e4m3"), device_blocks(cuda, *b, "e4m3")
    y = TAB.matmul_blocks(qa.view(3, 20, 512), sa.view(3, 20, 4), qb, sb, out_dtype=torch.float32)
    assert y.shape == (3, 20, 300) and np.array_equal(y.cpu().numpy().reshape(60, 300), want)
    turned = sa.view(torch.uint8).t().contiguous().t().view(torch.float8_e8m0fnu)
    wide = torch.zeros(3, 9, dtype=torch.uint8, device=cuda)
    wide[:, 1::2] = sb.view(torch.uint8)
    y = TAB.matmul_blocks(qa, turned, qb, wide[:, 1::2].view(torch.float8_e8m0fnu), out_dtype=torch.float32)
    assert np.array_equal(y.cpu().numpy(), want)
    part = ref.values(*a, "e4m3")[10:50, 128:400] @ ref.values(*b, "e4m3")[128:256, 128:400].T
    y = TAB.matmul_blocks(qa[10:50, 128:400], sa[10:50, 1:4], qb[128:256, 128:400], sb[1:2, 1:4], out_dtype=torch.float32)
    assert np.array_equal(y.cpu().numpy(), part)
    empty = TAB.matmul_blocks(qa[:, :0], sa[:, :0], qb[:, :0], sb[:, :0])
    assert empty.shape == (60, 300) and not empty.any()
    assert TAB.matmul_blocks(qa[:0], sa[:0], qb, sb).shape == (0, 300) and TAB.matmul_blocks(qa, sa, qb[:0], sb[:0]).shape == (60, 0)
    l = _cabi.lib()
    for M, N in ((60, 299), (3, 200), (1, 77)):
        out = torch.full((M + 1, 304), 7.0, device=cuda)
        assert l.tab_matmul_blocks_launch(qa.data_ptr(), 0, 512, sa.data_ptr(), 1, 4, 1, qb.data_ptr(), 0, 512, sb.data_ptr(), 128, 4, 1, out.data_ptr(), 0, 304, M, N, 512,
                                          torch.cuda.current_stream().cuda_stream) == 0
        assert np.array_equal(out[:M, :N].cpu().numpy(), want[:M, :N]) and bool((out[:, N:] == 7).all()) and bool((out[M:] == 7).all())


@pytest.mark.gpu
def test_matmul_blocks_argument_errors(cuda):
    q, s = TAB.quantize_blocks(torch.randn(4, 256, device=cuda))
    w, ws = TAB.quantize_blocks2d(torch.randn(300, 256, device=cuda))
    for args, words in [((q, s[:, :1], w, ws), "a_scales"), ((q, s[:3], w, ws), "a_scales has 3"), ((q, s, w, ws[:2]), "b_scales has 2"), ((q, s.float(), w, ws), "e8m0"),
                        ((q, s, w[:, :128], ws[:, :1]), "b must be"), ((q[:, 1:129], s[:, :1], w[:, :128], ws[:, :1]), "16 bytes"), ((q.float(), s, w, ws), "8-bit")]:
        with pytest.raises(RuntimeError, match=words):
            TAB.matmul_blocks(*args)
    with pytest.raises(RuntimeError, match="out_dtype"):
        TAB.matmul_blocks(q, s, w, ws, out_dtype=torch.float64)
    with pytest.raises(RuntimeError, match="float32, bfloat16 or float16"):
        TAB.quantize_blocks(torch.zeros(2, 2, device=cuda, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="contiguous rows"):
        TAB.quantize_blocks(torch.zeros(4, 8, device=cuda).t())


# ---- dense layers -----------------------------------------------------------------------------------------------------

def layer_reference(x, w, g, grad_format):
    """block_linear's result and gradients in float64."""
    v = lambda t, f="e4m3", square=False: ref.values(*ref.quantize(t, f, square), f)
    wv = v(w, square=True)
    return v(x) @ wv.T, v(g, grad_format) @ wv, v(g.T.copy(), grad_format) @ v(x.T.copy()).T


@pytest.mark.gpu
@pytest.mark.parametrize("grad_format", F8)
@pytest.mark.parametrize("M, N, K, type, wtype", [(1, 16, 40, "bf16", "fp32"), (70, 200, 129, "fp32", "fp32"), (260, 128, 384, "bf16", "bf16"), (130, 513, 256, "fp16", "fp32")])
def test_block_linear_gradients(cuda, M, N, K, type, wtype, grad_format):
    gen = torch.Generator().manual_seed(M)
    x, w = torch.randn(M, K, generator=gen).to(TYPES[type]), (torch.randn(N, K, generator=gen) / K ** 0.5).to(TYPES[wtype])
    g = torch.randn(M, N, generator=gen).to(TYPES[type])
    want = layer_reference(x.double().numpy(), w.double().numpy(), g.double().numpy(), grad_format)
    xd, wd = x.to(cuda).requires_grad_(), w.to(cuda).requires_grad_()
    y = tab_nn.block_linear(xd, wd, grad_dtype=F8[grad_format])
    y.backward(g.to(cuda))
    for got, wanted, terms, t in ((y, want[0], K, type), (xd.grad, want[1], N, type), (wd.grad, want[2], M, wtype)):
        got = got.detach().double().cpu().numpy()
        # additions as in test_matmul_blocks; the magnitudes that are summed are at most sqrt(terms) times their norm, here bounded by the largest value
        bound = np.abs(wanted).max() * 8 * terms ** 0.5 * terms * 2.0 ** -23 + np.abs(wanted) * torch.finfo(TYPES[t]).eps / 2 + 2.0 ** -25
        assert got.shape == wanted.shape and np.all(np.abs(got - wanted) <= bound)
    # only what is asked for
    assert torch.equal(torch.autograd.grad(tab_nn.block_linear(xd, w.to(cuda), grad_dtype=F8[grad_format]), xd, g.to(cuda))[0], xd.grad)
    assert torch.equal(torch.autograd.grad(tab_nn.block_linear(x.to(cuda), wd, grad_dtype=F8[grad_format]), wd, g.to(cuda))[0], wd.grad)


@pytest.mark.gpu
def test_block_linear_odd_gradients(cuda):
    """Gradients that autograd hands over expanded or transposed, leading dimensions, no rows at all."""
    w = torch.randn(96, 64, device=cuda)
    x = torch.randn(3, 5, 64, device=cuda, requires_grad=True)
    dx, = torch.autograd.grad(tab_nn.block_linear(x, w).sum(), x)
    full, = torch.autograd.grad(tab_nn.block_linear(x, w), x, torch.ones(3, 5, 96, device=cuda))
    assert dx.shape == x.shape and torch.equal(dx, full)
    g = torch.randn(96, 5, 3, device=cuda)
    a, = torch.autograd.grad(tab_nn.block_linear(x, w), x, g.permute(2, 1, 0))
    b, = torch.autograd.grad(tab_nn.block_linear(x, w), x, g.permute(2, 1, 0).contiguous())
    assert torch.equal(a, b)
    e, wl = torch.zeros(0, 64, device=cuda, requires_grad=True), w.clone().requires_grad_()
    y = tab_nn.block_linear(e, wl)
    dx, dw = torch.autograd.grad(y, (e, wl), torch.zeros(0, 96, device=cuda))
    assert y.shape == (0, 96) and dx.shape == (0, 64) and not dw.any()


@pytest.mark.gpu
def test_block_linear_module(cuda):
    w, x = torch.randn(200, 300, device=cuda), torch.randn(2, 9, 300, device=cuda, dtype=torch.bfloat16)
    m = tab_nn.BlockLinear.from_float(w)
    q, s = TAB.quantize_blocks(x)
    want = TAB.matmul_blocks(q, s, m.Wq, m.Ws)
    assert torch.equal(m(x), want) and torch.equal(m(q, s), want) and torch.equal(tab_nn.block_linear(x, w), want)
    other = tab_nn.BlockLinear.from_float(torch.zeros(200, 300, device=cuda))
    other.load_state_dict(m.state_dict())
    assert torch.equal(other(x), want)
    with pytest.raises(ValueError, match="300"):
        m(x[..., :128])


@pytest.mark.gpu
def test_both_bodies_agree(cuda, monkeypatch):
    """The native bodies and those behind them (taken where the extension is missing): the same bits, values and gradients."""
    x, w = torch.randn(3, 45, 300, device=cuda, dtype=torch.bfloat16), torch.randn(130, 300, device=cuda)
    p, gate = torch.rand(300, device=cuda), torch.rand(3, 45, 1, device=cuda)

    def everything():
        out = [*TAB.quantize_blocks(x, columns=True), *TAB.quantize_blocks2d(w, torch.float8_e5m2, transposed=True)]
        out += [TAB.matmul_blocks(*out[:2], *out[4:6]), *TAB.residual_norm(x, x, pre_weight=p, post_weight=p, gate=gate, quantize=torch.float8_e4m3fn)]
        for plain in (False, True):
            leaves = [t.clone().requires_grad_() for t in (x, w, p, gate)]
            r, h = tab_nn.residual_norm(leaves[0], pre_weight=leaves[2]) if plain else tab_nn.residual_norm(leaves[0], x, pre_weight=leaves[2], post_weight=p, gate=leaves[3], residual_scale=0.5)
            y = tab_nn.block_linear(h, leaves[1])
            grads = torch.autograd.grad((y, r), leaves[:3 if plain else 4], (torch.ones_like(y), torch.ones_like(r)))
            out += [y.detach(), *grads]
        return [t.view(torch.uint8) if t.dtype.itemsize == 1 else t for t in out]

    if not TAB.ops._host():
        pytest.fail("the native bodies are not built")
    native = everything()
    monkeypatch.setattr(TAB.ops, "_native", False)
    for a, b in zip(native, everything()):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("native", [True, False])
def test_second_derivatives_are_refused(cuda, monkeypatch, native):
    if not native:
        monkeypatch.setattr(TAB.ops, "_native", False)
    x, w, p = (torch.randn(*s, device=cuda, requires_grad=True) for s in ((4, 128), (16, 128), (128,)))
    for y in (tab_nn.block_linear(x, w), tab_nn.residual_norm(x, pre_weight=p)[1]):
        g, = torch.autograd.grad(y.sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="differentiable"):
            g.sum().backward()


@pytest.mark.parametrize("K", [100, 256])
def test_block_linear_module_on_the_host(K):
    """Changes of type leave 8-bit values and scales as they are, from tensors without gaps between rows too, and rows start on 16 bytes."""
    wq, ws = torch.randint(0, 127, (40, K), dtype=torch.uint8), torch.randint(100, 140, (1, -(-K // 128)), dtype=torch.uint8)
    m = tab_nn.BlockLinear(wq.view(torch.float8_e4m3fn), ws.view(torch.float8_e8m0fnu))
    for change in (lambda m: m.half(), lambda m: m.to(torch.bfloat16), lambda m: torch.nn.Sequential(m).double()[0], lambda m: m.cpu(), copy.deepcopy):
        m = change(m)
        assert m.Wq.dtype == torch.float8_e4m3fn and m.Ws.dtype == torch.float8_e8m0fnu and m.Wq.stride(0) % 16 == 0 and m.Wq.data_ptr() % 16 == 0
        assert torch.equal(m.Wq.view(torch.uint8), wq) and torch.equal(m.Ws.view(torch.uint8), ws)


@pytest.mark.gpu
@pytest.mark.parametrize("K", [100, 256])
def test_block_linear_module_moves(cuda, K):
    w, x = torch.randn(70, K, device=cuda), torch.randn(9, K, device=cuda)
    m = tab_nn.BlockLinear.from_float(w)
    want = m(x)
    m = torch.nn.Sequential(m).half().cpu().cuda()[0]
    assert want.dtype == torch.bfloat16 and torch.equal(m(x), want) and torch.equal(tab_nn.BlockLinear(m.Wq.contiguous(), m.Ws)(x), want)


# ---- together, as they are used ---------------------------------------------------------------------------------------

def block_step(x, params, training):
    """A residual block's dense half: norm, up, rectifier squared, down, norm, gate, residual, next norm."""
    w1, w2, up, down, gate = params
    if training:
        h = tab_nn.residual_norm(x, pre_weight=w1)[1]
        y = tab_nn.block_linear(torch.relu(tab_nn.block_linear(h, up)).square(), down)
        return tab_nn.residual_norm(y, x, pre_weight=w1, post_weight=w2, gate=gate, residual_scale=0.9)
    _, q, s = TAB.residual_norm(x, pre_weight=w1, quantize=torch.float8_e4m3fn)
    y = torch.relu(up(q, s)).square()
    return TAB.residual_norm(down(y), x, pre_weight=w1, post_weight=w2, gate=gate, residual_scale=0.9)


def block_params(cuda, C, F):
    gen = torch.Generator(device=cuda).manual_seed(3)
    n = lambda *s: torch.randn(*s, device=cuda, generator=gen)
    return 1 + 0.1 * n(C), 1 + 0.1 * n(C), n(F, C) / C ** 0.5, n(C, F) / F ** 0.5, 0.5 + 0.1 * n(C)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 7, 200, 600])
def test_block_for_serving_and_training_agree(cuda, tokens):
    """The same block from prepared layers, its first norm handing over blocks, and in its differentiable form: equal but for values
    whose fp32 and bf16 forms round to different 8-bit floats (a step is 2^-3 of a value, its half 2^-4; few values, and a sum of many)."""
    C, F = 384, 1000
    params = block_params(cuda, C, F)
    x = torch.randn(tokens, C, device=cuda).bfloat16()
    served = block_step(x, (*params[:2], tab_nn.BlockLinear.from_float(params[2]), tab_nn.BlockLinear.from_float(params[3]), params[4]), False)
    trained = block_step(x, params, True)
    for a, b in zip(served, trained):
        assert float((a.float() - b.float()).norm() / b.float().norm()) <= 2.0 ** -4


@pytest.mark.gpu
def test_block_in_a_graph(cuda):
    """Forward and backward captured once and replayed on other inputs, beside a second graph and eager calls: the eager results, bit for bit."""
    C, F, T = 256, 520, 160
    params = [p.requires_grad_() for p in block_params(cuda, C, F)]
    inputs = [torch.randn(T, C, device=cuda).bfloat16() for _ in range(3)]

    def step(x):
        x = x.detach().requires_grad_()
        r, h = block_step(x, params, True)
        return [r.detach(), h.detach(), *torch.autograd.grad((r, h), (x, *params), (torch.ones_like(r), torch.ones_like(h)))]

    eager = [step(x) for x in inputs]
    graphs = []
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(inputs[0])
    torch.cuda.synchronize()
    for _ in range(2):
        place, g = inputs[0].clone(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(place)
        graphs.append((place, g, out))
    for i, (x, want) in enumerate(zip(inputs, eager)):
        place, g, out = graphs[i % 2]
        place.copy_(x)
        g.replay()
        other = step(inputs[(i + 1) % 3])
        assert all(torch.equal(a, b) for a, b in zip(out, want)) and all(torch.equal(a, b) for a, b in zip(other, eager[(i + 1) % 3]))


@pytest.mark.gpu
def test_streams_side_by_side(cuda):
    """The same calls on two streams at once: each one's own results."""
    C, F = 512, 700
    params = block_params(cuda, C, F)
    xs = [torch.randn(t, C, device=cuda).bfloat16() for t in (3, 300, 900, 40)]
    want = [block_step(x, params, True) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i in range(20):
        with torch.cuda.stream(streams[i % 2]):
            got.append(block_step(xs[i % 4], params, True))
    torch.cuda.synchronize()
    for i, pair in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(pair, want[i % 4]))
    assert _cabi.lib().tab_device_status() == 0


@pytest.mark.gpu
def test_empty_rows_and_sums(cuda):
    x = torch.randn(3, 0, device=cuda)
    q, s, qt, st = TAB.quantize_blocks(x, columns=True)
    assert q.shape == (3, 0) and s.shape == (3, 0) and qt.shape == (0, 3) and st.shape == (0, 1)
    assert not TAB.matmul_blocks(q, s, q, s).any()
    q, s = TAB.quantize_blocks(torch.randn(0, 128, device=cuda))
    assert q.shape == (0, 128) and s.shape == (0, 1)


@pytest.mark.gpu
def test_single_vectors(cuda):
    """Tensors of one dimension are one row, through every operator and both directions."""
    x, w, g = torch.randn(300, device=cuda), torch.randn(130, 300, device=cuda), torch.randn(130, device=cuda)
    q, s = TAB.quantize_blocks(x)
    q2, s2 = TAB.quantize_blocks(x[None])
    wq = TAB.quantize_blocks2d(w)
    assert q.shape == (300,) and s.shape == (3,) and torch.equal(q.view(torch.uint8), q2[0].view(torch.uint8)) and torch.equal(s.view(torch.uint8), s2[0].view(torch.uint8))
    assert torch.equal(TAB.matmul_blocks(q, s, *wq), TAB.matmul_blocks(q2, s2, *wq)[0])
    results = []
    for v, grad in ((x, g), (x[None], g[None])):
        leaves = [v.clone().requires_grad_(), w.clone().requires_grad_()]
        y = tab_nn.block_linear(*leaves)
        results.append([y.detach().reshape(-1), *(d.reshape(-1) for d in torch.autograd.grad(y, leaves, grad))])
    assert all(torch.equal(a, b) for a, b in zip(*results))
    p = torch.rand(300, device=cuda)
    one, many = TAB.residual_norm(x, x, pre_weight=p, gate=p), TAB.residual_norm(x[None], x[None], pre_weight=p, gate=p)
    assert all(torch.equal(a, b[0]) for a, b in zip(one, many))


@pytest.mark.gpu
def test_weights_changed_between_the_passes(cuda):
    """The backward pass multiplies what the forward pass did, whatever has become of the weights since; the norms' weights say so."""
    x, w, g = torch.randn(40, 256, device=cuda, requires_grad=True), torch.randn(64, 256, device=cuda, requires_grad=True), torch.randn(40, 64, device=cuda)
    want = torch.autograd.grad(tab_nn.block_linear(x, w), (x, w), g)
    y = tab_nn.block_linear(x, w)
    with torch.no_grad():
        w.mul_(3)
    got = torch.autograd.grad(y, (x, w), g)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    p = torch.rand(256, device=cuda, requires_grad=True)
    h = tab_nn.residual_norm(x, pre_weight=p)[1]
    with torch.no_grad():
        p.mul_(3)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        h.sum().backward()


@pytest.mark.gpu
@pytest.mark.parametrize("native", [True, False])
def test_negated_views(cuda, monkeypatch, native):
    """A view whose memory holds the negatives of its values is refused; as a gradient it is resolved."""
    if not native:
        monkeypatch.setattr(TAB.ops, "_native", False)
    x, w, p = torch.randn(5, 256, device=cuda), torch.randn(40, 256, device=cuda), torch.rand(256, device=cuda)
    n = torch._neg_view(x)
    for call in (lambda: TAB.quantize_blocks(n), lambda: TAB.quantize_blocks2d(n), lambda: TAB.residual_norm(n, pre_weight=p), lambda: TAB.residual_norm(x, n),
                 lambda: TAB.residual_norm(x, pre_weight=torch._neg_view(p)), lambda: TAB.residual_norm(x, gate=n), lambda: tab_nn.block_linear(x, torch._neg_view(w))):
        with pytest.raises(RuntimeError, match="negated"):
            call()
    leaves = [x.requires_grad_(), w.requires_grad_(), p.requires_grad_()]
    g, gh = torch.randn(5, 40, device=cuda), torch.randn(5, 256, device=cuda)
    for of, grad, result in ((leaves[:2], g, lambda: tab_nn.block_linear(x, w)), (leaves[::2], gh, lambda: tab_nn.residual_norm(x, pre_weight=p)[1])):
        got, want = (torch.autograd.grad(result(), of, v) for v in (torch._neg_view(grad), -grad))
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize("native", [True, False])
def test_tensors_kept_on_the_host(cuda, monkeypatch, native):
    """What the forward passes keep may be copied to the host and back, where rows of odd lengths lose the bytes between them."""
    if not native:
        monkeypatch.setattr(TAB.ops, "_native", False)
    x, w, p, g = torch.randn(37, 100, device=cuda, requires_grad=True), torch.randn(51, 100, device=cuda, requires_grad=True), torch.rand(100, device=cuda, requires_grad=True), torch.randn(37, 51, device=cuda)
    def grads(outside):
        with outside:
            y = tab_nn.block_linear(tab_nn.residual_norm(x, x, pre_weight=p, gate=x)[1], w)
        return torch.autograd.grad(y, (x, w, p), g)
    assert all(torch.equal(a, b) for a, b in zip(grads(contextlib.nullcontext()), grads(torch.autograd.graph.save_on_cpu())))


@pytest.mark.gpu
@pytest.mark.parametrize("M", [2, 40, 200, 2304])
def test_matmul_blocks_values_behind_the_sum(cuda, M):
    """Sums that end inside a block, and inside sixteen bytes, with NaN and live values right behind them in memory."""
    rng = np.random.default_rng(M)
    N, K, end = (1300 if M > 1000 else 300), 512, 401
    a, b = random_blocks(rng, M, K, "e4m3", False, True), random_blocks(rng, N, K, "e4m3", True, True)
    (qa, sa), (qb, sb) = device_blocks(cuda, *a, "e4m3"), device_blocks(cuda, *b, "e4m3")
    va, vb = ref.values(*a, "e4m3")[:, 128:end], ref.values(*b, "e4m3")[:, 128:end]
    for q in (qa, qb):
        q.view(torch.uint8)[:, end::2] = 0x7F
    y = TAB.matmul_blocks(qa[:, 128:end], sa[:, 1:4], qb[:, 128:end], sb[:, 1:4], out_dtype=torch.float32)
    assert np.array_equal(y.cpu().numpy(), va @ vb.T)


@pytest.mark.gpu
def test_the_same_leaf_twice(cuda):
    """One tensor in several places has the sum of their gradients (fp32, of terms below 2^6: roundings of three sums)."""
    x, p = torch.randn(33, 200, device=cuda, requires_grad=True), torch.rand(200, device=cuda, requires_grad=True)
    gr, gh = torch.randn(33, 200, device=cuda), torch.randn(33, 200, device=cuda)
    one = torch.autograd.grad(tab_nn.residual_norm(x, x, pre_weight=p, post_weight=p, gate=x), (x, p), (gr, gh))
    xs, ps = [x.detach().clone().requires_grad_() for _ in range(3)], [p.detach().clone().requires_grad_() for _ in range(2)]
    each = torch.autograd.grad(tab_nn.residual_norm(xs[0], xs[1], pre_weight=ps[0], post_weight=ps[1], gate=xs[2]), xs + ps, (gr, gh))
    for got, parts in zip(one, (each[:3], each[3:])):
        size = sum(t.abs() for t in parts)
        assert bool(((got - sum(parts)).abs() <= size * 4 * 2.0 ** -24).all())
    w = torch.randn(200, 200, device=cuda, requires_grad=True)
    both, = torch.autograd.grad(tab_nn.block_linear(w, w), w, torch.ones(200, 200, device=cuda))
    ws = [w.detach().clone().requires_grad_() for _ in range(2)]
    parts = torch.autograd.grad(tab_nn.block_linear(*ws), ws, torch.ones(200, 200, device=cuda))
    assert torch.equal(both, parts[0] + parts[1])


@pytest.mark.gpu
@pytest.mark.parametrize("M, N, K", [(3, 130, 2300), (41, 130, 2300), (133, 299, 2300), (2303, 1301, 2300)])
def test_matmul_blocks_scales_shared_by_blocks(cuda, M, N, K):
    """One scale for all blocks of a row, and scales block by block without a gap behind the last row: exact, as in test_matmul_blocks_exact."""
    rng = np.random.default_rng(M)
    a, b = random_blocks(rng, M, K, "e4m3", False, True), random_blocks(rng, N, K, "e4m3", False, True)
    (qa, sa), (qb, sb) = device_blocks(cuda, *a, "e4m3"), device_blocks(cuda, *b, "e4m3")
    f64 = lambda q, s: torch.from_numpy(ref.values(q, s, "e4m3")).to(cuda)
    row = sa.view(torch.uint8)[:, 3].contiguous()[:, None].expand(sa.shape).view(torch.float8_e8m0fnu)
    close = sb.view(torch.uint8).t().contiguous().t().view(torch.float8_e8m0fnu)
    want = f64(a[0], np.repeat(a[1][:, 3:4], a[1].shape[1], 1)) @ f64(*b).t()
    assert torch.equal(TAB.matmul_blocks(qa, row, qb, close, out_dtype=torch.float32).double(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("formats", [("e4m3", "e4m3"), ("e5m2", "e4m3"), ("e4m3", "e5m2"), ("e5m2", "e5m2")])
@pytest.mark.parametrize("M, N, K", [(1, 6000, 2000), (8, 4753, 1100), (3, 16390, 200), (5, 20001, 16)])
def test_matmul_blocks_few_rows_many_columns(cuda, M, N, K, formats):
    """More columns than the SMs take at once: exact, as in test_matmul_blocks_exact."""
    rng = np.random.default_rng(N)
    fa, fb = formats
    a, b = random_blocks(rng, M, K, fa, False, True), random_blocks(rng, N, K, fb, True, True)
    y = TAB.matmul_blocks(*device_blocks(cuda, *a, fa), *device_blocks(cuda, *b, fb), out_dtype=torch.float32)
    assert np.array_equal(y.cpu().numpy(), ref.values(*a, fa) @ ref.values(*b, fb).T)
