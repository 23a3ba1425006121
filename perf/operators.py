"""The 8-bit block operators and the normalised residual stream: what they are given, what they return, what they cost.

Three operators.  ``quantize``: values to 8-bit floats with one power-of-two scale for each block of 128.  ``product``: the matrix
product of two such operands, alone, behind the quantiser of its activations (``linear``), and as a training step of a dense layer
(``train``).  ``norm``: the norm after a block, its gate, the scaled residual and the norm before the next block, forward or forward and
backward.
"""
import math

import torch

own = False

FORMATS = {"e4m3": (torch.float8_e4m3fn, 448.0, 0.875, 9), "e5m2": (torch.float8_e5m2, 57344.0, 0.875, 16)}
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-6


def listed():
    return [
        # activations of a small decoding batch
        dict(name="quantize_16x4096", op="quantize", M=16, K=4096, type="bf16", format="e4m3", form="rows"),
        # activations of a training step, along both axes: for the product and for the weights' gradient
        dict(name="quantize_both_8192x4096", op="quantize", M=8192, K=4096, type="bf16", format="e4m3", form="both"),
        # weights of odd size, from fp32 master copies, in squares, with the transposed copy that a backward pass multiplies
        dict(name="quantize_square_2571x1411", op="quantize", M=2571, K=1411, type="fp32", format="e4m3", form="square"),
        # one token through a dense layer
        dict(name="linear_1x4096x4096", op="linear", M=1, N=4096, K=4096, type="bf16", format="e4m3"),
        # a decoding batch through a wider one, operands in hand
        dict(name="product_40x8192x2048", op="product", M=40, N=8192, K=2048, type="bf16", format="e4m3", squares=True),
        # a prompt
        dict(name="product_4096x8192x4096", op="product", M=4096, N=8192, K=4096, type="bf16", format="e4m3", squares=True),
        # odd sizes, gradients in the wider-ranged type, a scale per row on both sides, fp32 result
        dict(name="product_1003x2571x1413", op="product", M=1003, N=2571, K=1413, type="fp32", format="e5m2", squares=False),
        # a training step of a dense layer: result and both gradients
        dict(name="train_8192x4096x4096", op="train", M=8192, N=4096, K=4096, type="bf16", format="e4m3"),
        # one token between two blocks, handed on as 8-bit blocks
        dict(name="norm_1x4096", op="norm", M=1, K=4096, type="bf16", kind="rms", gate="channel", post=True, quantize=True, backward=False),
        # a prompt
        dict(name="norm_4096x8192", op="norm", M=4096, K=8192, type="bf16", kind="rms", gate="none", post=True, quantize=True, backward=False),
        # a training step
        dict(name="norm_train_8192x4096", op="norm", M=8192, K=4096, type="bf16", kind="rms", gate="channel", post=True, quantize=False, backward=True),
        # odd sizes, centred norms with shifts, a gate per token, fp32
        dict(name="norm_train_777x1001", op="norm", M=777, K=1001, type="fp32", kind="layer", gate="token", post=True, quantize=False, backward=True),
    ]


def _size(rng, low, high):
    n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    return min(high, max(low, n if rng.random() < 0.5 else (n + 63) // 64 * 64))


def draw(rng):
    op = rng.choice(["quantize", "linear", "product", "train", "norm"])
    case = dict(op=op, type=rng.choice(["bf16", "bf16", "fp16", "fp32"]))
    if op == "quantize":
        return dict(case, M=_size(rng, 1, 8192), K=_size(rng, 16, 4096), format=rng.choice(["e4m3", "e5m2"]), form=rng.choice(["rows", "both", "square"]))
    if op == "norm":
        quantize = rng.random() < 0.4
        return dict(case, M=_size(rng, 1, 4096), K=_size(rng, 16, 8192), kind=rng.choice(["rms", "layer"]), gate=rng.choice(["none", "channel", "token"]),
                    post=rng.random() < 0.7, quantize=quantize, backward=not quantize and rng.random() < 0.7)
    case.update(N=_size(rng, 16, 4096), K=_size(rng, 16, 4096), format="e4m3")
    if op == "product":
        return dict(case, M=_size(rng, 1, 4096), format=rng.choice(["e4m3", "e5m2"]), squares=rng.random() < 0.5)
    return dict(case, M=_size(rng, 1, 256 if op == "linear" else 4096))


def _blocks(n):
    return -(-n // 128)


def _amax(x):
    """Largest finite magnitude of each 128 values of the last dimension."""
    x = torch.nn.functional.pad(torch.where(torch.isfinite(x), x.abs(), 0.0), (0, -x.shape[-1] % 128))
    return x.reshape(*x.shape[:-1], -1, 128).amax(-1)


def _exponent(amax, format):
    """Least e with amax <= largest * 2^e, from the parts of amax = m * 2^k."""
    _, _, m0, k0 = FORMATS[format]
    m, k = torch.frexp(amax)
    return torch.where(amax == 0, 0, (k - k0 + (m > m0)).clamp(-127, 127)).to(torch.int32)


def _spread(e, n):
    """One value for each 128 of the last dimension -> one for each of its n elements."""
    return e.repeat_interleave(128, -1)[..., :n]


def _pack(x, e, format):
    q = torch.ldexp(x, -e)
    if format == "e4m3":
        q = torch.where(torch.isinf(q), math.nan, q)
    return q.to(FORMATS[format][0])


def _scale(e):
    return (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def _quantize(x, format):
    x = x.float()
    e = _exponent(_amax(x), format)
    return _pack(x, _spread(e, x.shape[-1]), format), _scale(e)


def _quantize_square(x, format):
    x = x.float()
    e = _exponent(_amax(_amax(x).t()).t().contiguous(), format)
    return _pack(x, _spread(_spread(e, x.shape[1]).t(), x.shape[0]).t(), format), _scale(e)


def _values(q, s):
    """What 8-bit floats and their scales stand for; scales of rows, or of squares (fewer of them than rows)."""
    s = _spread(s.float(), q.shape[1])
    return q.float() * (s if s.shape[0] == q.shape[0] else _spread(s.t(), q.shape[0]).t())


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    normal = lambda *size: torch.randn(*size, device="cuda", generator=gen)
    dt, M, K = TYPES[case["type"]], case["M"], case["K"]
    # channels differ in magnitude, as those of a language model's activations do
    x = normal(M, K) * torch.exp(0.8 * normal(K))
    state = {"case": case}
    if case["op"] == "norm":
        rows = {"none": None, "channel": (K,), "token": (M, 1)}[case["gate"]]
        shift = case["kind"] == "layer"
        state.update(y=x.to(dt), residual=(3 * normal(M, K)).to(dt), alpha=1.25, gate=None if rows is None else 0.5 + 0.2 * normal(*rows),
                     pre=(1 + 0.1 * normal(K), 0.1 * normal(K) if shift else None),
                     post=(1 + 0.1 * normal(K), 0.1 * normal(K) if shift else None) if case["post"] else (None, None))
        if case["backward"]:
            state.update(gr=normal(M, K).to(dt), gh=normal(M, K).to(dt))
        return state
    if case["op"] == "quantize":
        return dict(state, x=x.to(dt))
    w = normal(case["N"], K) / math.sqrt(K)
    if case["op"] == "train":
        return dict(state, x=x.to(dt), w=w, dy=(0.01 * normal(M, case["N"])).to(dt))
    if case["op"] == "linear":
        return dict(state, x=x.to(dt), w=_rows_on_16(*_quantize_square(w, case["format"])))
    a = _rows_on_16(*_quantize(x.to(dt), case["format"]))
    return dict(state, a=a, w=_rows_on_16(*(_quantize_square if case["squares"] else _quantize)(w, "e4m3")))


def _rows_on_16(q, s):
    """The layout that 8-bit operands are kept in: every row starts on 16 bytes."""
    held = torch.zeros(q.shape[0], -(-q.shape[1] // 16) * 16, dtype=torch.uint8, device=q.device)
    held[:, :q.shape[1]] = q.view(torch.uint8)
    return held.view(q.dtype)[:, :q.shape[1]], s.contiguous()


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(state):
    import tab_b200 as TAB
    from tab_b200 import nn as tab_nn
    case = state["case"]
    op, dt = case["op"], TYPES[case["type"]]
    if op == "quantize":
        f8 = FORMATS[case["format"]][0]
        if case["form"] == "square":
            return TAB.quantize_blocks2d(state["x"], f8, transposed=True)
        return TAB.quantize_blocks(state["x"], f8, columns=case["form"] == "both")
    if op == "linear":
        q, s = TAB.quantize_blocks(state["x"])
        return TAB.matmul_blocks(q, s, *state["w"], out_dtype=dt)
    if op == "product":
        return TAB.matmul_blocks(*state["a"], *state["w"], out_dtype=dt)
    if op == "train":
        x, w = state["x"].detach().requires_grad_(), state["w"].detach().requires_grad_()
        y = tab_nn.block_linear(x, w)
        return (y.detach(), *torch.autograd.grad(y, (x, w), state["dy"]))
    args = dict(residual=state["residual"], residual_scale=state["alpha"], gate=state["gate"], pre_weight=state["pre"][0], pre_bias=state["pre"][1],
                post_weight=state["post"][0], post_bias=state["post"][1], kind=case["kind"], eps=EPS)
    if not case["backward"]:
        return TAB.residual_norm(state["y"], **args, quantize=torch.float8_e4m3fn if case["quantize"] else None)
    leaves = {k: args[k].detach().requires_grad_() for k in ("residual", "gate", "pre_weight", "pre_bias", "post_weight", "post_bias") if args[k] is not None}
    y = state["y"].detach().requires_grad_()
    r, h = tab_nn.residual_norm(y, **{**args, **leaves})
    return (r.detach(), h.detach(), *torch.autograd.grad((r, h), (y, *leaves.values()), (state["gr"], state["gh"])))


def _run_plain(state):
    case = state["case"]
    op, dt = case["op"], TYPES[case["type"]]
    if op == "quantize":
        x = state["x"]
        if case["form"] == "rows":
            return _quantize(x, case["format"])
        if case["form"] == "both":
            return (*_quantize(x, case["format"]), *_quantize(x.t(), case["format"]))
        q, s = _quantize_square(x, case["format"])
        return q, s, q.t(), s.t()
    if op in ("linear", "product"):
        a = _quantize(state["x"], case["format"]) if op == "linear" else state["a"]
        return (_values(*a) @ _values(*state["w"]).t()).to(dt)
    if op == "train":
        x, w, dy = state["x"], _values(*_quantize_square(state["w"], "e4m3")), state["dy"]
        y = _values(*_quantize(x, "e4m3")) @ w.t()
        dx = _values(*_quantize(dy, "e4m3")) @ w
        dw = _values(*_quantize(dy.t(), "e4m3")) @ _values(*_quantize(x.t(), "e4m3")).t()
        return y.to(dt), dx.to(dt), dw
    return _norm_plain(state, case, dt)


def _normalise(v, kind, weight, bias):
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    v = v * (v.square().mean(-1, keepdim=True) + EPS).rsqrt() * weight
    return v if bias is None else v + bias


def _norm_plain(state, case, dt):
    """The gradients are those of the elementary operations; storing r in the type of y counts as the identity."""
    back = case["backward"]
    names = {"y": state["y"].float(), "residual": state["residual"].float(), "gate": state["gate"], "pre_weight": state["pre"][0], "pre_bias": state["pre"][1],
             "post_weight": state["post"][0], "post_bias": state["post"][1]}
    v = {k: t.detach().requires_grad_(back) for k, t in names.items() if t is not None}
    with torch.set_grad_enabled(back):
        u = _normalise(v["y"], case["kind"], v["post_weight"], v.get("post_bias")) if case["post"] else v["y"]
        r = state["alpha"] * v["residual"] + (u if "gate" not in v else v["gate"] * u)
        r = r + (r.detach().to(dt).float() - r.detach())
        h = _normalise(r, case["kind"], v["pre_weight"], v.get("pre_bias"))
    if case["quantize"]:
        return (r.to(dt), *_quantize(h, "e4m3"))
    if not back:
        return r.to(dt), h.to(dt)
    grads = torch.autograd.grad((r, h), tuple(v.values()), (state["gr"].float(), state["gh"].float()))
    return (r.detach().to(dt), h.detach().to(dt), *(g.to(dt) if k in ("y", "residual") else g for k, g in zip(v, grads)))


def work(case):
    """Every input read once, every output written once; an operation is a multiply or an add.  8-bit operands count one byte for each
    value and one for each scale."""
    M, K, b = case["M"], case["K"], TYPES[case["type"]].itemsize
    if case["op"] == "quantize":
        scales = {"rows": M * _blocks(K), "both": M * _blocks(K) + K * _blocks(M), "square": 2 * _blocks(M) * _blocks(K)}[case["form"]]
        return {"bytes": M * K * (b + (1 if case["form"] == "rows" else 2)) + scales, "flops": 2 * M * K}
    if case["op"] == "norm":
        params = 4 * K * (2 if case["post"] else 1) * (2 if case["kind"] == "layer" else 1) + 4 * {"none": 0, "channel": K, "token": M}[case["gate"]]
        out = M * K + M * _blocks(K) if case["quantize"] else M * K * b
        total = 3 * M * K * b + out + params
        if case["backward"]:
            total += 4 * M * K * b + params
        return {"bytes": total, "flops": M * K * (40 if case["backward"] else 14)}
    N = case["N"]
    if case["op"] == "train":
        return {"bytes": 2 * M * K * b + 2 * M * N * b + 8 * N * K, "flops": 6 * M * N * K}
    rows = M * K * b if case["op"] == "linear" else M * K + M * _blocks(K)
    squares = case["op"] == "linear" or case["squares"]
    return {"bytes": rows + N * K + (_blocks(N) if squares else N) * _blocks(K) + M * N * b, "flops": 2 * M * N * K}


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------------------

def _exact_blocks(x, format, square=False):
    """Values and scales, [M,K] and [M or blocks of M, blocks of K]."""
    largest = FORMATS[format][1]
    digits, lowest = (3, -6) if format == "e4m3" else (2, -14)
    M, K = x.shape
    full = torch.zeros(_blocks(M) * 128 if square else M, _blocks(K) * 128, dtype=torch.float64, device=x.device)
    full[:M, :K] = x
    full = full.reshape(full.shape[0] // 128 if square else M, 128 if square else 1, _blocks(K), 128)
    a = full.abs().amax((1, 3), keepdim=True)
    one = torch.ones_like(a)
    e = torch.ceil(torch.log2(torch.where(a > 0, a / largest, one)))
    e = torch.where(a > largest * torch.exp2(e), e + 1, e)
    e = torch.where((a > 0) & (a <= largest * torch.exp2(e - 1)), e - 1, e).clamp(-127, 127)
    s = torch.exp2(e)
    v = full / s
    step = torch.exp2(torch.floor(torch.log2(torch.where(v == 0, 1.0, v.abs()))).clamp(min=lowest) - digits)
    v = torch.round(v / step) * step
    return v.reshape(-1, _blocks(K) * 128)[:M, :K], s.reshape(-1, _blocks(K)), (v * s).reshape(-1, _blocks(K) * 128)[:M, :K]


def _exact_values(q, s):
    M, K = q.shape
    s = s.double().unsqueeze(-1).expand(-1, -1, 128).reshape(s.shape[0], -1)[:, :K]
    if s.shape[0] != M:
        s = s.unsqueeze(1).expand(-1, 128, -1).reshape(-1, K)[:M]
    return q.double() * s


def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op == "quantize":
        x = state["x"].double()
        if case["form"] == "square":
            q, s, _ = _exact_blocks(x, case["format"], True)
            return q, s, q.t(), s.t()
        q, s, _ = _exact_blocks(x, case["format"])
        return (q, s, *_exact_blocks(x.t(), case["format"])[:2]) if case["form"] == "both" else (q, s)
    if op == "linear":
        return torch.einsum("mk,nk->mn", _exact_blocks(state["x"].double(), case["format"])[2], _exact_values(*state["w"]))
    if op == "product":
        return torch.einsum("mk,nk->mn", _exact_values(*state["a"]), _exact_values(*state["w"]))
    if op == "train":
        x, dy = state["x"].double(), state["dy"].double()
        w = _exact_blocks(state["w"].double(), "e4m3", True)[2]
        along = lambda t: _exact_blocks(t.t(), "e4m3")[2].t()
        return (torch.einsum("mk,nk->mn", _exact_blocks(x, "e4m3")[2], w), torch.einsum("mn,nk->mk", _exact_blocks(dy, "e4m3")[2], w),
                torch.einsum("mn,mk->nk", along(dy), along(x)))
    return _exact_norm(state, case)


def _exact_norm(state, case):
    layer = case["kind"] == "layer"
    wide = lambda t: None if t is None else t.double()
    y, x, gate, alpha = state["y"].double(), state["residual"].double(), wide(state["gate"]), state["alpha"]
    (w1, b1), (w2, b2) = [tuple(map(wide, state[k])) for k in ("post", "pre")]

    def unit(v):
        centred = v - v.mean(1, keepdim=True) if layer else v
        inverse = 1 / torch.sqrt((centred * centred).mean(1, keepdim=True) + EPS)
        return centred * inverse, inverse

    def through(t, v, inverse):
        """Gradient at the input of `unit` for t at its output v."""
        t = t - v * (t * v).mean(1, keepdim=True) - (t.mean(1, keepdim=True) if layer else 0)
        return t * inverse

    g = 1.0 if gate is None else gate
    y1, i1 = unit(y)
    u = y if w1 is None else y1 * w1 + (0 if b1 is None else b1)
    r = alpha * x + g * u
    kept = r.to(TYPES[case["type"]]).double()
    r2, i2 = unit(kept)
    h = r2 * w2 + (0 if b2 is None else b2)
    if case["quantize"]:
        return (r, *_exact_blocks(h, "e4m3")[:2])
    if not case["backward"]:
        return r, h
    gr, gh = state["gr"].double(), state["gh"].double()
    dr = gr + through(gh * w2, r2, i2)
    du = dr * g
    grads = [du if w1 is None else through(du * w1, y1, i1), alpha * dr]
    if gate is not None:
        grads.append((dr * u).sum(0) if case["gate"] == "channel" else (dr * u).sum(1, keepdim=True))
    grads += [(gh * r2).sum(0)] + ([] if b2 is None else [gh.sum(0)])
    if w1 is not None:
        grads += [(du * y1).sum(0)] + ([] if b1 is None else [du.sum(0)])
    return (r, h, *grads)
