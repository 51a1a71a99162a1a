"""The linear cross entropy (output projection and masked softmax loss in one) against the formula in
64 bits, at the sizes, masks and types where it can go wrong, and its refusals.

Tolerances are worst-case bounds worked out in 64 bits for each output element, from the roundings
that the mode is documented to make (half a step: 2^-11 for f16, 2^-24 for f32) and from sums of n
terms in f32, whose error is at most n 2^-24 of the sum of magnitudes (the tensor core cuts the
low bits of every group of 16: n/16 steps of 2^-23, which is less)."""

import ctypes as C

import numpy as np
import pytest
import torch

SKIP = 0xFFFFFFFF
F16, F32 = torch.float16, torch.float32
MODES = ("F32", "F16", "F16X2")


# ------------------------------------------------------------------------------- refusals, without a GPU
@pytest.fixture(scope="module")
def lib():
    from ferrotensor_b200 import _build, _lib
    _build.build()
    return _lib.load()


def _raw(lib, p, ctx=1, hidden=0x10000000, weight=0x20000000, targets=0x30000000, weights=0x31000000, loss=0x32000000,
         gh=None, gw=None, ws=0x40000000, ws_bytes=1 << 40):
    """A call whose pointers nothing may follow: every refusal comes before any CUDA call.  `ctx` is
    zeroed memory in place of a context."""
    fake = C.create_string_buffer(1 << 16)
    h = C.cast(fake, C.c_void_p) if ctx else None
    return lib.ft_linear_cross_entropy(h, hidden, weight, targets, weights, loss, gh, gw, ws, ws_bytes, C.byref(p))


def _params(**kw):
    from ferrotensor_b200._lib import FtLinearCeParams
    d = dict(rows=8, hidden=64, vocab=1000, weight_vocab_major=0, hidden_type=0, weight_type=0, grad_hidden_type=0,
             grad_weight_type=0, vocab_piece=0, grad_scale=1.0)
    d.update(kw)
    return FtLinearCeParams(**d)


@pytest.mark.parametrize("params,call,message", [
    ({}, dict(ctx=0), "NULL"),
    ({}, dict(hidden=None), "NULL"),
    ({}, dict(weight=None), "NULL"),
    ({}, dict(targets=None), "NULL"),
    ({}, dict(loss=None), "NULL"),
    ({}, dict(weights=None, gh=0x50000000), "needs the rows' weights"),
    ({}, dict(ws=None), "workspace"),
    ({}, dict(ws_bytes=64), "workspace"),
    (dict(hidden=0), {}, "outside"),
    (dict(vocab=0), {}, "outside"),
    (dict(vocab=(1 << 24) + 1), {}, "outside"),
    (dict(hidden=(1 << 16) + 1), {}, "outside"),
    (dict(rows=(1 << 24) + 1), {}, "outside"),
    (dict(hidden_type=2), {}, "type"),
    (dict(grad_weight_type=7), {}, "type"),
    (dict(grad_scale=float("nan")), {}, "finite"),
    (dict(grad_scale=float("inf")), {}, "finite"),
    ({}, dict(hidden=0x10000002), "aligned"),
    (dict(hidden_type=1), dict(hidden=0x10000001), "aligned"),
    ({}, dict(targets=0x30000001), "aligned"),
    ({}, dict(gh=0x10000000), "overlaps hidden"),
    ({}, dict(gw=0x20000000 + 64 * 1000 * 4 - 4), "overlaps weight"),
    ({}, dict(gh=0x50000000, gw=0x50000000), "overlaps"),
    ({}, dict(loss=0x31000000), "overlaps weights"),
    ({}, dict(ws=0x20000000), "overlaps weight"),
])
def test_refusals(lib, params, call, message):
    assert _raw(lib, _params(**params), **call) == 1
    assert message in lib.ft_last_error().decode()


def test_workspace_sizes(lib):
    fake = C.create_string_buffer(1 << 16)
    h = C.cast(fake, C.c_void_p)
    n = C.c_size_t()
    for mode in range(3):
        assert lib.ft_ctx_set_gemm_mode(h, mode) == 0
        for rows, hidden, vocab, piece in ((0, 1, 1, 0), (1, 1, 1, 0), (4096, 64, 1000, 0), (4096, 65, 100003, 1), (1 << 24, 1 << 16, 1 << 24, 7)):
            got = []
            for gh, gw in ((0, 0), (1, 0), (1, 1)):
                p = _params(rows=rows, hidden=hidden, vocab=vocab, vocab_piece=piece)
                assert lib.ft_linear_cross_entropy_workspace(h, None, C.byref(p), gh, gw, C.byref(n)) == 0
                got.append(n.value)
            assert min(got) > 0 and max(got) < 1 << 60
    assert lib.ft_linear_cross_entropy_workspace(h, None, C.byref(_params(hidden=0)), 0, 0, C.byref(n)) == 1
    assert lib.ft_linear_cross_entropy_workspace(h, None, C.byref(_params()), 0, 0, None) == 1


def test_struct_layout_matches_header(tmp_path):
    import subprocess
    from pathlib import Path
    from ferrotensor_b200._lib import FtLinearCeParams as P
    root = Path(__file__).resolve().parent.parent
    src = tmp_path / "s.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "ft_cuda.h"\nint main(void) { printf("%zu %zu %zu\\n", '
                   'sizeof(FtLinearCeParams), offsetof(FtLinearCeParams, vocab_piece), offsetof(FtLinearCeParams, grad_scale)); return 0; }\n')
    subprocess.run(["gcc", "-I", str(root / "include"), str(src), "-o", str(tmp_path / "s")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "s")], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [C.sizeof(P), P.vocab_piece.offset, P.grad_scale.offset]


# ------------------------------------------------------------------------------- on the GPU
gpu = pytest.mark.gpu


@pytest.fixture(scope="module")
def eng(cuda_ctx):
    from ferrotensor_b200.engine import ComputeEngine
    return ComputeEngine(cuda_ctx)


def _ut(x):
    from ferrotensor_b200.engine import DType, UnifiedTensor
    kind = {F32: DType.F32, F16: DType.FP16, torch.int32: DType.U32}[x.dtype]
    return UnifiedTensor(x.reshape(-1).view(torch.uint8), list(x.shape), kind)


def _targets(y):
    """int64 targets with SKIP -> the int32 bit patterns the device reads"""
    return torch.where(y >= 1 << 31, y - (1 << 32), y).to(torch.int32).cuda()


def _make(t, h, v, types, vocab_major, mask, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    hk, wk = types
    w = (torch.randn((v, h) if vocab_major else (h, v), generator=g, device="cuda") * 0.1).to(wk)
    x = (torch.randn((t, h), generator=g, device="cuda") * scale).to(hk)
    y = torch.randint(0, v, (t,), generator=g, device="cuda")
    if mask == "half":
        y[torch.rand(t, generator=g, device="cuda") < 0.5] = SKIP
    elif mask == "all":
        y[:] = SKIP
    elif mask == "last":
        y[:-1] = SKIP
    elif mask == "prompts":
        y[: (2 * t) // 3] = SKIP
    elif mask == "beyond":
        y[::3] = v
        y[1::3] = SKIP
        y[2::9] = 0xFFFFFFFE
    a = (torch.rand(t, generator=g, device="cuda") + 0.5) / t
    a[::5] *= -1
    a[3::7] = 0
    return x, w, y, a


def _truth(x, w, y, a, s, vocab_major):
    """loss, dh, dW of the formula in 64 bits, W as [v, h]"""
    W = (w if vocab_major else w.t()).double()
    live = y != SKIP
    X = torch.where(live[:, None], x.double(), 0.0)
    z = X @ W.t()
    lse = torch.logsumexp(z, dim=1)
    inside = live & (y < W.shape[0])
    one = torch.zeros_like(z)
    one[inside, y[inside]] = 1.0
    loss = torch.where(inside, lse - (z * one).sum(1), 0.0)
    c = torch.where(live, a.double() * s, 0.0)[:, None]
    p = torch.exp(z - lse[:, None])
    g = (p - one) * c
    return dict(X=X, W=W, z=z, lse=lse, live=live, p=p, c=c, g=g, loss=loss, dh=g @ W, dW=g.t() @ X)


def _bounds(q, mode, types, gtypes):
    """worst-case error of loss, dh, dW (see the top of the file)"""
    X, W, p, c, g = q["X"].abs(), q["W"].abs(), q["p"], q["c"].abs(), q["g"].abs()
    h, v, t = X.shape[1], W.shape[0], X.shape[0]
    u, u16 = 2.0 ** -24, 2.0 ** -11
    # an f32 operand: rounded to f16 in that mode, to two halves (22 bits) in the split one; values far
    # below the tensor's largest fall under f16's smallest step, 2^-24 of a range that ends at 2^14
    # (2^-39 of the largest value, 2^-50 with the second half)
    def op(kind, m):
        if kind is F16 or mode == "F32":
            return 0.0, 0.0
        return (u16, float(m.max()) * 2.0 ** -37) if mode == "F16" else (2.0 ** -21, float(m.max()) * 2.0 ** -48)
    rx, ax = op(types[0], X)
    rw, aw = op(types[1], W)
    dX, dW_ = rx * X + ax, rw * W + aw
    mag = X @ W.t()
    dz = dX @ W.t() + X @ dW_.t() + dX @ dW_.t() + (h + 8) * u * mag
    worst = dz.max(dim=1, keepdim=True).values
    # exp, sum over the vocabulary, log: a few units in the last place each; the exponent's argument is
    # rounded relative to its size
    zspan = (q["z"] - q["lse"][:, None]).abs()
    soft = 2.0 ** -20 + 2 * u * (q["z"].abs().max(dim=1, keepdim=True).values + q["lse"].abs()[:, None])
    loss = (worst + dz.max(dim=1, keepdim=True).values)[:, 0] * 1.01 + soft[:, 0] * 2 + 2 * u * q["loss"].abs()
    dg = c * (p * torch.expm1(dz + worst + soft + 2 * u * zspan) + 4 * u * (p + 1.0))
    rg = {"F32": 0.0, "F16": u16, "F16X2": 2.0 ** -21}[mode]
    floor = float(c.max()) * (2.0 ** -37 if mode == "F16" else 2.0 ** -48)   # f16's smallest step under the carried scale
    dg = dg + rg * (g + dg) + (floor if mode != "F32" else 0.0)
    dg = torch.where(q["live"][:, None], dg, 0.0)
    G = g + dg
    dh_tol = dg @ (W + dW_) + g @ dW_ + (v + 64) * u * (G @ (W + dW_))
    dW_tol = dg.t() @ (X + dX) + g.t() @ dX + (t + 64) * u * (G.t() @ (X + dX))
    for kind, tol, val in ((gtypes[0], dh_tol, q["dh"]), (gtypes[1], dW_tol, q["dW"])):
        if kind is F16:
            tol += u16 * (val.abs() + tol) + 2.0 ** -25
        else:
            tol += 2 * u * (val.abs() + tol) + 1e-40
    return torch.where(q["live"], loss, 0.0), dh_tol, dW_tol


def _call(ctx, eng, mode, x, w, y, a, s, vocab_major, gtypes=(F32, F32), want="both", piece=0, guard=64):
    """The engine's call, with every output between guard values that must survive it."""
    from ferrotensor_b200.engine import GemmMode
    t, h = x.shape
    ctx.set_gemm_mode(GemmMode[mode])

    def room(shape, kind):
        n = int(np.prod(shape))
        flat = torch.full((n + 2 * guard,), float("nan"), dtype=kind, device="cuda")
        flat[:guard] = 7.0
        flat[guard + n:] = 7.0
        return flat, flat[guard:guard + n].view(shape)

    fl, loss = room((t,), F32)
    fh, gh = room((t, h), gtypes[0])
    fw, gw = room(tuple(w.shape), gtypes[1])
    try:
        f = eng.linear_cross_entropy_bt if vocab_major else eng.linear_cross_entropy
        ws_args = dict(grad_hidden=_ut(gh) if want != "none" else None, grad_weight=_ut(gw) if want == "both" else None)
        n = eng.linear_cross_entropy_workspace(ctx, _ut(x), _ut(w), vocab_piece=piece, vocab_major=vocab_major, **ws_args)
        # the workspace is dirty and odd in place, its neighbours are watched
        ws = torch.full((n + 128 + 2 * guard,), 0xFF, dtype=torch.uint8, device="cuda")
        from ferrotensor_b200.engine import DType, UnifiedTensor
        f(ctx, _ut(x), _ut(w), _ut(_targets(y)), _ut(a), _ut(loss), grad_scale=s, vocab_piece=piece,
          workspace=UnifiedTensor(ws[guard + 3:guard + 3 + n], [n // 4], DType.U32), **ws_args)
        ctx.synchronize()
        for flat, m in ((fl, t), (fh, t * h), (fw, w.numel())):
            assert (flat[:guard] == 7.0).all() and (flat[guard + m:] == 7.0).all(), "written outside an output"
        assert (ws[:guard + 3] == 0xFF).all() and (ws[guard + 3 + n:] == 0xFF).all(), "written outside the workspace"
    finally:
        ctx.set_gemm_mode(GemmMode.F32)
    return loss, (gh if want != "none" else None), (gw if want == "both" else None)


def _check(got, q, tols, vocab_major, what=""):
    for name, have, want, tol in (("loss", got[0], q["loss"], tols[0]), ("dh", got[1], q["dh"], tols[1]),
                                  ("dW", got[2], q["dW"], tols[2])):
        if have is None:
            continue
        if name == "dW" and not vocab_major:
            have = have.t()
        err = (have.double() - want).abs()
        bad = ~(err <= tol)
        assert not bad.any(), f"{what} {name}: {int(bad.sum())} of {bad.numel()} off, worst {float((err / (tol + 1e-300)).nan_to_num(1e9).max()):.3g} of the bound"


SIZES = [(1, 1, 1, 0), (1, 64, 500, 0), (3, 5, 7, 4), (5, 8, 257, 0), (77, 96, 1000, 256), (129, 72, 640, 0),
         (257, 200, 513, 512), (300, 575, 1003, 300), (40, 64, 4099, 1024), (1031, 24, 320, 0)]


@gpu
@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("types,gtypes", [((F16, F16), (F16, F16)), ((F32, F16), (F32, F32)), ((F32, F32), (F32, F32)),
                                          ((F16, F32), (F32, F16))])
@pytest.mark.parametrize("vocab_major", [False, True])
def test_values_and_gradients(cuda_ctx, eng, mode, types, gtypes, vocab_major):
    for i, (t, h, v, piece) in enumerate(SIZES):
        mask = ("none", "half", "prompts")[i % 3]
        s = 512.0 if F16 in gtypes else 1.0
        x, w, y, a = _make(t, h, v, types, vocab_major, mask, 100 + i)
        q = _truth(x, w, y, a, s, vocab_major)
        got = _call(cuda_ctx, eng, mode, x, w, y, a, s, vocab_major, gtypes, "both", piece)
        _check(got, q, _bounds(q, mode, types, gtypes), vocab_major, f"{(t, h, v, piece)}")


@gpu
@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("mask", ["all", "last", "beyond"])
def test_masks(cuda_ctx, eng, mode, mask):
    for t in (1, 6, 300):
        x, w, y, a = _make(t, 64, 777, (F16, F16), True, mask, 5)
        x[y == SKIP] = float("nan")          # what a skipped row holds reaches nothing
        a[y == SKIP] = float("inf")
        q = _truth(x, w, y, a, 2.0, True)
        for want in ("both", "hidden", "none"):
            got = _call(cuda_ctx, eng, mode, x, w, y, a, 2.0, True, (F32, F32), want)
            _check(got, q, _bounds(q, mode, (F16, F16), (F32, F32)), True, f"{t} {want}")
            dead = y == SKIP
            assert (got[0][dead] == 0).all() and (got[1] is None or (got[1][dead] == 0).all())
            if mask == "all" and got[2] is not None:
                assert (got[2] == 0).all()


@gpu
@pytest.mark.parametrize("mode", MODES)
def test_no_rows(cuda_ctx, eng, mode):
    x, w, y, a = _make(4, 32, 100, (F16, F16), True, "none", 5)
    loss, gh, gw = _call(cuda_ctx, eng, mode, x[:0], w, y[:0], a[:0], 1.0, True)
    assert loss.numel() == 0 and (gw == 0).all()


@gpu
@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("scale", [1e-6, 300.0])
def test_small_and_large_operands(cuda_ctx, eng, mode, scale):
    """f32 rows far from 1: tiny ones keep their bits, large ones make a one-hot softmax."""
    for types in ((F32, F32), (F32, F16)):
        x, w, y, a = _make(70, 40, 300, types, False, "half", 9, scale)
        q = _truth(x, w, y, a, 1.0, False)
        got = _call(cuda_ctx, eng, mode, x, w, y, a, 1.0, False)
        _check(got, q, _bounds(q, mode, types, (F32, F32)), False)


@gpu
@pytest.mark.parametrize("mode", MODES)
def test_infinities_and_nan_stay_in_their_rows(cuda_ctx, eng, mode):
    x, w, y, a = _make(20, 32, 200, (F16, F16), True, "none", 11)
    clean = _call(cuda_ctx, eng, mode, x, w, y, a, 1.0, True, want="hidden")
    x2 = x.clone()
    x2[4, 3] = float("nan")
    x2[9, 0] = float("inf")
    got = _call(cuda_ctx, eng, mode, x2, w, y, a, 1.0, True, want="hidden")
    rest = torch.ones(20, dtype=torch.bool, device="cuda")
    rest[[4, 9]] = False
    assert torch.equal(got[0][rest], clean[0][rest]) and torch.equal(got[1][rest], clean[1][rest])
    assert got[0][4].isnan() and got[1][4].isnan().any() and not got[0][9].isfinite()


@gpu
@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("vocab_major", [False, True])
def test_one_row_is_enough_and_bits_repeat(cuda_ctx, eng, mode, vocab_major):
    x, w, y, a = _make(700, 136, 1500, (F16, F16), vocab_major, "half", 13)
    first = _call(cuda_ctx, eng, mode, x, w, y, a, 8.0, vocab_major, (F16, F16), "both", 512)
    for _ in range(3):
        again = _call(cuda_ctx, eng, mode, x, w, y, a, 8.0, vocab_major, (F16, F16), "both", 512)
        assert all(torch.equal(p, r) for p, r in zip(first, again))


@gpu
@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("kind", [F16, F32])
def test_operands_that_begin_anywhere(cuda_ctx, eng, mode, kind):
    """Every tensor one element behind a 16-byte boundary."""
    x, w, y, a = _make(90, 64, 513, (kind, kind), True, "half", 17)

    def moved(v):
        flat = torch.zeros(v.numel() + 9, dtype=v.dtype, device="cuda")
        flat[1:1 + v.numel()] = v.reshape(-1)
        return flat[1:1 + v.numel()].view(v.shape)

    q = _truth(x, w, y, a, 4.0, True)
    got = _call(cuda_ctx, eng, mode, moved(x), moved(w), y, moved(a), 4.0, True, (kind, kind), guard=65)
    _check(got, q, _bounds(q, mode, (kind, kind), (kind, kind)), True)


@gpu
@pytest.mark.parametrize("mode", ["F32", "F16X2"])
def test_gradients_against_differences(cuda_ctx, eng, mode):
    """Central differences of the loss the call itself returns, (L(x + e d) - L(x - e d)) / 2e, against
    <dL/dx, d>.  L sums 24 f32 losses near 5, each within 2^-18, so the quotient is within
    24 x 2^-18 / e; the third derivative of a log-sum-exp along a change u of its logits is at most
    (2 max|u|)^3, which gives the e^2 / 6 term."""
    x, w, y, a = _make(24, 48, 90, (F32, F32), False, "none", 19)
    a = torch.ones_like(a)
    _, gh, gw = _call(cuda_ctx, eng, mode, x, w, y, a, 1.0, False)
    g = torch.Generator(device="cuda").manual_seed(1)
    e = 0.02
    for which in ("hidden", "weight"):
        d = torch.randn(x.shape if which == "hidden" else w.shape, generator=g, device="cuda")
        d = d / d.norm()
        up, down = ((x + e * d, x - e * d) if which == "hidden" else (w + e * d, w - e * d))
        vals = []
        for v in (up, down):
            xx, ww = (v, w) if which == "hidden" else (x, v)
            vals.append(float(_call(cuda_ctx, eng, mode, xx, ww, y, a, 1.0, False, want="none")[0].double().sum()))
        slope = float(((gh if which == "hidden" else gw).double() * d.double()).sum())
        u = (d @ w if which == "hidden" else x @ d).double().abs().amax(dim=1)
        third = float(((2 * u) ** 3).sum()) * e * e / 6
        noise = 24 * 2.0 ** -18 / e
        assert abs((vals[0] - vals[1]) / (2 * e) - slope) <= noise + third, which


@gpu
def test_agrees_with_the_separate_operators(cuda_ctx, eng):
    """matmul, masked_cross_entropy_weighted and the two gradient products on the same data, exact mode."""
    from ferrotensor_b200.engine import UnifiedTensor
    x, w, y, a = _make(50, 96, 400, (F32, F32), False, "half", 23)
    loss, gh, gw = _call(cuda_ctx, eng, "F32", x, w, y, a, 1.0, False)
    logits, grad = (UnifiedTensor.empty(cuda_ctx, [50, 400]) for _ in range(2))
    row, dh, dw = UnifiedTensor.empty(cuda_ctx, [50]), UnifiedTensor.empty(cuda_ctx, [50, 96]), UnifiedTensor.empty(cuda_ctx, [96, 400])
    eng.matmul(cuda_ctx, _ut(x), _ut(w), logits)
    eng.masked_cross_entropy_weighted(cuda_ctx, logits, _ut(_targets(y)), _ut(a), grad, row)
    eng.matmul_bt(cuda_ctx, grad, _ut(w), dh)
    eng.matmul_at(cuda_ctx, _ut(x), grad, dw)
    for mine, theirs in ((loss, row), (gh, dh), (gw, dw)):
        ref = torch.from_numpy(theirs.to_vec(cuda_ctx)).view(mine.shape).cuda()
        assert torch.allclose(mine, ref, rtol=1e-4, atol=2e-6)


@gpu
@pytest.mark.parametrize("mode", MODES)
def test_captured_and_replayed_on_another_stream(eng, mode):
    """A graph of the call follows its inputs; a second graph with its own workspace runs beside it."""
    from ferrotensor_b200.engine import ComputeEngine, CudaContext, DType, GemmMode, UnifiedTensor
    data = [_make(130, 64, 900, (F16, F16), True, "half", 31 + k) for k in range(3)]
    built = []
    for k in range(2):
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            ctx = CudaContext(0)
        ctx.set_gemm_mode(GemmMode[mode])
        e = ComputeEngine(ctx)
        x, w, y, a = (v.clone() for v in data[k])
        y = _targets(y)
        loss, gh, gw = torch.empty(130, device="cuda"), torch.empty_like(x), torch.empty_like(w)
        n = e.linear_cross_entropy_workspace(ctx, _ut(x), _ut(w), _ut(gh), _ut(gw), vocab_major=True)
        ws = torch.empty(n, dtype=torch.uint8, device="cuda")

        def call():
            e.linear_cross_entropy_bt(ctx, _ut(x), _ut(w), _ut(y), _ut(a), _ut(loss), _ut(gh), _ut(gw), 16.0,
                                      workspace=UnifiedTensor(ws, [n // 4], DType.U32))
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            call()
            side.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                call()
        built.append((graph, side, ctx, x, w, y, a, loss, gh, gw, ws))
    torch.cuda.synchronize()
    for k, (graph, side, ctx, x, w, y, a, loss, gh, gw, ws) in enumerate(built):
        nx, nw, ny, na = data[k + 1]
        x.copy_(nx); w.copy_(nw); y.copy_(_targets(ny)); a.copy_(na)
    torch.cuda.synchronize()
    for _ in range(3):
        for b in built:
            with torch.cuda.stream(b[1]):
                b[0].replay()
    torch.cuda.synchronize()
    for k, (graph, side, ctx, x, w, y, a, loss, gh, gw, ws) in enumerate(built):
        nx, nw, ny, na = data[k + 1]
        q = _truth(nx, nw, ny, na, 16.0, True)
        _check((loss, gh, gw), q, _bounds(q, mode, (F16, F16), (F16, F16)), True, f"graph {k}")


@gpu
def test_refusals_of_the_engine(cuda_ctx, eng):
    from ferrotensor_b200._lib import FtError
    from ferrotensor_b200.engine import DType, UnifiedTensor
    mk = lambda shape, kind=DType.F32: UnifiedTensor.empty_with_dtype(cuda_ctx, shape, kind)  # noqa: E731
    x, w, y, a, loss = mk([4, 8]), mk([8, 10]), mk([4], DType.U32), mk([4]), mk([4])
    bad = [
        dict(hidden=mk([4, 7])), dict(weight=mk([8])), dict(targets=mk([4])), dict(targets=mk([3], DType.U32)),
        dict(weights=mk([3])), dict(row_loss=mk([5])), dict(hidden=mk([4, 8], DType.U32)), dict(grad_hidden=mk([4, 9])),
        dict(grad_weight=mk([8, 9])), dict(grad_weight=mk([8, 10], DType.U32)), dict(vocab_piece=-1),
        dict(grad_hidden=mk([4, 8]), weights=None), dict(workspace=mk([4])), dict(grad_scale=float("nan")),
    ]
    for over in bad:
        args = dict(hidden=x, weight=w, targets=y, weights=a, row_loss=loss)
        args.update(over)
        with pytest.raises(FtError):
            eng.linear_cross_entropy(cuda_ctx, **args)
    with pytest.raises(FtError):
        eng.linear_cross_entropy_bt(cuda_ctx, x, w, y, a, loss)


@gpu
@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("vocab_major", [False, True])
def test_gradient_of_the_hidden_rows_alone(cuda_ctx, eng, mode, vocab_major):
    """A frozen head (its own way through the vocabulary): sizes around tiles, pieces and parts of K, rows
    whose maximum jumps by 2^60 and more from piece to piece, and rows that are sure of their target."""
    for i, (t, h, v, piece) in enumerate(SIZES + [(300, 64, 9000, 2048), (520, 320, 5000, 4096), (64, 128, 12000, 0)]):
        for types, gtypes in (((F16, F16), (F16, F16)), ((F32, F32), (F32, F32)), ((F32, F16), (F32, F32))):
            s = 512.0 if F16 in gtypes else 1.0
            x, w, y, a = _make(t, h, v, types, vocab_major, ("half", "none", "beyond")[i % 3], 300 + i)
            q = _truth(x, w, y, a, s, vocab_major)
            got = _call(cuda_ctx, eng, mode, x, w, y, a, s, vocab_major, gtypes, "hidden", piece)
            _check(got, q, _bounds(q, mode, types, gtypes), vocab_major, f"{(t, h, v, piece)}")


@gpu
@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("order", ["rising", "falling"])
def test_logits_that_jump_between_pieces(cuda_ctx, eng, mode, order):
    """One column of each piece carries logits of 0, 90, 180, 270, ...: what the pieces before have left is
    scaled away by far more than f32's smallest number, or the later ones are."""
    t, h, v, piece = 40, 32, 2048, 512
    x, w, y, a = _make(t, h, v, (F16, F16), True, "none", 41)
    w *= 0.1
    x[:, 0] = 30.0
    for k in range(4):
        w[k * 512 + 77, 0] = 3.0 * (k if order == "rising" else 3 - k)
    y[: t // 2] = 3 * 512 + 77 if order == "rising" else 77
    q = _truth(x, w, y, a, 1.0, True)
    for want in ("hidden", "both"):
        got = _call(cuda_ctx, eng, mode, x, w, y, a, 1.0, True, (F32, F32), want, piece)
        _check(got, q, _bounds(q, mode, (F16, F16), (F32, F32)), True, want)


@gpu
@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("vocab_major", [False, True])
def test_losses_alone(cuda_ctx, eng, mode, vocab_major):
    """No gradient: from one row to more than two tiles of rows, with everything skipped, odd widths, and a
    vocabulary that ends inside a tile of any width."""
    for i, (t, h, v) in enumerate([(1, 8, 9), (1, 576, 6001), (2, 40, 33), (31, 64, 20000), (64, 136, 3000), (65, 72, 777), (128, 64, 1024),
                                   (129, 64, 1025), (256, 31, 4096), (257, 48, 900), (520, 24, 1500)]):
        for types in ((F16, F16), (F32, F16), (F16, F32)):
            x, w, y, a = _make(t, h, v, types, vocab_major, ("none", "beyond", "half", "all")[i % 4], 500 + i)
            x[y == SKIP] = float("inf")
            q = _truth(x, w, y, a, 1.0, vocab_major)
            got = _call(cuda_ctx, eng, mode, x, w, y, a, 1.0, vocab_major, want="none")
            _check(got, q, _bounds(q, mode, types, (F32, F32)), vocab_major, f"{(t, h, v)}")


@gpu
@pytest.mark.parametrize("mode", MODES)
def test_a_very_large_vocabulary(cuda_ctx, eng, mode):
    """More columns than one grid of the exact products reaches, a hidden size of one."""
    v = (1 << 23) + 1001
    x, w, y, a = _make(3, 1, v, (F32, F32), False, "none", 61)
    y[1] = v - 1
    q = _truth(x, w, y, a, 1.0, False)
    got = _call(cuda_ctx, eng, mode, x, w, y, a, 1.0, False, want="none")
    _check(got, q, _bounds(q, mode, (F32, F32), (F32, F32)), False)


@gpu
def test_a_weight_beyond_two_to_the_31_elements(cuda_ctx, eng):
    """1.1 million columns of 2048 f16 values: offsets pass 32 bits in the weight and in its gradient.  The
    last columns count, everything is checked where it can be told cheaply: losses and dh against sums
    over blocks in f64, dW at its first and last columns."""
    from ferrotensor_b200.engine import GemmMode
    t, h, v = 5, 2048, 1_100_000
    g = torch.Generator(device="cuda").manual_seed(3)
    w = torch.empty((v, h), dtype=F16, device="cuda")
    for part in w.split(100_000):
        part.copy_(torch.randn(part.shape, generator=g, device="cuda") * 0.02)
    x = torch.randn((t, h), generator=g, device="cuda").to(F16)
    y = torch.tensor([0, v - 1, v // 2, SKIP, v - 2], device="cuda")
    w[v - 1] += x[1] * 0.003
    a = torch.full((t,), 0.25, device="cuda")
    loss, gh, gw = torch.empty(t, device="cuda"), torch.empty_like(x), torch.empty_like(w)
    cuda_ctx.set_gemm_mode(GemmMode.F16)
    try:
        eng.linear_cross_entropy_bt(cuda_ctx, _ut(x), _ut(w), _ut(_targets(y)), _ut(a), _ut(loss), _ut(gh), _ut(gw), grad_scale=4096.0)
        cuda_ctx.synchronize()
    finally:
        cuda_ctx.set_gemm_mode(GemmMode.F32)
    X = x.double()
    lse = torch.logsumexp(torch.stack([torch.logsumexp(X @ p.double().t(), 1) for p in w.split(100_000)]), 0)
    live = y != SKIP
    yy = torch.where(live, y, 0)
    want = torch.where(live, lse - (X * w[yy].double()).sum(1), 0.0)
    assert ((loss.double() - want).abs() <= 1e-5 * (1 + want.abs())).all()
    c = torch.where(live, 0.25 * 4096.0, 0.0)[:, None]
    dh = -c * w[yy].double()
    mag = dh.abs()
    at = 0
    for p in w.split(100_000):
        P = torch.exp(X @ p.double().t() - lse[:, None]) * c
        dh += P @ p.double()
        mag += P @ p.double().abs()
        for cols in (slice(0, 3), slice(len(p) - 3, len(p))):
            G = P[:, cols].clone()
            for r in range(t):
                k = int(yy[r]) - at - cols.start
                if live[r] and 0 <= k < 3:
                    G[r, k] -= float(c[r])
            dw = G.t() @ X
            # g and the result are rounded to f16 once each, relative to each row's share
            tol = 2.0 ** -10 * (G.abs().t() @ X.abs()) + 2.0 ** -24
            assert ((gw[at + cols.start:at + cols.stop].double() - dw).abs() <= tol).all(), at
        at += len(p)
    # every term of the sum carries a g (or E) rounded to f16, the sum loses at most 2^-23 of what it has come
    # to for each group of 16, the result is rounded to f16: against the sum of magnitudes
    assert ((gh.double() - dh).abs() <= (2.0 ** -11 + v / 16 * 2.0 ** -23) * mag + 2.0 ** -11 * dh.abs() + 2.0 ** -24).all()


# (rows, hidden, vocab): every number of rows that a kernel is built for and the first that it is not, hidden
# sizes and vocabularies off every vector width, slices that end inside a warp, vocabularies wide enough
# for one, two and four columns a lane, and one row of one value
FEW = [(1, 1, 1), (1, 576, 14400), (2, 130, 7111), (4, 36, 129), (5, 2, 3), (7, 513, 7106), (8, 260, 1000), (9, 64, 2050),
       (13, 67, 515), (16, 132, 4097), (16, 20, 15000), (17, 40, 300), (3, 2700, 200), (16, 2700, 90)]


@gpu
@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("types,gtypes", [((F16, F16), (F16, F16)), ((F32, F16), (F32, F32)), ((F32, F32), (F32, F32)),
                                          ((F16, F32), (F16, F16))])
@pytest.mark.parametrize("vocab_major", [False, True])
def test_few_rows(cuda_ctx, eng, mode, types, gtypes, vocab_major):
    for i, (t, h, v) in enumerate(FEW):
        mask = ("none", "half", "beyond", "last")[i % 4]
        s = 64.0 if F16 in gtypes else 1.0
        x, w, y, a = _make(t, h, v, types, vocab_major, mask, 300 + i)
        x[y == SKIP] = float("nan")
        a[y == SKIP] = float("inf")
        q = _truth(x, w, y, a, s, vocab_major)
        tols = _bounds(q, mode, types, gtypes)
        for want in ("both", "hidden", "none"):
            got = _call(cuda_ctx, eng, mode, x, w, y, a, s, vocab_major, gtypes, want)
            _check(got, q, tols, vocab_major, f"{(t, h, v)} {want}")
            again = _call(cuda_ctx, eng, mode, x, w, y, a, s, vocab_major, gtypes, want)
            assert all(p is None or torch.equal(p, r) for p, r in zip(got, again))


@gpu
@pytest.mark.parametrize("vocab_major", [False, True])
def test_few_rows_beside_infinite_weights(cuda_ctx, eng, vocab_major):
    """A skipped row's gradient is zero whatever the weights hold; so is what it adds to theirs."""
    x, w, y, a = _make(6, 40, 200, (F32, F32), vocab_major, "none", 3)
    y[[1, 4]] = SKIP
    x[1] = float("inf")
    if vocab_major:
        w[7, 3] = float("inf")
    else:
        w[3, 7] = float("inf")
    for mode in MODES:
        loss, gh, gw = _call(cuda_ctx, eng, mode, x, w, y, a, 1.0, vocab_major)
        assert (loss[[1, 4]] == 0).all() and (gh[[1, 4]] == 0).all()
        assert not loss[0].isfinite() and gw.isnan().any()
    y[:] = SKIP
    for mode in MODES:
        loss, gh, gw = _call(cuda_ctx, eng, mode, x, w, y, a, 1.0, vocab_major)
        assert (loss == 0).all() and (gh == 0).all() and (gw == 0).all()


@gpu
def test_few_rows_agree_with_many(cuda_ctx, eng):
    """The same rows alone and in a batch: both within the bound of the exact products, so within twice
    that of each other."""
    for vocab_major in (False, True):
        x, w, y, a = _make(40, 200, 3000, (F32, F32), vocab_major, "none", 21)
        many = _call(cuda_ctx, eng, "F32", x, w, y, a, 1.0, vocab_major, want="hidden")
        for r in (slice(0, 1), slice(3, 9), slice(20, 36)):
            q = _truth(x[r], w, y[r], a[r], 1.0, vocab_major)
            tol = _bounds(q, "F32", (F32, F32), (F32, F32))
            few = _call(cuda_ctx, eng, "F32", x[r], w, y[r], a[r], 1.0, vocab_major, want="hidden")
            assert ((few[0] - many[0][r]).abs() <= 2 * tol[0]).all() and ((few[1] - many[1][r]).abs() <= 2 * tol[1]).all()


@gpu
@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("vocab_major", [False, True])
def test_few_rows_captured(eng, mode, vocab_major):
    """A graph of a call of five rows follows its inputs, which rows are skipped included."""
    from ferrotensor_b200.engine import ComputeEngine, CudaContext, DType, GemmMode, UnifiedTensor
    first, second = (_make(5, 72, 1900, (F32, F32), vocab_major, "none", 61 + k) for k in range(2))
    second[2][3] = SKIP
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        ctx = CudaContext(0)
    ctx.set_gemm_mode(GemmMode[mode])
    e = ComputeEngine(ctx)
    x, w, y, a = (v.clone() for v in first)
    y = _targets(y)
    loss, gh, gw = torch.empty(5, device="cuda"), torch.empty_like(x), torch.empty_like(w)
    n = e.linear_cross_entropy_workspace(ctx, _ut(x), _ut(w), _ut(gh), _ut(gw), vocab_major=vocab_major)
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")
    f = e.linear_cross_entropy_bt if vocab_major else e.linear_cross_entropy

    def call():
        f(ctx, _ut(x), _ut(w), _ut(y), _ut(a), _ut(loss), _ut(gh), _ut(gw), 1.0, workspace=UnifiedTensor(ws, [n // 4], DType.U32))
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        call()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            call()
    torch.cuda.synchronize()
    for to, new in ((x, second[0]), (w, second[1]), (y, _targets(second[2])), (a, second[3])):
        to.copy_(new)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        graph.replay()
        graph.replay()
    torch.cuda.synchronize()
    q = _truth(second[0], second[1], second[2], second[3], 1.0, vocab_major)
    _check((loss, gh, gw), q, _bounds(q, mode, (F32, F32), (F32, F32)), vocab_major)
