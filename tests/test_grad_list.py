"""The global gradient norm and the clip by it over lists of tensors, against 64-bit sums.

The norm is a sum of squares in f64, rounded to f32 once: half a step, 2^-24 relative, and a unit of
f64 for each term.  A clipped value is factor * g: the factor is rounded to f32, the product to the
result's type, so 2^-24 + 2^-24 relative (+ 2^-11 for f16, + half of f16's or f32's smallest step)."""

import ctypes as C

import numpy as np
import pytest
import torch

F16, F32 = torch.float16, torch.float32


@pytest.fixture(scope="module")
def lib():
    from ferrotensor_b200 import _build, _lib
    _build.build()
    return _lib.load()


def _arrays(items):
    n = len(items)
    return ((C.c_void_p * n)(*[i[0] for i in items]), (C.c_size_t * n)(*[i[1] for i in items]), (C.c_int * n)(*[i[2] for i in items]))


@pytest.mark.parametrize("items,message", [
    ([(None, 4, 0)], "NULL"), ([(0x1000, 4, 2)], "type"), ([(0x1002, 4, 0)], "aligned"), ([(0x1001, 4, 1)], "aligned"),
    ([(0x1000, 1 << 50, 0)], "too large"), ([(0x1000, 4, 0), (0x2000, 4, -1)], "type"),
])
def test_refusals_of_a_list(lib, items, message):
    fake = C.create_string_buffer(1 << 16)
    out = C.c_void_p()
    assert lib.ft_grad_list_create(C.cast(fake, C.c_void_p), len(items), *_arrays(items), C.byref(out)) == 1
    assert message in lib.ft_last_error().decode() and not out.value


def test_null_arguments(lib):
    fake = C.create_string_buffer(1 << 16)
    h, out = C.cast(fake, C.c_void_p), C.c_void_p()
    assert lib.ft_grad_list_create(None, 0, None, None, None, C.byref(out)) == 1
    assert lib.ft_grad_list_create(h, 2, None, None, None, C.byref(out)) == 1
    assert lib.ft_grad_list_create(h, 0, None, None, None, None) == 1
    assert lib.ft_global_grad_norm(h, None, 1.0, None) == 1
    assert lib.ft_clip_grad_global_norm(None, None, None, 1.0, 1.0, None) == 1
    assert lib.ft_grad_list_destroy(None) == 0


gpu = pytest.mark.gpu


@pytest.fixture(scope="module")
def eng(cuda_ctx):
    from ferrotensor_b200.engine import ComputeEngine
    return ComputeEngine(cuda_ctx)


def _ut(x):
    from ferrotensor_b200.engine import DType, UnifiedTensor
    return UnifiedTensor(x.reshape(-1).view(torch.uint8), list(x.shape), DType.F32 if x.dtype is F32 else DType.FP16)


def _tensors(counts, kinds, seed, scale=1.0, offset=True):
    """Tensors that begin at any multiple of their element size, between guard values."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    out, whole = [], []
    for i, (n, k) in enumerate(zip(counts, kinds)):
        at = 16 + (i % 5 if offset else 0)
        flat = torch.full((n + 40,), 3.0, dtype=k, device="cuda")
        flat[at:at + n] = (torch.randn(n, generator=g, device="cuda") * scale * (1 + i % 4)).to(k)
        out.append(flat[at:at + n])
        whole.append((flat, at, n))
    return out, whole


def _guards_hold(whole):
    for flat, at, n in whole:
        assert (flat[:at] == 3.0).all() and (flat[at + n:] == 3.0).all()


def _true_norm(xs, s):
    return float(np.sqrt(sum(float(x.double().square().sum()) for x in xs))) * abs(s)


def _check_values(out, src, factor):
    for o, g in zip(out, src):
        want = g.double() * factor
        u = 2.0 ** -23 + (2.0 ** -11 if o.dtype is F16 else 0.0)
        tol = u * 1.01 * want.abs() + (2.0 ** -25 if o.dtype is F16 else 2.0 ** -150)
        assert ((o.double() - want).abs() <= tol).all()


SHAPES = [[1], [0, 5, 0], [256] * 64, [256] * 63 + [257], [16384], [100] * 40, [3, 1, 8192, 8193, 7], [100000, 33], [16] * 400, [2 * 8192 * 1300 + 5], [31] * 3 + [70001] * 9]


@gpu
@pytest.mark.parametrize("counts", SHAPES, ids=range(len(SHAPES)))
@pytest.mark.parametrize("kinds", [(F32,), (F16,), (F32, F16)], ids=["f32", "f16", "both"])
def test_norm_and_clip(cuda_ctx, eng, counts, kinds):
    from ferrotensor_b200.engine import GradientList
    ks = [kinds[i % len(kinds)] for i in range(len(counts))]
    xs, whole = _tensors(counts, ks, len(counts))
    norm = torch.full((5,), 9.0, device="cuda")
    nt = _ut(norm[:4])
    grads = GradientList(cuda_ctx, [_ut(x) for x in xs])
    for s in (1.0, -0.25):
        want = _true_norm(xs, s)
        eng.global_grad_norm(cuda_ctx, grads, nt, grad_scale=s)
        got = norm.tolist()
        assert abs(got[0] - want) <= 2.0 ** -23 * want and got[1:3] == [1.0, s] and got[4] == 9.0
        for max_norm, clipped in ((want * 0.5, True), (want * 2, False), (0.0, False), (-1.0, False), (float("inf"), False)):
            for to in ({F32: F32, F16: F16}, {F32: F32, F16: F32}, {F32: F16, F16: F16}):
                kept = [x.clone() for x in xs]
                ys, guard = _tensors(counts, [to[k] for k in ks], 1)
                eng.clip_grad_global_norm(cuda_ctx, grads, max_norm, nt, s, GradientList(cuda_ctx, [_ut(y) for y in ys]))
                factor = s * max_norm / (want + 1e-6) if clipped and want > max_norm else s
                got = norm.tolist()
                assert got[1] == 1.0 and abs(got[2] - factor) <= 2.0 ** -22 * abs(factor)
                _check_values(ys, kept, factor)
                _guards_hold(guard)
                assert all(torch.equal(x, k) for x, k in zip(xs, kept))
    _guards_hold(whole)


@gpu
@pytest.mark.parametrize("kinds", [(F32,), (F32, F16)], ids=["f32", "both"])
def test_in_place(cuda_ctx, eng, kinds):
    from ferrotensor_b200.engine import GradientList
    counts = [5, 20000, 8192, 1]
    ks = [kinds[i % len(kinds)] for i in range(len(counts))]
    for out_is_list in (False, True):
        xs, whole = _tensors(counts, ks, 3)
        kept = [x.clone() for x in xs]
        grads = GradientList(cuda_ctx, [_ut(x) for x in xs])
        same = GradientList(cuda_ctx, [_ut(x) for x in xs]) if out_is_list else None
        want = _true_norm(xs, 1.0)
        norm = torch.zeros(4, device="cuda")
        eng.clip_grad_global_norm(cuda_ctx, grads, want * 3, _ut(norm), out=same)      # below the limit: nothing changes
        assert all(torch.equal(x, k) for x, k in zip(xs, kept)) and norm[2] == 1.0
        eng.clip_grad_global_norm(cuda_ctx, grads, want / 3, out=same)                 # no norm asked for
        _check_values(xs, kept, want / 3 / (want + 1e-6))
        _guards_hold(whole)


@gpu
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_a_norm_that_is_not_finite_writes_nothing(cuda_ctx, eng, value):
    from ferrotensor_b200.engine import GradientList
    xs, _ = _tensors([9000, 40], [F32, F16], 5)
    xs[1][17] = value
    kept = [x.clone() for x in xs]
    ys, _ = _tensors([9000, 40], [F32, F32], 6)
    before = [y.clone() for y in ys]
    norm = torch.zeros(4, device="cuda")
    grads, out = (GradientList(cuda_ctx, [_ut(t) for t in ts]) for ts in (xs, ys))
    for o in (None, out):
        eng.clip_grad_global_norm(cuda_ctx, grads, 1.0, _ut(norm), 0.5, o)
        assert norm[1] == 0 and not norm[0].isfinite() and norm[2] == 0.5
    for a, b in zip(xs + ys, kept + before):
        assert torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0))


@gpu
@pytest.mark.parametrize("scale", [1e-25, 1e-42, 1e25])
def test_squares_outside_the_range_of_f32(cuda_ctx, eng, scale):
    from ferrotensor_b200.engine import GradientList
    xs, _ = _tensors([10000, 3], [F32, F32], 7, scale)
    norm = torch.zeros(4, device="cuda")
    eng.global_grad_norm(cuda_ctx, GradientList(cuda_ctx, [_ut(x) for x in xs]), _ut(norm))
    want = _true_norm(xs, 1.0)
    assert norm[1] == 1 and abs(float(norm[0]) - want) <= 2.0 ** -23 * want + 2.0 ** -149


@gpu
def test_a_tensor_listed_twice_counts_twice_and_is_not_written(cuda_ctx, eng):
    from ferrotensor_b200._lib import FtError
    from ferrotensor_b200.engine import GradientList
    xs, _ = _tensors([500], [F32], 8)
    twice = GradientList(cuda_ctx, [_ut(xs[0]), _ut(xs[0])])
    norm = torch.zeros(4, device="cuda")
    eng.global_grad_norm(cuda_ctx, twice, _ut(norm))
    want = _true_norm(xs, 1.0) * 2 ** 0.5
    assert abs(float(norm[0]) - want) <= 2.0 ** -23 * want
    with pytest.raises(FtError, match="overlap"):
        eng.clip_grad_global_norm(cuda_ctx, twice, 1.0)
    ys, _ = _tensors([500, 500], [F32, F32], 9)
    eng.clip_grad_global_norm(cuda_ctx, twice, want / 2, out=GradientList(cuda_ctx, [_ut(y) for y in ys]))
    assert torch.equal(ys[0], ys[1])


@gpu
def test_refusals(cuda_ctx, eng):
    from ferrotensor_b200._lib import FtError
    from ferrotensor_b200.engine import CudaContext, DType, GradientList, UnifiedTensor
    buf = torch.zeros(4096, device="cuda")
    part = lambda a, n, k=F32: _ut(buf.view(torch.uint8)[a:a + n * k.itemsize].view(k))  # noqa: E731
    src = GradientList(cuda_ctx, [part(0, 100), part(400, 100)])
    norm = _ut(torch.zeros(4, device="cuda"))
    for bad, what in [([part(4, 100), part(2000, 100)], "overlaps"), ([part(400, 100), part(0, 100)], "overlaps"),
                      ([part(0, 100, F16), part(4000, 100)], "overlaps"), ([part(1000, 100)], "different numbers"),
                      ([part(1000, 100), part(2000, 99)], "different numbers"), ([part(1000, 100), part(1200, 100)], "overlap")]:
        with pytest.raises(FtError, match=what):
            eng.clip_grad_global_norm(cuda_ctx, src, 1.0, norm, out=GradientList(cuda_ctx, bad))
    ok = GradientList(cuda_ctx, [part(1000, 100), part(2000, 100)])
    for args in (dict(max_norm=float("nan")), dict(grad_scale=float("inf")), dict(norm_out=part(100, 4)), dict(norm_out=part(2096, 4))):
        a = dict(max_norm=1.0, norm_out=norm, grad_scale=1.0)
        a.update(args)
        with pytest.raises(FtError):
            eng.clip_grad_global_norm(cuda_ctx, src, out=ok, **a)
    with pytest.raises(FtError):
        eng.global_grad_norm(cuda_ctx, src, part(100, 4))
    with pytest.raises(FtError):
        eng.global_grad_norm(cuda_ctx, src, _ut(torch.zeros(3, device="cuda")))
    with pytest.raises(FtError, match="another context"):
        eng.global_grad_norm(CudaContext(0), src, norm)
    with pytest.raises(FtError):
        GradientList(cuda_ctx, [UnifiedTensor.empty_with_dtype(cuda_ctx, [4], DType.U32)])
    with pytest.raises(FtError):
        GradientList(cuda_ctx, [UnifiedTensor(torch.zeros(8, dtype=torch.uint8, device="cuda"), [4], DType.F32)])


@gpu
def test_more_than_two_to_the_32_values(cuda_ctx, eng):
    """One tensor of 2^32 + 9 f16 ones and a half in its last place, clipped in place."""
    from ferrotensor_b200.engine import GradientList
    n = (1 << 32) + 9
    x = torch.ones(n, dtype=F16, device="cuda")
    x[-1] = 0.5
    norm = torch.zeros(4, device="cuda")
    want = (n - 0.75) ** 0.5
    eng.clip_grad_global_norm(cuda_ctx, GradientList(cuda_ctx, [_ut(x)]), want / 4, _ut(norm))
    assert abs(float(norm[0]) - want) <= 2.0 ** -23 * want
    factor = float(norm[2])
    assert abs(factor - 0.25) <= 1e-6
    assert float(x[-1]) == 0.125 and all(bool((p == 0.25).all()) for p in x[:-1].split(1 << 30))


@gpu
def test_captured_and_replayed(cuda_ctx):
    from ferrotensor_b200.engine import ComputeEngine, CudaContext, GradientList
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        ctx = CudaContext(0)
    eng = ComputeEngine(ctx)
    xs, _ = _tensors([30000, 77], [F32, F16], 11)
    ys, _ = _tensors([30000, 77], [F32, F32], 12)
    norm = torch.zeros(4, device="cuda")
    src, dst = (GradientList(ctx, [_ut(t) for t in ts]) for ts in (xs, ys))
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        eng.clip_grad_global_norm(ctx, src, 2.0, _ut(norm), out=dst)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            eng.clip_grad_global_norm(ctx, src, 2.0, _ut(norm), out=dst)
    for k in range(3):
        new, _ = _tensors([30000, 77], [F32, F16], 20 + k)
        for x, n in zip(xs, new):
            x.copy_(n)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graph.replay()
        torch.cuda.synchronize()
        want = _true_norm(xs, 1.0)
        assert abs(float(norm[0]) - want) <= 2.0 ** -23 * want
        _check_values(ys, xs, 2.0 / (want + 1e-6))


@gpu
def test_a_step_with_a_trained_head(cuda_ctx, eng):
    """Loss, both gradients, norm, clip and AdamW in a row, as a trainer makes the calls, twice in a row
    against the same step in 64 bits.  Gradients of 2^-11 operands (F16X2: 2^-21) give a norm and an
    update within the bounds of the operators; AdamW's first steps move a weight by at most lr, and
    its sign is only free where a gradient is smaller than its own error."""
    from ferrotensor_b200.engine import AdamParams, DType, GemmMode, GradientList, UnifiedTensor
    g = torch.Generator(device="cuda").manual_seed(3)
    t, h, v, lr, max_norm = 200, 64, 900, 1e-2, 0.05
    x = torch.randn((t, h), generator=g, device="cuda")
    w = torch.randn((h, v), generator=g, device="cuda") * 0.1
    y = torch.randint(0, v, (t,), generator=g, device="cuda", dtype=torch.int32)
    y[::4] = -1
    a = torch.full((t,), 1.0 / 150, device="cuda")
    gh, gw = torch.empty_like(x), torch.empty_like(w)
    m, s2 = torch.zeros_like(w), torch.zeros_like(w)
    loss, norm = torch.empty(t, device="cuda"), torch.zeros(4, device="cuda")
    W, M, S = w.double(), m.double(), s2.double()
    other = torch.randn(777, generator=g, device="cuda") * 1e-3       # an adapter's gradient in the same list
    first = other.clone()
    grads = GradientList(cuda_ctx, [_ut(gw), _ut(other)])
    yt = UnifiedTensor(y.view(torch.uint8), [t], DType.U32)
    cuda_ctx.set_gemm_mode(GemmMode.F16X2)
    try:
        for step in (1, 2):
            other.copy_(first)
            eng.linear_cross_entropy(cuda_ctx, _ut(x), _ut(w), yt, _ut(a), _ut(loss), _ut(gh), _ut(gw))
            eng.clip_grad_global_norm(cuda_ctx, grads, max_norm, _ut(norm))
            eng.adamw_update(cuda_ctx, _ut(w), _ut(gw), _ut(m), _ut(s2), AdamParams(lr=lr, weight_decay=0.0, eps=1e-3, t=float(step)))
            live = y >= 0
            X = torch.where(live[:, None], x.double(), 0.0)
            z = X @ W
            p = torch.softmax(z, 1)
            p[live, y[live].long()] -= 1
            G = torch.where(live[:, None], p / 150, 0.0)
            want_loss = torch.where(live, torch.logsumexp(z, 1) - z.gather(1, y.clamp(min=0).long()[:, None])[:, 0], 0.0)
            assert (loss.double() - want_loss).abs().max() <= 1e-4
            DW = X.t() @ G
            n = float((DW.square().sum() + first.double().square().sum()).sqrt())
            assert abs(float(norm[0]) - n) <= 1e-4 * n and n > max_norm
            DW = DW * (max_norm / (n + 1e-6))
            assert (gw.double() - DW).abs().max() <= 1e-4 * float(DW.abs().max())
            assert (other.double() - first.double() * max_norm / (n + 1e-6)).abs().max() <= 1e-4 * float(first.abs().max())
            M = 0.9 * M + 0.1 * DW
            S = 0.999 * S + 0.001 * DW * DW
            W = W - lr * (M / (1 - 0.9 ** step)) / ((S / (1 - 0.999 ** step)).sqrt() + 1e-3)
            # eps = 1e-3 is above every |gradient|, so an update is Lipschitz in it: lr / eps = 10
            assert (w.double() - W).abs().max() <= 10 * 1e-4 * float(DW.abs().max()) * 2 + 1e-6
    finally:
        cuda_ctx.set_gemm_mode(GemmMode.F32)


@gpu
def test_a_list_that_goes_away_during_a_capture(cuda_ctx):
    """The garbage collector may meet a list while the stream is being captured: the capture stands, and the
    graph and lists made later work."""
    from ferrotensor_b200.engine import ComputeEngine, CudaContext, GradientList
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        ctx = CudaContext(0)
    eng = ComputeEngine(ctx)
    xs, _ = _tensors([30000, 77], [F32, F16], 11)
    norm = torch.zeros(4, device="cuda")
    src, other = (GradientList(ctx, [_ut(x) for x in xs]) for _ in range(2))
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        eng.global_grad_norm(ctx, src, _ut(norm))
        eng.global_grad_norm(ctx, other, _ut(norm))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            eng.global_grad_norm(ctx, src, _ut(norm))
            other.close()
            eng.global_grad_norm(ctx, src, _ut(norm), grad_scale=2.0)
    for k in range(3):
        later = GradientList(ctx, [_ut(x) for x in xs])
        norm.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graph.replay()
        torch.cuda.synchronize()
        want = _true_norm(xs, 2.0)
        assert abs(float(norm[0]) - want) <= 2.0 ** -23 * want
        with torch.cuda.stream(side):
            eng.global_grad_norm(ctx, later, _ut(norm))
        torch.cuda.synchronize()
        assert abs(float(norm[0]) - want / 2) <= 2.0 ** -23 * want
        later.close()
    src.close()
    ctx.close()


def test_a_closed_list_of_outputs_is_refused(lib, monkeypatch):
    """It must not turn into "no list of outputs", which scales the gradients themselves."""
    from ferrotensor_b200 import engine
    made = []
    monkeypatch.setattr(engine, "call", lambda name, *a: made.append(name))
    fake = type("Ctx", (), {"handle": 1})()
    open_list, closed = (engine.GradientList.__new__(engine.GradientList) for _ in range(2))
    for li in (open_list, closed):
        li.ctx, li.tensors, li.handle = fake, [], C.c_void_p(64)
    closed.close()
    eng = engine.ComputeEngine.__new__(engine.ComputeEngine)
    try:
        with pytest.raises(engine.FtError, match="closed"):
            eng.clip_grad_global_norm(fake, open_list, 1.0, out=closed)
        eng.clip_grad_global_norm(fake, open_list, 1.0)
    finally:
        open_list.close()
    assert made == ["ft_grad_list_destroy", "ft_clip_grad_global_norm", "ft_grad_list_destroy"]
