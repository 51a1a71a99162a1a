"""The linear cross entropy where its tiles, signs and ranges meet: results of several tiles a block, rows that
are sure of their target, tokens far below the likeliest, sums over many rows, infinite logits.  The formula
in 64 bits and the bounds are those of the tests of its values; a tighter bound is derived where it is used."""

import numpy as np
import pytest
import torch

from tests.test_linear_ce import F16, F32, MODES, SKIP, _bounds, _call, _check, _make, _targets, _truth, _ut

gpu = pytest.mark.gpu


@pytest.fixture(scope="module")
def eng(cuda_ctx):
    from ferrotensor_b200.engine import ComputeEngine
    return ComputeEngine(cuda_ctx)


@pytest.mark.parametrize("what", ["hidden", "weight", "targets", "weights", "row_loss", "grad_hidden", "grad_weight", "workspace", "norm_out"])
def test_buffers_that_are_too_small_or_elsewhere(monkeypatch, what):
    """A tensor whose buffer is a byte short or on another device never reaches the library."""
    from ferrotensor_b200 import engine
    from ferrotensor_b200.engine import DType, FtError, UnifiedTensor
    calls = []
    monkeypatch.setattr(engine, "call", lambda name, *a: calls.append(name))
    ctx = type("Ctx", (), {"handle": 1, "device_index": -1})()      # (-1: what a tensor on the CPU gives)
    eng = engine.ComputeEngine.__new__(engine.ComputeEngine)

    def tensor(name, shape, kind=DType.F32):
        n = int(np.prod(shape)) * kind.size_bytes() - (name == short)
        storage = torch.empty(n, dtype=torch.uint8)
        if name == far:
            storage = type("Elsewhere", (), dict(nbytes=n, device="cuda:1", get_device=lambda self: 1, data_ptr=lambda self: 256))()
        return UnifiedTensor(storage, shape, kind)

    def run():
        if what == "norm_out":
            lists = engine.GradientList.__new__(engine.GradientList)
            lists.ctx, lists.tensors, lists.handle = ctx, [], None
            eng.global_grad_norm(ctx, lists, tensor("norm_out", [4]))
            eng.clip_grad_global_norm(ctx, lists, 1.0, tensor("norm_out", [4]))
            return
        t = {n: tensor(n, s, k) for n, s, k in (("hidden", [3, 8], DType.FP16), ("weight", [8, 5], DType.F32), ("targets", [3], DType.U32),
                                                ("weights", [3], DType.F32), ("row_loss", [3], DType.F32), ("grad_hidden", [3, 8], DType.F32),
                                                ("grad_weight", [8, 5], DType.FP16), ("workspace", [64], DType.U32))}
        eng.linear_cross_entropy(ctx, **t)

    short = far = None
    run()
    assert calls.pop() in ("ft_linear_cross_entropy", "ft_clip_grad_global_norm")
    calls.clear()
    if what != "workspace":                                        # (its size is the library's to judge)
        short = what
        with pytest.raises(FtError, match=what):
            run()
    short, far = None, what
    with pytest.raises(FtError, match=what):
        run()
    assert not calls


@gpu
@pytest.mark.parametrize("mode", ["F16", "F16X2"])
@pytest.mark.parametrize("vocab_major", [False, True])
@pytest.mark.parametrize("rows,hidden", [(64, 576), (300, 576), (64, 896), (300, 960), (130, 64)])
def test_f16_weight_gradients_of_many_tiles(cuda_ctx, eng, mode, vocab_major, rows, hidden):
    """Hidden sizes whose tiles give a warp an odd number of 32-column blocks (192, 224 and 64 columns), few
    rows (a tile is multiplied sooner than it is stored) and several tiles for every block: each element
    of every tile, and the same bits each time."""
    x, w, y, a = _make(rows, hidden, 30208, (F16, F16), vocab_major, "half", 700 + hidden)
    q = _truth(x, w, y, a, 512.0, vocab_major)
    tols = _bounds(q, mode, (F16, F16), (F16, F16))
    first = _call(cuda_ctx, eng, mode, x, w, y, a, 512.0, vocab_major, (F16, F16))
    _check(first, q, tols, vocab_major)
    for _ in range(4):
        again = _call(cuda_ctx, eng, mode, x, w, y, a, 512.0, vocab_major, (F16, F16))
        assert all(torch.equal(p, r) for p, r in zip(first, again))


def _sure(t, h, v, types, vocab_major, offset, seed):
    """Rows whose target stands 12 to 20 above a spread of others, all logits `offset` higher than that."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    w = torch.randn((v, h), generator=g, device="cuda") * 0.1
    w[:, 0] = 32.0 if offset else 0.0
    y = torch.randint(0, v, (t,), generator=g, device="cuda")
    rest = w[y].clone()
    rest[:, 0] = 0.0
    lift = 12.0 + 8.0 * torch.rand((t, 1), generator=g, device="cuda")
    x = rest * (lift / rest.square().sum(dim=1, keepdim=True))
    x[:, 0] = offset / 32.0
    a = (torch.rand(t, generator=g, device="cuda") + 0.5) / t
    x, w = x.to(types[0]), w.to(types[1])
    return x, (w if vocab_major else w.t().contiguous()), y, a


def _sure_bounds(q, y, mode, types):
    """The bounds of the values' tests, but relative for every element of g: one with probability p is wrong by
    a share of p (its logit's error, against the target's and the sum's), the target's by a share of 1 - p
    and by the sum of the exponentials, which is f32 near 1 and takes at most v / 64 + 32 roundings in a row.
    (What is held as f16 is scaled so that the largest lies in 2^13 to 2^14: f16's smallest step, of which a
    rounding is half, is then at most 2^-37 of the largest, with a second half too.)"""
    X, W, p, c, g = q["X"].abs(), q["W"].abs(), q["p"], q["c"].abs(), q["g"].abs()
    (t, h), v = X.shape, W.shape[0]
    u, u16 = 2.0 ** -24, 2.0 ** -11

    def op(kind, m):
        if kind is F16 or mode == "F32":
            return 0.0, 0.0
        return (u16 if mode == "F16" else 2.0 ** -21), float(m.max()) * 2.0 ** -37
    (rx, ax), (rw, aw) = op(types[0], X), op(types[1], W)
    dX, dW_ = rx * X + ax, rw * W + aw
    dz = dX @ W.t() + X @ dW_.t() + dX @ dW_.t() + (h + 8) * u * (X @ W.t())
    worst = dz.max(dim=1, keepdim=True).values
    soft = 2.0 ** -20 + 2 * u * (q["z"].abs().max(dim=1, keepdim=True).values + q["lse"].abs()[:, None])
    rel = torch.expm1(dz + worst + soft + 2 * u * (q["z"] - q["lse"][:, None]).abs()) + 4 * u
    at = torch.zeros_like(p, dtype=torch.bool)
    at[torch.arange(t, device="cuda"), y] = True
    off = -torch.expm1(-q["loss"])[:, None]
    sure = off * rel.max(dim=1, keepdim=True).values + (v / 64 + 32) * u
    loss = (sure / (1 - off))[:, 0] * 1.01 + 2 * u * q["loss"]
    dg = c * torch.where(at, sure, p * rel)
    rg = {"F32": 0.0, "F16": u16, "F16X2": 2.0 ** -21}[mode]
    dg = dg + rg * (g + dg) + (0.0 if mode == "F32" else float(c.max()) * 2.0 ** -37)
    G = g + dg
    dh = dg @ (W + dW_) + g @ dW_ + (v + 64) * u * (G @ (W + dW_))
    dW = dg.t() @ (X + dX) + g.t() @ dX + (t + 64) * u * (G.t() @ (X + dX))
    return loss, dh + 2 * u * (q["dh"].abs() + dh) + 1e-40, dW + 2 * u * (q["dW"].abs() + dW) + 1e-40


def _sure_case(ctx, eng, mode, offset, size, wants):
    """Loss and gradients keep their relative accuracy where 1 - p is 1e-2 to 1e-5: at the target, and at tokens
    that share its tile; whatever all logits have in common."""
    rows, hidden, vocab, piece = size
    for types in ((F16, F16), (F32, F32)):
        for vocab_major in (False, True):
            x, w, y, a = _sure(rows, hidden, vocab, types, vocab_major, offset, 800 + rows)
            q = _truth(x, w, y, a, 1.0, vocab_major)
            assert 1e-8 < float(-torch.expm1(-q["loss"]).min()) and float(q["loss"].max()) < 0.2
            tols = _sure_bounds(q, y, mode, types)
            for want in wants:
                got = _call(ctx, eng, mode, x, w, y, a, 1.0, vocab_major, (F32, F32), want, piece)
                _check(got, q, tols, vocab_major, f"{types} {vocab_major} {want}")


@gpu
@pytest.mark.parametrize("offset", [0.0, 1000.0])
@pytest.mark.parametrize("size", [(16, 64, 3000, 0), (17, 64, 3000, 0), (120, 64, 3000, 0), (300, 64, 3000, 1024), (300, 288, 3000, 0)])
def test_sure_rows_exact(cuda_ctx, eng, offset, size):
    _sure_case(cuda_ctx, eng, "F32", offset, size, ("both", "hidden", "none"))


@gpu
@pytest.mark.parametrize("offset", [0.0, 1000.0])
@pytest.mark.parametrize("mode", ["F16", "F16X2"])
@pytest.mark.parametrize("rows", [1, 17, 120, 300, 600])
def test_sure_rows_losses_alone(cuda_ctx, eng, mode, offset, rows):
    _sure_case(cuda_ctx, eng, mode, offset, (rows, 64, 3000, 0), ("none",))


@gpu
@pytest.mark.parametrize("offset", [0.0, 1000.0])
@pytest.mark.parametrize("mode,size", [("F16", (16, 64, 3000, 0)), ("F16", (17, 64, 3000, 0)), ("F16", (120, 64, 3000, 0)), ("F16", (300, 288, 3000, 0)),
                                       ("F16", (140, 64, 3000, 1024)), ("F16X2", (300, 64, 3000, 0)), ("F16X2", (140, 64, 3000, 1024))])
def test_sure_rows_both_gradients(cuda_ctx, eng, mode, offset, size):
    _sure_case(cuda_ctx, eng, mode, offset, size, ("both", "none"))


@gpu
@pytest.mark.parametrize("offset", [0.0, 1000.0])
@pytest.mark.parametrize("mode,size", [(m, z) for m in ("F16", "F16X2") for z in [(16, 64, 3000, 0), (17, 64, 3000, 0), (120, 64, 3000, 0), (300, 288, 3000, 0),
                                                                                  (140, 64, 3000, 1024), (1100, 64, 3000, 0)]])
def test_sure_rows_hidden_gradient_alone(cuda_ctx, eng, mode, offset, size):
    _sure_case(cuda_ctx, eng, mode, offset, size, ("hidden",))


@gpu
@pytest.mark.parametrize("offset", [0.0, 1000.0])
@pytest.mark.parametrize("size", [(17, 64, 3000, 0), (200, 64, 3000, 0), (300, 288, 3000, 0)])
def test_sure_rows_gradient_made_in_place(cuda_ctx, eng, offset, size):
    _sure_case(cuda_ctx, eng, "F16X2", offset, size, ("both",))


@gpu
@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("rows", [3, 17, 100, 300])
def test_logits_of_minus_infinity(cuda_ctx, eng, mode, rows):
    """Columns of the vocabulary masked by a weight of -inf: they take no probability, a row whose target is
    masked has an infinite loss, and dW stays finite (its row pulls the masked column by -w h).  dh, which
    has 0 x -inf in its sum, is not looked at."""
    for kind in ((F16,) if mode == "F16X2" else (F16, F32)):
        x, w, y, a = _make(rows, 40, 700, (kind, kind), True, "none", 51)
        x[:, 0] = 0.5
        w[5::7, 0] = float("-inf")
        y = torch.where(y % 7 == 5, y - 1, y)
        y[1::2] = 5
        W, X = w.double(), x.double()
        z = X @ W.t()
        keep = torch.ones(700, dtype=torch.bool, device="cuda")
        keep[5::7] = False
        finite = dict(zip(("x", "w"), (x, w[keep])))
        inner = torch.where(y == 5, 0, torch.cumsum(keep, 0)[y] - 1)
        q = _truth(finite["x"], finite["w"], torch.where(y == 5, SKIP, inner), a, 1.0, True)
        tols = _bounds(q, mode, (kind, kind), (F32, F32))
        got = _call(cuda_ctx, eng, mode, x, w, y, a, 1.0, True)
        masked = y == 5
        assert (z[:, 5] == float("-inf")).all() and (got[0][masked] == float("inf")).all()
        assert ((got[0].double() - q["loss"]).abs() <= tols[0])[~masked].all()
        # dW of all rows: the ones with a masked target have the same softmax and no one-hot term inside
        zk = z[:, keep]
        p = torch.softmax(zk, dim=1)
        p[~masked, inner[~masked]] -= 1
        g = p * a.double()[:, None]
        full = torch.zeros(700, 40, dtype=torch.float64, device="cuda")
        full[keep] = g.t() @ X
        full[5] = -(a.double()[masked] @ X[masked])
        size = torch.zeros(700, 40, dtype=torch.float64, device="cuda")
        size[keep] = g.abs().t() @ X.abs()
        size[5] = a.double()[masked].abs() @ X[masked].abs()
        # operands and g within half a step of f16 (2^-21 and exact in the other modes), logits within 1e-2 for that
        rel = {"F32": 1e-4, "F16": 2e-2 if kind is F32 else 2e-3, "F16X2": 1e-4}[mode]
        assert ((got[2].double() - full).abs() <= rel * size + 1e-7).all()


@gpu
@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("size", [1e-25, 1e-30])
def test_operands_whose_scales_multiply_to_nothing(cuda_ctx, eng, mode, size):
    """f32 operands far below 1: every logit is 0 to f32, so each loss is log(vocab) to a few units of 2^-24 of
    it, every probability 1 / vocab, and the gradients follow in the operands' own size."""
    for rows, hidden, vocab in ((70, 40, 300), (300, 40, 300), (300, 320, 600)):
        x, w, y, a = _make(rows, hidden, vocab, (F32, F32), True, "half", 9)
        x, w, a = x * size, w * size, a.abs() + 0.01
        q = _truth(x / size, w / size, y, a, 1.0, True)
        live = q["live"]
        one = torch.zeros_like(q["z"])
        one[live, y[live]] = 1.0
        g = torch.where(live[:, None], (1.0 / vocab - one) * a.double()[:, None], 0.0)
        # 22 bits of each operand and of g (11 in FT_GEMM_F16), f32 sums
        rel = 2.0 ** -9 if mode == "F16" else 2.0 ** -16
        dh, dW = g @ q["W"], g.t() @ q["X"]
        for want in ("both", "hidden", "none"):
            loss, gh, gw = _call(cuda_ctx, eng, mode, x, w, y, a, 1.0, True, want=want)
            assert ((loss.double() - torch.where(live, np.log(vocab), 0.0)).abs() <= 8 * 2.0 ** -24 * np.log(vocab)).all()
            if gh is not None:
                assert ((gh.double() / size - dh).abs() <= rel * (g.abs() @ q["W"].abs()) + 2.0 ** -149 / size).all()
            if gw is not None:
                assert ((gw.double() / size - dW).abs() <= rel * (g.abs().t() @ q["X"].abs()) + 2.0 ** -149 / size).all()


@gpu
def test_f16_products_over_a_million_rows(cuda_ctx, eng):
    """dW sums one product for each row.  All terms of a column are positive here, so what a sum in the tensor
    cores loses, which cuts low bits off with each group of 16 products, would add up: 65536 groups, 2^-23
    of the sum each at most, is 0.8%.  Rounding g to f16 gives 2^-11, logits a relative error of 72 x 2^-24 x
    sum |h W| < 2^-14 in p; the sums themselves are taken over 2048 rows (128 groups) and then in f32."""
    t, h, v = 1 << 20, 8, 256
    g = torch.Generator(device="cuda").manual_seed(77)
    x = (torch.rand((t, h), generator=g, device="cuda") + 0.5).to(F16)
    w = (torch.randn((v, h), generator=g, device="cuda") * 0.1).to(F16)
    y = torch.full((t,), 3, device="cuda")
    a = torch.rand(t, generator=g, device="cuda") / t
    dW = torch.zeros((v, h), dtype=torch.float64, device="cuda")
    for s in range(0, t, 1 << 17):
        X, A = x[s:s + (1 << 17)].double(), a[s:s + (1 << 17)].double()
        p = torch.softmax(X @ w.double().t(), dim=1)
        p[:, 3] -= 1
        dW += (p * A[:, None]).t() @ X
    got = _call(cuda_ctx, eng, "F16", x, w, y, a, 1.0, True, (F32, F32))
    rel = 2.0 ** -11 + 2.0 ** -14 + 128 * 2.0 ** -23 + (t / 2048 + 64) * 2.0 ** -24
    assert ((got[2].double() - dW).abs() <= rel * dW.abs()).all()


@gpu
@pytest.mark.parametrize("mode", MODES)
def test_losses_without_row_weights(cuda_ctx, eng, mode):
    """No gradient asked for: the rows' weights may be left out, and change nothing."""
    for t in (1, 16, 100, 300):
        x, w, y, a = _make(t, 64, 900, (F16, F16), True, "half", 9)
        with_weights = _call(cuda_ctx, eng, mode, x, w, y, a, 1.0, True, want="none")[0]
        from ferrotensor_b200.engine import GemmMode
        cuda_ctx.set_gemm_mode(GemmMode[mode])
        loss = torch.full((t,), 9.0, device="cuda")
        try:
            eng.linear_cross_entropy_bt(cuda_ctx, _ut(x), _ut(w), _ut(_targets(y)), None, _ut(loss))
            cuda_ctx.synchronize()
        finally:
            cuda_ctx.set_gemm_mode(GemmMode.F32)
        assert torch.equal(loss, with_weights)


@gpu
@pytest.mark.parametrize("types,gtypes", [((F32, F32), (F32, F32)), ((F16, F16), (F16, F16)), ((F32, F16), (F32, F16))])
@pytest.mark.parametrize("vocab_major", [False, True])
@pytest.mark.parametrize("rows,hidden,mask", [(700, 320, "half"), (257, 896, "none"), (900, 264, "prompts"), (513, 576, "last")])
def test_gradient_made_in_place_over_several_row_tiles(cuda_ctx, eng, types, gtypes, vocab_major, rows, hidden, mask):
    """The split mode with more than one tile of rows, some of them empty behind the last supervised row."""
    s = 512.0 if F16 in gtypes else 1.0
    x, w, y, a = _make(rows, hidden, 2100, types, vocab_major, mask, 900 + rows)
    x[y == SKIP] = float("nan")
    q = _truth(x, w, y, a, s, vocab_major)
    got = _call(cuda_ctx, eng, "F16X2", x, w, y, a, s, vocab_major, gtypes)
    _check(got, q, _bounds(q, "F16X2", types, gtypes), vocab_major)


@gpu
@pytest.mark.parametrize("offset", [200.0, 1000.0])
@pytest.mark.parametrize("mode", ["F16", "F16X2"])
@pytest.mark.parametrize("size", [(75, 100, 395, 0), (184, 492, 337, 0), (179, 144, 920, 0), (721, 752, 408, 0), (304, 60, 664, 300), (1100, 144, 920, 0)])
def test_sure_rows_beside_large_weights(cuda_ctx, eng, mode, offset, size):
    """A coordinate in which every weight is 32, the others near 0.1: dh there is a sum that comes to almost
    nothing, of which the target's own share must not be in two parts."""
    _sure_case(cuda_ctx, eng, mode, offset, size, ("hidden", "both"))
