"""Workloads of the operators at the end of a training step: the linear cross entropy (output projection and
masked softmax loss in one, with its gradients, no logits kept) and the global gradient norm with clipping over
a list of tensors.  `own` chooses between the elementary torch form and the engine's calls."""

import math

import numpy as np
import torch

own = False

SKIP = 0xFFFFFFFF

# Operand types of the linear cross entropy: (hidden and its gradient, weight, the weight's gradient).
TYPES = {
    "f16": (torch.float16, torch.float16, torch.float16),     # all in storage precision
    "mixed": (torch.float32, torch.float16, torch.float32),   # f32 activations, f16 head: the engine's usual pair
    "f32": (torch.float32, torch.float32, torch.float32),     # a head that is trained in f32
}


def listed():
    return [
        # scoring one token against a tied [vocab, hidden] head: the smallest call
        dict(name="score_one", op="loss", rows=1, hidden=576, vocab=49152, vocab_major=True, types="f16", grads="none", skipped=0.0),
        # the log-likelihood of a short answer, a vocabulary of 152 thousand
        dict(name="score_answer", op="loss", rows=77, hidden=896, vocab=151936, vocab_major=True, types="f16", grads="none", skipped=0.0),
        # a held-out batch with its prompts masked: forward only, f32 activations
        dict(name="held_out", op="loss", rows=4096, hidden=960, vocab=49152, vocab_major=False, types="mixed", grads="none", skipped=0.25),
        # adapter training: a frozen head, the gradient goes to the hidden rows (8 x 1024 tokens)
        dict(name="frozen_head", op="loss", rows=8192, hidden=2048, vocab=49152, vocab_major=False, types="f16", grads="hidden", skipped=0.0),
        # the same for f32 activations and an f32 gradient, fewer rows
        dict(name="frozen_head_f32", op="loss", rows=2048, hidden=2048, vocab=49152, vocab_major=False, types="mixed", grads="hidden", skipped=0.0),
        # a trained tied head, half of the tokens are prompt
        dict(name="trained_head", op="loss", rows=4096, hidden=896, vocab=151936, vocab_major=True, types="f16", grads="both", skipped=0.5),
        # a trained head all in f32
        dict(name="trained_head_f32", op="loss", rows=512, hidden=576, vocab=49152, vocab_major=True, types="f32", grads="both", skipped=0.0),
        # nothing a multiple of anything: an extended vocabulary, a ragged batch
        dict(name="odd_sizes", op="loss", rows=1531, hidden=575, vocab=50021, vocab_major=False, types="f16", grads="both", skipped=0.2),
        # the adapters of the smallest workload: launch latency
        dict(name="clip_tiny", op="clip", layers=2, hidden=32, ffn=64, rank=4, full=False, src="f32", dst="f32", odd=False, above=True),
        # rank-16 adapters of 24 blocks, clipped into the optimizer's buffers
        dict(name="clip_adapters", op="clip", layers=24, hidden=2048, ffn=8192, rank=16, full=False, src="f32", dst="f32", odd=False, above=True),
        # whole weights of 32 blocks: loss-scaled f16 gradients, unscaled and clipped into f32
        dict(name="clip_full", op="clip", layers=32, hidden=960, ffn=2560, rank=0, full=True, src="f16", dst="f32", odd=False, above=True),
        # the norm alone of gradients of both types and odd lengths
        dict(name="norm_odd", op="clip", layers=30, hidden=576, ffn=1536, rank=0, full=True, src="both", dst="none", odd=True, above=False),
    ]


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    if rng.random() < 0.7:
        while True:
            c = dict(op="loss", rows=_log_uniform(rng, 1, 8192), hidden=_log_uniform(rng, 64, 2048), vocab=_log_uniform(rng, 500, 152000),
                     vocab_major=rng.random() < 0.5, types=rng.choice(("f16", "f16", "mixed", "f32")), grads=rng.choice(("none", "hidden", "both")),
                     skipped=rng.choice((0.0, 0.1, 0.5, 0.9)))
            if rng.random() < 0.5:   # most real sizes are round, the others are not
                c["hidden"] = max(64, c["hidden"] // 64 * 64)
                c["vocab"] = max(512, c["vocab"] // 64 * 64)
            cost = c["rows"] * c["hidden"] * c["vocab"] * {"none": 1, "hidden": 2, "both": 3}[c["grads"]] * (1 if c["types"] == "f16" else 2)
            if cost <= 0.5 * 2 * 8192 * 2048 * 49152 and c["hidden"] * c["vocab"] <= 1.4e8:
                return c
    full = rng.random() < 0.4
    return dict(op="clip", layers=_log_uniform(rng, 1, 16 if full else 48), hidden=_log_uniform(rng, 32, 1024 if full else 4096), ffn=_log_uniform(rng, 64, 2048 if full else 8192),
                rank=0 if full else rng.choice((4, 8, 16, 32)), full=full, src=rng.choice(("f32", "f16", "both")), dst=rng.choice(("f32", "same", "none")),
                odd=rng.random() < 0.5, above=rng.random() < 0.7)


# ---- inputs -----------------------------------------------------------------------------------------------

def _supervised(case):
    return max(1, round(case["rows"] * (1.0 - case["skipped"])))


def _lengths(case):
    """Element counts of the gradient tensors: A and B of every adapter, or the seven linears and two norms of a block."""
    h, f, r = case["hidden"], case["ffn"], case["rank"]
    if case["full"]:
        block = [h * h] * 4 + [h * f] * 3 + [h, h]
    else:
        block = [h * r, r * h] * 4 + [h * r, r * f] * 2 + [f * r, r * h]
    counts = block * case["layers"]
    return [n + (i % 7 if case["odd"] else 0) for i, n in enumerate(counts)]


def _kinds(case, which):
    n = len(_lengths(case))
    kind = case["src"] if which == "src" or case["dst"] == "same" else case["dst"]
    if kind == "both":
        return [torch.float16 if i % 2 else torch.float32 for i in range(n)]
    return [torch.float16 if kind == "f16" else torch.float32] * n


def _views(flat, starts, counts, kinds):
    return [flat[s:s + n * k.itemsize].view(k) for s, n, k in zip(starts, counts, kinds)]


def _buffers(counts, kinds, odd):
    """One byte buffer with room for every tensor; odd: each begins at a multiple of its own element size only."""
    starts, at = [], 0
    for i, (n, k) in enumerate(zip(counts, kinds)):
        at = -(-at // 16) * 16 + (k.itemsize * (i % 5) if odd else 0)
        starts.append(at)
        at += n * k.itemsize
    return torch.zeros(-(-at // 16) * 16, dtype=torch.uint8, device="cuda"), starts


def prepare(case, seed):
    state = _inputs(case, seed)
    if own:
        state["call"] = _handles_loss(state) if case["op"] == "loss" else _handles_clip(state)
    return state


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return _inputs_loss(case, g) if case["op"] == "loss" else _inputs_clip(case, g)


def _inputs_loss(case, g):
    t, h, v = case["rows"], case["hidden"], case["vocab"]
    hk, wk, gk = TYPES[case["types"]]
    weight = (torch.randn((v, h) if case["vocab_major"] else (h, v), generator=g, device="cuda") * 0.02).to(wk)
    targets = torch.randint(0, v, (t,), generator=g, device="cuda")
    # normalised hidden rows that lean towards their target: by 0 to 12 in its logit
    rows = weight[targets] if case["vocab_major"] else weight.t()[targets]
    lean = torch.rand((t, 1), generator=g, device="cuda") * (12.0 / (0.02 ** 2 * h))
    hidden = (torch.randn((t, h), generator=g, device="cuda") + lean * rows.float()).to(hk)
    # prompt and padding tokens are skipped; a token weighs 1 / the tokens of its sequence
    skip = torch.randperm(t, generator=g, device="cuda")[:t - _supervised(case)]
    targets[skip] = -1
    weights = (0.5 + torch.rand(t, generator=g, device="cuda")) / t
    state = dict(case=case, hidden=hidden, weight=weight, targets=targets.to(torch.int32), weights=weights,
                 loss=torch.empty(t, device="cuda"), scale=65536.0 if gk is torch.float16 else 1.0)
    if case["grads"] != "none":
        state["grad_hidden"] = torch.empty_like(hidden)
    if case["grads"] == "both":
        state["grad_weight"] = torch.empty(weight.shape, dtype=gk, device="cuda")
    return state


def _inputs_clip(case, g):
    counts, kinds = _lengths(case), _kinds(case, "src")
    flat, starts = _buffers(counts, kinds, case["odd"])
    grads = _views(flat, starts, counts, kinds)
    loss_scale = 1024.0 if case["src"] != "f32" else 1.0
    kept = 1.0 if case["dst"] == "same" else loss_scale     # f16 results keep the loss scale, f32 ones are unscaled
    for i, x in enumerate(grads):
        x.copy_(torch.randn(x.shape, generator=g, device="cuda") * (1e-4 * (1 + i % 9) * loss_scale))
    rms = math.sqrt(sum(n * (1e-4 * (1 + i % 9)) ** 2 for i, n in enumerate(counts)))
    state = dict(case=case, grads=grads, scale=1.0 / kept, norm=torch.zeros(4, device="cuda"),
                 max_norm=rms * loss_scale / kept * (0.37 if case["above"] else 2.0))
    if case["dst"] != "none":
        to = _kinds(case, "dst")
        state["flat"], starts = _buffers(counts, to, case["odd"])
        state["out"] = _views(state["flat"], starts, counts, to)
    return state


# ---- one pass ---------------------------------------------------------------------------------------------

def run(state):
    if own:
        state["call"]()
        if state["case"]["op"] == "loss":
            return [state[k] for k in ("loss", "grad_hidden", "grad_weight") if k in state]
        return [state["norm"][:3]] + (_clipped(state) if "out" in state else [])
    return _plain_loss(state) if state["case"]["op"] == "loss" else _plain_clip(state)


def _clipped(state):
    """The clipped gradients whole: the buffer that they lie in where all are f32, else one tensor for each type."""
    if all(x.dtype is torch.float32 for x in state["out"]):
        return [state["flat"].view(torch.float32)]
    return [torch.cat([x for x in state["out"] if x.dtype is k]) for k in (torch.float32, torch.float16) if any(x.dtype is k for x in state["out"])]


def _plain_loss(s):
    case = s["case"]
    h, w = s["hidden"].float(), s["weight"].float()
    if case["vocab_major"]:
        w = w.t()
    live = s["targets"] >= 0
    target = torch.where(live, s["targets"], 0).long()
    z = h @ w
    top = z.amax(dim=1, keepdim=True)
    lse = (z - top).exp().sum(dim=1, keepdim=True).log() + top
    picked = z.gather(1, target[:, None])
    loss = torch.where(live, (lse - picked)[:, 0], 0.0)
    out = [loss]
    if case["grads"] != "none":
        scale = torch.where(live, s["weights"] * s["scale"], 0.0)[:, None]
        grad = (z - lse).exp() * scale
        grad.scatter_add_(1, target[:, None], -scale)
        out.append((grad @ w.t()).to(s["hidden"].dtype))
        if case["grads"] == "both":
            grad_w = grad.t() @ h if case["vocab_major"] else h.t() @ grad
            out.append(grad_w.to(s["grad_weight"].dtype))
    return out


def _plain_clip(s):
    total = torch.stack([g.double().square().sum() for g in s["grads"]]).sum()
    norm = total.sqrt() * abs(s["scale"])
    finite = torch.isfinite(norm)
    above = norm > s["max_norm"] if "out" in s else torch.zeros_like(finite)
    factor = torch.where(finite & above, s["scale"] * s["max_norm"] / (norm + 1e-6), s["scale"])
    out = [torch.stack([norm, finite.double(), factor]).float()]
    if "out" in s:
        f = factor.float()
        [o.copy_(torch.where(finite, g.float() * f, o)) for g, o in zip(s["grads"], s["out"])]
        out += _clipped(s)
    return out


# ---- the engine's calls -----------------------------------------------------------------------------------

_engine = []


def _open():
    from ferrotensor_b200.engine import ComputeEngine, CudaContext
    if not _engine:
        ctx = CudaContext(torch.cuda.current_device())
        _engine.extend((ctx, ComputeEngine(ctx)))
    return _engine


def _tensor(x):
    from ferrotensor_b200.engine import DType, UnifiedTensor
    kind = {torch.float32: DType.F32, torch.float16: DType.FP16, torch.int32: DType.U32}[x.dtype]
    return UnifiedTensor(x.view(-1).view(torch.uint8), list(x.shape), kind)


def _handles_loss(s):
    from ferrotensor_b200.engine import GemmMode
    ctx, eng = _open()
    case = s["case"]
    mode = GemmMode.F16 if case["types"] == "f16" else GemmMode.F16X2
    method = eng.linear_cross_entropy_bt if case["vocab_major"] else eng.linear_cross_entropy
    h, w, y, a, loss = (_tensor(s[k]) for k in ("hidden", "weight", "targets", "weights", "loss"))
    gh, gw = (_tensor(s[k]) if k in s else None for k in ("grad_hidden", "grad_weight"))

    def call():
        ctx.set_gemm_mode(mode)
        method(ctx, h, w, y, a, loss, grad_hidden=gh, grad_weight=gw, grad_scale=s["scale"])

    return call


def _handles_clip(s):
    from ferrotensor_b200.engine import GradientList
    ctx, eng = _open()
    norm = _tensor(s["norm"])
    grads = GradientList(ctx, [_tensor(x) for x in s["grads"]])
    if "out" not in s:
        return lambda: eng.global_grad_norm(ctx, grads, norm, grad_scale=s["scale"])
    out = GradientList(ctx, [_tensor(x) for x in s["out"]])
    return lambda: eng.clip_grad_global_norm(ctx, grads, s["max_norm"], norm, grad_scale=s["scale"], out=out)


# ---- what a pass cannot do without, and what it gives -------------------------------------------------------

def work(case):
    if case["op"] == "loss":
        t, h, v = _supervised(case), case["hidden"], case["vocab"]
        hk, wk, gk = TYPES[case["types"]]
        gemms = {"none": 1, "hidden": 2, "both": 3}[case["grads"]]
        moved = t * h * hk.itemsize + h * v * wk.itemsize + case["rows"] * 8
        if case["grads"] != "none":
            moved += case["rows"] * (h * hk.itemsize + 4)
        if case["grads"] == "both":
            moved += h * v * gk.itemsize
        return {"bytes": moved, "flops": 2.0 * gemms * t * h * v}
    counts = _lengths(case)
    moved = sum(n * k.itemsize for n, k in zip(counts, _kinds(case, "src")))
    if case["dst"] != "none":
        moved += sum(n * k.itemsize for n, k in zip(counts, _kinds(case, "dst")))
    return {"bytes": moved + 12, "flops": (2.0 if case["dst"] == "none" else 3.0) * sum(counts)}


def exact(case, seed):
    """The same in 64 bits from the definition: the vocabulary in blocks, rows one group at a time."""
    s = _inputs(case, seed)
    if case["op"] == "clip":
        norm = math.sqrt(float(sum(float(torch.dot(x, x)) for x in (g.double() for g in s["grads"])))) * s["scale"]
        factor = s["scale"]
        if "out" in s and norm > s["max_norm"]:
            factor *= s["max_norm"] / (norm + 1e-6)
        out = [np.array([norm, 1.0, factor])]
        if "out" in s:
            if all(x.dtype is torch.float32 for x in s["out"]):
                whole = torch.zeros(s["flat"].numel() // 4, dtype=torch.float64, device="cuda")
                for g, o in zip(s["grads"], s["out"]):
                    at = (o.data_ptr() - s["flat"].data_ptr()) // 4
                    whole[at:at + g.numel()] = g.double() * factor
                out.append(whole)
            else:
                pairs = list(zip(s["grads"], s["out"]))
                out += [torch.cat([g.double() * factor for g, o in pairs if o.dtype is k]) for k in (torch.float32, torch.float16) if any(o.dtype is k for _, o in pairs)]
        return out
    t, v = case["rows"], case["vocab"]
    w = s["weight"] if case["vocab_major"] else s["weight"].t()     # [vocab, hidden]
    loss = torch.zeros(t, dtype=torch.float64, device="cuda")
    dh = torch.zeros(s["hidden"].shape, dtype=torch.float64, device="cuda")
    dw = torch.zeros(w.shape if case["grads"] == "both" else (0, 0), dtype=torch.float64, device="cuda")
    rows = torch.nonzero(s["targets"] != -1)[:, 0]
    for part in rows.split(2048):
        h, y = s["hidden"][part].double(), s["targets"][part].long()
        blocks = [slice(a, min(a + 16384, v)) for a in range(0, v, 16384)]
        parts = [torch.logsumexp(h @ w[b].double().t(), dim=1) for b in blocks]
        lse = torch.logsumexp(torch.stack(parts), dim=0)
        loss[part] = lse - (h * w[y].double()).sum(dim=1)
        if case["grads"] == "none":
            continue
        a = s["weights"][part].double() * s["scale"]
        dh_part = -a[:, None] * w[y].double()
        for b in blocks:
            wb = w[b].double()
            p = torch.exp(h @ wb.t() - lse[:, None]) * a[:, None]
            dh_part += p @ wb
            if case["grads"] == "both":
                dw[b] += p.t() @ h
        dh[part] = dh_part
        if case["grads"] == "both":
            dw.index_add_(0, y, -a[:, None] * h)
    out = [loss]
    if case["grads"] != "none":
        out.append(dh)
    if case["grads"] == "both":
        out.append(dw if case["vocab_major"] else dw.t().contiguous())
    return out
