"""The gated linear recurrence, its gradient and its single step against the definition in 64 bits, and a training
step of a recurrent token model that runs it together with the operators on logits. Tolerances: ``room``."""
import math

import numpy as np
import pytest
import torch

import parpy_b200 as parpy
from parpy_b200 import kernels, ops
from parpy_b200.buffer import CudaBuffer

gpu = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
H = 2.0 ** -24
TILE = kernels.SCAN_TILE


def opts():
    return parpy.par({})


def define(g, x, h0, lens, dh=None, dlast=None):
    """States and gradients step by step in 64 bits, with the largest sums of absolute values on the way."""
    g, x = g.double().cpu(), x.double().cpu()
    b, t, d = g.shape
    lens = torch.full((b,), t) if lens is None else lens.cpu().clamp(0, t)
    state = torch.zeros(b, d, dtype=torch.float64) if h0 is None else h0.double().cpu()
    size = state.abs()
    f, keep = torch.sigmoid(g), torch.sigmoid(-g)
    out = {"h": torch.zeros_like(g), "size": torch.zeros_like(g)}
    before = torch.zeros_like(g)
    for i in range(t):
        live = (lens > i)[:, None]
        before[:, i] = state
        state = torch.where(live, f[:, i] * state + keep[:, i] * x[:, i], state)
        size = torch.where(live, f[:, i] * size + keep[:, i] * x[:, i].abs(), size)
        out["h"][:, i] = torch.where(live, state, out["h"][:, i])
        out["size"][:, i] = size
    out["last"], out["last_size"] = state, size
    if dh is None and dlast is None:
        return out
    dh = torch.zeros_like(g) if dh is None else dh.double().cpu()
    c = torch.zeros(b, d, dtype=torch.float64) if dlast is None else dlast.double().cpu()
    cs = c.abs()
    for name in ("dg", "dx", "r_size"):
        out[name] = torch.zeros_like(g)
    for i in range(t - 1, -1, -1):
        live = (lens > i)[:, None]
        r, rs = dh[:, i] + c, dh[:, i].abs() + cs
        out["dx"][:, i] = torch.where(live, keep[:, i] * r, out["dx"][:, i])
        out["dg"][:, i] = torch.where(live, r * (before[:, i] - x[:, i]) * f[:, i] * keep[:, i], out["dg"][:, i])
        out["r_size"][:, i] = torch.where(live, rs, out["r_size"][:, i])
        c, cs = torch.where(live, f[:, i] * r, c), torch.where(live, f[:, i] * rs, cs)
    out["dh0"], out["dh0_size"] = c, cs
    out["f"], out["keep"], out["x"] = f, keep, x
    return out


def room(g, t):
    """Relative to the sum of absolute values: a gate carries its exponent's rounding (|g| log2(e) 2^-24 twice), exp2's
    2^-22 (weighted by 1 - f in f, whole in 1 - f) and the reciprocal's and products' few steps; a term of the sum has
    passed at most min(t, 1 / (1 - f)) gates that matter, and as many additions and products."""
    fast = float(torch.sigmoid(-g.double().cpu()).mean())
    passed = min(t, 4.0 / max(fast, 1e-6)) + 24
    gate = float(g.double().abs().max()) * 1.5 * 2 * H
    return 2.0 ** -22 + (gate + 2.0 ** -22) * (1 + fast * passed) + 4 * H * passed


def close(got, want, tol):
    got, want = got.double().cpu(), want.double().cpu()
    assert torch.isfinite(got).all()
    over = (got - want).abs() - torch.broadcast_to(torch.as_tensor(tol, dtype=torch.float64), want.shape)
    assert not over.numel() or float(over.max()) <= 0, f"off by {float(over.max()):.3g} more than allowed"


def rounding(dtype, want):
    f = torch.finfo(dtype)
    return want.abs() * f.eps / 2 + f.tiny * f.eps / 2 + 2.0 ** -120


def inputs(b, t, d, dtype, seed, shift=2.0):
    gen = torch.Generator().manual_seed(seed)

    def normal(*s):
        return torch.randn(*s, generator=gen)
    return {"g": (normal(b, t, d) * 1.5 + shift).to(dtype).cuda(), "x": normal(b, t, d).to(dtype).cuda(),
            "h0": normal(b, d).cuda(), "dh": normal(b, t, d).to(dtype).cuda(), "dlast": normal(b, d).cuda()}


def run(s, lens, h0=True, dh=True, dlast=True):
    b, t, d = s["g"].shape
    dev = dict(device="cuda")
    out = {"h": torch.full_like(s["g"], 7.0), "last": torch.full((b, d), 7.0, **dev),
           "carry": torch.full((b, -(-t // TILE), d), math.nan, **dev), "dg": torch.full_like(s["g"], 7.0),
           "dx": torch.full_like(s["g"], 7.0), "dh0": torch.full((b, d), 7.0, **dev)}
    kernels.gated_scan(s["g"], s["x"], s["h0"] if h0 else None, lens, b, t, d, out["h"], out["last"], out["carry"],
                       opts=opts())
    kernels.gated_scan_grad(s["g"], s["x"], lens, b, t, d, out["carry"], s["dh"] if dh else None,
                            s["dlast"] if dlast else None, out["dg"], out["dx"], out["dh0"], opts=opts())
    return out


def check(s, lens, out, h0=True, dh=True, dlast=True):
    t, dtype = s["g"].shape[1], s["g"].dtype
    d = define(s["g"], s["x"], s["h0"] if h0 else None, lens, s["dh"] if dh else torch.zeros_like(s["dh"]),
               s["dlast"] if dlast else None)
    r = room(s["g"], t)
    close(out["h"], d["h"], rounding(dtype, d["h"]) + r * d["size"])
    close(out["last"], d["last"], r * d["last_size"] + 2.0 ** -120)
    close(out["dx"], d["dx"], rounding(dtype, d["dx"]) + 2 * r * d["keep"] * d["r_size"])
    both = d["r_size"] * (d["size"] + d["x"].abs() + (s["h0"].abs().cpu().double()[:, None] if h0 else 0)) * d["keep"]
    close(out["dg"], d["dg"], rounding(dtype, d["dg"]) + 3 * r * both)
    close(out["dh0"], d["dh0"], 2 * r * d["dh0_size"] + 2.0 ** -120)
    return d


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("b,t,d", [(1, 1, 1), (2, 3, 5), (1, 127, 64), (3, 128, 66), (2, 129, 33), (1, 1000, 2),
                                   (5, 300, 515), (1, 3000, 130), (40, 140, 256), (2, 1025, 64), (300, 17, 100)])
def test_scan_and_gradient(b, t, d, dtype):
    s = inputs(b, t, d, dtype, 100 * b + t + d)
    check(s, None, run(s, None))
    gen = torch.Generator().manual_seed(t)
    lens = torch.randint(0, t + 1, (b,), generator=gen)
    lens[0] = 0
    lens[-1] = t - 1
    lens = lens.cuda()
    out = run(s, lens)
    check(s, lens, out)
    for i, n in enumerate(lens.tolist()):
        for name in ("h", "dg", "dx"):
            assert not out[name][i, n:].any()
    out = run(s, lens.int(), h0=False, dlast=False)
    check(s, lens, out, h0=False, dlast=False)
    out = run(s, lens, dh=False)
    check(s, lens, out, dh=False)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_long_memory_and_closed_gates(dtype):
    b, t, d = 2, 5000, 70
    s = inputs(b, t, d, dtype, 1)
    s["g"][:, :, ::3] = 12.0           # hardly forgets: 1 - f = 6e-6
    s["g"][:, :, 1::3] = -100.0        # f = 0: h = x
    s["g"][0, 100:140] = math.inf      # f = 1: the state passes
    s["g"][1, 50:60] = -math.inf
    finite = {**s, "g": s["g"].clamp(-100, 100)}
    out = run(s, None)
    want = define(s["g"], s["x"], s["h0"], None, s["dh"], s["dlast"])
    r = 2.0 ** -21 + 4 * H * 5000 + 200 * 3 * H            # every gate passed counts
    close(out["h"], want["h"], rounding(dtype, want["h"]) + r * want["size"])
    close(out["last"], want["last"], r * want["last_size"] + 2.0 ** -100)
    close(out["dx"], want["dx"], rounding(dtype, want["dx"]) + 2 * r * want["r_size"] * want["keep"] + 2.0 ** -100)
    # gates below -41.5 count as -41.5: there 0 < f - sigmoid(g) < exp(-41.5) < 2^-59, and dh0 = f r takes it times r
    close(out["dh0"], want["dh0"], 2 * r * want["dh0_size"] + 2.0 ** -100 + 2.0 ** -59 * want["r_size"][:, 0])
    assert torch.isfinite(out["dg"].float()).all() and torch.isfinite(run(finite, None)["dg"].float()).all()


@gpu
def test_padding_is_not_read_and_bad_lengths_are_clamped():
    b, t, d = 4, 200, 64
    s = inputs(b, t, d, BF16, 2)
    lens = torch.tensor([0, 1, 130, 200]).cuda()
    clean = run(s, lens)
    for i, n in enumerate(lens.tolist()):
        for name in ("g", "x", "dh"):
            s[name][i, n:] = math.nan
    dirty = run(s, lens)
    for name in ("h", "last", "dg", "dx", "dh0"):
        assert torch.equal(clean[name], dirty[name])
    s = inputs(b, t, d, BF16, 2)
    far = run(s, torch.tensor([-5, 1, 130, 1 << 40]).cuda())
    for name in ("h", "last", "dg", "dx", "dh0"):
        assert torch.equal(clean[name], far[name])
    nothing = run({k: v[:, :0] if v.dim() == 3 else v for k, v in s.items()}, None)
    assert torch.equal(nothing["last"], s["h0"]) and torch.equal(nothing["dh0"], s["dlast"])


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strided_arrays(dtype):
    # gate and input as halves of one projection, time before batch, an odd offset
    b, t, d = 3, 150, 40
    s = inputs(b, t, d, dtype, 3)
    plain = run(s, None)
    for pad in (0, 1):
        both = torch.empty(t, b, 2 * d + pad, dtype=dtype, device="cuda")
        v = {**s, "g": both[:, :, :d].transpose(0, 1), "x": both[:, :, d + pad:].transpose(0, 1)}
        v["g"].copy_(s["g"])
        v["x"].copy_(s["x"])
        grads = torch.full((b, t, 2 * d + 3), 7.0, dtype=dtype, device="cuda")
        hs = torch.full((t, b, d + pad), 7.0, dtype=dtype, device="cuda")
        last = torch.empty_like(plain["last"])
        carry, dh0 = torch.empty_like(plain["carry"]), torch.empty_like(plain["dh0"])
        h = hs[:, :, pad:].transpose(0, 1)
        dg, dx = grads[:, :, :d], grads[:, :, d + 1:2 * d + 1]
        kernels.gated_scan(v["g"], v["x"], s["h0"], None, b, t, d, h, last, carry, opts=opts())
        kernels.gated_scan_grad(v["g"], v["x"], None, b, t, d, carry, s["dh"], s["dlast"], dg, dx, dh0, opts=opts())
        assert torch.equal(h, plain["h"]) and torch.equal(last, plain["last"])
        assert torch.equal(dg, plain["dg"]) and torch.equal(dx, plain["dx"]) and torch.equal(dh0, plain["dh0"])
        assert bool((grads[:, :, d] == 7).all()) and bool((grads[:, :, 2 * d + 1:] == 7).all())
    with pytest.raises(ValueError, match="overlap"):
        kernels.gated_scan(s["g"], s["x"], None, None, b, t, d, s["g"][:, :1].expand(b, t, d), None, None, opts=opts())
    with pytest.raises(ValueError, match="contiguous"):
        kernels.gated_scan(s["g"].transpose(1, 2), s["x"].transpose(1, 2), None, None, b, d, t,
                           torch.empty(b, d, t, dtype=dtype, device="cuda"), None, None, opts=opts())


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("n,d", [(1, 1), (3, 7), (8, 1024), (5, 515), (2000, 264)])
def test_step_is_one_step_of_the_scan(n, d, dtype):
    s = inputs(n, 1, d, dtype, n + d)
    h, last = torch.empty_like(s["g"][:, 0]), torch.empty(n, d, device="cuda")
    kernels.gated_step(s["g"][:, 0], s["x"][:, 0], s["h0"], n, d, h, last, opts=opts())
    want = define(s["g"], s["x"], s["h0"], None)
    r = room(s["g"], 1)
    close(last, want["last"], r * want["last_size"])
    close(h, want["h"][:, 0], rounding(dtype, want["h"][:, 0]) + r * want["size"][:, 0])
    out = run(s, None)
    assert torch.equal(out["last"], last) and torch.equal(out["h"][:, 0], h)
    state = s["h0"].clone()
    wide = torch.full((n, d + 9), 7.0, dtype=dtype, device="cuda")
    kernels.gated_step(s["g"][:, 0], s["x"][:, 0], state, n, d, wide[:, 3:3 + d], state, opts=opts())     # in place
    assert torch.equal(state, last) and torch.equal(wide[:, 3:3 + d], h)
    assert bool((wide[:, :3] == 7).all()) and bool((wide[:, 3 + d:] == 7).all())


@gpu
def test_prefill_then_steps_equal_one_scan():
    b, t, d = 3, 140, 96
    s = inputs(b, t, d, F32, 9)
    whole = run(s, None)
    cut = 131
    h, last = torch.empty(b, cut, d, device="cuda"), torch.empty(b, d, device="cuda")
    kernels.gated_scan(s["g"][:, :cut], s["x"][:, :cut], s["h0"], None, b, cut, d, h, last, None, opts=opts())
    one = torch.empty(b, d, device="cuda")
    for i in range(cut, t):
        kernels.gated_step(s["g"][:, i], s["x"][:, i], last, b, d, one, last, opts=opts())
        # the scan composes its runs in another order: a few roundings of the sums' size
        close(one, whole["h"][:, i].double(), 64 * H * 8)


@gpu
def test_finite_differences():
    b, t, d = 1, 140, 3
    s = inputs(b, t, d, F32, 4)
    out = run(s, None)

    def value(v):
        o = define(v["g"], v["x"], v["h0"], None)
        return float((o["h"] * v["dh"].double().cpu()).sum() + (o["last"] * v["dlast"].double().cpu()).sum())
    step = 2.0 ** -10
    for name, grad in (("g", "dg"), ("x", "dx"), ("h0", "dh0")):
        flat = out[grad].double().reshape(-1)
        for at in (0, 7, flat.numel() // 2, flat.numel() - 1):
            at = min(at, flat.numel() - 1)
            ends = []
            for sign in (1, -1):
                v = {k: a.double().cpu().clone() for k, a in s.items()}
                v[name].reshape(-1)[at] += sign * step
                ends.append(value(v))
            # the third derivative of a sum of at most some ten terms of size 10: step^2 times 20
            assert abs((ends[0] - ends[1]) / (2 * step) - float(flat[at])) <= 2.0 ** -14 + 20 * step ** 2


@gpu
def test_streams_graphs_and_repeated_calls():
    b, t, d = 2, 3000, 192
    s = inputs(b, t, d, BF16, 5)
    lens = torch.tensor([3000, 1111]).cuda()
    first = run(s, lens)
    again = run(s, lens)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        third = run(s, lens)
    side.synchronize()
    names = ("h", "last", "dg", "dx", "dh0")
    for name in names:
        assert torch.equal(first[name], again[name]) and torch.equal(first[name], third[name])
    buf = {name: torch.zeros_like(v) for name, v in first.items()}

    def both():
        o = opts()
        kernels.gated_scan(s["g"], s["x"], s["h0"], lens, b, t, d, buf["h"], buf["last"], buf["carry"], opts=o)
        kernels.gated_scan_grad(s["g"], s["x"], lens, b, t, d, buf["carry"], s["dh"], s["dlast"], buf["dg"], buf["dx"],
                                buf["dh0"], opts=o)
    both()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        both()
    for name in names:
        buf[name].zero_()
    lens.copy_(torch.tensor([5, 3000]))
    graph.replay()
    new = run(s, lens)
    torch.cuda.synchronize()
    for name in names:
        assert torch.equal(buf[name], new[name])


@gpu
def test_host_arrays():
    b, t, d = 2, 150, 6
    s = {k: v.cpu() for k, v in inputs(b, t, d, F32, 6).items()}
    h, last = np.zeros((b, t, d), np.float32), np.zeros((b, d), np.float32)
    carry = np.zeros((b, 2, d), np.float32)
    dg, dx, dh0 = np.zeros_like(h), np.zeros_like(h), np.zeros_like(last)
    lens = np.array([150, 20])
    kernels.gated_scan(s["g"].numpy(), s["x"].numpy(), s["h0"].numpy(), lens, b, t, d, h, last, carry, opts=opts())
    kernels.gated_scan_grad(s["g"].numpy(), s["x"].numpy(), lens, b, t, d, carry, s["dh"].numpy(), s["dlast"].numpy(),
                            dg, dx, dh0, opts=opts())
    out = {k: torch.from_numpy(v) for k, v in (("h", h), ("last", last), ("dg", dg), ("dx", dx), ("dh0", dh0))}
    check(s, torch.from_numpy(lens), out)
    assert not carry[1, 1].any()        # behind the sequence's end: as it was


# ---- the operators together: a training step of a recurrent token model -----------------------------------
def test_registered_sources_are_complete():
    from parpy_b200 import source
    for name in ("gated_scan", "gated_step", "token_logprobs", "distill_topk_grad"):
        text = source.kernel_source(name)
        assert '#include "' not in text and f"parpy_b200_{name}" in text


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_training_step_of_a_recurrent_model(dtype):
    """scan -> projection -> policy and distillation losses -> gradients, against 64-bit automatic differentiation."""
    b, t, d, m, k = 3, 150, 48, 777, 16
    gen = torch.Generator().manual_seed(11)

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=gen) * scale).to(dtype).cuda()
    g, x, w = normal(b, t, d, scale=1.5), normal(b, t, d), normal(m, d, scale=0.3)
    lens = torch.tensor([150, 71, 0]).cuda()
    tokens = torch.randint(0, m, (b, t), generator=gen).cuda()
    tokens[torch.arange(t).cuda()[None] >= lens[:, None]] = -1
    advantage, bonus = torch.randn(b * t, generator=gen).cuda(), torch.full((b * t,), 0.05).cuda()
    n = b * t
    bonus[tokens.reshape(-1) < 0] = 0.0
    teach = normal(n, m, scale=2.0)
    o = opts()
    dev = dict(device="cuda")
    # teacher's alternatives, then the student's step
    lse_t, top, at = torch.empty(n, **dev), torch.empty(n, k, **dev), torch.empty(n, k, dtype=torch.int64, **dev)
    kernels.token_logprobs(teach, None, n, m, k, 1.0, None, lse_t, None, top, at, opts=o)
    at[tokens.reshape(-1) < 0] = -1
    h, carry = torch.empty_like(x), torch.empty(b, 2, d, **dev)
    kernels.gated_scan(g, x, None, lens, b, t, d, h, None, carry, opts=o)
    z = h.reshape(n, d) @ w.t()
    logp, lse, ent = (torch.empty(n, **dev) for _ in range(3))
    loss, lse2, rest = (torch.empty(n, **dev) for _ in range(3))
    kernels.token_logprobs(z, tokens.reshape(-1), n, m, 0, 1.0, logp, lse, ent, None, None, opts=o)
    kernels.distill_topk(z, at, top, n, m, k, 1.0, True, loss, lse2, rest, opts=o)
    dz1, dz2 = torch.empty_like(z), torch.empty_like(z)
    kernels.token_logprobs_grad(z, tokens.reshape(-1), n, m, 1.0, lse, ent, advantage, bonus, dz1, opts=o)
    one = torch.ones(n, **dev)
    kernels.distill_topk_grad(z, at, top, n, m, k, 1.0, True, lse2, rest, one, dz2, opts=o)
    dz = dz1 + dz2
    dw, dh = dz.t() @ h.reshape(n, d), (dz @ w).reshape(b, t, d)
    dg, dx = torch.empty_like(g), torch.empty_like(x)
    kernels.gated_scan_grad(g, x, lens, b, t, d, carry, dh, None, dg, dx, None, opts=o)

    G, X, Wt = (v.double().requires_grad_() for v in (g, x, w))
    state, hs = torch.zeros(b, d, dtype=torch.float64, **dev), []
    f = torch.sigmoid(G)
    for i in range(t):
        live = (lens > i)[:, None]
        new = f[:, i] * state + (1 - f[:, i]) * X[:, i]
        hs.append(torch.where(live, new, torch.zeros_like(new)))
        state = torch.where(live, new, state)
    logits = torch.stack(hs, 1).reshape(n, d) @ Wt.t()
    ls = torch.log_softmax(logits, 1)
    given = (tokens.reshape(-1) >= 0).double()
    lp = ls[torch.arange(n), tokens.reshape(-1).clamp(min=0)] * given
    entropy = -(ls.exp() * ls).sum(1)
    col = at.clamp(min=0)
    q = top.double().exp() * given[:, None]
    sp = ls.gather(1, col)
    inside = torch.zeros(n, m, dtype=torch.bool, **dev).scatter_(1, col, True)
    restlog = torch.logsumexp(ls.masked_fill(inside, -math.inf), 1)
    left = 1 - q.sum(1)
    kl = (torch.xlogy(q, q) - q * sp).sum(1) + (torch.xlogy(left, left) - left * restlog) * given
    total = (lp * advantage.double()).sum() + (entropy * bonus.double()).sum() + kl.sum()
    total.backward()
    # h, z, dz, dh pass through the type once each (half a step, relative to the gradients' norm), products over d and m
    step = torch.finfo(dtype).eps / 2
    tol = 8 * step if dtype == BF16 else 2.0 ** -14      # matrix products in fp32 may run in tf32 (2^-11 a factor): off by default
    for got, want in ((dw, Wt.grad), (dx, X.grad), (dg, G.grad)):
        assert float((got.double() - want).norm()) <= tol * float(want.norm())
    sure = given.bool()
    close(loss[sure], kl.detach()[sure], 1e-3 if dtype == F32 else 0.2)


# ---- refusals --------------------------------------------------------------------------------------------
def call(name, *args):
    spec = ops.REGISTRY[name][0]
    return spec.adapter(opts(), *[CudaBuffer(a, a.shape, parpy.types.F32) if isinstance(a, torch.Tensor) else a
                                  for a in args])


def test_refusals():
    b, t, d = 2, 3, 4
    a, s = torch.zeros(b, t, d), torch.zeros(b, d)
    lens, carry = torch.zeros(b, dtype=torch.int64), torch.zeros(b, 1, d)

    def bad(name, good, place, value, error, match):
        args = list(good)
        args[place] = value
        with pytest.raises(error, match=match):
            call(name, *args)
    scan = [a, a, s, lens, b, t, d, torch.zeros(b, t, d), s, carry]
    bad("gated_scan", scan, 0, a.double(), TypeError, "dtype")
    bad("gated_scan", scan, 1, a.to(BF16), TypeError, "dtype")
    bad("gated_scan", scan, 1, torch.zeros(b, t, d + 1), RuntimeError, "expected shape")
    bad("gated_scan", scan, 2, torch.zeros(b, d, dtype=BF16), TypeError, "dtype")
    bad("gated_scan", scan, 3, torch.zeros(b), TypeError, "dtype")
    bad("gated_scan", scan, 4, -1, RuntimeError, "negative")
    bad("gated_scan", scan, 7, torch.zeros(1, 1, d).expand(b, t, d), ValueError, "overlap")
    bad("gated_scan", scan, 7, None, TypeError, "missing")
    bad("gated_scan", scan, 9, torch.zeros(b, 2, d), RuntimeError, "expected shape")
    grad = [a, a, lens, b, t, d, carry, a, s, torch.zeros(b, t, d), torch.zeros(b, t, d), s]
    bad("gated_scan_grad", grad, 6, None, TypeError, "missing")
    bad("gated_scan_grad", grad, 9, torch.zeros(1, t, d).expand(b, t, d), ValueError, "overlap")
    step = [s, s, s, b, d, torch.zeros(b, d), s]
    bad("gated_step", step, 2, torch.zeros(b, d + 1), RuntimeError, "expected shape")
    bad("gated_step", step, 5, torch.zeros(d).expand(b, d), ValueError, "overlap")


def test_native_entries_refuse_before_any_launch(native):
    lib = native.lib()
    st = (32, 8)

    def scan(dtype=0, b=2, t=4, d=8, g=64, gs=st, h=64, hs=st):
        return lib.parpy_b200_gated_scan(dtype, b, t, d, g, *gs, 64, *st, None, None, 1, h, *hs, None, None, None)
    for kw, match in ((dict(dtype=5), "element type"), (dict(b=-1), "shape"), (dict(g=None), "null"),
                      (dict(h=None), "null"), (dict(g=66), "misaligned"), (dict(hs=(8, 8)), "overlap"),
                      (dict(hs=(24, 8)), "overlap"), (dict(gs=(-8, 8)), "negative")):
        assert scan(**kw) != 0 and match in native.error_message(), (kw, native.error_message())
    assert lib.parpy_b200_gated_scan_grad(0, 2, 4, 8, 64, *st, 64, *st, None, 1, None, None, 0, 0, None, 64, *st, 64,
                                          *st, None, None) != 0
    assert "carry" in native.error_message()
    assert lib.parpy_b200_gated_step(0, 2, 8, 64, 8, 64, 8, 64, 64, 4, 64, None) != 0
    assert "overlap" in native.error_message()


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("d", [64, 33])
def test_channels_do_not_reach_one_another(d, dtype):
    # a NaN gate and a NaN input in one channel each, in the middle of a run; every other channel as without them
    b, t = 2, 300
    s = inputs(b, t, d, dtype, 8)
    clean = run(s, None)
    step = [torch.empty_like(s["g"][:, 0]), torch.empty(b, d, device="cuda")]
    s["g"][0, 133, 6] = math.nan
    s["x"][1, 20, 9] = math.nan
    s["g"][1, 0, 11] = math.nan
    dirty = run(s, None)
    hit = torch.zeros(b, d, dtype=torch.bool)
    hit[0, 6] = hit[1, 9] = hit[1, 11] = True
    others = ~hit.cuda()
    # a neighbour's gates may be rounded otherwise in the run of the NaN: a reciprocal of its own, 4 steps of a gate
    rel = 2.0 ** -20 if dtype == F32 else float(torch.finfo(dtype).eps)
    for name in ("h", "dg", "dx"):
        keep = others[:, None].expand(b, t, d)
        a, c = clean[name][keep].float(), dirty[name][keep].float()
        assert torch.isfinite(c).all() and float((a - c).abs().max()) <= rel * 16
    assert torch.isnan(dirty["h"][0, 133:, 6]).all() and torch.isfinite(dirty["h"][0, :133, 6]).all()
    assert torch.isnan(dirty["last"][hit]).all() and torch.isfinite(dirty["last"][others]).all()
    assert torch.isnan(dirty["dh0"][0, 6]) and torch.isfinite(dirty["dh0"][others]).all()
    kernels.gated_step(s["g"][:, 0], s["x"][:, 0], s["h0"], b, d, step[0], step[1], opts=opts())
    assert torch.isnan(step[1][1, 11]) and int(torch.isnan(step[1]).sum()) == 1


@gpu
def test_state_is_carried_in_place():
    # chunks of a long prefill: the state buffer goes in and comes out
    b, t, d = 2, 700, 136
    s = inputs(b, t, d, BF16, 10)
    whole = run(s, None)
    state = s["h0"].clone()
    h = torch.empty_like(s["g"])
    for at in range(0, t, 256):      # whole tiles: the same runs, composed the same way within a call
        n = min(256, t - at)
        kernels.gated_scan(s["g"][:, at:at + n], s["x"][:, at:at + n], state, None, b, n, d, h[:, at:at + n], state, None,
                           opts=opts())
    want = define(s["g"], s["x"], s["h0"], None)
    r = room(s["g"], t)
    close(state, want["last"], r * want["last_size"])
    close(h, want["h"], rounding(BF16, want["h"]) + r * want["size"])
    assert whole["last"].shape == state.shape


# ---- many rounds: the staged kernels' ring of three rounds of inputs goes round several times ----------------------
@gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("b,t,d", [(70, 900, 128), (1, 9000, 64), (40, 1500, 256), (4, 5000, 72), (3, 2500, 520)])
def test_many_rounds_of_staged_rows(b, t, d, dtype):
    s = inputs(b, t, d, dtype, b + t + d)
    check(s, None, run(s, None))
    # ends in every slot of the ring, at and beside the ends of runs, tiles and rounds
    ends = torch.tensor([t, 0, 1, 128 * 5, 128 * 6 + 1, 128 * 4 - 1, t - 1, 7 * 16, 640 + 17, t - 130, 3 * 128 + 8])
    lens = ends[torch.arange(b) % len(ends)].cuda()
    out = run(s, lens)
    check(s, lens, out)
    for i, n in enumerate(lens.tolist()):
        for name in ("h", "dg", "dx"):
            assert not out[name][i, n:].any()
    check(s, lens, run(s, lens, h0=False, dh=False), h0=False, dh=False)
    check(s, lens, run(s, lens, dlast=False), dlast=False)


@gpu
def test_chunks_give_the_whole_sequence():
    # a prefill in chunks with the state in place against one call: each is within its bound of the definition
    b, t, d = 2, 900, 136
    s = inputs(b, t, d, F32, 14)
    whole = run(s, None)
    state, h = s["h0"].clone(), torch.empty_like(s["g"])
    for at in range(0, t, 250):
        n = min(250, t - at)
        kernels.gated_scan(s["g"][:, at:at + n], s["x"][:, at:at + n], state, None, b, n, d, h[:, at:at + n], state, None,
                           opts=opts())
    want = define(s["g"], s["x"], s["h0"], None)
    r = room(s["g"], t)
    close(state, whole["last"], 2 * r * want["last_size"])
    close(h, whole["h"], 2 * (rounding(F32, want["h"]) + r * want["size"]))


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("d", [70, 72])
def test_gate_gradient_at_open_and_closed_gates(d, dtype):
    b, t = 2, 3000
    s = inputs(b, t, d, dtype, 15)
    s["g"][:, :, ::3] = 12.0
    s["g"][:, :, 1::3] = -100.0
    s["g"][0, 100:140] = math.inf
    s["g"][1, 50:60] = -math.inf
    out = run(s, None)
    floor = -87.0 if dtype == F32 else -41.5              # gates below count as this
    want = define(s["g"].double().clamp(min=floor), s["x"], s["h0"], None, s["dh"], s["dlast"])
    r = 2.0 ** -21 + 4 * H * t + 200 * 3 * H
    both = want["r_size"] * (want["size"] + want["x"].abs() + s["h0"].abs().cpu().double()[:, None]) * want["keep"]
    # behind a closed gate f (1 - f) is f, from the exponential of the whole gate value
    close(out["dg"], want["dg"], rounding(dtype, want["dg"]) + 3 * r * both)
    closed = (s["g"] <= -100.0).cpu()
    near = torch.where(closed, want["dg"], torch.zeros_like(want["dg"]))
    got = torch.where(closed, out["dg"].double().cpu(), torch.zeros_like(want["dg"]))
    close(got, near, rounding(dtype, near) + 3 * r * both * torch.sigmoid(torch.tensor(floor, dtype=torch.float64)) +
          2.0 ** -120)


@gpu
@pytest.mark.parametrize("d", [5, 64])
def test_closed_gates_in_32_bits(d):
    # an fp32 gate keeps its own value down to -87: f = exp(g) to a relative error, where 16-bit types stop at -41.5
    b, t = 3, 4
    s = inputs(b, t, d, F32, 17)
    s["g"] = -torch.linspace(40.0, 86.0, b * t * d).reshape(b, t, d).cuda()
    s["x"].zero_()
    one = {k: (v[:, :1].contiguous() if v.dim() == 3 else v) for k, v in s.items()}
    out = run(one, None, dlast=False)
    f = torch.exp(one["g"].double().cpu())          # sigmoid and exp agree to exp(-40)
    # the exponent's roundings of 86 log2(e), exp2, the sum with 1, the reciprocal and the products
    rel = 86.0 * 1.5 * 2 * H + 2.0 ** -22 + 8 * H
    h0, dh = s["h0"].double().cpu(), one["dh"].double().cpu()[:, 0]
    close(out["last"], f[:, 0] * h0, rel * f[:, 0] * h0.abs() + 2.0 ** -148)
    close(out["dh0"], f[:, 0] * dh, rel * f[:, 0] * dh.abs() + 2.0 ** -148)
    h, last = torch.empty(b, d, device="cuda"), torch.empty(b, d, device="cuda")
    kernels.gated_step(one["g"][:, 0], one["x"][:, 0], s["h0"], b, d, h, last, opts=opts())
    assert torch.equal(last, out["last"])


@gpu
def test_an_infinite_input_stays_in_its_channel():
    # from its step on an infinity leaves infinities or NaN (a product of gates that has underflowed, times it) in its
    # channel, and nothing anywhere else
    b, t, d = 2, 2000, 72
    for dtype in (F32, BF16):
        s = inputs(b, t, d, dtype, 16)
        clean = run(s, None)
        s["x"][0, 700, 6] = math.inf
        s["h0"][1, 9] = -math.inf
        dirty = run(s, None)
        hit = torch.zeros(b, d, dtype=torch.bool, device="cuda")
        hit[0, 6] = hit[1, 9] = True
        for name in ("h", "dx"):
            keep = (~hit)[:, None].expand(b, t, d)
            assert torch.equal(clean[name][keep], dirty[name][keep])
        assert torch.equal(clean["last"][~hit], dirty["last"][~hit]) and not torch.isfinite(dirty["last"][hit]).any()
        assert torch.equal(clean["h"][0, :700, 6], dirty["h"][0, :700, 6])
        assert not torch.isfinite(dirty["h"][0, 700:, 6]).any() and not torch.isfinite(dirty["h"][1, :, 9]).any()
