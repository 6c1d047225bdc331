"""Log-probabilities of tokens, distillation from a teacher's best columns, and their gradients, against the
definitions in 64 bits. Tolerances follow from the arithmetic (2^-24 for each 32-bit rounding, 2^-22 for the hardware's
exp2, half a step of the output type), see ``room``."""
import math

import numpy as np
import pytest
import torch

import parpy_b200 as parpy
from parpy_b200 import kernels, ops
from parpy_b200.buffer import CudaBuffer

gpu = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
INF = math.inf
H = 2.0 ** -24


def opts():
    return parpy.par({})


# ---- the definitions ----------------------------------------------------------------------------
def logsumexp(z):
    """log(sum(exp)) of each row, -inf for a row without a finite entry, NaN with a NaN or +inf."""
    m = z.amax(1, keepdim=True)
    m = torch.where(torch.isinf(m) & (m < 0), torch.zeros_like(m), m)
    return (m + torch.log(torch.exp(z - m).sum(1, keepdim=True)))[:, 0]


def best(x, k):
    """Columns of the k largest values of each row, ties by the lowest column."""
    return torch.sort(x + 0.0, dim=1, descending=True, stable=True).indices[:, :k]


def define_logprobs(x, tokens, k, t):
    z = x.double().cpu() / t
    lse = logsumexp(z)
    m = z.amax(1, keepdim=True)
    m = torch.where(m == -INF, torch.zeros_like(m), m)
    logps = z - m - logsumexp(z - m)[:, None]      # large common offsets leave first
    logps[lse == -INF] = -INF
    p = torch.exp(logps)
    ent = -torch.where(p == 0, torch.zeros_like(p), p * logps).sum(1)
    tok = tokens.cpu().long()
    rows = torch.arange(len(z))
    logp = torch.where(tok < 0, torch.zeros_like(lse), logps[rows, tok.clamp(0, z.shape[1] - 1)])
    logp[tok >= z.shape[1]] = math.nan
    at = best(x.double().cpu(), k)
    top = torch.gather(logps, 1, at)
    broken = torch.isnan(lse)
    at[broken] = -1
    return {"lse": lse, "logp": logp, "entropy": ent, "top": top, "at": at, "p": p, "logps": logps}


def define_logprobs_grad(d, tokens, dlogp, dent, t):
    tok, rows = tokens.cpu().long(), torch.arange(len(tokens))
    m = d["p"].shape[1]
    dl = torch.where(tok >= 0, dlogp.double().cpu(), torch.zeros(len(tok), dtype=torch.float64))
    p, logps = d["p"], d["logps"]
    inside = torch.where(p == 0, torch.zeros_like(p), p * (logps + d["entropy"][:, None]))
    dz = -dl[:, None] * p - dent.double().cpu()[:, None] * inside
    dz[rows, tok.clamp(0, m - 1)] += torch.where(tok < m, dl, torch.zeros_like(dl))
    dz[d["lse"] == -INF] = 0.0
    dz[(tok >= m) | torch.isnan(d["lse"])] = math.nan
    return dz / t


def define_distill(x, index, values, t, tail, dloss):
    """Row by row, from the formulas."""
    z = x.double().cpu() / t
    n, m = z.shape
    lse = logsumexp(z)
    out = {"loss": torch.zeros(n, dtype=torch.float64), "lse": lse, "rest": torch.zeros(n, dtype=torch.float64),
           "dx": torch.zeros(n, m, dtype=torch.float64)}
    for i in range(n):
        cols, seen = [], set()
        broken = bool(torch.isnan(lse[i]))
        for j, c in enumerate(index[i].tolist()):
            if c >= m:
                broken = True
            elif c >= 0 and c not in seen:
                seen.add(c)
                cols.append((c, float(values[i, j])))
        mask = torch.zeros(m, dtype=torch.bool)
        mask[[c for c, _ in cols]] = True
        rest = float(logsumexp(z[i:i + 1].masked_fill(mask, -INF))[0])
        out["rest"][i] = rest
        v = torch.tensor([v for _, v in cols], dtype=torch.float64)
        if tail:
            q = torch.exp(v)
        else:
            q = torch.softmax(v, 0) if len(cols) and float(v.max()) != -INF else torch.zeros_like(v)
        if not bool(torch.isfinite(q).all()):
            broken = True
        logp = [float(z[i, c]) - float(lse[i]) if float(z[i, c]) > -INF else -INF for c, _ in cols]
        loss = sum(float(a) * (math.log(float(a)) - b) for a, b in zip(q, logp) if float(a) > 0)
        left = 0.0
        if tail and len(cols) < m:
            left = max(0.0, 1.0 - float(q.sum()))
            if left > 0:
                gap = rest - float(lse[i]) if rest > -INF else -INF
                loss += left * (math.log(left) - gap)
        mass = float(q.sum()) + left
        p = torch.exp(z[i] - lse[i]) if float(lse[i]) > -INF else torch.zeros(m, dtype=torch.float64)
        dz = mass * p
        if left > 0 and rest > -INF:
            dz -= torch.where(mask, torch.zeros_like(p), left * torch.exp(z[i] - rest))
        for (c, _), a in zip(cols, q):
            dz[c] -= a
        if float(lse[i]) == -INF:
            dz.zero_()
        if broken:
            loss = math.nan
            dz[:] = math.nan
        out["loss"][i] = loss
        out["dx"][i] = dz * float(dloss[i]) / t
    return out


# ---- tolerances -----------------------------------------------------------------------------------
def room(x, t):
    """Relative error that a row's sum of exponentials may carry: its exponent t = (x - ref) c has three roundings of
    its size (weighted by the terms' probabilities: at most the entropy in bits plus the 8 bits that ref may lie below
    the maximum), exp2 2^-22, and a sum of M terms over at least min(M, 128) threads with a tree above them."""
    m = x.shape[1]
    bits = math.log2(m) + 8 + 16
    return 2.0 ** -22 + H * (3 * bits + m / min(m, 512) + 24)


def close(got, want, tol):
    got, want = got.double().cpu(), want.double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    inf = torch.isinf(want)
    assert torch.equal(torch.isinf(got), inf) and torch.equal(got[inf], want[inf])
    ok = torch.isfinite(want)
    err = (got - want).abs()[ok]
    tol = torch.broadcast_to(torch.as_tensor(tol, dtype=torch.float64), want.shape)[ok]
    assert bool((err <= tol).all()), f"off by {float((err - tol).max()):.3g} more than {float(tol.max()):.3g}"


def rounding(dtype, want):
    """Half a step of the output type, of its smallest step below the normal range."""
    f = torch.finfo(dtype)
    return want.abs() * f.eps / 2 + f.tiny * f.eps / 2 + 2.0 ** -126


# ---- inputs -----------------------------------------------------------------------------------------
def logits(n, m, dtype, seed, scale=3.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(n, m, generator=g) * scale).to(dtype)


def run_logprobs(x, tokens, k, t, entropy=True, at_type=torch.int64):
    n, m = x.shape
    out = {"logp": torch.full((n,), 7.0, device="cuda"), "lse": torch.full((n,), 7.0, device="cuda"),
           "entropy": torch.full((n,), 7.0, device="cuda") if entropy else None,
           "top": torch.full((n, k), 7.0, device="cuda") if k else None,
           "at": torch.full((n, k), -7, dtype=at_type, device="cuda") if k else None}
    kernels.token_logprobs(x, tokens, n, m, k, t, out["logp"], out["lse"], out["entropy"], out["top"], out["at"],
                           opts=opts())
    return out


def check_logprobs(x, tokens, k, t, out):
    d = define_logprobs(x, tokens, k, t)
    r = room(x, t)
    finite = torch.where(torch.isfinite(d["lse"]), d["lse"].abs(), torch.zeros_like(d["lse"]))
    close(out["lse"], d["lse"], r + 2 * H * finite)
    lp = torch.where(torch.isfinite(d["logp"]), d["logp"].abs(), torch.zeros_like(finite))
    close(out["logp"], d["logp"], r + H * (finite + lp) + 2 * H * finite)
    if out["entropy"] is not None:
        close(out["entropy"], d["entropy"], 2 * r * (d["entropy"].nan_to_num(0.0) + 10) + r)
    if k:
        tl = torch.where(torch.isfinite(d["top"]), d["top"].abs(), torch.zeros_like(d["top"]))
        close(out["top"], d["top"], r + H * tl + 3 * H * finite[:, None])
        assert torch.equal(out["at"].cpu().long(), d["at"])
    return d


SHAPES = [(1, 1), (3, 2), (5, 7), (4, 129), (2, 1023), (3, 4096), (2, 16385), (1, 65536), (300, 5003), (1, 262144),
          (700, 300), (40, 40009)]


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape", SHAPES)
def test_logprobs_and_gradient(shape, dtype):
    n, m = shape
    x = logits(n, m, dtype, 7 * n + m).cuda()
    g = torch.Generator().manual_seed(3)
    tokens = torch.randint(0, m, (n,), generator=g)
    tokens[1::7] = -1
    tokens = tokens.cuda()
    t = [1.0, 0.7, 2.0][(n + m) % 3]
    k = min(m, [0, 1, 5, 20, 128][(n + 2 * m) % 5])
    out = run_logprobs(x, tokens, k, t)
    d = check_logprobs(x, tokens, k, t, out)
    dl, de = torch.randn(n, generator=g).cuda(), torch.randn(n, generator=g).cuda()
    dx = torch.full_like(x, 7.0)
    kernels.token_logprobs_grad(x, tokens, n, m, t, out["lse"], out["entropy"], dl, de, dx, opts=opts())
    want = define_logprobs_grad(d, tokens, dl, de, t)
    size = d["p"] * (dl.cpu().abs()[:, None] + de.cpu().abs()[:, None] *
                     (d["logps"].abs().clamp(max=200.0) + d["entropy"][:, None])) / t
    # p: exponent's roundings, lse's rounding, exp2; log p and the entropy carry their own errors
    rel = room(x, t) + 3 * H * d["lse"].abs()[:, None] + 4 * H * d["logps"].abs().clamp(max=200.0)
    off = d["p"] * de.cpu().abs()[:, None] * (room(x, t) * 20 + H * 400) / t
    close(dx, want, rounding(dtype, want) + size * rel + off + dl.cpu().abs()[:, None] * 2 * H / t)
    # without the entropy's part, in place
    y = x.clone()
    kernels.token_logprobs_grad(y, tokens, n, m, t, out["lse"], None, dl, None, y, opts=opts())
    want = define_logprobs_grad(d, tokens, dl, torch.zeros(n), t)
    close(y, want, rounding(dtype, want) + size * rel + dl.cpu().abs()[:, None] * 2 * H / t)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("m", [1, 9, 700, 33000, 70001])
def test_logprobs_of_masked_and_broken_rows(m, dtype):
    low = torch.finfo(dtype).min
    x = logits(12, m, dtype, m)
    x[0] = -INF
    x[1] = -INF
    x[1, m // 2] = 3.0
    x[2] = low
    x[3, ::2] = low
    x[4, m // 3] = math.nan
    x[5, -1] = INF
    x[6] = 0.0
    x[6, ::3] = -0.0
    x[7] = torch.linspace(-5, 5, m).to(dtype)
    x[8] = torch.linspace(5, -5, m).to(dtype)
    x[9] = -INF
    x[9, :max(1, m // 50)] = 1.0
    x[10] = 100.0 if dtype != F16 else 60000.0
    x[11, 0] = -INF
    tokens = torch.tensor([0, m // 2, 0, 0, 0, 0, m - 1, -1, m, 0, -5, 0], dtype=torch.int32)
    xd, td = x.cuda(), tokens.cuda()
    for k in (1, min(m, 33), min(m, 128)):
        for t in (1.0, 4.0):
            out = run_logprobs(xd, td, k, t, at_type=torch.int32)
            d = check_logprobs(xd, td, k, t, out)
    dl = torch.ones(12, device="cuda")
    dx = torch.full_like(xd, 7.0)
    kernels.token_logprobs_grad(xd, td, 12, m, t, out["lse"], out["entropy"], dl, dl, dx, opts=opts())
    want = define_logprobs_grad(d, td, dl, dl, t)
    assert torch.equal(torch.isnan(dx).cpu(), torch.isnan(want))
    assert not dx[0].cpu().any()                                        # nothing in the row
    size = d["p"] * (1 + d["logps"].abs().clamp(max=200.0) + d["entropy"][:, None]) / t
    finite = torch.where(torch.isfinite(d["lse"]), d["lse"].abs(), torch.zeros_like(d["lse"]))[:, None]
    rel = room(xd, t) * 20 + 400 * H + 3 * H * finite.clamp(max=1e5)
    ok = [0, 1, 3, 6, 7, 8, 9, 10, 11]
    close(dx[ok], want[ok], (rounding(dtype, want) + size.nan_to_num(0) * rel + 2 * H)[ok])


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_sharp_rows_stay_probabilities(dtype):
    # one column holds nearly everything: log-probabilities not above 0, entropies not below, whatever rounds
    n, m = 400, 2051
    g = torch.Generator().manual_seed(2)
    x = torch.randn(n, m, generator=g)
    x[torch.arange(n), torch.randint(0, m, (n,), generator=g)] = 12.0 + 40.0 * torch.rand(n, generator=g)
    x = x.to(dtype).cuda()
    tokens = x.float().argmax(1)
    for t in (1.0, 0.05):
        out = run_logprobs(x, tokens, 3, t)
        check_logprobs(x, tokens, 3, t, out)
        assert float(out["logp"].max()) <= 0 and float(out["top"].max()) <= 0 and float(out["entropy"].min()) >= 0
        dx = torch.empty_like(x)
        big = torch.full((n,), 1e9, device="cuda")
        kernels.token_logprobs_grad(x, tokens, n, m, t, out["lse"], out["entropy"], big, big, dx, opts=opts())
        assert torch.isfinite(dx.float()).all()


@gpu
@pytest.mark.parametrize("m", [24, 1000, 70001])
def test_broken_rows_report_every_alternative_as_none(m):
    # NaN of either sign, one or everywhere, and an infinity: NaN and -1 in all K places, the other rows as they are
    x = torch.randn(6, m, generator=torch.Generator().manual_seed(m))
    nan = torch.tensor([0xffc00000 - (1 << 32), 0x7fc00000], dtype=torch.int32).view(F32)
    x[1] = nan[0]
    x[2] = nan[1]
    x[3, m // 2] = nan[0]
    x[4, ::2] = nan[0]
    x[5, 3] = INF
    tokens = torch.zeros(6, dtype=torch.int64, device="cuda")
    for dtype in (F32, BF16, F16):
        xd = x.to(dtype).cuda()
        for k in (1, 20, min(m, 24)):
            out = run_logprobs(xd, tokens, k, 1.0)
            assert bool((out["at"][1:] == -1).all()) and torch.isnan(out["top"][1:]).all()
            assert torch.isnan(out["lse"][1:]).all() and torch.isnan(out["entropy"][1:]).all()
            check_logprobs(xd[:1], tokens[:1], k, 1.0, {name: v[:1] for name, v in out.items()})


@gpu
def test_many_candidates_for_few_places():
    # a thread's columns lie one stride apart: give every one of many threads a run of values above all others, so
    # that far more columns pass the selection's first bound than its list holds
    m, k = 131072, 100
    for dtype, per in ((BF16, 8), (F32, 4)):
        x = torch.full((300, m), -4.0).to(dtype)
        g = torch.Generator().manual_seed(9)
        for stride in (128, 512, 1024, 2048, 4096):
            cols = (torch.arange(0, m, stride * per)[:, None] + torch.arange(per)[None, :]).reshape(-1)
            x[0 if stride < 512 else stride // 512, cols] = torch.randn(len(cols), generator=g).to(dtype)
        x[9, :m // 2] = 1.0
        x[10] = torch.randn(m, generator=g).abs().to(dtype)
        xd = x.cuda()
        for rows in (slice(0, 300), slice(0, 11)):      # one CTA a row, and several
            tok = torch.zeros(xd[rows].shape[0], dtype=torch.int64, device="cuda")
            out = run_logprobs(xd[rows], tok, k, 1.0)
            assert torch.equal(out["at"].cpu(), best(x[rows].double(), k))


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rows_that_lie_apart_and_start_anywhere(dtype):
    n, m = 33, 1237
    wide = logits(n + 1, m + 91, dtype, 5).cuda()
    grad = torch.full((n, m + 55), 7.0, dtype=dtype, device="cuda")
    tokens = torch.arange(n, device="cuda")
    for c0 in (0, 1, 3, 8):
        x, dx = wide[1:, c0:c0 + m], grad[:, 7:7 + m]
        out = run_logprobs(x, tokens, 7, 1.0)
        d = check_logprobs(x, tokens, 7, 1.0, out)
        dl = torch.ones(n, device="cuda")
        kernels.token_logprobs_grad(x, tokens, n, m, 1.0, out["lse"], None, dl, None, dx, opts=opts())
        want = define_logprobs_grad(d, tokens, dl, torch.zeros(n), 1.0)
        close(dx, want, rounding(dtype, want) + d["p"] * (room(x, 1.0) + 400 * H) + 2 * H)
        assert bool((grad[:, :7] == 7).all()) and bool((grad[:, 7 + m:] == 7).all())   # beside the rows: as they were
    with pytest.raises(ValueError, match="contiguous"):
        kernels.token_logprobs(wide[:, ::2], tokens, n + 1, (m + 91 + 1) // 2, 0, 1.0, None, out["lse"], None, None,
                               None, opts=opts())
    with pytest.raises(ValueError, match="overlap"):
        one = torch.empty(m, dtype=dtype, device="cuda")
        kernels.token_logprobs_grad(wide[1:, :m], tokens, n, m, 1.0, out["lse"], None, dl, None, one.expand(n, m),
                                    opts=opts())


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_gradient_into_rows_of_another_pitch(dtype):
    n, m = 21, 1030
    x = logits(n, m, dtype, 15).cuda()
    tokens = torch.arange(n, device="cuda")
    dl = torch.ones(n, device="cuda")
    out = run_logprobs(x, tokens, 0, 1.0)
    plain = torch.empty_like(x)
    kernels.token_logprobs_grad(x, tokens, n, m, 1.0, out["lse"], None, dl, None, plain, opts=opts())
    for pad, c0 in ((2, 2), (1, 1), (4, 0), (16, 8), (34, 6)):
        wide = torch.full((n, m + pad), 7.0, dtype=dtype, device="cuda")
        kernels.token_logprobs_grad(x, tokens, n, m, 1.0, out["lse"], None, dl, None, wide[:, c0:c0 + m], opts=opts())
        assert torch.equal(wide[:, c0:c0 + m], plain)
        assert bool((wide[:, :c0] == 7).all()) and bool((wide[:, c0 + m:] == 7).all())

@gpu
def test_host_arrays_and_optional_outputs():
    n, m, k = 6, 500, 3
    x = logits(n, m, F32, 1)
    tokens = np.arange(n, dtype=np.int64)
    lse, top, at = np.zeros(n, np.float32), np.zeros((n, k), np.float32), np.zeros((n, k), np.int64)
    kernels.token_logprobs(x.numpy(), None, n, m, k, 1.0, None, lse, None, top, at, opts=opts())
    d = define_logprobs(x, torch.from_numpy(tokens), k, 1.0)
    close(torch.from_numpy(lse), d["lse"], 1e-5)
    assert np.array_equal(at, d["at"].numpy())
    xb = x.to(BF16)                             # a host tensor without a NumPy type
    dx = torch.zeros(n, m, dtype=BF16)
    kernels.token_logprobs_grad(xb, tokens, n, m, 1.0, lse, None, np.ones(n, np.float32), None, dx, opts=opts())
    d = define_logprobs(xb, torch.from_numpy(tokens), 0, 1.0)
    want = define_logprobs_grad(d, torch.from_numpy(tokens), torch.ones(n), torch.zeros(n), 1.0)
    # lse is of the unrounded logits: up to half a step of the largest, 2^-8 |x|, away
    close(dx, want, rounding(BF16, want) + d["p"] * float(x.abs().max()) * 2.0 ** -7 + 2 * H)
    empty = torch.empty(0, m, device="cuda")
    kernels.token_logprobs(empty, None, 0, m, 0, 1.0, None, torch.empty(0, device="cuda"), None, None, None, opts=opts())


# ---- distillation -------------------------------------------------------------------------------------
def teacher(n, m, k, seed, dtype=F32):
    g = torch.Generator().manual_seed(seed)
    index = torch.stack([torch.randperm(m, generator=g)[:k] for _ in range(n)])
    values = (torch.log_softmax(torch.randn(n, k, generator=g) * 2, 1) - 0.1).to(dtype)
    return index, values


def run_distill(x, index, values, t, tail, dloss):
    n, m = x.shape
    k = index.shape[1]
    dev = dict(device="cuda")
    loss, lse = torch.full((n,), 7.0, **dev), torch.full((n,), 7.0, **dev)
    rest = torch.full((n,), 7.0, **dev) if tail else None
    dx = torch.full((n, m), 7.0, dtype=x.dtype, **dev)
    kernels.distill_topk(x, index, values, n, m, k, t, tail, loss, lse, rest, opts=opts())
    kernels.distill_topk_grad(x, index, values, n, m, k, t, tail, lse, rest, dloss, dx, opts=opts())
    return {"loss": loss, "lse": lse, "rest": rest, "dx": dx}


def check_distill(x, index, values, t, tail, dloss, out):
    d = define_distill(x, index.cpu(), values.float().cpu(), t, tail, dloss.cpu())
    r = room(x, t)

    def size(v):
        return torch.where(torch.isfinite(v), v.abs(), torch.zeros_like(v))
    lse = size(d["lse"])
    close(out["lse"], d["lse"], r + 3 * H * lse)
    z = torch.where(torch.isfinite(x), x, torch.zeros_like(x)).double().cpu() / t
    # q carries expf's error (2 steps) and its normaliser's; log q - log p the errors of lse and of its own size
    big = 40.0 + lse + z.abs().amax(1)
    close(out["loss"], d["loss"], r + 8 * H * big + 4 * H * size(d["loss"]))
    if tail:
        close(out["rest"], d["rest"], r + 3 * H * size(d["rest"]))
    w = dloss.double().cpu().abs()[:, None] / t
    p = torch.exp(z - lse_safe(d["lse"])[:, None])
    rest = torch.where(torch.isfinite(d["rest"]), d["rest"], torch.full_like(d["rest"], INF))
    pr = torch.exp(z - rest[:, None]).clamp(max=1.0)
    tol = rounding(x.dtype, d["dx"].nan_to_num(0)) + w * (p + pr * tail + 1e-30) * (r + 8 * H * big[:, None])
    cols = index.cpu().clamp(0, x.shape[1] - 1).long()
    tol.scatter_add_(1, cols, (w * 8 * H * big[:, None]).expand_as(cols).contiguous())
    close(out["dx"], d["dx"], tol)
    return d


def lse_safe(v):
    return torch.where(torch.isfinite(v), v, torch.full_like(v, INF))


@gpu
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("n,m,k", [(1, 1, 1), (3, 2, 1), (4, 9, 9), (5, 130, 64), (2, 1025, 5), (40, 5003, 20),
                                   (1, 65536, 128), (300, 4096, 8), (2, 40009, 1000)])
def test_distill_and_gradient(n, m, k, dtype, tail):
    x = logits(n, m, dtype, n + m + k).cuda()
    index, values = teacher(n, m, k, m)
    g = torch.Generator().manual_seed(1)
    dloss = torch.randn(n, generator=g).cuda()
    t = [1.0, 2.0, 0.7][(n + m) % 3]
    out = run_distill(x, index.cuda(), values.cuda(), t, tail, dloss)
    check_distill(x, index, values, t, tail, dloss, out)


@gpu
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("m", [40, 33000])
def test_distill_lists_and_rows_out_of_the_ordinary(m, tail):
    n, k = 14, 12
    x = logits(n, m, F32, 2)
    index, values = teacher(n, m, k, 4)
    index[0] = -1                                   # no entry
    index[1, 3:] = -1
    index[2] = index[2, 0]                          # one column, many times
    index[3, 5] = m                                 # past the vocabulary
    index[4, 5] = m + (1 << 33)
    values[5] = -INF                                # entries without mass
    values[6, :6] = -INF
    x[7] = -INF                                     # nothing in the student's row
    x[8, index[8, 2]] = -INF                        # the student excludes what the teacher wants
    x[9] = -INF
    x[9, index[9]] = torch.randn(k)                 # the student has nothing outside the list
    x[10] -= 200.0
    x[10, index[10]] += 200.0                       # next to nothing outside the list
    x[11, 5] = math.nan
    values[12, 4] = math.nan
    x[13] = torch.finfo(F32).min
    dloss = torch.ones(n).cuda()
    xd = x.cuda()
    out = run_distill(xd, index.cuda(), values.cuda(), 1.0, tail, dloss)
    rows = [i for i in range(n) if i != 13]
    sub = {name: (v[rows] if v is not None else None) for name, v in out.items()}
    check_distill(xd[rows], index[rows], values[rows], 1.0, tail, dloss[rows], sub)
    # lowest values everywhere are a uniform row: lse is of their size, the gradient of a uniform p
    assert torch.isfinite(out["dx"][13]).all()
    # 32-bit indices and 16-bit teachers
    small = index.clone()
    small[4, 5] = -1
    i32 = run_distill(xd, small.int().cuda(), values.cuda(), 1.0, tail, dloss)
    i64 = run_distill(xd, small.cuda(), values.cuda(), 1.0, tail, dloss)
    for name in ("loss", "lse", "dx"):
        assert torch.equal(i32[name].view(torch.int32), i64[name].view(torch.int32))
    for half in (BF16, F16):
        vh = values.to(half)
        a = run_distill(xd, small.cuda(), vh.cuda(), 1.0, tail, dloss)
        b = run_distill(xd, small.cuda(), vh.float().cuda(), 1.0, tail, dloss)
        assert torch.equal(a["dx"].view(torch.int32), b["dx"].view(torch.int32))


@gpu
@pytest.mark.parametrize("tail", [False, True])
def test_distill_whole_vocabulary_in_place_and_finite_differences(tail):
    n, m = 4, 24
    x = logits(n, m, F32, 3, scale=1.0)
    index = torch.arange(m).repeat(n, 1)
    values = torch.log_softmax(torch.randn(n, m, generator=torch.Generator().manual_seed(8)), 1)
    dloss = torch.ones(n).cuda()
    out = run_distill(x.cuda(), index.cuda(), values.cuda(), 1.0, tail, dloss)
    check_distill(x.cuda(), index, values, 1.0, tail, dloss, out)
    index, values = index[:, :5], values[:, :5]
    out = run_distill(x.cuda(), index.cuda(), values.cuda(), 1.5, tail, dloss)
    step = 2.0 ** -6
    for j in (0, 4, 5, 23):
        a, b = x.clone(), x.clone()
        a[:, j] += step
        b[:, j] -= step
        up = run_distill(a.cuda(), index.cuda(), values.cuda(), 1.5, tail, dloss)["loss"].double()
        down = run_distill(b.cuda(), index.cuda(), values.cuda(), 1.5, tail, dloss)["loss"].double()
        # losses of size 4 carry 2^-21 each over a step of 2^-5; the third derivative is below 1: step^2 / 6
        assert torch.allclose((up - down) / (2 * step), out["dx"][:, j].double(), rtol=0, atol=2.0 ** -14 + step ** 2)
    y = x.cuda()
    kernels.distill_topk_grad(y, index.cuda(), values.cuda(), n, m, 5, 1.5, tail, out["lse"], out["rest"], dloss, y,
                              opts=opts())
    assert torch.equal(y, out["dx"])


@gpu
def test_teacher_from_the_alternatives_of_its_own_logits():
    # the teacher's rows give the list, the student's rows the loss; against the same student the tail's loss is 0
    n, m, k = 9, 8191, 32
    x = logits(n, m, BF16, 12).cuda()
    out = run_logprobs(x, torch.zeros(n, dtype=torch.int64, device="cuda"), k, 1.5)
    d = run_distill(x, out["at"], out["top"], 1.5, True, torch.ones(n, device="cuda"))
    # each log q - log p is off by the roundings of lse and of both logarithms
    assert float(d["loss"].abs().max()) <= room(x, 1.5) * 4 + 40 * 8 * H
    assert float(d["dx"].float().abs().max()) <= room(x, 1.5) * 4 + 40 * 8 * H


@gpu
def test_streams_graphs_and_repeated_calls():
    n, m, k = 37, 30011, 9
    x = logits(n, m, BF16, 4).cuda()
    tokens = torch.arange(n, device="cuda")
    index, values = (v.cuda() for v in teacher(n, m, k, 6))
    dloss = torch.ones(n, device="cuda")
    first = run_logprobs(x, tokens, k, 1.0)
    dist = run_distill(x, index, values, 1.0, True, dloss)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = run_logprobs(x, tokens, k, 1.0)
    side.synchronize()
    for name in first:
        assert torch.equal(first[name], again[name])          # no order of atomics shows
    buf = {name: torch.zeros_like(v) for name, v in first.items()}
    dbuf = {name: torch.zeros_like(v) for name, v in dist.items()}

    def both():
        o = opts()
        kernels.token_logprobs(x, tokens, n, m, k, 1.0, buf["logp"], buf["lse"], buf["entropy"], buf["top"], buf["at"],
                               opts=o)
        kernels.distill_topk(x, index, values, n, m, k, 1.0, True, dbuf["loss"], dbuf["lse"], dbuf["rest"], opts=o)
        kernels.distill_topk_grad(x, index, values, n, m, k, 1.0, True, dbuf["lse"], dbuf["rest"], dloss, dbuf["dx"],
                                  opts=o)
    both()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        both()
    keep = x.clone()
    x.copy_(logits(n, m, BF16, 5))
    graph.replay()
    new = run_logprobs(x, tokens, k, 1.0)
    torch.cuda.synchronize()
    assert all(torch.equal(buf[name], new[name]) for name in buf)
    x.copy_(keep)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(buf[name], first[name]) for name in buf)
    assert all(torch.equal(dbuf[name], dist[name]) for name in dbuf)


# ---- refusals: before any launch, so they need no GPU ------------------------------------------------
def wrap(t):
    return None if t is None else CudaBuffer(t, t.shape, parpy.types.F32)


def call(name, *args):
    spec = ops.REGISTRY[name][0]
    return spec.adapter(opts(), *[wrap(a) if isinstance(a, torch.Tensor) else a for a in args])


def test_refusals_of_logprobs():
    n, m = 3, 8
    x, tok, v = torch.zeros(n, m), torch.zeros(n, dtype=torch.int64), torch.zeros(n)
    top, at = torch.zeros(n, 2), torch.zeros(n, 2, dtype=torch.int64)
    good = [x, tok, n, m, 2, 1.0, v, v, v, top, at]

    def bad(place, value, error, match):
        args = list(good)
        args[place] = value
        with pytest.raises(error, match=match):
            call("token_logprobs", *args)
    bad(0, torch.zeros(n, m + 1), RuntimeError, "expected shape")
    bad(0, torch.zeros(n, m, dtype=torch.float64), TypeError, "dtype")
    bad(0, torch.zeros(m, n).t(), ValueError, "contiguous")
    bad(1, torch.zeros(n), TypeError, "dtype")
    bad(1, None, TypeError, "missing")
    bad(4, 9, RuntimeError, "outside")
    bad(4, -1, RuntimeError, "outside")
    bad(5, 0.0, RuntimeError, "temperature")
    bad(5, math.nan, RuntimeError, "temperature")
    bad(7, None, TypeError, "missing")
    bad(9, torch.zeros(n, 3), RuntimeError, "expected shape")
    bad(10, torch.zeros(n, 2), TypeError, "dtype")
    grad = [x, tok, n, m, 1.0, v, v, v, v, torch.zeros(n, m)]

    def bad_grad(place, value, error, match):
        args = list(grad)
        args[place] = value
        with pytest.raises(error, match=match):
            call("token_logprobs_grad", *args)
    bad_grad(9, torch.zeros(n, m, dtype=BF16), TypeError, "dtype")
    bad_grad(9, torch.zeros(m).expand(n, m), ValueError, "overlap")
    bad_grad(6, None, TypeError, "missing")
    bad_grad(1, None, TypeError, "missing")


def test_refusals_of_distill():
    n, m, k = 3, 8, 2
    x, v = torch.zeros(n, m), torch.zeros(n)
    index, values = torch.zeros(n, k, dtype=torch.int64), torch.zeros(n, k)
    good = [x, index, values, n, m, k, 1.0, True, v, v, v]

    def bad(place, value, error, match):
        args = list(good)
        args[place] = value
        with pytest.raises(error, match=match):
            call("distill_topk", *args)
    bad(1, torch.zeros(n, k), TypeError, "dtype")
    bad(1, torch.zeros(n, 3, dtype=torch.int64), RuntimeError, "expected shape")
    bad(2, torch.zeros(n, k, dtype=torch.int64), TypeError, "dtype")
    bad(5, 0, RuntimeError, "outside")
    bad(5, 1025, RuntimeError, "outside")
    bad(6, 1e5, RuntimeError, "temperature")
    bad(10, None, TypeError, "missing")


def test_native_entries_refuse_before_any_launch(native):
    lib = native.lib()
    for args, match in [
            ((None, 9, 8, 3, 8, None, 1, 1.0, 0, None, None, None, None, None, 1, None), "element type"),
            ((None, 0, 8, -1, 8, None, 1, 1.0, 0, None, None, None, None, None, 1, None), "shape"),
            ((None, 0, 8, 3, 0, None, 1, 1.0, 0, None, None, None, None, None, 1, None), "shape"),
            ((None, 0, 7, 3, 8, None, 1, 1.0, 0, None, None, None, None, None, 1, None), "pitch"),
            ((None, 0, 8, 3, 8, None, 1, 0.0, 0, None, None, None, None, None, 1, None), "temperature"),
            ((None, 0, 8, 3, 8, None, 1, 1.0, 0, None, None, None, None, None, 1, None), "null"),
            ((6, 0, 8, 3, 8, None, 1, 1.0, 0, None, 64, None, None, None, 1, None), "misaligned"),
            ((64, 0, 8, 3, 8, None, 1, 1.0, 129, None, 64, None, None, None, 1, None), "outside"),
            ((64, 0, 8, 3, 8, None, 1, 1.0, 0, 64, 64, None, None, None, 1, None), "null")]:
        assert lib.parpy_b200_token_logprobs(*args) != 0
        assert match in native.error_message(), (match, native.error_message())
    assert lib.parpy_b200_token_logprobs_grad(64, 0, 8, 3, 8, None, 1, 1.0, 64, None, None, None, 64, 12, None) != 0
    assert "in place" in native.error_message()
    assert lib.parpy_b200_distill_topk(64, 0, 8, 3, 8, 64, 1, 64, 7, 2, 1.0, 0, 64, 64, None, None) != 0
    assert "element type" in native.error_message()
    assert lib.parpy_b200_distill_topk(64, 0, 8, 3, 8, 64, 1, 64, 0, 2, 1.0, 1, 64, 64, None, None) != 0
    assert "null" in native.error_message()


# ---- rows that a CTA takes after its first -----------------------------------------------------------------
# As many CTAs as are resident take rows in turn: at most 32 warps an SM, 148 SMs, so 4736 rows of one warp, 1184 of 128
# threads and 592 of 256 are in flight at once. Every test below has more rows than that, rows that start at every
# alignment, and tokens, lists and masks of each row's own.
@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,m,k,entropy", [(5000, 61, 3, True), (5000, 300, 0, True), (2600, 2101, 0, True),
                                           (2600, 3001, 0, False), (1300, 2101, 7, True), (1300, 9001, 20, True),
                                           (700, 40009, 20, True), (700, 17003, 128, False)])
def test_logprobs_of_more_rows_than_ctas(n, m, k, entropy, dtype):
    x = logits(n, m, dtype, n + m + k)
    x += (torch.arange(n) % 23 - 11).to(dtype)[:, None]     # each row its own reference
    x[3::16] = torch.where(torch.arange(m) % 8 == 5, x[3::16], torch.full((), -INF, dtype=dtype))
    x[n - 40::9] = -INF
    x[n - 39::9, m // 2] = math.nan
    tokens = torch.arange(n) * 37 % m
    tokens[5::11] = -1
    tokens[n - 30] = m
    xd, td = x.cuda(), tokens.cuda()
    out = run_logprobs(xd, td, k, 0.7, entropy=entropy)
    d = check_logprobs(xd, td, k, 0.7, out)
    if entropy and k == 0:
        dl, de = torch.linspace(-2, 2, n).cuda(), torch.linspace(1, -1, n).cuda()
        dx = torch.full_like(xd, 7.0)
        kernels.token_logprobs_grad(xd, td, n, m, 0.7, out["lse"], out["entropy"], dl, de, dx, opts=opts())
        want = define_logprobs_grad(d, td, dl, de, 0.7)
        p, surprise = d["p"].nan_to_num(0), d["logps"].abs().clamp(max=200.0).nan_to_num(0)
        size = p * (dl.cpu().abs()[:, None] + de.cpu().abs()[:, None] * (surprise + d["entropy"].nan_to_num(0)[:, None]))
        finite = torch.where(torch.isfinite(d["lse"]), d["lse"].abs(), torch.zeros_like(d["lse"]))
        rel = room(xd, 0.7) + 3 * H * finite[:, None] + 4 * H * surprise
        off = p * de.cpu().abs()[:, None] * (room(xd, 0.7) * 20 + H * 400)
        close(dx, want, rounding(dtype, want.nan_to_num(0)) + (size * rel + off) / 0.7 +
              dl.cpu().abs()[:, None] * 2 * H / 0.7)


def distill_rows(x, index, values, t, tail):
    """``define_distill`` without a gradient, for lists of distinct columns: all rows at once."""
    z = x.double().cpu() / t
    used = index >= 0
    v = torch.where(used, values.double(), torch.full((), -INF, dtype=torch.float64))
    q = torch.exp(v) if tail else torch.softmax(v, 1)
    lse = logsumexp(z)
    lp = z.gather(1, index.clamp(min=0)) - lse[:, None]
    loss = torch.where(q > 0, q * (torch.log(q) - lp), torch.zeros_like(q)).sum(1)
    spot = torch.where(used, index, torch.full_like(index, z.shape[1]))
    mask = torch.zeros(z.shape[0], z.shape[1] + 1, dtype=torch.bool).scatter_(1, spot, True)[:, :-1]
    rest = logsumexp(z.masked_fill(mask, -INF))
    if tail:
        left = 1.0 - q.sum(1)
        loss += left * (torch.log(left) - (rest - lse))
    return loss, lse, rest


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,m,k,tail", [(2600, 3001, 20, False), (2600, 1999, 33, True), (1300, 9001, 20, True),
                                        (1300, 17003, 64, False)])
def test_distill_of_more_rows_than_ctas(n, m, k, tail, dtype):
    x = logits(n, m, dtype, n + m)
    x += (torch.arange(n) % 23 - 11).to(dtype)[:, None]
    start, step = torch.arange(n)[:, None] * 131 % m, torch.arange(n)[:, None] % (m // k - 1) + 1
    index = (start + step * torch.arange(k)) % m                  # distinct columns, another list in every row
    g = torch.Generator().manual_seed(k)
    values = torch.log_softmax(torch.randn(n, k, generator=g) * 2, 1) - 0.1
    index[7::13, k // 2:] = -1
    dloss = torch.linspace(-1, 1, n).cuda()
    xd = x.cuda()
    out = run_distill(xd, index.cuda(), values.cuda(), 0.7, tail, dloss)
    loss, lse, rest = distill_rows(x, index, values, 0.7, tail)
    r = room(xd, 0.7)
    big = 40.0 + lse.abs() + x.double().abs().amax(1) / 0.7
    close(out["lse"], lse, r + 3 * H * lse.abs())
    close(out["loss"], loss, r + 8 * H * big + 4 * H * loss.abs())
    if tail:
        close(out["rest"], rest, r + 3 * H * rest.abs())
    # the gradient's rows have a CTA each: a sample of them against the definition
    rows = torch.arange(0, n, n // 40)
    sub = {name: (v[rows.cuda()] if v is not None else None) for name, v in out.items()}
    check_distill(xd[rows.cuda()], index[rows], values[rows], 0.7, tail, dloss.cpu()[rows], sub)


# ---- broken rows of a distillation -----------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("m", [24, 9001])
def test_distill_rows_with_an_infinity_or_nan_are_nan(m, tail):
    # +inf or NaN in a listed column while nothing else is left, under a teacher that wants that column or does not,
    # and in a column that is not listed while the teacher wants columns which the student has masked
    n, k = 8, 4
    x = torch.full((n, m), -INF)
    index = (torch.arange(k) * 3 + torch.arange(n)[:, None]) % m
    values = torch.log(torch.tensor([0.4, 0.3, 0.2, 0.05])).repeat(n, 1)
    x[0, index[0]] = torch.tensor([1.0, INF, 0.5, 2.0])
    x[1, index[1]] = torch.tensor([1.0, INF, 0.5, 2.0])
    values[1, 1] = -INF                          # the teacher has no use for it
    x[2, index[2]] = torch.tensor([1.0, math.nan, 0.5, 2.0])
    values[2, 1] = -INF
    x[3, index[3, 0]] = INF
    values[3, 0] = -INF
    x[4] = 0.0
    x[4, index[4]] = -INF
    x[4, m - 1] = math.nan
    x[5] = 0.0
    x[5, 5] = INF
    index[5] = -1                                # nothing listed
    x[6] = 0.0                                   # sound
    x[7, index[7]] = 1.0                         # sound: nothing outside the list
    out = run_distill(x.cuda(), index.cuda(), values.cuda(), 1.0, tail, torch.ones(n).cuda())
    for name in ("loss", "lse"):
        assert torch.isnan(out[name][:6]).all() and not torch.isnan(out[name][6:]).any(), name
    assert torch.isnan(out["dx"][:6]).all() and not torch.isnan(out["dx"][6:]).any()


# ---- rows far from zero ------------------------------------------------------------------------------------
def shifted(x):
    """A row's logits below its largest, in 64 bits: log-probabilities, losses and gradients are the same, and no sum has
    the size of the row's offset."""
    x = x.double().cpu()
    top = x.amax(1, keepdim=True)
    return x - torch.where(torch.isinf(top), torch.zeros_like(top), top)


def far_rows(m, dtype, seed):
    """Rows of the type's lowest and highest values, of large common offsets, and masked with the lowest value."""
    low, high = torch.finfo(dtype).min, torch.finfo(dtype).max
    x = logits(8, m, dtype, seed)
    x[0] = low                                        # a mask of the lowest value over the whole row
    x[1] = low
    x[1, 1::3] = -INF
    x[2, ::2] = low                                   # ordinary: under such a mask
    x[3] = high
    x[4] = (x[4].float() * 8 + 3e4).to(dtype)
    x[5] = (x[5].float() * 8 - 3e4).to(dtype)
    x[6] = (x[6].float() + 700.0).to(dtype)
    return x


@gpu
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("m", [9, 1000, 33000])
def test_distill_loss_of_rows_far_from_zero(m, dtype, tail):
    k = 6
    for t in (1.0, 0.5, 0.01):
        x = far_rows(m, dtype, m)
        n = x.shape[0]
        index, values = teacher(n, m, k, m + 1)
        out = run_distill(x.cuda(), index.cuda(), values.cuda(), t, tail, torch.ones(n).cuda())
        near = shifted(x)
        loss, _, _ = distill_rows(near, index, values, t, tail)
        # q carries expf's error; log q - log p that of the row's sum, and a rounding of its own size
        size = torch.where(torch.isfinite(near), near.abs(), torch.zeros_like(near)).gather(1, index).amax(1) / t
        tol = room(x, t) + 8 * H * (40.0 + size) + 4 * H * loss.abs().nan_to_num(posinf=0.0)
        close(out["loss"], loss.float(), tol)          # past the type's range: an infinity
        assert torch.isfinite(out["lse"]).all()       # limited to the range of its type


@gpu
def test_teacher_values_far_from_zero():
    # a teacher's logits with a common offset, or of the lowest value: the same probabilities as without
    n, m, k = 5, 300, 9
    x = logits(n, m, F32, 31)
    index, values = teacher(n, m, k, 32)
    values = (values * 64).round() / 64                      # offsets below leave them exact
    far = values + torch.tensor([0.0, 512.0, -30000.0, 60000.0, 0.0])[:, None]
    values[4], far[4] = 0.0, torch.finfo(F32).min
    dloss = torch.ones(n).cuda()
    out = run_distill(x.cuda(), index.cuda(), far.cuda(), 1.0, False, dloss)
    check_distill(x.cuda(), index, values, 1.0, False, dloss, out)
    # q only: the loss is free of the offset's size
    loss, lse, _ = distill_rows(x, index, values, 1.0, False)
    close(out["loss"], loss, room(x, 1.0) + 8 * H * (40.0 + lse.abs() + x.double().abs().amax(1)))


COARSE = {F32: 64.0 * H, BF16: 1024.0 * H, F16: 1024.0 * H}     # |lse| up to which its 32 bits serve the gradient


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("m", [1, 9, 1000, 33000, 200003])
def test_gradient_of_rows_far_from_zero(m, dtype):
    # probabilities come from differences to the row's own sum, however large the offset or small the temperature:
    # no term of the tolerance has the size of lse beyond the bound up to which its 32 bits are used
    for t in (1.0, 0.5, 0.01, 1e-4):
        x = far_rows(m, dtype, m + 1)
        n = x.shape[0]
        tokens = (torch.arange(n) * 7 % m).cuda()
        xd = x.cuda()
        out = run_logprobs(xd, tokens, 0, t)
        d = define_logprobs(shifted(x), tokens, 0, t)
        assert torch.isfinite(out["lse"]).all()
        dl, de = torch.linspace(1, 2, n).cuda(), torch.linspace(0.5, -1, n).cuda()
        size = d["p"] * (dl.cpu().abs()[:, None] + de.cpu().abs()[:, None] *
                         (d["logps"].abs().clamp(max=200.0) + d["entropy"][:, None])) / t
        rel = room(x, t) + COARSE[dtype] + 4 * H * d["logps"].abs().clamp(max=200.0)
        off = d["p"] * de.cpu().abs()[:, None] * (room(x, t) * 20 + H * 400) / t
        for bonus in (de, None):
            want = define_logprobs_grad(d, tokens, dl, de if bonus is not None else torch.zeros(n), t)
            tol = rounding(dtype, want) + size * rel + off + dl.cpu().abs()[:, None] * 2 * H / t
            tol = tol + 210.0 * 2.0 ** -126 / t     # exp2 gives 0 below 2^-126, times |dlogp| + |dentropy| (|log p| + entropy)
            dx = torch.full_like(xd, 7.0)
            kernels.token_logprobs_grad(xd, tokens, n, m, t, out["lse"], out["entropy"], dl, bonus, dx, opts=opts())
            close(dx, want, tol)
            for rows in (slice(0, n), slice(0, 1)):      # in place, many rows and one
                y = xd[rows].clone()
                kernels.token_logprobs_grad(y, tokens[rows], y.shape[0], m, t, out["lse"][rows], out["entropy"][rows],
                                            dl[rows], bonus[rows] if bonus is not None else None, y, opts=opts())
                close(y, want[rows], tol[rows])


@gpu
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("m", [9, 1000, 33000])
def test_distill_gradient_of_rows_far_from_zero(m, dtype, tail):
    k = 6
    for t in (1.0, 0.5, 0.01):
        x = far_rows(m, dtype, m + 2)
        x[7] = (x[7].float() - 90.0).to(dtype)
        n = x.shape[0]
        index, values = teacher(n, m, k, m + 3)
        x[7, index[7]] = (x[7, index[7]].float() + 90.0).to(dtype)     # nearly nothing outside the list
        dloss = torch.linspace(0.5, 1, n)
        xd, idx, val = x.cuda(), index.cuda(), values.cuda()
        out = run_distill(xd, idx, val, t, tail, dloss.cuda())
        near = shifted(x)
        d = define_distill(near, index, values, t, tail, dloss)
        w = dloss.double()[:, None] / t
        p = torch.exp(near / t - d["lse"][:, None])
        rest = torch.where(torch.isfinite(d["rest"]), d["rest"], torch.full_like(d["rest"], INF))
        pr = torch.exp(near / t - rest[:, None]).clamp(max=1.0)
        rel = room(x, t) + 2 * COARSE[dtype] + 8 * H * (40.0 + torch.log(p).abs().clamp(max=200.0))
        # exp2 gives 0 below 2^-126: an absolute error of p and pr, which w scales like every other
        tol = rounding(dtype, d["dx"]) + w * ((p + pr * tail) * rel + 2.0 ** -125)
        tol.scatter_add_(1, index, (w * 8 * H * 40.0).expand(n, k).contiguous())
        close(out["dx"], d["dx"], tol)
        y = xd.clone()
        kernels.distill_topk_grad(y, idx, val, n, m, k, t, tail, out["lse"], out["rest"], dloss.cuda(), y, opts=opts())
        close(y, d["dx"], tol)


@gpu
def test_gradient_takes_a_sum_over_more_columns_as_it_is():
    # a vocabulary in two halves on two devices: each half's gradient from the sum over both, near zero and far from it
    n, m = 6, 2002
    x = logits(n, m, F32, 41)
    x[3:] += 200.0
    tokens = torch.arange(n)
    out = run_logprobs(x.cuda(), tokens.cuda(), 0, 1.0)
    dl = torch.ones(n).cuda()
    none = torch.full((n,), -1)
    d = define_logprobs(x, tokens, 0, 1.0)
    want = define_logprobs_grad(d, tokens, dl, torch.zeros(n), 1.0)
    for half, tok in ((slice(0, m // 2), tokens), (slice(m // 2, m), none)):
        part, dx = x[:, half].contiguous().cuda(), torch.empty(n, m // 2, device="cuda")
        scale = dl if tok is tokens else 3.0 * dl       # without a token there is no term
        kernels.token_logprobs_grad(part, tok.cuda(), n, m // 2, 1.0, out["lse"], None, scale, None, dx, opts=opts())
        expect = want[:, half] if tok is tokens else torch.zeros(n, m // 2)
        close(dx, expect, d["p"][:, half] * (room(x, 1.0) + 250 * H + 80 * H) + 2.0 ** -22)
    # the entropy's term needs no token
    ones = torch.ones(n).cuda()
    want = define_logprobs_grad(d, none, dl, ones, 1.0)
    for half in (slice(0, m // 2), slice(m // 2, m)):
        part, dx = x[:, half].contiguous().cuda(), torch.empty(n, m // 2, device="cuda")
        kernels.token_logprobs_grad(part, None, n, m // 2, 1.0, out["lse"], out["entropy"], None, ones, dx, opts=opts())
        size = d["p"][:, half] * (d["logps"][:, half].abs() + d["entropy"][:, None])
        close(dx, want[:, half], size * (room(x, 1.0) + 330 * H) + d["p"][:, half] * (room(x, 1.0) * 20 + H * 400))


@gpu
def test_gradients_in_place_captured_and_at_once():
    # few rows in place (a row's CTAs share a sum where it is far from zero) and with a list, each in a graph of its own,
    # both replayed at once on two streams over new logits
    n, m, k = 3, 70001, 9
    tokens, dl = torch.arange(n, device="cuda") * 5, torch.ones(n, device="cuda")
    index, values = (v.cuda() for v in teacher(n, m, k, 51))
    for dtype in (F32, BF16):
        source = logits(n, m, dtype, 50).cuda()
        y, z = torch.empty_like(source), torch.empty_like(source)
        logp, lse, entropy = (torch.empty(n, device="cuda") for _ in range(3))
        loss, lse2, rest = (torch.empty(n, device="cuda") for _ in range(3))

        def one(y=y):
            o = opts()
            y.copy_(source)
            kernels.token_logprobs(y, tokens, n, m, 0, 0.5, logp, lse, entropy, None, None, opts=o)
            kernels.token_logprobs_grad(y, tokens, n, m, 0.5, lse, entropy, dl, dl, y, opts=o)

        def other(z=z):
            o = opts()
            z.copy_(source)
            kernels.distill_topk(z, index, values, n, m, k, 0.5, True, loss, lse2, rest, opts=o)
            kernels.distill_topk_grad(z, index, values, n, m, k, 0.5, True, lse2, rest, dl, z, opts=o)
        graphs = []
        for call in (one, other):
            call()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                call()
            graphs.append(graph)
        streams = [torch.cuda.Stream() for _ in graphs]
        for offset in (0.0, 2000.0, -300.0):
            source.copy_(logits(n, m, dtype, 52) + torch.tensor([offset, 0.0, -offset])[:, None].to(dtype))
            torch.cuda.synchronize()
            for _ in range(3):
                for graph, stream in zip(graphs, streams):
                    with torch.cuda.stream(stream):
                        graph.replay()
            torch.cuda.synchronize()
            got = y.clone(), z.clone()
            out = run_logprobs(source, tokens, 0, 0.5)
            apart = torch.empty_like(source)
            kernels.token_logprobs_grad(source, tokens, n, m, 0.5, out["lse"], out["entropy"], dl, dl, apart, opts=opts())
            d = define_logprobs(shifted(source), tokens, 0, 0.5)
            want = define_logprobs_grad(d, tokens, dl, dl, 0.5)
            size = d["p"] * (1 + d["logps"].abs().clamp(max=200.0) + d["entropy"][:, None]) / 0.5
            rel = room(source, 0.5) + COARSE[dtype] + 4 * H * d["logps"].abs().clamp(max=200.0)
            tol = rounding(dtype, want) + size * rel + d["p"] * (room(source, 0.5) * 20 + H * 400) / 0.5 + 4 * H + 2.0 ** -117
            close(apart, want, tol)
            close(got[0], want, tol)
            same = run_distill(source, index, values, 0.5, True, dl)
            assert torch.equal(got[1], same["dx"]) and torch.equal(loss, same["loss"])
