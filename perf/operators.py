"""Cases of the language-model operators: token log-probabilities with entropy and top alternatives, distillation
from a teacher's top logits (both with their gradients), and the gated linear recurrence with its gradient and its
single-token step. ``listed`` names fixed cases, ``draw`` makes more of the same ranges, ``run`` makes one pass,
through this package's kernels where ``own`` is true and in plain torch operations where it is not, and ``exact``
computes the same outputs in 64 bits from the definitions.

Definitions (z = x / temperature, one row of M logits; -inf marks a column that a mask took out):

  token_logprobs   lse = log sum exp z;  logp = z[token] - lse (0 for a negative token);
                   entropy = -sum p log p, p = exp(z - lse);  the K largest of x, ties to the lowest column
  its gradient     dx = (dlogp (onehot(token) - p) - dentropy p (log p + entropy)) / temperature
  distill_topk     q = softmax(values) over a row's listed columns, or with `tail` q = exp(values) and the rest
                   bucket (1 - sum q) against the student's mass outside the list;
                   loss = sum q (log q - log p[column]) [+ q_rest (log q_rest - log p_rest)]
  its gradient     dx = dloss d loss / d z / temperature
  gated_scan       f = sigmoid(g);  h_t = f_t h_{t-1} + (1 - f_t) x_t, h zero and the state held from lens on
  its gradient     r_t = dh_t + f_{t+1} r_{t+1};  dx = (1 - f) r;  dg = r (h_{t-1} - x) f (1 - f);  dh0 = f_1 r_1
  gated_step       one step of the recurrence for every row of a decoding batch
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
LOGITS = 4096 * 131072     # logits of the largest listed case
STEPS = 65536 * 2048       # gate values of the largest listed recurrence


def listed():
    return [
        # one row per decoding step: the log-probability of the sampled token and eight alternatives
        {"name": "logprobs decode", "op": "logprobs", "dtype": "f32", "N": 1, "M": 65536, "K": 8, "T": 1.0, "grad": False},
        # scoring a batch of answers under a large vocabulary, twenty alternatives for each position
        {"name": "logprobs score", "op": "logprobs", "dtype": "bf16", "N": 4096, "M": 131072, "K": 20, "T": 1.0,
         "grad": False},
        # policy training: log-probability and entropy, both with a gradient, at a sampling temperature
        {"name": "logprobs train", "op": "logprobs", "dtype": "bf16", "N": 4096, "M": 65536, "K": 0, "T": 0.7,
         "grad": True},
        # the same on an odd vocabulary (rows start at every alignment) in 32 bits, with alternatives
        {"name": "logprobs train odd", "op": "logprobs", "dtype": "f32", "N": 777, "M": 40009, "K": 5, "T": 1.0,
         "grad": True},
        # distillation step on a large vocabulary, the teacher's 64 best renormalised
        {"name": "distill train", "op": "distill", "dtype": "bf16", "N": 4096, "M": 131072, "K": 64, "T": 1.0,
         "tail": False},
        # odd sizes in 32 bits, with the bucket of all other columns
        {"name": "distill tail odd", "op": "distill", "dtype": "f32", "N": 1023, "M": 32771, "K": 20, "T": 1.0,
         "tail": True},
        # a small microbatch at a softened temperature: latency counts
        {"name": "distill small", "op": "distill", "dtype": "f16", "N": 32, "M": 16384, "K": 8, "T": 2.0, "tail": True},
        # prefill of one long document
        {"name": "scan prefill", "op": "scan", "dtype": "bf16", "B": 1, "T": 65536, "D": 2048, "ragged": False,
         "grad": False},
        # training on a padded batch of ragged sequences (the benchmark's 1000 to 4000 steps)
        {"name": "scan train", "op": "scan", "dtype": "bf16", "B": 16, "T": 4000, "D": 2048, "ragged": True,
         "grad": True},
        # odd sizes in 32 bits
        {"name": "scan train odd", "op": "scan", "dtype": "f32", "B": 5, "T": 1999, "D": 515, "ragged": True,
         "grad": True},
        # one token for a few sequences
        {"name": "step small", "op": "step", "dtype": "bf16", "N": 8, "D": 1024},
        # one token for a large serving batch
        {"name": "step batch", "op": "step", "dtype": "bf16", "N": 2048, "D": 8192},
    ]


def _spread(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["logprobs", "logprobs", "distill", "distill", "scan", "scan", "step"])
    case = {"op": op, "dtype": rng.choice(["bf16", "bf16", "f16", "f32"])}
    if op in ("logprobs", "distill"):
        m = _spread(rng, 16, 262144)
        most = LOGITS // (2 if case["dtype"] == "f32" else 1)
        case |= {"M": m, "N": _spread(rng, 1, max(1, min(8192, most // m))), "T": rng.choice([1.0, 0.7, 1.3, 2.0])}
        if op == "logprobs":
            grad = rng.random() < 0.5
            case |= {"K": min(m, rng.choice([0, 1, 5, 20, 64])), "grad": grad}
        else:
            case |= {"K": min(m // 4, _spread(rng, 1, 128)), "tail": rng.random() < 0.5}
    elif op == "scan":
        d, t = _spread(rng, 1, 8192), _spread(rng, 1, 65536)
        grad = rng.random() < 0.5
        most = STEPS // (4 if grad or case["dtype"] == "f32" else 1)
        t = min(t, max(1, most // d))
        case |= {"D": d, "T": t, "B": _spread(rng, 1, max(1, min(64, most // (d * t)))),
                 "ragged": rng.random() < 0.5, "grad": grad}
    else:
        case |= {"N": _spread(rng, 1, 4096), "D": _spread(rng, 1, 16384)}
    return case


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, shift=0.0, to=torch.float32):
        v = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)
        return v.mul_(scale).add_(shift).to(to)

    def whole(low, high, *shape):
        return torch.randint(low, high, shape, generator=gen, device="cuda", dtype=torch.int64)

    def empty(*shape, to=torch.float32):
        return torch.empty(shape, device="cuda", dtype=to)

    s = dict(case)
    if case["op"] in ("logprobs", "distill"):
        n, m, k = case["N"], case["M"], case["K"]
        s["x"] = normal(n, m, scale=3.0, to=dtype)
        if n > 1:   # constrained decoding: every 16th row keeps about one column in eight
            some = s["x"][::16]
            some.masked_fill_(torch.rand(some.shape, generator=gen, device="cuda") > 0.125, -math.inf)
            s["x"][::16, m // 2] = 1.0
        s["lse"] = empty(n)
        if case["op"] == "distill" or case["grad"]:
            s["dx"] = empty(n, m, to=dtype)
    if case["op"] == "logprobs":
        tokens = whole(0, m, n)
        if n > 1:
            tokens[::16] = m // 2
            tokens[1::16] = -1      # positions of a prompt: no token to score
        s |= {"tokens": tokens, "logp": empty(n), "entropy": empty(n),
              "top": empty(n, k) if k else None, "at": empty(n, k, to=torch.int64) if k else None,
              "dlogp": normal(n), "dentropy": normal(n, scale=0.01)}
    elif case["op"] == "distill":
        start, step = whole(0, m, n, 1), whole(1, max(2, m // max(1, k)), n, 1)
        index = (start + step * torch.arange(k, device="cuda")) % m
        values = torch.log_softmax(normal(n, k, scale=2.0), 1) + math.log(0.9)
        if n > 1:
            s["x"][::16] = torch.where(torch.isinf(s["x"][::16]), torch.full((), -12.0, device="cuda", dtype=dtype),
                                       s["x"][::16])
            index[1::16, k // 2:] = -1      # a teacher that gave fewer
        s |= {"index": index, "values": values, "loss": empty(n), "rest": empty(n), "dloss": normal(n)}
    elif case["op"] == "scan":
        b, t, d = case["B"], case["T"], case["D"]
        s |= {"g": normal(b, t, d, scale=1.5, shift=3.0, to=dtype), "x": normal(b, t, d, to=dtype),
              "h0": normal(b, d), "h": empty(b, t, d, to=dtype), "last": empty(b, d), "lens": None, "carry": None}
        if case["ragged"]:
            s["lens"] = whole(t // 4, t + 1, b)
            s["lens"][0] = t
        if case["grad"]:
            s |= {"dh": normal(b, t, d, to=dtype), "dlast": normal(b, d), "dg": empty(b, t, d, to=dtype),
                  "dx": empty(b, t, d, to=dtype), "dh0": empty(b, d), "carry": empty(b, (t + 127) // 128, d)}
    else:
        n, d = case["N"], case["D"]
        s |= {"g": normal(n, d, scale=1.5, shift=3.0, to=dtype), "x": normal(n, d, to=dtype),
              "state": normal(n, d), "h": empty(n, d, to=dtype), "last": empty(n, d)}
    return s


# ---- the plain forms ----------------------------------------------------------------------------
def _lse(z):
    m = z.amax(1, keepdim=True)
    m = torch.where(torch.isinf(m), torch.zeros_like(m), m)
    return (m + torch.log(torch.exp(z - m).sum(1, keepdim=True)))[:, 0]


def _plain_logprobs(s):
    x, tokens, dtype = s["x"], s["tokens"], s["x"].dtype
    z = x.float() / s["T"]
    lse = _lse(z)
    given = tokens >= 0
    logp = torch.where(given, z.gather(1, tokens.clamp(min=0)[:, None])[:, 0] - lse, torch.zeros_like(lse))
    logps = z - lse[:, None]
    p = torch.exp(logps)
    entropy = -torch.where(p > 0, p * logps, torch.zeros_like(p)).sum(1)
    out = {"logp": logp, "lse": lse, "entropy": entropy}
    if s["K"]:
        # the order of (value, lowest column) as one whole number: the float's bits made monotone, then the column
        bits = (x.float() + 0.0).view(torch.int32).to(torch.int64)
        order = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
        column = torch.arange(x.shape[1], device=x.device)
        at = (order * (1 << 31) + ((1 << 31) - 1 - column)).topk(s["K"], dim=1).indices
        out |= {"top": logps.gather(1, at), "at": at}
    if s["grad"]:
        inside = torch.where(p > 0, p * (logps + entropy[:, None]), torch.zeros_like(p))
        dlogp = torch.where(given, s["dlogp"], torch.zeros_like(lse))
        dx = -dlogp[:, None] * p - s["dentropy"][:, None] * inside
        dx.scatter_add_(1, tokens.clamp(min=0)[:, None], dlogp[:, None])
        out["dx"] = (dx / s["T"]).to(dtype)
    return out


def _plain_distill(s):
    x, index, k = s["x"], s["index"], s["K"]
    z = x.float() / s["T"]
    lse = _lse(z)
    earlier = torch.ones(k, k, dtype=torch.bool, device=x.device).tril(-1)
    used = (index >= 0) & ~((index[:, :, None] == index[:, None, :]) & earlier).any(2)
    v = torch.where(used, s["values"].float(), torch.full_like(s["values"], -math.inf))
    zero = torch.zeros_like(v)
    logp = z.gather(1, index.clamp(min=0)) - lse[:, None]
    if not s["tail"]:
        logq = v - _lse(v)[:, None]
        q = torch.exp(logq)
        loss = torch.where(q > 0, q * (logq - logp), zero).sum(1)
        dz = torch.exp(z - lse[:, None]) * q.sum(1, keepdim=True)
        dz.scatter_add_(1, index.clamp(min=0), torch.where(used, -q, zero))
        return {"loss": loss, "lse": lse, "dx": (dz * (s["dloss"] / s["T"])[:, None]).to(x.dtype)}
    q = torch.exp(v)
    listed_at = torch.zeros(z.shape, dtype=torch.bool, device=x.device)
    row = torch.arange(z.shape[0], device=x.device)[:, None].expand_as(index)
    listed_at[row[used], index[used]] = True
    rest = _lse(z.masked_fill(listed_at, -math.inf))
    left = (1.0 - torch.exp(v.double()).sum(1)).clamp(min=0.0)     # next to a border: 64 bits
    term = torch.where(left > 0, left * (torch.log(left) - (rest - lse).double()), torch.zeros_like(left))
    loss = torch.where(q > 0, q * (v - logp), zero).sum(1) + term.float()
    left = left.float()
    total = q.sum(1) + left
    dz = total[:, None] * torch.exp(z - lse[:, None])
    dz -= torch.where(listed_at, torch.zeros_like(z), left[:, None] * torch.exp(z - rest[:, None]))
    dz.scatter_add_(1, index.clamp(min=0), torch.where(used, -q, zero))
    return {"loss": loss, "lse": lse, "rest": rest, "dx": (dz * (s["dloss"] / s["T"])[:, None]).to(x.dtype)}


def _recurrence(logf, u, first):
    """h_t = exp(logf_t) h_{t-1} + u_t along dimension 1, in closed form: with L the running sum of logf, h_t =
    exp(L_t) (first + sum_s exp(-L_s) u_s), positive and negative u apart in logarithms. L grows with the length and
    its differences are what counts, hence 64 bits."""
    total = torch.cumsum(logf, 1)
    up = torch.exp(total + torch.logcumsumexp(torch.log(u.clamp(min=0.0)) - total, 1))
    down = torch.exp(total + torch.logcumsumexp(torch.log((-u).clamp(min=0.0)) - total, 1))
    return up - down + torch.exp(total) * first[:, None]


def _plain_scan(s):
    dtype, (b, t, d) = s["x"].dtype, s["x"].shape
    g, x, h0 = s["g"].double(), s["x"].double(), s["h0"].double()
    logf = -torch.log1p(torch.exp(-g))
    keep = 1.0 / (1.0 + torch.exp(g))       # 1 - f
    inside = torch.ones(b, t, 1, dtype=torch.bool, device=g.device)
    if s["lens"] is not None:
        inside = (torch.arange(t, device=g.device) < s["lens"][:, None])[:, :, None]
        logf = torch.where(inside, logf, 0.0)
        keep = torch.where(inside, keep, 0.0)
    state = _recurrence(logf, keep * x, h0)
    out = {"h": torch.where(inside, state, 0.0).to(dtype), "last": state[:, -1].float()}
    if s["grad"]:
        before = torch.cat([h0[:, None], state[:, :-1]], 1)
        dh = torch.where(inside, s["dh"].double(), 0.0)
        back = torch.cat([torch.zeros_like(logf[:, :1]), logf.flip(1)[:, :-1]], 1)
        r = _recurrence(back, dh.flip(1), s["dlast"].double()).flip(1)
        f = torch.exp(logf)
        out |= {"dx": (keep * r).to(dtype), "dg": (r * (before - x) * f * keep).to(dtype),
                "dh0": (f[:, 0] * r[:, 0]).float()}
    return out


def _plain_step(s):
    g, x = s["g"].float(), s["x"].float()
    last = s["state"] / (1.0 + torch.exp(-g)) + x / (1.0 + torch.exp(g))
    return {"h": last.to(s["x"].dtype), "last": last}


# ---- one pass -----------------------------------------------------------------------------------
def _own(s):
    from parpy_b200 import kernels, par
    opts = par({})
    if s["op"] == "logprobs":
        n, m, k, t = s["N"], s["M"], s["K"], s["T"]
        kernels.token_logprobs(s["x"], s["tokens"], n, m, k, t, s["logp"], s["lse"], s["entropy"], s["top"], s["at"],
                               opts=opts)
        out = {"logp": s["logp"], "lse": s["lse"], "entropy": s["entropy"]}
        if k:
            out |= {"top": s["top"], "at": s["at"]}
        if s["grad"]:
            kernels.token_logprobs_grad(s["x"], s["tokens"], n, m, t, s["lse"], s["entropy"], s["dlogp"],
                                        s["dentropy"], s["dx"], opts=opts)
            out["dx"] = s["dx"]
        return out
    if s["op"] == "distill":
        n, m, k, t, tail = s["N"], s["M"], s["K"], s["T"], s["tail"]
        rest = s["rest"] if tail else None
        kernels.distill_topk(s["x"], s["index"], s["values"], n, m, k, t, tail, s["loss"], s["lse"], rest, opts=opts)
        kernels.distill_topk_grad(s["x"], s["index"], s["values"], n, m, k, t, tail, s["lse"], rest, s["dloss"],
                                  s["dx"], opts=opts)
        out = {"loss": s["loss"], "lse": s["lse"], "dx": s["dx"]}
        return out | {"rest": rest} if tail else out
    if s["op"] == "scan":
        b, t, d = s["B"], s["T"], s["D"]
        kernels.gated_scan(s["g"], s["x"], s["h0"], s["lens"], b, t, d, s["h"], s["last"], s["carry"], opts=opts)
        out = {"h": s["h"], "last": s["last"]}
        if s["grad"]:
            kernels.gated_scan_grad(s["g"], s["x"], s["lens"], b, t, d, s["carry"], s["dh"], s["dlast"], s["dg"],
                                    s["dx"], s["dh0"], opts=opts)
            out |= {"dg": s["dg"], "dx": s["dx"], "dh0": s["dh0"]}
        return out
    kernels.gated_step(s["g"], s["x"], s["state"], s["N"], s["D"], s["h"], s["last"], opts=opts)
    return {"h": s["h"], "last": s["last"]}


def run(state):
    if own:
        return _own(state)
    plain = {"logprobs": _plain_logprobs, "distill": _plain_distill, "scan": _plain_scan, "step": _plain_step}
    return plain[state["op"]](state)


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] in ("logprobs", "distill"):
        n, m, k = case["N"], case["M"], case["K"]
        grad = case["op"] == "distill" or case["grad"]
        # a gradient needs the row's sums before its first value: the logits twice, the gradient once
        moved = n * m * size * (3 if grad else 1) + n * (24 + 12 * k)
        return {"bytes": moved, "flops": n * m * (14 if grad else 7)}
    if case["op"] == "scan":
        b, t, d = case["B"], case["T"], case["D"]
        # forward g, x -> h; backward g, x, dh -> dg, dx. Steps behind a sequence's end need no reading: ragged
        # lengths run from a quarter to the whole, five eighths on average
        e = b * t * d
        read, written = (2 + 3, 1 + 2) if case["grad"] else (2, 1)
        share = 0.625 if case["ragged"] and b > 1 else 1.0
        return {"bytes": int(e * size * (read * share + written)) + 16 * b * d, "flops": e * (30 if case["grad"] else 10)}
    n, d = case["N"], case["D"]
    return {"bytes": n * d * (3 * size + 8), "flops": n * d * 10}


# ---- the definitions in 64 bits -----------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    dtype = torch.float64
    if case["op"] in ("logprobs", "distill"):
        parts = []
        rows = max(1, (1 << 26) // case["M"])
        for at in range(0, case["N"], rows):
            here = slice(at, at + rows)
            z = s["x"][here].to(dtype) / case["T"]
            logps = torch.log_softmax(z, 1)
            p = logps.exp()
            got = {"lse": torch.logsumexp(z, 1)}
            each = torch.arange(z.shape[0], device=z.device)
            if case["op"] == "logprobs":
                tokens = s["tokens"][here]
                given = (tokens >= 0).to(dtype)
                one = tokens.clamp(min=0)
                got["logp"] = logps[each, one].nan_to_num(neginf=0.0) * given
                surprise = torch.where(p > 0, -logps, torch.zeros_like(p))
                got["entropy"] = torch.linalg.vecdot(p, surprise)
                if case["K"]:
                    got["top"] = logps.topk(case["K"], dim=1).values
                if case["grad"]:
                    dlogp, dent = s["dlogp"][here].to(dtype) * given, s["dentropy"][here].to(dtype)
                    dz = p * (dent[:, None] * (surprise - got["entropy"][:, None]) - dlogp[:, None])
                    dz[each, one] += dlogp
                    got["dx"] = dz / case["T"]
            else:
                index, values = s["index"][here], s["values"][here].to(dtype)
                k = case["K"]
                spot = torch.where(index >= 0, index, torch.full_like(index, case["M"]))
                # teacher's mass over the vocabulary and one spare column; the lists of these inputs are distinct
                q = values.exp() * (index >= 0)
                if not case["tail"]:
                    q = q / q.sum(1, keepdim=True)
                teacher = torch.zeros(z.shape[0], case["M"] + 1, dtype=dtype, device=z.device).scatter_(1, spot, q)
                inlist = torch.zeros_like(teacher, dtype=torch.bool).scatter_(1, spot, True)[:, :-1]
                teacher = teacher[:, :-1]
                got["loss"] = (torch.xlogy(teacher, teacher) - torch.where(inlist & (teacher > 0), teacher * logps,
                                                                           torch.zeros_like(p))).sum(1)
                dz = p * teacher.sum(1, keepdim=True) - teacher
                if case["tail"]:
                    left = (1.0 - teacher.sum(1)).clamp(min=0.0)
                    got["rest"] = torch.logsumexp(z.masked_fill(inlist, -math.inf), 1)
                    got["loss"] += torch.xlogy(left, left) - left * (got["rest"] - got["lse"])
                    outside = torch.softmax(z.masked_fill(inlist, -math.inf), 1)
                    dz += left[:, None] * (p - outside)
                got["dx"] = dz * (s["dloss"][here].to(dtype) / case["T"])[:, None]
                del k
            parts.append(got)
        out = {name: torch.cat([g[name] for g in parts]) for name in parts[0]}
        if case.get("K") and case["op"] == "logprobs":
            out["at"] = None
        return out
    if case["op"] == "scan":
        b, t, d = case["B"], case["T"], case["D"]
        if b * t * d > 140_000_000:
            return None
        lens = s["lens"] if s["lens"] is not None else torch.full((b,), t, device="cuda")
        state = s["h0"].to(dtype)
        states = torch.empty(b, t + 1, d, dtype=dtype, device="cuda")
        states[:, 0] = state
        h = torch.zeros(b, t, d, dtype=dtype, device="cuda")
        for i in range(t):
            f = torch.sigmoid(s["g"][:, i].to(dtype))
            alive = (lens > i)[:, None]
            new = torch.lerp(s["x"][:, i].to(dtype), state, f)
            state = torch.where(alive, new, state)
            states[:, i + 1] = state
            h[:, i] = torch.where(alive, new, h[:, i])
        out = {"h": h, "last": state}
        if case["grad"]:
            dg, dx = torch.zeros_like(h), torch.zeros_like(h)
            r = s["dlast"].to(dtype)
            for i in range(t - 1, -1, -1):
                f = torch.sigmoid(s["g"][:, i].to(dtype))
                alive = (lens > i)[:, None]
                now = r + s["dh"][:, i].to(dtype)
                dx[:, i] = torch.where(alive, now - f * now, dx[:, i])
                dg[:, i] = torch.where(alive, now * (states[:, i] - s["x"][:, i].to(dtype)) * (f - f * f), dg[:, i])
                r = torch.where(alive, f * now, r)
            out |= {"dg": dg, "dx": dx, "dh0": r}
        return out
    f = torch.sigmoid(s["g"].to(dtype))
    last = f * s["state"].to(dtype) + (1.0 - f) * s["x"].to(dtype)
    return {"h": last, "last": last}
