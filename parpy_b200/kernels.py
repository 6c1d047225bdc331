"""The reduction-heavy functions of the reference's tests and benchmarks, bound
to their native kernels under the reference's names and signatures: ``softmax``
(test/test_softmax.py:11-26), the twelve row / axis / full reductions
(test/test_reduce.py:12-70), ``spmv_row`` (test/test_spmv.py:12-18) and the
SDDMM kernels (benchmarks/sddmm.py:21-41,63-70). All take ``opts=`` and write
their outputs in place. ``sum_max`` is this package's fused one-pass sum + max
of a long vector.

Beside them stand operators of language models on the same kinds of data: on rows of
vocabulary logits ``token_logprobs`` and ``distill_topk`` with their gradients; over
padded sequences the recurrence ``gated_scan`` with its gradient and, for decoding,
``gated_step``. They take float32, bfloat16 and float16 and, for CUDA arrays, rows that
lie apart (a slice of a wider matrix); arguments that may be ``None`` are named in their
docstrings, and outputs overlap inputs only where those say so."""
from . import jit
from ._native import SCAN_TILE


@jit
def softmax(x, N, M, out):
    """out[i,:] = softmax(x[i,:])"""


def _bind_reduce(name):
    def template(x, out, N):
        pass
    template.__name__ = name
    template.__qualname__ = name
    return jit(template)


sum_rows, prod_rows, max_rows, min_rows = (_bind_reduce(f"{o}_rows") for o in ("sum", "prod", "max", "min"))
sum_axis, prod_axis, max_axis, min_axis = (_bind_reduce(f"{o}_axis") for o in ("sum", "prod", "max", "min"))
sum_2d, prod_2d, max_2d, min_2d = (_bind_reduce(f"{o}_2d") for o in ("sum", "prod", "max", "min"))


@jit
def spmv_row(A, x, y):
    """y[row] += sum(A.values[i] * x[A.cols[i]]) over the row's non-zeros"""


@jit
def parpy_sddmm_decompress_csr(C_crows, C_rows, N):
    """C_rows[i] = row of non-zero i"""


@jit
def parpy_sddmm_csr_kernel(A, B, C, D, N, alpha, beta):
    """D[i] = alpha * dot(A[row_i,:], B[:,col_i]) + beta * C.values[i]; fills C.rows"""


@jit
def parpy_sddmm_coo_kernel(A, B, C, D, alpha, beta):
    """D[i] = alpha * dot(A[C.rows[i],:], B[:,C.cols[i]]) + beta * C.values[i]"""


def sum_max(x):
    """(sum, max) of a float32 CUDA tensor of any shape in one pass over it;
    returns a 2-element CUDA tensor."""
    import ctypes
    import torch
    from . import _native
    if not (isinstance(x, torch.Tensor) and x.is_cuda and x.dtype == torch.float32 and x.is_contiguous()):
        raise TypeError("sum_max expects a contiguous float32 CUDA tensor")
    out = torch.empty(2, dtype=torch.float32, device=x.device)
    P = ctypes.c_void_p
    rc = _native.lib().parpy_b200_sum_max(P(x.data_ptr()), x.numel(), P(out.data_ptr()),
                                          P(out.data_ptr() + 4), P(torch.cuda.current_stream().cuda_stream))
    _native.check(rc, "sum_max")
    return out


@jit
def normalize_rows(t, nrows, ncols):
    """t[i,:] /= sum(t[i,:]), in place"""


@jit
def sum_exp_3d(x, N, M, out):
    """x = exp(x) in place; out[i,j] = sum(x[i,j,:])"""


@jit
def spmm_cell(A, B, C):
    """C[i,j] += sum over row i's non-zeros of A.values[a] * B.values[A.cols[a], j]"""


@jit
def token_logprobs(x, tokens, N, M, K, temperature, logp, lse, entropy, top_logp, top_index):
    """For every row of logits x[N,M], with z = x / temperature: lse = log(sum(exp(z))),
    logp = z[tokens] - lse (0 for a negative token, NaN for one past the row), the
    entropy of softmax(z), and the K (at most 128) largest columns in falling order, ties by the lowest:
    their log-probabilities top_logp[N,K] and numbers top_index[N,K]. A logit of -inf is a column that a
    mask took out; a row of nothing else has lse and logp -inf and entropy 0; a row with a
    NaN or +inf gets NaN (top_index -1). ``tokens`` with ``logp``, ``entropy``, and for K = 0 ``top_logp``
    and ``top_index`` may be None. lse (and entropy) are what the gradient needs; lse stops at the range
    of float32."""


@jit
def token_logprobs_grad(x, tokens, N, M, temperature, lse, entropy, dlogp, dentropy, dx):
    """dx[N,M] = gradient of sum(dlogp * logp + dentropy * entropy) with respect to x, in x's
    type; dx may be x, and must not overlap it otherwise. ``dlogp`` (then ``tokens``) and ``dentropy``
    (then ``entropy``) may be None. ``lse`` and ``entropy`` are what ``token_logprobs`` wrote for the same
    arguments. The alternatives are reported, not differentiated. A row without a finite logit gets zeros.
    Rows with abs(lse) above 64 (16-bit types: 1024) are summed again, which costs them a second pass."""


@jit
def distill_topk(x, index, values, N, M, K, temperature, tail, loss, lse, rest):
    """loss[N] = distance of the student's softmax(x / temperature) from a teacher known by its K (at most 1024)
    best columns index[N,K] and their logits or log-probabilities values[N,K], at the temperature wanted
    (what ``token_logprobs`` gives as top_index and top_logp). Without ``tail`` the teacher's
    probabilities are renormalised over the list: sum(q * (log(q) - log(p))). With it q = exp(values),
    and the mass that the list leaves is compared with the student's mass outside the list. A
    negative index is an entry not given, a column's second mention is not used, an index past the row
    makes it NaN. Also writes lse[N] and, with a tail, rest[N] (else None), which the gradient needs."""


@jit
def distill_topk_grad(x, index, values, N, M, K, temperature, tail, lse, rest, dloss, dx):
    """dx[N,M] = gradient of sum(dloss * loss) with respect to x, in x's type; dx may be x (few long rows
    take longer then: one CTA a row), and must not overlap it otherwise. ``lse`` and ``rest`` are what
    ``distill_topk`` wrote for the same arguments; rows where one of them is above 64 (16-bit types: 1024)
    in size are summed again."""


@jit
def gated_scan(g, x, h0, lens, B, T, D, h, last, carry):
    """For every sequence and channel of g, x [B,T,D]: f = sigmoid(g), h[t] = f[t] * h[t-1] + (1 - f[t]) * x[t]
    from the state h0[B,D] (None: zeros), in 32 bits, h rounded once to the type of x. From lens[b]
    (None: T; clamped to [0, T]) on the state is held and h is zero. ``last`` [B,D] (or None) is the final state,
    ``carry`` [B,ceil(T/SCAN_TILE),D] (or None) the states that ``gated_scan_grad`` starts from; both float32,
    as h0; last may be h0. CUDA arrays g, x, h may be strided between sequences and between steps. An infinity or
    NaN makes the later steps of its channel infinite or NaN. Gates below -41.5 (float32: -87) count as that."""


@jit
def gated_scan_grad(g, x, lens, B, T, D, carry, dh, dlast, dg, dx, dh0):
    """dg, dx [B,T,D] and dh0 [B,D] (or None) = gradients of sum(dh * h) + sum(dlast * last); dh or dlast
    may be None. ``carry`` is what ``gated_scan`` wrote for the same inputs. dg and dx are zero from lens[b] on."""


@jit
def gated_step(g, x, state, N, D, h, last):
    """One step for N rows: last = sigmoid(g) * state + (1 - sigmoid(g)) * x in float32 (last may be
    state), h[N,D] the same in the type of x."""
