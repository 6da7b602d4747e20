"""Neural-network compositions: host-side mirror of ops/nn.rs and ops/metric.rs.

With fusion on (the default) softmax, softmax_cross_entropy and layer_norm over the LAST axis become
single graph nodes that the backend runs as one fused row kernel; in every other case — and always
with `var.set_fusion(False)` — they are the reference's compositions of maps and reductions, op for
op.  Both forms are compared against each other and against the CPU oracle by the parity tests.
"""
from collections import namedtuple

import numpy as np

from . import abi
from .shape import Shape, norm_axes
from .tensor import FLOAT, UINT, INT
from .var import Var, fusion_enabled, gt, into_var, part


def relu(x):
    """nn.rs:33-40: float(x > 0) * x."""
    x = into_var(x)
    return gt(x, 0.0).float() * x


def gelu(x):
    """erf-GELU 0.5*x*(1+erf(x/sqrt 2)) from the reference's own maps (UnaryMap::Erf, map.rs:104)."""
    x = into_var(x)
    return (x * 0.5) * ((x / 1.4142135381698608).erf() + 1.0)


def softmax_composed(x, axes):
    """nn.rs:42-56."""
    x = into_var(x)
    axes = norm_axes(axes, x.rank)
    xm = x.max(axes, True)
    y = (x - xm).exp()
    s = y.sum(axes, True)
    return y / s


def softmax(x, axes):
    x = into_var(x)
    axes = norm_axes(axes, x.rank)
    if fusion_enabled() and axes == [x.rank - 1] and x.dtype == FLOAT:
        return Var(Shape(x.extents), FLOAT, "softmax", [x])
    return softmax_composed(x, axes)


def log_sum_exp(x, axes):
    """nn.rs:58-68."""
    x = into_var(x)
    axes = norm_axes(axes, x.rank)
    c = x.max(axes, True)
    return (x - c).exp().sum(axes, True).log() + c


def softmax_cross_entropy_composed(x1, x2):
    """nn.rs:70-82."""
    x1, x2 = into_var(x1), into_var(x2)
    log_z = x1 - log_sum_exp(x1, 1)
    log_p = log_z.gather(x2, 1)
    return -log_p.sum(1, False)


def softmax_cross_entropy(x1, x2):
    x1, x2 = into_var(x1), into_var(x2)
    if (fusion_enabled() and x1.rank == 2 and x2.rank == 2 and x2.extents == [x1.extents[0], 1]
            and x1.dtype == FLOAT and x2.dtype in (UINT, INT)):
        return Var(Shape([x1.extents[0]]), FLOAT, "softmax_ce", [x1, x2])
    return softmax_cross_entropy_composed(x1, x2)


def layer_norm_composed(x, axes, gamma, beta, eps):
    """nn.rs:84-100."""
    x = into_var(x)
    axes = norm_axes(axes, x.rank)
    m = x.mean(axes, True)
    v = x.var(axes, True)
    xc = (x - m) / (v + float(eps)).sqrt()
    return xc * gamma + beta


def layer_norm(x, axes, gamma, beta, eps):
    x, gamma, beta = into_var(x), into_var(gamma), into_var(beta)
    axes = norm_axes(axes, x.rank)
    n = x.extents[-1]
    ok = lambda p: p.size() == 1 or (p.size() == n and p.extents[-1] == n)
    if fusion_enabled() and axes == [x.rank - 1] and x.dtype == FLOAT and ok(gamma) and ok(beta):
        return Var(Shape(x.extents), FLOAT, "layer_norm", [x, gamma, beta], {"eps": float(eps)})
    return layer_norm_composed(x, axes, gamma, beta, eps)


def accuracy(logits, labels):
    """metric.rs:4-16: float(sum_0(argmax_1(logits, keep) == labels)) / B."""
    logits, labels = into_var(logits), into_var(labels)
    hit = logits.argmax(1, True)
    from .var import eq
    return eq(hit, labels).sum(0, False).float() / float(logits.extents[0])


# ----------------------------------------------------------------------------- operators of language models
# These have one kernel each and no composition: they run the same with fusion on and off.
def embedding(table, ids, scale=1.0):
    """scale * table[ids]: [V, E] and ids of rank 1..7 (uint or int) -> ids' extents and E.  An id outside 0..V-1 (-1, say)
    is no token: its row is zero and it adds nothing to the gradient.  Embedding::pass (layers.rs:406-463) gathers
    through an expanded index tensor and its gradient scatters with additions in any order; here the gradient sorts the
    tokens and adds each row's in a fixed order."""
    table, ids = into_var(table), into_var(ids)
    if table.dtype != FLOAT or ids.dtype not in (UINT, INT):
        raise abi.DTypeError(abi.ERR_DTYPE, "embedding: a float table and uint or int ids expected")
    if table.rank != 2 or ids.rank >= abi.MAX_RANK:
        raise abi.ShapeError(abi.ERR_SHAPE, "embedding: a [V, E] table and ids of rank 1..7 expected")
    return Var(Shape(list(ids.extents) + [table.extents[1]]), FLOAT, "embedding", [table, ids], {"scale": float(np.float32(scale))})


TokenLogprobs = namedtuple("TokenLogprobs", "logprob entropy lse top_ids top_logprobs")


def token_logprobs(logits, tokens=None, top=0, scale=1.0):
    """Log probabilities under softmax(scale * logits) over the last axis: of `tokens` (uint or int, the leading extents),
    the entropy, the log of the sum of exponentials and, with top > 0, the `top` most likely indexes with their log
    probabilities, largest first and equal ones by index.  A token outside the vocabulary (-100, say) is no token: its
    log probability is 0 and has no gradient.  logprob and entropy have gradients; the rest is for reading.
    -logprob is softmax_cross_entropy (nn.rs:70-82)."""
    logits = into_var(logits)
    if logits.dtype != FLOAT:
        raise abi.DTypeError(abi.ERR_DTYPE, "token_logprobs: float logits expected")
    lead = list(logits.extents[:-1]) or [1]
    ins = [logits]
    if tokens is not None:
        tokens = into_var(tokens)
        if tokens.dtype not in (UINT, INT):
            raise abi.DTypeError(abi.ERR_DTYPE, "token_logprobs: uint or int tokens expected")
        if list(tokens.extents) != lead:
            raise abi.ShapeError(abi.ERR_SHAPE, f"token_logprobs: tokens {tokens.extents} for logits {logits.extents}")
        ins.append(tokens)
    scale = float(np.float32(scale))
    if not 0.0 < scale <= 2.0 ** 127:
        raise abi.SageError(abi.ERR_ARG, "token_logprobs: scale must be positive and at most 2^127")
    if not 0 <= top <= min(abi.MAX_TOP, logits.extents[-1]):
        raise abi.ShapeError(abi.ERR_SHAPE, f"token_logprobs: {top} alternatives of {logits.extents[-1]} (at most {abi.MAX_TOP})")
    lse = Var(Shape(lead), FLOAT, "token_lse", ins, {"scale": scale, "top": int(top)})
    tail = list(logits.extents[:-1]) + [top]
    return TokenLogprobs(
        Var(Shape(lead), FLOAT, "token_logprob", [logits, lse, tokens]) if tokens is not None else None,
        Var(Shape(lead), FLOAT, "token_entropy", [logits, lse]),
        lse,
        part(lse, "top_ids", tail, UINT) if top else None,
        part(lse, "top_logprobs", tail, FLOAT) if top else None)


def token_logprobs_grad(logits, lse, tokens=None, g_logprob=None, g_entropy=None):
    """The gradient of token_logprobs: the logits', from those of its log probabilities (which need the tokens) and entropies, one
    of them at least.  lse: the node that token_logprobs gave for these logits, which holds the scale and the entropy too.  It
    has no gradient of its own."""
    if lse.op != "token_lse":
        raise abi.SageError(abi.ERR_ARG, "token_logprobs_grad: the lse of token_logprobs expected")
    if g_logprob is None and g_entropy is None:
        raise abi.SageError(abi.ERR_ARG, "token_logprobs_grad: no gradient given")
    if g_logprob is not None and tokens is None:
        raise abi.SageError(abi.ERR_ARG, "token_logprobs_grad: g_logprob needs tokens")
    ins = [logits, lse] + [v for v in (tokens, g_logprob, g_entropy) if v is not None]
    return Var(Shape(logits.extents), FLOAT, "token_logprobs_grad", ins, {"logprob": g_logprob is not None, "entropy": g_entropy is not None})


def cross_attention(q, k, v, mask=None, scale=None):
    """softmax(scale * q . k^T) . v over the keys that `mask` ([N, Lk], 0 = hidden) leaves visible: q [N, H, Lq, D], k and v
    [N, G, Lk, D] with G dividing H (query head h reads key head h / (H/G)), D = 32 or 64, scale 1/sqrt(D) by default.
    A query without a visible key gives zeros; what hidden keys hold is not used.  MultiHeadAttention::pass
    (bert.rs:262-271) with the keys and values of another sequence, and a gradient of its own, which has none in turn."""
    q, k, v = into_var(q), into_var(k), into_var(v)
    ins = [q, k, v]
    if mask is not None:
        ins.append(into_var(mask))
    if any(x.dtype != FLOAT for x in ins):
        raise abi.DTypeError(abi.ERR_DTYPE, "cross_attention: float operands expected")
    if q.rank != 4 or k.rank != 4 or v.extents != k.extents:
        raise abi.ShapeError(abi.ERR_SHAPE, "cross_attention: q [N, H, Lq, D], k and v [N, G, Lk, D] expected")
    n, h, _, d = q.extents
    if k.extents[0] != n or k.extents[3] != d or h % k.extents[1] != 0:
        raise abi.ShapeError(abi.ERR_SHAPE, f"cross_attention: q {q.extents} does not go with k {k.extents}")
    if d not in (32, 64):
        raise abi.ShapeError(abi.ERR_SHAPE, f"cross_attention: head size {d} (32 and 64 are built)")
    if mask is not None and list(ins[3].extents) != [n, k.extents[2]]:
        raise abi.ShapeError(abi.ERR_SHAPE, f"cross_attention: mask {ins[3].extents}, expected {[n, k.extents[2]]}")
    scale = 1.0 / np.sqrt(d) if scale is None else scale
    return Var(Shape(q.extents), FLOAT, "cross_attention", ins, {"scale": float(np.float32(scale))})
