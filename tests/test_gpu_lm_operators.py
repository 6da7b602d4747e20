"""The language-model operators on the GPU, through the C ABI and the front end, against the plain 64-bit implementations
of tests/lm_reference.py with the tolerances derived there."""
import ctypes as C

import numpy as np
import pytest

import sage_amd as S
from sage_amd import abi, bert, nn, optim
from sage_amd import var as V
from sage_amd.grad import grad, grad_param
from sage_amd.layers import Dense, Embedding, Layer
from sage_amd.shape import Shape, default_strides
from sage_amd.tensor import FLOAT, INT, UINT, Buffer, Tensor
from sage_amd.var import Program, Var
from tests import lm_reference as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = S.Context()
    yield c
    c.close()


def say(*a):
    print("[case]", *a, flush=True)


def dev(ctx, a):
    return Tensor.from_numpy(ctx, a)


def strided(ctx, a, pad=3, order=None, offset=0):
    """`a` on the device with its axes in memory order `order` (the last axis stays last) and `pad` further elements behind
    each innermost row, `offset` elements into its buffer; what lies between the elements is NaN."""
    a = np.asarray(a)
    order = list(range(a.ndim)) if order is None else order
    ext = [a.shape[i] for i in order]
    ext[-1] += pad
    st = default_strides(ext)
    host = np.full(int(np.prod(ext)) + offset, np.nan if a.dtype == np.float32 else 7, a.dtype)
    strides = [0] * a.ndim
    for i, ax in enumerate(order):
        strides[ax] = st[i]
    view = np.lib.stride_tricks.as_strided(host[offset:], a.shape, [s * 4 for s in strides])
    view[...] = a
    t = dev(ctx, host)
    return Tensor(t.buf, t.dtype, Shape(list(a.shape), strides, offset))


def ref(t):
    """The argument for a tensor, which lives as long as the argument does."""
    if t is None:
        return None
    c = t.c()
    c.keep = t
    return C.byref(c)


def near(got, want, tol, what):
    got, want, tol = np.asarray(got, np.float64), np.asarray(want, np.float64), np.broadcast_to(np.asarray(tol, np.float64), np.shape(want))
    assert got.shape == want.shape, f"{what}: {got.shape} for {want.shape}"
    assert np.array_equal(np.isnan(got), np.isnan(want)), f"{what}: NaN in other places"
    inf = np.isinf(want)
    assert np.array_equal(np.isinf(got), inf) and np.array_equal(got[inf], want[inf]), f"{what}: infinities differ"
    ok = np.isfinite(want)
    if ok.any():
        off = np.abs(got[ok] - want[ok]) - tol[ok]
        assert off.max() <= 0, f"{what}: {np.abs(got[ok] - want[ok])[off.argmax()]:.3g} off, {tol[ok][off.argmax()]:.3g} allowed"


def same_bits(a, b):
    return np.array_equal(np.ascontiguousarray(a).view(np.uint32), np.ascontiguousarray(b).view(np.uint32))


# ----------------------------------------------------------------------------- embedding
def zipf_ids(rng, n, v):
    return np.minimum(np.exp(rng.random(n) * np.log(v + 1)).astype(np.int64) - 1, v - 1)


@pytest.mark.parametrize("n,v,e", [(1, 1, 1), (1, 5, 768), (7, 3, 64), (64, 1000, 33), (257, 10, 260), (300, 70000, 4), (4096, 500, 96), (5, 100, 2050),
                                   (128, 3, 768), (128, 1000, 24), (127, 40000, 8), (129, 20, 70), (100, 700, 13), (8000, 4000, 12), (3, 6, 17001), (90, 2633, 538)])
def test_embedding_and_gradient(ctx, n, v, e):
    say("embedding", n, v, e)
    rng = np.random.default_rng(n + v + e)
    table, g = R.f32(rng.standard_normal((v, e))), R.f32(rng.standard_normal((n, e)))
    ids = zipf_ids(rng, n, v).astype(np.int32)
    ids[rng.random(n) < 0.1] = -1
    ids[rng.random(n) < 0.05] = v
    t, i = dev(ctx, table), dev(ctx, ids)
    y = nn.embedding(Var.new(t), Var.new(i), 1.7).eval(ctx).numpy()
    assert same_bits(y, R.embedding(table, ids, 1.7))
    out = dev(ctx, np.full((v, e), np.nan, np.float32))
    gd = dev(ctx, g)
    want, tol = R.embedding_grad(g, ids, v, 1.7)
    first = None
    for _ in range(3):
        ctx.check(ctx._lib.sg_embedding_grad(ctx.handle, ref(gd), ref(i), C.c_float(1.7), ref(out)))
        got = out.numpy()
        near(got, want, tol, "gtable")
        assert first is None or same_bits(got, first)  # the same bits every time
        first = got


@pytest.mark.parametrize("n,distinct", [(2048, 1), (5000, 1), (20000, 3), (8193, 2), (70000, 5), (16384, 16384), (140000, 7), (128, 1)])
def test_embedding_gradient_of_long_runs_and_many_tokens(ctx, n, distinct):
    """All tokens on a few rows of a large table, and every token on a row of its own."""
    say("runs", n, distinct)
    rng = np.random.default_rng(n)
    v, e = 300000, 20
    ids = (rng.integers(0, distinct, n) * (v // distinct)).astype(np.uint32)
    if distinct == n:
        ids = rng.permutation(v)[:n].astype(np.uint32)
    g = R.f32(rng.standard_normal((n, e)))
    out = Tensor.uninit(ctx, [v, e])
    ctx.check(ctx._lib.sg_embedding_grad(ctx.handle, ref(dev(ctx, g)), ref(dev(ctx, ids)), C.c_float(0.5), ref(out)))
    want, tol = R.embedding_grad(g, ids, v, 0.5)
    near(out.numpy(), want, tol, "gtable")


@pytest.mark.parametrize("n,v", [(9000, 500), (8193, 511), (20000, 512), (70000, 60000), (30000, 262143), (9000, 262144), (140000, 60000)])
def test_embedding_gradient_of_sorts_over_several_launches(ctx, n, v):
    """One, two and three passes; the second pass counted by the first, or (many tiles) by a launch of its own; a gradient
    with padded rows and permuted axes; the largest ids of their tables, and unknown ones."""
    say("sort", n, v)
    rng = np.random.default_rng(n + v)
    ids = zipf_ids(rng, n, v).astype(np.uint32).reshape(2, n // 2) if n % 2 == 0 else zipf_ids(rng, n, v).astype(np.uint32).reshape(1, n)
    ids[:, ::7] = v - 1
    ids[:, ::11] = rng.integers(0, v, ids[:, ::11].shape)
    ids[:, ::13] = v
    ids[:, ::17] = 0xFFFFFFFF
    g = R.f32(rng.standard_normal((*ids.shape, 8)))
    want, tol = R.embedding_grad(g, ids, v, 1.0)
    for gd in (dev(ctx, g), strided(ctx, g, pad=1, order=[1, 0, 2])):
        out = dev(ctx, np.full((v, 8), np.nan, np.float32))
        ctx.check(ctx._lib.sg_embedding_grad(ctx.handle, ref(gd), ref(dev(ctx, ids)), C.c_float(1.0), ref(out)))
        near(out.numpy(), want, tol, "gtable")


def test_embedding_strided_operands(ctx):
    """Ids of a wider batch (its last position dropped), a broadcast batch, a table and a gradient with padded or permuted rows."""
    rng = np.random.default_rng(3)
    table = R.f32(rng.standard_normal((50, 36)))
    ids = rng.integers(0, 50, (4, 9)).astype(np.uint32)
    whole = dev(ctx, ids)
    cut = Tensor(whole.buf, UINT, Shape([4, 8], [9, 1], 1))
    for tab in (dev(ctx, table), strided(ctx, table, pad=5, offset=1), strided(ctx, table, pad=4)):
        out = Tensor.uninit(ctx, [4, 8, 36])
        ctx.check(ctx._lib.sg_embedding(ctx.handle, ref(tab), ref(cut), C.c_float(0.25), ref(out)))
        assert same_bits(out.numpy(), R.embedding(table, ids[:, 1:], 0.25))
    g = R.f32(rng.standard_normal((4, 8, 36)))
    want, tol = R.embedding_grad(g, ids[:, 1:], 50, 0.25)
    for gd in (dev(ctx, g), strided(ctx, g, pad=1), strided(ctx, g, pad=4, order=[1, 0, 2]), strided(ctx, g, pad=0, order=[1, 0, 2], offset=2)):
        out = Tensor.uninit(ctx, [50, 36])
        ctx.check(ctx._lib.sg_embedding_grad(ctx.handle, ref(gd), ref(cut), C.c_float(0.25), ref(out)))
        near(out.numpy(), want, tol, "gtable")
    one = dev(ctx, g[0, 0])  # a gradient broadcast over all tokens
    out = Tensor.uninit(ctx, [50, 36])
    ctx.check(ctx._lib.sg_embedding_grad(ctx.handle, ref(Tensor(one.buf, FLOAT, Shape([4, 8, 36], [0, 0, 1], 0))), ref(cut), C.c_float(1.0), ref(out)))
    want, tol = R.embedding_grad(np.broadcast_to(g[0, 0], g.shape), ids[:, 1:], 50, 1.0)
    near(out.numpy(), want, tol, "broadcast gradient")
    row = Tensor(whole.buf, UINT, Shape([6, 9], [0, 1], 9))  # one sequence six times
    out = Tensor.uninit(ctx, [6, 9, 36])
    ctx.check(ctx._lib.sg_embedding(ctx.handle, ref(dev(ctx, table)), ref(row), C.c_float(1.0), ref(out)))
    assert same_bits(out.numpy(), R.embedding(table, np.broadcast_to(ids[1], (6, 9)), 1.0))


def test_embedding_of_unknown_tokens_only(ctx):
    ids = dev(ctx, np.full((3, 4), -1, np.int32))
    table = dev(ctx, np.full((5, 8), np.nan, np.float32))
    assert not nn.embedding(Var.new(table), Var.new(ids)).eval(ctx).numpy().any()
    g = Var.new(dev(ctx, np.full((3, 4, 8), np.nan, np.float32)))
    t = Var.new(table)
    assert not grad(nn.embedding(t, Var.new(ids)), [t], seed=g)[0].eval(ctx).numpy().any()


# ----------------------------------------------------------------------------- log probabilities
def run_logprobs(ctx, x, tokens, scale, top=0, shape=None):
    """x: a Tensor or an array [.., C]."""
    x = x if isinstance(x, Tensor) else dev(ctx, x)
    lead = list(x.extents[:-1]) or [1]
    outs = {k: Tensor.from_numpy(ctx, np.full(lead, np.nan, np.float32)) for k in ("logprob", "entropy", "lse")}
    ids = tops = None
    if top:
        ids, tops = Tensor.uninit(ctx, list(x.extents[:-1]) + [top], UINT), Tensor.uninit(ctx, list(x.extents[:-1]) + [top])
    tok = tokens if tokens is None or isinstance(tokens, Tensor) else dev(ctx, tokens)
    ctx.check(ctx._lib.sg_token_logprobs(ctx.handle, ref(x), ref(tok), C.c_float(scale), ref(outs["logprob"]) if tok is not None else None, ref(outs["entropy"]),
                                         ref(outs["lse"]), ref(ids), ref(tops)))
    r = {k: v.numpy() for k, v in outs.items()}
    if top:
        r["top_ids"], r["top_logprobs"] = ids.numpy(), tops.numpy()
    r["dev"] = (x, tok, outs)
    return r


def check_logprobs(ctx, x, tokens, scale, top):
    want = R.logprobs(x, tokens, scale, top)
    got = run_logprobs(ctx, x, tokens, scale, top)
    t_lp, t_h = R.logprobs_tol(x, scale)
    far = np.abs(np.where(np.isfinite(x), x, 0)).max(1) * scale
    near(got["lse"], want["lse"], t_lp + 2 * R.U * far, "lse")
    near(got["entropy"], want["entropy"], t_h, "entropy")
    near(got["logprob"], want["logprob"], t_lp + 2 * R.U * np.abs(np.where(np.isfinite(want["logprob"]), want["logprob"], 0)), "logprob")
    if top:
        assert np.array_equal(got["top_ids"], want["top_ids"])
        near(got["top_logprobs"], want["top_logprobs"], t_lp[:, None] + 2 * R.U * np.abs(np.where(np.isfinite(want["top_logprobs"]), want["top_logprobs"], 0)), "top")
    return want, got


@pytest.mark.parametrize("rows,c,top", [(1, 1, 1), (1, 2, 2), (3, 63, 5), (2, 64, 64), (5, 257, 20), (1, 30522, 5), (4, 50257, 32), (37, 4099, 64), (300, 1000, 1), (2, 131071, 64), (1500, 203, 3)])
@pytest.mark.parametrize("scale", [1.0, 1.7])
def test_token_logprobs(ctx, rows, c, top, scale):
    say("logprobs", rows, c, top, scale)
    rng = np.random.default_rng(rows * c + top)
    x = R.f32(rng.standard_normal((rows, c)) * 3 + rng.standard_normal(c))
    tokens = rng.integers(0, c, rows).astype(np.int32)
    tokens[rng.random(rows) < 0.2] = -100
    check_logprobs(ctx, x, tokens, scale, top)


@pytest.mark.parametrize("c", [40, 1000, 20000])
def test_token_logprobs_of_masked_vocabularies_and_ties(ctx, c):
    """Rows with -inf, with nothing else, with one token left, with equal logits (all, and rising blocks), far from 0, in
    rising and in falling order."""
    say("masked", c)
    rng = np.random.default_rng(c)
    x = R.f32(rng.standard_normal((9, c)))
    x[0, rng.random(c) < 0.9] = -np.inf
    x[1] = -np.inf
    x[2] = -np.inf
    x[2, c - 3] = 4.0
    x[3] = 0.5
    x[4] = np.arange(c) // 7
    x[5] = np.sort(x[5])
    x[6] = np.sort(x[6])[::-1]
    x[7] = x[7] * 50 + 1000
    x[8] = np.where(np.arange(c) % 2, 0.0, -0.0)
    tokens = np.array([0, 5, c - 3, c - 1, 3, 0, 0, 2, c], np.int32)
    want, got = check_logprobs(ctx, x, tokens, 1.0, 32)
    assert got["entropy"][1] == 0 and np.isneginf(got["lse"][1])
    gl, ge = R.f32(rng.standard_normal(9)), R.f32(rng.standard_normal(9))
    xd, tok, outs = got["dev"]
    out = Tensor.uninit(ctx, [9, c])
    ctx.check(ctx._lib.sg_token_logprobs_grad(ctx.handle, ref(xd), ref(tok), C.c_float(1.0), ref(outs["lse"]), ref(outs["entropy"]), ref(dev(ctx, gl)), ref(dev(ctx, ge)), ref(out)))
    near(out.numpy(), R.logprobs_grad(want, 1.0, gl, ge), R.logprobs_grad_tol(want, x, 1.0, gl, ge), "glogits")


@pytest.mark.parametrize("c", [50, 5000, 70001])
def test_token_logprobs_of_nan_and_infinity(ctx, c):
    rng = np.random.default_rng(c)
    x = R.f32(rng.standard_normal((4, c)))
    x[0, c // 2] = np.nan
    x[1, 3] = np.inf
    x[2] = np.nan
    r = run_logprobs(ctx, x, np.array([0, 0, -1, 0], np.int32), 1.0, 8)
    for row in range(3):
        assert np.isnan(r["lse"][row]) and np.isnan(r["entropy"][row]) and np.isnan(r["top_logprobs"][row]).all()
    assert np.isnan(r["logprob"][:2]).all() and r["logprob"][2] == 0
    assert np.array_equal(r["top_ids"][0], np.argsort(-np.where(np.isnan(x[0]), -np.inf, x[0]), kind="stable")[:8])
    assert r["top_ids"][1, 0] == 3 and np.array_equal(r["top_ids"][2], np.arange(8))
    assert np.isfinite(r["lse"][3])


@pytest.mark.parametrize("rows,c", [(1, 1), (3, 64), (5, 257), (2, 30522), (129, 1023)])
def test_token_logprobs_gradient(ctx, rows, c):
    say("logprobs grad", rows, c)
    rng = np.random.default_rng(rows + c)
    x = R.f32(rng.standard_normal((rows, c)) * 2)
    tokens = rng.integers(0, c, rows).astype(np.int32)
    tokens[::3] = -100
    gl, ge = R.f32(rng.standard_normal(rows)), R.f32(rng.standard_normal(rows))
    want, got = check_logprobs(ctx, x, tokens, 0.8, 0)
    xd, tok, outs = got["dev"]
    for a, b in ((gl, ge), (gl, None), (None, ge)):
        out = Tensor.uninit(ctx, [rows, c])
        ctx.check(ctx._lib.sg_token_logprobs_grad(ctx.handle, ref(xd), ref(tok) if a is not None else None, C.c_float(0.8), ref(outs["lse"]),
                                                  ref(outs["entropy"]) if b is not None else None, ref(dev(ctx, a)) if a is not None else None,
                                                  ref(dev(ctx, b)) if b is not None else None, ref(out)))
        near(out.numpy(), R.logprobs_grad(want, 0.8, a, b), R.logprobs_grad_tol(want, x, 0.8, a, b), "glogits")
    # in place, with a gradient broadcast over the rows
    one = dev(ctx, gl[:1])
    ctx.check(ctx._lib.sg_token_logprobs_grad(ctx.handle, ref(xd), ref(tok), C.c_float(0.8), ref(outs["lse"]), None, ref(Tensor(one.buf, FLOAT, Shape([rows], [0], 0))), None, ref(xd)))
    all_same = np.full(rows, gl[0])
    near(xd.numpy(), R.logprobs_grad(want, 0.8, all_same), R.logprobs_grad_tol(want, x, 0.8, all_same), "in place")


@pytest.mark.parametrize("c", [300, 20001])
def test_token_logprobs_of_rows_far_from_zero(ctx, c):
    """A row moved by a constant has the same probabilities and gradients: multiples of 1/64 moved by 2^17 are exact, so the
    tolerance is that of the row that was not moved.  A row of the type's lowest value throughout is uniform."""
    rng = np.random.default_rng(c)
    x = R.f32(np.round(rng.standard_normal((3, c)) * 128) / 64)
    moved = x.copy()
    moved[0] += 2.0 ** 17
    moved[1] -= 2.0 ** 17
    x[2], moved[2] = 0.0, np.finfo(np.float32).min
    tokens = rng.integers(0, c, 3).astype(np.int32)
    gl, ge = R.f32(rng.standard_normal(3)), R.f32(rng.standard_normal(3))
    want, t_lp, t_h = R.logprobs(x, tokens, 1.0), *R.logprobs_tol(x, 1.0)
    got = run_logprobs(ctx, moved, tokens, 1.0, 6)
    near(got["logprob"], want["logprob"], t_lp, "logprob")
    near(got["entropy"], want["entropy"], t_h, "entropy")
    assert np.array_equal(got["top_ids"], R.logprobs(x, None, 1.0, 6)["top_ids"])
    xd, tok, outs = got["dev"]
    out = Tensor.uninit(ctx, [3, c])
    for to in (out, xd):  # beside the logits and in their place
        ctx.check(ctx._lib.sg_token_logprobs_grad(ctx.handle, ref(xd), ref(tok), C.c_float(1.0), ref(outs["lse"]), ref(outs["entropy"]), ref(dev(ctx, gl)), ref(dev(ctx, ge)),
                                                  ref(to)))
        near(to.numpy(), R.logprobs_grad(want, 1.0, gl, ge), R.logprobs_grad_tol(want, x, 1.0, gl, ge), "glogits")


def test_token_logprobs_strided_operands(ctx):
    """[2, 3, C] logits with padded rows at every alignment and permuted leading axes; strided tokens; a rank-1 call."""
    rng = np.random.default_rng(9)
    for c in (100, 1027):
        x = R.f32(rng.standard_normal((2, 3, c)))
        tokens = rng.integers(0, c, (2, 3)).astype(np.int32)
        want = R.logprobs(x.reshape(6, c), tokens.reshape(6), 1.0, 7)
        t_lp, t_h = R.logprobs_tol(x.reshape(6, c), 1.0)
        tok = strided(ctx, tokens, pad=2, order=[0, 1])
        for pad, order, offset in ((0, [0, 1, 2], 1), (1, [0, 1, 2], 0), (2, [1, 0, 2], 3), (4, [1, 0, 2], 0)):
            got = run_logprobs(ctx, strided(ctx, x, pad, order, offset), tok, 1.0, 7)
            near(got["logprob"].reshape(6), want["logprob"], t_lp, "logprob")
            near(got["entropy"].reshape(6), want["entropy"], t_h, "entropy")
            assert np.array_equal(got["top_ids"].reshape(6, 7), want["top_ids"])
    got = run_logprobs(ctx, x[0, 0].copy(), tokens[0, :1].copy(), 1.0, 7)
    near(got["logprob"], want["logprob"][:1], t_lp[:1], "rank 1")
    assert np.array_equal(got["top_ids"], want["top_ids"][0])


# ----------------------------------------------------------------------------- cross attention
def cross_case(rng, n, h, g, lq, lk, d):
    q, k, v, go = (R.f32(rng.standard_normal(s)) for s in ((n, h, lq, d), (n, g, lk, d), (n, g, lk, d), (n, h, lq, d)))
    return q, k, v, go


def run_cross(ctx, q, k, v, mask, scale, go=None, out=None):
    n, h, lq, d = q.extents
    out = Tensor.from_numpy(ctx, np.full(q.extents, np.nan, np.float32)) if out is None else out
    lse = Tensor.uninit(ctx, [n, h, lq])
    ctx.check(ctx._lib.sg_cross_attention(ctx.handle, ref(q), ref(k), ref(v), ref(mask), C.c_float(scale), ref(out), ref(lse)))
    r = {"out": out, "lse": lse}
    if go is not None:
        nan = lambda e: Tensor.from_numpy(ctx, np.full(e, np.nan, np.float32))  # noqa: E731
        r.update(gq=nan(q.extents), gk=nan(k.extents), gv=nan(k.extents))
        ctx.check(ctx._lib.sg_cross_attention_grad(ctx.handle, ref(q), ref(k), ref(v), ref(mask), C.c_float(scale), ref(out), ref(lse), ref(go), ref(r["gq"]),
                                                   ref(r["gk"]), ref(r["gv"])))
    return {key: t.numpy() for key, t in r.items()}


def check_cross(ctx, q, k, v, mask, scale, go, tensors=None):
    t = tensors or [dev(ctx, a) for a in (q, k, v, go)]
    got = run_cross(ctx, *t[:3], None if mask is None else dev(ctx, mask), scale, t[3])
    clean = lambda a: a if mask is None else np.where((np.asarray(mask) != 0)[:, None, :, None], a, np.float32(0))  # noqa: E731
    kc, vc = clean(k), clean(v)
    out, lse, _ = R.cross(q, kc, vc, mask, scale)
    t_out, t_lse = R.cross_tol(q, kc, vc, mask, scale)
    near(got["out"], out, t_out, "out")
    near(got["lse"], lse, t_lse, "lse")
    for name, want, tol in zip(("gq", "gk", "gv"), R.cross_grad(q, kc, vc, mask, scale, go), R.cross_grad_tol(q, kc, vc, mask, scale, go)):
        near(got[name], want, tol, name)
    return got


CROSS = [(1, 1, 1, 1, 1, 32), (1, 1, 1, 1, 1, 64), (2, 3, 3, 5, 7, 64), (1, 2, 1, 33, 65, 32), (3, 4, 2, 1, 200, 64), (2, 12, 12, 1, 513, 64), (2, 8, 2, 31, 130, 32),
         (1, 4, 1, 129, 64, 64), (2, 2, 2, 128, 128, 64), (1, 1, 1, 300, 33, 32), (1, 6, 3, 2, 1000, 32), (1, 1, 1, 3, 3000, 64), (9, 12, 4, 4, 96, 64)]


@pytest.mark.parametrize("n,h,g,lq,lk,d", CROSS)
def test_cross_attention_and_gradient(ctx, n, h, g, lq, lk, d):
    say("cross", n, h, g, lq, lk, d)
    rng = np.random.default_rng(n + h + lq + lk)
    q, k, v, go = cross_case(rng, n, h, g, lq, lk, d)
    check_cross(ctx, q, k, v, None, 1 / np.sqrt(d), go)


@pytest.mark.parametrize("n,h,g,lq,lk,d", [(4, 4, 2, 9, 150, 64), (4, 2, 2, 1, 700, 32), (5, 6, 2, 70, 257, 32), (4, 3, 1, 130, 128, 64), (3, 1, 1, 2, 64, 64)])
def test_cross_attention_masks(ctx, n, h, g, lq, lk, d):
    """Lengths, holes, a single visible key, an empty row; hidden keys hold NaN and infinities."""
    say("masks", n, h, g, lq, lk, d)
    rng = np.random.default_rng(lk)
    q, k, v, go = cross_case(rng, n, h, g, lq, lk, d)
    mask = np.zeros((n, lk), np.float32)
    mask[0, :lk // 2 + 1] = 1.0
    mask[1] = np.where(rng.random(lk) < 0.4, -2.5, 0.0)  # anything but 0 is visible
    if n > 3:
        mask[3, lk - 1] = 1e-30
    hidden = np.broadcast_to((mask == 0)[:, None, :, None], k.shape)
    k[hidden], v[hidden] = np.nan, np.inf
    got = check_cross(ctx, q, k, v, mask, 0.2, go)
    assert not got["out"][2].any() and np.isneginf(got["lse"][2]).all() and not got["gq"][2].any() and not got["gk"][2].any() and not got["gv"][2].any()
    again = run_cross(ctx, *[dev(ctx, a) for a in (q, k, v)], dev(ctx, mask), 0.2, dev(ctx, go))
    assert all(same_bits(got[x], again[x]) for x in got)


# More workgroups than the chip holds (the longest sequences first; more than 256 sequences), walks split over workgroups, every
# number of wavefronts side by side, few rows over many keys.
@pytest.mark.parametrize("n,h,g,lq,lk,d,masked", [
    (24, 12, 12, 70, 96, 32, True), (24, 12, 12, 70, 96, 64, True), (300, 2, 1, 40, 50, 32, True), (40, 8, 4, 200, 130, 64, True), (24, 12, 12, 96, 128, 64, False),
    (5, 4, 4, 9, 2000, 64, True), (8, 16, 4, 100, 200, 32, False), (9, 12, 12, 512, 33, 64, True), (1, 1, 1, 2000, 2000, 64, False), (1, 1, 1, 2000, 2000, 32, True),
    (22, 12, 12, 250, 40, 32, True), (4, 2, 2, 200, 31, 32, True), (40, 12, 12, 97, 100, 32, True), (3, 2, 2, 700, 300, 32, False), (2, 2, 2, 1, 7000, 32, False), (2, 4, 2, 2, 5000, 64, True), (2, 8, 1, 1, 3000, 64, True),
    (300, 1, 1, 8, 70, 32, True), (1, 2, 1, 1, 4000, 32, True), (2, 3, 1, 1, 900, 32, True), (1, 4, 2, 1, 600, 64, True),
    (32, 12, 12, 352, 70, 64, True), (32, 12, 12, 352, 140, 64, False), (44, 12, 12, 520, 40, 32, True), (6, 4, 2, 30, 700, 64, True), (7, 8, 2, 60, 300, 32, True)])
def test_cross_attention_of_many_and_of_long_sequences(ctx, n, h, g, lq, lk, d, masked):
    """Against the formula; rows that begin at any element give the bits that aligned ones give."""
    say("paths", n, h, g, lq, lk, d, masked)
    rng = np.random.default_rng(n * lq + lk)
    q, k, v, go = cross_case(rng, n, h, g, lq, lk, d)
    mask = None
    if masked:
        lengths = rng.integers(0, lk + 1, n)
        lengths[:1] = lk
        mask = R.f32((np.arange(lk)[None] < lengths[:, None]) & (rng.random((n, lk)) < 0.9))
    got = check_cross(ctx, q, k, v, mask, 1 / np.sqrt(d), go)
    m = None if mask is None else strided(ctx, mask, pad=1, offset=1)
    again = run_cross(ctx, *[strided(ctx, a, pad=1, offset=1) for a in (q, k, v)], m, 1 / np.sqrt(d), strided(ctx, go, pad=3, offset=2))
    for name in got:
        assert same_bits(got[name], again[name]), name


def test_cross_attention_large_scores_do_not_overflow(ctx):
    rng = np.random.default_rng(5)
    q, k, v, go = cross_case(rng, 1, 2, 2, 40, 300, 64)
    check_cross(ctx, q * 30, k, v, None, 1.0, go)
    check_cross(ctx, q, k - 100 * q[:, :, :1], v, None, 1.0, go)  # all scores far below 0
    check_cross(ctx, q, k, v, None, -0.5, go)


@pytest.mark.parametrize("d", [32, 64])
def test_cross_attention_layouts(ctx, d):
    """Heads side by side, padded and unaligned rows, broadcast keys, gradients and masks, outputs in the merged layout."""
    rng = np.random.default_rng(d)
    n, h, g, lq, lk = 2, 4, 2, 37, 70
    q, k, v, go = cross_case(rng, n, h, g, lq, lk, d)
    for pad, order, offset in ((0, [0, 2, 1, 3], 0), (1, [0, 2, 1, 3], 0), (4, [0, 1, 2, 3], 4), (3, [2, 0, 1, 3], 1)):
        check_cross(ctx, q, k, v, None, 0.3, go, [strided(ctx, a, pad, order, offset) for a in (q, k, v, go)])
    kb = np.broadcast_to(k[:1, :1], k.shape)
    t = dev(ctx, k[0, 0])
    shared = Tensor(t.buf, FLOAT, Shape([n, g, lk, d], [0, 0, d, 1], 0))
    gt = dev(ctx, go[0, 0, 0])
    check_cross(ctx, q, kb, kb, None, 0.3, np.broadcast_to(go[0, 0, 0], go.shape), [dev(ctx, q), shared, shared, Tensor(gt.buf, FLOAT, Shape([n, h, lq, d], [0, 0, 0, 1], 0))])
    # one mask for the whole batch; outputs with heads side by side leave what lies between rows alone
    mask = dev(ctx, np.where(rng.random(lk) < 0.5, 1.0, 0.0).astype(np.float32))
    m = Tensor(mask.buf, FLOAT, Shape([n, lk], [0, 1], 0))
    wide = dev(ctx, np.full((n, lq, h, d + 4), 7.0, np.float32))
    view = Tensor(wide.buf, FLOAT, Shape([n, h, lq, d], [lq * h * (d + 4), d + 4, h * (d + 4), 1], 0))
    got = run_cross(ctx, dev(ctx, q), dev(ctx, k), dev(ctx, v), m, 0.3, out=view)["out"]
    mm = np.broadcast_to(mask.numpy(), (n, lk))
    near(got, R.cross(q, k, v, mm, 0.3)[0], R.cross_tol(q, k, v, mm, 0.3)[0], "merged out")
    assert (wide.numpy()[..., d:] == 7.0).all()


# ----------------------------------------------------------------------------- AdamW
SIZES = [1, 3, 255, 256, 257, 1000, 4096, 4097, 10000]


def adamw_arrays(ctx, xs):
    arr = (abi.sg_tensor * len(xs))(*[x.c() for x in xs])
    arr.keep = xs
    return arr


HYPER = (1e-2, 0.9, 0.999, 1e-8, 0.1)


def hyper():
    lr, b1, b2, eps, wd = HYPER
    return abi.sg_adam_hyper(lr, b1, b2, float(np.float32(1) - np.float32(b1)), float(np.float32(1) - np.float32(b2)), eps, wd)


def test_adamw_32_bit_states(ctx):
    """150 tensors (three launches), some unaligned: the moments bit for bit, three steps."""
    say("adamw 32")
    rng = np.random.default_rng(0)
    sizes = (SIZES * 17)[:150]
    value, m, v = ([R.f32(rng.standard_normal(n)) for n in sizes] for _ in range(3))
    v = [np.abs(x) for x in v]
    up = lambda xs: [strided(ctx, x, 0, None, i % 3) for i, x in enumerate(xs)]  # noqa: E731
    dv, dm, ds = up(value), up(m), up(v)
    for t in (1, 2, 3):
        g = [R.f32(rng.standard_normal(n)) for n in sizes]
        dg = up(g)
        h = hyper()
        ctx.check(ctx._lib.sg_adamw_update(ctx.handle, len(sizes), *[adamw_arrays(ctx, x) for x in (dv, dg, dm, ds)], None, None, ref(dev(ctx, R.f32([t]))), C.byref(h), 0))
        for i in range(len(sizes)):
            m[i], v[i] = R.adamw_moments(m[i], v[i], g[i], 0.9, 0.999)
            assert same_bits(dm[i].numpy(), m[i]) and same_bits(ds[i].numpy(), v[i]), (t, i)
            want, tol = R.adamw_value(value[i], m[i], v[i], t, *HYPER)
            value[i] = dv[i].numpy()
            near(value[i], want, tol, f"value {i}")


@pytest.mark.parametrize("far", [0, 1])
def test_adamw_8_bit_states(ctx, far):
    """Bytes and scales exactly as defined, over 20 steps from zero states; far: gradients over many octaves, blocks of zeros."""
    say("adamw 8", far)
    rng = np.random.default_rng(1)
    sizes = SIZES * 8  # 72 tensors: two launches
    value = [R.f32(rng.standard_normal(n)) for n in sizes]
    codes = [[np.zeros(n, np.uint8) for n in sizes] for _ in range(2)]
    scales = [[np.zeros(-(-n // 256), np.float32) for n in sizes] for _ in range(2)]
    dv = [strided(ctx, x, 0, None, i % 3) for i, x in enumerate(value)]
    dm, ds = ([dev(ctx, R.pack(c)) for c in cs] for cs in codes)
    dms, dss = ([dev(ctx, s) for s in sc] for sc in scales)
    for t in range(1, 21):
        g = [R.f32(rng.standard_normal(n) * (np.exp(12 * rng.standard_normal(n)) if far else 1.0)) for n in sizes]
        if far:
            g[4][:256] = 0.0
            g[5][::2] = 0.0
        h = hyper()
        ctx.check(ctx._lib.sg_adamw_update(ctx.handle, len(sizes), *[adamw_arrays(ctx, x) for x in (dv, [dev(ctx, x) for x in g], dm, ds, dms, dss)],
                                           ref(dev(ctx, R.f32([t]))), C.byref(h), 77))
        for i, n in enumerate(sizes):
            m, v = R.adamw_moments(R.decode(codes[0][i], scales[0][i], True), R.decode(codes[1][i], scales[1][i], False), g[i], 0.9, 0.999)
            want, tol = R.adamw_value(value[i], m, v, t, *HYPER)
            value[i] = dv[i].numpy()
            near(value[i], want, tol, f"value {i} step {t}")
            nm, nv = R.noise(n, t, 77)
            codes[0][i], scales[0][i] = R.encode(m, True, nm)
            codes[1][i], scales[1][i] = R.encode(v, False, nv)
            if t in (1, 2, 7, 20):
                assert np.array_equal(dm[i].numpy(), R.pack(codes[0][i])) and np.array_equal(ds[i].numpy(), R.pack(codes[1][i])), (t, i)
                assert same_bits(dms[i].numpy(), scales[0][i]) and same_bits(dss[i].numpy(), scales[1][i]), (t, i)
    outs = [[Tensor.uninit(ctx, [n]) for n in sizes] for _ in range(2)]
    ctx.check(ctx._lib.sg_adamw_state_read(ctx.handle, len(sizes), *[adamw_arrays(ctx, x) for x in (dm, ds, dms, dss, *outs)]))
    for i in range(len(sizes)):
        assert same_bits(outs[0][i].numpy(), R.decode(codes[0][i], scales[0][i], True)) and same_bits(outs[1][i].numpy(), R.decode(codes[1][i], scales[1][i], False))


def test_adamw_not_finite_gradient_spoils_its_own_only(ctx):
    n = 600
    g = np.ones(n, np.float32)
    g[300], g[10] = np.inf, np.nan
    for bits in (32, 8):
        p = Var.new(dev(ctx, np.ones(n, np.float32)))
        opt = optim.AdamW(1e-2, state_bits=bits)
        opt.update({p: Var.new(dev(ctx, g))}, ctx)
        m, v = (x.numpy() for x in opt.state(p, ctx))
        bad = ~np.isfinite(p.value.numpy())
        assert bad[10] and bad[300] and bad.sum() == 2
        spoilt = ~np.isfinite(m)
        assert spoilt.sum() == (2 if bits == 32 else 512) and not spoilt[512:].any() and np.isnan(v[10])


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_optimizer_eager_compiled_and_captured(ctx, bits):
    """update(), a compiled program and its replayed graph take the same steps, bit for bit."""
    rng = np.random.default_rng(2)
    shapes = [(33, 7), (256,), (1,), (64, 65)]
    start = [R.f32(rng.standard_normal(s)) for s in shapes]
    steps = [[R.f32(rng.standard_normal(s)) for s in shapes] for _ in range(6)]

    def fresh():
        params = [Var.new(dev(ctx, a.copy())) for a in start]
        grads = [Var.new(dev(ctx, a)) for a in steps[0]]
        return params, grads, optim.AdamW(1e-2, state_bits=bits, seed=5)

    p1, g1, o1 = fresh()
    for s in steps:
        for gv, a in zip(g1, s):
            gv.value.copy_from_numpy(a)
        o1.update(dict(zip(p1, g1)), ctx)
    p2, g2, o2 = fresh()
    prog = o2.compile(dict(zip(p2, g2)), ctx)  # the first step
    for i, s in enumerate(steps[1:]):
        for gv, a in zip(g2, s):
            gv.value.copy_from_numpy(a)
        if i == 2:
            prog.capture()
        prog.run()
        ctx.sync()
    for a, b in zip(p1, p2):
        assert same_bits(a.value.numpy(), b.value.numpy())
        for x, y in zip(o1.state(a, ctx), o2.state(b, ctx)):
            assert list(x.extents) == list(a.extents) and same_bits(x.numpy(), y.numpy())
    prog.release_graph()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("count", [63, 64, 65, 72, 73, 100, 101, 230])
def test_adamw_of_many_tensors(ctx, bits, count):
    """As many as a launch's table holds, one more, several launches: each tensor gets the step it gets alone, whatever its place
    (the noise of 8-bit states depends on the element, not on the tensor)."""
    say("adamw tensors", bits, count)
    rng = np.random.default_rng(count)
    sizes = [int(n) for n in rng.choice([1, 5, 64, 300, 4096, 4097, 9000], count)]
    one = {}
    for n in set(sizes):
        a, g = R.f32(np.cos(np.arange(n))), R.f32(np.sin(np.arange(n)))
        p, opt = Var.new(dev(ctx, a)), optim.AdamW(1e-2, state_bits=bits)
        opt.update({p: Var.new(dev(ctx, g))}, ctx)
        one[n] = a, g, p.value.numpy(), [x.numpy() for x in opt.state(p, ctx)]
    params = [Var.new(dev(ctx, one[n][0])) for n in sizes]
    opt = optim.AdamW(1e-2, state_bits=bits)
    opt.update({p: Var.new(dev(ctx, one[n][1])) for p, n in zip(params, sizes)}, ctx)
    for p, n in zip(params, sizes):
        assert same_bits(p.value.numpy(), one[n][2])
        for x, y in zip(opt.state(p, ctx), one[n][3]):
            assert same_bits(x.numpy(), y)


def test_adamw_takes_strided_gradients_and_a_broadcast_one(ctx):
    rng = np.random.default_rng(4)
    a, g = R.f32(rng.standard_normal((6, 10))), R.f32(rng.standard_normal((10, 6)))
    p, q = Var.new(dev(ctx, a)), Var.new(dev(ctx, a))
    gt = dev(ctx, g)
    turned = Var.new(Tensor(gt.buf, FLOAT, Shape([6, 10], [1, 6], 0)))
    o1, o2 = optim.AdamW(1e-2), optim.AdamW(1e-2)
    for _ in range(2):
        o1.update({p: turned}, ctx)
        o2.update({q: Var.new(dev(ctx, g.T.copy()))}, ctx)
    assert same_bits(p.value.numpy(), q.value.numpy())
    r = Var.new(dev(ctx, a))
    prog = optim.AdamW(1e-2).compile({r: turned}, ctx)
    prog.run()
    assert same_bits(p.value.numpy(), r.value.numpy())
    with pytest.raises(abi.ShapeError):
        o1.update({p: Var.new(gt)}, ctx)


# ----------------------------------------------------------------------------- together
class Reader(Layer):
    """Tokens that attend to an encoder's states and predict the next token: the operators as a training step uses them."""

    def __init__(self, vocab, dim, heads, kv_heads, state_bits):
        self.embedding = Embedding(vocab, dim, scale=np.sqrt(dim))
        self.cross = bert.CrossAttention(dim, heads, num_kv_heads=kv_heads)
        self.head = Dense(dim, vocab)
        self.opt = optim.AdamW(1e-3, state_bits=state_bits)

    def params(self):
        return self.embedding.params() + self.cross.params() + self.head.params()

    def pass_(self, ids, states, mask):
        return self.head.pass_(self.cross.pass_(self.embedding.pass_(ids), states, mask))


def reader_in_64_bits(arrays, ids, states, mask, targets, heads, kv):
    """The same step with torch's float64 autograd: the loss and the gradients of every parameter."""
    import torch
    ps = [torch.tensor(np.asarray(a, np.float64), requires_grad=True) for a in arrays]
    emb, wq, bq, wk, bk, wv, bv, wo, bo, ga, be, wh, bh = ps
    n, l = ids.shape
    e = emb.shape[1]
    d = e // heads
    known = torch.tensor(ids >= 0)
    x = emb[torch.tensor(np.where(ids >= 0, ids, 0)).long()] * float(np.float32(np.sqrt(e))) * known[..., None]
    st = torch.tensor(states.astype(np.float64))
    q = (x @ wq + bq).view(n, l, heads, d).transpose(1, 2)
    k = (st @ wk + bk).view(n, -1, kv, d).transpose(1, 2).repeat_interleave(heads // kv, 1)
    v = (st @ wv + bv).view(n, -1, kv, d).transpose(1, 2).repeat_interleave(heads // kv, 1)
    s = (q @ k.transpose(2, 3)) / np.sqrt(d)
    s = s.masked_fill(torch.tensor(mask == 0)[:, None, None, :], -1e300)
    a = (torch.softmax(s, 3) @ v).transpose(1, 2).reshape(n, l, e) * torch.tensor((mask != 0).any(1)).double()[:, None, None]
    y = a @ wo + bo + x
    mu, var = y.mean(2, keepdim=True), (y ** 2).mean(2, keepdim=True) - y.mean(2, keepdim=True) ** 2
    z = ((y - mu) / (var + 1e-5).sqrt() * ga + be) @ wh + bh
    lp = torch.log_softmax(z, 2)
    ok = torch.tensor(targets >= 0)
    chosen = torch.where(ok, lp.gather(2, torch.tensor(np.where(targets >= 0, targets, 0)).long()[..., None])[..., 0], torch.zeros((), dtype=torch.float64))
    h = -(lp.exp() * lp).sum(2)
    loss = (-chosen - 0.01 * h).sum()
    loss.backward()
    return float(loss.detach()), [p.grad.numpy() for p in ps]


@pytest.mark.parametrize("bits", [32, 8])
def test_a_training_step_of_all_operators(ctx, bits):
    """Embedding, cross attention, log probabilities and AdamW as one program: gradients against float64 autograd, then the
    compiled and captured step with eager work between the replays against the eager one."""
    rng = np.random.default_rng(7)
    vocab, dim, heads, kv, n, l, lk = 211, 128, 4, 2, 3, 9, 21
    model = Reader(vocab, dim, heads, kv, bits)
    arrays = [R.f32(rng.standard_normal(p.extents) * (1.0 if i == 0 else 0.1)) for i, p in enumerate(model.params())]
    ids = rng.integers(0, vocab, (n, l)).astype(np.int32)
    ids[0, -3:] = -1
    targets = rng.integers(0, vocab, (n, l)).astype(np.int32)
    targets[0, -3:] = -100
    mask = np.ones((n, lk), np.float32)
    mask[1, 10:], mask[2] = 0.0, 0.0
    states = R.f32(rng.standard_normal((n, lk, dim)))

    def build():
        for p, a in zip(model.params(), arrays):
            p.set(dev(ctx, a))
        model.opt = optim.AdamW(1e-3, state_bits=bits)
        r = nn.token_logprobs(model.pass_(Var.new(dev(ctx, ids)), Var.new(dev(ctx, states)), Var.new(dev(ctx, mask))), Var.new(dev(ctx, targets)), top=3)
        loss = (-r.logprob - r.entropy * 0.01).sum([0, 1], False)
        return r, loss, grad_param(loss, model)

    r, loss, grads = build()
    want_loss, want = reader_in_64_bits(arrays, ids, states, mask, targets, heads, kv)
    prog = Program(ctx, [loss, r.top_ids] + list(grads.values())).bind()
    # products of length 128 to 211 and sums of at most 27 rows behind one another: 1e-4 of the largest element, as for models
    assert abs(float(loss.value.numpy()[0]) - want_loss) < 1e-4 * abs(want_loss)
    for i, (g, w, p) in enumerate(zip(grads.values(), want, model.params())):
        # a constant added to every key moves no probability, so the key bias's gradient is a sum that cancels to 0: its
        # terms are the key weight's without the factors of unit size that the states are, and so is what rounding leaves
        size = np.abs(want[i - 1] if p is model.cross.key_proj.bias else w).max()
        near(g.value.numpy(), w.reshape(g.extents), 1e-4 * size + 1e-12, p.label)
    assert r.top_ids.value.extents == [n, l, 3]
    step = model.opt.compile(grads, ctx)
    for _ in range(3):
        prog.run()
        step.run()
    eager = [p.value.numpy() for p in model.params()]
    r, loss, grads = build()
    prog = Program(ctx, [loss] + list(grads.values())).bind()
    step = model.opt.compile(grads, ctx)
    prog.capture()
    step.capture()
    for _ in range(3):
        prog.run()
        nn.softmax(Var.new(dev(ctx, states)), [2]).eval(ctx)  # other work of the program in between
        ctx.sync()
        step.run()
    # the sums of the composed parts (LayerNorm's gradient among them) are the same launches, so the bits are too
    for a, p in zip(eager, model.params()):
        assert same_bits(a, p.value.numpy()), p.label
    prog.release_graph()
    step.release_graph()


def test_two_captured_programs_and_an_eager_call_keep_their_workspaces_apart(ctx):
    """Two graphs of the calls that use workspaces, replayed in turn with eager calls of other sizes between them."""
    rng = np.random.default_rng(8)

    def program(n, v, seed):
        rr = np.random.default_rng(seed)
        ids, g = zipf_ids(rr, n, v).astype(np.uint32), R.f32(rr.standard_normal((n, 40)))
        q, k, vv, _ = cross_case(rr, 1, 2, 2, 1, 900 + n, 64)
        x = R.f32(rr.standard_normal((2, 40000)))
        table = Var.empty([v, 40])
        seedv = Var.new(dev(ctx, g))
        ge = Var(Shape([v, 40]), FLOAT, "embedding_grad", [seedv, Var.new(dev(ctx, ids))], {"scale": 1.0})
        at = nn.cross_attention(*[Var.new(dev(ctx, a)) for a in (q, k, vv)])
        lp = nn.token_logprobs(Var.new(dev(ctx, x)), top=9)
        prog = Program(ctx, [ge, at, lp.top_ids, lp.entropy])
        return prog, [o.numpy() for o in prog.outputs], (table,)

    p1, w1, _ = program(700, 90, 1)
    p2, w2, _ = program(9000, 1000, 2)
    p1.capture()
    p2.capture()
    for _ in range(3):
        for p, w in ((p1, w1), (p2, w2)):
            p.run()
            nn.cross_attention(*[Var.new(dev(ctx, R.f32(rng.standard_normal((1, 3, s, 32))))) for s in (1, 2000, 2000)]).eval(ctx)
            ctx.sync()
            for o, a in zip(p.outputs, w):
                assert same_bits(o.numpy(), a)
    p1.release_graph()
    p2.release_graph()


def test_serving_steps_reuse_the_states_keys(ctx):
    """Token by token against the whole sequence at once: each query attends on its own."""
    rng = np.random.default_rng(11)
    layer = bert.CrossAttention(128, 2, num_kv_heads=1)
    for p in layer.params():
        p.set(dev(ctx, R.f32(rng.standard_normal(p.extents) * 0.1)))
    x, states = R.f32(rng.standard_normal((2, 4, 128))), R.f32(rng.standard_normal((2, 300, 128)))
    mask = np.ones((2, 300), np.float32)
    mask[1, 200:] = 0.0
    m = Var.new(dev(ctx, mask))
    whole = layer.pass_(Var.new(dev(ctx, x)), Var.new(dev(ctx, states)), m).eval(ctx).numpy()
    k, v = (Var.new(t.eval(ctx)) for t in layer.keys_values(Var.new(dev(ctx, states))))
    for i in range(4):
        one = layer.attend(Var.new(dev(ctx, x[:, i:i + 1])), k, v, m).eval(ctx).numpy()
        # two different splits of the same sums behind products of length 128: 1e-4 of the layer's unit variance
        near(one[:, 0], whole[:, i], 1e-4, "token")

def test_out_of_memory_is_reported_and_harmless(ctx):
    c = S.Context(capacity=1 << 20)
    rng = np.random.default_rng(12)
    ids, g, out = dev(c, rng.integers(0, 50, 3000).astype(np.uint32)), dev(c, R.f32(rng.standard_normal((3000, 64)))), dev(c, np.zeros((50, 64), np.float32))
    hold = Tensor.uninit(c, [(c.mem_stats()["capacity"] - c.mem_stats()["used"]) // 4 - 16])
    with pytest.raises(abi.OutOfMemory):
        c.check(c._lib.sg_embedding_grad(c.handle, ref(g), ref(ids), C.c_float(1.0), ref(out)))
    del hold
    c.check(c._lib.sg_embedding_grad(c.handle, ref(g), ref(ids), C.c_float(1.0), ref(out)))
    want, tol = R.embedding_grad(g.numpy(), ids.numpy(), 50, 1.0)
    near(out.numpy(), want, tol, "gtable")
    del ids, g, out
    c.close()


def test_rows_beyond_two_to_the_31_elements(ctx):
    """Rows 2^24 + 4 elements apart in one buffer of 8.7 GB: the last ones begin behind element 2^31."""
    rows, stride = 130, (1 << 24) + 4
    assert (rows - 1) * stride > 1 << 31
    buf = Buffer(ctx, ((rows - 1) * stride + 4096) * 4)

    def view(offset, extents):
        return Tensor(buf, FLOAT, Shape(extents, [0] * (len(extents) - 2) + [stride, 1], offset))

    def far(a, offset, extents=None):
        for i, row in enumerate(a):
            ctx.check(ctx._lib.sg_memcpy_h2d(ctx.handle, C.c_void_p(buf.ptr + (i * stride + offset) * 4), row.ctypes.data_as(C.c_void_p), row.nbytes))
        return view(offset, extents or list(a.shape))

    def back(offset, cols):
        out = np.empty((rows, cols), np.float32)
        for i in range(rows):
            ctx.check(ctx._lib.sg_memcpy_d2h(ctx.handle, out[i].ctypes.data_as(C.c_void_p), C.c_void_p(buf.ptr + (i * stride + offset) * 4), cols * 4))
        return out

    rng = np.random.default_rng(21)
    for lq, d in ((40, 64), (1, 64), (50, 32)):
        say("far cross", lq, d)
        q, k, v, go = cross_case(rng, 1, 1, 1, lq, rows, d)
        kf, vf = (far(x[0, 0], o, [1, 1, rows, d]) for x, o in ((k, 0), (v, 64)))
        out, lse, gq = Tensor.uninit(ctx, [1, 1, lq, d]), Tensor.uninit(ctx, [1, 1, lq]), Tensor.uninit(ctx, [1, 1, lq, d])
        qd, god = dev(ctx, q), dev(ctx, go)
        ctx.check(ctx._lib.sg_cross_attention(ctx.handle, ref(qd), ref(kf), ref(vf), None, C.c_float(0.1), ref(out), ref(lse)))
        near(out.numpy(), R.cross(q, k, v, None, 0.1)[0], R.cross_tol(q, k, v, None, 0.1)[0], "out")
        ctx.check(ctx._lib.sg_cross_attention_grad(ctx.handle, ref(qd), ref(kf), ref(vf), None, C.c_float(0.1), ref(out), ref(lse), ref(god), ref(gq),
                                                   ref(view(128, [1, 1, rows, d])), ref(view(192, [1, 1, rows, d]))))
        want, tol = R.cross_grad(q, k, v, None, 0.1, go), R.cross_grad_tol(q, k, v, None, 0.1, go)
        for got, w, t, name in zip((gq.numpy()[0, 0], back(128, d), back(192, d)), want, tol, ("gq", "gk", "gv")):
            near(got, w[0, 0], np.broadcast_to(t, w.shape)[0, 0], name)
    say("far embedding")
    table, ids = R.f32(rng.standard_normal((rows, 60))), rng.permutation(rows).astype(np.uint32)
    out = Tensor.uninit(ctx, [rows, 60])
    ctx.check(ctx._lib.sg_embedding(ctx.handle, ref(far(table, 256)), ref(dev(ctx, ids)), C.c_float(2.0), ref(out)))
    assert same_bits(out.numpy(), R.embedding(table, ids, 2.0))
    ctx.check(ctx._lib.sg_embedding_grad(ctx.handle, ref(view(256, [rows, 60])), ref(dev(ctx, ids)), C.c_float(2.0), ref(out)))
    want, tol = R.embedding_grad(table, ids, rows, 2.0)
    near(out.numpy(), want, tol, "gtable")
    say("far logprobs")
    x, tokens = R.f32(rng.standard_normal((rows, 1001))), rng.integers(0, 1001, rows).astype(np.int32)
    got = run_logprobs(ctx, far(x, 512), tokens, 1.0, 3)
    want = R.logprobs(x, tokens, 1.0, 3)
    near(got["logprob"], want["logprob"], R.logprobs_tol(x, 1.0)[0], "logprob")
    assert np.array_equal(got["top_ids"], want["top_ids"])


def test_captured_in_a_caching_context_beside_another_context(ctx):
    """A graph whose workspaces come from the chunks of a caching allocator keeps them while eager calls of this context and of
    another one, on a stream of its own, take and give back workspaces."""
    c = S.Context(use_cache=True)
    rng = np.random.default_rng(31)

    def calls(where, n, lk):
        ids, g = zipf_ids(rng, n, 400).astype(np.uint32), R.f32(rng.standard_normal((n, 24)))
        q, k, v, go = cross_case(rng, 2, 2, 1, 20, lk, 32)
        mask = R.f32(np.arange(lk)[None] < np.array([[lk], [lk // 3]]))
        x = R.f32(rng.standard_normal((3, 30000)))
        new = lambda a: Var.new(dev(where, a))  # noqa: E731
        vs = [new(a) for a in (q, k, v)]
        at = nn.cross_attention(*vs, new(mask))
        lp = nn.token_logprobs(new(x), top=5)
        return Program(where, [Var(Shape([400, 24]), FLOAT, "embedding_grad", [new(g), new(ids)], {"scale": 1.0}), at,
                               *grad(at, vs, seed=new(go)), lp.top_ids, lp.entropy])
    prog = calls(c, 9000, 1500)
    want = [o.numpy() for o in prog.outputs]
    other = calls(ctx, 3000, 700)
    other_want = [o.numpy() for o in other.outputs]
    prog.capture()
    for i in range(3):
        prog.run()
        other.run()
        again = calls(c, 1000 + 3000 * i, 200 + 600 * i)
        del again
        c.sync()
        ctx.sync()
        for p, w in ((prog, want), (other, other_want)):
            for o, a in zip(p.outputs, w):
                assert same_bits(o.numpy(), a)
    prog.release_graph()
    del prog
    c.close()


def test_a_copy_of_bound_outputs_is_a_snapshot(ctx):
    """The transposed output and gradients of a bound program, copied: later runs of the program, and writes into one of two
    targets, leave the copies alone."""
    rng = np.random.default_rng(41)
    q, k, v, go = cross_case(rng, 2, 4, 2, 6, 30, 32)
    vs = [Var.new(dev(ctx, a)) for a in (q, k, v)]
    y = nn.cross_attention(*vs)
    nodes = [y, *grad(y, vs, seed=Var.new(dev(ctx, go)))]
    prog = Program(ctx, nodes).bind()
    copies = [x.transpose(2, 1).copy().eval(ctx) for x in nodes]
    first = [c.numpy() for c in copies]
    for c, x in zip(first, nodes):
        assert same_bits(c, x.value.numpy().transpose(0, 2, 1, 3))
    for t, a in zip(vs, (q, k, v)):
        t.value.copy_from_numpy(a * np.float32(0.5))
    prog.run()
    for c, a, x in zip(copies, first, nodes):
        assert same_bits(c.numpy(), a) and not same_bits(a, x.value.numpy().transpose(0, 2, 1, 3))
    out = nn.cross_attention(*vs)
    one, two = V.evaluate(ctx, [out, out.transpose(2, 1).copy()])
    kept = one.numpy()
    two.copy_from_numpy(np.zeros(two.extents, np.float32))
    assert same_bits(one.numpy(), kept) and kept.any()


@pytest.mark.parametrize("c", [50, 9001, 30522])
@pytest.mark.parametrize("scale", [1.0, 1.4])
def test_token_logprobs_gradient_of_tokens_hidden_by_the_lowest_value(ctx, c, scale):
    """Vocabularies masked with the type's lowest number: what -inf in its place gives, so 0 at hidden tokens (a hidden
    target keeps its own gradient, which is exact); near 0 and far from it, beside the logits and in their place."""
    say("hidden", c, scale)
    rng = np.random.default_rng(c)
    x = R.f32(rng.standard_normal((4, c)) * 2)
    x[2] += 700.0
    hidden = rng.random((4, c)) < 0.5
    tokens = np.array([7, 3, 11, -100], np.int32)
    hidden[np.arange(3), tokens[:3]] = [False, True, False]
    hidden[:, 20] = False
    clean = np.where(hidden, np.float32(-np.inf), x)
    x[hidden] = np.finfo(np.float32).min
    want = R.logprobs(clean, tokens, scale)
    gl, ge = R.f32(rng.standard_normal(4)), R.f32(rng.standard_normal(4))
    for a, b in ((gl, ge), (gl, None), (None, ge)):
        xd = dev(ctx, x)
        got = run_logprobs(ctx, xd, tokens, scale)
        _, tok, outs = got["dev"]
        ref_g, tol = R.logprobs_grad(want, scale, a, b), R.logprobs_grad_tol(want, clean, scale, a, b)
        if a is not None:
            ref_g[1, 3] = np.float32(scale) * gl[1]
        for out in (Tensor.uninit(ctx, [4, c]), xd):
            ctx.check(ctx._lib.sg_token_logprobs_grad(ctx.handle, ref(xd), ref(tok) if a is not None else None, C.c_float(scale), ref(outs["lse"]),
                                                      ref(outs["entropy"]) if b is not None else None, ref(dev(ctx, a)) if a is not None else None,
                                                      ref(dev(ctx, b)) if b is not None else None, ref(out)))
            g = out.numpy()
            near(g, ref_g, tol, "glogits")
            hit = hidden.copy()
            hit[1, 3] = False
            assert not g[hit].any()


@pytest.mark.parametrize("c", [40, 20000])
@pytest.mark.parametrize("scale", [0.5, 1.0, 1.4])
def test_token_logprobs_of_hidden_tokens_are_as_low_as_their_logits(ctx, c, scale):
    """Logits near the type's lowest value beside ordinary ones: their log probabilities are finite where the number is (three
    roundings: the distance, its scaling, the sum), as given tokens and among the alternatives."""
    say("low", c, scale)
    rng = np.random.default_rng(c)
    x = R.f32(rng.standard_normal((6, c)) * 2)
    x[4:] += 500.0
    low = np.array([np.finfo(np.float32).min, -2.5e38, -1e38], np.float32)
    hidden = np.ones((6, c), bool)
    hidden[:, 5:9] = False
    clean = np.where(hidden, np.float32(-np.inf), x)
    x[hidden] = low[rng.integers(0, 3, hidden.sum())]
    tokens = np.array([0, 6, c - 1, 30, 12, 7], np.int32)
    want, t_lp = R.logprobs(clean, None, scale), R.logprobs_tol(clean, scale)[0]
    lp = x.astype(np.float64) * float(np.float32(scale)) - want["lse"][:, None]
    lp[np.abs(lp) > np.finfo(np.float32).max * (1 + R.U)] = -np.inf
    tol = t_lp[:, None] + 4 * R.U * np.where(np.isfinite(lp), np.abs(lp), 0.0)
    got = run_logprobs(ctx, x, tokens, scale, 16)
    at = np.arange(6)
    near(got["logprob"], lp[at, tokens], tol[at, tokens], "logprob")
    order = np.argsort(-x.astype(np.float64), axis=1, kind="stable")[:, :16]
    assert np.array_equal(got["top_ids"], order)
    near(got["top_logprobs"], np.take_along_axis(lp, order, 1), np.take_along_axis(tol, order, 1), "alternatives")
    near(got["lse"], want["lse"], t_lp + 2 * R.U * np.abs(want["lse"]), "lse")
    near(got["entropy"], want["entropy"], R.logprobs_tol(clean, scale)[1], "entropy")


def test_token_logprobs_of_more_rows_than_a_launch_has_in_x(ctx):
    """2^24 + 77 rows of 6 logits, each one logit behind the one above: a workgroup a row is more than 2^32 threads."""
    rows, c, top = (1 << 24) + 77, 6, 2
    rng = np.random.default_rng(51)
    base = R.f32(rng.standard_normal(rows + c - 1))
    tokens = rng.integers(-1, c, rows).astype(np.int32)
    x = Tensor(dev(ctx, base).buf, FLOAT, Shape([rows, c], [1, 1], 0))
    got = run_logprobs(ctx, x, tokens, 1.0, top)
    gl = R.f32(rng.standard_normal(rows))
    _, tok, outs = got["dev"]
    out = Tensor.uninit(ctx, [rows, c])
    ctx.check(ctx._lib.sg_token_logprobs_grad(ctx.handle, ref(x), ref(tok), C.c_float(1.0), ref(outs["lse"]), None, ref(dev(ctx, gl)), None, ref(out)))
    g = out.numpy()
    for k in ("logprob", "entropy", "lse"):
        assert np.isfinite(got[k]).all(), k
    at = np.concatenate([np.arange(2000), np.arange((1 << 21) - 500, (1 << 21) + 500), np.arange(rows - 3000, rows), rng.integers(0, rows, 50000)])
    part = base[at[:, None] + np.arange(c)]
    want = R.logprobs(part, tokens[at], 1.0, top)
    t_lp, t_h = R.logprobs_tol(part, 1.0)
    near(got["logprob"][at], want["logprob"], t_lp, "logprob")
    near(got["entropy"][at], want["entropy"], t_h, "entropy")
    assert np.array_equal(got["top_ids"][at], want["top_ids"])
    near(g[at], R.logprobs_grad(want, 1.0, gl[at]), R.logprobs_grad_tol(want, part, 1.0, gl[at]), "glogits")


def test_embedding_of_more_tokens_and_rows_than_a_launch_has_in_x(ctx):
    """2^26 tokens of one value (ids of each sequence one behind those above), and the gradient of a few tokens in a table of
    2^28 rows: more than 2^32 threads either way."""
    rng = np.random.default_rng(52)
    n, l, v = 8193, 8192, 1000
    base, table = rng.integers(0, v + 1, n + l - 1).astype(np.uint32), R.f32(rng.standard_normal((v, 1)))
    ids = Tensor(dev(ctx, base).buf, UINT, Shape([n, l], [1, 1], 0))
    out = dev(ctx, np.full((n, l, 1), np.nan, np.float32))
    ctx.check(ctx._lib.sg_embedding(ctx.handle, ref(dev(ctx, table)), ref(ids), C.c_float(0.3), ref(out)))
    got, once = out.numpy(), R.embedding(table, base, 0.3)[:, 0]
    assert same_bits(got, np.lib.stride_tricks.sliding_window_view(once, l)[..., None])
    del out
    v = (1 << 28) + 100
    at = np.array([3, v - 1, 1 << 26, 3, v - 1, 0xFFFFFFFF, (1 << 28) - 1], np.uint32)
    g = R.f32(rng.standard_normal((at.size, 1)))
    out = Tensor.uninit(ctx, [v, 1])
    ctx.check(ctx._lib.sg_embedding_grad(ctx.handle, ref(dev(ctx, g)), ref(dev(ctx, at)), C.c_float(1.5), ref(out)))
    got = out.numpy()[:, 0]
    for row in set(at.tolist()) - {0xFFFFFFFF}:
        mine = g[at == row, 0].astype(np.float64)
        near(got[row], mine.sum() * 1.5, (mine.size + 2) * R.U * np.abs(mine).sum() * 1.5, f"row {row}")
        got[row] = 0.0
    assert not got.any()


def test_adamw_of_gradients_in_the_parameters_memory(ctx):
    """Gradients that are other parameters' values (of a product of two parameters, say), views of them or the parameter itself:
    read as they are in front of the step, eager and compiled.  Two parameters in one memory are refused."""
    rng = np.random.default_rng(61)
    a, b, c = (R.f32(rng.standard_normal((300, 400))) for _ in range(3))

    def params():
        return [Var.new(dev(ctx, x)) for x in (a, b, c)]

    def crossed(p):
        flat = p[0].value
        return {p[0]: Var.new(p[1].value), p[1]: Var.new(flat.with_shape(Shape([300, 400]))), p[2]: Var.new(p[2].value)}
    for bits in (32, 8):
        want = params()
        opt = optim.AdamW(1e-2, state_bits=bits)
        eager, compiled = params(), params()
        o1, o2 = optim.AdamW(1e-2, state_bits=bits), optim.AdamW(1e-2, state_bits=bits)
        prog = None
        for _ in range(3):
            x, y, z = (dev(ctx, p.value.numpy()) for p in want)
            opt.update({want[0]: Var.new(y), want[1]: Var.new(x), want[2]: Var.new(z)}, ctx)
            o1.update(crossed(eager), ctx)
            if prog is None:
                prog = o2.compile(crossed(compiled), ctx)
            else:
                prog.run()
            for w, e, p in zip(want, eager, compiled):
                assert same_bits(w.value.numpy(), e.value.numpy()) and same_bits(w.value.numpy(), p.value.numpy())
    whole = dev(ctx, a)
    half = lambda o, n: Var.new(Tensor(whole.buf, FLOAT, Shape([n], [1], o)))  # noqa: E731
    gh = Var.new(dev(ctx, b[0, :100].copy()))
    optim.AdamW(1e-2).update({half(0, 100): gh, half(100, 100): gh}, ctx)  # beside one another in one buffer
    for two in ([half(0, 100), half(99, 100)], [half(5, 100), half(5, 100)]):
        with pytest.raises(abi.SageError):
            optim.AdamW(1e-2).update({p: gh for p in two}, ctx)
        with pytest.raises(abi.SageError):
            optim.AdamW(1e-2).compile({p: gh for p in two}, ctx)
