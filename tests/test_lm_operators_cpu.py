"""The language-model operators without a GPU: every refusal of the C ABI (arguments are checked before the context, so a
null context gives the same status), the front end's shapes and gradient graphs, and the 64-bit formulas the GPU tests
compare with against finite differences."""
import ctypes as C

import numpy as np
import pytest

from sage_amd import abi, bert, nn, optim
from sage_amd.grad import grad
from sage_amd.shape import default_strides
from sage_amd.tensor import FLOAT, INT, UINT
from sage_amd.var import Var
from tests import lm_reference as R

OK_BUT_NO_CONTEXT = abi.ERR_ARG


def desc(extents, dtype=abi.FLOAT, strides=None, base=4096):
    t = abi.sg_tensor()
    t.base, t.dtype, t.rank = base, dtype, len(extents)
    for i, (e, s) in enumerate(zip(extents, default_strides(extents) if strides is None else strides)):
        t.extents[i], t.strides[i] = e, s
    return t


def call(fn, *args):
    return getattr(abi.lib(), fn)(None, *[C.byref(a) if isinstance(a, abi.sg_tensor) else a for a in args])


# ----------------------------------------------------------------------------- refusals
def emb(table=None, ids=None, out=None):
    return call("sg_embedding", table or desc([10, 8]), ids or desc([2, 3], UINT), C.c_float(1.0), out or desc([2, 3, 8]))


def emb_grad(gout=None, ids=None, gtable=None):
    return call("sg_embedding_grad", gout or desc([2, 3, 8]), ids or desc([2, 3], INT), C.c_float(1.0), gtable or desc([10, 8]))


def test_embedding_refusals():
    assert emb() == emb_grad() == OK_BUT_NO_CONTEXT
    assert emb(table=desc([10, 8], strides=[1, 10])) == abi.ERR_SHAPE
    assert emb(table=desc([8])) == abi.ERR_SHAPE
    assert emb(table=desc([10, 8], UINT)) == abi.ERR_DTYPE
    assert emb(table=desc([10, 8], base=None)) == abi.ERR_ARG
    assert emb(ids=desc([2, 3])) == abi.ERR_DTYPE
    assert emb(ids=desc([3, 2], UINT)) == abi.ERR_SHAPE
    assert emb(ids=desc([6], UINT)) == abi.ERR_SHAPE
    assert emb(out=desc([2, 3, 9])) == abi.ERR_SHAPE
    assert emb(out=desc([2, 3, 8], strides=[24, 8, 2])) == abi.ERR_SHAPE
    assert emb(out=desc([2, 3, 8], INT)) == abi.ERR_DTYPE
    assert emb(ids=desc([2, 3], UINT, strides=[0, 1])) == OK_BUT_NO_CONTEXT  # any strides for an input
    assert emb_grad(gout=desc([2, 3, 8], strides=[0, 0, 1])) == OK_BUT_NO_CONTEXT
    assert emb_grad(gout=desc([2, 3, 8], strides=[24, 8, 0])) == abi.ERR_SHAPE
    assert emb_grad(gout=desc([2, 4, 8])) == abi.ERR_SHAPE
    assert emb_grad(gtable=desc([10, 8], strides=[9, 1])) == abi.ERR_SHAPE
    assert emb_grad(gtable=desc([10, 4])) == abi.ERR_SHAPE
    assert emb_grad(ids=desc([2, 3], abi.LONG)) == abi.ERR_DTYPE


def lp(logits=None, tokens=0, scale=1.0, logprob=0, entropy=0, lse=0, ids=None, tops=None):
    pick = lambda x, d: d if x == 0 else x  # noqa: E731
    return call("sg_token_logprobs", logits or desc([2, 3, 50]), pick(tokens, desc([2, 3], INT)), C.c_float(scale), pick(logprob, desc([2, 3])),
                pick(entropy, desc([2, 3])), pick(lse, desc([2, 3])), ids, tops)


def lp_grad(logits=None, tokens=0, scale=1.0, lse=0, entropy=0, gl=0, ge=0, out=None):
    pick = lambda x, d: d if x == 0 else x  # noqa: E731
    return call("sg_token_logprobs_grad", logits or desc([2, 3, 50]), pick(tokens, desc([2, 3], INT)), C.c_float(scale), pick(lse, desc([2, 3])),
                pick(entropy, desc([2, 3])), pick(gl, desc([2, 3], strides=[0, 0])), pick(ge, desc([2, 3])), out or desc([2, 3, 50]))


def test_token_logprobs_refusals():
    assert lp() == lp_grad() == OK_BUT_NO_CONTEXT
    assert lp(ids=desc([2, 3, 5], UINT), tops=desc([2, 3, 5])) == OK_BUT_NO_CONTEXT
    assert lp(logits=desc([2, 3, 50], strides=[150, 1, 3])) == abi.ERR_SHAPE
    assert lp(logits=desc([2, 3, 50], INT)) == abi.ERR_DTYPE
    for bad in (0.0, -1.0, float("nan"), float("inf")):
        assert lp(scale=bad) == lp_grad(scale=bad) == abi.ERR_ARG
    assert lp(tokens=desc([2, 3])) == abi.ERR_DTYPE
    assert lp(tokens=desc([6], INT)) == abi.ERR_SHAPE
    assert lp(tokens=None) == abi.ERR_ARG and lp(tokens=None, logprob=None) == OK_BUT_NO_CONTEXT
    assert lp(logprob=desc([2, 3], strides=[0, 1])) == abi.ERR_SHAPE
    assert lp(entropy=desc([2, 4])) == abi.ERR_SHAPE
    assert lp(lse=None) == abi.ERR_ARG and lp(lse=desc([6])) == abi.ERR_SHAPE
    assert lp(ids=desc([2, 3, 5], UINT)) == lp(tops=desc([2, 3, 5])) == abi.ERR_ARG
    assert lp(ids=desc([2, 3, 5], INT), tops=desc([2, 3, 5])) == abi.ERR_DTYPE
    assert lp(ids=desc([2, 3, 5], UINT), tops=desc([2, 3, 4])) == abi.ERR_SHAPE
    assert lp(ids=desc([2, 3, 51], UINT), tops=desc([2, 3, 51])) == abi.ERR_SHAPE
    assert lp(logits=desc([2, 3, 500]), ids=desc([2, 3, 65], UINT), tops=desc([2, 3, 65])) == abi.ERR_SHAPE
    assert lp(ids=desc([2, 3, 5], UINT, strides=[20, 5, 1]), tops=desc([2, 3, 5])) == abi.ERR_SHAPE
    assert lp(logits=desc([50]), tokens=desc([1], INT), logprob=desc([1]), entropy=None, lse=desc([1])) == OK_BUT_NO_CONTEXT
    assert lp_grad(gl=None, ge=None) == abi.ERR_ARG
    assert lp_grad(tokens=None) == abi.ERR_ARG and lp_grad(tokens=None, gl=None) == OK_BUT_NO_CONTEXT
    assert lp_grad(entropy=None) == abi.ERR_ARG and lp_grad(entropy=None, ge=None) == OK_BUT_NO_CONTEXT
    assert lp_grad(lse=None) == abi.ERR_ARG
    assert lp_grad(ge=desc([2, 4])) == abi.ERR_SHAPE
    assert lp_grad(out=desc([2, 3, 50], strides=[160, 50, 1])) == abi.ERR_SHAPE
    assert lp_grad(out=desc([6, 50])) == abi.ERR_SHAPE
    # in place of logits with padded rows or of one row for all: other places than the gradient's
    assert lp_grad(logits=desc([2, 3, 50], strides=[160, 50, 1])) == lp_grad(logits=desc([2, 3, 50], strides=[0, 0, 1])) == abi.ERR_SHAPE
    assert lp_grad(logits=desc([2, 3, 50], strides=[160, 50, 1]), out=desc([2, 3, 50], base=8192)) == OK_BUT_NO_CONTEXT


Q, K, M, L = [2, 4, 5, 32], [2, 2, 7, 32], [2, 7], [2, 4, 5]


def ca(q=None, k=None, v=None, mask=0, out=None, lse=0):
    return call("sg_cross_attention", q or desc(Q), k or desc(K), v or desc(K), desc(M) if mask == 0 else mask, C.c_float(1.0), out or desc(Q),
                desc(L) if lse == 0 else lse)


def ca_grad(lse=0, gout=None, gq=None, gk=None, gv=None, out=None):
    return call("sg_cross_attention_grad", desc(Q), desc(K), desc(K), desc(M), C.c_float(1.0), out or desc(Q), desc(L) if lse == 0 else lse,
                gout or desc(Q), gq or desc(Q), gk or desc(K), gv or desc(K))


def test_cross_attention_refusals():
    assert ca() == ca_grad() == OK_BUT_NO_CONTEXT
    assert ca(mask=None, lse=None) == OK_BUT_NO_CONTEXT
    assert ca(q=desc(Q, strides=[640, 32, 128, 1]), out=desc(Q, strides=[640, 32, 128, 1])) == OK_BUT_NO_CONTEXT  # heads side by side
    assert ca(q=desc([2, 4, 5, 48]), k=desc([2, 2, 7, 48]), v=desc([2, 2, 7, 48]), out=desc([2, 4, 5, 48])) == abi.ERR_SHAPE
    assert ca(q=desc([4, 5, 32])) == abi.ERR_SHAPE
    assert ca(k=desc([2, 3, 7, 32]), v=desc([2, 3, 7, 32])) == abi.ERR_SHAPE  # 4 heads over 3
    assert ca(k=desc([1, 2, 7, 32])) == ca(k=desc([2, 2, 7, 64])) == ca(v=desc([2, 2, 8, 32])) == abi.ERR_SHAPE
    assert ca(k=desc(K, strides=[448, 224, 1, 7])) == abi.ERR_SHAPE
    assert ca(q=desc(Q, UINT)) == abi.ERR_DTYPE
    assert ca(mask=desc([2, 8])) == ca(mask=desc([7])) == ca(mask=desc(M, strides=[14, 2])) == abi.ERR_SHAPE
    assert ca(mask=desc(M, INT)) == abi.ERR_DTYPE
    assert ca(mask=desc(M, strides=[0, 1])) == OK_BUT_NO_CONTEXT  # one mask for all sequences
    assert ca(out=desc(Q, strides=[640, 160, 0, 1])) == abi.ERR_SHAPE  # queries on one address
    assert ca(out=desc(Q, strides=[640, 160, 16, 1])) == abi.ERR_SHAPE  # rows that overlap
    assert ca(out=desc([2, 4, 6, 32])) == abi.ERR_SHAPE
    assert ca(lse=desc([2, 4, 5], strides=[40, 10, 2])) == ca(lse=desc([8, 5])) == abi.ERR_SHAPE
    assert ca_grad(lse=None) == abi.ERR_ARG
    assert ca_grad(gout=desc(Q, strides=[0, 0, 0, 1])) == OK_BUT_NO_CONTEXT  # a broadcast gradient
    assert ca_grad(gout=desc(Q, strides=[0, 0, 0, 0])) == abi.ERR_SHAPE
    assert ca_grad(gq=desc(Q, strides=[640, 0, 32, 1])) == ca_grad(gk=desc(K, strides=[0, 224, 32, 1])) == abi.ERR_SHAPE
    assert ca_grad(gv=desc(Q)) == abi.ERR_SHAPE


def adamw(n=2, ext=(300, 7), bits=8, step=None, hyper=0, drop=None, **over):
    """over: an array's name -> the tensors to hand over instead."""
    ext = list(ext)
    arrays = {"value": [desc([e]) for e in ext], "grad": [desc([e]) for e in ext]}
    if bits == 8:
        for s in ("m", "v"):
            arrays[s] = [desc([(e + 3) // 4], UINT) for e in ext]
        for s in ("ms", "vs"):
            arrays[s] = [desc([(e + 255) // 256]) for e in ext]
    else:
        arrays["m"] = arrays["v"] = arrays["value"]
        arrays["ms"] = arrays["vs"] = None
    arrays.update(over)
    if drop:
        arrays[drop] = None
    c = lambda a: None if a is None else (abi.sg_tensor * len(a))(*a)  # noqa: E731
    h = abi.sg_adam_hyper(1e-3, 0.9, 0.999, 0.1, 0.001, 1e-8, 0.01) if hyper == 0 else hyper
    return abi.lib().sg_adamw_update(None, n, *[c(arrays[x]) for x in ("value", "grad", "m", "v", "ms", "vs")], C.byref(step or desc([1])),
                                     C.byref(h) if h is not None else None, 1)


def test_adamw_refusals():
    assert adamw() == adamw(bits=32) == OK_BUT_NO_CONTEXT
    assert adamw(n=0) == OK_BUT_NO_CONTEXT and adamw(n=-1) == abi.ERR_ARG
    for a in ("value", "grad", "m", "v", "ms", "vs"):
        assert adamw(drop=a) == abi.ERR_ARG
    assert adamw(hyper=None) == abi.ERR_ARG
    assert adamw(hyper=abi.sg_adam_hyper(1e-3, 1.0, 0.999, 0.0, 0.001, 1e-8, 0.0)) == abi.ERR_ARG
    assert adamw(hyper=abi.sg_adam_hyper(1e-3, 0.9, float("nan"), 0.1, 0.001, 1e-8, 0.0)) == abi.ERR_ARG
    assert adamw(step=desc([2])) == abi.ERR_SHAPE and adamw(step=desc([1], INT)) == abi.ERR_DTYPE
    assert adamw(grad=[desc([300]), desc([8])]) == abi.ERR_SHAPE
    assert adamw(value=[desc([300], strides=[2]), desc([7])]) == abi.ERR_SHAPE
    assert adamw(m=[desc([75]), desc([2])]) == abi.ERR_DTYPE
    assert adamw(m=[desc([300], UINT), desc([2], UINT)]) == abi.ERR_SHAPE
    assert adamw(vs=[desc([1]), desc([1])]) == abi.ERR_SHAPE
    assert adamw(bits=32, v=[desc([300]), desc([6])]) == abi.ERR_SHAPE
    arr = lambda *t: (abi.sg_tensor * len(t))(*t)  # noqa: E731
    ok = [arr(desc([75], UINT)), arr(desc([75], UINT)), arr(desc([2])), arr(desc([2])), arr(desc([300])), arr(desc([300]))]
    read = abi.lib().sg_adamw_state_read
    assert read(None, 1, *ok) == OK_BUT_NO_CONTEXT and read(None, -1, *ok) == abi.ERR_ARG
    assert read(None, 1, *ok[:5], None) == abi.ERR_ARG
    assert read(None, 1, *ok[:5], arr(desc([301]))) == abi.ERR_SHAPE
    assert read(None, 1, arr(desc([76], UINT)), *ok[1:]) == abi.ERR_SHAPE


# ----------------------------------------------------------------------------- the front end
def test_front_end_shapes_and_refusals():
    table, ids = Var.empty([10, 8]), Var.empty([2, 3], UINT)
    assert nn.embedding(table, ids, 2.0).extents == [2, 3, 8]
    logits = Var.empty([2, 3, 50])
    r = nn.token_logprobs(logits, Var.empty([2, 3], INT), top=4)
    assert r.logprob.extents == r.entropy.extents == r.lse.extents == [2, 3]
    assert r.top_ids.extents == r.top_logprobs.extents == [2, 3, 4] and r.top_ids.dtype == UINT
    assert nn.token_logprobs(logits).logprob is None and nn.token_logprobs(logits).top_ids is None
    q, k, m = Var.empty(Q), Var.empty(K), Var.empty(M)
    assert nn.cross_attention(q, k, k, m).extents == Q
    for bad in (lambda: nn.embedding(Var.empty([10]), ids), lambda: nn.embedding(table, Var.empty([1] * 8, UINT)),
                lambda: nn.token_logprobs(logits, Var.empty([6], INT)), lambda: nn.token_logprobs(logits, top=51),
                lambda: nn.token_logprobs(Var.empty([2, 500]), top=65), lambda: nn.token_logprobs(logits, top=-1),
                lambda: nn.cross_attention(q, Var.empty([2, 3, 7, 32]), Var.empty([2, 3, 7, 32])), lambda: nn.cross_attention(q, k, q),
                lambda: nn.cross_attention(Var.empty([2, 4, 5, 40]), Var.empty([2, 2, 7, 40]), Var.empty([2, 2, 7, 40])),
                lambda: nn.cross_attention(q, k, k, Var.empty([2, 8])), lambda: nn.cross_attention(Var.empty([4, 5, 32]), k, k)):
        with pytest.raises(abi.ShapeError):
            bad()
    for bad in (lambda: nn.embedding(Var.empty([10, 8], UINT), ids), lambda: nn.embedding(table, Var.empty([2, 3])),
                lambda: nn.token_logprobs(logits, Var.empty([2, 3])), lambda: nn.token_logprobs(ids),
                lambda: nn.cross_attention(q, k, k, Var.empty(M, UINT))):
        with pytest.raises(abi.DTypeError):
            bad()
    with pytest.raises(abi.SageError):
        nn.token_logprobs(logits, scale=0.0)
    with pytest.raises(ValueError):
        optim.AdamW(1e-3, state_bits=16)


def test_gradient_graphs_of_the_operators():
    table, ids = Var.empty([10, 8]), Var.empty([2, 3], UINT)
    g = grad(nn.embedding(table, ids, 2.0), [table])[0]
    assert g.op == "embedding_grad" and g.extents == [10, 8] and g.attrs["scale"] == 2.0
    seed = Var.empty([2, 3, 8])
    g2 = grad(nn.embedding(table, ids, 2.0), [table], seed=seed)[0]
    assert grad(g2, [seed])[0].op == "embedding"
    logits, tokens = Var.empty([6, 50]), Var.empty([6], INT)
    r = nn.token_logprobs(logits, tokens)
    one = grad(r.logprob, [logits])[0]
    assert one.attrs == {"logprob": True, "entropy": False}
    both = grad(r.logprob + r.entropy * 0.1, [logits])[0]  # one pass over the logits for both
    assert both.op == "token_logprobs_grad" and both.attrs == {"logprob": True, "entropy": True} and both.inputs[2] is tokens
    q, k, v, m = Var.empty(Q), Var.empty(K), Var.empty(K), Var.empty(M)
    gq, gk, gv = grad(nn.cross_attention(q, k, v, m), [q, k, v])
    assert gq.op == "cross_attention_grad" and gk.inputs[0] is gq and gv.inputs[0] is gq and gk.extents == gv.extents == K
    layer = bert.CrossAttention(64, 2, num_kv_heads=1)
    y = layer.pass_(Var.empty([2, 5, 64]), Var.empty([2, 7, 64]), Var.empty([2, 7]))
    assert y.extents == [2, 5, 64] and len(grad(y, layer.params())) == len(layer.params())


# ----------------------------------------------------------------------------- the formulas against differences
def directional(f, x, d, h=1e-5):
    return (f(x + h * d) - f(x - h * d)) / (2 * h)


def test_formulas_against_finite_differences():
    rng = np.random.default_rng(0)
    x, w1, w2 = rng.standard_normal((3, 11)), rng.standard_normal(3), rng.standard_normal(3)
    tok = np.array([4, -100, 10])

    def f(z):
        r = R.logprobs(z, tok, 1.5)
        return (r["logprob"] * w1 + r["entropy"] * w2).sum()
    g = R.logprobs_grad(R.logprobs(x, tok, 1.5), 1.5, w1, w2)
    d = rng.standard_normal(x.shape)
    assert abs(directional(f, x, d) - (g * d).sum()) < 1e-7
    q, k, v = rng.standard_normal((2, 4, 3, 32)), rng.standard_normal((2, 2, 5, 32)), rng.standard_normal((2, 2, 5, 32))
    mask = np.array([[1, 0, 1, 1, 0], [0, 0, 0, 0, 0]], np.float32)
    go = rng.standard_normal(q.shape)
    grads = R.cross_grad(q, k, v, mask, 0.3, go)
    for i, (a, ga) in enumerate(zip((q, k, v), grads)):
        d = rng.standard_normal(a.shape)
        assert abs(directional(lambda z: (R.cross(*[z if j == i else b for j, b in enumerate((q, k, v))], mask, 0.3)[0] * go).sum(), a, d) - (ga * d).sum()) < 1e-6
    assert not grads[0][1].any() and not grads[1][0][:, 1].any()


# ----------------------------------------------------------------------------- the 8-bit form
@pytest.mark.parametrize("signed", [True, False])
def test_eight_bit_states_round_trip_and_keep_their_mean(signed):
    rng = np.random.default_rng(1)
    x = R.f32(np.exp(rng.uniform(-3, 0, 1000)) * (np.sign(rng.standard_normal(1000)) if signed else 1.0))
    x[17] = 0.0
    draws = []
    for t in range(1, 400):
        codes, scale = R.encode(x, signed, R.noise(x.size, t, 3)[0 if signed else 1])
        y = R.decode(codes, scale, signed)
        assert np.all(np.abs(y - x) <= 2.0 ** -3 * np.abs(x))  # at most one step of 3 mantissa bits
        draws.append(y)
        # what the bytes stand for is kept as it is (the scale may be another one, if the largest was rounded down)
        assert np.array_equal(R.decode(*R.encode(y, signed, np.zeros(x.size, np.int64)), signed), y)
        assert np.array_equal(R.unpack(R.pack(codes), x.size), codes)
    # a draw is off by a step at most, with variance at most step^2 / 4: 399 draws' mean by 6 deviations of step / 2 / sqrt(399)
    assert np.all(np.abs(np.mean(draws, 0) - x) <= 6 * 2.0 ** -4 / np.sqrt(399) * np.abs(x) + 1e-12)


def test_eight_bit_states_at_the_borders():
    c, s = R.encode(R.f32([0.0] * 300), False, np.full(300, 0xFFFF))
    assert not c.any() and not R.decode(c, s, False).any() and s.shape == (2,)
    c, s = R.encode(R.f32([1e30, 1e-30, 0.0]), False, np.zeros(3, np.int64))
    y = R.decode(c, s, False)
    assert c[1] == 1 and y[1] > 0 and c[2] == 0  # a second moment that is not zero does not become zero
    c, s = R.encode(R.f32([1.99, -1.99, 1.0]), True, np.full(3, 0xFFFF))
    assert np.all(np.abs(R.decode(c, s, True)[:2]) == 2.0)  # rounded up past the mantissa: the scale has room
    c, s = R.encode(R.f32([np.inf, 1.0]), True, np.zeros(2, np.int64))
    assert np.isnan(s[0]) and np.isnan(R.decode(c, s, True)).all()


# ----------------------------------------------------------------------------- copies own their memory
def evaluated(targets):
    """The targets' tensors, and how many copies (maps) were launched, on a context without a device."""
    from sage_amd.var import _Evaluator
    from tests.test_host_cpu import _DryCtx

    class Log:
        def __init__(self, lib):
            self.lib, self.maps = lib, 0

        def __getattr__(self, name):
            self.maps += name == "sg_map"
            return getattr(self.lib, name)
    ctx = _DryCtx()
    ctx._lib = Log(ctx._lib)
    ev = _Evaluator(ctx, targets)
    return [ev.get(t) for t in targets], ctx._lib.maps


def cross_nodes():
    from tests.test_host_cpu import _DryCtx, _data
    ctx = _DryCtx()
    q, k, v = (_data(ctx, *e) for e in (Q, K, K))
    y = nn.cross_attention(q, k, v)
    return y, *grad(y, [q, k, v], seed=_data(ctx, *Q))


def bound(*nodes):
    for n, t in zip(nodes, evaluated(list(nodes))[0]):
        n.value = t


@pytest.mark.parametrize("which", [0, 1, 2, 3])
def test_copies_of_cross_attentions_tensors_have_memory_of_their_own(which):
    """The operator leaves heads side by side, so the copy of its transposed output or gradients finds the layout it asks for;
    it may take that memory over only where nobody else can see it."""
    y = cross_nodes()[which]
    (a, b), maps = evaluated([y, y.transpose(2, 1).copy()])  # both asked for
    assert a.buf is not b.buf and maps == 1
    y = cross_nodes()[which]
    (a, b), maps = evaluated([y.transpose(2, 1), y.transpose(2, 1).copy()])  # the permuted view asked for
    assert a.buf is not b.buf and maps == 1
    y = cross_nodes()[which]
    (a, b), maps = evaluated([y.transpose(2, 1).copy(), y.transpose(2, 1).copy()])  # two copies
    assert a.buf is not b.buf
    y = cross_nodes()[which]
    (a, b), maps = evaluated([y.transpose(2, 1).copy(), y.slice(0, 0, 1)])  # another view
    assert a.buf is not b.buf and maps == 1
    nodes = cross_nodes()
    bound(*nodes)  # as Program.bind leaves them
    (a,), maps = evaluated([nodes[which].transpose(2, 1).copy()])
    assert a.buf is not nodes[which].value.buf and maps == 1
    if which >= 2:  # the same output of a bound operator, or asked for beside the copy
        y, gq, gk, gv = cross_nodes()
        bound(gq)
        (a,), maps = evaluated([(gk, gv)[which - 2].transpose(2, 1).copy()])
        assert a.buf is not gq.value.parts[("gk", "gv")[which - 2]].buf and maps == 1
        y, gq, gk, gv = cross_nodes()
        again = Var(gk.shape, FLOAT, "part", [gq], dict((gk, gv)[which - 2].attrs))
        (a, b), maps = evaluated([again, (gk, gv)[which - 2].transpose(2, 1).copy()])
        assert a.buf is not b.buf and maps == 1


def test_merged_heads_inside_a_step_take_no_copy():
    y, gq, gk, gv = cross_nodes()
    merged = [x.transpose(2, 1).view([2, -1, x.extents[1] * 32]) for x in (y, gq, gk, gv)]
    outs, maps = evaluated(merged)
    assert maps == 0 and len({id(t.buf) for t in outs}) == 4


def test_token_logprobs_refuse_a_scale_whose_logarithm_to_base_2_overflows():
    """scale * log2(e) is what the kernels multiply by: beyond 2^127 it may be infinite, and 0 times it NaN."""
    for scale in (2.0 ** 127 * (1 + 2.0 ** -23), 3.4e38):
        assert lp(scale=scale) == lp_grad(scale=scale) == abi.ERR_ARG
        with pytest.raises(abi.SageError):
            nn.token_logprobs(Var.empty([2, 3, 50]), scale=scale)
    assert lp(scale=2.0 ** 127) == lp_grad(scale=2.0 ** 127) == OK_BUT_NO_CONTEXT
    assert np.isfinite(np.float32(2.0 ** 127) * np.float32(1.44269504088896340736))


@pytest.mark.parametrize("signed,bottom", [(True, -15), (False, -31)])
def test_eight_bit_states_at_the_bottom_of_a_block(signed, bottom):
    """Beside a largest of 1, whose power of two is 1: the mean is kept from 1.125 * 2^bottom on; below, a first moment loses it
    and becomes zero under 2^bottom, a second moment is held at 1.125 * 2^bottom."""
    lowest = 1.125 * 2.0 ** bottom
    x = R.f32([1.0] + [lowest * f for f in (1.0, 1.05, 1.3, 1.77, 3.1, 7.7)] + [2.0 ** bottom * f for f in (1.06, 1.0, 0.999, 0.5, 0.25, 2.0 ** -20)])
    assert np.all(x > 0)
    n = 999
    draws = np.array([R.decode(*R.encode(x, signed, R.noise(x.size, t, 3)[0 if signed else 1]), signed) for t in range(1, n + 1)])
    # a draw is off by at most a step of 1/8 with variance at most its square / 4: the mean by 6 deviations
    assert np.all(np.abs(draws.mean(0) - x)[:7] <= 6 * 2.0 ** -4 / np.sqrt(n) * x[:7])
    if signed:
        # 1.06 is 0.06 / 0.125 of the way from 2^bottom, which is no number of the block, to the smallest: else 0
        part = 0.06 / 0.125
        assert set(np.unique(draws[:, 7])) == {np.float32(0), np.float32(lowest)}
        assert abs((draws[:, 7] > 0).mean() - part) <= 6 * 0.5 / np.sqrt(n)
        assert not draws[:, 8:].any()
    else:
        assert np.all(draws[:, 7:] == np.float32(lowest))


def test_cross_attention_refuses_more_pairs_than_a_launch_has_workgroups():
    """2^24 workgroups of 256 threads are more than a launch takes; refused in front of the context, like any argument."""
    def both(n, heads):
        q, k, m, lse = [n, heads, 1, 32], [n, heads, 2, 32], [n, 2], [n, heads, 1]
        return (call("sg_cross_attention", desc(q), desc(k), desc(k), desc(m), C.c_float(1.0), desc(q), desc(lse)),
                call("sg_cross_attention_grad", desc(q), desc(k), desc(k), desc(m), C.c_float(1.0), desc(q), desc(lse), desc(q), desc(q), desc(k), desc(k)))
    assert both(1 << 24, 1) == both(1 << 12, 1 << 12) == both((1 << 24) - 7, 1) == (abi.ERR_SHAPE, abi.ERR_SHAPE)
    assert both((1 << 24) - 8, 1) == (OK_BUT_NO_CONTEXT, OK_BUT_NO_CONTEXT)


def test_token_logprobs_grad_refuses_what_it_cannot_compute():
    logits, tokens, g = Var.empty([6, 50]), Var.empty([6], INT), Var.empty([6])
    lse = nn.token_logprobs(logits, tokens).lse
    assert nn.token_logprobs_grad(logits, lse, tokens, g).extents == nn.token_logprobs_grad(logits, lse, g_entropy=g).extents == [6, 50]
    for bad in (lambda: nn.token_logprobs_grad(logits, lse, None, g), lambda: nn.token_logprobs_grad(logits, lse, tokens),
                lambda: nn.token_logprobs_grad(logits, Var.empty([6]), tokens, g)):
        with pytest.raises(abi.SageError):
            bad()
    q, k = Var.empty(Q), Var.empty(K)  # gradients of these gradients are refused, not wrong
    for first in (grad(nn.cross_attention(q, k, k), [q])[0], nn.token_logprobs_grad(logits, lse, tokens, g)):
        with pytest.raises(ValueError):
            grad(first, [q if first.op == "cross_attention_grad" else logits])
