"""Timed cases of the language-model operators: the embedding lookup and its gradient by sorted tokens, cross
attention to an encoder's states, log probabilities of given tokens, and the AdamW step over many tensors.

`own` chooses between the plain form (elementary torch operations in 32 bits) and the calls a program makes of
the library through its C ABI; `prepare` makes the same state for both.  The library works on borrowed pointers
and on a stream of its own, so `prepare` ends by waiting for the copies and fills it issued.
"""
import math

import numpy as np
import torch

own = False

I32 = torch.int32
LOW = 0xFFFFFFFF


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # a few new tokens of a serving batch: nothing but latency
        {"name": "embedding 8 tokens", "op": "embedding", "tokens": 8, "vocab": 30522, "width": 768, "ignored": 0.0, "grad": False},
        # the training batch of the repository's benchmark configuration (32 x 128 tokens), both directions
        {"name": "embedding 4096 train", "op": "embedding", "tokens": 4096, "vocab": 30522, "width": 768, "ignored": 0.0, "grad": True},
        # a long padded batch (64 x 512): frequent tokens come thousands of times, padding is no token
        {"name": "embedding 32768 padded", "op": "embedding", "tokens": 32768, "vocab": 30522, "width": 768, "ignored": 0.3, "grad": True},
        # serving: the next token's alternatives for four sequences
        {"name": "logprobs 4 rows top 5", "op": "logprobs", "rows": 4, "vocab": 30522, "top": 5, "scale": 1.25, "ignored": 0.0, "grad": False},
        # scoring given texts, with alternatives, an odd vocabulary
        {"name": "logprobs 1021 rows top 20", "op": "logprobs", "rows": 1021, "vocab": 50257, "top": 20, "scale": 1.0, "ignored": 0.1, "grad": False},
        # the loss of a training step and its gradient, with an entropy term; ignored positions
        {"name": "logprobs 4096 train", "op": "logprobs", "rows": 4096, "vocab": 30522, "top": 0, "scale": 1.0, "ignored": 0.2, "grad": True},
        # serving: one new token of each sequence reads the encoder's states
        {"name": "cross 1 query", "op": "cross", "batch": 32, "heads": 12, "kv_heads": 12, "queries": 1, "keys": 512, "size": 64, "grad": False},
        # a ragged batch with shared heads of size 32, odd lengths, both directions
        {"name": "cross 333 x 1001 train", "op": "cross", "batch": 7, "heads": 8, "kv_heads": 2, "queries": 333, "keys": 1001, "size": 32, "grad": True},
        # a training step at the longest length of the repository's encoder
        {"name": "cross 512 x 512 train", "op": "cross", "batch": 32, "heads": 12, "kv_heads": 12, "queries": 512, "keys": 512, "size": 64, "grad": True},
        # a small model: many small tensors, so the number of launches counts
        {"name": "adamw small", "op": "adamw", "layers": 4, "width": 64, "vocab": 151, "bits": 32, "step": 3},
        # a model of about 80 million values, states in 32 bits
        {"name": "adamw 32 bits", "op": "adamw", "layers": 12, "width": 640, "vocab": 30522, "bits": 32, "step": 100},
        # the same with 8-bit states
        {"name": "adamw 8 bits", "op": "adamw", "layers": 12, "width": 640, "vocab": 30522, "bits": 8, "step": 1000},
    ]


def _log(rng, lo, hi):
    """A whole number of lo..hi, spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["embedding", "logprobs", "cross", "adamw"])
    if op == "embedding":
        return {"op": op, "tokens": _log(rng, 1, 32768), "vocab": _log(rng, 100, 30522), "width": _log(rng, 24, 768),
                "ignored": rng.choice([0.0, 0.1, 0.5]), "grad": rng.random() < 0.7}
    if op == "logprobs":
        vocab = _log(rng, 1000, 60000)
        return {"op": op, "rows": _log(rng, 1, max(1, min(4096, 4096 * 30522 // vocab))), "vocab": vocab, "top": rng.choice([0, 1, 5, 20, 32]),
                "scale": rng.choice([1.0, 0.5, 1.4]), "ignored": rng.choice([0.0, 0.3]), "grad": rng.random() < 0.5}
    if op == "cross":
        kv, group, size = rng.choice([1, 2, 3, 4, 8, 12]), rng.choice([1, 1, 2, 3, 4]), rng.choice([32, 64])
        queries = 1 if rng.random() < 0.3 else _log(rng, 2, 512)
        keys = _log(rng, 8, 4096)  # with a single state the gradients of queries and keys are zero but for rounding
        most = 32 * 12 * 512 * 512 * 64
        batch = max(1, min(_log(rng, 1, 32), most // (kv * group * queries * keys * size)))
        return {"op": op, "batch": batch, "heads": kv * group, "kv_heads": kv, "queries": queries, "keys": keys, "size": size,
                "grad": queries > 1 and rng.random() < 0.6}
    return {"op": op, "layers": rng.randint(1, 12), "width": _log(rng, 16, 640), "vocab": _log(rng, 50, 30522), "bits": rng.choice([8, 32]),
            "step": rng.choice([1, 2, 10, 5000])}


# ------------------------------------------------------------------------------------------------ what a case consists of
def _lengths(case):
    """Visible states of each sequence of a cross-attention batch: full, shrinking to half, and the last of three or more has none."""
    n, keys = case["batch"], case["keys"]
    lengths = [max(1, math.ceil(keys * (1.0 - 0.5 * b / n))) for b in range(n)]
    if n >= 3:
        lengths[-1] = 0
    return lengths


def _sizes(case):
    """Element counts of a transformer's parameters."""
    w, per_layer = case["width"], []
    for _ in range(4):
        per_layer += [w * w, w]
    per_layer += [w * 4 * w, 4 * w, 4 * w * w, w, w, w, w, w]
    return [case["vocab"] * w] + per_layer * case["layers"]


def _starts(sizes):
    """Where each tensor starts in one flat buffer, every start a multiple of 256 elements; and the buffer's size."""
    starts, at = [], 0
    for n in sizes:
        starts.append(at)
        at += (n + 255) // 256 * 256
    return starts, at


def _adamw_constants():
    """lr, beta1, beta2, eps, weight_decay, 1 - beta1, 1 - beta2: the betas are 32-bit numbers, their complements exact."""
    b1, b2 = np.float32(0.9), np.float32(0.999)
    return 1e-4, float(b1), float(b2), 1e-8, 0.01, float(np.float32(1) - b1), float(np.float32(1) - b2)


SEED = 20240131  # of the rounding of 8-bit states


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*ext):
        return torch.randn(*ext, generator=g, device="cuda")

    def uniform(*ext):
        return torch.rand(*ext, generator=g, device="cuda")

    s = dict(case)
    if case["op"] == "embedding":
        n, v, w = case["tokens"], case["vocab"], case["width"]
        ids = torch.exp(uniform(n) * math.log(v + 1)).long() - 1  # the r-th most frequent token with probability ~ 1/r
        ids = torch.where(uniform(n) < case["ignored"], -torch.ones_like(ids), ids.clamp(0, v - 1))
        s.update(ids=ids.to(I32), table=normal(v, w) * 0.02, factor=float(np.float32(math.sqrt(w))), out=torch.empty(n, w, device="cuda"))
        if case["grad"]:
            s.update(gout=normal(n, w), gtable=torch.empty(v, w, device="cuda"))
    elif case["op"] == "logprobs":
        r, c, k = case["rows"], case["vocab"], case["top"]
        tokens = (uniform(r) * c).long().clamp(0, c - 1)
        tokens = torch.where(uniform(r) < case["ignored"], torch.full_like(tokens, -100), tokens)
        s.update(logits=normal(r, c) * 2.0 + normal(c), tokens=tokens.to(I32), logprob=torch.empty(r, device="cuda"), entropy=torch.empty(r, device="cuda"),
                 lse=torch.empty(r, device="cuda"))
        if k:
            s.update(top_ids=torch.empty(r, k, dtype=I32, device="cuda"), top_logprobs=torch.empty(r, k, device="cuda"))
        if case["grad"]:
            s.update(g_logprob=-(0.5 + uniform(r)) / r, g_entropy=-0.01 * uniform(r) / r, glogits=torch.empty(r, c, device="cuda"))
    elif case["op"] == "cross":
        n, h, kv, lq, lk, d = (case[x] for x in ("batch", "heads", "kv_heads", "queries", "keys", "size"))
        order = torch.randperm(n, generator=g, device="cuda")
        lengths = torch.tensor(_lengths(case), device="cuda")[order]
        # projections leave heads side by side: [batch, length, heads * size]
        s.update(q=normal(n, lq, h * d), k=normal(n, lk, kv * d), v=normal(n, lk, kv * d), mask=(torch.arange(lk, device="cuda") < lengths[:, None]).float(),
                 out=torch.empty(n, lq, h * d, device="cuda"), lse=torch.empty(n, h, lq, device="cuda"), factor=float(np.float32(1.0 / math.sqrt(d))))
        if case["grad"]:
            s.update(gout=normal(n, lq, h * d), gq=torch.empty(n, lq, h * d, device="cuda"), gk=torch.empty(n, lk, kv * d, device="cuda"),
                     gv=torch.empty(n, lk, kv * d, device="cuda"))
    else:
        sizes = _sizes(case)
        starts, total = _starts(sizes)
        first = torch.zeros(total, dtype=I32, device="cuda")
        at = torch.tensor(starts, device="cuda")
        first[at] = at.to(I32)
        place = torch.arange(total, device="cuda", dtype=I32) - torch.cummax(first, 0)[0].to(I32)  # an element's index in its tensor
        count = torch.repeat_interleave(torch.tensor(sizes, device="cuda"), torch.tensor([(n + 255) // 256 * 256 for n in sizes], device="cuda"))
        inside = place < count  # what is not lies between two tensors, holds zeros and stays so
        zero = torch.zeros((), device="cuda")
        grad = torch.where(inside, normal(total) * 0.01 * torch.exp(normal(total)), zero)
        s.update(value=torch.where(inside, normal(total) * 0.02, zero), grad=grad, place=place, step_t=torch.full((1,), float(case["step"]), device="cuda"))
        m, v = grad * 0.3, grad * grad * 0.5
        if case["bits"] == 8:
            (m, ms), (v, vs) = _encode(m, True, None), _encode(v, False, None)
            s.update(m=m, v=v, m_scale=ms, v_scale=vs, m_out=torch.zeros(total, device="cuda"), v_out=torch.zeros(total, device="cuda"))
        else:
            s.update(m=m, v=v)
    torch.cuda.synchronize()
    return s


# ------------------------------------------------------------------------------------------------ 8-bit states
def _encode(x, signed, noise):
    """Blocks of 256 values -> bytes and a power of two a block.  A byte of an unsigned state holds 5 exponent and 3
    mantissa bits, of a signed one a sign, 4 and 3; the block's largest value, rounded up, has the largest exponent.
    `noise` (20 bits a value) is added below the kept bits before they are cut off; None adds half a step."""
    bits = x.abs().view(I32).view(-1, 256)
    e = ((bits.amax(1) + 0xFFFFF) >> 23).clamp(33, 255)
    top = 127 if signed else 255
    c = ((bits + (0x80000 if noise is None else noise.view(-1, 256))) >> 20) - (e * 8 + 7 - top)[:, None]
    c = c.clamp(0, top)
    if signed:
        c = torch.where((x.view(-1, 256) < 0) & (c > 0), c + 128, c)
    else:
        c = torch.where(bits > 0, c.clamp(1, top), c)  # a second moment that is not zero is not rounded to it
    return c.to(torch.uint8).view(-1), (e << 23).view(torch.float32)


def _decode(codes, scale, signed):
    c = codes.view(-1, 256).to(I32)
    e = scale.view(I32) >> 23
    top = 127 if signed else 255
    low = c & 127 if signed else c
    x = ((low + (e * 8 + 7 - top)[:, None]) << 20).view(torch.float32)
    x = torch.where(low == 0, torch.zeros_like(x), x)
    return (torch.where(c > 127, -x, x) if signed else x).reshape(-1)


def _noise(place, step):
    """32 bits for each element from its index, the step and the seed: 16 of them for either moment."""
    h = (place.long() * 0x9E3779B9 + (SEED + step * 0xAC502949)) & LOW
    h = ((h ^ (h >> 16)) * 0x82D3099F) & LOW
    h = ((h ^ (h >> 15)) * 0x2ACAE79F) & LOW
    h = h ^ (h >> 16)
    return ((h & 0xFFFF) << 4).to(I32), ((h >> 16) << 4).to(I32)


# ------------------------------------------------------------------------------------------------ the plain forms
def _plain_embedding(s):
    known = (s["ids"] >= 0) & (s["ids"] < s["vocab"])
    at = torch.where(known, s["ids"], 0).long()
    out = torch.where(known[:, None], s["table"][at] * s["factor"], 0.0)
    if not s["grad"]:
        return {"out": out}
    part = torch.where(known[:, None], s["gout"], 0.0)
    return {"out": out, "gtable": torch.zeros_like(s["table"]).index_add_(0, at, part) * s["factor"]}


def _plain_logprobs(s):
    c = s["vocab"]
    z = s["logits"] * s["scale"]
    known = (s["tokens"] >= 0) & (s["tokens"] < c)
    at = torch.where(known, s["tokens"], 0).long()
    d = z - z.amax(1, keepdim=True)
    e = torch.exp(d)
    total = e.sum(1)
    entropy = torch.log(total) - (e * d).sum(1) / total
    lp = d - torch.log(total)[:, None]
    r = {"logprob": torch.where(known, lp.gather(1, at[:, None])[:, 0], 0.0), "entropy": entropy}
    if s["top"]:
        # largest first, equal ones by index: the logit's bits in rising order above, the index in falling order below
        bits = s["logits"].view(I32).long()
        key = ((torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits)) << 32) + (LOW - torch.arange(c, device=z.device))
        ids = torch.topk(key, s["top"], dim=1)[0]
        ids = LOW - (ids & LOW)
        r.update(top_ids=ids.to(I32), top_logprobs=lp.gather(1, ids))
    if s["grad"]:
        p = torch.exp(lp)
        gl = torch.where(known, s["g_logprob"], 0.0)[:, None]
        grad = -gl * p - s["g_entropy"][:, None] * p * (lp + entropy[:, None])
        r["glogits"] = grad.scatter_add_(1, at[:, None], gl) * s["scale"]
    return r


def _plain_cross(s):
    n, h, kv, lq, lk, d = (s[x] for x in ("batch", "heads", "kv_heads", "queries", "keys", "size"))
    rows = h // kv * lq  # the heads that share keys, one below the other
    split = lambda x, heads: x.view(n, -1, heads, d).transpose(1, 2)  # noqa: E731
    merge = lambda x: x.reshape(n, h, lq, d).transpose(1, 2).reshape(n, lq, h * d)  # noqa: E731
    q = split(s["q"], h).reshape(n, kv, rows, d)
    k, v = split(s["k"], kv).contiguous(), split(s["v"], kv).contiguous()
    score = torch.matmul(q, k.transpose(2, 3).contiguous()) * s["factor"]
    score = torch.where(s["mask"][:, None, None, :] != 0, score, -math.inf)
    top = score.amax(3, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(3, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    o = torch.matmul(p, v)
    if not s["grad"]:
        return {"out": merge(o)}
    go = split(s["gout"], h).reshape(n, kv, rows, d)
    gp = torch.matmul(go, v.transpose(2, 3).contiguous())
    gs = p * (gp - (go * o).sum(3, keepdim=True)) * s["factor"]
    side = lambda x: x.transpose(1, 2).reshape(n, lk, kv * d)  # noqa: E731
    return {"out": merge(o), "gq": merge(torch.matmul(gs, k)), "gk": side(torch.matmul(gs.transpose(2, 3).contiguous(), q)),
            "gv": side(torch.matmul(p.transpose(2, 3).contiguous(), go))}


def _plain_adamw(s):
    lr, b1, b2, eps, decay, c1, c2 = _adamw_constants()
    eight = s["bits"] == 8
    m = _decode(s["m"], s["m_scale"], True) if eight else s["m"]
    v = _decode(s["v"], s["v_scale"], False) if eight else s["v"]
    g, t = s["grad"], s["step_t"].double()
    m = m * b1 + g * c1
    v = v * b2 + g * g * c2
    far = 1.0 / (1.0 - torch.pow(b1, t)).float()
    wide = 1.0 / (1.0 - torch.pow(b2, t)).float()
    s["value"] -= lr * (m * far / (torch.sqrt(v * wide) + eps) + decay * s["value"])
    if eight:
        nm, nv = _noise(s["place"], s["step"])
        m, ms = _encode(m, True, nm)
        v, vs = _encode(v, False, nv)
        s["m"].copy_(m), s["v"].copy_(v), s["m_scale"].copy_(ms), s["v_scale"].copy_(vs)
        m, v = _decode(m, ms, True), _decode(v, vs, False)
        return {"value": s["value"], "m": m, "v": v}
    s["m"].copy_(m), s["v"].copy_(v)
    return {"value": s["value"], "m": s["m"], "v": s["v"]}


# ------------------------------------------------------------------------------------------------ the library's calls
_handle = []


def _context():
    """The program's one context."""
    if not _handle:
        from sage_amd import Context
        _handle.append(Context(torch.cuda.current_device()))
    return _handle[0]


def _own(s):
    """The calls of one pass with the descriptors of the state's tensors; a program builds these once and keeps them, as it
    keeps a recorded graph's."""
    import ctypes as C

    from sage_amd import abi
    ctx = _context()
    lib, kept = ctx._lib, []
    kinds = {torch.float32: abi.FLOAT, I32: abi.INT}

    def desc(x, extents=None, strides=None, dtype=None, offset=0):
        ext = list(x.shape) if extents is None else list(extents)
        t = abi.sg_tensor(x.data_ptr(), kinds[x.dtype] if dtype is None else dtype, len(ext))
        t.extents[:len(ext)], t.strides[:len(ext)] = ext, list(x.stride()) if strides is None else list(strides)
        t.offset = offset
        kept.append(t)
        return C.byref(t)

    def opt(name, **how):
        return desc(s[name], **how) if name in s else None

    calls = []
    if s["op"] == "embedding":
        calls.append((lib.sg_embedding, (desc(s["table"]), desc(s["ids"]), C.c_float(s["factor"]), desc(s["out"]))))
        if s["grad"]:
            calls.append((lib.sg_embedding_grad, (desc(s["gout"]), desc(s["ids"]), C.c_float(s["factor"]), desc(s["gtable"]))))
    elif s["op"] == "logprobs":
        scale = C.c_float(s["scale"])
        calls.append((lib.sg_token_logprobs, (desc(s["logits"]), desc(s["tokens"]), scale, desc(s["logprob"]), desc(s["entropy"]), desc(s["lse"]),
                                              opt("top_ids", dtype=abi.UINT), opt("top_logprobs"))))
        if s["grad"]:
            calls.append((lib.sg_token_logprobs_grad, (desc(s["logits"]), desc(s["tokens"]), scale, desc(s["lse"]), desc(s["entropy"]),
                                                       desc(s["g_logprob"]), desc(s["g_entropy"]), desc(s["glogits"]))))
    elif s["op"] == "cross":
        n, h, kv, lq, lk, d = (s[x] for x in ("batch", "heads", "kv_heads", "queries", "keys", "size"))
        at_q = dict(extents=[n, h, lq, d], strides=[lq * h * d, d, h * d, 1])
        at_k = dict(extents=[n, kv, lk, d], strides=[lk * kv * d, d, kv * d, 1])
        ins = (desc(s["q"], **at_q), desc(s["k"], **at_k), desc(s["v"], **at_k), desc(s["mask"]), C.c_float(s["factor"]))
        calls.append((lib.sg_cross_attention, ins + (desc(s["out"], **at_q), desc(s["lse"]) if s["grad"] else None)))
        if s["grad"]:
            calls.append((lib.sg_cross_attention_grad, ins + (desc(s["out"], **at_q), desc(s["lse"]), desc(s["gout"], **at_q), desc(s["gq"], **at_q),
                                                              desc(s["gk"], **at_k), desc(s["gv"], **at_k))))
    else:
        lr, b1, b2, eps, decay, c1, c2 = _adamw_constants()
        sizes = _sizes(s)
        starts, _ = _starts(sizes)
        hyper, noise = abi.sg_adam_hyper(lr, b1, b2, c1, c2, eps, decay), C.c_uint32(SEED)

        def table(name, per, dtype=None):
            """One descriptor for each tensor; `per` of its elements share one of this buffer's."""
            t = (abi.sg_tensor * len(sizes))()
            for i, (n, at) in enumerate(zip(sizes, starts)):
                t[i].base, t[i].dtype, t[i].rank, t[i].offset = s[name].data_ptr(), abi.FLOAT if dtype is None else dtype, 1, at // per
                t[i].extents[0], t[i].strides[0] = (n + per - 1) // per, 1
            kept.append(t)
            return t

        if s["bits"] == 8:
            states = (table("m", 4, abi.UINT), table("v", 4, abi.UINT), table("m_scale", 256), table("v_scale", 256))
            calls.append((lib.sg_adamw_update, (len(sizes), table("value", 1), table("grad", 1)) + states + (desc(s["step_t"]), C.byref(hyper), noise)))
            calls.append((lib.sg_adamw_state_read, (len(sizes),) + states + (table("m_out", 1), table("v_out", 1))))
        else:
            calls.append((lib.sg_adamw_update, (len(sizes), table("value", 1), table("grad", 1), table("m", 1), table("v", 1), None, None,
                                                desc(s["step_t"]), C.byref(hyper), noise)))
        kept.append(hyper)
    names = {"embedding": ("out", "gtable"), "logprobs": ("logprob", "entropy", "top_ids", "top_logprobs", "glogits"), "cross": ("out", "gq", "gk", "gv")}
    if s["op"] == "adamw":
        eight = s["bits"] == 8
        outs = {"value": s["value"], "m": s["m_out" if eight else "m"], "v": s["v_out" if eight else "v"]}
    else:
        outs = {x: s[x] for x in names[s["op"]] if x in s}
    return ctx, calls, outs, kept


def run(state):
    if not own:
        return {"embedding": _plain_embedding, "logprobs": _plain_logprobs, "cross": _plain_cross, "adamw": _plain_adamw}[state["op"]](state)
    if "calls" not in state:
        state["calls"] = _own(state)
    ctx, calls, outs, _ = state["calls"]
    for fn, args in calls:
        ctx.check(fn(ctx.handle, *args))
    return outs


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    if case["op"] == "embedding":
        n, v, w = case["tokens"], case["vocab"], case["width"]
        rank = np.arange(v, dtype=np.float64)
        share = np.log((rank + 2) / (rank + 1)) / math.log(v + 1) * (1 - case["ignored"])
        distinct = float((1.0 - np.exp(n * np.log1p(-np.minimum(share, 1 - 1e-12)))).sum())
        moved = 4 * n + 4 * w * (distinct + n)
        if case["grad"]:
            moved += 4 * n + 4 * w * (n * (1 - case["ignored"]) + v)
        return {"bytes": moved, "flops": n * w * (2 if case["grad"] else 1)}
    if case["op"] == "logprobs":
        cells = case["rows"] * case["vocab"]
        return {"bytes": 4 * cells * (3 if case["grad"] else 1), "flops": cells * (11 if case["grad"] else 5)}
    if case["op"] == "cross":
        n, h, kv, lq, lk, d = (case[x] for x in ("batch", "heads", "kv_heads", "queries", "keys", "size"))
        seen = sum(_lengths(case))
        moved = 4 * (2 * n * h * lq * d + 2 * kv * seen * d + n * lk)
        if case["grad"]:
            moved += 4 * (3 * n * h * lq * d + 2 * kv * seen * d + 2 * n * kv * lk * d)
        return {"bytes": moved, "flops": (14 if case["grad"] else 4) * h * lq * seen * d}
    n = sum(_sizes(case))
    # value and gradient, the states twice; with 8-bit states also their values, which the pass returns
    return {"bytes": n * (12 + 16 if case["bits"] == 32 else 12 + 4 + 8), "flops": 14 * n}


# ------------------------------------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "embedding":
        # one column of ones for each known token: both directions as sums over rows, by token order
        ids = s["ids"].long()
        known = ids.ge(0) & ids.lt(case["vocab"])
        padded = torch.cat([s["table"].double(), torch.zeros(1, case["width"], dtype=torch.float64, device="cuda")])
        row = torch.where(known, ids, case["vocab"])
        r = {"out": padded[row] * s["factor"]}
        if case["grad"]:
            r["gtable"] = torch.zeros_like(padded).index_add_(0, row, s["gout"].double())[:-1] * s["factor"]
        return r
    if case["op"] == "logprobs":
        parts = [_exact_rows(case, s, at, min(case["rows"], at + 512)) for at in range(0, case["rows"], 512)]
        return {k: torch.cat([p[k] for p in parts]) for k in parts[0]}
    if case["op"] == "cross":
        parts = [_exact_sequence(case, s, b) for b in range(case["batch"])]
        return {k: torch.stack([p[k] for p in parts]) for k in parts[0]}
    lr, b1, b2, eps, decay, _, _ = _adamw_constants()
    g, t = s["grad"].double(), case["step"]
    m, v = s["m"], s["v"]
    if case["bits"] == 8:
        m, v = _decode(m, s["m_scale"], True), _decode(v, s["v_scale"], False)
    m = b1 * m.double() + (1 - b1) * g
    v = b2 * v.double() + (1 - b2) * g.square()
    value = s["value"].double()
    value = value - lr * (m / -math.expm1(t * math.log(b1)) / ((v / -math.expm1(t * math.log(b2))).sqrt() + eps) + decay * value)
    if case["bits"] == 8:  # which of two codes a state becomes hangs on its last bit
        return {"value": value, "m": None, "v": None}
    return {"value": value, "m": m, "v": v}


def _exact_rows(case, s, lo, hi):
    logits, tokens = s["logits"][lo:hi], s["tokens"][lo:hi].long()
    known = tokens.ge(0) & tokens.lt(case["vocab"])
    hot = torch.zeros_like(logits, dtype=torch.float64)
    hot[known.nonzero()[:, 0], tokens[known]] = 1.0
    z = logits.double() * float(np.float32(case["scale"]))
    lp = z - torch.logsumexp(z, 1, keepdim=True)
    p = lp.exp()
    entropy = -(p * lp).sum(1)
    r = {"logprob": (hot * lp).sum(1), "entropy": entropy}
    if case["top"]:
        order = torch.sort(logits, dim=1, descending=True, stable=True)[1][:, :case["top"]]
        r.update(top_ids=order.to(I32), top_logprobs=lp.gather(1, order))
    if case["grad"]:
        gl, ge = s["g_logprob"][lo:hi, None].double(), s["g_entropy"][lo:hi, None].double()
        r["glogits"] = float(np.float32(case["scale"])) * (gl * (hot - p * hot.sum(1, keepdim=True)) - ge * p * (lp + entropy[:, None]))
    return r


def _exact_sequence(case, s, b):
    h, kv, d = case["heads"], case["kv_heads"], case["size"]
    seen = s["mask"][b].nonzero()[:, 0]
    heads = lambda x, n: x[b].double().view(-1, n, d).permute(1, 0, 2).contiguous()  # noqa: E731
    q, k, v = heads(s["q"], h), heads(s["k"], kv), heads(s["v"], kv)
    owner = torch.arange(h, device="cuda") // (h // kv)
    ks, vs = k[:, seen][owner], v[:, seen][owner]
    p = torch.softmax(torch.bmm(q, ks.transpose(1, 2).contiguous()) * s["factor"], 2)
    o = torch.bmm(p, vs)
    join = lambda x: x.permute(1, 0, 2).reshape(-1, x.shape[0] * d)  # noqa: E731
    r = {"out": join(o)}
    if case["grad"]:
        go = heads(s["gout"], h)
        gs = p * (torch.bmm(go, vs.transpose(1, 2).contiguous()) - (go * o).sum(2, keepdim=True)) * s["factor"]
        gk, gv = torch.zeros_like(k), torch.zeros_like(v)
        gk[:, seen] = torch.bmm(gs.transpose(1, 2).contiguous(), q).view(kv, h // kv, -1, d).sum(1)
        gv[:, seen] = torch.bmm(p.transpose(1, 2).contiguous(), go).view(kv, h // kv, -1, d).sum(1)
        r.update(gq=join(torch.bmm(gs, ks)), gk=join(gk), gv=join(gv))
    return r
