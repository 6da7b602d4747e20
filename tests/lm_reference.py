"""Plain 64-bit implementations of the language-model operators, and how far 32-bit arithmetic may be from them.

U is half a step of fp32 relative to the value.  A sum of n terms in any order is off by at most (n + 1) U times the sum
of the terms' magnitudes (one rounding for each product and each addition on the longest path)."""
import numpy as np

U = 2.0 ** -24


def f32(x):
    return np.asarray(x, np.float32)


# ----------------------------------------------------------------------------- embedding
def embedding(table, ids, scale):
    ids = np.asarray(ids).astype(np.int64) & 0xFFFFFFFF
    known = ids < table.shape[0]
    rows = table[np.where(known, ids, 0)] * np.float32(scale)  # one rounding: the same bits
    return np.where(known[..., None], rows, np.float32(0))


def embedding_grad(gout, ids, rows, scale):
    """(sums, tolerance): a row of c tokens has c products (none: the scale comes last) and additions, and the scale."""
    ids = np.asarray(ids).astype(np.int64).reshape(-1) & 0xFFFFFFFF
    g = np.asarray(gout, np.float64).reshape(ids.size, -1)
    out, mag, count = np.zeros((rows, g.shape[1])), np.zeros((rows, g.shape[1])), np.zeros(rows)
    known = ids < rows
    np.add.at(out, ids[known], g[known])
    np.add.at(mag, ids[known], np.abs(g[known]))
    np.add.at(count, ids[known], 1)
    s = float(np.float32(scale))
    return out * s, (count + 2)[:, None] * U * mag * abs(s)


# ----------------------------------------------------------------------------- log probabilities
def logprobs(logits, tokens, scale, top=0):
    """dict of 64-bit results for finite or -inf logits [R, C]."""
    x = np.asarray(logits, np.float64)
    z = x * float(np.float32(scale))
    m = z.max(1, keepdims=True)
    empty = np.isneginf(m)
    d = np.where(empty, -np.inf, z - np.where(empty, 0.0, m))
    e = np.exp(d)
    s = e.sum(1, keepdims=True)
    with np.errstate(divide="ignore", invalid="ignore"):
        lp = np.where(empty, -np.inf, d - np.log(s))
        p = np.where(np.isneginf(lp), 0.0, np.exp(lp))
        h = -np.where(p > 0, p * lp, 0.0).sum(1)
        lse = np.where(empty, -np.inf, m + np.log(s))[:, 0]
    r = {"lse": lse, "entropy": h, "lp": lp, "p": p}
    if tokens is not None:
        t = np.asarray(tokens).astype(np.int64) & 0xFFFFFFFF
        known = t < x.shape[1]
        r["logprob"] = np.where(known, np.take_along_axis(lp, np.where(known, t, 0)[:, None], 1)[:, 0], 0.0)
        r["token"], r["known"] = t, known
    if top:
        order = np.argsort(-np.where(np.isnan(x), -np.inf, x), axis=1, kind="stable")[:, :top]
        r["top_ids"], r["top_logprobs"] = order.astype(np.uint32), np.take_along_axis(lp, order, 1)
    return r


def logprobs_tol(logits, scale):
    """(of a log probability, of the entropy), absolute, per row.  z is one rounding of |z| U, the difference to the maximum
    another of at most 2 |z| U, the exponential's argument in base 2 as much again, an exponential and a logarithm 4 U
    each; the sums go in chains of at most C/256 + 64 additions.  t/s weighs the same errors with the distances |d|."""
    x = np.asarray(logits, np.float64) * float(np.float32(scale))
    x = np.where(np.isfinite(x), x, 0.0)
    far = np.abs(x).max(1)
    rel = U * (x.shape[1] / 256 + 80 + 8 * far)
    return rel + 4 * U * far, 2 * rel * (2 + 2 * far)


def logprobs_grad(ref, scale, g_logprob=None, g_entropy=None):
    c = float(np.float32(scale))
    lp, p, h = ref["lp"], ref["p"], ref["entropy"][:, None]
    out = np.zeros_like(p)
    if g_logprob is not None:
        hot = np.zeros_like(p)
        rows = np.nonzero(ref["known"])[0]
        hot[rows, ref["token"][rows]] = 1.0
        gl = np.asarray(g_logprob, np.float64)[:, None] * ref["known"][:, None]
        out += gl * (hot - p)
    if g_entropy is not None:
        ge = np.asarray(g_entropy, np.float64)[:, None]
        out -= np.where(p > 0, ge * p * (np.where(p > 0, lp, 0.0) + h), 0.0)
    return np.where(np.isneginf(lp), 0.0, out) * c


def logprobs_grad_tol(ref, logits, scale, g_logprob=None, g_entropy=None):
    """p carries the relative error of a log probability, log p + H the two absolute ones, the rest 8 roundings."""
    c = float(np.float32(scale))
    t_lp, t_h = (t[:, None] for t in logprobs_tol(logits, scale))
    p = ref["p"]
    lph = np.where(p > 0, np.abs(np.where(p > 0, ref["lp"], 0.0) + ref["entropy"][:, None]), 0.0)
    gl = 0.0 if g_logprob is None else np.abs(np.asarray(g_logprob, np.float64))[:, None]
    ge = 0.0 if g_entropy is None else np.abs(np.asarray(g_entropy, np.float64))[:, None]
    rel = 2 * t_lp + 8 * U
    return c * (p * rel * (gl + ge * lph) + ge * p * (t_lp + t_h) + 8 * U * (gl * (p + 1) + ge * p * lph)) + 1e-37


# ----------------------------------------------------------------------------- cross attention
def cross(q, k, v, mask, scale):
    """q [N,H,Lq,D], k, v [N,G,Lk,D], mask [N,Lk] or None -> out, lse, P (64 bits)."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    n, h, _, _ = q.shape
    r = h // k.shape[1]
    seen = np.ones((n, k.shape[2]), bool) if mask is None else np.asarray(mask) != 0
    k = np.where(seen[:, None, :, None], k, 0.0).repeat(r, 1)
    v = np.where(seen[:, None, :, None], v, 0.0).repeat(r, 1)
    s = np.einsum("nhid,nhjd->nhij", q, k) * float(np.float32(scale))
    s = np.where(seen[:, None, None, :], s, -np.inf)
    m = s.max(3, keepdims=True)
    e = np.exp(s - np.where(np.isneginf(m), 0.0, m))
    l = e.sum(3, keepdims=True)
    p = e / np.where(l == 0, 1.0, l)
    with np.errstate(divide="ignore"):
        lse = np.where(np.isneginf(m), -np.inf, np.where(np.isneginf(m), 0.0, m) + np.log(l))[..., 0]
    return np.einsum("nhij,nhjd->nhid", p, v), lse, p


def cross_grad(q, k, v, mask, scale, gout):
    q, k, v, go = (np.asarray(x, np.float64) for x in (q, k, v, gout))
    n, g, lk, d = k.shape
    r = q.shape[1] // g
    out, _, p = cross(q, k, v, mask, scale)
    c = float(np.float32(scale))
    seen = np.ones((n, lk), bool) if mask is None else np.asarray(mask) != 0
    kk = np.where(seen[:, None, :, None], k, 0.0).repeat(r, 1)
    vv = np.where(seen[:, None, :, None], v, 0.0).repeat(r, 1)
    ds = p * (np.einsum("nhid,nhjd->nhij", go, vv) - (go * out).sum(3, keepdims=True))
    gq = np.einsum("nhij,nhjd->nhid", ds, kk) * c
    gk = (np.einsum("nhij,nhid->nhjd", ds, q) * c).reshape(n, g, r, lk, d).sum(2)
    gv = np.einsum("nhij,nhid->nhjd", p, go).reshape(n, g, r, lk, d).sum(2)
    return gq, gk, gv


def cross_tol(q, k, v, mask, scale, gout=None):
    """Tolerances of out, lse (and gq, gk, gv), element by element.  A score is a sum of D products, scaled, shifted and
    scaled again for base 2: E.  P is off by 2E (itself and the sum it is divided by) and a sum of Lk; the rest follows the
    formulas with magnitudes in the place of values."""
    q, k, v = (np.abs(np.asarray(x, np.float64)) for x in (q, k, v))
    n, g, lk, d = k.shape
    r = q.shape[1] // g
    c = abs(float(np.float32(scale)))
    out, lse, p = cross(q, k, v, mask, scale)  # only for shapes and magnitudes below
    seen = np.ones((n, lk), bool) if mask is None else np.asarray(mask) != 0
    k = np.where(seen[:, None, :, None], k, 0.0).repeat(r, 1)
    v = np.where(seen[:, None, :, None], v, 0.0).repeat(r, 1)
    s = np.einsum("nhid,nhjd->nhij", q, k) * c
    top = np.where(seen[:, None, None, :], s, 0.0).max(3, keepdims=True)
    e = (d + 8) * U * top  # of any score of the row, absolute
    rel = 2 * e + (lk + 64) * U
    t_out = rel * v.max(2, keepdims=True)
    t_lse = (rel + 4 * U * (top + 8))[..., 0]
    if gout is None:
        return t_out, t_lse
    go = np.abs(np.asarray(gout, np.float64))
    return t_out, t_lse, rel, e, (q, k, v, go, c, r, g, d)


def cross_grad_tol(q, k, v, mask, scale, gout):
    t_out, _, rel, _, (aq, ak, av, go, c, r, g, d) = cross_tol(q, k, v, mask, scale, gout)
    out, lse, p = cross(q, k, v, mask, scale)
    n, h, lq, _ = aq.shape
    lk = ak.shape[2]
    dp = np.einsum("nhid,nhjd->nhij", go, av)
    delta = (go * np.abs(out)).sum(3, keepdims=True)
    t_delta = (d + 2) * U * delta + (go * t_out).sum(3, keepdims=True)
    # Below the smallest normal number 2^-126 an exponential has no relative precision: it is a multiple of 2^-149, or 0
    # where the hardware flushes.  So P is off by 2^-126 besides, whatever it is, in everything that it weighs.
    tiny = 2.0 ** -126
    t_ds = p * ((rel + 8 * U) * (dp + delta) + (d + 4) * U * dp + t_delta) + tiny * (dp + delta)
    ds = p * (dp + delta)
    t_gq = c * (np.einsum("nhij,nhjd->nhid", t_ds, ak) + (lk + 8) * U * np.einsum("nhij,nhjd->nhid", ds, ak))
    rows = lq * r + 8
    fold = lambda x: x.reshape(n, g, r, lk, d).sum(2)  # noqa: E731
    t_gk = fold(c * (np.einsum("nhij,nhid->nhjd", t_ds, aq) + rows * U * np.einsum("nhij,nhid->nhjd", ds, aq)))
    t_gv = fold(np.einsum("nhij,nhid->nhjd", p * rel + tiny, go) + rows * U * np.einsum("nhij,nhid->nhjd", p, go))
    return t_gq, t_gk, t_gv


# ----------------------------------------------------------------------------- AdamW
def adamw_moments(m, v, g, beta1, beta2):
    """The moments in fp32, each product and sum rounded on its own: the same bits as the kernel's."""
    b1, b2 = np.float32(beta1), np.float32(beta2)
    return f32(f32(m) * b1 + f32(g) * (np.float32(1) - b1)), f32(f32(v) * b2 + f32(g) * f32(g) * (np.float32(1) - b2))


def adamw_value(value, m, v, t, lr, beta1, beta2, eps, decay):
    """(64-bit value, tolerance): the update is about 16 roundings and library functions of at most 4 U, the value one more."""
    b1, b2 = float(np.float32(beta1)), float(np.float32(beta2))
    lr, eps, decay = (float(np.float32(x)) for x in (lr, eps, decay))
    m, v, x = (np.asarray(a, np.float64) for a in (m, v, value))
    step = m / (1 - b1 ** t) / (np.sqrt(v / (1 - b2 ** t)) + eps)
    return x - lr * (step + decay * x), 2 * U * np.abs(x) + lr * (64 * U * np.abs(step) + 8 * U * decay * np.abs(x)) + 1e-44


def noise(n, t, seed):
    i = np.arange(n, dtype=np.uint64)
    low = np.uint64(0xFFFFFFFF)
    h = (i * np.uint64(0x9E3779B9) + np.uint64(seed) + np.uint64(t) * np.uint64(0xAC502949)) & low
    h = ((h ^ (h >> np.uint64(16))) * np.uint64(0x82D3099F)) & low
    h = ((h ^ (h >> np.uint64(15))) * np.uint64(0x2ACAE79F)) & low
    h ^= h >> np.uint64(16)
    return (h & np.uint64(0xFFFF)).astype(np.int64), (h >> np.uint64(16)).astype(np.int64)


def encode(x, signed, noise16):
    """Bytes [n] and scales [ceil(n/256)] of fp32 values."""
    x = f32(x)
    n, nb = x.size, -(-x.size // 256)
    bits = np.zeros(nb * 256, np.int64)
    bits[:n] = np.abs(x).view(np.uint32)
    r = np.zeros(nb * 256, np.int64)
    r[:n] = noise16
    bits, r = bits.reshape(nb, 256), r.reshape(nb, 256)
    e = np.clip((bits.max(1) + 0xFFFFF) >> 23, 33, 255)
    top = 127 if signed else 255
    c = np.clip(((bits + (r << 4)) >> 20) - (e * 8 + 7 - top)[:, None], 0, top)
    if not signed:
        c = np.where((bits > 0) & (c == 0), 1, c)
    c = c.reshape(-1)[:n]
    if signed:
        c = np.where((x < 0) & (c > 0), c + 128, c)
    scale = np.where(e == 255, 0x7FC00000, e << 23).astype(np.uint32).view(np.float32)
    return c.astype(np.uint8), scale


def decode(codes, scale, signed):
    e = (scale.view(np.uint32).astype(np.int64) >> 23) & 255
    e = e.repeat(256)[:codes.size]
    top = 127 if signed else 255
    low = (codes & 127 if signed else codes).astype(np.int64)
    x = (np.where(low > 0, low + e * 8 + 7 - top, 0) << 20).astype(np.uint32).view(np.float32)
    x = np.where(low == 0, np.float32(0), x)
    x = np.where(e == 255, np.float32(np.nan), x)
    return np.where(signed & (codes > 127), -x, x).astype(np.float32)


def pack(codes):
    """Bytes four to a word, element 4w + j in byte j of word w."""
    b = np.zeros(-(-codes.size // 4) * 4, np.uint8)
    b[:codes.size] = codes
    return b.view(np.uint32)


def unpack(words, n):
    return np.ascontiguousarray(words).view(np.uint8)[:n].copy()
