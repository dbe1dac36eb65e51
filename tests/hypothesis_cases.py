"""Plain 64-bit forms of the tree and beam operators, and their tolerances."""
import numpy as np

from oracle import oracle

D, H, HD, QKV = 768, 12, 64, 2304
U = 2.0 ** -24  # half a step of an fp32 value near 1



def inv_freq():
    """The graph's fp32 frequencies: torch's fp32 evaluation, six of which sit
    one step away from the correctly rounded value."""
    import torch
    return (1.0 / (10000 ** (torch.arange(0, HD, 2).float() / HD))).numpy()


def rope32(x, pos):
    """x [..., H * 64] fp32 at positions pos [...], in the fp32 operations that
    the rings use (bit for bit): cos and sin in double of the fp32 angle."""
    x = x.reshape(*x.shape[:-1], x.shape[-1] // HD, HD // 2, 2).astype(np.float32)
    a = (np.asarray(pos).astype(np.float32)[..., None] * inv_freq()).astype(np.float64)[..., None, :]
    c, s = np.cos(a).astype(np.float32), np.sin(a).astype(np.float32)
    out = np.stack((x[..., 0] * c + -x[..., 1] * s, x[..., 1] * c + x[..., 0] * s), -1)
    return out.reshape(*out.shape[:-3], out.shape[-3] * HD)


def chains(parent, n):
    out = []
    for i in range(n):
        out.append((out[parent[i]] if parent[i] >= 0 else []) + [i])
    return out


def random_parents(rng, B, T, back=5):
    return np.maximum(np.arange(T)[None] - rng.integers(1, back + 2, (B, T)), -1).astype(np.int32)


def tree_reference(ring, qkv, parent, pos0, n, bf16):
    """ring = (k [C][768], v, slot_pos [C]) as stored; one sequence.  Returns
    (out [n][768], bound [n][768]) in 64 bits.

    bound, in steps U of fp32 arithmetic: a score is a sum of 64 products (and
    the roped, scaled q, which is the same bits): at most 66 U sum |q k| / 8.  Its
    weight exp(s - m) adds |s - m| 2 U (the difference, and the product with
    log2 e) and 4 U (the hardware exponential and the rescaling of a state).
    A quotient of two sums of weights doubles that, and the sums themselves
    round at most once per term: (terms + 16) U, all relative to sum w |v| / sum w.
    """
    k, v, sp = ring
    C = len(sp)
    q = rope32(qkv[:n, :D], pos0 + np.array([len(c) - 1 for c in chains(parent, n)], np.int64))
    ks, vs = np.empty((n, D), np.float32), qkv[:n, 2 * D:].astype(np.float32)
    cs = chains(parent, n)
    for i, c in enumerate(cs):
        ks[i] = rope32(qkv[i, D:2 * D], pos0 + len(c) - 1)
    if bf16:
        ks, vs = oracle.bf16_round(ks), oracle.bf16_round(vs)
    out, bound = np.zeros((n, D)), np.zeros((n, D))
    for i, c in enumerate(cs):
        pos = pos0 + len(c) - 1
        c = c[-C:]  # those that its window holds
        live = (sp >= 0) & (sp < pos0) & (pos - sp.astype(np.int64) < C)
        kk = np.concatenate((k[live], ks[c])).astype(np.float64).reshape(-1, H, HD)
        vv = np.concatenate((v[live], vs[c])).astype(np.float64).reshape(-1, H, HD)
        qq = q[i].astype(np.float64).reshape(H, HD)
        with np.errstate(invalid="ignore", over="ignore"):
            s = np.einsum("nhd,hd->hn", kk, qq) / 8
            a = np.einsum("nhd,hd->hn", np.abs(kk), np.abs(qq)) / 8
            m = s.max(1, keepdims=True)
            w = np.exp(s - m)
            o = np.einsum("hn,nhd->hd", w, vv) / w.sum(1)[:, None]
            d = (66 * a + 2 * np.abs(s - m) + 4).max(1) * 2 + len(kk) + 16
            bo = np.einsum("hn,nhd->hd", w, np.abs(vv)) / w.sum(1)[:, None] * d[:, None] * U
        out[i], bound[i] = o.reshape(-1), bo.reshape(-1)
    return out, bound


def beam_reference(logits, scores, n_out, done=None, end_id=-1, seen=None, penalty=1.2):
    """One voice: logits [W][V] fp32, scores [W].  (scores, parent, token, done)
    of the n_out best, by a full sort: c falling, then beam, logit, id."""
    W, V = logits.shape
    z = np.where(np.isnan(logits), -np.inf, logits).astype(np.float32)
    if seen is not None:
        bits = np.unpackbits(np.ascontiguousarray(seen).view(np.uint8), axis=-1,
                             bitorder="little")[:, :V].astype(bool)
        p = np.float32(penalty)
        z = np.where(bits, np.where(z < 0, z * p, z / p), z).astype(np.float32)
    rows = []
    for w in range(W):
        sc = float(scores[w])
        if done is not None and done[w]:
            rows.append((sc, w, 0.0, end_id))
            continue
        m = z[w].max()
        if m == -np.inf:
            continue
        with np.errstate(invalid="ignore"):
            d = np.where(z[w] == m, 0.0, z[w].astype(np.float64) - np.float64(m))
            c = sc + (d - np.log(np.exp(d).sum()))
        top = np.lexsort((np.arange(V), -z[w].astype(np.float64)))[:n_out]
        rows += [(c[v], w, -float(z[w, v]), int(v)) for v in top if z[w, v] > -np.inf]
    rows = sorted((r for r in rows if r[0] > -np.inf), key=lambda r: (-r[0], r[1], r[2], r[3]))[:n_out]
    out = np.full(n_out, -np.inf), np.full(n_out, -1), np.full(n_out, -1), np.ones(n_out, int)
    for k, (c, w, _, v) in enumerate(rows):
        out[0][k], out[1][k], out[2][k], out[3][k] = c, w, v, int(end_id >= 0 and v == end_id)
    return out
