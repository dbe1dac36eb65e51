"""Several hypotheses per voice: the operators, sized over the range of their use.

A program that decodes with more than one hypothesis per voice does one of two
things.  It drafts a tree of coming rows, has every node of it attend the
voice's ring and its own ancestors in one pass, and then commits the rows of
the path that the model confirms.  Or it keeps a beam: each step it takes the
best continuations over all of a voice's beams and the vocabulary, and moves
the rings of the beams that go on to where they go on.  The cases take these
four operators from one voice (an interactive program) to a server's batch, in
both storage types of the rings and both types of the activations.

With `own` false a pass is the plain form: elementary torch operations in 32
bits (64 where angles, long sums and near ties need them).  With `own` true it
is the calls of mockbird_amd.Context.  Inputs come from the seed alone and are
the same for both.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

D, H, HD, QKV, CODES, LAYERS = 768, 12, 64, 2304, 1024, 12
PENALTY = 1.2
END = 7  # the id that ends a beam


def listed():
    return [
        # One layer's attention of drafted trees.  One interactive voice with a
        # short draft, in fp32.
        {"name": "tree_1x8_f32", "op": "tree", "voices": 1, "nodes": 8, "shortest": 8,
         "capacity": 1024, "kv": "f32", "q": "f32"},
        # A small server: eight voices with up to 16 nodes each.
        {"name": "tree_8x16_bf16", "op": "tree", "voices": 8, "nodes": 16, "shortest": 5,
         "capacity": 2048, "kv": "bf16", "q": "f32"},
        # Wide fp32 trees of odd and ragged sizes over an odd ring.
        {"name": "tree_24x61_f32", "op": "tree", "voices": 24, "nodes": 61, "shortest": 17,
         "capacity": 1001, "kv": "f32", "q": "f32"},
        # The server's batch: 64 voices on long texts, bf16 throughout.
        {"name": "tree_64x16_bf16", "op": "tree", "voices": 64, "nodes": 16, "shortest": 16,
         "capacity": 2048, "kv": "bf16", "q": "bf16"},
        # Few voices with the widest trees over a very long cache.
        {"name": "tree_3x64_long_bf16", "op": "tree", "voices": 3, "nodes": 64, "shortest": 40,
         "capacity": 16384, "kv": "bf16", "q": "f32"},
        # The accepted path of every layer into the rings: one voice, and the
        # server's batch.
        {"name": "commit_1x5_f32", "op": "commit", "voices": 1, "nodes": 24, "path": 5,
         "capacity": 256, "kv": "f32", "q": "f32"},
        {"name": "commit_64x8_bf16", "op": "commit", "voices": 64, "nodes": 16, "path": 8,
         "capacity": 128, "kv": "bf16", "q": "bf16"},
        # A beam over one audio channel's codes for one voice; for 64 voices
        # with the repetition penalty; and over the text vocabulary.
        {"name": "beam_1x4_codes", "op": "beam", "voices": 1, "beams": 4, "vocab": CODES,
         "choose": 4, "logits": "f32", "penalty": False},
        {"name": "beam_64x8_codes_penalty", "op": "beam", "voices": 64, "beams": 8, "vocab": CODES,
         "choose": 8, "logits": "f32", "penalty": True},
        {"name": "beam_16x8_text", "op": "beam", "voices": 16, "beams": 8, "vocab": 32000,
         "choose": 16, "logits": "f32", "penalty": False},
        # The rings of every layer follow the chosen beams, over the rows that
        # are not the shared prompt's: one voice, and a server's 32.
        {"name": "reorder_1x4_f32", "op": "reorder", "voices": 1, "beams": 4, "rows": 60,
         "capacity": 512, "kv": "f32"},
        {"name": "reorder_32x4_bf16", "op": "reorder", "voices": 32, "beams": 4, "rows": 300,
         "capacity": 512, "kv": "bf16"},
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))

    op = rng.choice(("tree", "tree", "commit", "beam", "beam", "reorder"))
    kv, q = rng.choice(("f32", "bf16")), rng.choice(("f32", "bf16"))
    if op == "tree":
        voices, nodes = log(1, 64), log(1, 64)
        slots = min(131072 if kv == "bf16" else 65536, (1 << 21) // nodes)
        return {"op": op, "voices": voices, "nodes": nodes, "shortest": rng.randint(1, nodes),
                "capacity": log(64, min(16384, slots // voices)), "kv": kv, "q": q}
    if op == "commit":
        path = log(1, 16)
        return {"op": op, "voices": log(1, 64), "nodes": rng.randint(path, 64), "path": path,
                "capacity": rng.randint(32, 128), "kv": kv, "q": q}
    if op == "beam":
        voices, beams = log(1, 64), log(1, 16)
        return {"op": op, "voices": voices, "beams": beams,
                "vocab": log(256, min(32000, 4096000 // (voices * beams))),
                "choose": rng.choice((beams, 2 * beams)), "logits": q,
                "penalty": rng.random() < 0.5}
    voices, beams = log(1, 32), log(2, 16)
    rows = log(8, min(1000, 38400 // (voices * beams)))
    return {"op": op, "voices": voices, "beams": beams, "rows": rows,
            "capacity": rng.randint(rows, 2 * rows), "kv": kv}


def work(case):
    op, e, s = case["op"], 2 if case.get("kv") == "bf16" else 4, 2 if case.get("q") == "bf16" else 4
    if op == "tree":
        # positions U[1, 3C): five sixths of the slots are live
        B, T = case["voices"], (case["nodes"] + case["shortest"]) / 2
        slots = B * case["capacity"] * 5 / 6
        return {"bytes": slots * (2 * D * e + 4) + B * T * (QKV * s + D * 4),
                "flops": 4 * D * T * (slots + B * T / 4)}
    if op == "commit":
        # K and V of the path's rows, read and written
        return {"bytes": LAYERS * case["voices"] * (case["path"] + 1) / 2 * (2 * D * (s + e) + 4),
                "flops": 0}
    if op == "beam":
        rows, V = case["voices"] * case["beams"], case["vocab"]
        words = (rows + case["voices"] * case["choose"]) * V / 8
        return {"bytes": rows * V * (2 if case["logits"] == "bf16" else 4)
                + (words if case["penalty"] else 0), "flops": 4 * rows * V}
    # parents drawn with repeats: each beam that is some parent is read once,
    # each beam that is not its own is written
    W, n = case["beams"], (case["rows"] + 1) // 2 + case["rows"] // 4
    moved = case["voices"] * W * ((1 - (1 - 1 / W) ** W) + (1 - 1 / W))
    return {"bytes": LAYERS * moved * n * (2 * D * e + 4), "flops": 0}


# ------------------------------------------------------------------- inputs

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def _i32(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()


def _dtype(name):
    return torch.bfloat16 if name == "bf16" else torch.float32


def _inv():
    """The graph's frequencies of the 32 pairs of a head, as it holds them."""
    return (1.0 / (10000 ** (torch.arange(0, HD, 2).float() / HD))).cuda()


def _slot_positions(pos0, capacity):
    """The positions [B][C] that a wrapping ring's slots hold after pos0[b] rows."""
    slot = np.arange(capacity)
    last = pos0[:, None] - 1
    p = last - (last - slot) % capacity
    return np.where(p >= 0, p, -1).astype(np.int32)


def _rings(g, layers, seqs, capacity, kv, pos0):
    """K, V [layers, seqs, H, C, 64] and positions [layers, seqs, C]."""
    shape = (layers, seqs, H, capacity, HD)
    sp = _i32(_slot_positions(pos0, capacity)).expand(layers, seqs, capacity).contiguous()
    return _randn(g, *shape, dtype=_dtype(kv)), _randn(g, *shape, dtype=_dtype(kv)), sp


def _tree_inputs(case, seed):
    """Trees drafted as programs draft them: a node's parent is one of the
    last few before it, so that chains and branches mix."""
    B, T = case["voices"], case["nodes"]
    r = np.random.default_rng([seed, 1])
    n = r.integers(case.get("shortest", T), T + 1, size=B)
    n[0] = T
    parent = np.arange(T)[None] - r.integers(1, 7, size=(B, T))
    pos0 = r.integers(1, 3 * case["capacity"], size=B).astype(np.int32)
    return n.astype(np.int32), np.maximum(parent, -1).astype(np.int32), pos0


def _commit_inputs(case, seed):
    """Paths of ascending nodes, of 1 to case["path"] rows."""
    B = case["voices"]
    r = np.random.default_rng([seed, 2])
    path = np.sort(np.argsort(r.random((B, case["nodes"])), 1)[:, :case["path"]], 1)
    n = r.integers(1, case["path"] + 1, size=B)
    pos0 = r.integers(1, 3 * case["capacity"], size=B)
    return path.astype(np.int32), n.astype(np.int32), pos0.astype(np.int32)


# ------------------------------------------------------------------- prepare

def prepare(case, seed):
    return globals()["_prepare_" + case["op"]](case, seed)


def _own_rings(state):
    """The rings as the library holds them, in place of the plain tensors."""
    import mockbird_amd as mb

    k, v, sp = state["rings"]
    layers, seqs, _, capacity, _ = k.shape
    ctx = mb.Context(n_layers=layers, capacity=capacity, max_seqs=seqs, max_rows=64, vocab=16,
                     kv_dtype=mb.MB_KV_BF16 if k.dtype == torch.bfloat16 else mb.MB_KV_F32)
    ctx.set_stream(torch.cuda.current_stream().cuda_stream)
    views = [torch.as_tensor(a, device="cuda") for a in ctx.ring_view()]
    for to, src in zip(views, (k, v, sp)):
        to.view(src.dtype).copy_(src)
    state["rings"] = [to.view(src.dtype) for to, src in zip(views, (k, v, sp))]
    state["ctx"] = ctx


def _prepare_tree(case, seed):
    g = _generator(seed)
    n, parent, pos0 = _tree_inputs(case, seed)
    B, T = case["voices"], case["nodes"]
    state = {"case": case, "rings": _rings(g, 1, B, case["capacity"], case["kv"], pos0),
             "qkv": _randn(g, B, T, QKV, dtype=_dtype(case["q"])), "parent": _i32(parent),
             "pos0": _i32(pos0), "n": _i32(n), "max_pos": int(pos0.max()) + T - 1, "inv": _inv(),
             "out": torch.zeros((B, T, D), device="cuda")}
    if own:
        _own_rings(state)
        size = state["ctx"].tree_attention_work(B, T, state["max_pos"])
        state["work"] = torch.empty(size, dtype=torch.uint8, device="cuda")
    return state


def _prepare_commit(case, seed):
    g = _generator(seed)
    path, n, pos0 = _commit_inputs(case, seed)
    B = case["voices"]
    state = {"case": case, "rings": _rings(g, LAYERS, B, case["capacity"], case["kv"], pos0),
             "qkv": _randn(g, LAYERS, B, case["nodes"], QKV, dtype=_dtype(case["q"])),
             "path": _i32(path), "n": _i32(n), "pos0": _i32(pos0), "inv": _inv()}
    if own:
        _own_rings(state)
    return state


def _beam_inputs(case, seed):
    """Logits of a peaked distribution, running scores with a few beams that
    have ended, and histories of 40 ids per beam."""
    g = _generator(seed)
    B, W, V = case["voices"], case["beams"], case["vocab"]
    logits = _randn(g, B, W, V).mul_(3).to(_dtype(case["logits"]))
    scores = _randn(g, B, W).mul_(2).sub_(20)
    r = np.random.default_rng([seed, 3])
    done = _i32(r.random((B, W)) < 0.1)
    seen = None
    if case["penalty"]:
        words = np.zeros((B, W, -(-V // 32)), np.uint32)
        ids = r.integers(0, V, size=(B, W, 40))
        b, w = np.arange(B)[:, None, None], np.arange(W)[None, :, None]
        np.bitwise_or.at(words, (b, w, ids // 32), np.uint32(1) << (ids % 32).astype(np.uint32))
        seen = _i32(words.view(np.int32))
    return logits, scores, done, seen


def _prepare_beam(case, seed):
    logits, scores, done, seen = _beam_inputs(case, seed)
    B, W, V, n = case["voices"], case["beams"], case["vocab"], case["choose"]
    state = {"case": case, "logits": logits, "scores": scores, "done": done, "seen": seen,
             "by": torch.tensor(PENALTY, dtype=torch.float32, device="cuda")}
    if own:
        import mockbird_amd as mb

        ctx = mb.Context(n_layers=1, capacity=8, max_seqs=1, max_rows=8, vocab=16)
        ctx.set_stream(torch.cuda.current_stream().cuda_stream)
        state["ctx"] = ctx
        state["work"] = torch.empty(ctx.beam_select_work(B, W, V, n), dtype=torch.uint8,
                                    device="cuda")
        state["out"] = {"scores": torch.zeros((B, n), device="cuda")}
        for name in ("parent", "token", "done"):
            state["out"][name] = torch.zeros((B, n), dtype=torch.int32, device="cuda")
        if seen is not None:
            state["out"]["seen"] = torch.zeros((B, n, seen.shape[-1]), dtype=torch.int32,
                                               device="cuda")
    return state


def _prepare_reorder(case, seed):
    B, W, n = case["voices"], case["beams"], case["rows"]
    r = np.random.default_rng([seed, 4])
    parent = r.integers(0, W, size=(B, W))
    count = r.integers((n + 1) // 2, n + 1, size=B)
    first = r.integers(0, 2 * case["capacity"], size=B)
    last = (first + count).repeat(W)
    state = {"case": case, "parent": _i32(parent), "first": _i32(first), "last": _i32(first + count),
             "rings": _rings(_generator(seed), LAYERS, B * W, case["capacity"], case["kv"], last)}
    if own:
        _own_rings(state)
    return state


# ----------------------------------------------------------------------- run

def run(state):
    return globals()["_run_" + state["case"]["op"]](state, state["case"])


def _half(t):
    """1 (MB_DT_BF16) for bf16 tensors, 0 (MB_DT_F32) for fp32 ones."""
    return int(t.dtype == torch.bfloat16)


def _rope(x, pos, inv):
    """x [..., heads, 64] in 32 bits at positions pos [...]: the angle is the
    fp32 product of the position and the graph's fp32 frequencies."""
    a = (pos.to(torch.float32)[..., None] * inv).double()[..., None, :]
    c, s = a.cos().float(), a.sin().float()
    x0, x1 = x[..., 0::2], x[..., 1::2]
    return torch.stack((x0 * c - x1 * s, x1 * c + x0 * s), -1).flatten(-2)


def _twice(m):
    return (m @ m).clamp_(max=1)


def _ancestors(parent):
    """[B, T, T]: 1 where column j is row i itself or an ancestor of it, from
    the 64th power of the matrix of single steps."""
    T = parent.shape[1]
    node = torch.arange(T, device=parent.device)
    step = ((parent[..., None] == node) | (node[:, None] == node)).float()
    return _twice(_twice(_twice(_twice(_twice(_twice(step))))))


def _run_tree(s, case):
    if own:
        ctx, B, T = s["ctx"], case["voices"], case["nodes"]
        ctx.tree_attention_dev(0, B, T, s["qkv"].data_ptr(), s["parent"].data_ptr(),
                               s["pos0"].data_ptr(), s["n"].data_ptr(), s["max_pos"],
                               s["out"].data_ptr(), s["work"].data_ptr(), s["work"].numel(),
                               qkv_dtype=_half(s["qkv"]))
        return s["out"]
    k, v, sp = (t[0] for t in s["rings"])
    T, C = case["nodes"], case["capacity"]
    anc = _ancestors(s["parent"])
    pos0 = s["pos0"][:, None]
    pos = pos0 + anc.sum(-1).int() - 1
    x = s["qkv"].float().unflatten(-1, (3, H, HD))
    q = _rope(x[:, :, 0], pos, s["inv"]).transpose(1, 2) * 0.125
    kn = _rope(x[:, :, 1], pos, s["inv"]).to(k.dtype).float().transpose(1, 2)
    vn = x[:, :, 2].to(v.dtype).float().transpose(1, 2)
    cached = (sp >= 0) & (sp < pos0)
    cached = cached[:, None] & (pos[..., None] - sp[:, None] < C)
    score = torch.cat((q @ k.float().transpose(-1, -2), q @ kn.transpose(-1, -2)), -1)
    sees = torch.cat((cached, anc > 0), -1)[:, None]
    score = torch.where(sees, score, -torch.inf)
    p = (score - score.amax(-1, keepdim=True)).exp()
    o = (p[..., :C] @ v.float() + p[..., C:] @ vn) / p.sum(-1, keepdim=True)
    there = torch.arange(T, device="cuda") < s["n"][:, None]
    return torch.where(there[..., None], o.transpose(1, 2).flatten(2), 0)


def _run_commit(s, case):
    k, v, sp = s["rings"]
    B, P, C = case["voices"], case["path"], case["capacity"]
    if own:
        s["ctx"].tree_commit_dev(0, LAYERS, B, case["nodes"], s["qkv"].data_ptr(),
                                 s["pos0"].data_ptr(), P, s["path"].data_ptr(), s["n"].data_ptr(),
                                 qkv_dtype=_half(s["qkv"]))
        return s["rings"]
    # rows behind a path's end repeat its last
    row = torch.minimum(torch.arange(P, device="cuda"), s["n"][:, None] - 1)
    pos = s["pos0"][:, None] + row
    slot, b = pos.long() % C, torch.arange(B, device="cuda")[:, None]
    x = s["qkv"][:, b, s["path"].gather(1, row).long()].float().unflatten(-1, (3, H, HD))
    k[:, b, :, slot] = _rope(x[:, :, :, 1], pos, s["inv"]).to(k.dtype).permute(1, 2, 0, 3, 4)
    v[:, b, :, slot] = x[:, :, :, 2].to(v.dtype).permute(1, 2, 0, 3, 4)
    sp[:, b, slot] = pos.int()
    return s["rings"]


def _run_beam(s, case):
    B, W, V, n = case["voices"], case["beams"], case["vocab"], case["choose"]
    seen = s["seen"]
    if own:
        o = s["out"]
        s["ctx"].beam_select_dev(
            B, W, V, n, s["logits"].data_ptr(), s["scores"].data_ptr(), o["scores"].data_ptr(),
            o["parent"].data_ptr(), o["token"].data_ptr(), s["work"].data_ptr(),
            s["work"].numel(), logits_dtype=_half(s["logits"]), end_id=END,
            done_ptr=s["done"].data_ptr(), done_out_ptr=o["done"].data_ptr(),
            seen_ptr=seen.data_ptr() if seen is not None else None,
            seen_out_ptr=o["seen"].data_ptr() if seen is not None else None, penalty=PENALTY)
        return o
    z = s["logits"].float()
    bit = torch.arange(32, device="cuda", dtype=torch.int32)
    if seen is not None:
        used = ((seen[..., None] >> bit) & 1).flatten(2)[..., :V] != 0
        z = torch.where(used, torch.where(z < 0, z * s["by"], z / s["by"]), z)
    z = z.double()  # scores of two beams may be a few units of the 24th bit apart
    z = z - z.amax(-1, keepdim=True)
    c = s["scores"].double()[..., None] + (z - z.exp().sum(-1, keepdim=True).log())
    # an ended beam goes on as it is, by END alone
    ended = s["done"][..., None] != 0
    at_end = torch.arange(V, device="cuda") == END
    c = torch.where(ended, torch.where(at_end, s["scores"].double()[..., None], -torch.inf), c)
    c = torch.nn.functional.pad(c.flatten(1), (0, max(0, n - W * V)), value=-torch.inf)
    best, at = c.sort(dim=-1, descending=True, stable=True)
    best, at = best[:, :n], at[:, :n]
    parent, token = at // V, at % V
    none = best == -torch.inf  # fewer continuations than are asked for
    o = {"scores": best.float(), "parent": torch.where(none, -1, parent).int(),
         "token": torch.where(none, -1, token).int(), "done": (none | (token == END)).int()}
    if seen is not None:
        words = seen.gather(1, parent[..., None].expand(B, n, seen.shape[-1]))
        word = (token // 32)[..., None]
        new = words.gather(2, word) | (1 << (token % 32))[..., None].int()
        o["seen"] = torch.where(none[..., None], 0, words.scatter(2, word, new))
    return o


def _run_reorder(s, case):
    k, v, sp = s["rings"]
    B, W, n, C = case["voices"], case["beams"], case["rows"], case["capacity"]
    if own:
        s["ctx"].ring_reorder_dev(0, LAYERS, B * W, W, s["parent"].data_ptr(),
                                  s["first"].data_ptr(), s["last"].data_ptr(), n)
        return s["rings"]
    # rows behind a voice's last repeat it
    row = torch.minimum(s["first"][:, None] + torch.arange(n, device="cuda"), s["last"][:, None] - 1)
    slot = (row.long() % C).repeat_interleave(W, 0)
    to = torch.arange(B * W, device="cuda")[:, None]
    src = (s["parent"] + W * torch.arange(B, device="cuda")[:, None]).reshape(-1, 1)
    k[:, to, :, slot] = k[:, src, :, slot]
    v[:, to, :, slot] = v[:, src, :, slot]
    sp[:, to, slot] = sp[:, src, slot]
    return s["rings"]


# --------------------------------------------------------------------- exact

def exact(case, seed):
    if case["op"] == "reorder":  # nothing is computed
        return None
    return globals()["_exact_" + case["op"]](case, seed)


def _turned(x, pos):
    """x [..., heads, 64] in 64 bits at positions pos [...], each pair as a
    complex number times exp(i angle)."""
    a = (pos.to(torch.float32)[..., None] * _inv()).double()[..., None, :]
    z = torch.view_as_complex(x.double().unflatten(-1, (HD // 2, 2)).contiguous())
    return torch.view_as_real(z * torch.polar(torch.ones_like(a), a)).flatten(-2)


def _kept(x, kv):
    """x as a ring of that storage holds it, in 64 bits."""
    return x.float().to(torch.bfloat16).double() if kv == "bf16" else x


def _exact_tree(case, seed):
    B, T, C, kv = case["voices"], case["nodes"], case["capacity"], case["kv"]
    g = _generator(seed)
    n, parent, pos0 = _tree_inputs(case, seed)
    k, v, sp = _rings(g, 1, B, C, kv, pos0)
    x = _randn(g, B, T, QKV, dtype=_dtype(case["q"])).double().unflatten(-1, (3, H, HD))
    out = torch.zeros((B, T, D), dtype=torch.float64, device="cuda")
    for b in range(B):
        chains = []
        for i in range(int(n[b])):
            chains.append((chains[parent[b, i]] if parent[b, i] >= 0 else []) + [i])
        depth = torch.tensor([len(c) - 1 for c in chains], device="cuda")
        mine = torch.zeros((len(chains), len(chains)), dtype=torch.bool, device="cuda")
        for i, c in enumerate(chains):
            mine[i, c] = True
        pos = int(pos0[b]) + depth
        y = x[b, :len(chains)]
        q = _turned(y[:, 0], pos).transpose(0, 1)
        keys = torch.cat((k[0, b].double(), _kept(_turned(y[:, 1], pos), kv).transpose(0, 1)), 1)
        vals = torch.cat((v[0, b].double(), _kept(y[:, 2], kv).transpose(0, 1)), 1)
        p = sp[0, b].long()
        old = (p >= 0) & (p < int(pos0[b])) & (pos[:, None] - p < C)
        w = torch.matmul(q, keys.transpose(1, 2).contiguous()) / 8
        w = w.masked_fill(~torch.cat((old, mine), 1), -torch.inf).softmax(-1)
        out[b, :len(chains)] = torch.matmul(w, vals).transpose(0, 1).flatten(1)
    return out


def _exact_commit(case, seed):
    B, C, kv = case["voices"], case["capacity"], case["kv"]
    g = _generator(seed)
    path, n, pos0 = _commit_inputs(case, seed)
    k, v, _ = _rings(g, LAYERS, B, C, kv, pos0)
    x = _randn(g, LAYERS, B, case["nodes"], QKV, dtype=_dtype(case["q"])).unflatten(-1, (3, H, HD))
    k, v = k.double(), v.double()
    for b in range(B):
        pos = int(pos0[b]) + torch.arange(int(n[b]), device="cuda")
        y = x[:, b, torch.from_numpy(path[b, :n[b]].astype(np.int64)).cuda()]
        k[:, b, :, pos % C] = _kept(_turned(y[:, :, 1], pos), kv).transpose(1, 2)
        v[:, b, :, pos % C] = _kept(y[:, :, 2].double(), kv).transpose(1, 2)
    return [k, v, None]


def _exact_beam(case, seed):
    logits, scores, done, seen = _beam_inputs(case, seed)
    B, W, V, n = case["voices"], case["beams"], case["vocab"], case["choose"]
    out = torch.zeros((B, n), dtype=torch.float64, device="cuda")
    for b in range(B):
        z = logits[b].double()
        if seen is not None:
            bits = np.unpackbits(seen[b].cpu().numpy().view(np.uint8), axis=-1, bitorder="little")
            used = torch.from_numpy(bits[:, :V].astype(bool)).cuda()
            # the penalty is an fp32 number
            by = float(np.float32(PENALTY))
            z = torch.where(used, torch.where(z < 0, z * by, z / by), z)
        c = scores[b].double()[:, None] + z.log_softmax(-1)
        for w in torch.nonzero(done[b]).flatten().tolist():
            c[w] = -torch.inf
            c[w, END] = scores[b, w].double()
        out[b] = c.flatten().topk(n).values
    return {"scores": out, "parent": None, "token": None, "done": None, "seen": None}
