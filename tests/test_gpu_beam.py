"""Beam search: the choice over beams and ids against a full 64-bit sort, and
the move of the rings, through the C ABI."""
import numpy as np
import pytest

import mockbird_amd as mb
from conftest import say
from hypothesis_cases import D, QKV, U, beam_reference
from oracle import oracle

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    with mb.Context(n_layers=1, capacity=4, max_seqs=1, max_rows=4) as c:
        yield c


def _check(got, logits, scores, n, done=None, end_id=-1, seen=None, penalty=1.2):
    """Ids and flags equal.  Scores: the sum of exponentials is off by at most
    2^-21 relative (each term 4 U of the hardware exponential and its argument,
    a sum of 16 four roundings), which is 2^-21 in its logarithm; then one
    rounding to fp32."""
    so, parent, token, dn, seen_out = got
    for b in range(len(logits)):
        c, p, t, d = beam_reference(logits[b], scores[b], n, None if done is None else done[b],
                                    end_id, None if seen is None else seen[b], penalty)
        assert np.array_equal(parent[b], p), (b, parent[b], p)
        assert np.array_equal(token[b], t), (b, token[b], t)
        assert np.array_equal(dn[b], d), b
        fin = np.isfinite(c)
        assert np.array_equal(so[b][~fin], c[~fin].astype(np.float32))
        assert (np.abs(so[b][fin] - c[fin]) <= 2.0 ** -21 + np.abs(c[fin]) * U).all()
        if seen is not None:
            for k in range(n):
                want = np.zeros(seen.shape[-1], np.uint32)
                if p[k] >= 0:
                    want = seen[b, p[k]].copy()
                    want[t[k] // 32] |= np.uint32(1) << np.uint32(t[k] % 32)
                assert np.array_equal(seen_out[b, k], want), (b, k)


def _seen(rng, B, W, V, ids=10):
    s = np.zeros((B, W, (V + 31) // 32), np.uint32)
    at = rng.integers(0, V, (B, W, ids))
    np.bitwise_or.at(s, (np.arange(B)[:, None, None], np.arange(W)[None, :, None], at // 32),
                     np.uint32(1) << (at % 32).astype(np.uint32))
    return s


@pytest.mark.parametrize("V", [1, 2, 31, 33, 64, 1000, 1023, 1024, 1025, 2049, 4096, 4097, 32003,
                               66001])
@pytest.mark.parametrize("W,n", [(1, 1), (3, 5), (8, 8), (17, 32), (32, 9)])
def test_beam_select(ctx, V, W, n):
    """Vocabularies around the scans' edges (one workgroup per voice, and parts
    of a row), more choices than continuations, ended beams, histories."""
    say(f"beam V={V} W={W} n={n}")
    rng = np.random.default_rng([V, W, n])
    B = 3 if V * W < 200_000 else 2
    logits = rng.standard_normal((B, W, V), dtype=np.float32) * 3
    scores = rng.standard_normal((B, W), dtype=np.float32) * 2 - 10
    _check(ctx.beam_select(logits, scores, n), logits, scores, n)
    done = (rng.random((B, W)) < 0.3).astype(np.int32)
    seen = _seen(rng, B, W, V)
    end = V // 2
    for pen in (1.2, 0.75):
        got = ctx.beam_select(logits, scores, n, done, end, seen, pen)
        _check(got, logits, scores, n, done, end, seen, pen)


@pytest.mark.parametrize("V", [100, 2000, 5000])
def test_beam_ties(ctx, V):
    """Equal logits: the lower id; equal beams: the lower beam, whatever the
    place of a row in memory."""
    rng = np.random.default_rng(31)
    logits = np.repeat(rng.integers(-3, 3, (2, 1, V)).astype(np.float32), 5, 1)
    logits[1] = 0.25  # every logit alike
    scores = np.full((2, 5), -1.5, np.float32)
    _check(ctx.beam_select(logits, scores, 12), logits, scores, 12)
    parent, token = ctx.beam_select(logits, scores, 12)[1:3]
    assert (parent[1] == 0).all() and np.array_equal(token[1], np.arange(12))


@pytest.mark.parametrize("V", [70, 1024, 2000, 9000])
def test_beam_first_step_and_not_finite(ctx, V):
    """Beams of score -inf or NaN do not go on; NaN and -inf logits are not
    chosen, a row of nothing else gives nothing; +inf logits share the whole."""
    say(f"beam not finite V={V}")
    rng = np.random.default_rng([32, V])
    W, n = 6, 10
    logits = rng.standard_normal((4, W, V), dtype=np.float32)
    scores = np.zeros((4, W), np.float32)
    scores[0, 1:] = -np.inf                  # a first step
    logits[1, 0] = np.nan
    logits[1, 1] = -np.inf
    logits[1, 2, ::2] = np.nan
    logits[1, 3, 1:] = -np.inf
    logits[1, 4, [3, V - 1]] = np.inf
    scores[1, 5] = np.nan
    logits[2] = -np.inf                      # nothing goes on
    logits[3, :, 5:] = -np.inf               # few continuations, and a beam that ended
    done = np.zeros((4, W), np.int32)
    done[3, 2] = 1
    scores[3] = -np.inf
    scores[3, 2:4] = [-4, -3]
    got = ctx.beam_select(logits, scores, n, done, 2)
    _check(got, logits, scores, n, done, 2)
    assert (got[1][2] == -1).all() and (got[3][2] == 1).all()
    assert list(got[2][1][:2]) == [0, 3] or set(got[2][1][:3]) == {0, 3, V - 1}


@pytest.mark.parametrize("V,W", [(1024, 8), (2001, 8), (7001, 5)])
def test_beam_device_form(ctx, V, W):
    """bf16 logits (many ties) in rows at odd offsets, another stream, a
    workspace of any content, optional outputs left out."""
    import torch
    say(f"beam device form V={V}")
    rng = np.random.default_rng([33, V])
    B, n = 4, 16
    z = oracle.bf16_round(rng.standard_normal((B, W, V + 3), dtype=np.float32) * 3)
    scores = rng.standard_normal((B, W), dtype=np.float32)
    size = ctx.beam_select_work(B, W, V, n)
    assert (size > 0) == (V > 4096)
    st = torch.cuda.Stream()
    try:
        ctx.set_stream(st.cuda_stream)
        with torch.cuda.stream(st):
            t = torch.from_numpy(z).cuda().to(torch.bfloat16)
            s = torch.from_numpy(scores).cuda()
            so = torch.zeros(B, n, device="cuda")
            parent, token = (torch.zeros(B, n, dtype=torch.int32, device="cuda") for _ in range(2))
            work = torch.full((max(size, 16),), 255, dtype=torch.uint8, device="cuda")
            ctx.beam_select_dev(B, W, V, n, t.data_ptr() + 2, s.data_ptr(), so.data_ptr(),
                                parent.data_ptr(), token.data_ptr(), work.data_ptr(), work.numel(),
                                logits_dtype=mb.MB_DT_BF16, logits_stride=V + 3)
            rows = z.reshape(-1)[1:]
            rows = np.stack([rows[r * (V + 3):r * (V + 3) + V] for r in range(B * W)])
            _check((so.cpu().numpy(), parent.cpu().numpy(), token.cpu().numpy(),
                    np.where(parent.cpu().numpy() < 0, 1, 0), None), rows.reshape(B, W, V), scores, n)
    finally:
        ctx.set_stream(None)


@pytest.mark.parametrize("V", [1024, 2001, 9001])
def test_beam_graph_replays(ctx, V):
    """Captured and replayed with eager work between, every replay as the eager call."""
    import torch
    B, W, n = 3, 4, 4
    z, s = torch.randn(B, W, V, device="cuda"), torch.randn(B, W, device="cuda")
    out = [[torch.zeros(B, n, device="cuda")] +
           [torch.zeros(B, n, dtype=torch.int32, device="cuda") for _ in range(2)] for _ in range(2)]
    size = max(16, ctx.beam_select_work(B, W, V, n))
    work = [torch.empty(size, dtype=torch.uint8, device="cuda") for _ in range(2)]

    def call(i):
        ctx.set_stream(torch.cuda.current_stream().cuda_stream)
        ctx.beam_select_dev(B, W, V, n, z.data_ptr(), s.data_ptr(), *(x.data_ptr() for x in out[i]),
                            work[i].data_ptr(), size)

    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call(0)
    for _ in range(4):
        z.normal_()
        s.normal_()
        g.replay()
        call(1)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(*out))


# ---------------------------------------------------------------- reorder

KV = [("f32", mb.MB_KV_F32), ("bf16", mb.MB_KV_BF16)]


def _rings(c):
    return [[c.read_ring(l, b) for b in range(c.cfg.max_seqs)] for l in range(c.cfg.n_layers)]


def _fill(c, rng):
    C = c.capacity
    for l in range(c.cfg.n_layers):
        for b in range(c.cfg.max_seqs):
            last = int(rng.integers(0, 3 * C if c.cfg.wrap else C))
            sp = last - (last - np.arange(C)) % C
            c.write_ring(l, b, 0, rng.standard_normal((C, D), dtype=np.float32),
                         rng.standard_normal((C, D), dtype=np.float32),
                         np.where(sp >= 0, sp, -1).astype(np.int32))


@pytest.mark.parametrize("name,kv", KV)
@pytest.mark.parametrize("W,C", [(1, 5), (2, 1), (3, 7), (4, 33), (5, 64), (8, 20), (16, 9), (32, 6)])
def test_ring_reorder(name, kv, W, C):
    """Permutations, repeats, beams that stay and parents that are none; ranges
    that wrap, are empty, exceed the ring, or are every slot; other layers and
    sequences stay.  Bit for bit."""
    say(f"reorder W={W} C={C} kv={name}")
    rng = np.random.default_rng([W, C])
    G, L = 3, 3
    with mb.Context(n_layers=L, capacity=C, max_seqs=G * W + 1, max_rows=8, kv_dtype=kv) as c:
        _fill(c, rng)
        for mode in range(3):
            before = _rings(c)
            parent = rng.integers(0, W, (G, W)).astype(np.int32)
            parent[0] = rng.permutation(W)
            if W > 2:
                parent[1, 1:3] = [-1, W]
            a = z = None
            if mode < 2:
                a = rng.integers(0, 4 * C, G).astype(np.int32)
                z = (a + [rng.integers(0, C + 1), C + 3, 0 if mode else 1]).astype(np.int32)
            c.ring_reorder(1, 2, parent, a, z)
            after = _rings(c)
            for l in range(L):
                for b in range(G * W + 1):
                    g, w = divmod(b, W)
                    want = [x.copy() for x in before[l][b]]
                    if l >= 1 and g < G and 0 <= parent[g, w] < W:
                        slots = np.arange(C) if a is None else \
                            np.arange(a[g], min(z[g], a[g] + C)) % C
                        src = before[l][g * W + parent[g, w]]
                        for x, y in zip(want, src):
                            x[slots] = y[slots]
                    for x, y in zip(want, after[l][b]):
                        assert np.array_equal(x, y), (mode, l, b)


@pytest.mark.parametrize("name,kv", KV)
def test_ring_reorder_device_form_non_wrapping(name, kv):
    """Ranges beyond a non-wrapping ring are cut at its end; a bound on the rows
    that is too small or large sizes the launch alone."""
    import torch
    rng = np.random.default_rng(41)
    W, C = 2, 30
    with mb.Context(n_layers=1, capacity=C, max_seqs=2 * W, max_rows=8, kv_dtype=kv, wrap=False) as c:
        c.set_stream(torch.cuda.current_stream().cuda_stream)
        for most in (1, 30, 10 ** 6):
            _fill(c, rng)
            before = _rings(c)[0]
            parent = torch.tensor([1, 0, 1, 1], dtype=torch.int32, device="cuda")
            a = torch.tensor([-5, 22], dtype=torch.int32, device="cuda")
            z = torch.tensor([17, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
            c.ring_reorder_dev(0, 1, 2 * W, W, parent.data_ptr(), a.data_ptr(), z.data_ptr(), most)
            after = _rings(c)[0]
            for b, src, s in ((0, 1, slice(0, 17)), (1, 0, slice(0, 17)), (2, 3, slice(22, 30)), (3, 3, slice(0))):
                for x, y, o in zip(before[b], before[src], after[b]):
                    w = x.copy()
                    w[s] = y[s]
                    assert np.array_equal(w, o), (most, b)


@pytest.mark.parametrize("name,kv", KV)
def test_a_beam_search(name, kv):
    """Select, reorder, append and attend for several steps, the choice's arrays
    handed on on the device: rings and outputs are those of beams whose whole
    history a second context appends from the start."""
    import torch
    say(f"beam search kv={name}")
    rng = np.random.default_rng(42)
    B, W, V, C, P, steps = 2, 4, 60, 64, 7, 12
    rows = rng.standard_normal((B * W, V, QKV), dtype=np.float32)  # the row that an id appends
    prompt = rng.standard_normal((B, P, QKV), dtype=np.float32).repeat(W, 0)
    hist = [[] for _ in range(B * W)]
    dev = lambda x: torch.from_numpy(np.ascontiguousarray(x)).cuda()  # noqa: E731
    with mb.Context(n_layers=1, capacity=C, max_seqs=B * W, max_rows=64, kv_dtype=kv) as a, \
            mb.Context(n_layers=1, capacity=C, max_seqs=B * W, max_rows=64, kv_dtype=kv) as s:
        a.set_stream(torch.cuda.current_stream().cuda_stream)
        a.ring_write_rows(0, prompt, np.zeros(B * W), np.full(B * W, P))
        scores = np.full((B, W), -np.inf, np.float32)
        scores[:, 0] = 0
        scores = dev(scores)
        parent, token = (torch.zeros(B, W, dtype=torch.int32, device="cuda") for _ in range(2))
        first = dev(np.full(B, P, np.int32))
        for t in range(steps):
            logits = rng.standard_normal((B, W, V), dtype=np.float32) * 2
            z, new = dev(logits), torch.zeros(B, W, device="cuda")
            a.beam_select_dev(B, W, V, W, z.data_ptr(), scores.data_ptr(), new.data_ptr(),
                              parent.data_ptr(), token.data_ptr())
            c, p, i = beam_reference(logits[0], scores[0].cpu().numpy(), W)[:3]
            assert np.array_equal(parent[0].cpu().numpy(), p) and np.array_equal(token[0].cpu().numpy(), i)
            scores = new
            to = dev(np.full(B, P + t, np.int32))
            a.ring_reorder_dev(0, 1, B * W, W, parent.data_ptr(), first.data_ptr(), to.data_ptr(), t)
            torch.cuda.synchronize()
            p, i = parent.cpu().numpy(), token.cpu().numpy()
            hist = [hist[g * W + p[g, w]] + [i[g, w]] for g in range(B) for w in range(W)]
            new_rows = np.stack([rows[0, h[-1]] for h in hist])
            pos = np.full(B * W, P + t, np.int32)
            _, out = a.append_attend(0, new_rows, pos)
            s.ring_reset()
            s.ring_write_rows(0, prompt, np.zeros(B * W), np.full(B * W, P))
            s.ring_write_rows(0, np.stack([rows[0, h] for h in hist]), np.full(B * W, P),
                              np.full(B * W, t + 1))
            q, want = s.append_attend(0, new_rows, pos)
            assert np.array_equal(out, want), t
            for b in range(B * W):
                for x, y in zip(a.read_ring(0, b), s.read_ring(0, b)):
                    assert np.array_equal(x, y), (t, b)
