"""Drafted trees: their attention over the rings against a 64-bit form, and the
commit of a path against the row writes, through the C ABI."""
import numpy as np
import pytest

import mockbird_amd as mb
from conftest import say
from hypothesis_cases import D, H, HD, QKV, random_parents, rope32, tree_reference
from oracle import oracle

pytestmark = pytest.mark.gpu

KV = [("f32", mb.MB_KV_F32), ("bf16", mb.MB_KV_BF16)]


def _fill(ctx, rng, layer, pos0):
    """Each sequence's ring after pos0[b] appended rows (random K and V)."""
    C = ctx.capacity
    slot = np.arange(C)
    for b, p in enumerate(pos0):
        last = int(p) - 1
        sp = last - (last - slot) % C
        sp = np.where(sp >= 0, sp, -1).astype(np.int32)
        ctx.write_ring(layer, b, 0, rng.standard_normal((C, D), dtype=np.float32),
                       rng.standard_normal((C, D), dtype=np.float32), sp)


def _check(ctx, layer, got, qkv, parent, pos0, n, bf16):
    for b in range(len(pos0)):
        want, bound = tree_reference(ctx.read_ring(layer, b), qkv[b], parent[b], int(pos0[b]),
                                     int(n[b]), bf16)
        err = np.abs(got[b, :n[b]] - want)
        assert (err <= bound).all(), (b, float((err / bound).max()), float(err.max()))


@pytest.mark.parametrize("name,kv", KV)
@pytest.mark.parametrize("T,C", [(1, 1), (2, 3), (7, 16), (15, 31), (16, 32), (17, 33), (31, 100),
                                 (33, 257), (48, 64), (49, 65), (64, 40), (64, 300)])
def test_tree_attention(name, kv, T, C):
    """Empty, partly filled, full and wrapped rings; ragged trees, one of them
    empty; rows past a tree's nodes and the rings stay as they are."""
    say(f"tree T={T} C={C} kv={name}")
    rng = np.random.default_rng([T, C, kv])
    pos0 = np.array([0, 1, max(0, C - 1), C, C + 5, 3 * C + 1], np.int32)
    n = np.array([T, max(1, T - 1), T, 0, max(1, T // 2), T], np.int32)
    B = len(pos0)
    with mb.Context(n_layers=2, capacity=C, max_seqs=B + 1, max_rows=64, kv_dtype=kv) as ctx:
        _fill(ctx, rng, 1, pos0)
        before = [ctx.read_ring(1, b) for b in range(B)]
        qkv = rng.standard_normal((B, T, QKV), dtype=np.float32)
        parent = random_parents(rng, B, T)
        parent[4] = np.arange(-1, T - 1)  # a chain
        parent[5] = -1                    # a star
        out = np.full((B, T, D), 7.0, np.float32)
        got = ctx.tree_attention(1, qkv, parent, pos0, n, out)
        _check(ctx, 1, got, qkv, parent, pos0, n, kv == mb.MB_KV_BF16)
        for b in range(B):
            assert (got[b, n[b]:] == 7.0).all()
            for x, y in zip(before[b], ctx.read_ring(1, b)):
                assert np.array_equal(x, y)


@pytest.mark.parametrize("name,kv", KV)
@pytest.mark.parametrize("B,T,C", [(1, 5, 5000), (2, 64, 3001), (70, 3, 200)])
def test_tree_attention_split_and_many(name, kv, B, T, C):
    """Windows shared by many workgroups, and more sequences than the chip holds at once."""
    say(f"tree B={B} T={T} C={C} kv={name}")
    rng = np.random.default_rng([B, T, C])
    pos0 = rng.integers(C // 2, 3 * C, B).astype(np.int32)
    n = rng.integers(1, T + 1, B).astype(np.int32)
    with mb.Context(n_layers=1, capacity=C, max_seqs=B, max_rows=64, kv_dtype=kv) as ctx:
        _fill(ctx, rng, 0, pos0)
        qkv = rng.standard_normal((B, T, QKV), dtype=np.float32)
        parent = random_parents(rng, B, T)
        got = ctx.tree_attention(0, qkv, parent, pos0, n)
        _check(ctx, 0, got, qkv, parent, pos0, n, kv == mb.MB_KV_BF16)
        # the same call again gives the same bits
        assert np.array_equal(got, ctx.tree_attention(0, qkv, parent, pos0, n))


@pytest.mark.parametrize("name,kv", KV)
@pytest.mark.parametrize("B,T", [(20, 40), (21, 33), (22, 64), (41, 17), (42, 16), (43, 5), (64, 50), (64, 3), (65, 2)])
def test_tree_attention_as_sequences_and_as_a_line(name, kv, B, T):
    """Around the numbers of sequences from which each has workgroups of its own;
    windows of all lengths, several sequences without nodes or rows."""
    say(f"tree B={B} T={T} kv={name}")
    rng = np.random.default_rng([B, T])
    C = 90
    pos0 = rng.integers(0, 3 * C, B).astype(np.int32)
    pos0[rng.integers(0, B, 3)] = 0
    n = rng.integers(0, T + 1, B).astype(np.int32)
    n[rng.integers(0, B, 4)] = 0
    with mb.Context(n_layers=1, capacity=C, max_seqs=B, max_rows=64, kv_dtype=kv) as ctx:
        _fill(ctx, rng, 0, pos0)
        qkv = rng.standard_normal((B, T, QKV), dtype=np.float32)
        parent = random_parents(rng, B, T)
        got = ctx.tree_attention(0, qkv, parent, pos0, n)
        _check(ctx, 0, got, qkv, parent, pos0, n, kv == mb.MB_KV_BF16)
        # the same call again gives the same bits
        assert np.array_equal(got, ctx.tree_attention(0, qkv, parent, pos0, n))
        n[:] = 0  # nothing at all
        out = np.full((B, T, D), 5.0, np.float32)
        assert (ctx.tree_attention(0, qkv, parent, pos0, n, out) == 5.0).all()


@pytest.mark.parametrize("name,kv", KV)
@pytest.mark.parametrize("B,T,C", [(5, 40, 2500), (12, 3, 3000), (1, 64, 1600)])
def test_tree_attention_of_ragged_windows_on_a_line(name, kv, B, T, C):
    """Long windows beside short and empty ones, cut into equal pieces: sequences that
    begin inside a piece, end in it, or have no nodes."""
    say(f"tree line B={B} T={T} C={C} kv={name}")
    rng = np.random.default_rng([B, T, C])
    pos0 = rng.integers(0, 3 * C, B).astype(np.int32)
    pos0[0], pos0[B // 2] = 2 * C + 7, 0 if B > 1 else C
    n = rng.integers(1, T + 1, B).astype(np.int32)
    n[0] = T
    if B > 2:
        n[2] = 0
    with mb.Context(n_layers=1, capacity=C, max_seqs=B, max_rows=64, kv_dtype=kv) as ctx:
        assert ctx.tree_attention_work(B, T, int(pos0.max())) > 0
        _fill(ctx, rng, 0, pos0)
        qkv = rng.standard_normal((B, T, QKV), dtype=np.float32)
        parent = random_parents(rng, B, T)
        out = np.full((B, T, D), 5.0, np.float32)
        got = ctx.tree_attention(0, qkv, parent, pos0, n, out)
        for b in range(B):
            assert (got[b, n[b]:] == 5.0).all()
        _check(ctx, 0, got, qkv, parent, pos0, n, kv == mb.MB_KV_BF16)
        assert np.array_equal(got, ctx.tree_attention(0, qkv, parent, pos0, n, out.copy()))


@pytest.mark.parametrize("B,T,C", [(3, 6, 40), (70, 6, 40), (6, 6, 1500), (6, 40, 1500), (30, 40, 40)])
def test_tree_device_positions_that_do_not_fit(B, T, C):
    """Sequences at positions below 0 or above 2^31 - 65, and negative and too large
    counts, on the device: left out, or taken to rows_max."""
    import torch
    rng = np.random.default_rng(14)
    say(f"tree positions B={B} T={T} C={C}")
    pos0 = rng.integers(0, 2 * C, B).astype(np.int32)
    n = np.full(B, T, np.int32)
    n[1] = 2 ** 31 - 1
    good = np.ones(B, bool)
    for b, (p, m) in ((0, (-1, T)), (2, (2 ** 31 - 64, T)), (B - 2, (7, -2 ** 31 if T > 32 else -5)),
                      (B - 1, (-2 ** 31, T))):
        pos0[b], n[b], good[b] = p, m, False
    with mb.Context(n_layers=1, capacity=C, max_seqs=B, max_rows=64) as ctx:
        _fill(ctx, rng, 0, np.where(good, pos0, 0))
        ctx.set_stream(torch.cuda.current_stream().cuda_stream)
        rows = rng.standard_normal((B, T, QKV), dtype=np.float32)
        parent = random_parents(rng, B, T)
        q, w, p, c = (torch.from_numpy(x).cuda() for x in (rows, parent, pos0, n))
        out = torch.full((B, T, D), 3.0, device="cuda")
        _dev(ctx, 0, q, w, p, c, 2 ** 31 - 1, out)
        got = out.cpu().numpy()
        at = np.flatnonzero(good)
        assert (got[~good] == 3.0).all()
        for b in at:
            want, bound = tree_reference(ctx.read_ring(0, b), rows[b], parent[b], int(pos0[b]), T, False)
            assert (np.abs(got[b] - want) <= bound).all(), b


@pytest.mark.parametrize("name,kv", KV)
def test_tree_equals_appending_its_paths(name, kv):
    """Every node's output is what mb_append_attend ends with when its path is
    appended row by row: the window evicts alike.  Both are within their bounds
    of the 64-bit form, so they are within the sum of both of each other."""
    say(f"tree against appends kv={name}")
    rng = np.random.default_rng(5)
    C, T, p0 = 24, 12, 50
    qkv = rng.standard_normal((1, T, QKV), dtype=np.float32)
    parent = random_parents(rng, 1, T, 3)
    with mb.Context(n_layers=1, capacity=C, max_seqs=1, max_rows=64, kv_dtype=kv) as ctx:
        _fill(ctx, rng, 0, [p0])
        ring = ctx.read_ring(0, 0)
        got = ctx.tree_attention(0, qkv, parent, [p0], [T])
        _, bound = tree_reference(ring, qkv[0], parent[0], p0, T, kv == mb.MB_KV_BF16)
        for i in range(T):
            path, j = [], i
            while j >= 0:
                path.insert(0, j)
                j = parent[0, j]
            ctx.write_ring(0, 0, 0, *ring)
            for d, j in enumerate(path):
                _, o = ctx.append_attend(0, qkv[:, j], [p0 + d])
            assert (np.abs(o[0] - got[0, i]) <= 2 * bound[i]).all(), i


@pytest.mark.parametrize("name,kv", KV)
@pytest.mark.parametrize("bad", [False, True])
@pytest.mark.parametrize("T,C,pos0", [(2, 1, 0), (2, 1, 7), (20, 3, 0), (40, 33, 50), (64, 7, 2), (64, 63, 200)])
def test_tree_of_chains_longer_than_the_ring(name, kv, bad, T, C, pos0):
    """A node does not see ancestors that its own appends would have evicted: the
    result is that of appending the chain row by row."""
    say(f"long chains T={T} C={C} pos0={pos0} kv={name} bad={bad}")
    rng = np.random.default_rng([T, C, pos0, bad])
    parent = np.stack((np.arange(-1, T - 1), np.maximum(np.arange(T) - 2, -1))).astype(np.int32)
    at, n = np.full(2, pos0, np.int32), np.full(2, T, np.int32)
    qkv = rng.standard_normal((2, T, QKV), dtype=np.float32)
    if bad:  # evicted by the last row of the first chain, and seen by earlier ones
        qkv[0, 0, 2 * D] = np.inf
    with mb.Context(n_layers=1, capacity=C, max_seqs=2, max_rows=64, kv_dtype=kv) as ctx:
        _fill(ctx, rng, 0, at)
        got = ctx.tree_attention(0, qkv, parent, at, n)
        for b in range(2):
            want, bound = tree_reference(ctx.read_ring(0, b), qkv[b], parent[b], pos0, T, kv == mb.MB_KV_BF16)
            fine = np.isfinite(want)
            assert np.array_equal(got[b][~fine], want[~fine].astype(np.float32), equal_nan=True)
            assert (np.abs(got[b][fine] - want[fine]) <= bound[fine]).all()
            assert fine.all() == (b == 1 or not bad)
            assert fine[-1].all()


@pytest.mark.parametrize("name,kv", KV)
def test_tree_does_not_see_a_dropped_draft(name, kv):
    """Slots at pos0 and later (an earlier draft, rolled back) are not seen, in
    whatever state."""
    rng = np.random.default_rng(6)
    C, p0 = 64, 30
    with mb.Context(n_layers=1, capacity=C, max_seqs=1, max_rows=64, kv_dtype=kv) as ctx:
        _fill(ctx, rng, 0, [p0])
        qkv = rng.standard_normal((1, 9, QKV), dtype=np.float32)
        parent = random_parents(rng, 1, 9)
        want = ctx.tree_attention(0, qkv, parent, [p0], [9])
        ctx.ring_write_rows(0, rng.standard_normal((1, 20, QKV), dtype=np.float32), [p0], [20])
        assert np.array_equal(want, ctx.tree_attention(0, qkv, parent, [p0], [9]))
        k = np.full((20, D), np.nan, np.float32)
        ctx.write_ring(0, 0, p0, k, k)
        got = ctx.tree_attention(0, qkv, parent, [p0], [9])
        _check(ctx, 0, got, qkv, parent, [p0], [9], kv == mb.MB_KV_BF16)


@pytest.mark.parametrize("name,kv", KV)
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("B,C", [(1, 150), (24, 150), (70, 150), (1, 1500), (3, 1500)])
def test_tree_not_finite(name, kv, bad, B, C):
    """Values that are not finite reach exactly the nodes that see them: in empty
    slots and rows behind the nodes none, in a slot that only the shallow nodes
    still hold and in a drafted row its descendants.  (1500 slots: windows
    shared by workgroups.)"""
    say(f"tree {bad} kv={name} B={B} C={C}")
    rng = np.random.default_rng(8)
    T = 20
    pos0 = np.full(B, C + 250, np.int32)
    pos0[0] = C + 110
    n = np.full(B, T - 2, np.int32)
    qkv = rng.standard_normal((B, T, QKV), dtype=np.float32)
    parent = np.repeat(random_parents(rng, 1, T, 4), B, 0)
    bf16 = kv == mb.MB_KV_BF16
    with mb.Context(n_layers=1, capacity=C, max_seqs=B, max_rows=64, kv_dtype=kv) as ctx:
        _fill(ctx, rng, 0, pos0)
        clean = ctx.tree_attention(0, qkv, parent, pos0, n)
        k, v, sp = ctx.read_ring(0, 0)
        # an emptied slot, and rows behind the nodes
        k2, v2, sp2 = k.copy(), v.copy(), sp.copy()
        k2[17], v2[17], sp2[17] = bad, bad, -1
        ctx.write_ring(0, 0, 0, k2, v2, sp2)
        qkv[:, T - 2:] = bad
        got = ctx.tree_attention(0, qkv, parent, pos0, n)
        assert np.isfinite(got).all()
        _check(ctx, 0, got[:1], qkv, parent, pos0[:1], n[:1], bf16)
        assert np.array_equal(got[1:], clean[1:])
        # V of the oldest position that a node at pos0 holds and deeper ones do not: head 3
        ctx.write_ring(0, 0, 0, k, v, sp)
        s = int(np.argmax(sp == pos0[0] - C + 1))
        v2 = v.copy()
        v2[s, 3 * HD:4 * HD] = bad
        ctx.write_ring(0, 0, 0, k, v2, sp)
        got = ctx.tree_attention(0, qkv, parent, pos0, n)
        for i in range(T - 2):
            at = got[0, i].reshape(H, HD)
            want = clean[0, i].reshape(H, HD)
            if parent[0, i] < 0:
                assert (np.isnan(at[3]) if np.isnan(bad) else at[3] == bad).all(), i
            else:
                assert np.isfinite(at[3]).all(), i
            assert np.array_equal(np.delete(at, 3, 0), np.delete(want, 3, 0))
        # a drafted V row: its descendants and itself
        ctx.write_ring(0, 0, 0, k, v, sp)
        q2 = qkv.copy()
        q2[0, 4, 2 * D:] = bad
        got = ctx.tree_attention(0, q2, parent, pos0, n)
        for i in range(T - 2):
            j, sees = i, False
            while j >= 0:
                sees, j = sees or j == 4, parent[0, j]
            ok = np.isnan(got[0, i]) if np.isnan(bad) else got[0, i] == bad
            assert ok.all() if sees else np.isfinite(got[0, i]).all(), i
        assert np.array_equal(got[1:], clean[1:])
        # a drafted K row of NaN or an infinity that takes the whole weight or none
        q2 = qkv.copy()
        q2[0, 4, D:2 * D] = 0
        q2[0, 4, D] = bad
        got = ctx.tree_attention(0, q2, parent, pos0, n)
        for i in range(T - 2):
            j, sees = i, False
            while j >= 0:
                sees, j = sees or j == 4, parent[0, j]
            if not sees:
                assert np.isfinite(got[0, i]).all(), i
            elif np.isnan(bad):
                assert np.isnan(got[0, i, :HD]).all()


@pytest.mark.parametrize("name,kv", KV)
def test_tree_large_values(name, kv):
    """q near the largest float over K of its reciprocal's size."""
    rng = np.random.default_rng(9)
    C, T, p0 = 40, 5, 33
    qkv = rng.standard_normal((1, T, QKV), dtype=np.float32)
    qkv[0, 2, :D] = 0
    qkv[0, 2, 0:D:HD] = 3.4e38
    parent = np.full((1, T), -1, np.int32)
    with mb.Context(n_layers=1, capacity=C, max_seqs=1, max_rows=64, kv_dtype=kv) as ctx:
        _fill(ctx, rng, 0, [p0])
        k, v, sp = ctx.read_ring(0, 0)
        k *= 1e-37
        ctx.write_ring(0, 0, 0, k, v, sp)
        qkv[:, :, D:2 * D] *= 1e-37
        got = ctx.tree_attention(0, qkv, parent, [p0], [T])
        _check(ctx, 0, got, qkv, parent, [p0], [T], kv == mb.MB_KV_BF16)


@pytest.mark.parametrize("name,kv", KV)
def test_tree_far_positions(name, kv):
    """Beyond the table of angles and up to the last position that fits."""
    rng = np.random.default_rng(10)
    C, T = 37, 6
    pos0 = np.array([65_533, 1_000_003, 2 ** 31 - 65], np.int32)
    qkv = rng.standard_normal((3, T, QKV), dtype=np.float32)
    parent = random_parents(rng, 3, T, 2)
    n = np.full(3, T, np.int32)
    with mb.Context(n_layers=1, capacity=C, max_seqs=3, max_rows=64, kv_dtype=kv) as ctx:
        _fill(ctx, rng, 0, pos0)
        got = ctx.tree_attention(0, qkv, parent, pos0, n)
        _check(ctx, 0, got, qkv, parent, pos0, n, kv == mb.MB_KV_BF16)


def _dev(ctx, layer, qkv, parent, pos0, n, max_pos, out, work=None, **kw):
    B, T = parent.shape
    size = ctx.tree_attention_work(B, T, max_pos)
    if work is None:
        import torch
        work = torch.full((max(size, 16),), 255, dtype=torch.uint8, device="cuda")  # NaN everywhere
    ctx.tree_attention_dev(layer, B, T, qkv.data_ptr(), parent.data_ptr(), pos0.data_ptr(),
                           None if n is None else n.data_ptr(), max_pos, out.data_ptr(),
                           work.data_ptr(), work.numel(), **kw)
    return work


@pytest.mark.parametrize("name,kv", KV)
@pytest.mark.parametrize("half", [False, True])
def test_tree_device_form(name, kv, half):
    """Strided rows of both types, a workspace of any content, a bound on the
    positions that is larger than needed, no counts, another stream, parents
    that are no earlier node, a sequence left out."""
    import torch
    say(f"tree device form kv={name} bf16 rows={half}")
    rng = np.random.default_rng(12)
    B, T, C = 3, 18, 700
    pos0 = np.array([650, 2000, -4], np.int32)
    rows = rng.standard_normal((B, T, QKV + 16), dtype=np.float32)
    if half:
        rows = oracle.bf16_round(rows)
    parent = random_parents(rng, B, T)
    wild = parent.copy()
    wild[parent < 0] = rng.choice([-2 ** 31, -7, 2 ** 31 - 1, 64, 999], (parent < 0).sum())
    wild[0, 3], parent[0, 3] = 3, -1  # its own parent
    with mb.Context(n_layers=1, capacity=C, max_seqs=B, max_rows=64, kv_dtype=kv) as ctx:
        _fill(ctx, rng, 0, np.maximum(pos0, 0))
        st = torch.cuda.Stream()
        ctx.set_stream(st.cuda_stream)
        with torch.cuda.stream(st):
            q = torch.from_numpy(rows).cuda()
            q = q.to(torch.bfloat16) if half else q
            p, w = torch.from_numpy(pos0).cuda(), torch.from_numpy(wild).cuda()
            out = torch.full((B, T, D + 4), 3.0, device="cuda")
            for bound in (2100, 2 ** 31 - 1):
                _dev(ctx, 0, q, w, p, None, bound, out, qkv_dtype=int(half), qkv_stride=QKV + 16,
                     out_stride=D + 4)
                got = out.cpu().numpy()
                n = np.full(B, T, np.int32)
                _check(ctx, 0, got[:2, :, :D], rows[:, :, :QKV], parent, pos0[:2], n,
                       kv == mb.MB_KV_BF16)
                assert (got[2] == 3.0).all() and (got[..., D:] == 3.0).all()


def test_tree_graph_replays():
    """Two captured graphs with a workspace each, replayed several times with
    eager work between, on inputs that change: every replay as the eager call."""
    import torch
    rng = np.random.default_rng(13)
    B, T, C = 1, 24, 1500
    with mb.Context(n_layers=2, capacity=C, max_seqs=B, max_rows=64, kv_dtype=mb.MB_KV_BF16) as ctx:
        _fill(ctx, rng, 0, [1400])
        _fill(ctx, rng, 1, [1400])
        qkv = torch.randn(2, B, T, QKV, device="cuda")
        parent = torch.from_numpy(random_parents(rng, B, T)).cuda()
        pos0 = torch.tensor([1400], dtype=torch.int32, device="cuda")
        outs = [torch.zeros(B, T, D, device="cuda") for _ in range(2)]
        want = torch.zeros(B, T, D, device="cuda")
        size = ctx.tree_attention_work(B, T, 2000)
        works = [torch.empty(size, dtype=torch.uint8, device="cuda") for _ in range(3)]
        graphs = []
        for i in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                ctx.set_stream(torch.cuda.current_stream().cuda_stream)
                _dev(ctx, i, qkv[i], parent, pos0, None, 2000, outs[i], works[i])
            graphs.append(g)
        ctx.set_stream(torch.cuda.current_stream().cuda_stream)
        for r in range(4):
            qkv.normal_()
            pos0.fill_(1400 - 300 * r)
            for i in (0, 1):
                graphs[i].replay()
            for i in (0, 1):
                _dev(ctx, i, qkv[i], parent, pos0, None, 2000, want, works[2])
                torch.cuda.synchronize()
                assert torch.equal(want, outs[i]), (r, i)


# ----------------------------------------------------------------- commit

@pytest.mark.parametrize("name,kv", KV)
@pytest.mark.parametrize("wrap", [True, False])
def test_commit_is_the_row_write_of_the_path(name, kv, wrap):
    """All layers in one call, ragged paths (one empty, repeated and falling
    nodes, in a wrapping ring one longer than the ring): every ring bit for bit
    what mb_ring_write_rows leaves of the gathered rows."""
    say(f"commit kv={name} wrap={wrap}")
    rng = np.random.default_rng(20)
    L, B, T, P, C = 3, 5, 20, 12, 10 if wrap else 200
    pos0 = np.array([0, 7, 95, 3, 64], np.int32)
    n = np.array([P, 1, 5, 0, 9], np.int32)
    path = rng.integers(0, T, (B, P)).astype(np.int32)
    qkv = rng.standard_normal((L, B, T, QKV), dtype=np.float32)
    with mb.Context(n_layers=L + 1, capacity=C, max_seqs=B, max_rows=64, kv_dtype=kv, wrap=wrap) as a, \
            mb.Context(n_layers=L + 1, capacity=C, max_seqs=B, max_rows=64, kv_dtype=kv, wrap=wrap) as b:
        a.tree_commit(1, qkv, pos0, path, n)
        for l in range(L):
            rows = qkv[l][np.arange(B)[:, None], path]
            # (a host write takes at most `capacity` rows: the last ones of a longer path)
            cut = np.maximum(0, n - C)
            shifted = np.stack([np.roll(rows[i], -cut[i], 0) for i in range(B)])
            b.ring_write_rows(l + 1, shifted, pos0 + cut, n - cut)
        for l in range(L + 1):
            for s in range(B):
                for x, y in zip(a.read_ring(l, s), b.read_ring(l, s)):
                    assert np.array_equal(x, y), (l, s)


@pytest.mark.parametrize("name,kv", KV)
def test_commit_device_form(name, kv):
    """bf16 rows with strides, path entries that are no rows, no counts."""
    import torch
    rng = np.random.default_rng(21)
    L, B, T, P, C = 2, 3, 9, 4, 16
    rows = oracle.bf16_round(rng.standard_normal((L, B, T, QKV + 8), dtype=np.float32))
    path = rng.integers(0, T, (B, P)).astype(np.int32)
    path[1] = [2, -1, T, 5]
    pos0 = np.array([14, 40, -3], np.int32)
    with mb.Context(n_layers=L, capacity=C, max_seqs=B, max_rows=64, kv_dtype=kv) as ctx:
        ctx.set_stream(torch.cuda.current_stream().cuda_stream)
        pad = torch.zeros(L, B * T * (QKV + 8) + 64, dtype=torch.bfloat16, device="cuda")
        pad[:, :-64] = torch.from_numpy(rows).cuda().reshape(L, -1).to(torch.bfloat16)
        p, q = torch.from_numpy(pos0).cuda(), torch.from_numpy(path).cuda()
        ctx.tree_commit_dev(0, L, B, T, pad.data_ptr(), p.data_ptr(), P, q.data_ptr(), None,
                            qkv_dtype=mb.MB_DT_BF16, qkv_stride=QKV + 8, layer_stride=pad.shape[1])
        for l in range(L):
            for b in range(B):
                k, v, sp = ctx.read_ring(l, b)
                want = np.full(C, -1)
                for i in range(P):
                    if pos0[b] >= 0 and 0 <= path[b, i] < T:
                        pos = int(pos0[b]) + i
                        want[pos % C] = pos
                        x = rows[l, b, path[b, i]]
                        kk = rope32(x[D:2 * D], pos)
                        kk = oracle.bf16_round(kk) if kv == mb.MB_KV_BF16 else kk
                        assert np.array_equal(k[pos % C], kk) and np.array_equal(v[pos % C], x[2 * D:QKV])
                assert np.array_equal(sp, want), (l, b)


@pytest.mark.parametrize("name,kv", KV)
def test_draft_verify_commit_go_on(name, kv):
    """The operators as a program runs them: attend a tree in every layer, commit
    the chosen path, draft again from its end.  The rings and outputs are those of
    a second context that appends the path row by row."""
    say(f"draft, commit, draft kv={name}")
    rng = np.random.default_rng(22)
    L, B, T, C = 2, 2, 14, 48
    pos0 = np.array([5, 40], np.int32)
    bf16 = kv == mb.MB_KV_BF16
    with mb.Context(n_layers=L, capacity=C, max_seqs=B, max_rows=64, kv_dtype=kv) as a, \
            mb.Context(n_layers=L, capacity=C, max_seqs=B, max_rows=64, kv_dtype=kv) as s:
        for l in range(L):
            seed = rng.integers(1 << 30)
            _fill(a, np.random.default_rng(seed), l, pos0)
            _fill(s, np.random.default_rng(seed), l, pos0)
        for _ in range(6):
            qkv = rng.standard_normal((L, B, T, QKV), dtype=np.float32)
            parent = random_parents(rng, B, T, 2)
            leaf = rng.integers(0, T, B)
            path, n = np.zeros((B, T), np.int32), np.zeros(B, np.int32)
            for b in range(B):
                c, j = [], int(leaf[b])
                while j >= 0:
                    c.insert(0, j)
                    j = int(parent[b, j])
                path[b, :len(c)], n[b] = c, len(c)
            outs = [a.tree_attention(l, qkv[l], parent, pos0, np.full(B, T)) for l in range(L)]
            for l in range(L):
                _check(a, l, outs[l], qkv[l], parent, pos0, np.full(B, T), bf16)
            a.tree_commit(0, qkv, pos0, path, n)
            for l in range(L):
                rows = qkv[l][np.arange(B)[:, None], path]
                s.ring_write_rows(l, rows, pos0, n)
                for b in range(B):
                    for x, y in zip(a.read_ring(l, b), s.read_ring(l, b)):
                        assert np.array_equal(x, y)
            pos0 = (pos0 + n).astype(np.int32)


def test_ring_view_is_the_rings():
    import torch
    for _, kv in KV:
        with mb.Context(n_layers=2, capacity=6, max_seqs=3, max_rows=8, kv_dtype=kv) as ctx:
            ctx.ring_write_rows(1, np.random.default_rng(3).standard_normal((3, 4, QKV), dtype=np.float32),
                                [0, 1, 4], [4, 3, 4])
            k, v, sp = (torch.as_tensor(x, device="cuda") for x in ctx.ring_view())
            k, v = (x.view(torch.bfloat16) if kv == mb.MB_KV_BF16 else x for x in (k, v))
            for b in range(3):
                kk, vv, pp = ctx.read_ring(1, b)
                assert np.array_equal(kk, k[1, b].float().transpose(0, 1).reshape(6, D).cpu().numpy())
                assert np.array_equal(vv, v[1, b].float().transpose(0, 1).reshape(6, D).cpu().numpy())
                assert np.array_equal(pp, sp[1, b].cpu().numpy())
            v[0, 2] = 2.5
            torch.cuda.synchronize()
            assert (ctx.read_ring(0, 2)[1] == 2.5).all() and (ctx.read_ring(0, 1)[1] == 0).all()
