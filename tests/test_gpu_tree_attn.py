"""Tree attention over the paged cache against the oracle's softmax in 64 bits.

Bounds, fixed before the first run. With u = eps(type) / 2, the relative error of a weight p_j is
at most u (its rounding to the type for the product with V; absent in float32 runs) plus
e = 2 ds + (n + D + 16) 2^-23: ds = (D + 4) 2^-23 max_j scale sum_d |q_d k_jd| is the error of a score
(D products summed in float32, truncated or rounded), n 2^-23 that of sums over n keys in float32, and
16 * 2^-23 covers the exponential and its argument (|x| below 64, 2 ulp). The output, a weighted
mean, is off by at most (u + e) sum_j p_j |v_j| / sum p, and its own rounding by u |out|; the
log-sum-exp by ds + (n + 16) 2^-23 + |lse| 2^-23."""

import math

import numpy as np
import pytest
import torch

from oracle.paged_oracle import tree_attention as oracle_attention

pytestmark = pytest.mark.gpu

cab = pytest.importorskip("cab_attention")
from cab_attention import PagedKVCache, _lib  # noqa: E402
from cab_attention.eviction import select_indices_batched  # noqa: E402
from cab_attention.kernels import flash_attention_forward, tree_attention  # noqa: E402

BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def _device_status_clean():
    yield
    assert _lib.device_status() == 0


def random_parents(n, T, g, branch=0.7):
    """Parents before children; several roots now and then."""
    p = torch.zeros(n, T, dtype=torch.int64)
    for b in range(n):
        for t in range(T):
            back = int(torch.randint(1, 4, (1,), generator=g))
            p[b, t] = max(-1, t - back) if torch.rand(1, generator=g) < branch else int(torch.randint(-1, max(t, 1), (1,), generator=g))
        p[b, 0] = -1
    return p


def build(lens, H, S, D, dtype, seed=0, fill=math.nan, slots_first=False, extra=2):
    """A pool in which everything but the sequences' tokens is `fill`."""
    g = torch.Generator().manual_seed(seed)
    counts = [-(-n // S) for n in lens]
    W, P = max(counts + [1]) + 1, sum(counts) + extra
    order = torch.randperm(P, generator=g)
    table = torch.full((len(lens), W), -1, dtype=torch.int32)
    shape = (P, S, H, D) if slots_first else (P, H, S, D)
    kp, vp = (torch.full(shape, fill, dtype=dtype) for _ in range(2))
    if slots_first:
        kp, vp = kp.transpose(1, 2), vp.transpose(1, 2)
    ks, vs, at = [], [], 0
    for b, n in enumerate(lens):
        pages = order[at:at + counts[b]]
        at += counts[b]
        table[b, :counts[b]] = pages.int()
        k, v = ((torch.randn(H, n, D, generator=g) + 0.5 * torch.randn(H, 1, D, generator=g)).to(dtype) for _ in range(2))
        for x in range(n):
            kp[pages[x // S], :, x % S] = k[:, x]
            vp[pages[x // S], :, x % S] = v[:, x]
        ks.append(k.float().numpy())
        vs.append(v.float().numpy())

    def put(t):
        return t.transpose(1, 2).contiguous().cuda().transpose(1, 2) if slots_first else t.cuda()

    return put(kp), put(vp), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), ks, vs


def bounds(n, D, dtype, scale_abs, absv, out, lse):
    u = 0.0 if dtype == FP else torch.finfo(dtype).eps / 2
    ds = (D + 4) * 2.0 ** -23 * scale_abs
    e = 2 * ds + (n + D + 16) * 2.0 ** -23
    round_out = torch.finfo(dtype).eps / 2
    lim_out = (u + e)[..., None] * absv + round_out * np.abs(out) + 1e-30
    lim_lse = ds + (n + 16) * 2.0 ** -23 + np.where(np.isfinite(lse), np.abs(lse), 0) * 2.0 ** -23
    return lim_out, lim_lse


def check(got, lse, q, ks, vs, nodes, scale, dtype, parents=None, mask=None, rows=None, there=None):
    got, lse, q = got.float().cpu().numpy().astype(np.float64), lse.cpu().numpy(), q.float().cpu().numpy()
    for i in range(q.shape[0]):
        r = i if rows is None else rows[i]
        m = nodes[i]
        par = None if parents is None else parents if parents.dim() == 1 else parents[i]
        msk = None if mask is None else mask if mask.dim() == 2 else mask[i]
        w, wl, absv, absqk = oracle_attention(q[i], ks[r], vs[r], m, scale, None if par is None else par.tolist(),
                                              None if msk is None else msk.numpy(), None if there is None else there[r])
        lo, ll = bounds(ks[r].shape[1], q.shape[3], dtype, absqk, absv, w, wl)
        assert np.isfinite(got[i]).all()
        assert (np.abs(got[i] - w) <= lo).all(), (i, np.max(np.abs(got[i] - w) / lo))
        dead = np.isneginf(wl)
        assert np.array_equal(dead, np.isneginf(lse[i]))
        with np.errstate(invalid="ignore"):
            assert (np.where(dead, 0, np.abs(lse[i] - wl)) <= ll).all(), i
        assert (got[i][dead] == 0).all()


# n is len(ctx): context lengths, with T nodes on top
CASES = [
    # Hq, Hkv, D, S, T, ctx, tree, dtype
    (8, 8, 64, 16, 1, [0, 1, 15, 127], "chain", BF),
    (8, 2, 128, 16, 1, [128, 300, 1025], "chain", BF),
    (4, 1, 128, 64, 1, [5000], "chain", HF),
    (8, 2, 128, 8, 3, [7, 250], "parents", BF),
    (6, 2, 128, 32, 17, [0, 100, 513], "parents", BF),
    (4, 4, 64, 128, 64, [64, 1000], "parents", HF),
    (4, 1, 128, 64, 64, [63, 700], "parents", BF),       # 256 rows a KV head
    (2, 2, 128, 16, 129, [1, 400], "mask", BF),
    (8, 1, 64, 256, 40, [300, 17], "mask", HF),          # 320 rows a KV head
    (5, 1, 128, 16, 7, [333, 0, 90], "mask", BF),        # a group that does not divide the tile
    (2, 1, 128, 64, 300, [0, 77, 1100], "chain", BF),
    (1, 1, 64, 16, 513, [40], "chain", BF),
    (4, 2, 64, 16, 5, [0, 30, 200], "parents", FP),
    (4, 2, 128, 64, 33, [90, 1], "mask", FP),
    (8, 8, 256, 16, 2, [100], "chain", FP),
    (3, 1, 80, 24, 6, [100, 31], "parents", HF),         # head_dim and page size off the tensor-core path
    (4, 4, 64, 20, 3, [100, 31], "chain", BF),
    (2, 1, 7, 1, 4, [33], "mask", FP),
    (2, 2, 128, 48, 2, [500, 3], "chain", BF),
    # up to 8 rows on CUDA cores
    (3, 1, 80, 24, 2, [100, 31, 0], "parents", HF),
    (8, 1, 256, 16, 1, [700, 1], "chain", FP),
    (4, 4, 8, 3, 7, [33, 400], "mask", FP),
    (8, 8, 128, 48, 3, [500, 3], "parents", BF),
    (1, 1, 64, 16, 1, [0, 31, 32, 3000], "chain", FP),
    (2, 1, 128, 64, 1, [2000], "chain", FP),
]


@pytest.mark.parametrize("Hq,H,D,S,T,ctx,tree,dtype", CASES)
def test_matches_oracle(Hq, H, D, S, T, ctx, tree, dtype):
    g = torch.Generator().manual_seed(T * 31 + D)
    n = len(ctx)
    nodes = [max(T - 3 * i, 0 if i else T) for i in range(n)]
    lens = [c + m for c, m in zip(ctx, nodes)]
    kp, vp, table, seq, ks, vs = build(lens, H, S, D, dtype, seed=D + T)
    q = torch.randn(n, Hq, T, D, generator=g).to(dtype)
    parents = random_parents(n, T, g) if tree == "parents" else None
    mask = torch.rand(n, T, T, generator=g) < 0.3 if tree == "mask" else None  # some rows see no node
    out, lse = tree_attention(q.cuda(), kp, vp, table, seq, parents=None if parents is None else parents.cuda(),
                              tree_mask=None if mask is None else mask.cuda(),
                              num_nodes=torch.tensor(nodes).cuda(), return_lse=True)
    check(out, lse, q, ks, vs, nodes, 1 / math.sqrt(D), dtype, parents, mask)


# shapes of the scheduling: many sequences, heads that fill a tile or exceed it, long rows cut between
# CTAs, short rows in wide tables, large pages
SHAPES = [
    # Hq, Hkv, D, S, T, ctx, width (pages of a table row, 0: as needed), dtype
    (4, 2, 64, 16, 2, [37 * i % 400 for i in range(40)], 0, BF),
    (2, 2, 128, 16, 1, [11 * i % 90 for i in range(150)], 0, HF),
    (2, 1, 64, 64, 3, [5 + 7 * i for i in range(33)], 2048, BF),
    (128, 1, 128, 32, 3, [700, 20], 0, BF),     # a node fills a tile
    (130, 1, 64, 16, 2, [50], 0, BF),           # more heads than a tile has rows: CUDA cores
    (96, 1, 64, 16, 9, [300, 1000], 0, HF),     # one node a group, groups side by side
    (8, 8, 128, 512, 4, [1500, 511, 512], 0, BF),
    (1, 1, 128, 128, 2, [70001], 0, BF),
    (2, 1, 64, 16, 6, [40003, 3], 4096, HF),
    (4, 1, 64, 16, 700, [10], 0, BF),           # 2800 rows of a KV head: several sets of groups
    # more than 128 sequences whose rows are cut between CTAs
    (4, 2, 64, 16, 2, [53 * i % 120 + 2500 * (i % 50 == 7) for i in range(150)], 0, BF),
    (2, 1, 128, 32, 70, [3100] + [i % 3 for i in range(128)], 0, HF),
    (1, 1, 64, 64, 1, [0] * 299 + [6000], 0, BF),
    (8, 2, 64, 16, 40, [31 * i % 200 for i in range(257)], 64, BF),   # 160 rows a KV head, a pair of groups
]


@pytest.mark.parametrize("Hq,H,D,S,T,ctx,width,dtype", SHAPES)
def test_schedule_shapes(Hq, H, D, S, T, ctx, width, dtype):
    g = torch.Generator().manual_seed(T + Hq)
    n = len(ctx)
    nodes = [max(1, T - i % 2) for i in range(n)]
    kp, vp, table, seq, ks, vs = build([c + m for c, m in zip(ctx, nodes)], H, S, D, dtype, seed=Hq + S)
    if width:
        table = torch.nn.functional.pad(table, (0, width - table.shape[1]), value=-1)
    q = torch.randn(n, Hq, T, D, generator=g).to(dtype)
    out, lse = tree_attention(q.cuda(), kp, vp, table, seq, num_nodes=torch.tensor(nodes).cuda(), return_lse=True)
    if T * Hq * sum(ctx) < 3e6:
        check(out, lse, q, ks, vs, nodes, 1 / math.sqrt(D), dtype)
        return
    pick = sorted({0, 1, T // 2, T - 1} & set(range(min(nodes))))  # some rows of large cases
    for t in pick:
        for i in range(n):
            m = nodes[i]
            kk, vv = ks[i][:, :len(ks[i][0]) - m + t + 1], vs[i][:, :len(vs[i][0]) - m + t + 1]
            check(out[i:i + 1, :, t:t + 1], lse[i:i + 1, :, t:t + 1], q[i:i + 1, :, t:t + 1], [kk], [vv], [1],
                  1 / math.sqrt(D), dtype)


@pytest.mark.parametrize("dtype,D,S", [(BF, 128, 64), (HF, 64, 16), (FP, 64, 16)])
@pytest.mark.parametrize("up", [True, False])
def test_scores_that_grow_or_fall_along_the_cache(dtype, D, S, up):
    """The reference of the weights changes again and again, or never after the first tile."""
    T, n = 5, 1700
    kp, vp, table, seq, ks, vs = build([n], 1, S, D, dtype, fill=0.0)
    ramp = torch.linspace(-1, 1, n) if up else torch.linspace(1, -1, n)
    k = (0.1 * torch.from_numpy(ks[0][0]) + 6.0 * ramp[:, None]).to(dtype)
    for x in range(n):
        kp[int(table[0, x // S]), 0, x % S] = k[x].cuda()
    q = (torch.rand(1, 2, T, D) + 0.5).to(dtype)
    out, lse = tree_attention(q.cuda(), kp, vp, table, seq, return_lse=True)
    check(out, lse, q, [k.float().numpy()[None]], vs, [T], 1 / math.sqrt(D), dtype)


@pytest.mark.parametrize("dtype,S,D", [(BF, 16, 128), (HF, 64, 64), (FP, 16, 64)])
def test_infinite_scores(dtype, S, D):
    """+inf among the seen scores gives NaN as softmax does; -inf is a weight of 0."""
    kp, vp, table, seq, ks, vs = build([300], 1, S, D, dtype)
    q = torch.ones(1, 1, 2, D, dtype=dtype, device="cuda")
    clean = tree_attention(q, kp, vp, table, seq)
    page, slot = int(table[0, 37 // S]), 37 % S
    keep = kp[page, 0, slot].clone()
    kp[page, 0, slot] = math.inf
    assert torch.isnan(tree_attention(q, kp, vp, table, seq)).all()
    kp[page, 0, slot] = -math.inf
    low = tree_attention(q, kp, vp, table, seq)
    there = np.ones(300, dtype=bool)
    there[37] = False
    w, wl, absv, absqk = oracle_attention(q[0].float().cpu().numpy(), ks[0], vs[0], 2, D ** -0.5, there=there)
    lo, _ = bounds(300, D, dtype, absqk, absv, w, wl)
    assert (np.abs(low[0].float().cpu().numpy() - w) <= lo).all()
    kp[page, 0, slot] = keep
    assert torch.equal(tree_attention(q, kp, vp, table, seq), clean)


@pytest.mark.parametrize("dtype,S,D", [(BF, 16, 128), (HF, 64, 64), (FP, 16, 64), (BF, 24, 128)])
def test_strides_rows_and_out(dtype, S, D):
    """Slot-major pages, a query in [n, T, H, D] memory, an output view, rows out of order and twice,
    one tree for all, a scale of its own."""
    g = torch.Generator().manual_seed(5)
    Hq, H, T = 8, 2, 9
    lens = [200, 9, 90, 411]
    kp, vp, table, seq, ks, vs = build(lens, H, S, D, dtype, slots_first=True)
    rows = [3, 1, 3, 0, 2]
    q = torch.randn(5, T, Hq, D, generator=g).to(dtype).cuda().transpose(1, 2)
    hold = torch.full((5, Hq, T + 2, D + 8), 7.0, dtype=dtype, device="cuda")
    out = hold[:, :, 1:T + 1, :D]
    parents = random_parents(1, T, g)[0]
    got, lse = tree_attention(q, kp, vp, table, seq, parents=parents.cuda(), rows=torch.tensor(rows, device="cuda"),
                              softmax_scale=0.21, out=out, return_lse=True)
    assert got is out
    check(out, lse, q, ks, vs, [T] * 5, 0.21, dtype, parents, rows=rows)
    mine = torch.zeros_like(hold, dtype=torch.bool)
    mine[:, :, 1:T + 1, :D] = True
    assert (hold[~mine] == 7.0).all()
    # an output and a query that start off a 16-byte boundary
    odd = torch.empty(5 * Hq * T * D + 1, dtype=dtype, device="cuda")[1:].view(5, Hq, T, D)
    tree_attention(odd.copy_(q), kp, vp, table, seq, parents=parents.cuda(), rows=torch.tensor(rows, device="cuda"),
                   softmax_scale=0.21, out=odd)
    assert torch.equal(odd, out)


@pytest.mark.parametrize("dtype,S,D,T,Hq", [(BF, 16, 128, 40, 4), (HF, 64, 64, 12, 4), (FP, 16, 64, 12, 4),
                                            (BF, 16, 128, 150, 4), (FP, 16, 64, 7, 2)])
def test_what_is_not_seen_does_not_reach_the_output(dtype, S, D, T, Hq):
    """Nodes with NaN or infinite keys and values change only the nodes that see them."""
    g = torch.Generator().manual_seed(9)
    H, ctx = 2, 100
    kp, vp, table, seq, ks, vs = build([ctx + T], H, S, D, dtype)
    q = torch.randn(1, Hq, T, D, generator=g).to(dtype).cuda()
    parents = random_parents(1, T, g, branch=0.3)
    parents[0, 3:5] = 0
    clean = tree_attention(q, kp, vp, table, seq, parents=parents.cuda())
    bad = {3: math.nan, 4: math.inf}
    for u, x in bad.items():
        page, slot = int(table[0, (ctx + u) // S]), (ctx + u) % S
        kp[page, :, slot] = math.nan
        vp[page, :, slot, ::2] = x
        vp[page, 1, slot, 1::2] = -x
    got = tree_attention(q, kp, vp, table, seq, parents=parents.cuda())
    sees = torch.zeros(T, dtype=torch.bool)
    for t in range(T):
        u = t
        while u >= 0:
            sees[t] |= u in bad
            u = int(parents[0, u])
    assert sees.any() and not sees.all()
    assert torch.equal(got[:, :, ~sees], clean[:, :, ~sees])
    assert torch.isnan(got[:, :, sees]).all()  # the keys are NaN
    # finite keys, infinite values: a node that sees one gets that infinity
    for u in bad:
        page, slot = int(table[0, (ctx + u) // S]), (ctx + u) % S
        kp[page, :, slot] = 0.25
        vp[page, :, slot] = math.inf
        vp[page, :, slot, 5] = -math.inf
        vp[page, :, slot, 6] = 1.0
    got = tree_attention(q, kp, vp, table, seq, parents=parents.cuda())
    assert torch.equal(got[:, :, ~sees], clean[:, :, ~sees])
    assert (got[:, :, sees, 7] == math.inf).all() and (got[:, :, sees, 5] == -math.inf).all()
    assert torch.isfinite(got[:, :, sees, 6]).all()


@pytest.mark.parametrize("dtype,S", [(BF, 16), (BF, 64), (FP, 16)])
def test_sequences_that_cannot_be_read(dtype, S):
    """Rows out of range, more nodes than tokens, a length past the row: 0 and -inf; pages out of
    range: their tokens are left out."""
    D, H, T = 64, 2, 4
    lens = [100, 100, 3, 100, 100]
    kp, vp, table, seq, ks, vs = build(lens, H, S, D, dtype)
    seq[3] = 100000
    table[4, 0] = -1
    table[4, 1] = kp.shape[0]
    q = torch.randn(7, 4, T, D).to(dtype)
    rows = [0, 1, 2, 3, 4, -1, 5]
    out, lse = tree_attention(q.cuda(), kp, vp, table, seq, rows=torch.tensor(rows, dtype=torch.int32, device="cuda"),
                              num_nodes=torch.tensor([4, 0, 4, 4, 4, 4, 4], device="cuda"), return_lse=True)
    dead = [1, 2, 3, 5, 6]
    assert (out[dead] == 0).all() and torch.isneginf(lse[dead]).all()
    there = [np.ones(x, dtype=bool) for x in lens]
    there[4][:2 * S] = False
    check(out[[0, 4]], lse[[0, 4]], q[[0, 4]], ks, vs, [4, 4], 1 / 8, dtype, rows=[0, 4], there=there)


def test_parents_that_do_not_come_first_are_roots():
    """A parent at or after its child ends the walk."""
    D, S, T = 64, 16, 6
    kp, vp, table, seq, ks, vs = build([50], 1, S, D, BF)
    q = torch.randn(1, 1, T, D).to(BF)
    parents = torch.tensor([0, 5, 1, 3, -7, 2])
    want = torch.tensor([-1, -1, 1, -1, -1, 2])
    out, lse = tree_attention(q.cuda(), kp, vp, table, seq, parents=parents.cuda(), return_lse=True)
    check(out, lse, q, ks, vs, [T], 1 / 8, BF, want)


def test_equals_flash_attention_on_a_dense_cache():
    """A chunk's chain over a whole prompt is the last rows of causal attention."""
    H, D, N, T, S = 4, 128, 700, 130, 64
    kp, vp, table, seq, ks, vs = build([N], H, S, D, BF)
    q = torch.randn(1, H, N, D).to(BF).cuda()
    k, v = (torch.from_numpy(x[0])[None].to(BF).cuda() for x in (ks, vs))
    full = flash_attention_forward(q, k, v, causal=True)
    got = tree_attention(q[:, :, -T:], kp, vp, table, seq)
    # both round P and the output to bf16: at most two roundings of each apart
    assert (got.float() - full[:, :, -T:].float()).abs().max() <= 4 * 2.0 ** -8 * v.float().abs().max()


def test_deterministic_two_streams_and_graph():
    g = torch.Generator().manual_seed(2)
    H, Hq, D, S, T = 2, 8, 128, 16, 8
    lens = [3000, 37, 900, 2100]
    kp, vp, table, seq, ks, vs = build(lens, H, S, D, BF)
    q = torch.randn(4, Hq, T, D, generator=g).to(BF).cuda()
    parents = random_parents(4, T, g).cuda().int()
    first = tree_attention(q, kp, vp, table, seq, parents=parents)
    outs = []
    torch.cuda.synchronize()
    for s in [torch.cuda.Stream() for _ in range(4)]:
        with torch.cuda.stream(s):
            outs += [tree_attention(q, kp, vp, table, seq, parents=parents) for _ in range(5)]
    torch.cuda.synchronize()
    assert all(torch.equal(o, first) for o in outs)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            o = tree_attention(q, kp, vp, table, seq, parents=parents)
        graphs.append((graph, o))
    for graph, _ in graphs:
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, first) for _, o in graphs)
    seq[0] = 1500
    seq[1] = 8
    for graph, _ in graphs:
        graph.replay()
    want = tree_attention(q, kp, vp, table, seq, parents=parents)
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for _, o in graphs) and not torch.equal(want, first)


def test_pages_past_32_bits():
    P = 2 ** 31 // (2 * 64 * 128) + 40
    kp = torch.empty(P, 2, 64, 128, dtype=BF, device="cuda")
    vp = torch.empty_like(kp)
    ks, vs, table, seq, kn, vn = build([200], 2, 64, 128, BF)
    at = [P - 1, P - 30, 5, P - 7]
    big = torch.tensor([at], dtype=torch.int32, device="cuda")
    for j, pg in enumerate(at):
        kp[pg], vp[pg] = ks[table[0, j]], vs[table[0, j]]
    q = torch.randn(1, 4, 3, 128).to(BF).cuda()
    assert torch.equal(tree_attention(q, kp, vp, big, seq), tree_attention(q, ks, vs, table[:, :4].contiguous(), seq))


def test_refusals():
    kp, vp, table, seq, _, _ = build([50, 20], 2, 16, 64, BF)
    q = torch.randn(2, 4, 3, 64, device="cuda").to(BF)
    i32 = dict(dtype=torch.int32, device="cuda")
    par = torch.zeros(2, 3, **i32)
    msk = torch.ones(3, 3, dtype=torch.bool, device="cuda")
    for kw in [dict(parents=par, tree_mask=msk), dict(parents=par[:, :2]), dict(parents=par.float()),
               dict(tree_mask=msk.int()), dict(tree_mask=msk[:2]), dict(num_nodes=torch.ones(3, **i32)),
               dict(rows=torch.zeros(1, **i32)), dict(softmax_scale=0.0), dict(softmax_scale=-1.0),
               dict(softmax_scale=math.inf), dict(out=torch.empty(2, 4, 3, 32, device="cuda", dtype=BF)),
               dict(parents=par.cpu()), dict(num_nodes=torch.ones(2, dtype=torch.int32))]:
        with pytest.raises((ValueError, RuntimeError)):
            tree_attention(q, kp, vp, table, seq, **kw)
    for bad in [(q.float(), kp, vp, table, seq), (q[:, :3], kp, vp, table, seq), (q[..., :32], kp, vp, table, seq),
                (q, kp, vp.float(), table, seq), (q, kp, vp, table.long(), seq), (q, kp, vp, table, seq.long()),
                (q, kp, vp, table, seq[:1]), (q.repeat(2, 1, 1, 1), kp, vp, table, seq), (q[0], kp, vp, table, seq),
                (q, kp[0], vp[0], table, seq)]:
        with pytest.raises((ValueError, RuntimeError)):
            tree_attention(*bad)
    empty = tree_attention(q[:0], kp, vp, table, seq, rows=torch.zeros(0, **i32))
    assert empty.shape == (0, 4, 3, 64)
    assert tree_attention(q[:, :, :0], kp, vp, table, seq).shape == (2, 4, 0, 64)


@pytest.mark.parametrize("dtype,S,D", [(BF, 16, 128), (HF, 64, 64), (FP, 16, 64)])
def test_decoding_with_forks_drafts_and_eviction(dtype, S, D):
    """The operators as a program uses them: a prompt in two chunks, two samples from it, a draft
    tree whose path is accepted, an eviction, a decode step, the rows freed."""
    g = torch.Generator().manual_seed(1)
    H, Hq, L = 2, 8, 2
    cache = PagedKVCache.allocate(L, 80, H, S, D, num_rows=3, max_pages=24, dtype=dtype)
    cache.k_pages.fill_(math.nan)
    cache.v_pages.fill_(math.nan)
    held = {0: [np.zeros((L, 2, H, 0, D), dtype=np.float32)][0]}

    def add(rows, T):
        cache.extend(T, torch.tensor(rows, device="cuda"))
        for layer in range(L):
            k, v = ((torch.randn(len(rows), T, H, D, generator=g)).to(dtype).transpose(1, 2) for _ in range(2))
            cache.write(layer, k.cuda(), v.cuda(), rows=torch.tensor(rows, device="cuda"))
            new = torch.stack([k, v], 1).float().numpy()
            for i, r in enumerate(rows):
                if layer == 0:
                    held[r] = np.concatenate([held[r], np.zeros((L, 2, H, T, D), dtype=np.float32)], axis=3)
                held[r][layer][:, :, -T:] = new[i]

    def attend(rows, T, parents=None):
        for layer in range(L):
            q = torch.randn(len(rows), Hq, T, D, generator=g).to(dtype)
            out, lse = cache.attend(layer, q.cuda(), parents=None if parents is None else parents.cuda(),
                                    rows=torch.tensor(rows, device="cuda"), return_lse=True)
            ks, vs = ({r: held[r][layer][x] for r in held} for x in (0, 1))
            check(out, lse, q, ks, vs, [T] * len(rows), 1 / math.sqrt(D), dtype, parents, rows=rows)

    add([0], 150)
    attend([0], 150)
    add([0], 61)
    attend([0], 61)
    cache.fork(torch.tensor([0, 0], device="cuda"), torch.tensor([1, 2], device="cuda"))
    held[1], held[2] = held[0].copy(), held[0].copy()
    start = cache.seq_lens.clone()
    parents = torch.tensor([-1, 0, 0, 1, 1, 2, 3])
    add([0, 1, 2], 7)
    attend([2, 0, 1], 7, parents)
    paths = [[0, 1, 3, 6], [0, 2], [0]]
    keep = torch.tensor([p + [-1] * (4 - len(p)) for p in paths], device="cuda")
    cache.compact(keep, torch.tensor([len(p) for p in paths], dtype=torch.int32, device="cuda"), start=start)
    for r, p in enumerate(paths):
        held[r] = np.concatenate([held[r][:, :, :, :211], held[r][:, :, :, 211:][:, :, :, p]], axis=3)
    imp = torch.rand(1, held[1].shape[3], generator=g).cuda()
    keep, counts = select_indices_batched(held[1].shape[3], 70, imp)
    cache.compact(keep, counts[:, 0], src=torch.tensor([1], device="cuda"))
    held[1] = held[1][:, :, :, keep[0, :int(counts[0, 0])].cpu().numpy()]
    add([0, 1, 2], 1)
    attend([0, 1, 2], 1)
    cache.check()
    cache.truncate(torch.tensor([100, 50, 10], device="cuda"))
    for r, x in enumerate([100, 50, 10]):
        held[r] = held[r][:, :, :, :x]
    add([1], 3)
    attend([1], 3)
    attend([0], 1)
    cache.free()
    cache.check()
    assert cache.free_pages() == 80 and int(cache.seq_lens.sum()) == 0
