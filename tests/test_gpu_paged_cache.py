"""The paged KV cache's page updates and writes against the plain oracle: page numbers, lengths,
use counts, status and every byte of the pages are equal, also behind the sequences."""

import random

import numpy as np
import pytest
import torch

from oracle.paged_oracle import PagedOracle

pytestmark = pytest.mark.gpu

cab = pytest.importorskip("cab_attention")
from cab_attention import PagedKVCache, _lib  # noqa: E402
from cab_attention.eviction import select_indices_batched  # noqa: E402


@pytest.fixture(autouse=True)
def _device_status_clean():
    yield
    assert _lib.device_status() == 0


def make(L=2, P=40, H=2, S=16, D=64, R=6, W=10, dtype=torch.bfloat16, seed=0, slots_first=False):
    """A cache with random pages (so copies from a wrong place show) and its oracle."""
    g = torch.Generator().manual_seed(seed)
    shape = (L, P, S, H, D) if slots_first else (L, P, H, S, D)
    k, v = (torch.randn(shape, generator=g).to(dtype).cuda() for _ in range(2))
    if slots_first:
        k, v = k.transpose(2, 3), v.transpose(2, 3)
    i32 = dict(dtype=torch.int32, device="cuda")
    c = PagedKVCache(k, v, torch.full((R, W), -1, **i32), torch.zeros(R, **i32), torch.zeros(P, **i32),
                     torch.zeros(1, **i32))
    return c, oracle_of(c)


def oracle_of(c):
    o = PagedOracle(*(t.float().cpu().numpy() for t in (c.k_pages, c.v_pages)),
                    *(t.cpu().numpy().astype(np.int64) for t in (c.block_table, c.seq_lens, c.ref_counts)))
    o.status = int(c.status.item())
    return o


def same(c, o):
    assert int(c.status.item()) == o.status
    for name in ("lens", "refs", "table"):
        t = {"lens": c.seq_lens, "refs": c.ref_counts, "table": c.block_table}[name]
        assert np.array_equal(t.cpu().numpy(), getattr(o, name)), name
    assert np.array_equal(c.k_pages.float().cpu().numpy(), o.k, equal_nan=True)
    assert np.array_equal(c.v_pages.float().cpu().numpy(), o.v, equal_nan=True)


def dev(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device="cuda")


def pairs(src, dst=None, start=None, keep=None, grow=None):
    n = len(src)
    pick = lambda x, i: x[i] if isinstance(x, (list, tuple)) else x  # noqa: E731
    return [dict(src=src[i], dst=src[i] if dst is None else dst[i], start=pick(start, i),
                 keep=None if keep is None else keep[i], grow=0 if grow is None else pick(grow, i)) for i in range(n)]


@pytest.mark.parametrize("S,D,dtype,first", [(16, 64, torch.bfloat16, False), (5, 24, torch.float16, True),
                                             (64, 128, torch.float32, False), (1, 3, torch.bfloat16, False),
                                             (128, 64, torch.float16, True), (33, 6, torch.bfloat16, True)])
@pytest.mark.parametrize("seed", [0, 1])
def test_random_calls_match_oracle(S, D, dtype, first, seed):
    rng = random.Random(seed * 1000 + S)
    R, W, P = 6, 7, 30
    c, o = make(P=P, S=S, D=D, R=R, W=W, dtype=dtype, seed=seed, slots_first=first)
    for _ in range(60):
        n = rng.randint(1, R)
        rows = rng.sample(range(R), n)
        op = rng.choice(["extend", "extend", "write", "truncate", "free", "fork", "compact", "compact", "accept", "branch"])
        lens = [int(x) for x in o.lens]
        if op == "extend":
            grow = [rng.choice([0, 1, S - 1, S, rng.randint(0, 2 * S)]) for _ in rows]
            c.extend(dev(grow), dev(rows))
            o.update(pairs(rows, grow=grow), copies=False)
        elif op == "write":
            T = rng.randint(1, 2 * S)
            m = [min(lens[r], rng.randint(0, T)) for r in rows]
            k, v = (torch.randn(n, T, 2, D).to(dtype).cuda().transpose(1, 2) for _ in range(2))
            c.write(1, k, v, dev(m), dev(rows))
            o.write(1, k.float().cpu().numpy(), v.float().cpu().numpy(), rows, m)
        elif op == "truncate":
            new = [rng.randint(0, lens[r]) for r in rows]
            c.truncate(dev(new), dev(rows, torch.int64))
            o.update(pairs(rows, start=new))
        elif op == "free":
            c.free(dev(rows))
            o.update(pairs(rows, start=0), copies=False)
        elif op == "fork":
            src = [rng.randrange(R) for _ in rows]
            c.fork(dev(src), dev(rows))
            o.update(pairs(src, rows))
        else:
            src = [rng.randrange(R) for _ in rows] if op == "branch" else rows
            start = [rng.randint(0, lens[r]) if op == "accept" else 0 for r in src]
            keep = []
            for r, a in zip(src, start):
                room = lens[r] - a
                ks = rng.sample(range(room), rng.randint(0, room)) if room else []
                if rng.random() < 0.7:
                    ks.sort()
                if ks and rng.random() < 0.3:
                    ks[: len(ks) // 2] = range(len(ks) // 2)
                if ks and rng.random() < 0.2:
                    ks[-1] = ks[0]  # the same token twice
                keep.append(ks)
            K = max(len(x) for x in keep) + rng.randint(0, 2)
            pad = [x + [-1] * (K - len(x)) for x in keep]
            kt = dev(pad, rng.choice([torch.int32, torch.int64])).reshape(n, K)
            c.compact(kt, dev([[len(x), 9] for x in keep])[:, 0], start=dev(start), src=dev(src),
                      dst=dev(rows) if op == "branch" else None)
            o.update(pairs(src, rows, start=start, keep=keep))
        same(c, o)
        if o.status:  # refused for want of pages or table room: nothing changed; go on
            with pytest.raises(RuntimeError):
                c.check()
            o.status = 0
        assert int((c.ref_counts < 0).sum()) == 0


def test_refusals_leave_the_cache_as_it_was():
    c, o = make(P=8, S=16, R=4, W=6)
    c.extend(dev([40, 20, 0, 5]))
    o.update(pairs([0, 1, 2, 3], grow=[40, 20, 0, 5]), copies=False)
    same(c, o)
    calls = [
        (lambda: c.extend(16 * 3), 1),                                   # 8 pages, 6 used
        (lambda: c.extend(97, dev([2])), 2),                             # 6 pages a row
        (lambda: c.extend(1, dev([4])), 4),
        (lambda: c.extend(1, dev([-1])), 4),
        (lambda: c.extend(1, dev([2 ** 32], torch.int64)), 4),           # not row 0
        (lambda: c.truncate(dev([2 ** 32 + 3], torch.int64), dev([0])), 8),
        (lambda: c.extend(1, dev([1, 1])), 4),
        (lambda: c.fork(dev([0, 0]), dev([2, 2])), 4),
        (lambda: c.truncate(41, dev([0])), 8),
        (lambda: c.truncate(dev([-1]), dev([0])), 8),
        (lambda: c.extend(dev([-1]), dev([0])), 8),
        (lambda: c.compact(dev([[0, 40]]), src=dev([0])), 8),            # position past the row
        (lambda: c.compact(dev([[0, -1]]), src=dev([0])), 8),
        (lambda: c.compact(dev([[0, 1]]), dev([3]), src=dev([0])), 8),   # more than the list has
        (lambda: c.compact(dev([[0, 1]]), start=dev([41]), src=dev([0])), 8),
        (lambda: c.write(0, *(torch.zeros(1, 2, 6, 64, dtype=torch.bfloat16, device="cuda"),) * 2, rows=dev([3])), 8),
        (lambda: c.write(0, *(torch.zeros(1, 2, 1, 64, dtype=torch.bfloat16, device="cuda"),) * 2, rows=dev([9])), 4),
    ]
    for call, bit in calls:
        call()
        o.status = bit
        same(c, o)
        c.extend(1, dev([2]))  # frozen until the refusal has been seen
        same(c, o)
        with pytest.raises(RuntimeError, match="paged KV cache"):
            c.check()
        o.status = 0
    c.check()
    c.extend(1, dev([2]))
    o.update(pairs([2], grow=1), copies=False)
    same(c, o)


def test_bad_table_is_refused():
    c, o = make(P=8, S=16, R=3, W=4)
    c.extend(dev([40, 20, 0]))
    c.block_table[0, 1] = 8
    o = oracle_of(c)
    c.free(dev([0]))
    assert int(c.status.item()) == 16
    c.status.zero_()
    same(c, o)
    c.block_table[0, 1] = c.block_table[0, 0]
    c.seq_lens[2] = 1000  # longer than its row
    o = oracle_of(c)
    c.fork(dev([2]), dev([1]))
    assert int(c.status.item()) == 16
    c.status.zero_()
    same(c, o)


@pytest.mark.parametrize("n,K,P", [(3, 5000, 4000), (40, 700, 9000), (1, 60000, 9000)])
def test_eviction_selection_feeds_compact(n, K, P):
    """The policy's list and counts go into compact as they are; big enough for the cluster form."""
    S, N = 16, 2 * K
    g = torch.Generator().manual_seed(K)
    c, _ = make(L=1, P=P + n * (N // S + 1), H=1, S=S, D=8, R=n, W=N // S + 1, seed=K)
    c.extend(N)
    imp = torch.rand(n, N, generator=g).cuda()
    keep, counts = select_indices_batched(N, K, imp)
    o = oracle_of(c)
    c.compact(keep, counts[:, 0])
    c.check()
    o.update(pairs(list(range(n)), start=0, keep=[keep[i, :int(counts[i, 0])].tolist() for i in range(n)]))
    same(c, o)


def test_many_pairs_and_swapped_rows():
    n = 1024
    c, _ = make(L=1, P=5000, H=1, S=4, D=8, R=n, W=6, seed=3)
    g = torch.Generator().manual_seed(1)
    c.extend(torch.randint(0, 15, (n,), generator=g).cuda())
    o = oracle_of(c)
    src = torch.randint(0, n, (n,), generator=g)
    dst = torch.randperm(n, generator=g)
    c.fork(src.cuda(), dst.cuda())
    o.update(pairs(src.tolist(), dst.tolist()))
    same(c, o)
    c.check()
    with pytest.raises(RuntimeError, match="1024"):
        c.fork(torch.zeros(n + 1, dtype=torch.int32, device="cuda"), torch.arange(n + 1, device="cuda"))


def test_pages_past_32_bits():
    """Element offsets above 2^31 in the pages."""
    P = 2 ** 31 // (2 * 64 * 128) + 40
    k = torch.empty(1, P, 2, 64, 128, dtype=torch.bfloat16, device="cuda")
    v = torch.empty_like(k)
    i32 = dict(dtype=torch.int32, device="cuda")
    refs = torch.ones(P, **i32)
    refs[-20:] = 0
    c = PagedKVCache(k, v, torch.full((2, 8), -1, **i32), torch.zeros(2, **i32), refs, torch.zeros(1, **i32))
    c.extend(300, dev([0]))
    kk, vv = (torch.randn(1, 2, 300, 128, device="cuda").to(torch.bfloat16) for _ in range(2))
    c.write(0, kk, vv, rows=dev([0]))
    c.compact(torch.arange(1, 300, 2, device="cuda")[None], src=dev([0]), dst=dev([1]))
    c.check()
    pg = c.block_table[1, :3].long()
    assert pg.tolist() == [P - 15, P - 14, P - 13]
    got = k[0, pg].transpose(0, 1).reshape(2, 192, 128)[:, :150]
    assert torch.equal(got, kk[0, :, 1::2])
    assert torch.equal(v[0, pg].transpose(0, 1).reshape(2, 192, 128)[:, :150], vv[0, :, 1::2])


def test_graph_replay_and_side_stream():
    c, _ = make(P=60, S=16, R=4, W=12)
    c.extend(dev([30, 20, 10, 3]))
    keep, num, start = dev([[0, 2], [1, 3], [0, 1], [0, 2]]), dev([2, 1, 2, 2]), c.seq_lens.clone()
    k = torch.randn(4, 2, 5, 64, device="cuda").to(torch.bfloat16)

    def step():  # draft five tokens, accept a path, keep it
        start.copy_(c.seq_lens)
        c.extend(5)
        c.write(0, k, k)
        c.compact(keep, num, start=start)

    o = oracle_of(c)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step()
        graph.replay()
        graph.replay()
    torch.cuda.current_stream().wait_stream(side)
    for _ in range(3):
        at = o.lens.tolist()
        o.update(pairs([0, 1, 2, 3], grow=5), copies=False)
        o.write(0, k.float().cpu().numpy(), k.float().cpu().numpy())
        o.update(pairs([0, 1, 2, 3], start=at, keep=[[0, 2], [1], [0, 1], [0, 2]]))
    same(c, o)
    c.check()


@pytest.mark.parametrize("S,D,lens", [(16, 64, [3, 40, 0, 17]), (16, 128, [900, 5, 700, 60])])
def test_queued_steps_equal_waited_ones(S, D, lens):
    """Decode steps queued without a wait, so that each kernel is launched while those before it run,
    give what the same steps give with a wait after every call."""
    def steps(wait):
        c, _ = make(L=1, P=400, S=S, D=D, R=4, W=64, seed=1)
        pause = torch.cuda.synchronize if wait else (lambda: None)
        g = torch.Generator(device="cuda").manual_seed(4)
        kv = torch.randn(8, 4, 2, 3, D, device="cuda", generator=g).to(torch.bfloat16)
        first = torch.randn(4, 2, max(lens), D, device="cuda", generator=g).to(torch.bfloat16)
        c.extend(dev(lens))
        pause()
        c.write(0, first, first, dev(lens))
        pause()
        outs = []
        for i in range(40):
            n = c.seq_lens.clone()
            c.extend(3)
            pause()
            c.write(0, kv[i % 8], kv[(i + 3) % 8])
            pause()
            outs.append(c.attend(0, kv[(i + 1) % 8].repeat_interleave(2, 1)))
            pause()
            c.compact(dev([[0, 2], [1, 0], [0, 0], [2, 1]]), dev([2, 1, 2, 1]), start=n)
            pause()
            if i % 5 == 4:
                c.fork(dev([0, 1]), dev([2, 3]))
                pause()
        c.check()
        return outs + [c.k_pages, c.v_pages, c.block_table, c.seq_lens, c.ref_counts]

    want = steps(True)
    for _ in range(3):
        for x, y in zip(steps(False), want):
            assert torch.equal(x, y)
