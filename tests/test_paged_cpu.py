"""The paged KV cache without a GPU: C-ABI argument checks, refusals of the Python layer, and
the oracle's own invariants."""

import ctypes
import random

import numpy as np
import pytest
import torch

from cab_attention import PagedKVCache, _lib
from cab_attention.kernels import tree_attention
from oracle.paged_oracle import PagedOracle, tree_attention as oracle_attention


@pytest.fixture(scope="module")
def lib():
    import cab_build
    cab_build.build()
    return _lib.lib()


def fake_cache(**change):
    c = _lib.PageCache()
    for name in ("k_pages", "v_pages", "block_table", "seq_lens", "ref_counts", "status"):
        setattr(c, name, 16)
    c.layers, c.pages, c.heads, c.page_size, c.dim = 1, 8, 2, 16, 64
    c.k_strides[:] = c.v_strides[:] = (8 * 2 * 16 * 64, 2 * 16 * 64, 16 * 64, 64)
    c.rows, c.width, c.table_stride, c.dtype = 4, 6, 6, 2
    for name, value in change.items():
        setattr(c, name, value)
    return c


def test_c_abi_refusals(lib):
    size = _lib._c_size(0)
    fake = ctypes.c_void_p(256)

    def update(c, n=2, src=None, keep=None, keep_bytes=8, cols=0, grow=0, copies=1, ws=fake, nbytes=1 << 20):
        return lib.cab_pages_update(c, src, None, n, None, -1, keep, keep_bytes, cols, cols, None, 1, None, grow, copies,
                                    ws, nbytes, None)

    assert lib.cab_pages_update_workspace_size(fake_cache(), 2, ctypes.byref(size)) == 0 and size.value > 0
    assert lib.cab_pages_update_workspace_size(fake_cache(), 0, ctypes.byref(size)) == 2
    assert lib.cab_pages_update_workspace_size(fake_cache(), 1025, ctypes.byref(size)) == 2
    assert lib.cab_pages_update_workspace_size(fake_cache(pages=0), 2, ctypes.byref(size)) == 1
    assert lib.cab_pages_update_workspace_size(fake_cache(width=1 << 28), 2, ctypes.byref(size)) == 2
    assert update(None) == 1
    assert update(fake_cache(status=None)) == 1
    assert update(fake_cache(k_pages=None)) == 1
    assert update(fake_cache(table_stride=5)) == 1
    assert update(fake_cache(dtype=7)) == 2
    assert update(fake_cache(), n=5) == 1                 # five rows of four
    assert update(fake_cache(), grow=-1) == 1
    assert update(fake_cache(), cols=4) == 1              # no list
    assert update(fake_cache(), keep=fake, keep_bytes=2, cols=4) == 1
    assert update(fake_cache(), keep=fake, cols=4, copies=0) == 1
    assert update(fake_cache(), nbytes=8) == 5
    assert update(fake_cache(), ws=None) == 5

    s3 = _lib._i64_3(2048, 1024, 64)
    write = lambda c, layer=0, n=1, T=1, k=fake, m=1: lib.cab_pages_write(c, layer, k, fake, n, T, s3, s3, None, None, m, None)  # noqa: E731
    assert write(fake_cache(), layer=1) == 1
    assert write(fake_cache(), n=5) == 1
    assert write(fake_cache(), T=0) == 1
    assert write(fake_cache(), m=2) == 1
    assert write(fake_cache(), k=None) == 1

    def attend(c, n=1, Hq=4, T=2, layer=0, q=fake, parents=None, mask=None, scale=0.1, ws=fake, nbytes=1 << 30):
        return lib.cab_tree_attn_fwd(c, layer, q, fake, None, n, Hq, T, s3, s3, None, None, parents, 0, mask, 0, scale,
                                     ws, nbytes, None)

    assert attend(fake_cache(), q=None) == 1
    assert attend(fake_cache(), Hq=3) == 1
    assert attend(fake_cache(), T=0) == 1
    assert attend(fake_cache(), n=5) == 1
    assert attend(fake_cache(), layer=1) == 1
    assert attend(fake_cache(), parents=fake, mask=fake) == 1
    assert attend(fake_cache(), T=1025, parents=fake) == 2
    for scale in (0.0, -1.0, float("inf"), float("nan")):
        assert attend(fake_cache(), scale=scale) == 1
    assert attend(fake_cache(dim=257)) == 2
    assert attend(fake_cache(dtype=5)) == 2
    assert lib.cab_tree_attn_workspace_size(fake_cache(), 1, 4, 2, None) == 1


def test_cpu_tensors_are_refused():
    k = torch.zeros(1, 4, 2, 16, 64)
    i = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="no CPU implementation"):
        PagedKVCache(k, k, torch.zeros(4, 4, dtype=torch.int32), i, i, i[:1])
    with pytest.raises(RuntimeError, match="no CPU implementation"):
        tree_attention(torch.zeros(1, 2, 1, 64), k[0], k[0], torch.zeros(1, 4, dtype=torch.int32), i[:1])


@pytest.mark.parametrize("seed", range(6))
def test_oracle_keeps_every_rows_tokens(seed):
    """After any calls a row holds the tokens that a plain list model holds, use counts equal the
    table's entries, and a page that is not full is in one row."""
    rng = random.Random(seed)
    S, R, W, P = rng.choice([1, 3, 16]), 5, 6, 24
    shape = (1, P, 1, S, 1)
    o = PagedOracle(np.zeros(shape), np.zeros(shape), np.full((R, W), -1), np.zeros(R, dtype=np.int64),
                    np.zeros(P, dtype=np.int64))
    model, tag = [[] for _ in range(R)], 0.0
    for _ in range(80):
        n = rng.randint(1, R)
        rows = rng.sample(range(R), n)
        op = rng.choice(["extend", "cut", "fork", "compact"])
        if op == "extend":
            grow = [rng.randint(0, S + 1) for _ in rows]
            o.update([dict(src=r, dst=r, grow=g) for r, g in zip(rows, grow)], copies=False)
            if not o.status:
                k = np.zeros((n, 1, S + 1, 1))
                for i, (r, g) in enumerate(zip(rows, grow)):
                    for t in range(g):
                        tag += 1
                        k[i, 0, t, 0] = tag
                        model[r] = model[r] + [tag]
                o.write(0, k, k, rows, grow)
        elif op == "cut":
            new = [rng.randint(0, len(model[r])) for r in rows]
            o.update([dict(src=r, dst=r, start=a) for r, a in zip(rows, new)])
            if not o.status:
                for r, a in zip(rows, new):
                    model[r] = model[r][:a]
        else:
            src = [rng.randrange(R) for _ in rows]
            start = [None if op == "fork" else rng.randint(0, len(model[s])) for s in src]
            keep = [[] if a is None or a == len(model[s]) else
                    [rng.randrange(len(model[s]) - a) for _ in range(rng.randint(0, 4))] for s, a in zip(src, start)]
            o.update([dict(src=s, dst=r, start=a, keep=x) for s, r, a, x in zip(src, rows, start, keep)])
            if not o.status:
                old = [list(x) for x in model]
                for s, r, a, x in zip(src, rows, start, keep):
                    model[r] = list(old[s]) if a is None else old[s][:a] + [old[s][a + y] for y in x]
        o.status = 0
        used = np.zeros(P, dtype=np.int64)
        for r in range(R):
            assert o.tokens(0, r)[0].reshape(-1).tolist() == model[r]
            for j in range(o.pages_of(len(model[r]))):
                used[o.table[r, j]] += 1
            assert (o.table[r, o.pages_of(len(model[r])):] == -1).all()
        assert np.array_equal(used, o.refs)
        for r in range(R):
            if len(model[r]) % S:
                assert o.refs[o.table[r, len(model[r]) // S]] == 1


def test_oracle_attention_is_softmax():
    rng = np.random.default_rng(0)
    q, k, v = rng.normal(size=(4, 3, 8)), rng.normal(size=(2, 10, 8)), rng.normal(size=(2, 10, 8))
    out, lse, _, _ = oracle_attention(q, k, v, 3, 0.3, parents=[-1, 0, 0])
    seen = torch.ones(3, 10, dtype=torch.bool)
    seen[:, 7:] = torch.tensor([[1, 0, 0], [1, 1, 0], [1, 0, 1]], dtype=torch.bool)
    kt, vt = (torch.from_numpy(x).repeat_interleave(2, 0) for x in (k, v))
    s = (torch.from_numpy(q) @ kt.transpose(1, 2) * 0.3).masked_fill(~seen, -torch.inf)
    assert np.allclose(out, (torch.softmax(s, -1) @ vt).numpy(), atol=1e-12)
    assert np.allclose(lse, torch.logsumexp(s, -1).numpy(), atol=1e-12)


def test_operators_are_registered_with_fakes():
    from torch._subclasses.fake_tensor import FakeTensorMode
    for name in ("tree_attn", "pages_extend", "pages_write", "pages_compact", "pages_fork", "pages_truncate"):
        assert hasattr(torch.ops.cab, name), name
    with FakeTensorMode():
        q = torch.empty(3, 8, 5, 128, dtype=torch.bfloat16, device="cuda")
        k = torch.empty(20, 2, 16, 128, dtype=torch.bfloat16, device="cuda")
        i = torch.empty(3, 7, dtype=torch.int32, device="cuda")
        out, lse = torch.ops.cab.tree_attn(q, k, k, i, i[:, 0], None, None, None, None, 0.0)
        assert out.shape == q.shape and out.dtype == q.dtype and lse.shape == (3, 8, 5) and lse.dtype == torch.float32
