"""Refused calls of the paged cache leave it as it was, also where only one of many rows is at fault."""

import pytest
import torch

from test_gpu_paged_cache import dev, make, oracle_of, same

pytestmark = pytest.mark.gpu

from cab_attention import _lib  # noqa: E402


@pytest.fixture(autouse=True)
def _device_status_clean():
    yield
    assert _lib.device_status() == 0


# the second has more table entries to check than a CTA of the write looks at by itself
@pytest.mark.parametrize("R,S,T", [(64, 16, 40), (600, 4, 21)])
@pytest.mark.parametrize("at", [0, 37, 63])
@pytest.mark.parametrize("fault", ["count", "negative", "row", "twice", "table", "length"])
def test_one_bad_row_in_a_write(R, S, T, at, fault):
    H, D = 4, 64
    W = 60 // S + 2
    c, _ = make(L=1, P=R * W, H=H, S=S, D=D, R=R, W=W, seed=at)
    c.extend(dev([T + i % 17 for i in range(R)]))
    rows = torch.randperm(R, generator=torch.Generator().manual_seed(1)).to(torch.int32).cuda()
    num = dev([T - i % 3 for i in range(R)])
    k, v = (torch.randn(R, T, H, D, device="cuda").to(torch.bfloat16).transpose(1, 2) for _ in range(2))
    good = rows.clone(), num.clone(), c.block_table.clone(), c.seq_lens.clone()
    row = int(rows[at])
    if fault == "count":
        num[at] = T + 1
        bit = 8
    elif fault == "negative":
        num[at] = -1
        bit = 8
    elif fault == "row":
        rows[at] = R
        bit = 4
    elif fault == "twice":
        rows[at] = rows[(at + 20) % R]
        bit = 4
    elif fault == "table":
        c.block_table[row, (int(c.seq_lens[row]) - 1) // S] = c.num_pages
        bit = 16
    else:
        c.seq_lens[row] = W * S + 1
        bit = 8
    o = oracle_of(c)
    for _ in range(3):
        c.write(0, k, v, num, rows)
        o.status = bit
        same(c, o)
        with pytest.raises(RuntimeError, match="paged KV cache"):
            c.check()
    rows, num = good[:2]
    c.block_table.copy_(good[2])
    c.seq_lens.copy_(good[3])
    o = oracle_of(c)
    c.write(0, k, v, num, rows)
    c.check()
    o.write(0, k.float().cpu().numpy(), v.float().cpu().numpy(), rows.tolist(), num.tolist())
    same(c, o)


@pytest.mark.parametrize("T", [1, 3000])
def test_a_write_after_a_refusal_does_nothing(T):
    c, _ = make(P=800, S=4, W=800)
    c.extend(dev([3000, 1]), dev([0, 1]))
    c.extend(1, dev([9]))
    o = oracle_of(c)
    assert o.status == 4
    kv = torch.ones(1, 2, T, 64, dtype=torch.bfloat16, device="cuda")
    c.write(0, kv, kv, rows=dev([0]))
    same(c, o)
    c.write(0, kv, kv, rows=dev([-1]))  # the refusal that was there stays the only one
    same(c, o)


def test_counts_that_do_not_fit():
    """Numbers past 31, 32, 63 and 64 bits are refused like any count that is too large."""
    c, _ = make(P=20, R=3, W=6)
    c.extend(dev([40, 16, 0]))
    c.check()
    o = oracle_of(c)
    for big in (2 ** 31 - 1, 2 ** 31, 2 ** 32 + 1, 2 ** 63 - 1, 2 ** 63, 2 ** 64 + 1, 10 ** 30):
        for call, bit in ((lambda: c.extend(big), 2), (lambda: c.extend(big, dev([1])), 2),
                          (lambda: c.truncate(big), 8),
                          (lambda: c.compact(dev([[0]]), start=big, src=dev([0])), 8)):
            call()
            o.status = bit
            same(c, o)
            with pytest.raises(RuntimeError, match="paged KV cache"):
                c.check()
            o.status = 0


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_counts_of_an_empty_list(dtype):
    """A keep list without columns holds no positions, whatever keep_num says."""
    c, _ = make(P=20, R=3, W=6)
    c.extend(dev([40, 16, 5]))
    o = oracle_of(c)
    empty = torch.empty(2, 0, dtype=dtype, device="cuda")
    c.compact(empty, dev([0, 2]), start=7, src=dev([0, 1]))
    o.status = 8
    same(c, o)
    with pytest.raises(RuntimeError, match="paged KV cache"):
        c.check()
    c.compact(empty, dev([0, 0]), start=7, src=dev([0, 1]))
    c.compact(empty[:1], start=3, src=dev([2]))
    c.check()
    assert c.seq_lens.tolist() == [7, 7, 3]
