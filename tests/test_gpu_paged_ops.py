"""torch.ops.cab's paged-cache operators: the same results as PagedKVCache's methods, schemas and
fake implementations (opcheck), and a compiled decode step."""

import pytest
import torch

pytestmark = pytest.mark.gpu

cab = pytest.importorskip("cab_attention")
from cab_attention import PagedKVCache, _lib  # noqa: E402


@pytest.fixture(autouse=True)
def _device_status_clean():
    yield
    assert _lib.device_status() == 0


def make(seed=0):
    torch.manual_seed(seed)
    c = PagedKVCache.allocate(1, 24, 2, 16, 64, num_rows=4, max_pages=8)
    c.k_pages.normal_()
    c.v_pages.normal_()
    return c


def tensors(c):
    return (c.k_pages, c.v_pages, c.block_table, c.seq_lens, c.ref_counts, c.status)


def dev(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def test_operators_equal_the_methods():
    a, b = make(), make()
    k = torch.randn(4, 2, 40, 64, device="cuda").to(torch.bfloat16)
    q = torch.randn(4, 8, 3, 64, device="cuda").to(torch.bfloat16)
    grow, keep, num = dev([40, 20, 0, 7]), dev([[0, 3, 5]] * 2), dev([3, 2])
    ops, t = torch.ops.cab, tensors(b)
    a.extend(grow)
    ops.pages_extend(*t, grow, None)
    a.write(0, k, k, num_new=grow)
    ops.pages_write(*t, 0, k, k, grow, None)
    a.compact(keep, num, start=dev([10, 5]), src=dev([0, 1]))
    ops.pages_compact(*t, keep, num, dev([10, 5]), dev([0, 1]), None)
    a.fork(dev([0, 1]), dev([2, 3]))
    ops.pages_fork(*t, dev([0, 1]), dev([2, 3]))
    a.truncate(dev([4, 4, 4, 4]))
    ops.pages_truncate(*t, dev([4, 4, 4, 4]), None)
    for x, y in zip(tensors(a), t):
        assert torch.equal(x, y)
    parents = dev([-1, 0, 0])
    want = a.attend(0, q, parents=parents, return_lse=True)
    got = ops.tree_attn(q, b.k_pages[0], b.v_pages[0], b.block_table, b.seq_lens, None, None, parents, None, 0.0)
    assert all(torch.equal(x, y) for x, y in zip(want, got))
    a.check()


def test_opcheck():
    c = make()
    c.extend(20)
    q = torch.randn(4, 8, 3, 64, device="cuda").to(torch.bfloat16)
    torch.library.opcheck(torch.ops.cab.tree_attn.default,
                          (q, c.k_pages[0], c.v_pages[0], c.block_table, c.seq_lens, None, None, dev([-1, 0, 0]), None, 0.0),
                          test_utils=("test_schema", "test_faketensor"))
    for op, args in ((torch.ops.cab.pages_extend.default, (dev([1, 0, 2, 3]), None)),
                     (torch.ops.cab.pages_fork.default, (dev([0]), dev([1]))),
                     (torch.ops.cab.pages_compact.default, (dev([[0, 2]]), None, None, dev([2]), None)),
                     (torch.ops.cab.pages_truncate.default, (dev([1, 1, 1, 1]), None)),
                     (torch.ops.cab.pages_write.default, (0, q[:, :2], q[:, :2], dev([1, 0, 1, 0]), None))):
        torch.library.opcheck(op, (*tensors(c), *args), test_utils=("test_schema", "test_faketensor"))


def test_compiled_step_matches_eager():
    q = torch.randn(4, 8, 1, 64, device="cuda").to(torch.bfloat16)
    k = torch.randn(4, 2, 1, 64, device="cuda").to(torch.bfloat16)

    def step(q, k, kp, vp, table, lens, refs, status, one):
        torch.ops.cab.pages_extend(kp, vp, table, lens, refs, status, one, None)
        torch.ops.cab.pages_write(kp, vp, table, lens, refs, status, 0, k, k, None, None)
        return torch.ops.cab.tree_attn(q, kp[0], vp[0], table, lens, None, None, None, None, 0.0)[0]

    a, b = make(), make()
    for c in (a, b):
        c.extend(dev([30, 0, 3, 16]))
    eager = step(q, k, *tensors(a), dev([1, 1, 1, 1]))
    compiled = torch.compile(step, fullgraph=True, backend="aot_eager")(q, k, *tensors(b), dev([1, 1, 1, 1]))
    assert torch.equal(eager, compiled)
    assert all(torch.equal(x, y) for x, y in zip(tensors(a), tensors(b)))
