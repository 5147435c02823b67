"""Tree attention over batches in which sequences, or groups of query rows, have no node: slots that sit
out a step, trees of different sizes in one call. Their rows are 0 and -inf, and those of the others
are the oracle's within the bounds of ``test_gpu_tree_attn``."""

import math

import pytest
import torch

from test_gpu_tree_attn import BF, HF, build, check, random_parents

pytestmark = pytest.mark.gpu

from cab_attention import _lib  # noqa: E402
from cab_attention.kernels import tree_attention  # noqa: E402


@pytest.fixture(autouse=True)
def _device_status_clean():
    yield
    assert _lib.device_status() == 0


# table_tokens: tokens that a table row has room for; up to 512 no unit is cut, else units are cut between CTAs
CASES = [
    # Hq, Hkv, D, S, T, ctx, nodes, tree, dtype
    (8, 8, 128, 16, 1, [200] * 64, [i % 2 for i in range(64)], "chain", BF),
    (8, 8, 64, 16, 1, [128 + 7 * i % 272 for i in range(96)], [int(i % 4 == 3) for i in range(96)], "chain", HF),
    (8, 8, 128, 64, 2, [400 - 3 * i for i in range(64)], [2 * (i // 8 % 2) for i in range(64)], "chain", BF),
    (8, 2, 128, 16, 33, [130 + 5 * i for i in range(48)], [33 - i % 3 for i in range(48)], "mask", BF),
    (8, 2, 64, 16, 33, [130 + 5 * i for i in range(48)], [33 - i % 3 for i in range(48)], "parents", BF),
    (4, 1, 128, 64, 300, [200, 150, 170, 128] * 4, [1, 1, 1, 300] * 4, "chain", BF),
    (4, 1, 64, 32, 70, [129, 300, 128, 256] * 10, [0, 70, 1, 33] * 10, "parents", HF),
    (2, 1, 128, 16, 1, [300] * 300, [int(i % 7 == 6) for i in range(300)], "chain", BF),
]


@pytest.mark.parametrize("Hq,H,D,S,T,ctx,nodes,tree,dtype", CASES)
@pytest.mark.parametrize("table_tokens", [0, 2048])
def test_rows_without_a_node(Hq, H, D, S, T, ctx, nodes, tree, dtype, table_tokens):
    g = torch.Generator().manual_seed(T * 7 + D)
    n = len(ctx)
    kp, vp, table, seq, ks, vs = build([c + m for c, m in zip(ctx, nodes)], H, S, D, dtype, seed=T + S)
    if table_tokens:
        table = torch.nn.functional.pad(table, (0, table_tokens // S - table.shape[1]), value=-1)
    q = torch.randn(n, Hq, T, D, generator=g).to(dtype)
    parents = random_parents(n, T, g) if tree == "parents" else None
    mask = torch.rand(n, T, T, generator=g) < 0.5 if tree == "mask" else None
    call = dict(parents=None if parents is None else parents.cuda(), tree_mask=None if mask is None else mask.cuda(),
                num_nodes=torch.tensor(nodes).cuda(), return_lse=True)
    q_dev = q.cuda()
    out, lse = tree_attention(q_dev, kp, vp, table, seq, **call)
    check(out, lse, q, ks, vs, nodes, 1 / math.sqrt(D), dtype, parents, mask)
    for i, m in enumerate(nodes):
        assert (out[i, :, m:] == 0).all() and torch.isneginf(lse[i, :, m:]).all()
    for _ in range(20):  # the same whatever the timing
        again, lse_again = tree_attention(q_dev, kp, vp, table, seq, **call)
        assert torch.equal(again, out) and torch.equal(lse_again, lse)


@pytest.mark.parametrize("D", [64, 128])
def test_zeros_into_an_output_off_16_bytes(D):
    """Rows without a node of an output that is written element by element; what lies between stays."""
    lens = [300, 200, 140]
    kp, vp, table, seq, ks, vs = build(lens, 2, 16, D, BF)
    q = torch.randn(3, 4, 3, D).to(BF)
    hold = torch.full((3 * 4 * 3 * (D + 3) + 1,), 7.0, dtype=BF, device="cuda")
    out = hold[1:].view(3, 4, 3, D + 3)[..., :D]
    nodes = torch.tensor([0, 3, 0], device="cuda")
    _, lse = tree_attention(q.cuda(), kp, vp, table, seq, num_nodes=nodes, out=out, return_lse=True)
    check(out, lse, q, ks, vs, [0, 3, 0], 1 / math.sqrt(D), BF)
    assert (out[::2] == 0).all() and (hold[1:].view(3, 4, 3, D + 3)[..., D:] == 7.0).all() and float(hold[0]) == 7.0


@pytest.mark.parametrize("D,S,T,Hq,dtype", [(64, 16, 1, 8, HF), (128, 16, 1, 8, BF), (128, 16, 7, 24, BF), (64, 64, 3, 40, HF)])
@pytest.mark.parametrize("table_tokens", [0, 2048])
def test_infinite_values_of_nodes_in_many_short_rows(D, S, T, Hq, dtype, table_tokens):
    """Many units after one another in a CTA, every other one with infinite values at its nodes: each row gets its
    own nodes' infinities, in every run."""
    n, H = 400, 8
    lens = [T + 3 * i % 120 for i in range(n)]
    kp, vp, table, seq, _, _ = build(lens, H, S, D, dtype)
    if table_tokens:
        table = torch.nn.functional.pad(table, (0, table_tokens // S - table.shape[1]), value=-1)
    q = torch.randn(n, Hq, T, D).to(dtype).cuda()
    odd = torch.arange(1, n, 2)
    for i in odd.tolist():
        x = lens[i] - T  # node 0: every node sees it
        vp[int(table[i, x // S]), :, x % S, 5::16] = math.inf
        vp[int(table[i, x // S]), :, x % S, 9::16] = -math.inf
    first = tree_attention(q, kp, vp, table, seq)
    for i, got in ((odd, first[odd.cuda()]), (odd - 1, first[odd.cuda() - 1])):
        hit = bool(i[0] % 2)
        assert ((got[..., 5::16] == math.inf) == hit).all() and ((got[..., 9::16] == -math.inf) == hit).all()
        assert torch.isfinite(got[..., 0::16]).all()
    for _ in range(20):
        assert torch.equal(tree_attention(q, kp, vp, table, seq), first)
