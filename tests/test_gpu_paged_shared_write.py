"""Writes that reach back into pages shared by rows: the last sequence's values stay, in every run."""

import pytest
import torch

from test_gpu_paged_cache import dev, make, oracle_of, same

pytestmark = pytest.mark.gpu

from cab_attention import _lib  # noqa: E402


@pytest.fixture(autouse=True)
def _device_status_clean():
    yield
    assert _lib.device_status() == 0


@pytest.mark.parametrize("S,R", [(1, 6), (4, 150), (16, 60)])
@pytest.mark.parametrize("listed", [False, True])
def test_last_sequence_counts(S, R, listed):
    H, D, T, held = 4, 64, 10, 64
    c, _ = make(L=1, P=held // S + 5 * R, H=H, S=S, D=D, R=R, W=held // S + 5)
    c.extend(held, dev([2]))
    others = [r for r in range(R) if r != 2]
    c.fork(dev([2] * len(others)), dev(others))
    c.extend(dev([i % 4 for i in range(R)]))
    c.check()
    o = oracle_of(c)
    g = torch.Generator().manual_seed(S)
    rows = torch.randperm(R, generator=g).tolist() if listed else list(range(R))
    num = [T - 3 * i % 11 if i % 5 else 0 for i in range(R)]
    for _ in range(10):
        k, v = (torch.randn(R, T, H, D, generator=g).to(torch.bfloat16).cuda().transpose(1, 2) for _ in range(2))
        c.write(0, k, v, dev(num), dev(rows) if listed else None)
        o.write(0, k.float().cpu().numpy(), v.float().cpu().numpy(), rows, num)
        same(c, o)
    c.check()
