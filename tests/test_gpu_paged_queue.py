"""Calls of the paged cache queued one behind the other without a wait between them, so that each kernel is
launched while those before it run: the results are those of the same calls with a wait after each."""

import pytest
import torch

from test_gpu_paged_cache import dev, make

pytestmark = pytest.mark.gpu

from cab_attention import _lib  # noqa: E402


@pytest.fixture(autouse=True)
def _device_status_clean():
    yield
    assert _lib.device_status() == 0


@pytest.mark.parametrize("S,D,lens", [(16, 64, [3, 1200, 0, 717]), (16, 128, [900, 5, 2300, 60])])
def test_attention_directly_after_a_change_of_lengths(S, D, lens):
    """extend -> attend, truncate -> attend and free -> attend with nothing between: rows are cut between
    CTAs, so which partial sums are joined follows from lengths that the call before writes."""
    g = torch.Generator(device="cuda").manual_seed(4)
    q = torch.randn(4, 8, 4, D, device="cuda", generator=g).to(torch.bfloat16)

    def steps(wait):
        c, _ = make(L=1, P=700, S=S, D=D, R=4, W=200, seed=1)
        pause = torch.cuda.synchronize if wait else (lambda: None)
        c.extend(dev(lens))
        pause()
        outs = []
        for i in range(30):
            c.extend(dev([4, 31 + i, 7 * i % 60, 4]))
            pause()
            outs += c.attend(0, q, return_lse=True)
            pause()
            c.truncate(dev([lens[j] + i for j in range(4)]))
            pause()
            outs += c.attend(0, q, num_nodes=dev([4, 0, min(4, lens[2] + i), 1]), return_lse=True)
            pause()
            if i % 10 == 9:
                c.free(dev([2]))
                pause()
                outs += c.attend(0, q, num_nodes=dev([4, 1, 0, 4]), return_lse=True)
                pause()
                c.extend(dev([lens[2] + i]), dev([2]))
                pause()
        c.check()
        return outs + [c.block_table, c.seq_lens, c.ref_counts]

    want = steps(True)
    for _ in range(5):
        for x, y in zip(steps(False), want):
            assert torch.equal(x, y)


def test_check_waits_for_calls_on_other_streams():
    c, _ = make(P=20, R=3, W=6)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)  # about a tenth of a second
        c.extend(20, dev([0]))
    assert c.free_pages() == 18
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)
        c.extend(1, dev([7]))
    with pytest.raises(RuntimeError, match="outside the table"):
        c.check()
    c.check()


@pytest.mark.parametrize("R,T", [(24, 3), (300, 5)])
def test_captured_steps_with_idle_rows(R, T):
    """extend, write, attend and truncate in one graph, replayed with other idle rows each time; 300 rows of 5 tokens
    have more table entries than the write checks by itself."""
    S, D, H = 4, 64, 2
    c, _ = make(L=1, P=R * 80, H=H, S=S, D=D, R=R, W=80, seed=3)
    lens = [130 + 7 * i % 150 for i in range(R)]
    c.extend(dev(lens))
    first = torch.randn(R, H, 280, D, device="cuda").to(torch.bfloat16)
    c.write(0, first, first, dev(lens))
    c.check()
    k, q = (torch.randn(R, x, T, D, device="cuda").to(torch.bfloat16) for x in (H, 2 * H))
    num, start = dev([T] * R), c.seq_lens.clone()

    def step():
        c.extend(num)
        c.write(0, k, k, num)
        out = c.attend(0, q, num_nodes=num, return_lse=True)
        c.truncate(start)
        return out

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for x in range(12):
        num.copy_(dev([(T - i % 2 if (i + x) % 3 else 0) if x % 4 else T * ((i // 8 + x) % 2) for i in range(R)]))
        want = [t.clone() for t in step()]
        state = [t.clone() for t in (c.block_table, c.seq_lens, c.ref_counts)]
        for _ in range(3):
            graph.replay()
            assert all(torch.equal(a, b) for a, b in zip(held, want))
            assert all(torch.equal(a, b) for a, b in zip((c.block_table, c.seq_lens, c.ref_counts), state))
    c.check()
