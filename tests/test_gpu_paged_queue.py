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
