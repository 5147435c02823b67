"""Caches used by several host threads at once, each on its own stream."""

import threading

import pytest
import torch

from test_gpu_paged_cache import dev, make

pytestmark = pytest.mark.gpu

from cab_attention import _lib  # noqa: E402


@pytest.fixture(autouse=True)
def _device_status_clean():
    yield
    assert _lib.device_status() == 0


def together(*jobs):
    errors, start = [], threading.Barrier(len(jobs))

    def run(job):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                start.wait()
                job()
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    torch.cuda.synchronize()
    threads = [threading.Thread(target=run, args=(j,)) for j in jobs]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not errors, errors


def test_updates_of_different_sizes():
    """A call of 1024 rows needs more shared memory than one of 750, both more than a launch gets unasked."""
    def job(rows):
        c, _ = make(L=1, P=5000, H=1, S=4, D=8, R=1024, W=6, seed=rows)
        at = dev(list(range(rows)))

        def run():
            for _ in range(1500):
                c.extend(1, at)
                c.truncate(0, at)
        return run, c

    jobs = [job(n) for n in (1024, 750, 1024, 750)]
    together(*(run for run, _ in jobs))
    for _, c in jobs:
        c.check()
        assert c.free_pages() == 5000


def test_attention_with_different_head_dims():
    """One kernel on CUDA cores takes head_dim 129 to 256, with shared memory by the dimension."""
    def job(D):
        c, _ = make(L=1, P=8, H=1, S=16, D=D, R=1, W=8, dtype=torch.float32)
        c.extend(100)
        q = torch.randn(1, 1, 40, D, device="cuda")
        want = c.attend(0, q)
        outs = []

        def run():
            outs.extend(c.attend(0, q) for _ in range(1500))
        return run, outs, want

    jobs = [job(D) for D in (256, 136, 248, 144)]
    together(*(run for run, _, _ in jobs))
    for _, outs, want in jobs:
        assert all(torch.equal(o, want) for o in outs)
