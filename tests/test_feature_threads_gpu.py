"""The feature operators from several host threads at once (their calls hold no
lock): every call succeeds and gives what it gives alone."""

import threading

import pytest
import torch

import dot
from tests import util as U

pytestmark = pytest.mark.gpu
DEV = "cuda"


def together(jobs, repeats):
    """Runs every job(its own stream) `repeats` times in a thread of its own; returns what was raised."""
    raised, start = [], threading.Barrier(len(jobs))

    def loop(job):
        stream = torch.cuda.Stream()
        start.wait()
        with torch.cuda.stream(stream):
            for _ in range(repeats):
                try:
                    job()
                except Exception as e:   # noqa: BLE001
                    raised.append(repr(e))
        stream.synchronize()

    threads = [threading.Thread(target=loop, args=(job,)) for job in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    return raised


def test_norms_with_other_numbers_of_groups():
    """One kernel with four sizes of shared memory, its opt-in set by all threads."""
    jobs, results = [], []
    for G, C, S in ((8, 64, 30000), (512, 4096, 900), (16, 128, 20000), (256, 2048, 1500)):
        x = torch.randn(1, S, C, generator=U.gen(G)).to(DEV).half()
        want, got = dot.group_norm_act(x, G), []
        results.append((want, got))
        jobs.append(lambda x=x, G=G, got=got: (got.clear(), got.append(dot.group_norm_act(x, G))))
    torch.cuda.synchronize()
    assert together(jobs, 1000) == []
    for want, got in results:
        assert torch.equal(got[0], want)


def test_training_calls():
    jobs, results = [], []
    freqs = dot.rotary_freqs((8, 8), device=DEV)
    for G, C, S in ((8, 64, 3000), (2900, 2900, 40), (32, 256, 900)):
        x = torch.randn(2, S, C, generator=U.gen(G)).to(DEV).requires_grad_(True)
        pos = torch.randint(0, 90, (S, 2), generator=U.gen(S)).to(DEV)

        def step(x=x, G=G, pos=pos):
            y = dot.group_norm_act(x, G)
            q = dot.rotary(y[..., :64].unflatten(-1, (2, 32)), pos, freqs)
            return y.detach(), q.detach(), torch.autograd.grad(q, x, torch.ones_like(q))[0]

        want, got = step(), []
        results.append((want, got))
        jobs.append(lambda step=step, got=got: (got.clear(), got.append(step())))
    torch.cuda.synchronize()
    assert together(jobs, 100) == []
    for want, got in results:
        assert all(torch.equal(a, b) for a, b in zip(got[0], want))
