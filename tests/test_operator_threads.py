"""Calls of one operator from two threads at once, each of its own size: a kernel's
limits are not those of the other thread's call."""

import threading

import pytest
import torch

from test_distill import make
from test_paged4 import filled, heads, ints


def together(jobs, turns, device):
    """Runs each job's call ``turns`` times in a thread and a stream of its own, all at
    once; returns their last results."""
    start, errors, results = threading.Barrier(len(jobs)), [], [None] * len(jobs)

    def work(i, call):
        try:
            with torch.cuda.stream(torch.cuda.Stream(device)):
                start.wait()
                for _ in range(turns):
                    results[i] = call()
                torch.cuda.current_stream(device).synchronize()
        except Exception as e:  # noqa: BLE001 (reported by the test)
            errors.append(e)

    torch.cuda.synchronize(device)
    threads = [threading.Thread(target=work, args=x) for x in enumerate(jobs)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    return results


def same(results, wants):
    for got, want in zip(results, wants):
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
def test_distillation_of_two_vocabularies(cuda_device):
    from autoindexer_b200 import distill_loss_and_grad

    jobs = []
    for V in (300, 780001):  # (slices of 1.2 and 195 KB)
        args = [y.to(cuda_device) for y in make((1,), V, 4, torch.float32, V)]
        jobs.append(lambda args=args: distill_loss_and_grad(*args))
    wants = [job() for job in jobs]
    same(together(jobs, 6000, cuda_device), wants)


@pytest.mark.gpu
def test_attention_of_two_batches(cuda_device):
    from autoindexer_b200 import paged_attention_4bit

    jobs = []
    for B in (1, 700):
        lens = [20 + i % 3 for i in range(B)]
        cache, table = filled(B, 1, 32, 16, lens, torch.float32, 5, cuda_device)
        q = heads(B, 4, 1, 32, torch.bfloat16, 6, cuda_device)
        jobs.append(lambda args=(q, *cache, table, ints(lens, cuda_device)): [paged_attention_4bit(*args)])
    wants = [job() for job in jobs]
    same(together(jobs, 3000, cuda_device), wants)


@pytest.mark.gpu
@pytest.mark.parametrize("prefix_len", [0, 3000])
def test_shared_prefix_attention_of_two_batches(prefix_len, cuda_device):
    from autoindexer_b200 import shared_prefix_attention

    H, S, D = 2, 16, 64
    pages = [heads(200, H, S, D, torch.bfloat16, s, cuda_device).contiguous() for s in (1, 2)]
    prefix = torch.arange(-(-prefix_len // S), dtype=torch.int32, device=cuda_device) if prefix_len else None
    jobs = []
    for B in (1, 700):
        table = torch.randint(0, 200, (B, 2), dtype=torch.int32, device=cuda_device)
        lens = ints([20 + i % 3 for i in range(B)], cuda_device)
        q = heads(B, 4, 1, D, torch.bfloat16, 6, cuda_device)
        jobs.append(lambda args=(q, *pages, prefix, prefix_len, table, lens): [shared_prefix_attention(*args)])
    wants = [job() for job in jobs]
    same(together(jobs, 3000, cuda_device), wants)
