"""Orders of different numbers of experts from several threads at once: their kernel needs more shared memory than a launch may have by itself from some 341 experts on."""
import threading

import pytest
import torch

from ccfuser_b200.ops.expert_sort import expert_order

pytestmark = pytest.mark.gpu


def test_calls_of_different_numbers_of_experts_from_several_threads():
    g = torch.Generator().manual_seed(1)
    experts = (1024, 400, 700, 1024)
    sets = [torch.randint(0, e, (22000, 2), generator=g).cuda() for e in experts]      # slots times experts above 2^24: blocks of 1024 threads
    sets[2] = sets[2][:6000]                                                           # below
    want = [expert_order(i.cpu(), e) for i, e in zip(sets, experts)]
    failed, start = [], threading.Barrier(len(experts))

    def work(k):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                start.wait(60)
                for _ in range(1500):
                    order = expert_order(sets[k], experts[k])
                torch.cuda.current_stream().synchronize()
                for a, b in zip(order, want[k]):
                    assert torch.equal(a.cpu(), b)
        except BaseException as e:
            failed.append(e)
            raise

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(k,)) for k in range(len(experts))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
