"""Calls of one kernel that need different amounts of shared memory, from several host threads: none takes from another what it was allowed."""
import threading

import pytest
import torch

import mlx_b200 as mb

pytestmark = pytest.mark.gpu


def in_a_thread(f):
    failed = []

    def work():
        try:
            f()
        except Exception as e:   # noqa: BLE001 (shown by the caller)
            failed.append(e)

    t = threading.Thread(target=work)
    t.start()
    t.join()
    assert not failed, failed


def routing(T):
    g = torch.Generator("cuda").manual_seed(T)
    logits, bias = torch.randn((T, 256), generator=g, device="cuda"), torch.randn(256, generator=g, device="cuda") * 0.1
    return lambda: mb.route_experts(logits, 8, "sigmoid", bias, groups=8, top_groups=4, group_best=2)


def grouping(T, n):
    ids = torch.randint(-1, n, (T,), generator=torch.Generator().manual_seed(T)).cuda()
    return lambda: mb.group_rows(ids, n)


# (more, less) of the same kernels: route_kernel; group_kernel and place_kernel; group_few_kernel
PAIRS = {"route": lambda: (routing(8192), routing(2048)), "group": lambda: (grouping(5000, 4096), grouping(5000, 2048)),
         "group few": lambda: (grouping(900, 4096), grouping(900, 600))}


@pytest.mark.parametrize("what", tuple(PAIRS))
def test_a_smaller_call_between_larger_ones(what):
    large, small = PAIRS[what]()
    ref = large()
    in_a_thread(small)
    assert all(torch.equal(p, q) for p, q in zip(large(), ref))
    in_a_thread(large)


def test_threads_that_call_at_the_same_time():
    pairs = [f() for f in PAIRS.values()]
    refs = [[f() for f in pair] for pair in pairs]
    bad = []

    def work(k):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for i in range(30):
                    for pair, ref in zip(pairs, refs):
                        got = pair[(i + k) % 2]()
                        if not all(torch.equal(p, q) for p, q in zip(got, ref[(i + k) % 2])):
                            bad.append("differs")
        except Exception as e:   # noqa: BLE001
            bad.append(e)

    torch.cuda.synchronize()
    ts = [threading.Thread(target=work, args=(k,)) for k in range(4)]
    [t.start() for t in ts]
    [t.join() for t in ts]
    assert not bad, bad
