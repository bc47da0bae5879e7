"""Group norm called by several host threads at once (run with -m gpu).

Calls of one kernel that need different amounts of shared memory above 48 KB: 1,000
channels in 500 groups, in 8 groups, and 900 in 6 share an instantiation. No call may fail,
and each result must be the bits that a call on its own gives.
"""
import threading

import pytest
import torch

from gnn_cuda_b200.GNN_cuda_common import norm_ops as M

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


@pytest.mark.parametrize("graphs", [True, False])
def test_threads_of_different_sizes(graphs):
    n = 300
    ptr = torch.tensor([0, 70, 300], dtype=torch.int32, device=DEV) if graphs else None
    jobs = []
    for c, groups in ((1000, 500), (1000, 8), (900, 6)):
        x = torch.randn(n, c, device=DEV)
        want = torch.empty_like(x)
        M.group_norm_forward_(x, groups, None, None, want, graph_ptr=ptr)
        jobs.append((x, groups, want, torch.empty_like(x), torch.cuda.Stream()))
    torch.cuda.synchronize()
    errors = []
    start = threading.Barrier(len(jobs))

    def work(x, groups, want, out, stream):
        try:
            with torch.cuda.stream(stream):
                start.wait()
                for _ in range(3000):
                    M.group_norm_forward_(x, groups, None, None, out, graph_ptr=ptr)
                stream.synchronize()
            if not torch.equal(out, want):
                errors.append("results differ")
        except Exception as e:  # noqa: BLE001 - reported by the main thread
            errors.append(repr(e))

    threads = [threading.Thread(target=work, args=j) for j in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert errors == []
