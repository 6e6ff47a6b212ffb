"""GPU test of routing calls from two threads at once, a handle and a stream each."""
import threading

import pytest
import torch

import gemm_sm100 as gs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens,top_k", [(100, 4), (8, 4)])
def test_two_threads_with_different_expert_counts(cuda, tokens, top_k):
    """The plan's shared memory grows with the experts (past the size that needs an opt-in, which is one setting of the
    kernel's for all threads): neither thread's calls may depend on the other's."""
    def buffers(experts):
        rows, ws = gs.moe_rows(tokens, experts, top_k), gs.moe_route_workspace(tokens, experts, top_k)
        i32 = dict(dtype=torch.int32, device="cuda")
        logits = torch.randn(tokens, experts, generator=torch.Generator().manual_seed(experts)).cuda()
        return logits, torch.empty(tokens, top_k, **i32), dict(
            weights=torch.empty(tokens, top_k, device="cuda"), offsets=torch.empty(experts + 1, **i32),
            slot_row=torch.empty(tokens, top_k, **i32), row_slot=torch.empty(rows, **i32), rows=rows,
            workspace=torch.empty(max(ws, 4), dtype=torch.uint8, device="cuda"), workspace_bytes=ws)

    sizes = (1024, 520)
    sets, failures = [buffers(e) for e in sizes], []
    torch.cuda.synchronize()
    start = threading.Barrier(2)

    def work(experts, logits, ids, kw):
        try:
            stream = torch.cuda.Stream()
            with gs.Handle(stream) as h:
                start.wait()
                for i in range(4000):
                    h.moe_route(tokens, experts, top_k, logits, gs.R_32F, experts, ids, **kw)
                    if i % 500 == 499:
                        stream.synchronize()
                stream.synchronize()
        except Exception as e:  # noqa: BLE001
            failures.append(e)

    threads = [threading.Thread(target=work, args=(e, *s)) for e, s in zip(sizes, sets)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures, failures
    for logits, ids, kw in sets:
        assert torch.equal(ids.long(), logits.topk(top_k).indices)
        assert int(kw["offsets"][-1]) == tokens * top_k
