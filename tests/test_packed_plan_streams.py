"""A plan's positions on other streams than the one they were made on, and in a graph's capture."""
import pytest
import torch

import cudatransformer_amd as ct

LENS = [3000, 0, 1, 4999]
WANT = torch.cat([torch.arange(n) for n in LENS])


def test_on_the_host():
    plan = ct.packed_plan(LENS, 2, 2, device="cpu")
    p = plan.positions()
    assert torch.equal(p, WANT) and plan.positions("cpu") is p
    empty = ct.packed_plan([], 2, 2, device="cpu").positions()
    assert empty.shape == (0,) and empty.dtype == torch.int64


@pytest.mark.gpu
def test_memory_is_kept_while_another_stream_reads_it():
    plan = ct.packed_plan(LENS, 2, 2)
    at = plan.positions().data_ptr()  # made on the current stream
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)  # what comes next on this stream waits for about 0.1 s
        out = plan.positions() + 1
        done = side.record_event()
    del plan
    others = [torch.full((sum(LENS),), -7, device="cuda") for _ in range(4)]  # of the same size, on the first stream
    assert not done.query()  # the side stream has not read the positions yet
    assert all(t.data_ptr() != at for t in others)
    side.synchronize()
    assert torch.equal(out.cpu(), WANT + 1)


@pytest.mark.gpu
def test_in_a_capture():
    plan, late = ct.packed_plan(LENS, 2, 2), ct.packed_plan(LENS, 2, 2)
    p = plan.positions("cuda")
    assert plan.positions() is p and plan.positions(torch.device("cuda", torch.cuda.current_device())) is p
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = plan.positions() * 2
        with pytest.raises(RuntimeError, match="capture"):
            late.positions()
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out.cpu(), WANT * 2)
