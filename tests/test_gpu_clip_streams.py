"""GPU: a gradient set's table is not handed to another tensor while a stream still has to read it."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_table_outlives_calls_on_other_streams():
    """A clipper made on one stream, used on another that is busy, and dropped: until the call has run, its table's memory serves no
    other tensor."""
    from trebi_amd.clip import GradClipper
    g = torch.Generator('cuda').manual_seed(0)
    grads = [torch.randn(5, device='cuda', generator=g) for _ in range(3000)]      # a table of a size of its own
    want = torch.cat(grads).double().norm()
    GradClipper(grads).clip_into(1.0)                       # everything is loaded, the pools are warm
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    clipper = GradClipper(grads)
    size, at = clipper.table.numel(), clipper.table.data_ptr()
    done = torch.cuda.Event()
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)                      # a tenth of a second
        flat, norm = clipper.clip_into(1.0)
        done.record()
    del clipper
    others = [torch.empty(size, dtype=torch.uint8, device='cuda') for _ in range(4)]
    assert not done.query()
    assert all(v.data_ptr() + size <= at or at + size <= v.data_ptr() for v in others)
    torch.cuda.synchronize()
    assert abs(float(norm) - float(want)) <= 2.0 ** -23 * float(want)
    again = [torch.empty(size, dtype=torch.uint8, device='cuda') for _ in range(8)]
    assert len({v.data_ptr() for v in others + again}) == 12


def test_calls_on_another_stream_can_be_captured():
    from trebi_amd.clip import GradClipper
    g = torch.Generator('cuda').manual_seed(0)
    grads = [torch.randn(n, device='cuda', generator=g) for n in (7, 4097, 100)]
    clipper = GradClipper(grads)
    clipper.clip_into(1.0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        flat, norm = clipper.clip_into(1.0)
    for k in range(4):
        for v in grads:
            v.normal_(generator=g)
        want, n = clipper.clip_into(1.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(flat, want) and torch.equal(norm, n), k
