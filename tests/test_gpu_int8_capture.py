"""Chunks over an int8 cache whose first call of a length is a graph capture."""
import pytest
import torch

from tests.test_gpu_int8_engine import _engine, _rows, pa  # noqa: F401  (pa: fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rope", [False, True])
def test_an_eager_chunk_behind_a_capture_that_was_never_replayed(pa, rope):  # noqa: F811
    """What a layer keeps from call to call may not be left to the kernels of a graph: the capture is the first call of its
    length, the eager step behind it comes before any replay."""
    D, bs, Hq, Hkv, T = 64, 16, 8, 2, 100
    g = torch.Generator(device="cuda").manual_seed(7)
    (cache, layer), (c2, l2) = (_engine(D, bs, Hq, Hkv, 3, rope=rope) for _ in range(2))
    x = _rows(g, 3, T, Hq, Hkv, D)
    lens = [100, 0, 31]
    cache.begin_step(lens, T)
    c2.begin_step(lens, T)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        replayed = layer.attend(*x, max_seq_len=400)
    want = l2.attend(*(t.clone() for t in x), max_seq_len=400).clone()
    assert torch.equal(layer.attend(*x, max_seq_len=400), want)
    for lens in ([100, 0, 31], [5, 64, 100], [0, 100, 0]):
        if lens != [100, 0, 31]:
            cache.begin_step(lens, T)
            c2.begin_step(lens, T)
        replayed.zero_()
        graph.replay()
        want = l2.attend(*(t.clone() for t in x), max_seq_len=400)
        torch.cuda.synchronize()
        assert torch.equal(replayed, want)


def test_two_captures_of_one_length_replayed_out_of_order(pa):  # noqa: F811
    D, bs, Hq, Hkv, T = 128, 16, 4, 2, 70
    g = torch.Generator(device="cuda").manual_seed(8)
    (cache, layer), (c2, l2) = (_engine(D, bs, Hq, Hkv, 2) for _ in range(2))
    lens = [70, 33]
    cache.begin_step(lens, T)
    c2.begin_step(lens, T)
    xs = [_rows(g, 2, T, Hq, Hkv, D) for _ in range(2)]
    graphs = []
    for x in xs:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            out = layer.attend(*x, max_seq_len=300)
    for i in (1, 0, 1):
        out.zero_()
        graphs[i].replay()
        want = l2.attend(*(t.clone() for t in xs[i]), max_seq_len=300)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
