"""The rotation's table of the token policy network, which all streams and graphs share."""
import pytest
import torch

from omoknuni_quantum_amd.synthetic.token_policy import RotaryTable

pytestmark = pytest.mark.gpu


def expected():
    cell = torch.arange(81)
    return torch.stack((cell // 9, cell % 9), 1).int(), 100.0 ** (-torch.arange(8).double() / 8)


def test_other_streams_find_it_whole(device):
    """It is there when `of` returns, however long the stream that asked first is busy."""
    tokens = torch.zeros(1, 81, dtype=torch.int32, device=device)
    places, freq = expected()
    first, other = torch.cuda.Stream(), torch.cuda.Stream()
    table = RotaryTable(9, 32)
    with torch.cuda.stream(first):
        torch.cuda._sleep(20_000_000)
        positions, frequencies, sections = table.of(tokens, False)
    with torch.cuda.stream(other):
        got = positions.clone(), frequencies.clone()
    other.synchronize()
    assert sections == (8, 8)
    assert torch.equal(got[0].cpu(), places)
    assert torch.allclose(got[1].cpu(), freq.repeat(2), rtol=1e-15)
    torch.cuda.synchronize()


def test_a_capture_does_not_make_it(device):
    """A graph's memory is not filled before a replay, and what it holds is not for others."""
    tokens = torch.zeros(1, 81, dtype=torch.int32, device=device)
    x = torch.zeros(4, device=device)
    table = RotaryTable(9, 32)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x.add_(1.0)
        with pytest.raises(RuntimeError, match="captured"):
            table.of(tokens, False)
    assert not table.held
    assert torch.equal(table.of(tokens, False)[0].cpu(), expected()[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = table.of(tokens, False)[0] + 1
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(held.cpu(), expected()[0] + 1)
