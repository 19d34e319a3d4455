"""What the token policy network reads from feature planes, on the CPU."""
import pytest
import torch

from omoknuni_quantum_amd.synthetic import token_policy


@pytest.mark.parametrize("board", [3, 15, 19])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16, torch.float64,
                                   torch.int8, torch.int32, torch.bool])
def test_tokens_of_planes_of_any_type(board, dtype):
    g = torch.Generator().manual_seed(board)
    content = torch.randint(0, 3, (4, board * board), generator=g)
    planes = torch.zeros(4, 18, board * board, dtype=dtype)
    planes[:, 0], planes[:, 1] = (content == 1).to(dtype), (content == 2).to(dtype)
    net = token_policy.TokenPolicy(board_size=board, dim=8, blocks=1, device="cpu")
    got = net.tokens(planes.view(4, 18, board, board))
    assert got.dtype == torch.int32
    assert torch.equal(got.long(), 3 * torch.arange(board * board) + content)
