"""The token policy network serves the weights that it has, whatever changed them, and leaves its
mode alone."""
import copy

import pytest
import torch

from omoknuni_quantum_amd.synthetic import token_policy
from tests.test_gpu_token_policy import tokens_of

pytestmark = pytest.mark.gpu


def network(device, seed=0):
    return token_policy.TokenPolicy(board_size=7, dim=32, blocks=2, seed=seed, device=device)


def of_fresh(net, tokens):
    """What a network that has served nothing yet gives with the same weights."""
    fresh = network(tokens.device, 9)
    fresh.load_state_dict(copy.deepcopy(net.state_dict()))
    return fresh.eval().serve(tokens)


def planes(positions, device, dtype=torch.float32):
    g = torch.Generator().manual_seed(positions)
    cell = torch.randint(0, 3, (positions, 7, 7), generator=g)
    f = torch.zeros(positions, 18, 7, 7)
    f[:, 0], f[:, 1] = cell == 1, cell == 2
    return f.to(device, dtype)


def _step(net):
    tokens = tokens_of(net, 3, 5, net.table.device)
    optimizer = torch.optim.AdamW(net.parameters(), lr=0.01)  # (steps of bounded size)
    logits, values = net(tokens)
    (logits.square().sum() + values.sum()).backward()
    optimizer.step()


def _copies(net):
    with torch.no_grad():
        for p in net.parameters():
            p.add_(0.1 * torch.randn_like(p))


def _data(net):
    for p in net.parameters():
        p.data.mul_(1.5)


def _of_a_parent(net):
    torch.nn.ModuleDict({"net": net}).load_state_dict(
        {"net." + k: v for k, v in network(net.table.device, 3).state_dict().items()})


def _of_a_block(net):
    net.blocks[1].load_state_dict(network(net.table.device, 4).blocks[1].state_dict())


@pytest.mark.parametrize("change", [_step, _copies, _data, _of_a_parent, _of_a_block])
@pytest.mark.parametrize("training", [False, True])
def test_serves_the_weights_that_it_has(device, change, training):
    net, f = network(device).train(training), planes(6, device)
    tokens = net.tokens(f)
    before, searched = net.serve(tokens), net.evaluate_batch(f)
    change(net)
    assert net.training == training
    after, want = net.serve(tokens), of_fresh(net, tokens)
    assert not torch.equal(before[0], after[0])
    assert all(torch.equal(a, b) for a, b in zip(after, want))
    again = net.evaluate_batch(f)
    assert not torch.equal(again[0], searched[0])
    assert torch.equal(again[1], want[1]) and net.training == training


def test_a_loop_that_searches_and_trains(device):
    """train() once, then searches and steps in turn: dropout stays on, and each search has the
    weights of its step."""
    net, f = network(device).train(), planes(4, device)
    tokens = net.tokens(f)
    for _ in range(3):
        net.evaluate_batch(f)
        assert net.training
        still = net(tokens)[0]
        net.steps += 1  # (another mask)
        assert not torch.equal(net(tokens)[0], still)
        _step(net)
        assert all(torch.equal(a, b) for a, b in zip(net.serve(tokens), of_fresh(net, tokens)))


def test_an_evaluator_keeps_its_weights(device):
    net, f = network(device), planes(5, device)
    evaluator = net.evaluator()
    first = evaluator.evaluate_batch(f)
    for change in (_step, _copies, _data):
        change(net)
        assert all(torch.equal(a, b) for a, b in zip(evaluator.evaluate_batch(f), first))
    assert not torch.equal(net.evaluate_batch(f)[0], first[0])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_policies_of_full_boards_are_zero(device, dtype):
    """A row that the mask leaves nothing of has no policy, and the others theirs."""
    f = planes(5, device, dtype)
    f[1, 0], f[1, 1] = 1, 0
    f[3, 0] = 1 - f[3, 1]
    policies, values = network(device).evaluate_batch(f)
    occupied = ((f[:, 0] + f[:, 1]) > 0).flatten(1)
    full = torch.tensor([False, True, False, True, False], device=device)
    assert torch.equal(occupied.all(1), full)
    assert not bool(policies[occupied].any())
    # 49 float32 terms
    assert float((policies.double().sum(1) - (~full).double()).abs().max()) < 60 * 2.0**-24
    assert bool(values.isfinite().all())
