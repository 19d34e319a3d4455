"""The token policy network: the operators of net_ops together, as an evaluator of searches and in
training on what the searches return."""
import pytest
import torch

from omoknuni_quantum_amd.synthetic import token_policy

pytestmark = pytest.mark.gpu


def plain_forward(net, tokens):
    """The network in plain torch, float64, without dropout."""
    table = net.table.detach().double()
    h = table[tokens.long()] * net.dim**0.5

    def norm(h, w):
        return h * torch.rsqrt(h.square().mean(-1, keepdim=True) + 1e-6) * w.detach().double()

    for b in net.blocks:
        y = norm(h, b.norm_cells).transpose(1, 2) @ b.cells.weight.detach().double().t()
        h = h + y.transpose(1, 2)
        y = norm(h, b.norm_channels) @ b.up.weight.detach().double().t()
        h = h + torch.nn.functional.gelu(y) @ b.down.weight.detach().double().t()
    y = norm(h, net.norm_out)
    logits = y @ net.policy.weight.detach().double().t() + net.policy.bias.detach().double()
    v = y.mean(1) @ net.value.weight.detach().double().t() + net.value.bias.detach().double()
    return logits[..., 0], torch.tanh(v)[:, 0]


def tokens_of(net, positions, seed, device):
    g = torch.Generator().manual_seed(seed)
    cells = net.board**2
    return (3 * torch.arange(cells) + torch.randint(0, 3, (positions, cells), generator=g)).to(
        device, torch.int32)


def test_forward_and_serving(device):
    net = token_policy.TokenPolicy(board_size=9, dim=64, blocks=2, device=device).eval()
    t = tokens_of(net, 5, 3, device)
    want = [x.cpu() for x in plain_forward(net.double().cpu(), t.cpu())]
    net = net.float().to(device)
    got = [x.detach().cpu().double() for x in net(t)]
    # float32 products of 64 and 128 terms on values of order 1
    assert float((got[0] - want[0]).abs().max()) < 1e-4
    assert float((got[1] - want[1]).abs().max()) < 1e-4
    served = [x.cpu().double() for x in net.serve(t)]
    # bfloat16 layers and one product in 4 significant bits a block: a few percent of the spread
    spread = float(want[0].std())
    assert float((served[0] - want[0]).pow(2).mean().sqrt()) < 0.1 * spread
    assert float((served[1] - want[1]).abs().max()) < 0.1


def test_gradients_of_the_network(device):
    """Every parameter's gradient in training mode against the difference of the loss along it."""
    net = token_policy.TokenPolicy(board_size=7, dim=32, blocks=1, dropout=0.2, device=device)
    t = tokens_of(net, 6, 4, device)
    g = torch.Generator(device=device).manual_seed(5)
    up = torch.randn(6, 49, generator=g, device=device)
    net.train()

    def value():
        logits, v = net(t)
        return (logits.double() * up).sum() + v.double().sum()

    value().backward()
    for name, p in net.named_parameters():
        v = torch.randn(p.shape, generator=g, device=device)
        v = v / v.norm() * p.detach().norm().clamp(min=0.1)
        step = 1e-2
        with torch.no_grad():
            keep = p.clone()
            p.copy_(keep + step * v)
            high = value()
            p.copy_(keep - step * v)
            low = value()
            p.copy_(keep)
        slope = float((high - low) / (2 * step))
        # float32 values of order 100 differenced over 2e-2, and the step's third order
        assert slope == pytest.approx(float((p.grad * v).sum()), rel=3e-2, abs=3e-2), name


def test_search_then_train(device):
    net = token_policy.TokenPolicy(board_size=9, dim=64, blocks=2, device=device)
    tokens, target, legal, actions, old = token_policy.searched_positions(net, 8, 64, 20, 3)
    assert bool((target[~legal] == 0).all())
    assert float((target.sum(1) - 1).abs().max()) < 1e-5
    assert bool(legal.gather(1, actions[:, None]).all())
    optimizer = torch.optim.AdamW(net.parameters(), lr=2e-3)
    outcome = torch.ones(8, device=device)
    said = [net.train_step(optimizer, tokens, target, legal, actions, torch.zeros(8, device=device),
                           old, outcome) for _ in range(15)]
    assert said[-1]["kl"] < 0.8 * said[0]["kl"] and said[-1]["value"] < said[0]["value"]
    # the trained network searches again, with its new weights
    assert token_policy.searched_positions(net, 8, 64, 20, 4)[1].shape == target.shape
