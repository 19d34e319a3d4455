"""The token policy network whose cells attend to one another: the head norms, the attention and the
log-probabilities together, as an evaluator of searches and in training."""
import math

import pytest
import torch

from omoknuni_quantum_amd.synthetic import token_policy

pytestmark = pytest.mark.gpu


def make(device, board=9, dim=64, blocks=2, heads=4, kv_heads=2, **kw):
    net = token_policy.TokenPolicy(board_size=board, dim=dim, blocks=blocks, heads=heads,
                                   kv_heads=kv_heads, device=device, **kw)
    with torch.no_grad():  # (weights other than ones)
        g = torch.Generator().manual_seed(11)
        for b in net.blocks:
            for w in (b.norm_q, b.norm_k):
                w.copy_(torch.rand(w.shape, generator=g) + 0.5)
    return net


def board_tokens(boards, size, largest, seed):
    """Random positions on boards of `size`, cells numbered as on the largest board."""
    g = torch.Generator().manual_seed(seed)
    cell = (torch.arange(size)[:, None] * largest + torch.arange(size)).flatten()
    return (3 * cell + torch.randint(0, 3, (boards, size * size), generator=g)).int()


def plain_forward(net, tokens):
    """The network in plain torch, float64, without dropout: one board [cells]."""
    table = net.table.detach().double().cpu()
    tokens = tokens.long()
    h = table[tokens] * net.dim**0.5
    place = torch.stack((tokens // 3 // net.board, tokens // 3 % net.board), 1).double()

    def w(p):
        return p.detach().double().cpu()

    def norm(x, weight):
        return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w(weight)

    for b in net.blocks:
        width = net.dim // b.heads
        pairs = width // 2
        first = pairs - pairs // 2
        freq = torch.cat([100.0 ** (-torch.arange(n).double() / n) for n in (first, pairs // 2)])
        angle = torch.cat((place[:, :1] * freq[:first], place[:, 1:] * freq[first:]), 1)[:, None]

        def turn(x):
            x, y = x[..., :pairs], x[..., pairs:]
            return torch.cat((x * angle.cos() - y * angle.sin(), y * angle.cos() + x * angle.sin()), -1)

        qkv = (norm(h, b.norm_cells) @ w(b.qkv.weight).t()).view(len(tokens), -1, width)
        q, k, v = qkv.split((b.heads, b.kv_heads, b.kv_heads), 1)
        q, k = turn(norm(q, b.norm_q)), turn(norm(k, b.norm_k))
        k, v = (t.repeat_interleave(b.heads // b.kv_heads, 1).transpose(0, 1) for t in (k, v))
        p = torch.softmax(q.transpose(0, 1) @ k.transpose(1, 2) / width**0.5, 2)
        h = h + (p @ v).transpose(0, 1).flatten(1) @ w(b.out.weight).t()
        y = norm(h, b.norm_channels) @ w(b.up.weight).t()
        h = h + torch.nn.functional.gelu(y) @ w(b.down.weight).t()
    y = norm(h, net.norm_out)
    logits = y @ w(net.policy.weight).t() + w(net.policy.bias)
    return logits[:, 0], torch.tanh(y.mean(0) @ w(net.value.weight).t() + w(net.value.bias))[0]


def test_forward_and_serving(device):
    net = make(device).eval()
    t = board_tokens(5, 9, 9, 3)
    want = [plain_forward(net, x) for x in t]
    logits, values = (x.detach() for x in net(t.to(device)))
    served = net.serve(t.to(device))
    spread = float(torch.stack([x for x, _ in want]).std())
    for i, (x, v) in enumerate(want):
        # float32 products of 64 and 128 terms on values of order 1
        assert float((logits[i].cpu() - x).abs().max()) < 1e-4
        assert abs(float(values[i]) - float(v)) < 1e-4
        # bfloat16 layers and one product in 4 significant bits a block: a few percent of the spread
        assert float((served[0][i].cpu().double() - x).pow(2).mean().sqrt()) < 0.1 * spread
        assert abs(float(served[1][i]) - float(v)) < 0.1


def test_packed_boards_of_different_sizes(device):
    net = make(device).eval()
    boards = [board_tokens(1, n, 9, n)[0] for n in (7, 9, 5, 9, 8)]
    starts = torch.tensor([0] + [len(b) for b in boards]).cumsum(0).int()
    logits, values = net(torch.cat(boards).to(device), starts.to(device))
    assert logits.shape == (int(starts[-1]),) and values.shape == (5,)
    for i, b in enumerate(boards):
        x, v = plain_forward(net, b)
        got = logits[starts[i]:starts[i + 1]].detach().cpu()
        assert float((got - x).abs().max()) < 1e-4 and abs(float(values[i]) - float(v)) < 1e-4
    with pytest.raises(ValueError, match="heads"):
        token_policy.TokenPolicy(9, 64, 1, device=device)(boards[0].to(device), starts.to(device))
    with pytest.raises(ValueError, match="divide"):
        token_policy.TokenPolicy(9, 64, 1, device=device, heads=5)


@pytest.mark.parametrize("packed", [False, True])
def test_gradients_of_the_network(device, packed):
    """Every parameter's gradient in training mode against the difference of the loss along it."""
    net = make(device, board=7, dim=32, blocks=1, dropout=0.2)
    if packed:
        boards = [board_tokens(1, n, 7, n)[0] for n in (7, 4, 6, 7)]
        starts = torch.tensor([0] + [len(b) for b in boards]).cumsum(0).int().to(device)
        args = (torch.cat(boards).to(device), starts)
    else:
        args = (board_tokens(6, 7, 7, 4).to(device),)
    g = torch.Generator(device=device).manual_seed(5)
    net.train()
    up = torch.randn(net(*args)[0].shape, generator=g, device=device)

    def value():
        logits, v = net(*args)
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


def test_search_then_train_with_an_entropy_bonus(device):
    net = make(device, heads=4, kv_heads=4)
    tokens, target, legal, actions, old = token_policy.searched_positions(net, 8, 64, 20, 3)
    optimizer = torch.optim.AdamW(net.parameters(), lr=1e-3)
    args = (tokens, target, legal, actions, torch.zeros(8, device=device), old,
            torch.ones(8, device=device))
    net.eval()
    before = net(tokens)[0].detach()
    net.p = 0.0
    with torch.no_grad():
        logq = torch.log_softmax(before.double().masked_fill(~legal, -math.inf), 1)
        entropy = -torch.where(legal, logq.exp() * logq, 0.0).sum(1).mean()
    said = net.train_step(optimizer, *args, entropy_coef=0.01)
    # a mean of sums of 81 float32 terms
    assert said["entropy"] == pytest.approx(float(entropy), abs=1e-4)
    assert said["loss"] == pytest.approx(said["policy"] + said["value"] - 0.01 * said["entropy"],
                                         abs=1e-5)
    assert "entropy" not in net.train_step(optimizer, *args)
    for p in net.parameters():
        assert p.grad is not None and bool(torch.isfinite(p.grad).all())


def test_best_moves(device):
    net = make(device)
    g = torch.Generator().manual_seed(8)
    content = torch.randint(0, 3, (4, 9, 9), generator=g)
    content[1] = 1
    content[1, 0, 0], content[1, 4, 4] = 0, 0  # (two free cells)
    planes = torch.stack((content == 1, content == 2), 1).to(device, torch.float32)
    served = net.evaluator()
    moves, logp, entropy = served.best_moves(planes, 3)
    policies, _ = served.evaluate_batch(planes)
    want = torch.where(policies > 0, -policies * policies.log(), 0.0).sum(1)
    # float32 sums of 81 terms on either side
    assert float((entropy - want).abs().max()) < 1e-4
    for i in range(4):
        free = (content[i].flatten() == 0).sum()
        n = min(3, int(free))
        assert bool((moves[i, n:] == -1).all()) and bool((logp[i, n:] == -math.inf).all())
        p = policies[i]
        assert torch.allclose(logp[i, :n].exp(), p[moves[i, :n]], rtol=1e-4)
        assert torch.allclose(p.sort(descending=True)[0][:n], p[moves[i, :n]], rtol=1e-4)


def test_example_runs(device, capsys):
    assert len(token_policy.main(steps=2, positions=4, heads=4)) == 2
    assert "step 1" in capsys.readouterr().out
