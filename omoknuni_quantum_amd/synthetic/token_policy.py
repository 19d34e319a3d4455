"""A small policy network over board tokens that searches with the package's MCTS and trains on
what the searches return: the operators of ``net_ops`` in one path.

A position is one token per cell, ``3 * cell + content`` (0 empty, 1 the mover's stone, 2 the
other's), looked up in one table; two kinds of layer alternate on the residual, a product over
the cells and one over the channels, each behind a root-mean-square norm of the residual sum; the
policy is one logit per cell, the value a mean over the cells.

* ``evaluator()`` has ``evaluate_batch(features)`` (the protocol of ``MCTS``): the norms before the
  channel products give them their input in 8 bits with a scale for every row, and so are those
  products' weights.  It holds the weights as they were when it was made; the network's own
  ``evaluate_batch`` lays them out at every call.
* ``train_step(...)``: dropout on every branch (fused into the norms), the clipped policy loss
  against the searches' policies over the legal cells, the table's gradient over sorted tokens.

``python -m omoknuni_quantum_amd.synthetic.token_policy`` searches a batch of random Gomoku
positions, trains on the visit distributions and prints the loss of every step.
"""
from __future__ import annotations

import math

import numpy as np
import torch
import torch.nn as nn
import torch.nn.functional as F

from .. import net_ops


def position_tokens(features: torch.Tensor) -> torch.Tensor:
    """int32 [positions, cells] of feature planes [positions, planes, board, board]: plane 0
    holds the mover's stones, plane 1 the other's."""
    # (in whole numbers: bfloat16 planes would round tokens above 256)
    own, other = (features[:, k].flatten(1).to(torch.int32) for k in (0, 1))
    cell = torch.arange(own.shape[1], device=own.device, dtype=torch.int32)
    return 3 * cell + own + 2 * other


class _Block(nn.Module):
    """A product over the cells and one over the channels (times `widen` and back)."""

    def __init__(self, cells: int, dim: int, widen: int):
        super().__init__()
        self.norm_cells = nn.Parameter(torch.ones(dim))
        self.norm_channels = nn.Parameter(torch.ones(dim))
        self.cells = nn.Linear(cells, cells, bias=False)
        self.up = nn.Linear(dim, widen * dim, bias=False)
        self.down = nn.Linear(widen * dim, dim, bias=False)

    def mix(self, y):
        """Over the cells, as a product of matrices (rows: position and channel)."""
        b, c, d = y.shape
        rows = y.transpose(1, 2).reshape(b * d, c)
        return self.cells(rows).view(b, d, c).transpose(1, 2).contiguous()


class TokenPolicy(nn.Module):
    """The network, its evaluator and its training step."""

    input_channels = 18

    def __init__(self, board_size: int = 15, dim: int = 128, blocks: int = 3, widen: int = 2,
                 dropout: float = 0.1, seed: int = 0, device: str = "cuda"):
        super().__init__()
        self.board, self.dim, self.p, self.seed = board_size, dim, dropout, seed
        c = board_size * board_size
        with torch.random.fork_rng(devices=[]):
            torch.manual_seed(seed)
            self.table = nn.Parameter(torch.randn(3 * c, dim) / dim)
            self.blocks = nn.ModuleList(_Block(c, dim, widen) for _ in range(blocks))
            self.norm_out = nn.Parameter(torch.ones(dim))
            self.policy = nn.Linear(dim, 1)
            self.value = nn.Linear(dim, 1)
        self.steps = 0
        self.to(device)

    # ---- training --------------------------------------------------------------------------
    def tokens(self, features: torch.Tensor) -> torch.Tensor:
        """position_tokens(features)."""
        return position_tokens(features)

    def forward(self, tokens: torch.Tensor):
        """(logits [positions, cells], values [positions]) for training; a new dropout mask for
        every branch and every value of `steps`, which train_step counts."""
        p = self.p if self.training else 0.0
        use = self.steps * (2 * len(self.blocks) + 1)
        branch = net_ops.token_embedding(tokens, self.table, math.sqrt(self.dim))
        h = None
        for block in self.blocks:
            y, h = net_ops.add_rms_norm(branch, h, block.norm_cells, p=p, seed=self.seed,
                                        offset=use)
            y, h = net_ops.add_rms_norm(block.mix(y), h, block.norm_channels, p=p,
                                        seed=self.seed, offset=use + 1)
            branch = block.down(F.gelu(block.up(y)))
            use += 2
        y, _ = net_ops.add_rms_norm(branch, h, self.norm_out, p=p, seed=self.seed, offset=use)
        return self.policy(y)[..., 0], torch.tanh(self.value(y.mean(1)))[:, 0]

    def train_step(self, optimizer, tokens, target, legal, actions, advantages, old_logp, outcome,
                   clip: float = 0.2, kl_coef: float = 1.0) -> dict:
        """One step on positions with the searches' policies `target` [positions, cells], the
        moves played, their advantages and log-probabilities when they were played, and the
        games' outcomes.  Returns the losses."""
        self.train()
        logits, values = self(tokens)
        loss, _, kl = net_ops.clipped_policy_loss(logits, actions, advantages, old_logp, clip,
                                                  clip, kl_coef, target=target, legal=legal)
        value_loss = F.mse_loss(values, outcome)
        total = loss.mean() + value_loss
        optimizer.zero_grad(set_to_none=True)
        total.backward()
        optimizer.step()
        self.steps += 1
        said = torch.stack((total, loss.mean(), kl.mean(), value_loss)).detach().tolist()
        return dict(zip(("loss", "policy", "kl", "value"), said))

    # ---- serving ---------------------------------------------------------------------------
    def evaluator(self) -> "Evaluator":
        """The network for serving, with its weights as they are now: make another one when they
        have changed.  (Making one takes 0.2 ms, 32 positions of 15 x 15 cells 0.5 ms.)"""
        return Evaluator(self)

    def serve(self, tokens: torch.Tensor):
        """evaluator().serve(tokens)."""
        return self.evaluator().serve(tokens)

    def evaluate_batch(self, features: torch.Tensor):
        """evaluator().evaluate_batch(features)."""
        return self.evaluator().evaluate_batch(features)


class Evaluator:
    """A TokenPolicy's weights laid out for serving, copies all: bfloat16, the channel products'
    weights in 8 bits with a scale per output column, the heads in float32.  Without dropout,
    whatever mode the network is in."""

    @torch.no_grad()
    def __init__(self, net: TokenPolicy):
        def copy(p, dtype=torch.bfloat16):
            return p.detach().to(dtype, copy=True)

        self.input_channels, self.dim = net.input_channels, net.dim
        self.table, self.norm_out = copy(net.table), copy(net.norm_out)
        self.blocks = []
        for b in net.blocks:
            w = b.up.weight.detach().float()
            scale = (w.abs().amax(1, keepdim=True) / 448.0).clamp_(min=2.0**-126)
            self.blocks.append((copy(b.norm_cells), copy(b.cells.weight), copy(b.norm_channels),
                                (w / scale).to(torch.float8_e4m3fn), scale.t().contiguous(),
                                copy(b.down.weight)))
        self.heads = [(copy(h.weight, torch.float32), copy(h.bias, torch.float32))
                      for h in (net.policy, net.value)]

    @torch.no_grad()
    def serve(self, tokens: torch.Tensor):
        """(logits, values) as TokenPolicy.forward without dropout, in bfloat16 and 8 bits."""
        branch, h = net_ops.token_embedding(tokens, self.table, math.sqrt(self.dim)), None
        b, c, d = branch.shape
        for norm_cells, cells, norm_channels, up, up_scale, down in self.blocks:
            y, h = net_ops.add_rms_norm(branch, h, norm_cells)
            y = F.linear(y.transpose(1, 2).reshape(b * d, c), cells)
            y = y.view(b, d, c).transpose(1, 2).contiguous()
            q, scales, h = net_ops.add_rms_norm_fp8(y, h, norm_channels)
            y = torch._scaled_mm(q.view(b * c, d), up.t(), scale_a=scales.view(b * c, 1),
                                 scale_b=up_scale, out_dtype=torch.bfloat16)
            branch = F.linear(F.gelu(y), down).view(b, c, d)
        y, _ = net_ops.add_rms_norm(branch, h, self.norm_out)
        y = y.float()
        policy, value = self.heads
        return (F.linear(y, *policy)[..., 0],
                torch.tanh(F.linear(y.mean(1), *value))[:, 0])

    def evaluate_batch(self, features: torch.Tensor):
        """(policies [positions, cells], values [positions]) of feature planes.  The policy of a
        full board is zero."""
        logits, values = self.serve(position_tokens(features))
        occupied = (features[:, 0] + features[:, 1]).flatten(1) > 0
        policies = torch.softmax(logits.masked_fill_(occupied, -math.inf), 1)
        return policies.masked_fill_(occupied, 0.0), values  # (NaN where all are)


def searched_positions(net: TokenPolicy, positions: int, simulations: int, stones: int,
                       seed: int, wave: int = 32):
    """Random Gomoku positions, searched with the network: (tokens, visit distributions, legal
    cells, moves drawn from them, the network's log-probabilities of those moves)."""
    from ..core.mcts import MCTS
    from ..core.mcts_config import GameType, MCTSConfig
    from . import games

    bs = net.board
    boards = games.random_boards(positions, bs, stones, seed)
    config = MCTSConfig(num_simulations=simulations, max_wave_size=wave, c_puct=1.4,
                        virtual_loss=3.0, game_type=GameType.GOMOKU, board_size=bs,
                        device="cuda", num_trees=positions, seed=seed,
                        max_tree_nodes=1024 + 2 * simulations * bs * bs)
    evaluator = net.evaluator()
    policies = MCTS(config, evaluator).search_batch(boards)
    device = net.table.device
    flat = torch.from_numpy(np.ascontiguousarray(boards).reshape(positions, -1)).to(device)
    # player 1 moves on an even number of stones
    mover = torch.where((flat != 0).sum(1) % 2 == 0, 1, 2)[:, None]
    planes = torch.stack(((flat == mover), (flat != 0) & (flat != mover)), 1)
    tokens = net.tokens(planes.view(positions, 2, bs, bs).to(torch.int32))
    target = torch.from_numpy(np.ascontiguousarray(policies)).to(device, torch.float32)
    legal = flat == 0
    g = torch.Generator(device=device).manual_seed(seed)
    actions = torch.multinomial(target, 1, generator=g)[:, 0]
    with torch.no_grad():
        logits = evaluator.serve(tokens)[0].masked_fill(~legal, -math.inf)
        old = torch.log_softmax(logits, 1).gather(1, actions[:, None])[:, 0]
    return tokens, target, legal, actions, old


def main(steps: int = 20, positions: int = 64) -> list:
    net = TokenPolicy()
    optimizer = torch.optim.AdamW(net.parameters(), lr=2e-3)
    tokens, target, legal, actions, old = searched_positions(net, positions, 128, 60, 1)
    g = torch.Generator(device=tokens.device).manual_seed(2)
    outcome = torch.randint(0, 2, (positions,), generator=g, device=tokens.device) * 2.0 - 1.0
    losses = []
    for step in range(steps):
        # (no critic here: the outcomes stand in for the moves' advantages)
        said = net.train_step(optimizer, tokens, target, legal, actions, 0.1 * outcome, old,
                              outcome)
        losses.append(said["loss"])
        print(f"step {step}: loss {said['loss']:.4f}, policy {said['policy']:.4f}, "
              f"kl {said['kl']:.4f}, value {said['value']:.4f}", flush=True)
    return losses


if __name__ == "__main__":
    main()
