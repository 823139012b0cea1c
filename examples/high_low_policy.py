"""A recurrent policy for the high-low trading game: played a move at a time, trained on
whole games.

    python examples/high_low_policy.py --envs 256 --updates 3

Every seat of every env is one row of the batch. Each block is ``join_norm`` -> projection ->
``short_conv`` -> ``state_scan`` -> projection, and a feed-forward block follows it:
``join_norm`` -> ``gated_linear`` -> projection. ``log_probs`` gives the log probabilities of
the four parts of a move and their entropies. While games are played, the blocks'
convolution windows and scan states are carried from move to move (``short_conv_step``,
``state_scan_step``); the update runs the same weights over the recorded observations at
once, and its log probabilities start out as those the moves were drawn from. The update is
plain policy gradient on the rewards since a seat's last action, with a baseline and a bonus
for entropy.
"""
import argparse
import math
import os
import sys

import numpy as np
import torch
from torch import nn

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if os.path.join(ROOT, "astra-cuda_amd") not in sys.path:
    sys.path.insert(0, os.path.join(ROOT, "astra-cuda_amd"))

import astra_cuda as astra  # noqa: E402
from astra_cuda import sequence as seq  # noqa: E402


class Block(nn.Module):
    """One sequence block of width D: H heads of P features with states of N values."""

    def __init__(self, D, H, P, N, taps=4):
        super().__init__()
        self.H, self.P, self.N, self.taps = H, P, N, taps
        self.mixed = H * P + 2 * N
        self.inp = nn.Linear(D, self.mixed + H + D, bias=False)  # x, B, C; dt; the join's gate
        self.out = nn.Linear(H * P, D, bias=False)
        self.conv_weight = nn.Parameter(torch.randn(self.mixed, taps) / math.sqrt(taps))
        self.conv_bias = nn.Parameter(torch.zeros(self.mixed))
        self.log_rate = nn.Parameter(torch.linspace(0.0, math.log(16.0), H))
        self.skip = nn.Parameter(torch.ones(H))
        step = torch.exp(torch.linspace(math.log(1e-2), math.log(0.3), H))
        self.dt_bias = nn.Parameter(step + torch.log(-torch.expm1(-step)))
        self.post_weight = nn.Parameter(torch.ones(D))
        self.scale = nn.Parameter(torch.full((D,), 0.5))

    def new_state(self, batch, device, dtype):
        return (torch.zeros(batch, self.taps - 1, self.mixed, device=device, dtype=dtype),
                torch.zeros(batch, self.H, self.P, self.N, device=device))

    def _parts(self, n):
        mixed, dt, gate = self.inp(n).split([self.mixed, self.H, n.shape[-1]], dim=-1)
        return mixed, dt, gate

    def _heads(self, mixed):
        x, B, C = mixed.split([self.H * self.P, self.N, self.N], dim=-1)
        return x.unflatten(-1, (self.H, self.P)), B.unsqueeze(-2), C.unsqueeze(-2)

    def forward(self, n):
        """Normed input [batch, length, D] -> (the block's output, its gate)."""
        mixed, dt, gate = self._parts(n)
        x, B, C = self._heads(seq.short_conv(mixed, self.conv_weight, self.conv_bias))
        y = seq.state_scan(x, dt, -torch.exp(self.log_rate), B, C, self.skip, dt_bias=self.dt_bias)
        return self.out(y.flatten(-2)), gate

    def step(self, n, state):
        """One position [batch, D]; ``state`` moves on in place."""
        window, h = state
        mixed, dt, gate = self._parts(n)
        x, B, C = self._heads(seq.short_conv_step(mixed, window, self.conv_weight, self.conv_bias))
        y = seq.state_scan_step(x, dt, -torch.exp(self.log_rate), B, C, h, self.skip, dt_bias=self.dt_bias)
        return self.out(y.flatten(-2)), gate


class FeedForward(nn.Module):
    """Width D to the hidden width F and back, position by position."""

    def __init__(self, D, F):
        super().__init__()
        self.gate_weight = nn.Parameter(torch.randn(F, D) / math.sqrt(D))
        self.up_weight = nn.Parameter(torch.randn(F, D) / math.sqrt(D))
        self.out = nn.Linear(F, D, bias=False)
        self.post_weight = nn.Parameter(torch.ones(D))
        self.scale = nn.Parameter(torch.full((D,), 0.5))

    def forward(self, n):
        return self.out(seq.gated_linear(n, self.gate_weight, self.up_weight))


class Policy(nn.Module):
    """Observation -> logits of the four parts of a move (bid and ask price, bid and ask size)."""

    def __init__(self, observation, max_value, max_trade, D=128, blocks=2, H=4, P=32, N=32, F=None):
        super().__init__()
        self.sizes = [max_value, max_value, max_trade + 1, max_trade + 1]
        self.embed = nn.Linear(observation, D)
        self.norms = nn.ParameterList([nn.Parameter(torch.ones(D)) for _ in range(2 * blocks + 1)])
        self.blocks = nn.ModuleList([Block(D, H, P, N) for _ in range(blocks)])
        self.forwards = nn.ModuleList([FeedForward(D, F or 2 * D) for _ in range(blocks)])
        self.head = nn.Linear(D, sum(self.sizes))

    def _run(self, observation, mix):
        r = self.embed(observation)
        n = seq.rms_norm(r, self.norms[0])
        for i, (block, forward) in enumerate(zip(self.blocks, self.forwards)):
            u, gate = mix(i, block, n)
            r, n = seq.join_norm(r, u, block.post_weight, self.norms[2 * i + 1], gate=gate, scale=block.scale)
            r, n = seq.join_norm(r, forward(n), forward.post_weight, self.norms[2 * i + 2], scale=forward.scale)
        return Moves(self.head(n), self.sizes)

    def forward(self, observations):
        """[batch, length, observation]."""
        return self._run(observations, lambda i, block, n: block(n))

    def step(self, observation, states):
        """[batch, observation], with the blocks' states."""
        return self._run(observation, lambda i, block, n: block.step(n, states[i]))

    def new_states(self, batch, device, dtype=torch.float32):
        return [b.new_state(batch, device, dtype) for b in self.blocks]


class Moves:
    """What a policy would do: logits [..., entries] of a move's parts, one behind the other."""

    def __init__(self, logits, sizes):
        self.logits, self.sizes = logits, sizes

    def draw(self, generator):
        """An entry of each part [batch, 4]."""
        return torch.stack([torch.multinomial(torch.softmax(part, -1), 1, generator=generator).squeeze(1)
                            for part in self.logits.split(self.sizes, dim=-1)], -1)

    def judge(self, choice):
        """Log probability and entropy of moves [..., 4], each the sum over their parts."""
        log_prob, entropy = seq.log_probs(self.logits, choice, sizes=self.sizes)
        return log_prob.sum(-1), entropy.sum(-1)


def log_prob(moves, choice):
    """Sum over the parts of a move of the log probability of its choice [..., 4]."""
    return moves.judge(choice)[0]


def deal(game, generator, device):
    """A new state after the game's four chance moves: two candidate values, which of them
    settles, the seats' roles, and the customers' targets."""
    p = game.get_parameters()
    n, players = game.num_markets, game.players
    state = game.new_initial_state()
    top = p["max_contract_value"]
    values = torch.randint(1, top + 1, (n, 2), generator=generator, device=device, dtype=torch.int32)
    settle = torch.randint(0, 2, (n,), generator=generator, device=device, dtype=torch.int32)
    seats = torch.argsort(torch.rand(n, players, generator=generator, device=device), 1).to(torch.int32)
    sizes = torch.randint(1, p["customer_max_size"] + 1, (n, players - 3), generator=generator, device=device,
                          dtype=torch.int32)
    signs = torch.randint(0, 2, (n, players - 3), generator=generator, device=device, dtype=torch.int32) * 2 - 1
    for action in (values, settle, seats, sizes * signs):
        state.apply_action(action)
    return state


def play(game, policy, generator, device):
    """One episode of every env: observations [envs, seats, rounds, ...], choices [..., 4],
    their log probabilities and the rewards that each choice led to."""
    state = deal(game, generator, device)
    n, players, rounds = game.num_markets, game.players, game.steps_per_player
    width = game.observation_tensor_shape()[1]
    obs = torch.empty(n, players, rounds, width, device=device)
    choices = torch.empty(n, players, rounds, 4, dtype=torch.int64, device=device)
    logp, reward = (torch.zeros(n, players, rounds, device=device) for _ in range(2))
    states = [policy.new_states(n, device) for _ in range(players)]
    seen, since = torch.empty(n, width, device=device), torch.empty(n, device=device)
    with torch.no_grad():
        for t in range(rounds):
            for seat in range(players):
                if t:
                    state.fill_rewards_since_last_action(since, seat)
                    reward[:, seat, t - 1] = since
                state.fill_observation_tensor(seen)
                moves = policy.step(seen, states[seat])
                choice = moves.draw(generator)
                obs[:, seat, t], choices[:, seat, t] = seen, choice
                logp[:, seat, t] = log_prob(moves, choice)
                prices = choice[:, :2] + 1
                state.apply_action(torch.cat([prices, choice[:, 2:]], -1).to(torch.int32).contiguous())
        final = torch.empty(n, players, device=device)
        state.fill_returns(final)
        # what the game settles after the last moves
        reward[:, :, rounds - 1] = final - reward.sum(-1)
    return obs, choices, logp, reward


def update(policy, optimizer, obs, choices, reward):
    """One step of policy gradient over whole games; returns the loss and the new pass's log
    probabilities."""
    n, players, rounds, width = obs.shape
    moves = policy(obs.reshape(n * players, rounds, width))
    logp, entropy = (v.view(n, players, rounds) for v in moves.judge(choices.reshape(n * players, rounds, 4)))
    togo = reward.flip(-1).cumsum(-1).flip(-1)
    advantage = (togo - togo.mean((0, 1))) / (togo.std() + 1e-6)
    loss = -(advantage * logp + 0.01 * entropy).mean()
    optimizer.zero_grad(set_to_none=True)
    loss.backward()
    optimizer.step()
    return loss.item(), logp.detach()


def main(argv=None):
    p = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    p.add_argument("--envs", type=int, default=256)
    p.add_argument("--players", type=int, default=5)
    p.add_argument("--rounds", type=int, default=8)
    p.add_argument("--updates", type=int, default=3)
    p.add_argument("--seed", type=int, default=0)
    a = p.parse_args(argv)
    device = torch.device("cuda:0")
    torch.manual_seed(a.seed)
    generator = torch.Generator(device=device)
    generator.manual_seed(a.seed)
    astra.register_games()
    game = astra.load_game("high_low_trading", dict(num_markets=a.envs, players=a.players, steps_per_player=a.rounds,
                                                    max_contract_value=10, max_contracts_per_trade=2))
    policy = Policy(game.observation_tensor_shape()[1], 10, 2).to(device)
    optimizer = torch.optim.Adam(policy.parameters(), lr=1e-3)
    worst = 0.0
    for u in range(a.updates):
        obs, choices, played, reward = play(game, policy, generator, device)
        loss, learned = update(policy, optimizer, obs, choices, reward)
        gap = float((played - learned).abs().max())
        worst = max(worst, gap)
        print(f"update {u}: loss {loss:+.4f}, mean return {float(reward.sum(-1).mean()):+.3f}, "
              f"log probabilities of moves and of whole games differ by at most {gap:.1e}", flush=True)
    assert np.isfinite(worst) and all(bool(torch.isfinite(q).all()) for q in policy.parameters())
    return worst


if __name__ == "__main__":
    main()
