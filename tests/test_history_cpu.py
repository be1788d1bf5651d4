"""A policy with memory (pnp_amd.history, TQCConfig.history) on the CPU: the replay buffer's windows
against a search through what was added, the learner's refusals, and that a learner without history
is what it was."""
import pytest
import torch

from pnp_amd import tqc as T
from test_tqc_cpu import ToyReach


@pytest.mark.parametrize("steps,size", [(3, 8), (8, 8), (21, 8), (5, 1), (40, 16)])
def test_windows_are_the_sequences_that_were_added(steps, size):
    n, length = 3, 5
    g = torch.Generator().manual_seed(steps)
    buf = T.DictReplayBuffer(size * n, n, 4, 2, torch.device("cpu"), windows=True)
    assert buf.size == size
    told = []
    start = torch.ones(n, dtype=torch.bool)
    for k in range(steps):
        row = dict(obs=torch.randn(n, 4, generator=g), next=torch.randn(n, 4, generator=g), act=torch.randn(n, 2, generator=g),
                   rew=torch.randn(n, generator=g), done=(torch.rand(n, generator=g) < 0.2).float(), start=start)
        buf.add(row["obs"], row["next"], row["act"], row["rew"], row["done"], start)
        told.append(row)
        start = torch.rand(n, generator=g) < 0.2
    kept = told[-size:]
    obs, prev, starts, act, nobs, done, rew = buf.sample_windows(64, length, torch.Generator().manual_seed(1))
    seen = set()
    for i in range(64):
        # the one step that has this last observation
        (k, e), = [(k, e) for k in range(len(kept)) for e in range(n) if torch.equal(kept[k]["obs"][e], obs[i, -1])]
        seen.add((k, e))
        assert torch.equal(act[i], kept[k]["act"][e]) and torch.equal(nobs[i], kept[k]["next"][e])
        assert rew[i, 0] == kept[k]["rew"][e] and done[i, 0] == kept[k]["done"][e]
        for j in range(length):
            at = k - (length - 1) + j
            if at < 0:
                continue          # before the buffer's first step: hidden by the start below
            assert torch.equal(obs[i, j], kept[at]["obs"][e])
            begins = bool(kept[at]["start"][e]) or at == 0
            assert bool(starts[i, j]) == begins
            assert torch.equal(prev[i, j], torch.zeros(2) if begins else kept[at - 1]["act"][e])
    assert len(seen) > 1 or size * n == 1


def test_history_has_no_cpu_path():
    with pytest.raises(ValueError, match="HIP device"):
        T.TQC(ToyReach(4), T.TQCConfig(history=4))
    with pytest.raises(ValueError, match="negative"):
        T.TQC(ToyReach(4), T.TQCConfig(history=-1))


def test_learner_without_history_keeps_its_parts():
    agent = T.TQC(ToyReach(4), T.TQCConfig(net_arch=(16, 16), batch_size=8, buffer_size=64))
    assert agent.encoder is None and agent.buffer.starts is None
    assert agent.actor.latent[0].in_features == 25 and "encoder" not in agent.state_dict()


def test_train_refuses_8_bits_without_history():
    from pnp_amd import train
    with pytest.raises(SystemExit):
        train.main(["--rollout-int8"])


def test_learner_refuses_8_bits_without_history():
    with pytest.raises(ValueError, match="set history"):
        T.TQC(ToyReach(4), T.TQCConfig(rollout_int8=True))
