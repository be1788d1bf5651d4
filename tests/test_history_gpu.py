"""A policy with memory on the device: the encoder (all sequence operators in a row) against 64-bit
formulas, forward and back; steps against windows; the learner that trains it and the command that
runs it."""
import pytest
import torch

import seq_plain as P
from test_tqc_cpu import ToyReach

pytestmark = pytest.mark.gpu


class DeviceReach(ToyReach):
    """ToyReach with its tensors on the device."""

    def __init__(self, *a, **k):
        super().__init__(*a, **k)
        self.device = torch.device("cuda", 0)

    def _up(self, t):
        return {k: self._up(v) for k, v in t.items()} if isinstance(t, dict) else t.cuda()

    def reset(self, mask=None):
        return self._up(super().reset(mask))

    def step(self, a):
        return tuple(self._up(t) for t in super().step(a.cpu()))


def encoder(seed=0, **kw):
    from pnp_amd.history import HistoryEncoder
    torch.manual_seed(seed)
    return HistoryEncoder(9, **{**dict(dim=24, layers=2, state=8), **kw}).cuda()


def plain_encoder(enc, x, starts):
    """The encoder in 64 bits by torch's own operations, differentiable."""
    w = {k: v.detach().double().cpu().requires_grad_(True) for k, v in enc.named_parameters()}

    def norm(s, g):
        return s / (s.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * g

    keep = torch.ones(x.shape[:2], dtype=torch.bool) if starts is None else starts == 0
    h, stream = x.double() @ w["embed.weight"].t() + w["embed.bias"], 0.0
    for k, blk in enumerate(enc.blocks):
        p = lambda n: w[f"blocks.{k}.{n}"]   # noqa: E731
        stream = stream + h
        u, z = (norm(stream, p("norm")) @ p("in_proj.weight").t()).chunk(2, -1)
        B, L, D = u.shape
        W, N = enc.width, enc.state
        held, us = [torch.zeros(B, D).double()] * (W - 1), []
        for t in range(L):
            held = [v * keep[:, t, None] for v in held] + [u[:, t]]
            us.append(sum(v * p("conv_weight")[:, j] for j, v in enumerate(held)) + p("conv_bias"))
            held = held[1:]
        u = torch.nn.functional.silu(torch.stack(us, 1))
        dt, Bm, Cm = torch.split(u @ p("x_proj.weight").t(), blk.split, -1)
        dt = P.softplus(dt @ p("dt_proj.weight").t() + p("dt_bias"))
        A, s, ys = -torch.exp(p("A_log")), torch.zeros(B, D, N).double(), []
        for t in range(L):
            s = torch.exp(dt[:, t, :, None] * A) * (s * keep[:, t, None, None]) + (dt[:, t] * u[:, t])[..., None] * Bm[:, t, None]
            ys.append((s * Cm[:, t, None]).sum(-1) + p("D") * u[:, t])
        h = (torch.stack(ys, 1) * torch.nn.functional.silu(z)) @ p("out_proj.weight").t()
    return norm(stream + h, w["norm"]), w


def far(got, ref):
    return float((got.detach().double().cpu() - ref).norm() / ref.norm())


@pytest.mark.parametrize("starts", [False, True])
def test_encoder_and_its_gradients(starts):
    """Relative 2-norms: two blocks of 6 operators, products of up to 48 terms; each rounding 2^-24, errors that grow
    by no more than a few between operators (norms, gates of order 1): a few hundred steps, 2e-5."""
    enc = encoder()
    g = torch.Generator().manual_seed(3)
    x = torch.randn(5, 21, 9, generator=g)
    at = (torch.rand(5, 21, generator=g) < 0.15).to(torch.uint8) if starts else None
    dy = torch.randn(5, 21, 24, generator=g)
    xg = x.cuda().requires_grad_(True)
    f = enc(xg, None if at is None else at.cuda())
    xd = x.double().requires_grad_(True)
    ref, w = plain_encoder(enc, xd, at)
    assert far(f, ref.detach()) < 2e-5
    names = [k for k, _ in enc.named_parameters()]
    got = torch.autograd.grad(f, [xg] + list(enc.parameters()), dy.cuda())
    want = torch.autograd.grad(ref, [xd] + [w[k] for k in names], dy.double())
    for k, a, b in zip(["x"] + names, got, want):
        assert far(a, b) < 2e-5, k


def test_steps_are_the_window():
    enc = encoder(1)
    g = torch.Generator().manual_seed(4)
    x, at = torch.randn(6, 30, 9, generator=g).cuda(), (torch.rand(6, 30, generator=g) < 0.1).cuda()
    with torch.no_grad():
        whole = enc(x, at)
        state = enc.new_state(6)
        for t in range(30):
            f = enc.step(x[:, t], state, reset=at[:, t])
            assert far(f, whole[:, t].double().cpu()) < 2e-5, t


def test_8_bit_steps():
    """A product of rows in 8 bits: each operand's rounding is uniform within +-max / 254, and a row's max is about 3
    times its rms: 0.7 % of the rms each, 1 % of the product.  Six products in a row, the gates between them of slope
    about 1: sqrt(6) %, twice that allowed."""
    enc = encoder(2, dim=64, state=16)
    g = torch.Generator().manual_seed(5)
    q = enc.int8_weights()
    a, b = enc.new_state(64), enc.new_state(64)
    for t in range(12):
        x = torch.randn(64, 9, generator=g).cuda()
        at = (torch.rand(64, generator=g) < 0.2).cuda()
        f, f8 = enc.step(x, a, reset=at), enc.step(x, b, reset=at, int8=q)
        assert far(f8, f.double().cpu()) < 0.05
        assert not torch.equal(f, f8)


def agent(**kw):
    from pnp_amd.tqc import TQC, TQCConfig
    return TQC(DeviceReach(8, horizon=12, seed=3), TQCConfig(**{**dict(net_arch=(32, 32), batch_size=16, buffer_size=8 * 64, learning_starts=8,
                                                            history=6, history_dim=32, seed=5), **kw}))


def test_rollout_features_are_the_windows_features():
    """With the weights at rest, the features that the rollout carries are those of a window that reaches back to the
    episode's start."""
    a = agent(history=16)
    a.total_timesteps = 10 ** 6
    a.reset()
    a.vecnorm.training = False      # (windows are normalised with the statistics of the update, the rollout with those of the step)
    for _ in range(9):
        a.collect_step()
    seen = a._recall(a._last_norm, {"state": [tuple(t.clone() for t in s) for s in a._mem["state"]], "act": a._mem["act"], "start": a._mem["start"]})
    a.collect_step()                # adds the step that `seen` belongs to
    b = a.buffer
    rows = torch.arange(0, b.pos, device="cuda")
    x = torch.cat([a._norm(dict(zip(("achieved_goal", "desired_goal", "observation"), torch.split(b.obs[:b.pos].reshape(-1, 25), [3, 3, 19], 1)))).view(-1, 8, 25),
                   b.actions[(rows - 1) % b.size] * (b.starts[:b.pos] == 0)[..., None]], dim=2).transpose(0, 1)
    with torch.no_grad():
        f = a.encoder(x, b.starts[:b.pos].t().contiguous())[:, -1]
    assert far(seen[:, 25:], f.double().cpu()) < 2e-5


def test_learner_steps_graph_and_checkpoint(tmp_path):
    a, b = agent(), agent(graph=False)
    for m in (a, b):
        m.total_timesteps = 10 ** 6
        m.reset()
        for _ in range(8):
            m.collect_step()
    before = [p.detach().clone() for p in a.encoder.parameters()]
    for k in range(3):
        la, lb = a.train(3), b.train(3)          # 3 eager steps, then the captured one, with eager work between
        for m in (a, b):
            m.collect_step()
        assert all(torch.isfinite(v).all() for n, v in la.items() if n != "lr")
        for x, y in zip(a._critic_params() + list(a.actor.parameters()), b._critic_params() + list(b.actor.parameters())):
            assert torch.equal(x, y), k
    assert a._graph is not None and b._graph is None
    assert all(not torch.equal(x, p) for x, p in zip(before, a.encoder.parameters()))
    assert all(not torch.equal(x, y) for x, y in zip(a.encoder_target.parameters(), a.encoder.parameters()))
    a.save(tmp_path / "m.pt")
    c = agent(seed=9)
    c.load(tmp_path / "m.pt")
    for x, y in zip(list(a.encoder.parameters()) + list(a.encoder_target.parameters()), list(c.encoder.parameters()) + list(c.encoder_target.parameters())):
        assert torch.equal(x, y)
    r, s = c.evaluate(DeviceReach(8, horizon=12, seed=8), 4)
    assert torch.isfinite(torch.tensor(r)) and 0 <= s <= 1


def test_learner_trains_the_encoder_by_the_critics_loss_alone():
    """The gradients that the step applies to the encoder are those of the critics' loss."""
    from pnp_amd.tqc import quantile_huber_loss
    a = agent(graph=False)
    a.total_timesteps = 10 ** 6
    a.reset()
    for _ in range(8):
        a.collect_step()
    state = a.gen.get_state()
    rec = {}
    with torch.no_grad():
        start = [p.clone() for p in a._critic_params()]
    a._update_torch(rec)
    with torch.no_grad():
        for p, v in zip(a._critic_params(), start):
            p.copy_(v)
    # the same batch and noise again, the loss written out
    b = agent(graph=False)
    b.load_state_dict(a.state_dict())
    with torch.no_grad():
        for p, q in zip(list(b.encoder_target.parameters()) + list(b.critic_target.parameters()), [*start[len(list(b.critic.parameters())):], *start[:len(list(b.critic.parameters()))]]):
            p.copy_(q)                # (the targets of the first step are the networks themselves)
        b.log_ent_coef.zero_()
    b.buffer, b.vecnorm = a.buffer, a.vecnorm
    b.actor.load_state_dict(agent().actor.state_dict())
    b.gen.set_state(state)
    obs, act, nobs, tobs, done, rew = b._sample_history()
    b.actor.action_log_prob(obs.detach(), b.gen)
    with torch.no_grad():
        na, nlp = b.actor.action_log_prob(nobs, b.gen)
        nq = torch.sort(b.critic_target(tobs, na).reshape(16, -1))[0][:, :46]
        tq = (rew + (1 - done) * 0.95 * (nq - nlp.reshape(-1, 1))).unsqueeze(1)
    grads = torch.autograd.grad(quantile_huber_loss(b.critic(obs, act), tq), b._critic_params())
    for x, y in zip(rec["critic"], grads):
        assert torch.allclose(x, y, rtol=1e-4, atol=1e-6 * float(y.abs().max()) + 1e-9)


@pytest.mark.parametrize("int8", [False, True])
def test_train_command_with_history(tmp_path, int8):
    from pnp_amd import train
    train.main(["--envs", "16", "--total-steps", "160", "--history", "4", "--history-dim", "32", "--gradient-steps", "5",
                "--ckpt-dir", str(tmp_path), "--eval-episodes", "2"] + (["--rollout-int8"] if int8 else []))
    d = torch.load(tmp_path / "tqc_final_dense.pt", weights_only=True)
    assert d["n_updates"] == 4 * 5          # past the 100 steps of random actions: 4 vector steps
    assert all(torch.isfinite(v).all() for v in d["encoder"].values())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_8_bit_steps_of_a_16_bit_encoder(dtype):
    """Against the same encoder's steps with products in its own type.  Six products in 8 bits: sqrt(6) % (as in fp32).
    Roundings to 16 bits on top, about 20 in each of the two ways: half a step of bf16 is 0.4 %, 0.23 % in the mean square,
    sqrt(40) of them 1.4 % (fp16: an eighth).  2.8 % in all, twice that allowed."""
    enc = encoder(2, dim=64, state=16).to(dtype)
    g = torch.Generator().manual_seed(5)
    q = enc.int8_weights()
    a, b = enc.new_state(64), enc.new_state(64)
    for t in range(12):
        x = torch.randn(64, 9, generator=g).cuda().to(dtype)
        at = (torch.rand(64, generator=g) < 0.2).cuda()
        with torch.no_grad():
            f, f8 = enc.step(x, a, reset=at), enc.step(x, b, reset=at, int8=q)
        assert f.dtype == f8.dtype == dtype and all(s[0].dtype == dtype for s in b)
        assert far(f8, f.double().cpu()) < 0.056
        assert not torch.equal(f, f8)
