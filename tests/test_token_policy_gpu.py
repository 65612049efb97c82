"""The token policy network: embedding, delta rule with positions, categorical head and AdamW together, against a plain
implementation in 64 bits, and stepwise acting against whole segments."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
F = torch.nn.functional


def network(seed=0, layers=1, vocab=37, actions=19, d_model=64, **kw):
    from memorax_b200 import blocks
    torch.manual_seed(seed)
    return blocks.TokenPolicyNet(vocab, actions, d_model=d_model, num_heads=2, head_dim=64, layers=layers, **kw).cuda().bfloat16()


def inputs(batch, steps, vocab=37, actions=19, seed=1, p_done=0.1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda n: torch.randint(0, n, (batch, steps), device="cuda", generator=g)
    return r(vocab), r(actions), torch.rand(batch, steps, device="cuda", generator=g) < p_done, torch.randn(batch, steps, device="cuda", generator=g)


def positions_of(done):
    out = torch.zeros(done.shape, dtype=torch.long)
    for b in range(done.shape[0]):
        at = -1
        for t in range(done.shape[1]):
            at = 0 if done[b, t] else at + 1
            out[b, t] = at
    return out.to(done.device)


def plain_policy(model, p, tokens, done, base=10000.0):
    """The network's logits in 64 bits; ``p``: parameters by name."""
    from oracle import memoroid_oracle as mo
    x = p["embed.weight"][tokens] * model.embed.scale
    pos = positions_of(done).double()
    for i in range(0, len(model.torso.blocks), 2):
        for j in (i, i + 1):
            n = f"torso.blocks.{j}."
            normed = F.layer_norm(x, x.shape[-1:], p[n + "module.norm.weight"], p[n + "module.norm.bias"], 1e-5)
            dense = lambda y, m: F.linear(y, p[m + ".weight"], p.get(m + ".bias"))
            if j == i:
                c, cell = n + "module.module.cell.", model.torso.blocks[j].module.module.cell
                heads = lambda t: t.view(*t.shape[:2], cell.num_heads, cell.head_dim)
                d = cell.head_dim
                angle = pos[..., None, None] * torch.tensor([base ** (-2 * k / d) for k in range(d // 2)], dtype=torch.float64, device=x.device)

                def turned(t):
                    t = F.normalize(heads(t), dim=-1, eps=1e-12)
                    a, b = t[..., :d // 2], t[..., d // 2:]
                    return torch.cat((a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()), -1)

                gates = dense(normed, c + "gate")
                beta, alpha = torch.sigmoid(gates[..., :cell.num_heads]), torch.exp(-F.softplus(gates[..., cell.num_heads:]))
                s0 = torch.zeros(x.shape[0], cell.num_heads, d, d, dtype=torch.float64, device=x.device)
                o, _ = mo.gdelta_seq(turned(dense(normed, c + "query")), turned(dense(normed, c + "key")), heads(dense(normed, c + "value")), alpha, beta, s0, done.double())
                out = dense(F.rms_norm(o.flatten(2), (cell.num_heads * d,), p[c + "norm.weight"], 1e-6), c + "output_projection")
            else:
                out = dense(F.gelu(dense(normed, n + "module.module.up"), approximate="tanh"), n + "module.module.down")
            x = x + torch.sigmoid(dense(x, n + "gate")) * out
    return F.linear(x, p["head.logits.weight"], p["head.logits.bias"])


def test_gradients_of_a_policy_loss():
    """bf16 through about twenty roundings a path (each at most 2^-8 of its value, of either sign): 2^-8 sqrt(20) is 1.7e-2 of a
    tensor's norm; gradients pass the same chain twice.  8e-2 is allowed of each parameter's gradient, 2e-2 of the loss's terms."""
    model = network()
    tokens, actions, done, advantage = inputs(4, 70)
    tokens[0, 5:9] = -1                                      # padding: no features, no gradient of a row
    actions[0, 5:9] = -1
    _, policy = model(tokens, done, actions=actions)
    loss = -(advantage * policy.log_prob).mean() - 0.01 * policy.entropy.mean()
    loss.backward()
    p = {n: t.detach().double().requires_grad_() for n, t in model.named_parameters()}
    keep = (tokens >= 0)
    padded = {**p, "embed.weight": torch.cat((p["embed.weight"], torch.zeros_like(p["embed.weight"][:1])))}
    logits = plain_policy(model, padded, torch.where(keep, tokens, 37), done)
    lp = logits.log_softmax(-1)
    entropy = -(lp.exp() * lp).sum(-1) * keep
    picked = torch.where(keep, lp.gather(-1, actions.clamp_min(0)[..., None])[..., 0], 0.0)
    want = -(advantage.double() * picked).mean() - 0.01 * entropy.mean()
    want.backward()
    off = lambda a, b: float((a.double() - b).norm() / b.norm())
    assert off(policy.log_prob, picked) <= 2e-2 and off(policy.entropy, entropy) <= 2e-2
    for n, t in model.named_parameters():
        assert t.grad is not None and off(t.grad, p[n].grad) <= 8e-2, (n, off(t.grad, p[n].grad))


def test_acting_step_by_step_is_the_segment():
    """Carries hold the state and the position: single steps, with resets, give what one call over the segment gives, up to the bf16
    roundings of the chunked and the stepwise form (as above, 3e-2 of a tensor's norm)."""
    model = network(layers=2)
    tokens, actions, done, _ = inputs(3, 20, p_done=0.15)
    with torch.no_grad():
        carry, whole = model(tokens, done, actions=actions, top=3)
        step_carry, parts = None, []
        for t in range(20):
            step_carry, got = model(tokens[:, t:t + 1], done[:, t:t + 1], step_carry, actions=actions[:, t:t + 1], top=3)
            parts.append(got)
        mid, first = model(tokens[:, :13], done[:, :13], actions=actions[:, :13])
        end, second = model(tokens[:, 13:], done[:, 13:], mid, actions=actions[:, 13:])
    off = lambda a, b: float((a.double() - b.double()).norm() / b.double().norm())
    assert off(torch.cat([p.log_prob for p in parts], 1), whole.log_prob) <= 3e-2
    assert off(torch.cat((first.log_prob, second.log_prob), 1), whole.log_prob) <= 3e-2
    for a, b, c in zip(carry, step_carry, end):
        if a is None:
            continue
        assert torch.equal(a[1], b[1]) and torch.equal(a[1], c[1])               # positions are whole numbers
        assert torch.equal(a[1][:, 0], positions_of(done)[:, -1] + 1)
        assert off(b[0], a[0]) <= 3e-2 and off(c[0], a[0]) <= 3e-2
    best = torch.cat([p.top_log_probs for p in parts], 1)
    assert bool((best[..., :-1] >= best[..., 1:]).all())


@pytest.mark.parametrize("kw", [{}, {"state_bits": 8}, {"master": True}, {"state_bits": 8, "master": True}])
def test_updates_run_and_move_every_parameter(kw):
    from memorax_b200 import blocks
    model = network(layers=2)
    trainer = blocks.TokenPolicyTrainer(model, lr=1e-2, check_every=2, **kw)
    before = [p.detach().clone() for p in model.parameters()]
    batch = inputs(4, 33)
    mask = torch.rand(4, 33, 19, device="cuda") < 0.8
    mask.scatter_(-1, batch[1][..., None], True)
    for _ in range(3):
        loss = trainer.step(*batch, mask=mask)
    assert math.isfinite(float(loss)) and trainer.optimiser.step_count == 3
    assert all(bool(p.isfinite().all()) and not torch.equal(p, b) for p, b in zip(model.parameters(), before))


def test_a_cell_without_positions_is_as_it_was():
    from memorax_b200.memoroid import DeltaNetCell, Memoroid
    torch.manual_seed(3)
    plain = Memoroid(DeltaNetCell(64, 64, 1)).cuda().bfloat16()
    torch.manual_seed(3)
    turned = Memoroid(DeltaNetCell(64, 64, 1, rotary_base=10000.0)).cuda().bfloat16()
    assert [n for n, _ in plain.named_parameters()] == [n for n, _ in turned.named_parameters()] and plain.state_dict().keys() == turned.state_dict().keys()
    assert len(plain.initialize_carry(None, (2, 64))) == 1
    state, position = turned.initialize_carry(None, (2, 64))
    x, done = torch.randn(2, 1, 64, device="cuda").bfloat16(), torch.zeros(2, 1, device="cuda")
    carry, y = turned(x, done, (state.cuda(), position.cuda()))
    assert carry[1].tolist() == [[1], [1]]
    (_,), z = plain(x, done)                       # at position 0 nothing is turned
    assert float((y.float() - z.float()).norm() / z.float().norm()) <= 3e-2
