"""What an AdamW optimiser holds, out and in again, and lists in which only some parameters have float32 copies."""
import pytest
import torch

pytestmark = pytest.mark.gpu

SETTING = dict(lr=1e-2, betas=(0.9, 0.95), weight_decay=0.1)


def model(seed):
    torch.manual_seed(seed)
    return torch.nn.Sequential(torch.nn.Linear(20, 33), torch.nn.Tanh(), torch.nn.Linear(33, 7))


def gradients(net, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randn(p.shape, device="cuda", generator=g).to(p.dtype) for p in net.parameters()]


@pytest.mark.parametrize("capturable", [False, True])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_run_is_resumed_with_its_float32_copies(dtype, bits, capturable):
    """The optimiser is built over fresh weights, then the model's and the optimiser's states are loaded: the next step is bit for bit the
    one of the run that went on."""
    from memorax_b200 import blocks
    one = model(0).cuda().to(dtype)
    build = lambda net: blocks.AdamW(net.parameters(), state_bits=bits, master=True, capturable=capturable, **SETTING)
    first = build(one)
    for k in range(5):
        first.step(gradients(one, k))
    saved = first.state_dict()
    weights = {k: v.clone() for k, v in one.state_dict().items()}
    two = model(1).cuda().to(dtype)
    second = build(two)
    two.load_state_dict(weights)
    second.load_state_dict(saved)
    for net, opt in ((one, first), (two, second)):
        opt.step(gradients(net, 9))
    assert second.step_count == 6
    for a, b in zip([*one.parameters(), *first.master], [*two.parameters(), *second.master], strict=True):
        assert torch.equal(a, b)
    for a, b, kept in zip(first.master, second.master, saved["master"]):
        assert a.data_ptr() != kept.data_ptr() != b.data_ptr() and not torch.equal(a, kept)      # the state is a copy


@pytest.mark.parametrize("bits", [32, 8])
def test_copies_of_a_state_without_any_are_made_from_the_loaded_parameters(bits):
    from memorax_b200 import blocks
    one, two = model(0).cuda().bfloat16(), model(1).cuda().bfloat16()
    first = blocks.AdamW(one.parameters(), state_bits=bits, **SETTING)
    first.step(gradients(one, 0))
    for state in (first.state_dict(), {k: v for k, v in first.state_dict().items() if k != "master"}):
        second = blocks.AdamW(two.parameters(), state_bits=bits, master=True, **SETTING)
        two.load_state_dict(one.state_dict())
        second.load_state_dict(state)
        assert all(torch.equal(p.detach().float(), c) for p, c in zip(two.parameters(), second.master))
        two.load_state_dict(model(1).bfloat16().state_dict())
    # the same through the moments' values: copies stay, are made again, or are given
    third = blocks.AdamW(two.parameters(), state_bits=bits, master=True, **SETTING)
    before = [x.clone() for x in third.master]
    two.load_state_dict(one.state_dict())
    third.load(*first.moments(), 1)
    assert all(torch.equal(a, b) for a, b in zip(third.master, before))
    third.load(*first.moments(), 1, master=True)
    assert all(torch.equal(p.detach().float(), c) for p, c in zip(two.parameters(), third.master))
    third.load(*first.moments(), 1, master=before)
    assert all(torch.equal(a, b) for a, b in zip(third.master, before))


@pytest.mark.parametrize("bits", [32, 8])
def test_a_state_that_does_not_fit_changes_nothing(bits):
    from memorax_b200 import blocks
    one, two = model(0).cuda().bfloat16(), model(1).cuda().bfloat16()
    first, second = (blocks.AdamW(net.parameters(), state_bits=bits, master=True, **SETTING) for net in (one, two))
    for net, opt in ((one, first), (two, second)):
        opt.step(gradients(net, 3))
    state, before = first.state_dict(), second.state_dict()
    flat = lambda s: [y for x in (s["m"], s["v"], s["master"]) for y in (x if isinstance(x, (tuple, list)) else (x,))]
    short = lambda held: tuple(x[:-1] for x in held) if isinstance(held, tuple) else held[:-1]
    for bad in ({**state, "v": short(state["v"])}, {**state, "master": state["master"][:-1]}, {**state, "master": [x[:1] for x in state["master"]]}):
        with pytest.raises(ValueError):
            second.load_state_dict(bad)
    m, v = first.moments()
    for bad in ((m, v[:-1], 7), (m, [x[:1] for x in v], 7), (m, v, 7, first.master[:-1])):
        with pytest.raises(ValueError):
            second.load(*bad)
    assert second.step_count == 1 and all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(flat(before), flat(second.state_dict())))
    with pytest.raises(ValueError, match="copies"):
        blocks.AdamW(two.parameters(), state_bits=bits, **SETTING).load_state_dict(state)


TYPES = [torch.bfloat16, torch.float32, torch.float16, torch.float32, torch.bfloat16]


def mixed(seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [(0.1 * torch.randn(n, device="cuda", generator=g)).to(t) for n, t in zip((300, 17, 513, 2049, 1), TYPES)]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("given", [False, True])
def test_copies_of_the_16_bit_parameters_of_a_list(bits, given):
    """Each parameter goes as in a list of its own type: the 16-bit ones with copies, the float32 ones without."""
    from memorax_b200 import blocks
    params = mixed(0)
    copies = [None if p.dtype == torch.float32 else p.float() for p in params]
    opt = blocks.AdamW(params, state_bits=bits, master=copies if given else True, **SETTING)
    alone = [p.clone() for p in params]
    singles = [blocks.AdamW([p], state_bits=bits, master=None if p.dtype == torch.float32 else True, **SETTING) for p in alone]
    for k in range(3):
        grads = mixed(k + 1)
        opt.step(grads)
        for single, g in zip(singles, grads):
            single.step([g])
    for i, (p, q, single) in enumerate(zip(params, alone, singles)):
        assert torch.equal(p, q)
        assert opt.master[i] is None if p.dtype == torch.float32 else torch.equal(opt.master[i], single.master[0])
    again = blocks.AdamW([p.clone() for p in params], state_bits=bits, master=True, **SETTING)
    again.load_state_dict(opt.state_dict())
    for o in (opt, again):
        o.step(grads)
    assert all(torch.equal(a, b) for a, b in zip(opt.params, again.params))
    again.load(*opt.moments(), 4, master=True)
    assert all(c is None or torch.equal(p.float(), c) for p, c in zip(again.params, again.master))


def test_copies_for_the_wrong_parameters_are_refused():
    from memorax_b200 import blocks
    half, single = torch.zeros(10, device="cuda").half(), torch.zeros(10, device="cuda")
    for master in ([None, None], [half.float(), single.clone()], [half.float()], [half, None], [single, None]):
        with pytest.raises(ValueError):
            blocks.AdamW([half, single], master=master)
    opt = blocks.AdamW([half, single], master=True)
    state = opt.state_dict()
    for master in ([None, None], [half.float(), single.clone()]):
        with pytest.raises(ValueError):
            opt.load_state_dict({**state, "master": master})


def test_a_graph_that_saved_a_copy_is_refused_after_a_step():
    from memorax_b200 import blocks
    params = [torch.ones(10, device="cuda").bfloat16() for _ in range(2)]
    copies = [p.float().requires_grad_() for p in params]
    kept, moved = ((c * c).sum() for c in copies)
    opt = blocks.AdamW(params, master=copies, **SETTING)
    opt.step([None, torch.ones(10, device="cuda").bfloat16()])
    kept.backward()
    assert torch.equal(copies[0].grad, torch.full((10,), 2.0, device="cuda"))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        moved.backward()
