"""AdamW over many tensors against its definition in 64 bits, step by step from the moments that are held.

Tolerances: each moment goes through three float32 roundings, the update through about ten (2^-20 of it), a stored value through
half a step of its type; 8-bit moments are off by half a step of e4m3 (2^-4 of the value, or half of its smallest number times
the block's scale; a root that would round to zero is the smallest number instead, off by at most that)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25}
RATE, BETAS, EPS, DECAY = 1e-2, (0.9, 0.95), 1e-8, 0.1


def make(shapes, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    params = [(0.1 * torch.randn(s, device="cuda", generator=g)).to(dtype) for s in shapes]
    grads = [(torch.randn(s, device="cuda", generator=g) * 10.0 ** torch.randint(-4, 2, s, device="cuda", generator=g)).to(dtype) for s in shapes]
    return params, grads


def blockwise(x):
    """A tensor's largest size in each 256, for every element."""
    flat = torch.nn.functional.pad(x.abs().flatten(), (0, -x.numel() % 256)).view(-1, 256)
    return flat.amax(1).repeat_interleave(256)[:x.numel()].view(x.shape)


def check_step(opt, grads, scale=1.0):
    before = [p.double() for p in (opt.master or opt.params)]
    m0, v0 = ([x.double() for x in side] for side in opt.moments())
    t = opt.step_count + 1
    opt.step(grads, grad_scale=scale)
    assert opt.step_count == t
    m1, v1 = opt.moments()
    for i, g in enumerate(grads):
        p = opt.params[i]
        if g is None:
            assert torch.equal((opt.master or opt.params)[i].double(), before[i]) and torch.equal(m1[i].double(), m0[i]) and torch.equal(v1[i].double(), v0[i])
            continue
        g = g.double() * scale
        m = BETAS[0] * m0[i] + (1 - BETAS[0]) * g
        v = BETAS[1] * v0[i] + (1 - BETAS[1]) * g * g
        m_size = BETAS[0] * m0[i].abs() + (1 - BETAS[0]) * g.abs()
        update = RATE / (1 - BETAS[0] ** t) / ((v / (1 - BETAS[1] ** t)).sqrt() + EPS)
        want = before[i] * (1 - RATE * DECAY) - update * m
        tol = 2.0 ** -20 * update * m_size + 2.0 ** -22 * before[i].abs()
        near = lambda got, to, tol: bool(((got.double() - to).abs() <= tol).all())
        if opt.master:
            assert near(opt.master[i], want, tol + 2.0 ** -149), f"master {i}"
            assert torch.equal(p, opt.master[i].to(p.dtype)), f"parameter {i} is not its copy's rounding"
        else:
            assert near(p, want, tol + HALF[p.dtype] * want.abs() * 1.01 + TINY[p.dtype]), f"parameter {i}"
        if opt.state_bits == 32:
            assert near(m1[i], m, 2.0 ** -22 * m_size + 2.0 ** -148) and near(v1[i], v, 2.0 ** -21 * v + 2.0 ** -148), f"moments {i}"
        else:
            unit_m, unit_v = blockwise(m) / 448, blockwise(v.sqrt()) / 448
            assert near(m1[i], m, (2.0 ** -4 + 2.0 ** -20) * m.abs() + 2.0 ** -20 * m_size + 2.0 ** -10 * 1.01 * unit_m + 2.0 ** -99), f"m {i}"
            root, got = v.sqrt(), v1[i].double().sqrt()
            assert near(got, root, (2.0 ** -4 + 2.0 ** -20) * root + 2.0 ** -9 * 1.01 * unit_v + 2.0 ** -99), f"v {i}"
            assert bool(((got > 0) | (root < 2.0 ** -70)).all()), f"v {i}: a root held as zero"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_what_8_bits_hold_is_what_single_roundings_give(dtype):
    """Codes and scales after some steps are bit for bit those of the same operations one by one: a number beside a border of the
    format would else be held a step of it away, and be its block's largest later."""
    from memorax_b200 import blocks
    params, _ = make([(100000,)], dtype)
    opt = blocks.AdamW(params, lr=RATE, betas=BETAS, eps=EPS, weight_decay=DECAY, state_bits=8)
    m = v = torch.zeros(100000, device="cuda")

    def hold(x, root):
        rows = torch.nn.functional.pad(x, (0, -x.numel() % 256)).view(-1, 256)
        top = rows.abs().amax(-1, keepdim=True)
        held = rows * (top.reciprocal() * 448.0)
        if root:
            held = torch.where(rows > 0, held.clamp_min(2.0 ** -9), held)
        return held.to(torch.float8_e4m3fn).flatten(), (top * (1.0 / 448.0)).flatten()

    for k in range(4):
        g = make([(100000,)], dtype, seed=k)[1][0]
        opt.step([g])
        g = g.float()
        m = m * BETAS[0] + g * (1.0 - BETAS[0])
        v = v * BETAS[1] + g * (1.0 - BETAS[1]) * g
        for (codes, scales), (want, want_scales) in ((opt.m, hold(m, False)), (opt.v, hold(v.sqrt(), True))):
            assert torch.equal(scales, want_scales) and torch.equal(codes.view(torch.uint8), want.view(torch.uint8))
        (m,), (v,) = opt.moments()


SHAPES = [(1,), (3, 5), (255,), (256,), (257,), (2048,), (8191,), (8192,), (8193,), (100, 333), (0,), (7,)]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype,master", [(torch.float32, None), (torch.bfloat16, None), (torch.bfloat16, True), (torch.float16, None), (torch.float16, True)])
def test_steps(bits, dtype, master):
    from memorax_b200 import blocks
    params, grads = make(SHAPES, dtype)
    opt = blocks.AdamW(params, lr=RATE, betas=BETAS, eps=EPS, weight_decay=DECAY, state_bits=bits, master=master)
    for k in range(4):
        check_step(opt, make(SHAPES, dtype, seed=k)[1], scale=0.5 if k == 2 else 1.0)
    check_step(opt, [g if i % 3 else None for i, g in enumerate(grads)])
    check_step(opt, [g.float() for g in grads])                          # float32 gradients of 16-bit parameters
    check_step(opt, [torch.zeros_like(g) for g in grads])


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("count", [1, 48, 49, 350, 351, 700, 701, 1500])
def test_many_tensors(bits, count):
    """Lists that take one launch, or several."""
    from memorax_b200 import blocks
    shapes = [(1 + 37 * i % 300,) for i in range(count)]
    params, grads = make(shapes, torch.bfloat16)
    opt = blocks.AdamW(params, lr=RATE, betas=BETAS, eps=EPS, weight_decay=DECAY, state_bits=bits)
    check_step(opt, grads)


def test_a_list_of_several_types():
    from memorax_b200 import blocks
    params = [make([s], t)[0][0] for s, t in (((300,), torch.float32), ((40, 9), torch.bfloat16), ((513,), torch.float16), ((5,), torch.bfloat16))]
    opt = blocks.AdamW(params, lr=RATE, betas=BETAS, eps=EPS, weight_decay=DECAY)
    check_step(opt, [torch.randn_like(p) for p in params])
    check_step(opt, [torch.randn(p.shape, device="cuda") for p in params])


@pytest.mark.parametrize("bits", [32, 8])
def test_unaligned_and_strided(bits):
    """Parameters cut out of one buffer anywhere, gradients that are views; what lies between the parameters stays."""
    from memorax_b200 import blocks
    flat = torch.randn(5000, device="cuda").bfloat16()
    before = flat.clone()
    params = [flat[1:1001], flat[1003:3004], flat[3010:4900].view(27, 70)]
    opt = blocks.AdamW(params, lr=RATE, betas=BETAS, eps=EPS, weight_decay=DECAY, state_bits=bits)
    wide = torch.randn(70, 27, device="cuda").bfloat16()
    check_step(opt, [torch.randn(2000, device="cuda").bfloat16()[::2], torch.ones((), device="cuda").bfloat16().expand(2001), wide.t()])
    for a, b in ((0, 1), (1001, 1003), (3004, 3010), (4900, 5000)):
        assert torch.equal(flat[a:b], before[a:b])


def test_parameters_of_a_model_and_version_counters():
    from memorax_b200 import blocks
    model = torch.nn.Sequential(torch.nn.Linear(8, 16), torch.nn.Tanh(), torch.nn.Linear(16, 1)).cuda()
    opt = blocks.AdamW(model.parameters(), lr=RATE, betas=BETAS, eps=EPS, weight_decay=DECAY)
    x = torch.randn(4, 8, device="cuda")
    model(x).square().mean().backward()
    check_step(opt, [p.grad for p in model.parameters()])
    opt.zero_grad()
    assert all(p.grad is None for p in model.parameters())
    loss = model(x).square().mean()
    kept = [p.detach().clone() for p in model.parameters()]
    opt.step()                                                            # no gradients: nothing moves
    assert all(torch.equal(a, b) for a, b in zip(kept, model.parameters()))
    loss.backward()
    loss = model(x).square().mean()
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


@pytest.mark.parametrize("bits", [32, 8])
def test_state_goes_out_and_in(bits):
    from memorax_b200 import blocks
    shapes = [(300,), (17, 31)]
    params, grads = make(shapes, torch.float32)
    build = lambda p: blocks.AdamW(p, lr=RATE, betas=BETAS, eps=EPS, weight_decay=DECAY, state_bits=bits)
    one = build([p.clone() for p in params])
    for _ in range(3):
        one.step(grads)
    two = build([p.clone() for p in one.params])
    two.load_state_dict(one.state_dict())
    three = build([p.clone() for p in one.params])
    three.load(*one.moments(), one.step_count)
    for opt in (one, two, three):
        opt.step(grads)
    assert two.step_count == three.step_count == 4
    for a, b, c in zip(one.params, two.params, three.params):
        assert torch.equal(a, b)
        # 8-bit blocks that are held anew keep their codes up to the scale's rounding
        assert float((a - c).abs().max()) <= (0.0 if bits == 32 else 1e-3)
    with pytest.raises(ValueError):
        build(params).load_state_dict({**one.state_dict(), "state_bits": 40 - bits})
    with pytest.raises(ValueError):
        build(params[:1]).load_state_dict(one.state_dict())


@pytest.mark.parametrize("bits", [32, 8])
def test_not_finite_gradients_stay_in_their_block(bits):
    from memorax_b200 import blocks
    params, grads = make([(1000,)], torch.float32)
    a, b = ([p.clone() for p in params] for _ in range(2))
    build = lambda p: blocks.AdamW(p, lr=RATE, betas=BETAS, eps=EPS, weight_decay=DECAY, state_bits=bits)
    one, two = build(a), build(b)
    bad = grads[0].clone()
    bad[300], bad[310] = math.nan, math.inf
    for g, opt in ((grads[0], one), (bad, two)):
        opt.step([g])
        opt.step([grads[0]])
    keep = torch.ones(1000, dtype=torch.bool, device="cuda")
    keep[256:512] = False
    assert torch.equal(a[0][keep], b[0][keep])
    if bits == 32:
        keep[256:512] = True
        keep[300] = keep[310] = False
        assert torch.equal(a[0][keep], b[0][keep])


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps_count(bits):
    from memorax_b200 import blocks
    shapes = [(300,), (17, 31)]
    params, grads = make(shapes, torch.bfloat16)
    a, b = ([p.clone() for p in params] for _ in range(2))
    kw = dict(lr=RATE, betas=BETAS, eps=EPS, weight_decay=DECAY, state_bits=bits, master=True)
    eager, held = blocks.AdamW(a, **kw), blocks.AdamW(b, capturable=True, **kw)
    static = [torch.zeros_like(g) for g in grads]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held.step(static)
    assert held.step_count == 0
    for k in range(3):
        for s, g in zip(static, make(shapes, torch.bfloat16, seed=k)[1]):
            s.copy_(g)
        graph.replay()
        eager.step(make(shapes, torch.bfloat16, seed=k)[1])
        if k == 1:
            held.lr.fill_(RATE / 2)
            eager.lr = RATE / 2
    assert held.step_count == eager.step_count == 3
    for x, y in zip(eager.master, held.master):
        assert float((x - y).abs().max()) <= 2.0 ** -20        # coefficients computed on the device: a rounding of lr's
    with pytest.raises(RuntimeError, match="capturable"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            eager.step(grads)
    torch.cuda.synchronize()


def test_step_on_another_stream():
    from memorax_b200 import blocks
    params, grads = make([(5000,)], torch.bfloat16)
    a, b = ([p.clone() for p in params] for _ in range(2))
    one, two = blocks.AdamW(a, lr=RATE), blocks.AdamW(b, lr=RATE)
    one.step(grads)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        two.step(grads)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(a[0], b[0])


def test_rate_that_is_not_on_the_device_is_refused():
    """``lr`` of a capturable optimiser may be put in its place anew, as one float32 on the parameters' device only."""
    from memorax_b200 import blocks
    p, g = torch.zeros(10, device="cuda"), torch.ones(10, device="cuda")
    opt = blocks.AdamW([p], lr=RATE, capturable=True)
    for bad in (torch.tensor(RATE), torch.tensor(RATE, device="cuda", dtype=torch.float64), torch.zeros(2, device="cuda")):
        opt.lr = bad
        with pytest.raises(ValueError, match="lr"):
            opt.step([g])
    opt.lr = torch.tensor(RATE, device="cuda")
    opt.step([g])
    assert opt.step_count == 1 and bool((p != 0).all())


def test_parameters_without_a_gradient_stay_as_autograd_saved_them():
    """A graph that saved one goes on; one that saved a parameter that took a step is refused."""
    from memorax_b200 import blocks
    a, b = (torch.ones(10, device="cuda").requires_grad_() for _ in range(2))
    kept, moved = (a * a).sum(), (b * b).sum()
    blocks.AdamW([a, b], lr=RATE).step([None, torch.ones(10, device="cuda")])
    kept.backward()
    assert torch.equal(a.grad, torch.full((10,), 2.0, device="cuda"))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        moved.backward()


def test_refusals():
    from memorax_b200 import blocks
    p = torch.zeros(10, device="cuda")
    for args, kw in ((([],), {}), (([p, p],), {}), (([p, p[3:]],), {}), (([p, torch.zeros(3)],), {}), (([p.double()],), {}), (([p], ), {"state_bits": 16}),
                     (([torch.zeros(4, 4, device="cuda").t()[:2]],), {}), (([p],), {"master": [p.clone()]}), (([p.half()],), {"master": [p[:5]]}),
                     (([p.half()],), {"master": [p, p]}), (([p],), {"betas": (1.0, 0.9)}), (([p],), {"eps": -1.0})):
        with pytest.raises(ValueError):
            blocks.AdamW(*args, **kw)
    opt = blocks.AdamW([p])
    for bad in ([], [p, p], [p[:5]], [p.half()], [p.cpu()], [p.view(2, 5)], [torch.zeros(10, device="cuda").to_sparse()]):
        with pytest.raises(ValueError):
            opt.step(bad)
    assert opt.step_count == 0
    p.data = torch.zeros(12, device="cuda")
    with pytest.raises(ValueError):
        opt.step([torch.zeros(12, device="cuda")])
