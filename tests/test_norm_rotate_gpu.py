"""Norm and position rotation of query and key heads, and its gradients, against the definition in 64 bits.

Tolerances: half a step of the type for what is stored; a head's sum of squares or products goes through d float32 additions
((d + 32) 2^-24 with what follows it), an angle is off by at most 2^-24 of a half turn and the sine's own 2^-22."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25}


def turn(x, angle, rot, interleaved, sign=1.0):
    y = x.clone()
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else (x[..., :rot // 2], x[..., rot // 2:rot])
    c, s = angle.cos(), sign * angle.sin()
    p, q = a * c - b * s, b * c + a * s
    if interleaved:
        y[..., 0:rot:2], y[..., 1:rot:2] = p, q
    else:
        y[..., :rot // 2], y[..., rot // 2:rot] = p, q
    return y


def pair_sizes(x, rot, interleaved):
    """|a| + |b| of each element's pair, |x| behind them."""
    y = x.abs().clone()
    if interleaved:
        s = y[..., 0:rot:2] + y[..., 1:rot:2]
        y[..., 0:rot:2], y[..., 1:rot:2] = s, s.clone()
    else:
        s = y[..., :rot // 2] + y[..., rot // 2:rot]
        y[..., :rot // 2], y[..., rot // 2:rot] = s, s.clone()
    return y


def check(q, k, rot, positions=None, weights=(None, None), norm="rms", eps=1e-6, interleaved=False, base=10000.0, dys=None):
    from memorax_b200 import ops
    dtype, d = q.dtype, q.shape[-1]
    plan = ops.RotaryPlan(rot, base=base, interleaved=interleaved)
    g = torch.Generator(device="cuda").manual_seed(1)
    leaves = [x.detach().requires_grad_() if x is not None else None for x in (q, k, *weights)]
    out = ops.norm_rotate(leaves[0], leaves[1], plan, positions, leaves[2], leaves[3], norm=norm, eps=eps)
    dys = dys or [torch.randn(x.shape, device="cuda", generator=g).to(dtype) for x in (q, k)]
    grads = torch.autograd.grad(out, [x for x in leaves if x is not None], dys)
    pos = torch.arange(q.shape[1], device="cuda") if positions is None else positions
    rates = torch.tensor([math.pow(base, -2 * i / rot) for i in range(rot // 2)], dtype=torch.float64, device="cuda")
    angle = pos.double().expand(q.shape[:2])[..., None, None] * rates
    far = float(pos.abs().max()) * 2.0 ** -52 if pos.numel() else 0.0     # the reference's own angle
    unit = (d + 32) * 2.0 ** -24 + far
    for i, (x, w, y, dy, dx) in enumerate(zip((q, k), weights, out, dys, grads)):
        assert y.dtype == dtype and y.shape == x.shape and y.is_contiguous() and dx.shape == x.shape
        x64 = x.detach().double()
        r = {"rms": lambda: (x64.square().mean(-1, keepdim=True) + eps).rsqrt(), "l2": lambda: 1 / x64.norm(dim=-1, keepdim=True).clamp_min(eps),
             None: lambda: torch.ones_like(x64[..., :1])}[norm]()
        n, w64 = x64 * r, torch.ones(d, dtype=torch.float64, device="cuda") if w is None else w.double()
        want = turn(n * w64, angle, rot, interleaved)
        bound = pair_sizes(n * w64, rot, interleaved)
        bad = (y.double() - want).abs() > unit * bound + HALF[dtype] * want.abs() * 1.01 + TINY[dtype]
        assert not bad.any(), f"y[{i}]: {int(bad.sum())} off, worst {float((y.double() - want).abs().max()):.3g}"
        gy = turn(dy.double(), angle, rot, interleaved, -1.0)
        gs = pair_sizes(dy.double(), rot, interleaved)
        wg = gy * w64
        div = {"rms": d, "l2": 1, None: math.inf}[norm]
        back, back_s = (n * wg).sum(-1, keepdim=True) / div, (n * w64 * gs).abs().sum(-1, keepdim=True) / div
        if norm == "l2":
            held = x64.norm(dim=-1, keepdim=True) <= eps
            back, back_s = torch.where(held, 0.0, back), torch.where(held, 0.0, back_s)
        want = r * (wg - n * back)
        tol = 3 * unit * r * ((w64 * gs).abs() + n.abs() * back_s) + HALF[dtype] * want.abs() * 1.01 + TINY[dtype]
        bad = (dx.double() - want).abs() > tol
        assert not bad.any(), f"dx[{i}]: {int(bad.sum())} off, worst {float((dx.double() - want).abs().max()):.3g}"
        if w is not None:
            want = (n * gy).sum((0, 1, 2))
            terms = x[..., 0].numel()
            tol = (terms + 2 * d + 64) * 2.0 ** -24 * (n.abs() * gs).sum((0, 1, 2)) + far * (n.abs() * gs).sum((0, 1, 2)) + HALF[dtype] * want.abs() * 1.01 + TINY[dtype]
            dw = grads[2 + i]
            assert dw.dtype == dtype and not ((dw.double() - want).abs() > tol).any(), f"dw[{i}]"
    again = ops.norm_rotate(q, k, plan, positions, *weights, norm=norm, eps=eps)
    assert all(torch.equal(a, b) for a, b in zip(out, again))
    repeat = torch.autograd.grad(ops.norm_rotate(leaves[0], leaves[1], plan, positions, leaves[2], leaves[3], norm=norm, eps=eps), [x for x in leaves if x is not None], dys)
    assert all(torch.equal(a, b) for a, b in zip(grads, repeat))
    return out


def make(b, t, hq, hk, d, dtype, seed=0, weights=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rn = lambda *s: torch.randn(*s, device="cuda", generator=g)
    q, k = (1.5 * rn(b, t, hq, d)).to(dtype), (0.7 * rn(b, t, hk, d)).to(dtype)
    return q, k, [(1 + 0.3 * rn(d)).to(dtype) for _ in range(2)] if weights else [None, None]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,rot", [(2, 2), (6, 4), (8, 2), (20, 20), (32, 32), (64, 16), (64, 64), (80, 40), (96, 96), (128, 128), (200, 100), (256, 128), (512, 512), (510, 254)])
def test_head_dims(dtype, interleaved, d, rot):
    q, k, w = make(2, 9, 3, 2, d, dtype)
    check(q, k, rot, weights=w, interleaved=interleaved)


@pytest.mark.parametrize("norm", ["rms", "l2", None])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("b,t,hq,hk", [(1, 1, 1, 1), (64, 1, 8, 8), (3, 37, 16, 1), (1, 700, 4, 4), (2, 1500, 7, 5)])
def test_norms_and_sizes(norm, dtype, b, t, hq, hk):
    q, k, w = make(b, t, hq, hk, 64, dtype, weights=norm == "rms")
    check(q, k, 64, weights=w, norm=norm)


@pytest.mark.parametrize("kind", ["int32", "row", "column", "one", "negative", "far", "expanded"])
def test_positions(kind):
    q, k, w = make(3, 10, 4, 2, 128, torch.float32)
    g = torch.Generator(device="cuda").manual_seed(2)
    p = torch.randint(0, 5000, (3, 10), device="cuda", generator=g)
    p = {"int32": p.int(), "row": p[0], "column": p[:, :1], "one": p[0, 0], "negative": -p, "far": p + (2 ** 31 - 6000), "expanded": p[:1, :1].expand(3, 10)}[kind]
    check(q, k, 128, p, w)


def test_far_positions_keep_their_angle():
    """At 2^40 a float64 product has lost the angle too: whole numbers modulo a turn say what it is."""
    from memorax_b200 import ops
    plan = ops.RotaryPlan(8, base=100.0)
    rates = [t % 2 ** 64 for t in plan.turns.tolist()]
    positions = [2 ** 40 + 12345, 2 ** 62 - 1, -(2 ** 50)]
    q = torch.zeros(1, 3, 1, 8, device="cuda")
    q[..., :4] = 1.0
    y, _ = ops.norm_rotate(q, q, plan, torch.tensor(positions, device="cuda"), norm=None)
    for j, p in enumerate(positions):
        for i, r in enumerate(rates):
            angle = 2 * math.pi * ((p * r) % 2 ** 64) / 2 ** 64
            assert abs(float(y[0, j, 0, i]) - math.cos(angle)) < 2.0 ** -20 and abs(float(y[0, j, 0, i + 4]) - math.sin(angle)) < 2.0 ** -20


def test_heads_of_one_projection_and_other_layouts():
    g = torch.Generator(device="cuda").manual_seed(3)
    joint = torch.randn(2, 21, (6 + 2 + 2) * 64, device="cuda", generator=g).bfloat16()
    q, k = joint[..., :6 * 64].unflatten(-1, (6, 64)), joint[..., 6 * 64:8 * 64].unflatten(-1, (2, 64))
    w = [(1 + 0.1 * torch.randn(64, device="cuda", generator=g)).bfloat16() for _ in range(2)]
    check(q, k, 64, weights=w)
    check(q[:, ::2], k[:, ::2], 64, weights=w)
    check(q.transpose(1, 2).contiguous().transpose(1, 2), k, 64, weights=w)          # (B, H, T, d) memory
    check(q.expand(2, 21, 6, 64)[:, :, :1].expand(2, 21, 6, 64), k, 64, weights=w)    # one head for all
    odd = torch.randn(2 * 21 * 8 * 64 + 3, device="cuda", generator=g).bfloat16()[3:].view(2, 21, 8, 64)
    check(odd[:, :, :6], odd[:, :, 6:], 64, weights=w)                                # addresses of two bytes' alignment
    check(q.transpose(2, 3).contiguous().transpose(2, 3), k, 64, weights=w)           # elements apart: copied
    dys = [torch.randn(2, 6, 21, 64, device="cuda", generator=g).bfloat16().transpose(1, 2), torch.randn(2, 21, 1, 64, device="cuda", generator=g).bfloat16().expand(2, 21, 2, 64)]
    check(q, k, 64, weights=w, dys=dys)


def test_zero_heads_and_large_values():
    q, k, w = make(1, 8, 2, 2, 64, torch.float32)
    q[0, 0], q[0, 1] = 0.0, 1e-9
    check(q, k, 64, weights=[None, None], norm="l2")
    check(q, k, 64, weights=w)
    check(q * 1e15, k * 1e-15, 64, weights=w)
    from memorax_b200 import ops
    q[0, 2, 0, 50] = math.inf        # behind the rotated part, without a norm: nobody else's
    y, _ = ops.norm_rotate(q, k, ops.RotaryPlan(32), norm=None)
    assert y[0, 2, 0, 50] == math.inf and y.isfinite().sum() == y.numel() - 1


def test_gradient_against_differences():
    from memorax_b200 import ops
    q, k, w = make(1, 3, 2, 1, 16, torch.float32)
    plan = ops.RotaryPlan(8)
    c = [torch.randn_like(x) for x in (q, k)]
    leaves = [x.clone().requires_grad_() for x in (q, k, *w)]
    f = lambda a: sum((y.double() * z).sum() for y, z in zip(ops.norm_rotate(a[0], a[1], plan, None, a[2], a[3]), c))
    grads = torch.autograd.grad(f(leaves), leaves)
    step = 2.0 ** -7
    for n, i in ((0, 3), (0, 77), (1, 5), (1, 40), (2, 1), (2, 9), (3, 15)):
        moved = [[x.detach().clone() for x in leaves] for _ in range(2)]
        for m, s in zip(moved, (step, -step)):
            m[n].view(-1)[i] += s
        diff = float(f(moved[0]) - f(moved[1])) / (2 * step)
        assert abs(diff - float(grads[n].view(-1)[i])) <= 50 * step ** 2 + 2.0 ** -18 / step


def test_only_one_output_used_and_shared_weights():
    from memorax_b200 import ops
    q, k, w = make(2, 5, 4, 2, 32, torch.float32)
    plan = ops.RotaryPlan(32)
    a, b, s = q.clone().requires_grad_(), k.clone().requires_grad_(), w[0].clone().requires_grad_()
    yq, yk = ops.norm_rotate(a, b, plan, None, s, s)
    ga, gb, gs = torch.autograd.grad(yq.sum(), (a, b, s), retain_graph=True)
    assert ga.any() and gs.any() and not gb.any()
    (both,) = torch.autograd.grad(yq.sum() + yk.sum(), s, retain_graph=True)
    (other,) = torch.autograd.grad(yk.sum(), s)
    assert float((both - gs - other).abs().max()) <= 2.0 ** -20 * float(both.abs().max() + gs.abs().max())


def test_nothing_and_refusals():
    from memorax_b200 import ops
    plan = ops.RotaryPlan(32)
    q, k, w = make(0, 5, 4, 2, 32, torch.float32)
    leaves = [x.requires_grad_() for x in (q, k, *w)]
    out = ops.norm_rotate(leaves[0], leaves[1], plan, None, leaves[2], leaves[3])
    grads = torch.autograd.grad(out[0].sum() + out[1].sum(), leaves)
    assert out[0].shape == (0, 5, 4, 32) and not grads[2].any() and not grads[3].any()
    q, k, w = make(2, 5, 4, 2, 32, torch.float32)
    z = lambda *s, **kw: torch.zeros(*s, device="cuda", **kw)
    for args, kw in (((q, k[:, :4], plan), {}), ((q, k.half(), plan), {}), ((q.double(), k.double(), plan), {}), ((q[..., :31], k[..., :31], plan), {}),
                     ((q[..., :30], k[..., :30], plan), {}), ((z(1, 1, 1, 514), z(1, 1, 1, 514), plan), {}), ((q, k, plan), {"q_weight": w[0]}),
                     ((q, k, plan), {"q_weight": w[0], "k_weight": w[1], "norm": "l2"}), ((q, k, plan), {"q_weight": w[0], "k_weight": w[1].half()}),
                     ((q, k, plan), {"q_weight": w[0], "k_weight": w[1][:16]}), ((q, k, plan, z(2, 5)), {}), ((q, k, plan, torch.zeros(5, dtype=torch.long)), {}),
                     ((q, k, plan), {"eps": -1e-6}), ((q, k, plan), {"norm": "layer"}), ((q.cpu(), k, plan), {}), ((q, k, ops.RotaryPlan(32, device="cpu")), {}), ((q[0], k[0], plan), {})):
        with pytest.raises(ValueError):
            ops.norm_rotate(*args, **kw)
    for bad in (z(3, 5, dtype=torch.long), z(2, 4, dtype=torch.long), z(1, 2, 5, dtype=torch.long), z(0, dtype=torch.long)):
        with pytest.raises(ValueError):
            ops.norm_rotate(q, k, plan, bad)
    leaf = q.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(ops.norm_rotate(leaf, k, plan)[0].sum(), leaf, create_graph=True)


def test_streams_and_graphs():
    from memorax_b200 import ops
    q, k, w = make(4, 33, 8, 2, 64, torch.bfloat16)
    plan = ops.RotaryPlan(64)
    dq, dk = torch.randn_like(q), torch.randn_like(k)

    def calls():
        leaves = [x.detach().requires_grad_() for x in (q, k, *w)]
        out = ops.norm_rotate(leaves[0], leaves[1], plan, None, leaves[2], leaves[3])
        return [*out, *torch.autograd.grad(out, leaves, (dq, dk))]

    want = calls()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            there = calls()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, there))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = calls()
    q.copy_(q.flip(0))
    w[0].mul_(2)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(held, calls()))
