"""The operators at the two ends of a network over discrete symbols, of its positions and of its update, as timed cases.

A case is a dict of plain values; its ``op`` says which operator it goes through:

* ``embed``    lookup of scaled rows of a table, ``ops.embedding``; ``grad``: and the table's gradient
* ``rotate``   norms of queries and keys for each head with the position rotation, ``ops.norm_rotate``; ``grad``: and the
               gradients of queries, keys and both weights
* ``logprob``  log probabilities of given tokens with entropy and top alternatives, ``ops.token_log_probs``; ``grad``: and
               the gradient of the logits
* ``adamw``    one AdamW step over a list of tensors, ``blocks.AdamW``

With ``own`` false ``run`` computes them from elementary torch operations in float32."""
import itertools
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
#: elements that share a scale in 8-bit optimiser states, and the largest number of their format
BLOCK, MOST = 256, 448.0
LR, BETAS, EPS, DECAY, STEP = 3e-4, (0.9, 0.999), 1e-8, 0.01, 100


def listed():
    return [
        # one acting step of 64 environments: a row each
        {"name": "embed-act", "op": "embed", "rows": 64, "vocab": 32768, "dim": 512, "dtype": "bf16", "grad": False},
        # a minibatch of 32 segments of 500 steps, a vocabulary that is no multiple of anything
        {"name": "embed-train", "op": "embed", "rows": 16000, "vocab": 50001, "dim": 512, "dtype": "bf16", "grad": True},
        # a large update: 64 segments of 1024 steps into a wide table
        {"name": "embed-train-wide", "op": "embed", "rows": 65536, "vocab": 131072, "dim": 1024, "dtype": "bf16", "grad": True},
        # one acting step at far positions, before the recurrent mixer
        {"name": "rotate-act", "op": "rotate", "batch": 64, "steps": 1, "heads": 8, "key_heads": 8, "dim": 128, "rotary": 128,
         "interleaved": False, "norm": "rms", "far": 1000000, "dtype": "bf16", "grad": False},
        # an update of a wide mixer with shared key heads, queries and keys cut out of one projection
        {"name": "rotate-train", "op": "rotate", "batch": 8, "steps": 2048, "heads": 32, "key_heads": 8, "dim": 128, "rotary": 128,
         "interleaved": False, "norm": "rms", "far": 4096, "dtype": "bf16", "grad": True},
        # float32 heads of 80 of which half are rotated, in pairs of neighbours; ragged lengths
        {"name": "rotate-train-part", "op": "rotate", "batch": 5, "steps": 1111, "heads": 6, "key_heads": 6, "dim": 80, "rotary": 40,
         "interleaved": True, "norm": "l2", "far": 2000, "dtype": "fp32", "grad": True},
        # one acting step: the chosen token and the eight best of each environment
        {"name": "logprob-act", "op": "logprob", "rows": 64, "vocab": 32768, "dtype": "bf16", "top": 8, "masked": False, "grad": False},
        # a policy loss over a whole vocabulary: both cotangents, odd rows
        {"name": "logprob-train", "op": "logprob", "rows": 8000, "vocab": 50001, "dtype": "bf16", "top": 0, "masked": False, "grad": True},
        # a policy with eighteen actions, some of them not allowed, over a whole rollout
        {"name": "logprob-actions", "op": "logprob", "rows": 131072, "vocab": 18, "dtype": "fp32", "top": 0, "masked": True, "grad": True},
        # the benchmark's value network: 512 features, four layers, bf16 with float32 copies
        {"name": "adamw-net", "op": "adamw", "layout": "net", "features": 512, "layers": 4, "vocab": 0, "dtype": "bf16", "bits": 32, "master": True},
        # many small and odd float32 tensors: what a step costs besides its bytes
        {"name": "adamw-ragged", "op": "adamw", "layout": "ragged", "count": 300, "most": 4001, "dtype": "fp32", "bits": 32, "master": False},
        # a wide network with a table, both moments in 8 bits
        {"name": "adamw-8bit", "op": "adamw", "layout": "net", "features": 2048, "layers": 8, "vocab": 50001, "dtype": "bf16", "bits": 8, "master": False},
    ]


def _log(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    op = rng.choice(("embed", "rotate", "logprob", "adamw"))
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    grad = rng.random() < 0.6
    if op == "embed":
        dim = rng.choice((64, 100, 256, 512, 1000, 1024, 2048))
        return {"op": op, "rows": _log(rng, 1, 65536 * 512 // max(dim, 512)), "vocab": _log(rng, 64, 131072 * 512 // max(dim, 512)),
                "dim": dim, "dtype": dtype, "grad": grad}
    if op == "rotate":
        dim = rng.choice((32, 64, 80, 96, 128, 256))
        key_heads = rng.choice((1, 2, 4, 6, 8))
        heads = key_heads * rng.choice((1, 2, 4))
        batch = _log(rng, 1, 64)
        most = 16384 * 40 * 128 // (2 * (heads + key_heads) * dim * batch)
        return {"op": op, "batch": batch, "steps": _log(rng, 1, max(1, min(8192, most))), "heads": heads, "key_heads": key_heads,
                "dim": dim, "rotary": rng.choice((dim, dim // 2)), "interleaved": rng.random() < 0.3,
                "norm": rng.choice(("rms", "rms", "l2")), "far": _log(rng, 1, 1000000), "dtype": dtype, "grad": grad}
    if op == "logprob":
        vocab = _log(rng, 2, 131072)
        return {"op": op, "rows": _log(rng, 1, min(131072, 200000000 // vocab)), "vocab": vocab, "dtype": dtype,
                "top": 0 if grad else min(vocab, rng.choice((0, 1, 5, 8, 20))), "masked": rng.random() < 0.3, "grad": grad}
    bits = rng.choice((8, 32))
    master = dtype != "fp32" and rng.random() < 0.5
    if rng.random() < 0.5:
        return {"op": op, "layout": "net", "features": 64 * _log(rng, 1, 16), "layers": rng.randint(1, 8), "vocab": _log(rng, 16, 20000),
                "dtype": dtype, "bits": bits, "master": master}
    return {"op": op, "layout": "ragged", "count": _log(rng, 1, 600), "most": _log(rng, 10, 60000), "dtype": dtype, "bits": bits,
            "master": master}


def _shapes(case):
    """The tensors of a list: a network's (projections, two-layer blocks, gates, norms, a table and a head), or odd ones."""
    if case["layout"] == "ragged":
        return [(1 + (7919 * i * i + 31 * i) % case["most"],) for i in range(case["count"])]
    f, layer = case["features"], []
    layer += [(f, f)] * 4 + [(16, f), (16,), (f,), (f,)]              # query, key, value, output, gates, norms
    layer += [(4 * f, f), (4 * f,), (f, 4 * f), (f,)]                 # the two-layer block
    layer += [(f, f), (f,)] * 2 + [(f,)] * 4                          # residual gates, norms
    return ([(case["vocab"], f)] if case["vocab"] else []) + layer * case["layers"] + [(f, 128), (f,), (1, f), (1,)]


def _layout(case):
    """(where each tensor starts in one buffer, its shape), and the buffer's length: starts are multiples of BLOCK."""
    shapes = _shapes(case)
    ends = list(itertools.accumulate(-(-math.prod(s) // BLOCK) * BLOCK for s in shapes))
    return list(zip([0, *ends[:-1]], shapes)), ends[-1]


def _ids(gen, rows, vocab):
    """Tokens as a corpus has them: the n-th most frequent one n times as rare as the first."""
    u = torch.rand(rows, generator=gen, device="cuda", dtype=torch.float64)
    return (torch.exp(u * math.log(vocab + 1.0)).floor().long() - 1).clamp_(0, vocab - 1)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    rn = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    state = {"case": case}
    if case["op"] == "embed":
        table = (rn(case["vocab"], case["dim"]) / math.sqrt(case["dim"])).to(dtype)
        state.update(ids=_ids(gen, case["rows"], case["vocab"]), table=table.requires_grad_(case["grad"]),
                     scale=math.sqrt(case["dim"]))
        if case["grad"]:
            state["dy"] = rn(case["rows"], case["dim"]).to(dtype)
    elif case["op"] == "rotate":
        b, t, hq, hk, d = case["batch"], case["steps"], case["heads"], case["key_heads"], case["dim"]
        joint = (1.5 * rn(b, t, (hq + 2 * hk) * d)).to(dtype)          # query | key | value of one projection
        weights = [(1.0 + 0.2 * rn(d)).to(dtype) for _ in range(2)] if case["norm"] == "rms" else [None, None]
        start = torch.randint(0, case["far"], (b, 1), generator=gen, device="cuda")
        state.update(q=joint[..., :hq * d].unflatten(-1, (hq, d)), k=joint[..., hq * d:(hq + hk) * d].unflatten(-1, (hk, d)),
                     weights=weights, positions=start + torch.arange(t, device="cuda"))
        if case["grad"]:
            state.update(wrt=[x.detach().requires_grad_() for x in (state["q"], state["k"], *weights) if x is not None],
                         dq=rn(b, t, hq, d).to(dtype), dk=rn(b, t, hk, d).to(dtype))
            state["q"], state["k"] = state["wrt"][:2]
            if weights[0] is not None:
                state["weights"] = state["wrt"][2:]
        if own:
            from memorax_b200 import ops
            state["plan"] = ops.RotaryPlan(case["rotary"], interleaved=case["interleaved"], device="cuda")
    elif case["op"] == "logprob":
        n, v = case["rows"], case["vocab"]
        logits = (3.0 * rn(n, v)).to(dtype)
        state.update(tokens=torch.randint(0, v, (n,), generator=gen, device="cuda"), mask=None)
        if case["masked"]:
            state["mask"] = torch.rand(n, v, generator=gen, device="cuda") < 0.7
            state["mask"].scatter_(1, state["tokens"][:, None], True)       # a token that was chosen was allowed
        if case["grad"]:
            logits.requires_grad_()
            state.update(dlp=rn(n), dent=0.01 * rn(n))
        state["logits"] = logits
    else:
        starts, size = _layout(case)
        real = torch.zeros(size, device="cuda")       # ones, and zeros behind a tensor that does not fill its last block
        for (at, shape) in starts:
            real[at:at + math.prod(shape)] = 1.0
        values, m, v = rn(size).mul_(0.05).mul_(real), rn(size).mul_(0.003).mul_(real), rn(size).square_().mul_(1e-4).mul_(real)
        flat, grads = values.to(dtype), rn(size).mul_(0.01).mul_(real).to(dtype)
        cut = lambda x: [x[at:at + math.prod(shape)].view(shape) for at, shape in starts]
        state.update(flat=flat, master=values if case["master"] else None)
        if own:
            from memorax_b200 import blocks
            state["grads"] = cut(grads)
            state["adamw"] = blocks.AdamW(cut(flat), lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY, state_bits=case["bits"],
                                          master=cut(values) if case["master"] else None)
            state["adamw"].load(cut(m), cut(v), STEP)
        else:
            eight = case["bits"] == 8
            state.update(grads=grads, step=STEP, m=_hold(m) if eight else m, v=_hold_root(v.sqrt()) if eight else v)
    return state


# ---------------------------------------------------------------------------------------------------- plain forms
def _embed(state):
    table, ids = state["table"], state["ids"]
    out = (table.detach()[ids].float() * state["scale"]).to(table.dtype)
    if not state["case"]["grad"]:
        return out
    total = torch.zeros(table.shape, device=table.device).index_add_(0, ids, state["dy"].float())
    return out, (total * state["scale"]).to(table.dtype)


def _angles(case, positions):
    """cos and sin (B, T, 1, R / 2): the angle in 64 bits, where a far position leaves digits behind its turns."""
    i = torch.arange(case["rotary"] // 2, device="cuda", dtype=torch.float64)
    angle = positions.double()[..., None, None] * 10000.0 ** (-2.0 * i / case["rotary"])
    return angle.cos().float(), angle.sin().float()


def _pairs(case, x):
    r = case["rotary"]
    return (x[..., 0:r:2], x[..., 1:r:2]) if case["interleaved"] else (x[..., :r // 2], x[..., r // 2:r])


def _join(case, a, b, x):
    turned = torch.stack((a, b), -1).flatten(-2) if case["interleaved"] else torch.cat((a, b), -1)
    return torch.cat((turned, x[..., case["rotary"]:]), -1)


def _turn(case, x, cos, sin):
    a, b = _pairs(case, x)
    return _join(case, a * cos - b * sin, b * cos + a * sin, x)


def _norm_scale(case, x):
    if case["norm"] == "rms":
        return torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)
    return 1.0 / x.square().sum(-1, keepdim=True).sqrt().clamp_min(1e-6)


def _rotate_one(case, x, weight, cos, sin):
    f = x.detach().float()
    n = f * _norm_scale(case, f)
    return _turn(case, n if weight is None else n * weight.detach().float(), cos, sin).to(x.dtype)


def _rotate_one_grad(case, x, weight, dy, cos, sin):
    f = x.detach().float()
    r = _norm_scale(case, f)
    n, g = f * r, _turn(case, dy.float(), cos, -sin)
    wg = g if weight is None else g * weight.detach().float()
    share = (n * wg).mean(-1, keepdim=True) if case["norm"] == "rms" else (n * wg).sum(-1, keepdim=True)
    dx = (r * (wg - n * share)).to(x.dtype)
    return dx, None if weight is None else (n * g).sum((0, 1, 2)).to(weight.dtype)


def _rotate(state):
    case, (wq, wk) = state["case"], state["weights"]
    cos, sin = _angles(case, state["positions"])
    out = _rotate_one(case, state["q"], wq, cos, sin), _rotate_one(case, state["k"], wk, cos, sin)
    if not case["grad"]:
        return out
    (dq, dwq), (dk, dwk) = (_rotate_one_grad(case, *a, cos, sin) for a in ((state["q"], wq, state["dq"]), (state["k"], wk, state["dk"])))
    return (*out, dq, dk) if wq is None else (*out, dq, dk, dwq, dwk)


def _logprob(state):
    case, logits, tokens, mask = state["case"], state["logits"].detach(), state["tokens"][:, None], state["mask"]
    z = logits.float()
    if mask is not None:
        z = z.masked_fill(~mask, -math.inf)
    shifted = z - z.amax(-1, keepdim=True)
    e = shifted.exp()
    total = e.sum(-1, keepdim=True)
    logs = shifted - total.log()
    p = e / total
    entropy = -torch.where(p > 0, p * logs, 0.0).sum(-1)
    out = (logs.gather(-1, tokens)[:, 0], entropy)
    if case["top"]:
        # value, then lowest index: float bits in the order of the values above the index's complement
        bits = z.view(torch.int32).long()
        key = (torch.where(bits < 0, -(bits & 0x7fffffff), bits) << 32) + (0x7fffffff - torch.arange(case["vocab"], device=z.device))
        best = key.topk(case["top"], -1).indices
        out = (*out, logs.gather(-1, best), best)
    if not case["grad"]:
        return out
    dlp, dent = state["dlp"][:, None], state["dent"][:, None]
    d = -p * dlp - torch.where(p > 0, p * (logs + entropy[:, None]), 0.0) * dent
    return (*out, d.scatter_add_(-1, tokens, dlp).to(logits.dtype))


def _hold(x):
    """Numbers as 8-bit floats with a scale for every BLOCK of them."""
    rows = x.view(-1, BLOCK)
    top = rows.abs().amax(-1, keepdim=True)
    top = torch.where(top < 2.0 ** -100, 0.0, top)
    held = rows * torch.where(top > 0, MOST / top, 0.0)
    return held.to(torch.float8_e4m3fn).flatten(), (top / MOST).flatten()


def _hold_root(x):
    """As _hold, of numbers that are not negative; one that is not zero is held as no less than the format's smallest."""
    rows = x.view(-1, BLOCK)
    top = rows.amax(-1, keepdim=True)
    top = torch.where(top < 2.0 ** -100, 0.0, top)
    held = rows * torch.where(top > 0, MOST / top, 0.0)
    held = torch.where((top > 0) & (rows > 0), held.clamp_min(2.0 ** -9), 0.0)
    return held.to(torch.float8_e4m3fn).flatten(), (top / MOST).flatten()


def _values(held):
    codes, scales = held
    return (codes.float().view(-1, BLOCK) * scales[:, None]).flatten()


def _adamw(state):
    case, master, m, v = state["case"], state["master"], state["m"], state["v"]
    eight = case["bits"] == 8
    state["step"] += 1
    c1, c2 = 1.0 - BETAS[0] ** state["step"], 1.0 - BETAS[1] ** state["step"]
    g = state["grads"].float()
    m_new = (_values(m) if eight else m) * BETAS[0] + g * (1.0 - BETAS[0])
    v_new = (_values(v).square() if eight else v) * BETAS[1] + g * (1.0 - BETAS[1]) * g
    root = v_new.sqrt()
    x = state["flat"].float() if master is None else master
    x = x * (1.0 - LR * DECAY) - m_new / (root * c2 ** -0.5 + EPS) * (LR / c1)
    if eight:
        m[0].copy_((held := _hold(m_new))[0]), m[1].copy_(held[1])
        v[0].copy_((held := _hold_root(root))[0]), v[1].copy_(held[1])
    else:
        m.copy_(m_new)
        v.copy_(v_new)
    if master is not None:
        master.copy_(x)
    state["flat"].copy_(x)
    return {"params": state["flat"], "master": master, "m": m, "v": v}


# -------------------------------------------------------------------------------------------------------- the calls
def run(state):
    case = state["case"]
    if not own:
        return {"embed": _embed, "rotate": _rotate, "logprob": _logprob, "adamw": _adamw}[case["op"]](state)
    from memorax_b200 import ops
    if case["op"] == "embed":
        out = ops.embedding(state["ids"], state["table"], state["scale"])
        return (out, *torch.autograd.grad(out, state["table"], state["dy"])) if case["grad"] else out
    if case["op"] == "rotate":
        out = ops.norm_rotate(state["q"], state["k"], state["plan"], state["positions"], *state["weights"], norm=case["norm"], eps=1e-6)
        return (*out, *torch.autograd.grad(out, state["wrt"], (state["dq"], state["dk"]))) if case["grad"] else out
    if case["op"] == "logprob":
        got = ops.token_log_probs(state["logits"], state["tokens"], mask=state["mask"], top=case["top"])
        out = (got.log_prob, got.entropy)
        if case["grad"]:
            return (*out, *torch.autograd.grad(out, state["logits"], (state["dlp"], state["dent"])))
        return (*out, got.top_log_probs, got.top_tokens) if case["top"] else out
    adamw = state["adamw"]
    adamw.step(state["grads"])
    return {"params": state["flat"], "master": state["master"], "m": adamw.m, "v": adamw.v}


def work(case):
    s = BYTES[case["dtype"]]
    if case["op"] == "embed":
        n, v, d = case["rows"], case["vocab"], case["dim"]
        # the rows that are read, as many as tokens of _ids's frequencies hit
        distinct = sum(-math.expm1(n * math.log1p(-math.log1p(1.0 / (i + 1.0)) / math.log(v + 1.0))) for i in range(v))
        forward = 8 * n + (distinct + n) * d * s
        return {"bytes": forward + ((n + v) * d * s if case["grad"] else 0), "flops": (2 if case["grad"] else 1) * n * d}
    if case["op"] == "rotate":
        tokens, width = case["batch"] * case["steps"], (case["heads"] + case["key_heads"]) * case["dim"]
        # queries and keys in and out; with gradients the cotangents in and the gradients out besides
        return {"bytes": tokens * (width * s * (4 if case["grad"] else 2) + 8), "flops": tokens * width * (20 if case["grad"] else 7)}
    if case["op"] == "logprob":
        n, v = case["rows"], case["vocab"]
        forward = n * (v * (s + case["masked"]) + 16 + 12 * case["top"])
        return {"bytes": forward + (n * (v * s + 8) if case["grad"] else 0), "flops": n * v * (12 if case["grad"] else 6)}
    shapes = _shapes(case)
    n = sum(math.prod(x) for x in shapes)
    state = 4 * n if case["bits"] == 32 else n + 4 * sum(-(-math.prod(x) // BLOCK) for x in shapes)
    # with float32 copies the 16-bit parameters are only written
    values = (8 + s if case["master"] else 2 * s) * n
    return {"bytes": values + s * n + 4 * state, "flops": 15 * n}


# ---------------------------------------------------------------------------------------- the definitions in 64 bits
def _exact_rotate(case, x, weight, dy, position):
    x = x.detach().double()
    d, r = x.shape[-1], case["rotary"]
    n2 = (x * x).sum(-1, keepdim=True)
    length = (n2 / d + 1e-6).sqrt() if case["norm"] == "rms" else n2.sqrt().clamp_min(1e-6)
    unit = x / length
    w = torch.ones(d, device=x.device, dtype=torch.float64) if weight is None else weight.detach().double()
    idx = torch.arange(r // 2, device=x.device)
    first, second = (2 * idx, 2 * idx + 1) if case["interleaved"] else (idx, idx + r // 2)
    theta = position.double()[:, :, None, None] / torch.pow(torch.tensor(10000.0, device=x.device, dtype=torch.float64), 2.0 * idx.double() / r)
    turn = torch.polar(torch.ones_like(theta), theta)
    y = unit * w
    z = torch.complex(y[..., first], y[..., second]) * turn
    y[..., first], y[..., second] = z.real, z.imag
    if dy is None:
        return y, None, None
    g = dy.double().clone()
    z = torch.complex(g[..., first], g[..., second]) * turn.conj()
    g[..., first], g[..., second] = z.real, z.imag
    gw = g * w
    along = (gw * unit).sum(-1, keepdim=True)
    dx = (gw - unit * along / (d if case["norm"] == "rms" else 1)) / length
    return y, dx, None if weight is None else torch.einsum("bthd,bthd->d", g, unit)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "embed":
        table, ids = s["table"].detach().double(), s["ids"]
        out = torch.index_select(table, 0, ids) * s["scale"]
        if not case["grad"]:
            return out
        order = torch.argsort(ids, stable=True)
        ends = torch.bincount(ids, minlength=case["vocab"]).cumsum(0)
        sums = torch.nn.functional.pad(s["dy"].double()[order].cumsum(0), (0, 0, 1, 0))[torch.nn.functional.pad(ends, (1, 0))]
        return out, (sums[1:] - sums[:-1]) * s["scale"]
    if case["op"] == "rotate":
        dq, dk = s.get("dq"), s.get("dk")
        yq, gq, wq = _exact_rotate(case, s["q"], s["weights"][0], dq, s["positions"])
        yk, gk, wk = _exact_rotate(case, s["k"], s["weights"][1], dk, s["positions"])
        return ((yq, yk) + ((gq, gk) if dq is not None else ()) + ((wq, wk) if wq is not None else ()))
    if case["op"] == "logprob":
        parts = []
        rows = max(1, 100000000 // case["vocab"])
        for at in range(0, case["rows"], rows):       # in pieces: 64 bits of everything at once do not fit
            z = s["logits"].detach()[at:at + rows].double()
            if s["mask"] is not None:
                z = torch.where(s["mask"][at:at + rows], z, torch.full_like(z, -math.inf))
            logs = z - torch.logsumexp(z, -1, keepdim=True)
            plogs = torch.special.entr(logs.exp())
            entropy = plogs.sum(-1)
            picked = torch.nn.functional.one_hot(s["tokens"][at:at + rows], case["vocab"]).bool()
            out = [torch.where(picked, logs, 0.0).sum(-1), entropy]
            if case["top"]:
                ranked = torch.sort(logs, dim=-1, descending=True, stable=True).values[:, :case["top"]]
                out += [ranked, None]
            if case["grad"]:
                p = logs.exp()
                a, b = s["dlp"][at:at + rows, None].double(), s["dent"][at:at + rows, None].double()
                out.append(a * (picked.double() - p) + b * (plogs - p * entropy[:, None]))
            parts.append(out)
        return [None if x[0] is None else torch.cat(x) for x in zip(*parts)]
    return _exact_adamw(case, s)


def _exact_adamw(case, s):
    """The step in 64 bits from what is held before it; in 8 bits the moments are held once more."""
    t, eight = STEP + 1, case["bits"] == 8
    block = torch.arange(s["flat"].numel(), device="cuda") // BLOCK
    m, v = (x[0].float().double() * x[1].double()[block] if eight else x.double() for x in (s["m"], s["v"]))
    v = v * v if eight else v
    g = s["grads"].double()
    m = BETAS[0] * m + (1.0 - BETAS[0]) * g
    v = BETAS[1] * v + (1.0 - BETAS[1]) * g * g
    x = (s["flat"] if s["master"] is None else s["master"]).double()
    x = x - LR * DECAY * x - LR * (m / (1.0 - BETAS[0] ** t)) / ((v / (1.0 - BETAS[1] ** t)).sqrt() + EPS)
    if eight:
        m, v = _exact_hold(m, block, False), _exact_hold(v.sqrt(), block, True)
    return {"params": x, "master": x if case["master"] else None, "m": m, "v": v}


def _exact_hold(x, block, root):
    top = torch.zeros(x.numel() // BLOCK, device="cuda", dtype=torch.float64).scatter_reduce_(0, block, x.abs(), "amax")
    unit = torch.where(top[block] > 0, x / (top / MOST)[block], 0.0)
    if root:
        unit = torch.where(x > 0, unit.clamp_min(2.0 ** -9), unit)
    return unit.float().to(torch.float8_e4m3fn).double(), top / MOST
