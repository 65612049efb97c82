"""Embedding lookup and its gradient, and token log probabilities, against their definitions in 64 bits.

Tolerances count roundings: half a step of the output's type (eps / 2 of the value), 2^-24 for every float32 operation that a
number goes through; sums of n terms in float32 are off by at most n 2^-24 times the sum of the terms' sizes."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8 / 1, torch.float16: 2.0 ** -11}   # half a step, relative
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25}    # half a step below the normal numbers
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def close(got, want, tol, what):
    got, want = got.double(), want.double()
    assert got.shape == want.shape, what
    bad = ~((got - want).abs() <= tol) & ~(got == want) & ~(got.isnan() & want.isnan())
    assert not bad.any(), f"{what}: {int(bad.sum())} off, worst {float((got - want).abs().nan_to_num().max()):.3g}"


# ---------------------------------------------------------------------------------------------------------- embedding
def embedding_reference(ids, table, scale, dy):
    vocab = table.shape[0]
    known = (ids >= 0) & (ids < vocab)
    at = torch.where(known, ids, 0).long()
    out = table.double()[at] * scale * known[..., None]
    flat, rows = at[known], dy.double()[known]
    zero = torch.zeros(table.shape, dtype=torch.float64, device=table.device)
    total, size = zero.clone().index_add_(0, flat, rows), zero.clone().index_add_(0, flat, rows.abs())
    count = torch.zeros(vocab, dtype=torch.float64, device=table.device).index_add_(0, flat, torch.ones_like(flat, dtype=torch.float64))
    return out, total * scale, size * abs(scale), count[:, None]


def check_embedding(ids, table, scale, seed=0):
    from memorax_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = table.dtype
    dy = torch.randn(*ids.shape, table.shape[1], device="cuda", generator=g).to(dtype)
    leaf = table.clone().requires_grad_()
    out = ops.embedding(ids, leaf, scale)
    (dw,) = torch.autograd.grad(out, leaf, dy)
    assert out.dtype == dw.dtype == dtype and dw.shape == table.shape
    want, want_dw, size, count = embedding_reference(ids, table, scale, dy)
    scale_step = 2.0 ** -24                                       # the scale itself is a float32 in the kernel
    close(out, want, want.abs() * (HALF[dtype] + 2 * 2.0 ** -24 + scale_step) + TINY[dtype], "out")
    close(dw, want_dw, want_dw.abs() * (HALF[dtype] + 2.0 ** -22) + size * (count + 2) * 2.0 ** -24 + TINY[dtype], "dw")
    assert torch.equal(out, ops.embedding(ids, table, scale))     # without a graph
    assert torch.equal(dw, torch.autograd.grad(ops.embedding(ids, leaf, scale), leaf, dy)[0])   # the same bits again


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab,dim", [(1, 1, 1), (1, 70000, 8), (7, 3, 5), (31, 1000, 100), (33, 33, 64), (1000, 17, 72), (2048, 511, 40), (2049, 512, 512),
                                            (5000, 513, 33), (20000, 300001, 16), (32769, 40, 8), (70000, 5, 24), (70001, 1000, 8), (262144, 70000, 4), (262145, 3000, 3), (300000, 1, 8)])
def test_embedding(dtype, rows, vocab, dim):
    g = torch.Generator(device="cuda").manual_seed(rows + vocab)
    table = torch.randn(vocab, dim, device="cuda", generator=g).to(dtype)
    check_embedding(torch.randint(0, vocab, (rows,), device="cuda", generator=g), table, 1.7)


@pytest.mark.parametrize("share", [0.5, 1.0])
def test_embedding_frequent_token(share):
    """One token takes half of all positions, or all: its sum crosses hundreds of runs."""
    g = torch.Generator(device="cuda").manual_seed(3)
    ids = torch.randint(0, 400, (9001,), device="cuda", generator=g)
    ids[torch.rand(9001, device="cuda", generator=g) < share] = 57
    check_embedding(ids, torch.randn(400, 96, device="cuda", generator=g).bfloat16(), 0.5)


@pytest.mark.parametrize("kind", ["int32", "shape", "strided", "outside", "all outside", "unaligned"])
def test_embedding_kinds_of_calls(kind):
    g = torch.Generator(device="cuda").manual_seed(5)
    table = torch.randn(300, 64, device="cuda", generator=g).bfloat16()
    ids = torch.randint(0, 300, (3, 50), device="cuda", generator=g)
    if kind == "int32":
        ids = ids.int()
    elif kind == "strided":
        ids = ids.t()
    elif kind == "outside":
        ids[0, :7], ids[2, 40:] = -1, 300
        ids[1, 3], ids[1, 4] = 2 ** 40, -2 ** 40
    elif kind == "all outside":
        ids[:] = -100
    elif kind == "unaligned":
        table = torch.randn(300 * 64 + 1, device="cuda", generator=g).bfloat16()[1:].view(300, 64)
    check_embedding(ids, table, -2.0)


@pytest.mark.parametrize("rows", [100, 40000])
def test_embedding_sorted_reversed_and_single_runs(rows):
    """Lists that are in order, in the opposite order, and in which every token comes exactly once, 32 or 33 times."""
    table = torch.randn(rows, 8, device="cuda")
    ids = torch.arange(rows, device="cuda")
    for order in (ids, ids.flip(0), ids // 32, ids // 33, (ids // 32).flip(0), (ids * 7919) % rows):
        check_embedding(order, table, 1.0)


def test_two_gradients_at_once_on_two_streams():
    from memorax_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(8)
    jobs = [(torch.randint(0, 3000, (n,), device="cuda", generator=g), torch.randn(3000, 64, device="cuda", generator=g).requires_grad_(), torch.randn(n, 64, device="cuda", generator=g))
            for n in (50000, 3000)]
    call = lambda ids, table, dy: torch.autograd.grad(ops.embedding(ids, table, 1.5), table, dy)[0]
    want = [call(*j) for j in jobs]
    streams = [torch.cuda.Stream() for _ in jobs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, (j, s) in enumerate(zip(jobs, streams)):
            with torch.cuda.stream(s):
                got[i].append(call(*j))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[i]) for i in range(2) for x in got[i])


def test_embedding_of_nothing():
    from memorax_b200 import ops
    table = torch.randn(5, 8, device="cuda").requires_grad_()
    out = ops.embedding(torch.zeros(0, 3, dtype=torch.long, device="cuda"), table)
    assert out.shape == (0, 3, 8)
    out.sum().backward()
    assert table.grad.shape == (5, 8) and not table.grad.any()


def test_embedding_gradient_of_expanded_and_transposed_cotangents():
    from memorax_b200 import ops
    table = torch.randn(40, 16, device="cuda").requires_grad_()
    ids = torch.arange(30, device="cuda") % 7
    (dw,) = torch.autograd.grad(ops.embedding(ids, table, 3.0).sum(), table)
    want = 3.0 * torch.bincount(ids, minlength=40).float()[:, None].expand(40, 16)
    assert torch.equal(dw, want)
    (dw,) = torch.autograd.grad(ops.embedding(ids, table).t().contiguous().t().sum(), table)
    assert torch.equal(dw, want / 3.0)


def test_embedding_refusals():
    from memorax_b200 import ops
    table, ids = torch.randn(5, 8, device="cuda"), torch.zeros(3, dtype=torch.long, device="cuda")
    for bad in ((ids.float(), table), (ids.cpu(), table), (ids, table.double()), (ids, table[0]), (ids, table[:0]), (ids, table.cpu())):
        with pytest.raises(ValueError):
            ops.embedding(*bad)
    leaf = table.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(ops.embedding(ids, leaf).square().sum(), leaf, create_graph=True)


# -------------------------------------------------------------------------------------------------- log probabilities
def logprob_reference(logits, tokens, mask, temperature, top, glp, gh):
    x = logits.double()
    vocab = x.shape[-1]
    if mask is not None:
        x = torch.where(mask.expand(x.shape).bool(), x, -math.inf)
    z = x / temperature
    empty = (z == -math.inf).all(-1, keepdim=True)
    bad = z.isnan().any(-1, keepdim=True) | (z == math.inf).any(-1, keepdim=True)
    m = torch.where(empty, 0.0, z.amax(-1, keepdim=True))
    logs = torch.where(empty, -math.inf, z - m - (z - m).exp().sum(-1, keepdim=True).log())
    p = torch.where(empty, 0.0, logs.exp())
    plogp = torch.where(p > 0, p * logs, 0.0)
    h = -plogp.sum(-1)
    spread = (p * torch.where(p > 0, (z - m).abs(), 0.0)).sum(-1)
    if bad.any():
        nan = torch.full_like(logs, math.nan)
        logs, p, plogp = (torch.where(bad, nan, t) for t in (logs, p, plogp))
        h = torch.where(bad[..., 0], math.nan, h)
    here = torch.ones_like(h, dtype=torch.bool)
    lp = None
    if tokens is not None:
        here = (tokens >= 0) & (tokens < vocab)
        lp = torch.where(here, logs.gather(-1, torch.where(here, tokens, 0).long()[..., None])[..., 0], 0.0)
    order = torch.sort(x.nan_to_num(nan=-math.inf, posinf=math.inf, neginf=-math.inf), dim=-1, descending=True, stable=True).indices[..., :top]
    a = glp if (glp is not None and tokens is not None) else torch.zeros_like(h)
    b = gh if gh is not None else torch.zeros_like(h)
    live = (here & ~empty[..., 0]).double()
    a, b = (a.double() * live)[..., None], (b.double() * live)[..., None]
    one = torch.zeros_like(p)
    if tokens is not None:
        one.scatter_(-1, torch.where(here, tokens, 0).long()[..., None], 1.0)
    if mask is not None:
        one = one * mask.expand(x.shape)
    hh = torch.where(here, h, 0.0)
    dx = (a * (one - p) - b * (plogp + p * h[..., None])) / temperature
    if mask is not None:
        dx = torch.where(mask.expand(x.shape).bool(), dx, 0.0)
    size = (a.abs() * (one + p) + b.abs() * (plogp.abs() + p * h[..., None].abs())) / temperature
    return lp, hh, logs.gather(-1, order), order, dx, size, spread, logs


def check_logprobs(logits, tokens=None, mask=None, temperature=1.0, top=0, backward=True, whole_top=True):
    from memorax_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(11)
    lead, vocab, dtype = logits.shape[:-1], logits.shape[-1], logits.dtype
    glp = torch.randn(lead, device="cuda", generator=g) if tokens is not None else None
    gh = torch.randn(lead, device="cuda", generator=g)
    lp, h, values, order, dx, size, spread, logs = logprob_reference(logits, tokens, mask, temperature, top, glp, gh)
    unit = 2.0 ** -22 * (vocab / 512 + 32)                     # a thread's share of the sum, exponents' and logarithms' roundings
    leaf = logits.detach().requires_grad_() if backward else logits
    got = ops.token_log_probs(leaf, tokens, mask, temperature, top)
    spread_safe = spread.nan_to_num()
    tol = lambda x: unit * (1 + spread_safe[(...,) + (None,) * (x.dim() - spread.dim())]) + 2.0 ** -21 * x.abs().nan_to_num(posinf=0.0, neginf=0.0)
    assert got.entropy.dtype == torch.float32
    close(got.entropy, h, tol(h) * 2, "entropy")
    if tokens is None:
        assert got.log_prob is None
    else:
        close(got.log_prob, lp, tol(lp), "log_prob")
    if top:
        assert got.top_tokens.dtype == torch.int64 and got.top_tokens.shape == (*lead, top)
        if whole_top:
            assert torch.equal(got.top_tokens, order)
            close(got.top_log_probs, values, tol(values), "top")
        assert int(got.top_tokens.min()) >= 0 and int(got.top_tokens.max()) < vocab
    else:
        assert got.top_tokens is None and got.top_log_probs is None
    if backward:
        outs = [(got.entropy, gh)] + ([(got.log_prob, glp)] if tokens is not None else [])
        (d,) = torch.autograd.grad([o for o, _ in outs], leaf, [c for _, c in outs])
        assert d.dtype == dtype and d.shape == logits.shape
        rel = (unit * (1 + spread_safe)[..., None] + 2.0 ** -21 * logs.abs().nan_to_num(posinf=0.0, neginf=0.0)) * 2
        close(d, dx, rel * size.nan_to_num() + HALF[dtype] * dx.abs().nan_to_num() * 1.01 + 2 * TINY[dtype] + 2.0 ** -120, "dlogits")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab,masked", [(1300, 1025, False), (1300, 2000, True), (1184, 4003, False), (2000, 8192, True), (1183, 1500, True), (1500, 9001, False), (40, 30001, True)])
def test_logprobs_of_many_middling_rows(dtype, rows, vocab, masked):
    """Where a warp takes a row, and the sizes around it; rows of which nothing is left among them."""
    g = torch.Generator(device="cuda").manual_seed(rows + vocab)
    logits = (2 * torch.randn(rows, vocab, device="cuda", generator=g)).to(dtype)
    logits[5] = -math.inf
    tokens = torch.randint(0, vocab, (rows,), device="cuda", generator=g)
    tokens[6] = -1
    mask = None
    if masked:
        mask = torch.rand(rows, vocab, device="cuda", generator=g) < 0.6
        mask[7] = False
    check_logprobs(logits, tokens, mask)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (1000, 18), (65, 33), (7, 128), (5, 129), (9, 1000), (4, 1024), (3, 1025), (5, 4097), (130, 5003), (2, 50001), (1, 131073),
                                        (300, 8192)])
def test_logprobs(dtype, rows, vocab):
    g = torch.Generator(device="cuda").manual_seed(rows + vocab)
    logits = (3 * torch.randn(rows, vocab, device="cuda", generator=g)).to(dtype)
    tokens = torch.randint(0, vocab, (rows,), device="cuda", generator=g)
    check_logprobs(logits, tokens, top=min(vocab, 1 + rows % 32))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("rows,vocab", [(1, 129), (37, 128), (1301, 257), (6, 1023), (1300, 1025), (1184, 70001), (1500, 33001), (2400, 3001)])
def test_logprobs_warps_and_walking_blocks(dtype, masked, rows, vocab):
    """Rows around the lengths and numbers at which a row goes to lanes, a warp or a walking block; each with odd starts."""
    g = torch.Generator(device="cuda").manual_seed(rows + vocab)
    logits = torch.randn(rows, vocab, device="cuda", generator=g).to(dtype)
    tokens = torch.randint(0, vocab, (rows,), device="cuda", generator=g)
    mask = None
    if masked:
        mask = torch.rand(rows, vocab, device="cuda", generator=g) < 0.6
        mask[torch.arange(rows, device="cuda"), tokens] = True
        mask[rows // 2] = False
    check_logprobs(logits, tokens, mask)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab", [(303105, 4), (303103, 5), (152001, 9), (152001, 8), (40001, 33), (9600, 128), (9470, 127), (9473, 65)])
def test_logprobs_of_many_short_rows(dtype, rows, vocab):
    """More rows than a wave: eight entries a lane; the last block not full, some rows without a token."""
    g = torch.Generator(device="cuda").manual_seed(rows)
    logits = torch.randn(rows, vocab, device="cuda", generator=g).to(dtype)
    tokens = torch.randint(-1, vocab, (rows,), device="cuda", generator=g)
    mask = torch.rand(rows, vocab, device="cuda", generator=g) < 0.6
    check_logprobs(logits, tokens, mask)
    check_logprobs(logits, tokens, None, top=3)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab,top", [(200, 32), (257, 1), (257, 3), (400, 20), (500, 32), (1000, 2), (1000, 32), (1023, 32), (1025, 32), (1024, 3)])
def test_logprobs_largest_of_short_rows(dtype, vocab, top):
    g = torch.Generator(device="cuda").manual_seed(vocab + top)
    logits = (torch.randn(150, vocab, device="cuda", generator=g) * 2).to(dtype)
    logits[3] = logits[3, 0]                      # all alike: the lowest indices
    logits[4, ::2] = -math.inf
    check_logprobs(logits, torch.randint(0, vocab, (150,), device="cuda", generator=g), None, top=top)


@pytest.mark.parametrize("temperature", [0.05, 0.7, 30.0])
@pytest.mark.parametrize("vocab", [40, 3001])
@pytest.mark.parametrize("masked", [False, True])
def test_logprobs_temperature_and_mask(temperature, vocab, masked):
    g = torch.Generator(device="cuda").manual_seed(vocab)
    logits = (2 * torch.randn(6, 5, vocab, device="cuda", generator=g)).bfloat16()
    tokens = torch.randint(0, vocab, (6, 5), device="cuda", generator=g).int()
    mask = torch.rand(6, 5, vocab, device="cuda", generator=g) < 0.5 if masked else None
    if masked:
        mask.scatter_(-1, tokens[..., None].long(), True)
        logits[0, 0][~mask[0, 0]] = math.nan                   # whatever a masked place holds
        logits[0, 1][~mask[0, 1]] = math.inf
        logits[0, 2][~mask[0, 2]] = 1e30
    if temperature < 0.1:      # z of some hundreds: sizes of the exponents' roundings are in the tolerance's logs
        logits = logits / 8
    check_logprobs(logits, tokens, mask, temperature, top=min(vocab, 9))


@pytest.mark.parametrize("vocab", [20, 1500])
def test_logprobs_special_rows(vocab):
    """Rows of which nothing is left, of one entry, of the type's lowest value, with infinities and NaN; tokens that are not there."""
    g = torch.Generator(device="cuda").manual_seed(1)
    logits = torch.randn(12, vocab, device="cuda", generator=g)
    tokens = torch.randint(1, vocab, (12,), device="cuda", generator=g)
    logits[0] = -math.inf
    logits[1], logits[1, 3], tokens[1] = -math.inf, 2.0, 3
    logits[2] = torch.finfo(torch.float32).min
    logits[3], logits[3, 5], tokens[3] = torch.finfo(torch.float32).min, 0.0, 5
    logits[4, 7] = math.nan
    logits[5, 9] = math.inf
    tokens[6], tokens[7] = -1, vocab
    logits[8, 4], tokens[8] = -math.inf, 4                      # the token itself has no probability
    logits[9] = 0.0                                             # all alike: ties
    logits[10] = 1e4 + logits[10]
    logits[11, ::2] = -math.inf
    check_logprobs(logits, tokens, top=0)
    fine = [i for i in range(12) if i not in (4, 5)]
    check_logprobs(logits[fine].contiguous(), tokens[fine].contiguous(), top=10)
    check_logprobs(logits[4:6], None, top=10, backward=False, whole_top=False)
    mask = torch.ones(12, vocab, dtype=torch.bool, device="cuda")
    mask[3], mask[9, 1:] = False, False
    mask[4, 7] = mask[5, 9] = False                             # NaN and infinity in masked places
    tokens[9] = 0
    check_logprobs(logits, tokens, mask, top=10)


@pytest.mark.parametrize("vocab,top", [(1024, 32), (1025, 32), (6000, 32), (70000, 20)])
@pytest.mark.parametrize("order", ["rising", "falling", "equal", "steps", "one thread"])
def test_logprobs_top_of_ordered_rows(vocab, top, order):
    """Values whose largest sit together, all alike, or all with the same few threads (more of them than the buffer holds)."""
    x = torch.arange(vocab, device="cuda", dtype=torch.float32) / vocab
    if order == "falling":
        x = -x
    elif order == "equal":
        x = torch.zeros_like(x)
    elif order == "steps":
        x = (x * 7).floor()
    elif order == "one thread":      # every 16-byte vector of the first threads is large
        x = torch.where(torch.arange(vocab, device="cuda") // 8 % 256 < 40, x + 5, x)
    check_logprobs(torch.stack((x, x.flip(0))).bfloat16(), None, top=top, backward=False)
    check_logprobs(torch.stack((x, x.flip(0), x)), None, top=top, backward=False)


@pytest.mark.parametrize("vocab", [50, 2001, 2048])
def test_logprobs_strides(vocab):
    g = torch.Generator(device="cuda").manual_seed(vocab)
    wide = torch.randn(4, 6, vocab + 24, device="cuda", generator=g).bfloat16()
    tokens = torch.randint(0, vocab, (4, 6), device="cuda", generator=g)
    check_logprobs(wide[..., :vocab], tokens, top=3)             # a padded vocabulary
    check_logprobs(wide[..., 3:vocab + 3], tokens, top=3)        # rows that begin anywhere
    check_logprobs(wide[:, :5, :vocab], tokens[:, :5], top=3)    # two strides
    check_logprobs(wide[:1, :, :vocab].expand(4, 6, vocab), tokens, top=3)
    check_logprobs(wide[..., :vocab].transpose(0, 1), tokens.t(), top=3)
    check_logprobs(wide[0, 0, :vocab], tokens[0, 0], top=3)      # one row
    mask = torch.rand(vocab, device="cuda", generator=g) < 0.8
    mask[0] = True
    check_logprobs(wide[..., :vocab], torch.zeros_like(tokens), mask, top=3)
    check_logprobs(wide[..., 1:vocab + 1], torch.zeros_like(tokens), mask.byte().expand(4, 6, vocab), top=3)


def test_logprobs_cotangents():
    """Only one of the outputs used, sums (an expanded cotangent), strided cotangents."""
    from memorax_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(2)
    logits = torch.randn(8, 1111, device="cuda", generator=g).requires_grad_()
    tokens = torch.randint(0, 1111, (8,), device="cuda", generator=g)
    p = logits.double().softmax(-1)
    one = torch.nn.functional.one_hot(tokens, 1111)
    # p = 2^(log p * log2 e): log p goes through two roundings, the constant and the product through one each, and an error e of
    # the exponent is one of e of p; so 4 * 2^-24 |log p| of p (twice that is allowed), besides 2^-20 for the sums and 2^x itself
    rel = 2.0 ** -20 + 2.0 ** -21 * p.log().abs()
    (d,) = torch.autograd.grad(ops.token_log_probs(logits, tokens).log_prob.sum(), logits)
    close(d, one - p, rel * (one + p), "sum of log_prob")
    (d,) = torch.autograd.grad(ops.token_log_probs(logits).entropy.sum(), logits)
    h = -(p * p.log()).sum(-1, keepdim=True)
    close(d, -p * (p.log() + h), 2.0 ** -17 * p * (p.log().abs() + h), "sum of entropy")
    w = torch.randn(8, 2, device="cuda", generator=g)[:, 0]
    (d,) = torch.autograd.grad(ops.token_log_probs(logits, tokens).log_prob, logits, w)
    close(d, w[:, None] * (one - p), rel * w[:, None].abs() * (one + p), "strided")
    got = ops.token_log_probs(logits, tokens, top=2)
    assert got.log_prob.requires_grad and not got.top_log_probs.requires_grad and not got.top_tokens.requires_grad


def test_logprobs_gradient_against_differences():
    from memorax_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(4)
    logits = torch.randn(3, 30, device="cuda", generator=g).requires_grad_()
    tokens, a, b = torch.tensor([1, 29, 7], device="cuda"), torch.randn(3, device="cuda", generator=g), torch.randn(3, device="cuda", generator=g)
    f = lambda x: (lambda r: (r.log_prob * a + r.entropy * b).double().sum())(ops.token_log_probs(x, tokens, temperature=0.8))
    (d,) = torch.autograd.grad(f(logits), logits)
    step = 2.0 ** -6
    for i in (0, 31, 67, 89):
        e = torch.zeros(90, device="cuda")
        e[i] = step
        diff = float(f(logits.detach() + e.view(3, 30)) - f(logits.detach() - e.view(3, 30))) / (2 * step)
        # third derivatives of some units times step^2 / 6, and the outputs' float32 roundings over the step
        assert abs(diff - float(d.view(-1)[i])) <= 20 * step ** 2 / 6 + 2.0 ** -19 / step


def test_logprobs_of_no_rows_and_refusals():
    from memorax_b200 import ops
    got = ops.token_log_probs(torch.zeros(0, 5, device="cuda"), torch.zeros(0, dtype=torch.long, device="cuda"), top=2)
    assert got.log_prob.shape == (0,) and got.top_tokens.shape == (0, 2)
    leaf = torch.zeros(0, 5, device="cuda").requires_grad_()
    assert torch.autograd.grad(ops.token_log_probs(leaf).entropy.sum(), leaf)[0].shape == (0, 5)
    x, t = torch.zeros(3, 40, device="cuda"), torch.zeros(3, dtype=torch.long, device="cuda")
    for args, kw in (((x.double(), t), {}), ((x, t[:2]), {}), ((x, t.float()), {}), ((x, t.cpu()), {}), ((x, t), {"top": 33}), ((x[:, :5], t), {"top": 6}),
                     ((x, t), {"temperature": 0.0}), ((x, t), {"temperature": -1.0}), ((x, t), {"temperature": math.nan}), ((x, t), {"temperature": math.inf}),
                     ((x, t), {"temperature": 1e-60}), ((x, t), {"temperature": 1e28}), ((x, t), {"mask": x}), ((x, t), {"mask": torch.ones(3, 40, dtype=torch.bool)}), ((x[:, :0], t), {})):
        with pytest.raises(ValueError):
            ops.token_log_probs(*args, **kw)
    with pytest.raises(RuntimeError):
        ops.token_log_probs(x, t, mask=torch.ones(2, 40, dtype=torch.bool, device="cuda"))
    leaf = x.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(ops.token_log_probs(leaf, t).log_prob.sum(), leaf, create_graph=True)


def test_calls_on_another_stream_and_in_a_graph():
    """A call on a side stream; forward and backward captured once and replayed on new contents."""
    from memorax_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(9)
    ids = torch.randint(0, 500, (700,), device="cuda", generator=g)
    table = torch.randn(500, 64, device="cuda", generator=g).bfloat16()
    logits = torch.randn(64, 5000, device="cuda", generator=g).bfloat16()
    dy = torch.randn(700, 64, device="cuda", generator=g).bfloat16()

    def calls():
        leaf, x = table.detach().requires_grad_(), logits.detach().requires_grad_()
        out = ops.embedding(ids, leaf, 2.0)
        got = ops.token_log_probs(x, ids[:64], top=4)
        return [out, *torch.autograd.grad(out, leaf, dy), got.log_prob, got.entropy, got.top_tokens, *torch.autograd.grad(got.log_prob.sum() + got.entropy.sum(), x)]

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
    ids.copy_(ids.flip(0))
    logits.copy_(logits.flip(0))
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(held, calls()))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [7, 300, 5001, 40000])
@pytest.mark.parametrize("held", [math.nan, math.inf, -math.inf])
def test_logprobs_rows_that_are_not_there_have_no_gradient(dtype, vocab, held):
    """Whatever is in them, and in their cotangents: zeros, and the other rows as without them."""
    from memorax_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(13)
    logits = torch.randn(9, vocab, device="cuda", generator=g).to(dtype)
    tokens = torch.randint(0, vocab, (9,), device="cuda", generator=g)
    clean = logits.clone().requires_grad_()
    gone = torch.tensor([2, 5], device="cuda")
    tokens[gone] = torch.tensor([-1, vocab], device="cuda")
    logits[2], logits[5, 1::3] = held, held
    cot = torch.randn(2, 9, device="cuda", generator=g)
    bad = cot.clone()
    bad[:, gone] = math.nan
    want = ops.token_log_probs(clean, tokens)
    want_dx, = torch.autograd.grad([want.log_prob, want.entropy], clean, list(cot))
    leaf = logits.requires_grad_()
    got = ops.token_log_probs(leaf, tokens)
    dx, = torch.autograd.grad([got.log_prob, got.entropy], leaf, list(bad))
    assert torch.equal(got.log_prob, want.log_prob) and torch.equal(got.entropy, want.entropy)
    assert torch.equal(dx, want_dx) and not dx[gone].any()


@pytest.mark.parametrize("vocab", [40, 3000])
def test_logprobs_hottest_and_coldest(vocab):
    """At the ends of the temperatures: even over what the mask leaves, and the largest alone."""
    from memorax_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(14)
    logits = torch.randn(5, vocab, device="cuda", generator=g)
    mask = torch.rand(5, vocab, device="cuda", generator=g) < 0.5
    mask[:, 3] = True
    tokens = torch.full((5,), 3, device="cuda")
    got = ops.token_log_probs(logits, tokens, mask, temperature=1e27)
    even = mask.sum(-1).double().log()
    # a sum of up to 3000 ones is exact; logf is within 2 units, and so is the difference: 4 eps of at most 8
    assert float((got.entropy - even).abs().max()) <= 32 * 2.0 ** -23 and float((got.log_prob + even).abs().max()) <= 32 * 2.0 ** -23
    cold = ops.token_log_probs(logits, logits.argmax(-1), temperature=1e-30)
    assert not cold.log_prob.any() and not cold.entropy.any()


def test_capture_beside_a_living_graph_is_refused():
    """A graph of the same parameter on the default stream: refused in a capture; released, the capture goes through."""
    from memorax_b200 import ops
    ids = torch.arange(20, device="cuda")
    weight = torch.randn(30, 8, device="cuda").requires_grad_()
    alive = ops.embedding(ids, weight)
    plan = ops.RotaryPlan(8)
    heads = torch.randn(1, 4, 2, 8, device="cuda").requires_grad_()
    turned = ops.norm_rotate(heads, heads.detach(), plan)
    for call in (lambda: ops.embedding(ids, weight), lambda: ops.token_log_probs(weight), lambda: ops.norm_rotate(heads, heads.detach(), plan)):
        with pytest.raises(RuntimeError, match="release it"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                call()
    want, = torch.autograd.grad(alive.sum(), weight)
    del alive, turned
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, = torch.autograd.grad(ops.embedding(ids, weight).sum(), weight)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(want, got)
