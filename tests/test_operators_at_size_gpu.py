"""The operators over discrete symbols where a thread block has more than one piece of work: AdamW with several turns a block, the
rotation's gradients with several tiles, the warps and blocks of many long rows of logits.  Tolerances are those of the operators'
own tests, whose checks these are."""
import math

import pytest
import test_adamw_gpu as adamw
import torch
from test_norm_rotate_gpu import check as check_rotate
from test_norm_rotate_gpu import make as make_rotate
from test_tokens_gpu import check_logprobs

pytestmark = pytest.mark.gpu

TYPES = [(torch.float32, None), (torch.bfloat16, None), (torch.bfloat16, True), (torch.float16, None), (torch.float16, True)]


def adamw_of(shapes, dtype, master, bits):
    """An optimiser whose first parameter begins two bytes behind an aligned address (float32: four)."""
    from memorax_b200 import blocks
    params, _ = adamw.make(shapes, dtype)
    params[0] = torch.cat((params[0][:1], params[0]))[1:]
    return blocks.AdamW(params, lr=adamw.RATE, betas=adamw.BETAS, eps=adamw.EPS, weight_decay=adamw.DECAY, state_bits=bits, master=master)


# A block takes 2048 elements a turn, as many turns as leave eight blocks an SM, sixteen at most; a tensor's last block has turns that its
# warps do not all take part in.
@pytest.mark.parametrize("turns", [2, 3, 4, 5, 16])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype,master", TYPES)
def test_adamw_turns(dtype, master, bits, turns):
    unit = 2048 * 1184 * turns // 8 // 2048 * 2048
    shapes = [(unit + 1,), (3 * unit + 255,), (2 * unit + 2047,), (2 * unit + 300,), (7,), (4097,), (2048 * turns,), (2048 * turns + 1,), (2048 * turns - 256,)]
    assert 2048 * 1184 * turns <= sum(math.prod(s) for s in shapes) < 2048 * 1184 * (turns + 1) or turns == 16
    opt = adamw_of(shapes, dtype, master, bits)
    for k in range(2):
        adamw.check_step(opt, adamw.make(shapes, dtype, seed=k + 1)[1])
    if dtype != torch.float32 and turns in (3, 16):
        adamw.check_step(opt, [g.float() for g in adamw.make(shapes, dtype, seed=5)[1]])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size", [5_000_001, 12_345_679, 40_000_000])
def test_adamw_8_bits_are_those_of_single_roundings(dtype, size):
    """``test_what_8_bits_hold_is_what_single_roundings_give`` over blocks of two, five and sixteen turns."""
    opt = adamw_of([(size,)], dtype, None, 8)
    m = v = torch.zeros(size, device="cuda")

    def hold(x, root):
        rows = torch.nn.functional.pad(x, (0, -x.numel() % 256)).view(-1, 256)
        top = rows.abs().amax(-1, keepdim=True)
        held = rows * (top.reciprocal() * 448.0)
        if root:
            held = torch.where(rows > 0, held.clamp_min(2.0 ** -9), held)
        return held.to(torch.float8_e4m3fn).flatten(), (top * (1.0 / 448.0)).flatten()

    for k in range(3):
        g = adamw.make([(size,)], dtype, seed=k)[1][0]
        opt.step([g])
        g = g.float()
        m = m * adamw.BETAS[0] + g * (1.0 - adamw.BETAS[0])
        v = v * adamw.BETAS[1] + g * (1.0 - adamw.BETAS[1]) * g
        for (codes, scales), (want, want_scales) in ((opt.m, hold(m, False)), (opt.v, hold(v.sqrt(), True))):
            assert torch.equal(scales, want_scales) and torch.equal(codes.view(torch.uint8), want.view(torch.uint8))
        (m,), (v,) = opt.moments()


# More tiles than the 1184 blocks of a launch with weights: a block's sums go on over several, the last of which is short; tiles that
# reach over sequences.
@pytest.mark.parametrize("b,t,hq,hk,d", [(8, 2048, 32, 8, 128), (8, 2048, 33, 1, 64), (8, 2047, 6, 6, 80), (1000, 37, 4, 2, 64), (5, 4001, 3, 1, 256)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rotation_of_several_tiles_a_block(b, t, hq, hk, d, dtype):
    q, k, w = make_rotate(b, t, hq, hk, d, dtype)
    g = torch.Generator(device="cuda").manual_seed(3)
    positions = torch.randint(0, 3000, (b, 1), device="cuda", generator=g) + torch.arange(t, device="cuda")
    check_rotate(q, k, d, positions, w)
    check_rotate(q, k, d // 2, positions, w, interleaved=True)


@pytest.mark.parametrize("d,rot", [(16, 16), (8, 4), (2, 2)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rotation_of_many_tokens_with_small_heads(d, rot, dtype):
    """The largest tiles there are: 512 tokens, whose angles and sums take all of the shared memory that a launch gets unasked."""
    q, k, w = make_rotate(3, 52001, 1, 1, d, dtype)
    check_rotate(q, k, rot, None, w)
    check_rotate(q, k, rot, None, (None, None), norm="l2", eps=1e-12)


# A warp a row with 32 entries at a time: from 5920 rows on, of more than 16384 bytes and at most 131072; blocks that walk the rows on either side.
@pytest.mark.parametrize("dtype,rows,vocab", [(torch.bfloat16, 5920, 8193), (torch.float16, 6001, 8200), (torch.float32, 5920, 4097), (torch.float32, 6001, 5003),
                                              (torch.bfloat16, 5919, 8193), (torch.bfloat16, 5921, 8192), (torch.float32, 5923, 4096), (torch.bfloat16, 5925, 20001)])
@pytest.mark.parametrize("masked", [False, True])
def test_many_long_rows(dtype, rows, vocab, masked):
    g = torch.Generator(device="cuda").manual_seed(rows + vocab)
    logits = (2 * torch.randn(rows, vocab, device="cuda", generator=g)).to(dtype)
    tokens = torch.randint(0, vocab, (rows,), device="cuda", generator=g)
    logits[11] = -math.inf
    logits[12, ::2] = -math.inf
    tokens[12], tokens[13], tokens[14] = 1, -1, vocab
    mask = None
    if masked:
        mask = torch.rand(rows, vocab, device="cuda", generator=g) < 0.6
        mask[torch.arange(rows, device="cuda"), tokens.clamp(0, vocab - 1)] = True
        mask[15] = False
        logits[16][~mask[16]] = math.nan
    check_logprobs(logits, tokens, mask)


@pytest.mark.parametrize("rows,vocab", [(5920, 32768), (5920, 32769)])
def test_rows_at_the_longest_of_a_warp(rows, vocab):
    """float32 rows of 131072 bytes, and of one entry more: the sums of a part of the rows against 64 bits."""
    from memorax_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(vocab)
    logits = 2 * torch.randn(rows, vocab, device="cuda", generator=g)
    tokens = torch.randint(0, vocab, (rows,), device="cuda", generator=g)
    got = ops.token_log_probs(logits, tokens)
    for at in (0, 2960, 5820):
        logs = logits[at:at + 100].double().log_softmax(-1)
        lp, h = logs.gather(-1, tokens[at:at + 100, None])[:, 0], -(logs.exp() * logs).sum(-1)
        unit = 2.0 ** -22 * (vocab / 512 + 32) * (1 + 10)          # as check_logprobs; distances to the largest are below ten on average
        assert bool(((got.log_prob[at:at + 100] - lp).abs() <= unit + 2.0 ** -21 * lp.abs()).all())
        assert bool(((got.entropy[at:at + 100] - h).abs() <= 2 * unit + 2.0 ** -20 * h).all())


def test_rows_apart_and_many():
    """The same from a wider buffer, whose rows begin at odd addresses."""
    g = torch.Generator(device="cuda").manual_seed(1)
    wide = torch.randn(5921, 8300, device="cuda", generator=g).bfloat16()
    tokens = torch.randint(0, 8201, (5921,), device="cuda", generator=g)
    check_logprobs(wide[:, 3:8204], tokens)
    mask = torch.rand(8201, device="cuda", generator=g) < 0.8
    mask[0] = True
    check_logprobs(wide[:, 5:8206], torch.zeros_like(tokens), mask)


# ---- tensors of more than 2^31 elements: what lies behind is as in a call of its own ----
def test_a_wide_table_and_many_rows():
    from memorax_b200 import ops
    vocab, dim = 2_100_001, 1024
    assert vocab * dim > 2 ** 31
    g = torch.Generator(device="cuda").manual_seed(1)
    ids = torch.randperm(vocab, device="cuda", generator=g)
    table = torch.randn(vocab, dim, device="cuda", generator=g, dtype=torch.bfloat16).requires_grad_()
    dy = torch.randn(vocab, dim, device="cuda", generator=g, dtype=torch.bfloat16)
    out = ops.embedding(ids, table, 3.0)
    (dw,) = torch.autograd.grad(out, table, dy)
    once = lambda x: (x.float() * 3.0).bfloat16()              # each token comes once: one product, rounded once
    back = torch.empty_like(ids)
    back[ids] = torch.arange(vocab, device="cuda")
    for at in (0, 2 ** 31 // dim - 50, vocab - 100):
        part = slice(at, at + 100)
        assert torch.equal(out[part], once(table.detach()[ids[part]])) and torch.equal(dw[part], once(dy[back[part]]))


def test_heads_behind_2_to_31_elements():
    from memorax_b200 import ops
    q = torch.randn(1, 530_000, 64, 64, device="cuda", dtype=torch.bfloat16)
    assert q.numel() > 2 ** 31
    k, plan = q[:, :, :1], ops.RotaryPlan(64)
    dys = [torch.randn(x.shape, device="cuda", dtype=torch.bfloat16) for x in (q, k)]

    def run(part):
        positions = torch.arange(530_000, device="cuda")[part]
        leaves = [x[:, part].detach().requires_grad_() for x in (q, k)]
        out = ops.norm_rotate(*leaves, plan, positions, norm="l2", eps=1e-12)
        return [*out, *torch.autograd.grad(out, leaves, [dy[:, part] for dy in dys])]

    whole = run(slice(None))
    for at in (0, 2 ** 31 // 4096 - 50, 529_900):
        for a, b in zip(whole, run(slice(at, at + 100))):
            assert torch.equal(a[:, at:at + 100], b)


@pytest.mark.parametrize("rows,vocab", [(45_000, 50_001), (2_200_001, 1000), (25_000_000, 100)])
def test_logits_behind_2_to_31_elements(rows, vocab):
    from memorax_b200 import ops
    assert rows * vocab > 2 ** 31
    logits = torch.randn(rows, vocab, device="cuda", dtype=torch.bfloat16).requires_grad_()
    tokens = torch.randint(0, vocab, (rows,), device="cuda")
    cot = torch.randn(2, rows, device="cuda")
    got = ops.token_log_probs(logits, tokens)
    (dx,) = torch.autograd.grad([got.log_prob, got.entropy], logits, list(cot))
    for at in (0, 2 ** 31 // vocab - 30, rows - 60):
        part = slice(at, at + 60)
        logs = logits.detach()[part].double().log_softmax(-1)
        p, one = logs.exp(), torch.nn.functional.one_hot(tokens[part], vocab)
        lp, h = (one * logs).sum(-1), -(p * logs).sum(-1)
        unit = 2.0 ** -22 * (vocab / 512 + 32) * (1 + 6)           # as check_logprobs
        assert bool(((got.log_prob[part] - lp).abs() <= unit + 2.0 ** -21 * lp.abs()).all())
        assert bool(((got.entropy[part] - h).abs() <= 2 * unit + 2.0 ** -20 * h).all())
        a, b = cot[0, part, None].double(), cot[1, part, None].double()
        want = a * (one - p) - b * p * (logs + h[:, None])
        size = a.abs() * (one + p) + b.abs() * p * (logs.abs() + h[:, None])
        assert bool(((dx[part] - want).abs() <= 2 * (unit + 2.0 ** -21 * logs.abs()) * size + 2.0 ** -8 * 1.01 * want.abs() + 2.0 ** -120).all())


@pytest.mark.parametrize("bits", [8, 32])
def test_a_parameter_behind_2_to_31_elements(bits):
    from memorax_b200 import blocks
    size = 2 ** 31 + 70_001
    g = torch.Generator(device="cuda").manual_seed(2)
    p = torch.randn(size, device="cuda", generator=g, dtype=torch.bfloat16)
    grad = torch.randn(size, device="cuda", generator=g, dtype=torch.bfloat16)
    parts = [slice(at, at + 69_632 if at else 100_096) for at in (0, 2 ** 31 - 2048, 2 ** 31 + 256)] + [slice(2 ** 31 + 65_536, size)]      # from multiples of 256 on
    alone = [p[part].clone() for part in parts]
    opts = [blocks.AdamW([x], lr=1e-2, state_bits=bits) for x in (p, *alone)]
    for _ in range(2):
        opts[0].step([grad])
        for opt, part in zip(opts[1:], parts):
            opt.step([grad[part]])
    for x, opt, part in zip(alone, opts[1:], parts):
        assert torch.equal(p[part], x)
        assert torch.equal(opts[0].moments()[0][0][part], opt.moments()[0][0]) if bits == 32 else torch.equal(opts[0].m[0].view(torch.uint8)[part], opt.m[0].view(torch.uint8)[:x.numel()])
