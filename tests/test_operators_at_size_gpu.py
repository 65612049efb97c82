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
