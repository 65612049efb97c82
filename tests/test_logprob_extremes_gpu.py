"""Log probabilities and their gradients at temperatures and cotangents near the ends of what is allowed."""
import math

import pytest
import torch
from test_tokens_gpu import check_logprobs

pytestmark = pytest.mark.gpu


# rows held in registers, by vectors, and by single entries (odd lengths in float32 do not lie alike)
@pytest.mark.parametrize("vocab", [18, 100, 1024, 4003])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("temperature", [1e-30, 1e-20, 1e-9, 1e-4, 1e10, 1e27])
def test_temperatures(vocab, dtype, temperature):
    """Cold rows are ties or one token; a place at -inf, or whose exponential is zero, has no gradient."""
    g = torch.Generator(device="cuda").manual_seed(vocab)
    logits = (3 * torch.randn(9, vocab, device="cuda", generator=g)).to(dtype)
    tokens = torch.randint(0, vocab, (9,), device="cuda", generator=g)
    tokens[:4] = logits[:4].float().argmax(-1)
    logits[1, ::3], logits[5, 1::2] = -math.inf, -math.inf
    logits[2, :5] = logits[2].max()
    logits[6] = torch.finfo(dtype).min
    logits[7] = logits[7, 0]
    tokens[1], tokens[5] = 1, 2
    tokens[8] = -1
    check_logprobs(logits, tokens, None, temperature)
    mask = torch.rand(9, vocab, device="cuda", generator=g) < 0.6
    mask[torch.arange(8, device="cuda"), tokens[:8]] = True
    mask[3] = False
    check_logprobs(logits, tokens, mask, temperature)


@pytest.mark.parametrize("vocab", [18, 1024, 4003])
@pytest.mark.parametrize("size", [1e9, 1e30])
def test_cotangents_beyond_the_numbers_when_divided(vocab, size):
    """A row of one token has no gradient, whatever its cotangents; where two share it, it is as large as it is."""
    from memorax_b200 import ops
    logits = torch.randn(3, vocab, device="cuda").requires_grad_()
    with torch.no_grad():
        logits[:, 4] = 20.0
        logits[1, 9] = 20.0
        logits[2, 5:9] = -math.inf
    out = ops.token_log_probs(logits, torch.tensor([4, 4, 4], device="cuda"), temperature=1e-30)
    (d,) = torch.autograd.grad((out.log_prob, out.entropy), logits, (torch.full((3,), size, device="cuda"), torch.full((3,), size, device="cuda")))
    want = torch.zeros(3, vocab, device="cuda")
    want[1, 4], want[1, 9] = math.inf, -math.inf               # (1 - 1/2) size / T, beyond float32
    assert torch.equal(d, want)
