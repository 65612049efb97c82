"""Calls whose kernels follow each other without a pause.  A call of small tensors is usually waited for by its own host code, so that each
kernel finds the ones in front finished; here they are queued behind one that takes some milliseconds, and each is resident before its
predecessor has written.  Two inputs in turn, so that what one call reads too early is another one's; the results are those of calls
that were waited for, bit for bit."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def rn(*shape, dtype=torch.float32, grad=False, scale=1.0):
    return (scale * torch.randn(*shape, device="cuda")).to(dtype).requires_grad_(grad)


def layer(make, bsz, steps, feat, dtype=torch.float32):
    from memorax_b200.memoroid import Memoroid
    model = Memoroid(make()).cuda().to(dtype)
    params = list(model.parameters())

    def inputs():
        return rn(bsz, steps, feat, dtype=dtype, grad=True), torch.rand(bsz, steps, device="cuda") < 0.05, rn(bsz, steps, feat, dtype=dtype)

    def call(x, done, gy):
        carry, y = model(x, done, None)
        return [y, *carry, *torch.autograd.grad(y, [x, *params], gy, allow_unused=True)]
    return inputs, call


def mamba(shape):
    from memorax_b200.memoroid import MambaCell
    bsz, steps, feat, heads = shape
    return layer(lambda: MambaCell(feat, num_heads=heads), bsz, steps, feat)


def product(m, n, k):
    from memorax_b200 import _C
    return lambda: (rn(m, k), rn(n, k), rn(n)), lambda x, w, b: [_C.linear_f32(x, w, b)]


def network():
    """A policy's update over tokens: embedding, rotated delta rule, log probabilities, AdamW."""
    from memorax_b200.blocks import AdamW, TokenPolicyNet
    torch.manual_seed(1)
    net = TokenPolicyNet(50, 18, d_model=64, num_heads=1, head_dim=64, layers=2).cuda().bfloat16()
    start = [p.detach().clone() for p in net.parameters()]

    def inputs():
        return torch.randint(0, 50, (3, 40), device="cuda"), torch.randint(0, 18, (3, 40), device="cuda"), torch.rand(3, 40, device="cuda") < 0.05, rn(3, 40)

    def call(observations, actions, done, advantage):
        with torch.no_grad():
            for p, s in zip(net.parameters(), start):
                p.copy_(s)
        adamw = AdamW(net.parameters(), lr=1e-2)
        for _ in range(2):
            adamw.zero_grad()
            _, policy = net(observations, done, actions=actions)
            (-(advantage * policy.log_prob).mean() - 0.01 * policy.entropy.mean()).backward()
            adamw.step()
        return [policy.log_prob.detach(), *(p.detach().clone() for p in net.parameters()), *(x.clone() for x in adamw.moments()[0])]
    return inputs, call


def cases():
    from memorax_b200 import memoroid as m
    bf = torch.bfloat16
    return {
        "mamba 16 heads": lambda: mamba((2, 17, 8, 16)), "mamba 17 heads": lambda: mamba((2, 17, 8, 17)), "mamba 2 heads": lambda: mamba((2, 65, 33, 2)),
        "lru": lambda: layer(lambda: m.LRUCell(48, 300), 3, 33, 48), "mingru": lambda: layer(lambda: m.MinGRUCell(64), 3, 33, 64),
        "linattn": lambda: layer(lambda: m.LinearAttentionCell(64, 64, 2), 2, 70, 64, bf),
        "deltanet": lambda: layer(lambda: m.DeltaNetCell(64, 64, 2), 2, 70, 64, bf),
        "mlstm": lambda: layer(lambda: m.mLSTMCell(64, 64, num_heads=2, tensor_cores=True), 2, 35, 64, bf),
        "long product": lambda: product(34, 8, 1040), "longer product": lambda: product(130, 300, 2100), "short product": lambda: product(34, 256, 8),
        "network": network,
    }


@pytest.mark.parametrize("name", ["mamba 16 heads", "mamba 17 heads", "mamba 2 heads", "lru", "mingru", "linattn", "deltanet", "mlstm", "long product",
                                  "longer product", "short product", "network"])
def test_kernels_behind_one_another(name):
    from memorax_b200 import ops
    torch.manual_seed(0)
    inputs, call = cases()[name]()
    given = [inputs() for _ in range(2)]
    held = lambda outs: [x.detach().clone() for x in outs if x is not None]
    want = []
    for args in given:
        torch.cuda.synchronize()
        want.append(held(call(*args)))
    torch.cuda.synchronize()
    for _ in range(12):
        got = []
        torch.cuda._sleep(8_000_000)                          # about four milliseconds
        for i in range(6):
            got.append((i % 2, held(call(*given[i % 2]))))
        ops.check_status()
        for i, outs in got:
            for at, (x, w) in enumerate(zip(outs, want[i], strict=True)):
                assert torch.equal(x, w), (name, at, float((x.double() - w.double()).abs().max()))


# few rows against a long contraction: four parts of 64 columns, added up by a launch of their own.  The bound is that of
# test_gemm32_f16_gpu.py: 2^-20 for eight truncating additions, 2^-21 for the small products and the float32 sums of the parts.
@pytest.mark.parametrize("m,n,k", [(34, 8, 1040), (34, 8, 1105), (3, 64, 1025), (128, 20, 4000)])
def test_products_in_parts(m, n, k):
    from memorax_b200 import _C, ops
    torch.manual_seed(k)
    x, w, b = rn(m, k), rn(n, k), rn(n)
    got = _C.linear_f32(x, w, b)
    ops.check_status()
    want, scale = x.double() @ w.double().t() + b.double(), x.abs().double() @ w.abs().double().t() + b.abs().double()
    assert bool(((got.double() - want).abs() <= (2.0 ** -20 + 2.0 ** -21) * scale).all())
