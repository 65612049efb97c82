"""Steps of the policy trainer that do not wait for the device."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("capturable", [False, True])
def test_a_step_waits_for_nothing_but_the_check_of_the_status(capturable):
    from memorax_b200 import blocks
    torch.manual_seed(0)
    net = blocks.TokenPolicyNet(37, 19, d_model=64, num_heads=1, head_dim=64, layers=1).cuda().bfloat16()
    trainer = blocks.TokenPolicyTrainer(net, check_every=5, lr=1e-2, capturable=capturable)
    batch = [torch.randint(0, n, (4, 33), device="cuda") for n in (37, 19)] + [torch.rand(4, 33, device="cuda") < 0.1, torch.randn(4, 33, device="cuda")]
    trainer.step(*batch)
    torch.cuda.set_sync_debug_mode("error")
    try:
        for _ in range(3):
            trainer.step(*batch)
    finally:
        torch.cuda.set_sync_debug_mode("default")
    trainer.step(*batch)                       # the fifth: checked
    assert trainer.optimiser.step_count == 5


def test_a_captured_step_is_the_eager_one():
    from memorax_b200 import blocks
    make = lambda: blocks.TokenPolicyNet(37, 19, d_model=64, num_heads=1, head_dim=64, layers=1).cuda().bfloat16()
    torch.manual_seed(0)
    nets = [make(), make()]
    nets[1].load_state_dict(nets[0].state_dict())
    eager, held = (blocks.TokenPolicyTrainer(net, check_every=1, lr=1e-2, capturable=True) for net in nets)
    batch = [torch.randint(0, n, (4, 33), device="cuda") for n in (37, 19)] + [torch.rand(4, 33, device="cuda") < 0.1, torch.randn(4, 33, device="cuda")]
    for _ in range(5):
        eager.step(*batch)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):              # a graph's first calls set kernels up
        for _ in range(2):
            held.step(*batch)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held.step(*batch)
    for _ in range(3):
        graph.replay()
    assert held.optimiser.step_count == eager.optimiser.step_count == 5
    for a, b in zip(nets[0].parameters(), nets[1].parameters()):
        assert torch.equal(a, b)
