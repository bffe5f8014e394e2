"""GPU tests of what lies around the decoder operators' kernels: the streams and memory of the objects they read, their
workspaces, and autograd's book of what was written."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF, F32 = torch.bfloat16, torch.float32


@pytest.fixture()
def ops(pkg):
    return pkg.decoder_attn


def rand(shape, dtype, seed, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * std).to(dtype).to(DEV)


def test_plan_dropped_before_its_kernel_has_run(ops):
    """A plan and a rotation made on one stream, used on another that is still busy, and dropped: what the first stream
    allocates then is other memory."""
    q, k, w = rand((70, 8, 64), BF, 1), rand((70, 2, 64), BF, 2), torch.ones(64, device=DEV)
    pos = torch.arange(70, dtype=torch.int32, device=DEV)
    make = lambda: (ops.CausalPlan([70], num_heads=8, num_kv_heads=2, head_dim=64, dtype=BF, device=DEV),
                    ops.TextRotary(64, 1e4, (12, 10, 10), True, DEV))
    call = lambda plan, rot: (ops.causal_attention(q, k, k, plan), *ops.qk_norm_rotary(q, k, None, w, w, pos, rot)[:2])
    want = call(*make())
    torch.cuda.synchronize()
    plan, rot = make()
    sizes = plan.items.shape, rot.table.shape
    at = plan.items.data_ptr(), rot.table.data_ptr()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(100_000_000)                            # some 50 ms
        got = call(plan, rot)
    del plan, rot
    taken = [torch.zeros(sizes[0], dtype=torch.int32, device=DEV) for _ in range(8)]
    taken += [torch.zeros(sizes[1], dtype=torch.int64, device=DEV) for _ in range(8)]
    assert not {t.data_ptr() for t in taken} & set(at)
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)
