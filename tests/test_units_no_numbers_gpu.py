"""The units with a limit and the square of relu on sums that are no numbers, in 16 and 32 bits: a comparison does not turn what
is no number into one."""

import pytest
import torch

from mini_llm_stack_b200.ops.kernels import Runtime
from test_experts_tc_gpu import routed

pytestmark = pytest.mark.gpu
ALPHA, LIMIT = 1.702, 7.0
NAN = float("nan")


@pytest.fixture(scope="module")
def ops():
    o = Runtime("cuda:0", torch.bfloat16).ops
    o.require_part("experts")
    return o


def inputs(m, n, k, mats, dtype):
    g = torch.Generator("cuda").manual_seed(m + n)
    a = torch.randn(m, k, generator=g, device="cuda").to(dtype)
    w = (torch.randn(mats, n, k, generator=g, device="cuda") * k ** -0.5).to(dtype)
    a[m - 1, 3] = NAN
    w[0, n // 3, 5] = NAN
    bad = torch.zeros(m, n, dtype=torch.bool, device="cuda")
    bad[m - 1] = True
    bad[:, n // 3] = True
    if mats == 2:
        w[1, n // 2, 7] = NAN
        bad[:, n // 2] = True
    return a, w, bad


@pytest.mark.parametrize("m", [1, 8, 40, 130, 700])
@pytest.mark.parametrize("n, k", [(256, 512), (2048, 4096)])
def test_products_in_16_bits(ops, m, n, k):
    a, w, bad = inputs(m, n, k, 2, torch.bfloat16)
    out = torch.full((m, n), -7.0, dtype=torch.bfloat16, device="cuda")
    ops.linear_clamped_glu(a, ops.interleave_gate_up(w[0], w[1]), out, ALPHA, LIMIT)
    assert torch.equal(out.isnan(), bad)
    a, w, bad = inputs(m, n, k, 1, torch.bfloat16)
    for bias in (None, torch.zeros(n, dtype=torch.bfloat16, device="cuda")):
        ops.linear_relu_squared(a, w[0], out, bias=bias)
        assert torch.equal(out.isnan(), bad)
    ops.check_status()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_element_by_element(ops, dtype):
    z = torch.tensor([[-2.0, 3.0, NAN, 0.0, NAN, 9.0, float("inf"), 1.0]], device="cuda").to(dtype)
    out = torch.empty_like(z)
    ops.relu_squared(z, out)
    assert out.tolist()[0][:2] == [0.0, 9.0] and out.isnan().tolist() == z.isnan().tolist() and out[0, 6].isinf()
    act = torch.empty(1, 4, dtype=dtype, device="cuda")
    ops.clamped_glu(z, act, ALPHA, LIMIT)
    assert act.isnan().tolist() == [[True, False, True, False]]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("t, experts, d, f", [(5, 3, 64, 48), (90, 4, 256, 136), (700, 4, 256, 384), (30, 3, 65, 33)])
@pytest.mark.parametrize("kind", ["clamped", "relu2"])
def test_products_by_expert(ops, t, experts, d, f, kind, dtype):
    g = torch.Generator("cuda").manual_seed(t)
    order_of = torch.Generator().manual_seed(t)
    chosen = torch.stack([torch.randperm(experts, generator=order_of)[:2] for _ in range(t)])
    work = routed(ops, chosen, torch.ones(t, 2), experts, experts)
    idx, order = work["idx"][:t * 2].long(), work["order"][:t * 2].long()
    h = torch.randn(t, d, generator=g, device="cuda").to(dtype)
    w = (torch.randn(experts, 2, f, d, generator=g, device="cuda") * d ** -0.5).to(dtype)
    h[t // 2, 3] = NAN
    w[1, 0, f // 3, 5] = NAN
    w[1, 1, f // 2, 5] = NAN
    y = torch.full((t * 2, f), -7.0, dtype=dtype, device="cuda")
    if kind == "relu2":
        ops.expert_relu_squared(h, w[:, 0].contiguous(), y, work, 2, False)
    else:
        ops.expert_glu(h, w.flatten(1, 2).contiguous(), y, work, 2, False, alpha=ALPHA, limit=LIMIT)
    ops.check_status()
    bad = torch.zeros(t * 2, f, dtype=torch.bool, device="cuda")
    bad[order // 2 == t // 2] = True
    bad[idx[order] == 1, f // 3] = True
    if kind == "clamped":
        bad[idx[order] == 1, f // 2] = True
    assert torch.equal(y.isnan(), bad)
