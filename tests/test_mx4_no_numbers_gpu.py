"""Units of 4-bit products on sums that are no numbers: such a sum leaves every unit as what it is, every other one as its
number, by every way that a product may take."""

import pytest
import torch

import plain_mx4 as plain
from mini_llm_stack_b200.ops.kernels import Runtime
from test_mx4_gpu import choices, gen, on_device, routed

pytestmark = pytest.mark.gpu
ALPHA, LIMIT = 1.702, 0.5


@pytest.fixture(scope="module")
def ops():
    return Runtime("cuda:0", torch.bfloat16).ops


# (rows, outputs, K): rows quantised in the product, by one block and by a cluster; few rows behind their quantisation; 64 and 192
# rows on a block; pairs by 192 and 256 weights, outputs at odd places among them.
SIZES = [(1, 40, 64), (3, 200, 700), (5, 16, 5000), (13, 70, 33000), (30, 200, 1100), (40, 200, 2300), (130, 1001, 300),
         (257, 2047, 2100), (257, 8192, 1100), (257, 4100, 2600), (257, 2048, 2100), (300, 2047, 4100), (200, 20000, 520),
         (400, 4100, 2100), (200, 8192, 2100), (700, 20000, 300), (2050, 6007, 520)]
KINDS = ["plain", "silu", "clamped", "relu2"]


def with_bad_blocks(x, places):
    """x with one value of each row that is named made no number; the rows."""
    for i, r in enumerate(places):
        x[r, (7 * r + 3) % x.shape[-1]] = (float("nan"), float("inf"), float("-inf"))[i % 3]
    return sorted(places)


@pytest.mark.parametrize("m, n, k", SIZES)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_products(ops, m, n, k, kind, dtype):
    g = torch.Generator("cuda").manual_seed(m + n + k)
    a = torch.randn(m, k, generator=g, device="cuda").to(dtype)
    w = (torch.randn(2, n, k, generator=g, device="cuda") * k ** -0.5).bfloat16()
    good, good_w = on_device(a), on_device(w)
    rows = with_bad_blocks(a, {0, m // 2, m - 1} if m > 1 else set())
    gate, up = {n // 3, n - 1}, {0, n // 2}                  # outputs whose gate's, or up's, weights are no numbers
    with_bad_blocks(w[0], gate)
    with_bad_blocks(w[1], up)
    paired = kind in ("silu", "clamped")
    out = torch.full((m, n), -7.0, dtype=dtype, device="cuda")
    if kind == "plain":
        ops.linear_mx4(a, ops.prepare_weight_mx4(w[0]), out)
    elif kind == "relu2":
        ops.linear_relu_squared_mx4(a, ops.prepare_weight_mx4(w[0]), out)
    else:
        ops.linear_glu_mx4(a, ops.prepare_weight_mx4(w, gate_up=True), out,
                           **(dict(alpha=ALPHA, limit=LIMIT) if kind == "clamped" else {}))
    ops.check_status()
    bad = torch.zeros(m, n, dtype=torch.bool, device="cuda")
    bad[rows] = True
    bad[:, sorted(gate | up if paired else gate)] = True
    assert torch.equal(out.isnan(), bad)
    want, off = plain.product(good, good_w[0])
    if kind == "relu2":
        z = want.clamp(min=0)
        want, off = z ** 2, (2 * z + off) * off + z ** 2 * plain.STEPS
    elif paired:
        other, off_other = plain.product(good, good_w[1])
        want, off = plain.unit(want, other, off, off_other, *((ALPHA, LIMIT) if kind == "clamped" else ()))
    far = (out.double() - want).abs() - off - plain.rounding(dtype, want)
    assert bool((far <= 0)[~bad].all()), float(far[~bad].max())


# tokens, experts, chosen, width in, width out: by blocks of 64 and of 192 rows, by pairs, tokens quantised once for all slots
EXPERTS = [(9, 4, 2, 96, 64), (70, 4, 2, 96, 72), (14000, 3, 1, 64, 1500), (900, 3, 2, 700, 3000), (1900, 4, 2, 1037, 301)]


@pytest.mark.parametrize("t, experts, top, d, f", EXPERTS)
@pytest.mark.parametrize("kind", ["silu", "clamped", "relu2"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("scale_in", [False, True])
def test_products_by_expert(ops, t, experts, top, d, f, kind, dtype, scale_in):
    g = gen("no numbers", t)
    idx = choices(t, experts, top, "even", g)
    work = routed(idx, torch.rand(t, top, generator=g) + 0.1, experts)
    h = torch.randn(t, d, generator=g).to(dtype)
    w = (torch.randn(experts, 2, f, d, generator=g) * d ** -0.5).bfloat16()
    tokens = with_bad_blocks(h, {1, t // 2, t - 1})
    gate, up = {f // 3, f - 1}, {0, f // 2}                  # of the last expert
    with_bad_blocks(w[-1, 0], gate)
    with_bad_blocks(w[-1, 1], up)
    y = torch.full((t * top, f), -7.0, dtype=dtype, device="cuda")
    if kind == "relu2":
        ops.expert_relu_squared_mx4(h.cuda(), ops.prepare_weight_mx4(w[:, 0].cuda()), y, work, top, scale_in)
    else:
        ops.expert_glu_mx4(h.cuda(), ops.prepare_weight_mx4(w.cuda(), gate_up=True), y, work, top, scale_in,
                           **(dict(alpha=ALPHA, limit=LIMIT) if kind == "clamped" else {}))
    ops.check_status()
    order = work["order"].cpu().long()
    bad = torch.zeros(t * top, f, dtype=torch.bool)
    bad[torch.isin(order // top, torch.tensor(tokens))] = True
    last = (idx.reshape(-1)[order] == experts - 1).nonzero()
    bad[last, torch.tensor(sorted(gate if kind == "relu2" else gate | up))] = True
    assert torch.equal(y.isnan().cpu(), bad)
