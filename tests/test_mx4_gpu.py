"""4-bit microscaled rows and their products against 64 bits."""

import threading
import zlib

import pytest
import torch

import plain_mx4 as plain
from mini_llm_stack_b200.ops.kernels import KernelError, Mx4, Runtime

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    return Runtime("cuda:0", torch.bfloat16).ops


def gen(*key):
    return torch.Generator().manual_seed(zlib.crc32(repr(key).encode()))


def values(ops, q, dtype=torch.float32):
    out = torch.full(q.shape, -5.0, dtype=dtype, device="cuda")
    ops.mx4_values(q, out)
    return out.cpu()


def same(a, b):
    return torch.equal(torch.nan_to_num(a.double(), nan=12345.0), torch.nan_to_num(b.double(), nan=12345.0))


def wide_rows(rows, k, g):
    """Rows whose blocks' sizes spread over many powers of two, with zeros and ties among them."""
    x = torch.randn(rows, k, generator=g) * torch.exp2(torch.randint(-20, 20, (rows, k // 32 + 1), generator=g).float()
                                                       ).repeat_interleave(32, 1)[:, :k]
    x[torch.rand(rows, k, generator=g) < 0.1] = 0.0
    ties = torch.randint(-32, 33, (rows, k), generator=g).float() / 4
    return torch.where(torch.rand(rows, 1, generator=g) < 0.3, ties, x)


SHAPES = [(1, 1), (1, 31), (2, 32), (3, 33), (5, 64), (7, 255), (128, 256), (129, 257), (130, 96), (300, 1000), (1, 14336)]


@pytest.mark.parametrize("rows, k", SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_become_the_nearest_values(ops, rows, k, dtype):
    x = wide_rows(rows, k, gen(rows, k)).to(dtype)
    q = ops.quantize_mx4(x.cuda())
    assert q.shape == (rows, k)
    want = plain.nearest(x)
    for out in (torch.float32, torch.bfloat16):
        assert same(values(ops, q, out), want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_ends_of_the_range(ops, dtype):
    info = torch.finfo(dtype)
    sub = 2.0 ** -133 if dtype == torch.bfloat16 else 2.0 ** -149
    rows = [[sub] * 32, [0.0] * 32, [-0.0] * 32, [info.max] * 32, [-info.max, sub] * 16, [2.0 ** -127 * 1.25, 2.0 ** -128] * 16,
            [info.smallest_normal] * 32, [2.0 ** -124, 2.0 ** -127] * 16, [float("inf")] + [1.0] * 31,
            [1.0] * 31 + [float("-inf")], [float("nan")] + [0.0] * 31, [1.0] * 31 + [float("nan")]]
    x = torch.tensor(rows, dtype=torch.float64).to(dtype)
    x = torch.cat([x, torch.ones(len(rows), 32, dtype=dtype)], 1)       # the block beside is a number
    got = values(ops, ops.quantize_mx4(x.cuda()))
    assert same(got, plain.nearest(x))
    assert torch.equal(got[:, 32:], torch.ones(len(rows), 32))


def test_rows_between_addresses_and_with_strides(ops):
    g = gen("strides")
    for dtype in (torch.bfloat16, torch.float32):
        big = wide_rows(40, 500, g).to(dtype).cuda()
        for view in (big[:, :256], big[:, 1:258], big[::2, 8:264], big[3:9, 100:133]):
            assert same(values(ops, ops.quantize_mx4(view)), plain.nearest(view.cpu()))
    flat = wide_rows(1, 64 * 8 + 1, g).cuda()[0]
    assert same(values(ops, ops.quantize_mx4(flat[1:].view(8, 64))), plain.nearest(flat[1:].view(8, 64).cpu()))


def test_matrices_on_top_of_one_another(ops):
    x = wide_rows(2 * 3 * 150, 96, gen("mats")).view(2, 3, 150, 96)
    q = ops.quantize_mx4(x.cuda())
    assert q.codes.shape == (900, 48) and q.scales.shape == (12, 2, 512)
    assert same(values(ops, q), plain.nearest(x))
    y = wide_rows(900, 96, gen("mats", 2)).view(2, 3, 150, 96)
    assert ops.quantize_mx4(y.cuda(), into=q) is q and same(values(ops, q), plain.nearest(y))


def test_gate_and_up_lie_interleaved(ops):
    for n in (16, 40, 129):
        x = wide_rows(3 * 2 * n, 70, gen("pairs", n)).view(3, 2, n, 70)
        q = ops.quantize_mx4(x.cuda(), gate_up=True)
        full = -(-n // 16) * 32
        assert q.codes.shape == (3 * full, 48)
        assert same(values(ops, q), plain.nearest(x))
        plain_q = ops.quantize_mx4(x.cuda())
        up_5 = q.codes.view(3, full, 48)[2, 16 + 5]
        assert torch.equal(up_5, plain_q.codes.view(3, 2, n, 48)[2, 1, 5])


# ------------------------------------------------------------------------------------- products
DENSE = [(1, 1, 1), (1, 128, 64), (1, 16, 32), (2, 130, 96), (16, 128, 256), (17, 200, 257), (31, 129, 1000), (32, 127, 320),
         (33, 136, 512), (8, 384, 5000), (13, 70, 33000), (32, 260, 2100), (64, 140, 600), (97, 40, 160), (191, 128, 64), (193, 257, 288), (385, 130, 700), (1, 300, 4096), (700, 260, 100)]


def dense_inputs(m, n, k, mats, dtype=torch.bfloat16):
    g = gen(m, n, k, mats)
    a = (torch.randn(m, k, generator=g) * torch.exp(torch.randn(k, generator=g))).to(dtype)
    w = (torch.randn(mats, n, k, generator=g) * k ** -0.5).bfloat16()
    return a, w


def near(got, want, off, dtype):
    got = got.cpu().double()
    far = (got - want).abs() - off - plain.rounding(dtype, want)
    assert got.shape == want.shape and bool((far <= 0).all()), float(far.max())


@pytest.mark.parametrize("m, n, k", DENSE)
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
def test_product(ops, m, n, k, out_dtype):
    a, w = dense_inputs(m, n, k, 1)
    out = torch.full((m, n), float("nan"), dtype=out_dtype, device="cuda")
    ops.linear_mx4(a.cuda(), ops.prepare_weight_mx4(w[0].cuda()), out)
    ops.check_status()
    want = plain.product(plain.nearest(a), plain.nearest(w[0]))
    near(out, *want, out_dtype)
    # rows that are 4-bit values already
    out.fill_(float("nan"))
    ops.linear_mx4(ops.quantize_mx4(a.cuda()), ops.prepare_weight_mx4(w[0].cuda()), out)
    ops.check_status()
    near(out, *want, out_dtype)


@pytest.mark.parametrize("m, n, k", DENSE)
@pytest.mark.parametrize("kind", ["silu", "clamped", "relu2"])
def test_product_with_a_unit(ops, m, n, k, kind):
    dtype = torch.float32 if (m + n + k) % 2 else torch.bfloat16
    a, w = dense_inputs(m, n, k, 1 if kind == "relu2" else 2, dtype)
    out = torch.full((m, n), float("nan"), dtype=dtype, device="cuda")
    qa, qw = plain.nearest(a), plain.nearest(w)
    if kind == "relu2":
        ops.linear_relu_squared_mx4(a.cuda(), ops.prepare_weight_mx4(w[0].cuda()), out)
        z, off = plain.product(qa, qw[0])
        want, off = z.clamp(min=0) ** 2, (2 * z.clamp(min=0) + off) * off + z ** 2 * plain.STEPS
    else:
        alpha, limit = (1.702, 0.5) if kind == "clamped" else (1.0, 0.0)
        ops.linear_glu_mx4(a.cuda(), ops.prepare_weight_mx4(w.cuda(), gate_up=True), out, alpha=alpha, limit=limit)
        g, u = plain.product(qa, qw[0]), plain.product(qa, qw[1])
        want, off = plain.unit(g[0], u[0], g[1], u[1], alpha, limit)
    ops.check_status()
    near(out, want, off, dtype)


# ------------------------------------------------------------------------------------- by expert
def routed(idx, weight, outputs):
    """The arrays of a step in which token t takes the outputs idx[t]."""
    flat = idx.reshape(-1)
    order = torch.sort(flat, stable=True).indices
    offsets = torch.searchsorted(flat[order], torch.arange(outputs + 1))
    return {"idx": flat.int().cuda(), "order": order.int().cuda(), "offsets": offsets.int().cuda(),
            "weight": weight.reshape(-1).cuda()}


def choices(t, outputs, top, spread, g):
    if spread == "one":                      # every token's first choice is the same expert
        idx = torch.stack([torch.randperm(outputs - 1, generator=g)[:top] + 1 for _ in range(t)])
        idx[:, 0] = 0
        return idx
    return torch.stack([torch.randperm(outputs, generator=g)[:top] for _ in range(t)])


EXPERTS = [  # tokens, experts, outputs without weights, top, d, f, spread
    (1, 3, 0, 1, 64, 16, "even"), (16, 4, 0, 1, 72, 40, "one"), (17, 4, 1, 2, 136, 128, "one"),
    (33, 5, 0, 2, 65, 131, "one"), (65, 9, 0, 2, 257, 136, "one"), (40, 2, 0, 1, 200, 129, "even"),
    (129, 3, 0, 2, 64, 96, "one"), (127, 2, 0, 2, 320, 264, "even"), (257, 3, 1, 2, 128, 72, "one"),
    (600, 4, 0, 1, 64, 130, "even"), (515, 2, 0, 1, 256, 384, "one"), (70, 300, 0, 3, 64, 32, "even"),
    (30, 1500, 3, 2, 40, 24, "even"), (2100, 5, 1, 3, 2900, 72, "one")]


@pytest.mark.parametrize("t, experts, identity, top, d, f, spread", EXPERTS)
@pytest.mark.parametrize("kind", ["silu", "clamped", "relu2"])
def test_products_by_expert(ops, t, experts, identity, top, d, f, spread, kind):
    g = gen(t, experts, kind)
    outputs = experts + identity
    idx = choices(t, outputs, top, spread, g)
    weight = torch.rand(t, top, generator=g) + 0.1
    work = routed(idx, weight, outputs)
    dtype = torch.float32 if kind == "clamped" else torch.bfloat16
    h = torch.randn(t, d, generator=g).to(dtype)
    w1 = (torch.randn(experts, 1 if kind == "relu2" else 2, f, d, generator=g) * d ** -0.5).bfloat16()
    w2 = (torch.randn(experts, d, f, generator=g) * f ** -0.5).bfloat16()
    n = t * top
    y = torch.full((n, f), 77.0, dtype=dtype, device="cuda")
    out = torch.full((n, d), 77.0, device="cuda")
    scale_in = kind == "silu"
    if kind == "relu2":
        ops.expert_relu_squared_mx4(h.cuda(), ops.prepare_weight_mx4(w1[:, 0].cuda()), y, work, top, scale_in)
    else:
        alpha, limit = (1.702, 0.5) if kind == "clamped" else (1.0, 0.0)
        ops.expert_glu_mx4(h.cuda(), ops.prepare_weight_mx4(w1.cuda(), gate_up=True), y, work, top, scale_in, alpha=alpha,
                           limit=limit)
    ops.expert_down_mx4(y, ops.prepare_weight_mx4(w2.cuda()), out, work, top, not scale_in)
    ops.check_status()
    order, flat, share = work["order"].cpu().long(), idx.reshape(-1), weight.reshape(-1).double()
    y, out = y.cpu(), out.cpu()
    qh, qy = plain.nearest(h), plain.nearest(y)
    for e in range(outputs):
        at = (flat[order] == e).nonzero()[:, 0]
        slot = order[at]
        if e >= experts:
            assert bool((y[at] == 77.0).all()) and bool((out[slot] == 77.0).all())    # nobody's: left as they were
            continue
        if at.numel() == 0:
            continue
        qw = plain.nearest(w1[e])
        s = share[slot, None] if scale_in else torch.ones((), dtype=torch.float64)
        sums = [plain.product(qh[slot // top], m) for m in qw]
        sums = [(z * s, (off + z.abs() * plain.STEPS) * s) for z, off in sums]
        if kind == "relu2":
            z, off = sums[0]
            want, off = z.clamp(min=0) ** 2, (2 * z.clamp(min=0) + off) * off + z ** 2 * plain.STEPS
        else:
            want, off = plain.unit(sums[0][0], sums[1][0], sums[0][1], sums[1][1], alpha, limit)
        near(y[at], want, off, dtype)
        z, off = plain.product(qy[at], plain.nearest(w2[e]))
        s = torch.ones((), dtype=torch.float64) if scale_in else share[slot, None]
        near(out[slot], z * s, (off + z.abs() * plain.STEPS) * s, torch.float32)


# ------------------------------------------------------------------------------------- more than one round of tiles
def on_device(x):
    """nearest() on the device: scales by frexp, which is exact."""
    k = x.shape[-1]
    v = torch.nn.functional.pad(x.double(), (0, -k % 32)).unflatten(-1, (-1, 32))
    top = v.abs().amax(-1, keepdim=True)
    scale = torch.ldexp(torch.ones_like(top), (torch.frexp(top).exponent - 3).clamp(min=-127))
    v = v / torch.where(top > 0, scale, 1.0)
    step = torch.where(v.abs() < 2, 0.5, torch.where(v.abs() < 4, 1.0, 2.0).double())
    return ((torch.round(v / step) * step).clamp(-6, 6) * torch.where(top > 0, scale, 1.0)).flatten(-2)[..., :k]


@pytest.mark.parametrize("m, n, k", [(65, 40000, 300), (150, 20500, 520), (260, 19000, 1100), (300, 15000, 300), (700, 9100, 700),
                                     (1500, 3000, 3300), (2050, 4100, 2600), (513, 700, 9000), (20000, 130, 300)])
@pytest.mark.parametrize("gated", [False, True])
def test_many_tiles(ops, m, n, k, gated):
    g = torch.Generator("cuda").manual_seed(m + n + k)
    a = torch.randn(m, k, generator=g, device="cuda").bfloat16()
    w = (torch.randn(2 if gated else 1, n, k, generator=g, device="cuda") * k ** -0.5).bfloat16()
    out = torch.full((m, n), float("nan"), dtype=torch.bfloat16, device="cuda")
    if gated:
        ops.linear_glu_mx4(a, ops.prepare_weight_mx4(w, gate_up=True), out)
    else:
        ops.linear_mx4(a, ops.prepare_weight_mx4(w[0]), out)
    ops.check_status()
    qa, qw = on_device(a), on_device(w)
    z, off = plain.product(qa, qw[0])
    if gated:
        z, off = plain.unit(z, plain.product(qa, qw[1])[0], off, plain.product(qa, qw[1])[1])
    far = (out.double() - z).abs() - off - plain.rounding(torch.bfloat16, z)
    assert bool((far <= 0).all()), float(far.max())


@pytest.mark.parametrize("t, experts, top, d, f", [(1200, 12, 4, 1100, 1000), (900, 3, 2, 700, 3000), (64, 60, 6, 1030, 600)])
def test_many_tiles_by_expert(ops, t, experts, top, d, f):
    g = torch.Generator("cuda").manual_seed(t)
    h = torch.randn(t, d, generator=g, device="cuda").bfloat16()
    w1 = (torch.randn(experts, 2, f, d, generator=g, device="cuda") * d ** -0.5).bfloat16()
    w2 = (torch.randn(experts, d, f, generator=g, device="cuda") * f ** -0.5).bfloat16()
    liked = torch.randn(t, experts, generator=g, device="cuda") + 2 * torch.randn(experts, generator=g, device="cuda")
    idx = liked.topk(top).indices
    work = routed(idx.cpu(), torch.softmax(torch.randn(t, top, generator=g, device="cuda"), 1).cpu(), experts)
    y = torch.full((t * top, f), float("nan"), dtype=torch.bfloat16, device="cuda")
    out = torch.full((t * top, d), float("nan"), device="cuda")
    ops.expert_glu_mx4(h, ops.prepare_weight_mx4(w1, gate_up=True), y, work, top, False)
    ops.expert_down_mx4(y, ops.prepare_weight_mx4(w2), out, work, top, True)
    ops.check_status()
    order, share = work["order"].long(), work["weight"].double()
    qh, qy, flat = on_device(h), on_device(y), idx.reshape(-1)
    for e in range(experts):
        at = (flat[order] == e).nonzero()[:, 0]
        if at.numel() == 0:
            continue
        slot, qw = order[at], on_device(w1[e])
        gate, up = (plain.product(qh[slot // top], m) for m in qw)
        want, off = plain.unit(gate[0], up[0], gate[1], up[1])
        assert bool(((y[at].double() - want).abs() <= off + plain.rounding(torch.bfloat16, want)).all()), e
        want, off = plain.product(qy[at], on_device(w2[e]))
        s = share[slot, None]
        far = (out[slot].double() - want * s).abs() - (off + want.abs() * plain.STEPS) * s - plain.rounding(torch.float32, want * s)
        assert bool((far <= 0).all()), (e, float(far.max()))


# ------------------------------------------------------------------------------------- what is no number
@pytest.mark.parametrize("m, n, k", [(3, 200, 300), (20, 200, 300), (40, 200, 2300), (100, 300, 300), (300, 300, 600),
                                     (600, 2100, 300)])
def test_what_is_no_number_stays_in_its_row(ops, m, n, k):
    a, w = dense_inputs(m, n, k, 1)
    want, off = plain.product(plain.nearest(a), plain.nearest(w[0]))
    bad_rows = {0: float("nan"), m // 2: float("inf"), m - 1: float("-inf")}
    for r, v in bad_rows.items():
        a[r, (7 * r) % k] = v
    w[0, n // 3, k - 1] = float("inf")
    out = torch.empty((m, n), dtype=torch.bfloat16, device="cuda")
    ops.linear_mx4(a.cuda(), ops.prepare_weight_mx4(w[0].cuda()), out)
    ops.check_status()
    out = out.cpu()
    bad = torch.zeros(m, n, dtype=torch.bool)
    bad[list(bad_rows)] = True
    bad[:, n // 3] = True
    assert bool(out[bad].isnan().all())
    assert bool(((out.double() - want).abs() <= off + plain.rounding(torch.bfloat16, want))[~bad].all())


def test_what_is_no_number_stays_with_its_slots(ops):
    t, experts, top, d, f = 70, 4, 2, 96, 64
    g = gen("nan experts")
    idx = choices(t, experts, top, "one", g)
    work = routed(idx, torch.ones(t, top), experts)
    h = torch.randn(t, d, generator=g).bfloat16()
    h[5, 90] = float("nan")
    w = (torch.randn(experts, 2, f, d, generator=g) * d ** -0.5).bfloat16()
    w[2, 0, 0, 0] = float("nan")
    y = torch.zeros((t * top, f), dtype=torch.bfloat16, device="cuda")
    ops.expert_glu_mx4(h.cuda(), ops.prepare_weight_mx4(w.cuda(), gate_up=True), y, work, top, False)
    order = work["order"].cpu().long()
    bad = torch.zeros(t * top, f, dtype=torch.bool)
    bad[order // top == 5] = True
    bad[idx.reshape(-1)[order] == 2, 0] = True
    assert torch.equal(y.isnan().cpu(), bad)


# ------------------------------------------------------------------------------------- how calls may be made
def test_empty_calls_and_edges(ops):
    w = ops.prepare_weight_mx4(torch.randn(40, 64, device="cuda"))
    ops.linear_mx4(torch.empty(0, 64, device="cuda"), w, torch.empty(0, 40, device="cuda"))
    q = ops.quantize_mx4(torch.empty(0, 64, device="cuda"))
    assert q.shape == (0, 64) and q.codes.shape == (0, 32)
    ops.mx4_values(q, torch.empty(0, 64, device="cuda"))
    pairs = ops.prepare_weight_mx4(torch.randn(2, 2, 24, 64, device="cuda"), gate_up=True)
    work = routed(torch.empty(0, 1, dtype=torch.long), torch.empty(0, 1), 2)
    ops.expert_glu_mx4(torch.empty(0, 64, device="cuda"), pairs, torch.empty(0, 24, device="cuda"), work, 1, False)
    ops.check_status()


@pytest.mark.parametrize("m", [1, 12, 40, 150, 400])
def test_nothing_beside_the_output_is_written(ops, m):
    n, k = 330, 700
    a, w = dense_inputs(m, n, k, 2)
    room = torch.full((m + 4, n), 9.0, dtype=torch.bfloat16, device="cuda")
    ops.linear_mx4(a.cuda(), ops.prepare_weight_mx4(w[0].cuda()), room[2:-2])
    ops.linear_glu_mx4(a.cuda(), ops.prepare_weight_mx4(w.cuda(), gate_up=True), room[2:-2])
    ops.check_status()
    assert bool((room[:2] == 9).all()) and bool((room[-2:] == 9).all()) and not bool((room[2:-2] == 9).all())


@pytest.mark.parametrize("m", [1, 8, 12, 40, 100, 300, 900])
def test_the_same_bits_each_time_and_on_another_stream(ops, m):
    a, w = dense_inputs(m, 1000, 2100, 1)
    a, held = a.cuda(), ops.prepare_weight_mx4(w[0].cuda())
    outs = []
    side = torch.cuda.Stream()
    for stream in (torch.cuda.current_stream(), torch.cuda.current_stream(), side):
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            out = torch.full((m, 1000), float("nan"), device="cuda")
            ops.linear_mx4(a, held, out)
        torch.cuda.current_stream().wait_stream(stream)
        outs.append(out)
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


def test_rows_with_a_stride(ops):
    for m in (5, 30, 200):
        big = torch.randn(m, 900, generator=gen("stride", m)).bfloat16().cuda()
        w = ops.prepare_weight_mx4(torch.randn(72, 300, generator=gen("w")).bfloat16().cuda())
        for view in (big[:, 8:308], big[:, 301:601], big[:, ::1][:, 600:]):
            out, want = torch.empty(m, 72, device="cuda"), torch.empty(m, 72, device="cuda")
            ops.linear_mx4(view, w, out)
            ops.linear_mx4(view.contiguous(), w, want)
            assert torch.equal(out, want)


def test_graphs_keep_their_memory(ops):
    """Captured calls, replayed behind calls that need more scratch memory, and on other inputs."""
    own = Runtime("cuda:0", torch.bfloat16).ops
    g = gen("graph")
    cases = []
    for m, n, k in ((6, 300, 600), (50, 300, 600), (400, 300, 600)):
        a = torch.randn(m, k, generator=g).bfloat16().cuda()
        w = own.prepare_weight_mx4(torch.randn(n, k, generator=g).bfloat16().cuda())
        cases.append((a, w, torch.empty(m, n, device="cuda")))
    t, experts, top = 90, 5, 2
    idx = choices(t, experts, top, "even", g)
    work = routed(idx, torch.ones(t, top), experts)
    h = torch.randn(t, 200, generator=g).bfloat16().cuda()
    w1 = own.prepare_weight_mx4(torch.randn(experts, 2, 64, 200, generator=g).bfloat16().cuda(), gate_up=True)
    y = torch.empty(t * top, 64, dtype=torch.bfloat16, device="cuda")

    def run():
        for a, w, out in cases:
            own.linear_mx4(a, w, out)
        own.expert_glu_mx4(h, w1, y, work, top, False)

    run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    big = torch.randn(3000, 4096, device="cuda").bfloat16()
    wide = own.prepare_weight_mx4(torch.randn(64, 4096, device="cuda"))
    own.linear_mx4(big, wide, torch.empty(3000, 64, device="cuda"))      # the scratch memory moves
    for a, _, _ in cases:
        a.copy_(torch.randn(a.shape, generator=g).bfloat16())
    h.copy_(torch.randn(h.shape, generator=g).bfloat16())
    filled = [torch.full((1 << 20,), 0xff, dtype=torch.uint8, device="cuda") for _ in range(64)]
    graph.replay()
    got = [out.clone() for _, _, out in cases] + [y.clone()]
    run()
    torch.cuda.synchronize()
    for a, b in zip(got, [out for _, _, out in cases] + [y]):
        assert torch.equal(a, b)
    assert all(bool((f == 0xff).all()) for f in filled)


def test_weights_written_anew_are_waited_for(ops):
    """A product right behind the quantisation of its weights, where kernels start under their predecessors."""
    g = gen("anew")
    a = torch.randn(4, 2048, generator=g).bfloat16().cuda()
    first, second = (torch.randn(4096, 2048, generator=g).bfloat16().cuda() for _ in range(2))
    out, want = torch.empty(4, 4096, device="cuda"), torch.empty(4, 4096, device="cuda")
    ops.linear_mx4(a, ops.prepare_weight_mx4(second), want)
    held = ops.prepare_weight_mx4(first)
    for _ in range(20):
        ops.quantize_mx4(first, into=held)
        ops.quantize_mx4(second, into=held)
        ops.linear_mx4(a, held, out)
    assert torch.equal(out, want)


def test_refusals(ops):
    w = ops.prepare_weight_mx4(torch.randn(40, 64, device="cuda"))
    a, out = torch.randn(3, 64, device="cuda"), torch.empty(3, 40, device="cuda")
    both = torch.zeros(400, device="cuda")
    for call in (lambda: ops.linear_mx4(a.cpu(), w, out), lambda: ops.linear_mx4(a, w, out.cpu()),
                 lambda: ops.linear_mx4(both[:192].view(3, 64), w, both[100:220].view(3, 40)),
                 lambda: ops.quantize_mx4(a.cpu()), lambda: ops.mx4_values(w, torch.empty(40, 64)),
                 lambda: ops.linear_mx4(ops.quantize_mx4(torch.randn(2, 3, 64, device="cuda")), w, out)):
        with pytest.raises(KernelError):
            call()
    ops.linear_mx4(a, w, out)
    ops.check_status()


# ------------------------------------------------------------------------------------- places beyond 32 bits
def test_many_rows_are_quantised(ops):
    """More than 2^32 values and 2^31 bytes of codes: repeated rows, whose codes repeat."""
    k, once, times = 4096, 4096, 270
    part = wide_rows(once, k, gen("many")).bfloat16().cuda()
    x = part.expand(times, once, k).reshape(times * once, k)
    assert x.numel() > 1 << 32
    few, many = ops.quantize_mx4(part), ops.quantize_mx4(x)
    assert many.codes.numel() > 1 << 31
    assert bool((many.codes.view(times, -1) == few.codes.view(1, -1)).all())
    assert bool((many.scales.view(times, -1) == few.scales.view(1, -1)).all())
    want = torch.empty_like(part)
    ops.mx4_values(few, want)
    x.fill_(-5.0)
    ops.mx4_values(many, x)
    assert bool((x.view(times, once, k) == want).all())


@pytest.mark.parametrize("gated", [False, True])
def test_large_outputs(ops, gated):
    """An output of more than 2^32 values: rows from its start, its middle and its end."""
    m, n, k = 70000, 62000, 64
    g = gen("large", gated)
    a = torch.randn(m, k, generator=g).bfloat16()
    w = torch.randn(2, n, k, generator=g).bfloat16()
    out = torch.empty(m, n, dtype=torch.bfloat16, device="cuda")
    if gated:
        ops.linear_glu_mx4(a.cuda(), ops.prepare_weight_mx4(w.cuda(), gate_up=True), out)
    else:
        ops.linear_mx4(a.cuda(), ops.prepare_weight_mx4(w[0].cuda()), out)
    ops.check_status()
    rows = torch.tensor([0, 1, 34999, 35000, 69887, 69888, 69998, 69999])
    assert out.numel() > 1 << 32
    qa, qw = plain.nearest(a[rows]), on_device(w.cuda()).cpu()
    want, off = plain.product(qa, qw[0])
    if gated:
        up, off_up = plain.product(qa, qw[1])
        want, off = plain.unit(want, up, off, off_up)
    near(out[rows.cuda()].cpu(), want, off, torch.bfloat16)


def test_large_outputs_by_expert(ops):
    """Slots' rows of more than 2^32 values, and every token's choices twice the same expert."""
    t, top, experts, d, f = 140000, 2, 3, 16384, 64
    g = gen("large experts")
    idx = torch.randint(0, experts, (t, 1), generator=g).expand(t, top).contiguous()
    weight = torch.rand(t, top, generator=g) + 0.1
    work = routed(idx, weight, experts)
    y = torch.randn(t * top, f, generator=g).bfloat16()
    w = torch.randn(experts, d, f, generator=g).bfloat16()
    out = torch.empty(t * top, d, device="cuda")
    assert out.numel() > 1 << 32
    ops.expert_down_mx4(y.cuda(), ops.prepare_weight_mx4(w.cuda()), out, work, top, True)
    ops.check_status()
    order, flat, share = work["order"].cpu().long(), idx.reshape(-1), weight.reshape(-1).double()
    qw = on_device(w.cuda()).cpu()
    for p in (0, 1, 100000, 140000, 200000, t * top - 2, t * top - 1):
        slot = int(order[p])
        z, off = plain.product(plain.nearest(y[p:p + 1]), qw[flat[slot]])
        near(out[slot:slot + 1].cpu(), z * share[slot], (off + z.abs() * plain.STEPS) * share[slot], torch.float32)


def test_two_models_at_once(ops):
    """Calls of two runtimes on two streams, few rows, many rows and routed ones side by side."""
    g = gen("two")
    other = Runtime("cuda:0", torch.bfloat16).ops
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    jobs = []
    for own in (ops, other):
        w = own.prepare_weight_mx4((torch.randn(3000, 2100, generator=g) * 0.1).bfloat16().cuda())
        pair = own.prepare_weight_mx4((torch.randn(2, 2100, 3000, generator=g) * 0.1).bfloat16().cuda(), gate_up=True)
        calls = []
        for m in (1, 9, 40, 300, 1100):
            a = torch.randn(m, 2100, generator=g).bfloat16().cuda()
            calls.append((own, w, pair, a, torch.empty(m, 3000, dtype=torch.bfloat16, device="cuda"),
                          torch.empty(m, 2100, device="cuda")))
        jobs.append(calls)

    def run(call):
        own, w, pair, a, mid, out = call
        own.linear_mx4(a, w, mid)
        own.linear_glu_mx4(mid, pair, out)

    want = []
    for calls in jobs:
        for call in calls:
            run(call)
        want.append([call[5].clone() for call in calls])
    torch.cuda.synchronize()
    for call in sum(jobs, []):
        call[5].fill_(-1.0)
    torch.cuda.synchronize()
    for _ in range(20):
        for i in range(len(jobs[0])):
            for calls, stream in zip(jobs, streams):
                with torch.cuda.stream(stream):
                    run(calls[i])
    torch.cuda.synchronize()
    for calls, results in zip(jobs, want):
        for call, result in zip(calls, results):
            assert torch.equal(call[5], result)
    ops.check_status()
    other.check_status()


@pytest.mark.parametrize("kind", ["silu", "relu2"])
def test_more_choices_than_lanes(ops, kind):
    """Tokens that are quantised once for 36 slots each."""
    assert 600 * 36 * 2 >= ops.MX4_ONCE
    test_products_by_expert(ops, 600, 40, 2, 36, 300, 48, "even", kind)


def test_streams_and_graphs_have_their_own_scratch(ops):
    """One runtime's products on two streams and out of two graphs, all at once."""
    g = gen("scratch")
    w = ops.prepare_weight_mx4((torch.randn(4000, 2100, generator=g) * 0.1).bfloat16().cuda())
    experts, top, t = 6, 2, 700
    w1 = ops.prepare_weight_mx4(torch.randn(experts, 2, 200, 2100, generator=g).bfloat16().cuda(), gate_up=True)
    jobs = []
    for i in range(4):
        idx = choices(t, experts, top, "even", g)
        jobs.append((torch.randn(t, 2100, generator=g).bfloat16().cuda(), torch.empty(t, 4000, device="cuda"),
                     routed(idx, torch.ones(t, top), experts), torch.empty(t * top, 200, dtype=torch.bfloat16, device="cuda")))

    def run(job):
        a, out, work, y = job
        ops.linear_mx4(a, w, out)
        ops.expert_glu_mx4(a, w1, y, work, top, False)

    want = []
    for job in jobs:
        run(job)
        want.append((job[1].clone(), job[3].clone()))
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for graph, job in zip(graphs, jobs):
        with torch.cuda.graph(graph):
            run(job)
    streams = [torch.cuda.Stream() for _ in range(4)]
    for job in jobs:
        job[1].fill_(-1.0)
        job[3].fill_(-1.0)
    torch.cuda.synchronize()
    for _ in range(15):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                if i < 2:
                    graphs[i].replay()
                else:
                    run(jobs[i])
    torch.cuda.synchronize()
    for job, (out, y) in zip(jobs, want):
        assert torch.equal(job[1], out) and torch.equal(job[3], y)
    ops.check_status()


# ------------------------------------------------------------------------------------- rows that suit no wide access
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows, k", [(1, 1), (3, 7), (1, 17), (2, 31), (5, 97), (9, 511), (4, 513), (130, 1003), (33, 2049), (700, 333)])
@pytest.mark.parametrize("before", [0, 1, 3, 6])
def test_rows_at_any_address(ops, rows, k, dtype, before):
    """Matrices that begin and end anywhere, among values that are no numbers; back into memory of which nothing else changes."""
    g = gen("anywhere", rows, k)
    x = wide_rows(rows, k, g).to(dtype).cuda()
    ld = k + 2
    buf = torch.full((before + rows * ld + 40,), float("nan"), dtype=dtype, device="cuda")
    strided = buf[before:before + rows * ld].view(rows, ld)[:, :k]
    strided.copy_(x)
    close = torch.full((before + rows * k + 40,), float("nan"), dtype=dtype, device="cuda")
    dense = close[before:before + rows * k].view(rows, k)
    dense.copy_(x)
    want = torch.empty((rows, k), dtype=torch.float32, device="cuda")
    ops.mx4_values(ops.quantize_mx4(x.clone()), want)
    assert same(want.cpu(), plain.nearest(x.cpu()))
    back = torch.full_like(close, -7.0)
    for m in (strided, dense):
        q = ops.quantize_mx4(m)
        into = back[before:before + rows * k].view(rows, k)
        into.fill_(-7.0)
        ops.mx4_values(q, into)
        assert torch.equal(into.float(), want)
        assert bool((back[:before] == -7.0).all()) and bool((back[before + rows * k:] == -7.0).all())
    for m in (1, 5, 16):                                 # and on the way into a product
        if rows >= m:
            w = ops.prepare_weight_mx4(torch.randn(40, k, generator=g).cuda())
            out, same_out = torch.empty(m, 40, device="cuda"), torch.empty(m, 40, device="cuda")
            ops.linear_mx4(strided[:m], w, out)
            ops.linear_mx4(x[:m].clone(), w, same_out)
            assert torch.equal(out, same_out)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["plain", "silu", "relu2"])
@pytest.mark.parametrize("m, n, k", [(700, 1501, 300), (1300, 2047, 520), (515, 3013, 1100), (2050, 777, 64)])
def test_outputs_that_begin_anywhere(ops, m, n, k, kind, dtype):
    """Rows of outputs at no 32-byte places, in tiles of many rows; nothing behind them is written."""
    g = gen("outputs", m, n, k)
    a = torch.randn(m, k, generator=g).bfloat16()
    w = (torch.randn(2, n, k, generator=g) * k ** -0.5).bfloat16()
    buf = torch.full((m * n + 64,), -7.0, dtype=dtype, device="cuda")
    out = buf[3:3 + m * n].view(m, n)
    if kind == "silu":
        ops.linear_glu_mx4(a.cuda(), ops.prepare_weight_mx4(w.cuda(), gate_up=True), out)
    elif kind == "relu2":
        ops.linear_relu_squared_mx4(a.cuda(), ops.prepare_weight_mx4(w[0].cuda()), out)
    else:
        ops.linear_mx4(a.cuda(), ops.prepare_weight_mx4(w[0].cuda()), out)
    ops.check_status()
    assert bool((buf[:3] == -7.0).all()) and bool((buf[3 + m * n:] == -7.0).all())
    qa, qw = on_device(a.cuda()), on_device(w.cuda())
    want, off = plain.product(qa, qw[0])
    if kind == "silu":
        up, off_up = plain.product(qa, qw[1])
        want, off = plain.unit(want, up, off, off_up)
    elif kind == "relu2":
        z = want.clamp(min=0)
        want, off = z ** 2, (2 * z + off) * off + z ** 2 * plain.STEPS
    near(out.cpu(), want.cpu(), off.cpu(), dtype)


@pytest.mark.parametrize("kind", ["silu", "relu2"])
def test_outputs_that_begin_anywhere_by_expert(ops, kind):
    test_products_by_expert(ops, 1900, 4, 1, 2, 1037, 301, "even", kind)


def test_one_column(ops):
    """Matrices [rows, 1] with any stride of their one column."""
    g = gen("one column")
    for dtype in (torch.bfloat16, torch.float32):
        x, w = torch.randn(1, 70, generator=g).to(dtype).cuda().t(), torch.randn(1, 33, generator=g).to(dtype).cuda().t()
        assert x.stride() == (1, 70)
        assert same(values(ops, ops.quantize_mx4(x)), plain.nearest(x.cpu()))
        for m in (70, 5):
            out = torch.full((m, 33), float("nan"), device="cuda")
            ops.linear_mx4(x[:m], ops.prepare_weight_mx4(w), out)
            assert torch.equal(out.cpu().double(), plain.nearest(x[:m].cpu()) @ plain.nearest(w.cpu()).T)   # one exact product each
    ops.check_status()


def test_two_threads_on_one_stream(ops):
    """Products whose rows are quantised in scratch memory of the stream, called by two threads at once; one of them
    asks for more and more of it."""
    own = Runtime("cuda:0", torch.bfloat16).ops
    g = gen("threads")
    w = own.prepare_weight_mx4((torch.randn(300, 2100, generator=g) * 0.1).bfloat16().cuda())
    w1 = own.prepare_weight_mx4(torch.randn(4, 72, 2100, generator=g).bfloat16().cuda())
    jobs = []
    for sizes in (range(70, 1500, 130), range(1400, 60, -130)):
        calls = []
        for m in sizes:
            a = torch.randn(m, 2100, generator=g).bfloat16().cuda()
            work = routed(choices(m, 4, 1, "even", g), torch.ones(m, 1), 4)
            calls.append((a, work, torch.empty(m, 300, device="cuda"), torch.empty(m, 72, device="cuda")))
        jobs.append(calls)

    def run(calls):
        for a, work, out, y in calls:
            own.linear_mx4(a, w, out)
            own.expert_relu_squared_mx4(a, w1, y, work, 1, False)

    for calls in jobs:
        run(calls)
    want = [[(out.clone(), y.clone()) for _, _, out, y in calls] for calls in jobs]
    for _, _, out, y in sum(jobs, []):
        out.fill_(-1.0)
        y.fill_(-1.0)
    own._mx4_rows.clear()
    threads = [threading.Thread(target=lambda c=calls: [run(c) for _ in range(5)]) for calls in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for calls, results in zip(jobs, want):
        for (_, _, out, y), (out_want, y_want) in zip(calls, results):
            assert torch.equal(out, out_want) and torch.equal(y, y_want)
    own.check_status()


@pytest.mark.parametrize("m", [1, 12, 60, 300])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_the_longest_rows(ops, m, dtype):
    """K as long as it may be, from its first value to its last."""
    n, k = 130, ops.MX4_MOST_K
    g = torch.Generator("cuda").manual_seed(m)
    a = torch.randn(m, k, generator=g, device="cuda").to(dtype)
    w = (torch.randn(n, k, generator=g, device="cuda") * k ** -0.5).bfloat16()
    q = ops.quantize_mx4(a)
    back = torch.empty_like(a)
    ops.mx4_values(q, back)
    assert torch.equal(back.double(), on_device(a))
    held = ops.prepare_weight_mx4(w)
    want, off = plain.product(on_device(a), on_device(w))
    for rows in (a, q):
        out = torch.full((m, n), float("nan"), device="cuda")
        ops.linear_mx4(rows, held, out)
        ops.check_status()
        far = (out.double() - want).abs() - off - plain.rounding(torch.float32, want)
        assert bool((far <= 0).all()), float(far.max())
