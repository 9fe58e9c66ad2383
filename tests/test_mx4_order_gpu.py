"""Float32 outputs of 4-bit products: a row's bits do not depend on the rows that it is multiplied beside, nor on its place among
them, so that a float32 run's tokens do not depend on the batch, on how a prompt is cut, or on a recomputation."""

import pytest
import torch
from safetensors.torch import load_file, save_file

from engine_helpers import Replayer, make_folder, tokens_for
from mini_llm_stack_b200.engine import runner
from mini_llm_stack_b200.ops.kernels import Runtime
from test_mx4_gpu import choices, gen, routed

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    return Runtime("cuda:0", torch.float32).ops


def spread(*shape, std=1.0, seed):
    """Values whose blocks of 32 differ by many powers of two: their products' sums are not exact in 24 bits, whatever the order."""
    g = torch.Generator("cuda").manual_seed(seed)
    blocks = -(-shape[-1] // 32)
    size = torch.exp2(torch.randint(-9, 10, (*shape[:-1], blocks), generator=g, device="cuda").float())
    return torch.randn(*shape, generator=g, device="cuda") * std * size.repeat_interleave(32, -1)[..., :shape[-1]]


def same_bits(a, b):
    return torch.equal(a.view(torch.int32), b.view(torch.int32))


# outputs, K: of one slice and of many, within and beyond what a product quantises itself, outputs at odd places
@pytest.mark.parametrize("n, k", [(40, 64), (200, 700), (1001, 2300), (2048, 5000), (16, 33000), (4100, 2600), (20000, 520),
                                  (8192, 2100), (4096, 14336)])
@pytest.mark.parametrize("kind", ["plain", "silu", "clamped", "relu2"])
def test_products(ops, n, k, kind):
    most = 2050 if n * k < 1 << 25 else 700
    a, w = spread(most, k, seed=n + k), spread(2, n, k, std=0.01, seed=n + k + 1)
    held = ops.prepare_weight_mx4(w if kind in ("silu", "clamped") else w[0], gate_up=kind in ("silu", "clamped"))

    def product(rows):
        out = torch.full((rows.shape[0], n), -7.0, device="cuda")
        if kind == "plain":
            ops.linear_mx4(rows, held, out)
        elif kind == "relu2":
            ops.linear_relu_squared_mx4(rows, held, out)
        else:
            ops.linear_glu_mx4(rows, held, out, **(dict(alpha=1.702, limit=0.5) if kind == "clamped" else {}))
        return out

    whole = product(a)
    for r0, m in [(0, 1), (77, 1), (3, 2), (0, 8), (5, 9), (64, 16), (1, 17), (0, 32), (130, 33), (200, 64), (0, 65), (100, 130),
                  (64, 257), (300, 400), (0, 699), (0, 1100), (550, 1500)]:
        if r0 + m <= most:
            assert same_bits(product(a[r0:r0 + m]), whole[r0:r0 + m]), (r0, m)
            if kind == "plain":
                out = torch.full((m, n), -7.0, device="cuda")
                ops.linear_mx4(ops.quantize_mx4(a[r0:r0 + m]), held, out)
                assert same_bits(out, whole[r0:r0 + m]), (r0, m, "quantised before")
    ops.check_status()


@pytest.mark.parametrize("experts, top, d, f", [(4, 2, 96, 72), (3, 2, 700, 3000), (4, 2, 1037, 301), (12, 4, 1100, 1000)])
@pytest.mark.parametrize("kind", ["silu", "clamped", "relu2"])
def test_products_by_expert(ops, experts, top, d, f, kind):
    g = gen("order", experts, d)
    most = 1900
    idx, weight = choices(most, experts, top, "even", g), torch.rand(most, top, generator=g) + 0.1
    h, w1 = spread(most, d, seed=d), spread(experts, 2, f, d, std=0.01, seed=d + 1)
    w2 = ops.prepare_weight_mx4(spread(experts, d, f, std=0.01, seed=d + 2))
    up = ops.prepare_weight_mx4(w1 if kind != "relu2" else w1[:, 0], gate_up=kind != "relu2")

    def products(t0, t):
        work = routed(idx[t0:t0 + t], weight[t0:t0 + t], experts)
        y, out = torch.full((t * top, f), -7.0, device="cuda"), torch.full((t * top, d), -7.0, device="cuda")
        if kind == "relu2":
            ops.expert_relu_squared_mx4(h[t0:t0 + t], up, y, work, top, True)
        else:
            ops.expert_glu_mx4(h[t0:t0 + t], up, y, work, top, kind == "clamped",
                               **(dict(alpha=1.702, limit=0.5) if kind == "clamped" else {}))
        ops.expert_down_mx4(y, w2, out, work, top, kind == "silu")
        return y[torch.argsort(work["order"])], out                  # by slot

    whole = products(0, most)
    for t0, t in [(0, 1), (9, 3), (0, 16), (100, 70), (3, 400), (300, 1000)]:
        for got, want in zip(products(t0, t), whole):
            assert same_bits(got, want[t0 * top:(t0 + t) * top]), (t0, t)
    ops.check_status()


@pytest.mark.parametrize("key", ["A", "D", "E"])
def test_cutting_does_not_change_bits(tmp_path, monkeypatch, key):
    """A float32 model with its feed-forwards in 4 bits: whole prompts, portions of them and decoded tokens."""
    monkeypatch.setattr("engine_helpers.load_model", lambda folder, dtype: runner.load_model(folder, dtype, ffn_weights="mxfp4"))
    folder, cfg, _ = make_folder(tmp_path, key, "float32", patch={"intermediate_size": 1408})
    weights = load_file(str(folder / "model.safetensors"))
    for i, name in enumerate(sorted(weights)):
        if "w_gate" in name or "w_up" in name or "w_down" in name:
            weights[name] = spread(*weights[name].shape, std=0.01, seed=i).cpu()
    save_file(weights, str(folder / "model.safetensors"))
    n = 140
    toks = {"r": tokens_for(cfg["vocab_size"], n, 9)}
    logits = []
    for steps in ([n], [50, 2, 37, 1, 1, 1, 48], [1] * 20 + [17, 16, 87]):
        r = Replayer(folder, "float32", num_blocks=16)
        for s in steps:
            r.step([("r", s)], toks)
        logits.append(r.logits("r"))
    assert same_bits(logits[0], logits[1]) and same_bits(logits[0], logits[2])
