"""Feed-forwards whose weights are held as 4-bit microscaled values: every part stage by stage against 64 bits, and whole
models through the engine."""

import pytest
import torch

import plain_llama as P
import plain_mx4 as plain
from engine_helpers import Replayer, make_folder, tokens_for
from mini_llm_stack_b200 import LLM
from mini_llm_stack_b200.config import EngineOptions, config_from_dict
from mini_llm_stack_b200.engine import runner
from mini_llm_stack_b200.ops.kernels import Runtime
from mini_llm_stack_b200.parts.feedforward import (ClampedGLUFeedForward, RoutedExperts, SquaredReluFeedForward,
                                                   SwiGLUFeedForward)
from tiny_configs import TINY_A, TINY_D
from tiny_zededra import Z_MIXED

pytestmark = pytest.mark.gpu
D, F = 200, 136


def bound(part, dtype, seed):
    rt = Runtime("cuda:0", dtype, "mxfp4")
    g = torch.Generator().manual_seed(seed)
    tensors = {n: (torch.randn(s.shape, generator=g) * (s.shape[-1] ** -0.5 if len(s.shape) > 1 else 0.1)).to(dtype).cuda()
               for n, s in part.tensor_specs().items()}
    part.bind(tensors, rt)
    return rt, {n: t.cpu() for n, t in tensors.items()}


def rows(t, dtype, seed):
    return torch.randn(t, D, generator=torch.Generator().manual_seed(seed)).to(dtype)


def close(got, want, off, dtype):
    far = (got.cpu().double() - want).abs() - off - plain.rounding(dtype, want)
    assert bool((far <= 0).all()), float(far.max())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("t", [1, 9, 70, 300])
@pytest.mark.parametrize("kind", ["swiglu", "clamped", "relu2", "relu2 with biases"])
def test_dense_feed_forwards(kind, t, dtype):
    part = {"swiglu": lambda: SwiGLUFeedForward(D, F), "clamped": lambda: ClampedGLUFeedForward(D, F, limit=0.7, alpha=1.3),
            "relu2": lambda: SquaredReluFeedForward(D, F),
            "relu2 with biases": lambda: SquaredReluFeedForward(D, F, biases=True)}[kind]()
    rt, w = bound(part, dtype, t)
    h = rows(t, dtype, t)
    out = part.forward(h.cuda(), None)
    rt.ops.check_status()
    act = rt.buffer("ffn_act", (t, F), dtype).cpu()
    q = plain.nearest
    if kind in ("swiglu", "clamped"):
        names = part.names
        g, u = plain.product(q(h), q(w[names[0]])), plain.product(q(h), q(w[names[1]]))
        want, off = plain.unit(g[0], u[0], g[1], u[1], *((1.3, 0.7) if kind == "clamped" else ()))
        down = w[names[2]]
    else:
        z, off = plain.product(q(h), q(w["up"]))
        if part.biases:
            out, b_down = out
            assert torch.equal(b_down.cpu(), w["down.b"])
            z, off = z + w["up.b"].double(), off + (z.abs() + 1) * plain.STEPS
        want, off = z.clamp(min=0) ** 2, (2 * z.clamp(min=0) + off) * off + z ** 2 * plain.STEPS
        down = w["down"]
    close(act, want, off, dtype)
    close(out, *plain.product(q(act), q(down)), dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("t", [1, 40, 330])
@pytest.mark.parametrize("unit, weigh, shared", [("gated", "input", False), ("gated", "output", True),
                                                 ("relu_squared", "output", False)])
def test_routed_experts(t, dtype, unit, weigh, shared):
    experts, top = 6, 2
    part = RoutedExperts(D, experts, top, F, shared=SwiGLUFeedForward(D, F, names=("gate", "up", "down")) if shared else None,
                         weigh=weigh, unit=unit, renormalise=True)
    rt, w = bound(part, dtype, t)
    h = rows(t, dtype, t + 1)
    delta = part.forward(h.cuda(), None).clone()
    rt.ops.check_status()
    n = t * top
    idx = rt.buffer("route_idx", (n,), torch.int32).cpu().long()
    order = rt.buffer("route_order", (n,), torch.int32).cpu().long()
    share = rt.buffer("route_weight", (n,), torch.float32).cpu().double()
    y, slots = rt.buffer("expert_act", (n, F), dtype).cpu(), rt.buffer("expert_out", (n, D), torch.float32).cpu()
    q = plain.nearest
    qh, qy = q(h), q(y)
    for e in range(experts):
        at = (idx[order] == e).nonzero()[:, 0]
        if not at.numel():
            continue
        slot = order[at]
        s_in = share[slot, None] if weigh == "input" else torch.ones((), dtype=torch.float64)
        s_out = share[slot, None] if weigh == "output" else torch.ones((), dtype=torch.float64)

        def sums(name):
            z, off = plain.product(qh[slot // top], q(w[f"e{e}.{name}"]))
            return z * s_in, (off + z.abs() * plain.STEPS) * s_in
        if unit == "gated":
            g, u = sums("gate"), sums("up")
            want, off = plain.unit(g[0], u[0], g[1], u[1])
        else:
            z, off = sums("up")
            want, off = z.clamp(min=0) ** 2, (2 * z.clamp(min=0) + off) * off + z ** 2 * plain.STEPS
        close(y[at], want, off, dtype)
        z, off = plain.product(qy[at], q(w[f"e{e}.down"]))
        close(slots[slot], z * s_out, (off + z.abs() * plain.STEPS) * s_out, torch.float32)
    want = slots.double().view(t, top, D).sum(1)
    size = slots.double().abs().view(t, top, D).sum(1)
    if shared:
        act = rt.buffer("ffn_act", (t, F), dtype).cpu()
        z, off = plain.product(q(act), q(w["shared.down"]))
        # the shared addend is rounded to the run's type before it is added
        want, size = want + z, size + off / plain.STEPS + plain.rounding(dtype, z) / plain.STEPS
    close(delta, want, size * plain.STEPS * 4, dtype)


def four_bit_swiglu(x, w_gate, w_up, w_down, rnd=P.ident):
    q = plain.nearest
    qx = q(x)
    g, u = qx @ q(w_gate).T, qx @ q(w_up).T
    act = (g * torch.sigmoid(g) * u).float()
    return (q(act) @ q(w_down).T).float()


@pytest.mark.parametrize("key", ["A", "D"])
def test_float32_logits(tmp_path, monkeypatch, key):
    """A whole model in float32 against the plain one with its feed-forwards in 4 bits, prompts cut in portions and decoded
    tokens among them.  Sums differ in their order, by parts of 2^-24, which moves a value over a border of the
    quantisation only where it lies that near to one: none of these does."""
    monkeypatch.setattr(P, "plain_swiglu", four_bit_swiglu)
    monkeypatch.setattr("engine_helpers.load_model", lambda folder, dtype: runner.load_model(folder, dtype, ffn_weights="mxfp4"))
    folder, cfg, w = make_folder(tmp_path, key, "float32")
    toks = {0: tokens_for(cfg["vocab_size"], 40, 1), 1: tokens_for(cfg["vocab_size"], 23, 2)}
    r = Replayer(folder, "float32", num_blocks=32)
    r.step([(0, 30), (1, 7)], toks)
    for _ in range(4):
        r.step([(0, 1), (1, 1)], toks)
    r.step([(0, 6), (1, 12)], toks)
    for rid in toks:
        want = P.plain_forward(w, cfg, toks[rid], P.ident)
        err = (r.logits(rid) - want).abs().max().item()
        assert err <= 5e-5 * want.abs().max().item(), (rid, err)


@pytest.mark.parametrize("raw", [TINY_A, TINY_D, Z_MIXED], ids=["dense", "dense wide", "experts"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_generation(raw, dtype):
    """Generation with 4-bit feed-forwards: the same tokens from graphs and without, and the option reaches the parts."""
    cfg = config_from_dict(dict(raw, dtype=dtype))
    prompts = [[5, 17, 3, 20, 41], list(range(1, 30))]
    opts = dict(ffn_weights="mxfp4", num_blocks=64)
    got = []
    for graphs in (True, False):
        llm = LLM.from_random(cfg, seed=11, dtype=dtype, options=EngineOptions(cuda_graphs=graphs, dtype=dtype, **opts))
        before = llm.model.runtime.ops.launches
        got.append(llm.generate(prompts, max_new_tokens=12))
        assert llm.model.runtime.ops.launches > before
        llm.model.runtime.ops.check_status()
    assert got[0] == got[1] and all(len(g) == 12 for g in got[0])
