"""4-bit microscaled rows: sizes in memory, what is refused before anything reaches a device, the engine's option."""

import copy
import pickle
import threading
import time

import pytest
import torch

from mini_llm_stack_b200.config import ConfigError, EngineOptions
from mini_llm_stack_b200.ops.kernels import KernelError, Mx4, Ops


@pytest.fixture
def ops():
    """The checks of the kernels' owner without a device: tensors of the CPU pass for its own."""
    o = Ops.__new__(Ops)
    o.device, o._device_index, o.sm_count, o.launches, o._part_libs = torch.device("cpu"), -1, 148, 0, {}

    def here(what, *tensors):
        assert all(isinstance(t, torch.Tensor) for t in tensors)

    def part(name):
        raise AssertionError("a kernel was asked for")

    o._mx4_here, o._part_lib = here, part
    return o


def test_sizes_in_memory():
    q = Mx4((3, 130, 70), "cpu")
    assert q.codes.shape == (390, 48) and q.scales.shape == (6, 2, 512) and q.lead == 1
    pair = Mx4((4, 2, 20, 300), "cpu", gate_up=True)
    assert pair.codes.shape == (4 * 64, 160) and pair.scales.shape == (4, 4, 512) and pair.lead == 1
    assert not pair.data.any()                       # 20 rows fill up to 32 a matrix: what fills up is zero
    assert Mx4((1, 1), "cpu").codes.shape == (1, 16)
    assert pair.codes_at % 16 == 0 and (pair.codes_at - pair.scales_at) % 1024 == 0


@pytest.mark.parametrize("n, k", [(1, 1), (130, 4096), (4096, 14336), (28672, 4096), (36000, 300), (40000, 300), (128256, 4096),
                                  (256, 1 << 20)])
def test_slices_are_eight_at_most_and_resident_at_once(n, k):
    steps, tiles = -(-k // 256), -(-n // 128)
    s = Mx4((n, k), "meta" if n * k > 1 << 24 else "cpu").few_rows_slice(148)
    if s == 0:
        assert tiles > 281
    else:
        slices = -(-steps // s)
        assert 1 <= slices <= 8 and tiles * slices <= 281 and (slices - 1) * s < steps


def test_rows_that_are_refused(ops):
    bad = [torch.zeros(3), torch.zeros(3, 4, dtype=torch.float16), torch.zeros(3, 0), torch.zeros(3, 4, dtype=torch.int32),
           torch.zeros(4, 8).t(), torch.zeros(4, 6, 8)[:, ::2], torch.zeros(8).expand(3, 8), torch.empty(1, (1 << 20) + 1, device="meta"),
           torch.zeros(1).expand((1 << 28) + 1, 1)]
    for x in bad:
        with pytest.raises(KernelError):
            ops.quantize_mx4(x)
    with pytest.raises(KernelError):
        ops.quantize_mx4(torch.zeros(3, 4, 8), gate_up=True)
    with pytest.raises(KernelError):
        ops.quantize_mx4(torch.zeros(1).expand(1 << 24, 2, 1, 1), gate_up=True)
    for into in (Mx4((3, 4), "cpu"), Mx4((2, 4, 8), "cpu"), torch.zeros(2, 4, 8)):
        with pytest.raises(KernelError):
            ops.quantize_mx4(torch.zeros(2, 4, 8), into=into, gate_up=True)
    q = Mx4((3, 64), "cpu")
    for out in (torch.zeros(3, 63), torch.zeros(64, 3).t(), torch.zeros(3, 64, dtype=torch.float16)):
        with pytest.raises(KernelError):
            ops.mx4_values(q, out)
    with pytest.raises(KernelError):
        ops.mx4_values(torch.zeros(3, 64), torch.zeros(3, 64))


def test_products_that_are_refused(ops):
    w, pair = Mx4((40, 64), "cpu"), Mx4((2, 40, 64), "cpu", gate_up=True)
    a, out = torch.zeros(3, 64), torch.zeros(3, 40)
    for call in (lambda: ops.linear_mx4(a, torch.zeros(40, 64), out), lambda: ops.linear_mx4(a, pair, out),
                 lambda: ops.linear_glu_mx4(a, w, out), lambda: ops.linear_mx4(a, Mx4((1, 40, 64), "cpu"), out),
                 lambda: ops.linear_mx4(a[:, :63], w, out), lambda: ops.linear_mx4(a, w, out[:2]),
                 lambda: ops.linear_mx4(a, w, torch.zeros(40, 3).t()), lambda: ops.linear_mx4(a.half(), w, out),
                 lambda: ops.linear_mx4(a, w, out.half()), lambda: ops.linear_mx4(torch.zeros(64, 3).t(), w, out),
                 lambda: ops.linear_mx4(torch.zeros(()), w, out), lambda: ops.linear_mx4(a[0], w, out),
                 lambda: ops.linear_relu_squared_mx4(a, pair, out),
                 lambda: ops.linear_mx4(torch.zeros(1).expand((1 << 28) + 1, 1), Mx4((1, 1), "cpu"),
                                        torch.zeros(1).expand((1 << 28) + 1, 1))):
        with pytest.raises(KernelError):
            call()
    room = torch.zeros(1000)
    with pytest.raises(KernelError, match="where the rows are"):
        ops.linear_mx4(room[:192].view(3, 64), w, room[191:311].view(3, 40))
    ops.linear_mx4(a[:0], w, out[:0])                # nothing to do: no kernel


def test_products_by_expert_that_are_refused(ops):
    w1, w2 = Mx4((2, 2, 40, 64), "cpu", gate_up=True), Mx4((2, 64, 40), "cpu")
    h, y, slots = torch.zeros(3, 64), torch.zeros(6, 40), torch.zeros(6, 64)
    i32 = dict(dtype=torch.int32)
    work = {"order": torch.zeros(6, **i32), "idx": torch.zeros(6, **i32), "offsets": torch.zeros(3, **i32), "weight": torch.zeros(6)}
    for call in (lambda: ops.expert_glu_mx4(h, w2, y, work, 2, False), lambda: ops.expert_down_mx4(y, w1, slots, work, 2, True),
                 lambda: ops.expert_glu_mx4(h, w1, y, work, 3, False), lambda: ops.expert_glu_mx4(h, w1, y, work, 0, False),
                 lambda: ops.expert_glu_mx4(h, w1, y[:, :39], work, 2, False),
                 lambda: ops.expert_down_mx4(y, w2, slots.bfloat16(), work, 2, True),
                 lambda: ops.expert_down_mx4(y[:5], w2, slots, work, 2, True),
                 lambda: ops.expert_glu_mx4(h, w1, y, dict(work, offsets=work["offsets"][:2]), 2, False),
                 lambda: ops.expert_glu_mx4(h, w1, y, dict(work, order=work["order"].long()), 2, False),
                 lambda: ops.expert_glu_mx4(h, w1, y, dict(work, idx=work["idx"][:5]), 2, False),
                 lambda: ops.expert_glu_mx4(h, w1, y, dict(work, weight=work["weight"].double()), 2, False),
                 lambda: ops.expert_relu_squared_mx4(h, w1, y, work, 2, False)):
        with pytest.raises(KernelError):
            call()


def test_the_engines_option():
    assert EngineOptions().ffn_weights is None
    opts = EngineOptions(ffn_weights="mxfp4", device="cpu")
    opts.check_against("bfloat16", "cpu", "mxfp4")
    with pytest.raises(ConfigError, match="mxfp4"):
        opts.check_against("bfloat16", "cpu")
    with pytest.raises(ConfigError, match="ffn_weights"):
        EngineOptions(ffn_weights="int4")
    EngineOptions(device="cpu").check_against("bfloat16", "cpu", "mxfp4")     # asks for nothing


def test_copies_have_their_own_memory():
    q = Mx4((2, 3, 40), "cpu", gate_up=False)
    q.data.copy_(torch.arange(q.data.numel()) % 251)
    q.settled = True
    twin = copy.deepcopy({"w": q})["w"]
    assert torch.equal(twin.data, q.data) and twin.shape == q.shape and twin.data.data_ptr() != q.data.data_ptr()
    assert twin.scales_at == twin.data.data_ptr() and twin.codes_at - twin.scales_at == q.codes_at - q.scales_at
    assert not twin.settled
    for refused in (copy.copy, pickle.dumps):
        with pytest.raises(TypeError):
            refused(q)


def test_more_experts_than_places_are_numbered_for(ops):
    many = Mx4((70000, 1, 1), "cpu")
    work = {"order": torch.zeros(2, dtype=torch.int32), "idx": torch.zeros(2, dtype=torch.int32),
            "offsets": torch.zeros(70001, dtype=torch.int32), "weight": torch.zeros(2)}
    with pytest.raises(KernelError, match="experts"):
        ops.expert_relu_squared_mx4(torch.zeros(1, 1), many, torch.zeros(2, 1), work, 2, False)


def test_a_single_column_may_have_any_stride(ops):
    """[rows, 1] of a transposed row is as contiguous as any: its one column's stride says nothing."""
    one = torch.zeros(1, 5).t()
    assert one.is_contiguous() and one.stride() == (1, 5) and one.contiguous().stride() == (1, 5)
    assert ops._mx4_ld(one, 1, "rows") == 1
    assert ops._mx4_ld(torch.zeros(7, 30)[:, 4:5], 1, "rows") == 30
    assert ops._mx4_ld(torch.zeros(1, 30)[:, ::30], 1, "rows") >= 1
    ops._stream, ops._status_at = lambda: 0, 0
    for call in (lambda: ops.quantize_mx4(one), lambda: ops.linear_mx4(one, Mx4((3, 1), "cpu"), torch.zeros(5, 3))):
        with pytest.raises(AssertionError, match="a kernel was asked for"):      # accepted
            call()
    for refused in (torch.zeros(1).expand(5, 1), torch.zeros(5, 2).t()[:, :2]):
        with pytest.raises(KernelError):
            ops._mx4_ld(refused, refused.shape[1], "rows")


@pytest.mark.parametrize("routed", [False, True])
def test_calls_of_two_threads_do_not_come_between_one_another(ops, monkeypatch, routed):
    """Quantisation and product are two kernels of a call that runs without the interpreter's lock, with scratch memory of
    the stream between them: a second thread's call on that stream waits for both, and for a larger buffer in the first one's place."""
    ops._stream, ops._status_at, ops._mx4_rows, ops._mx4_lock = lambda: 0, 0, {}, threading.Lock()
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    inside, met = [], []

    def kernels(*args):
        inside.append(threading.get_ident())
        held = ops._mx4_rows[0].data_ptr()
        time.sleep(0.002)
        met.append(len(inside) == 1 and ops._mx4_rows[0].data_ptr() == held)
        inside.pop()
        return 0

    ops._part_libs = {"mx4": {"product": kernels, "expert_product": kernels}}
    w, experts = Mx4((40, 4096), "cpu"), Mx4((2, 40, 4096), "cpu")

    def calls(sizes):
        for m in sizes:
            if routed:
                work = {n: torch.zeros(m + 3, dtype=torch.int32) for n in ("order", "idx", "offsets")}
                ops.expert_relu_squared_mx4(torch.zeros(m, 4096), experts, torch.zeros(m, 40),
                                            dict(work, weight=torch.zeros(m)), 1, False)
            else:
                ops.linear_mx4(torch.zeros(m, 4096), w, torch.zeros(m, 40))

    threads = [threading.Thread(target=calls, args=(range(m, m + 2000, 199),)) for m in (100, 150)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(met) == 22 and all(met)
