"""Plans of the row operators and the contractions in several host threads at once, and in new ones."""
from __future__ import annotations

import threading

import pytest
import torch

from einsum_ir_b200 import binary, cabi, operators as op
from tests._operators import contract64, quantized32
from tests.test_gpu_operators import CODE, F32, codes, gen, rows_of

pytestmark = pytest.mark.gpu


def in_threads(works, times):
    """each work (a function of a stream) `times` times in a host thread and stream of its own; raises what they raise"""
    failed, ready = [], threading.Barrier(len(works))

    def loop(work, stream):
        try:
            ready.wait(60)
            for _ in range(times):
                work(stream.cuda_stream)
        except Exception as e:
            failed.append(e)

    streams = [torch.cuda.Stream() for _ in works]
    torch.cuda.synchronize()
    threads = [threading.Thread(target=loop, args=(w, s), daemon=True) for w, s in zip(works, streams)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(120)
    assert not any(t.is_alive() for t in threads), "a call did not return"
    torch.cuda.synchronize()
    cabi.check_device_errors()
    assert not failed, failed[0]


def norm_backward_work(g, rows, cols, dtype):
    dy, h = rows_of(g, rows, cols, dtype), rows_of(g, rows, cols, dtype)
    rstd, dx, once = torch.rand(rows, generator=g, device="cuda") + 0.5, torch.empty_like(h), torch.empty_like(h)
    plan = op.NormPlan(rows, cols, CODE[dtype])
    plan.backward(dy, h, rstd, once)
    return (lambda stream: plan.backward(dy, h, rstd, dx, stream=stream)), lambda: torch.equal(dx, once)


def quantize_work(g, rows, cols, dtype, offset):
    x = rows_of(g, rows, cols, dtype, 0, offset)
    q, scale = torch.empty((rows, cols), device="cuda", dtype=torch.int8), torch.empty(rows, device="cuda")
    plan = op.QuantizePlan(rows, cols, CODE[dtype])
    return (lambda stream: plan.quantize(x, q, scale, stream=stream)), lambda: torch.equal(q, quantized32(x)[0])


@pytest.mark.parametrize("make", [
    # one kernel each, whose rows in shared memory take different room: ring, wide rows, rows off the grid
    lambda g: [norm_backward_work(g, 8, cols, F32) for cols in (4096, 1024, 2048)],
    lambda g: [norm_backward_work(g, 4, cols, F32) for cols in (17000, 18432)],
    lambda g: [quantize_work(g, 4, cols, F32, 0) for cols in (40000, 17000, 30000)],
    lambda g: [quantize_work(g, 8, cols, F32, 1) for cols in (7900, 3001)],
])
def test_plans_of_several_widths(cuda, make):
    works = make(gen(3))
    in_threads([w for w, _ in works], 2000)
    for _, right in works:
        assert right()


def contract_work(g, m, n, k):
    a, b = codes(g, m, k), codes(g, n, k)
    y = torch.empty((m, n), device="cuda")
    plan = op.Int8ContractPlan(m, n, k, dtype_out=cabi.FP32)
    want = contract64(a, b, None, None, None, 0).float()
    return (lambda stream: plan.contract(a, b, None, None, y, stream=stream)), lambda: torch.equal(y, want)


def bf16_work(g, m, n, k):
    # small whole numbers: the FP32 sums are exact
    a, b = (torch.randint(-8, 9, s, generator=g, device="cuda").bfloat16() for s in ((m, k), (n, k)))
    y = torch.empty((m, n), device="cuda")
    il, ir, io, names = binary.parse_binary("mk,nk->mn")
    sizes = {i: dict(m=m, n=n, k=k)[c] for i, c in enumerate(names)}
    plan = cabi.ContractPlan(binary.contraction_dims(il, ir, io, sizes), cabi.BF16, cabi.BF16, cabi.FP32)
    assert plan.family == cabi.FAMILY_TC
    want = (a.float() @ b.float().T)
    return (lambda stream: plan.contract(a, b, y, stream=stream)), lambda: torch.equal(y, want)


@pytest.mark.parametrize("make", [
    lambda g: [contract_work(g, 40, 512, 1024), contract_work(g, 300, 512, 1024), contract_work(g, 60, 512, 1000)],
    lambda g: [bf16_work(g, 1024, 1024, 512)],
])
def test_first_call_of_a_host_thread(cuda, make):
    """contractions that set up tensor maps before anything has made the context current in the thread"""
    works = make(gen(4))
    in_threads([w for w, _ in works], 200)
    for _, right in works:
        assert right()


def test_one_plan_in_several_host_threads(cuda):
    """plans whose calls share a workspace: packed operands, and partial weight gradients"""
    g = gen(6)
    m, n, k, rows, cols = 300, 1000, 1023, 700, 1500
    b, a = codes(g, n, k), [codes(g, m, k) for _ in range(3)]
    y = [torch.empty((m, n), device="cuda") for _ in range(3)]
    plan = op.Int8ContractPlan(m, n, k, dtype_out=cabi.FP32)
    in_threads([lambda s, i=i: plan.contract(a[i], b, None, None, y[i], stream=s) for i in range(3)], 300)
    for i in range(3):
        assert torch.equal(y[i], contract64(a[i], b, None, None, None, 0).float())
    norm = op.NormPlan(rows, cols, cabi.FP32)
    h, rstd = torch.randn(rows, cols, generator=g, device="cuda"), torch.rand(rows, generator=g, device="cuda") + 0.5
    dy = [torch.randn(rows, cols, generator=g, device="cuda") for _ in range(3)]
    dx, dw, once = torch.empty(3, rows, cols, device="cuda"), torch.empty(3, cols, device="cuda"), torch.empty(3, cols, device="cuda")
    for i in range(3):
        norm.backward(dy[i], h, rstd, dx[i], dweight=once[i])
    in_threads([lambda s, i=i: norm.backward(dy[i], h, rstd, dx[i], dweight=dw[i], stream=s) for i in range(3)], 300)
    assert torch.equal(dw, once)
