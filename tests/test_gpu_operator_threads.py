"""Plans of the row operators in several host threads at once."""
from __future__ import annotations

import threading

import pytest
import torch

from einsum_ir_b200 import cabi, operators as op
from tests._operators import quantized32
from tests.test_gpu_operators import CODE, F32, gen, rows_of

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
    threads = [threading.Thread(target=loop, args=(w, s)) for w, s in zip(works, streams)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
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
