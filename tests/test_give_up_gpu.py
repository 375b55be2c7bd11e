"""Blocks that give up a wait stay until the copies they have asked for have had the time to arrive, whichever of their warps gave up.

The first copy announces more bytes than it brings, so that the warp that reads what it brings gives up; the warp that issues the copies never waits
where all of them fit its ring, and has nothing to say about it."""
import pytest
import torch

from rust_deeplearning_b200.kernels import library, ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
WAIT = 50_000               # clock cycles a wait is given here
DRAIN = 200_000             # clock cycles the copies have (RDL_COPY_DRAIN_CYCLES)
FASTEST = 1.965e9           # the multiprocessors' highest clock


def rnd(shape, dtype, seed, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).to(DEV)


def head(rows, top):
    x, w = rnd((rows, 256), torch.bfloat16, 1), rnd((3000, 256), torch.bfloat16, 2, 0.1)
    return lambda status: ops.linear_logprobs(x, w, None, top, status=status)[1:]


def product_mx4(rows, k):
    w, x = ops.pack_mx4(rnd((300, k), torch.float32, 3)), rnd((rows, k), torch.bfloat16, 4)
    x = ops.pack_mx8(x) if rows > 16 else x
    return lambda status: (ops.linear_mx4(x, w, status=status),)


def product(rows, k):
    x, w = rnd((rows, k), torch.bfloat16, 5), rnd((300, k), torch.bfloat16, 6, 0.2)
    return lambda status: (ops.linear(x, w, status=status),)


CALLS = [(12, "linear_logprobs", lambda: head(40, 0)), (12, "linear_logprobs", lambda: head(40, 5)), (12, "linear_logprobs", lambda: head(200, 0)),
         (12, "linear_logprobs", lambda: head(300, 5)), (9, "mx_many_rows", lambda: product_mx4(140, 512)), (9, "mx_many_rows", lambda: product_mx4(400, 512)),
         (10, "mx_some_rows", lambda: product_mx4(40, 4096)), (8, "mx_few_rows", lambda: product_mx4(8, 512)),
         (7, "gemm_skinny", lambda: product(8, 512)), (7, "gemm_skinny", lambda: product(16, 9000))]


@pytest.mark.parametrize("case", range(len(CALLS)))
def test_a_block_that_gives_up_waits_for_its_copies(case):
    code, name, make = CALLS[case]
    lib, call = library.load(), make()
    want = call(None)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    torch.cuda.synchronize()
    try:
        lib.rdl_set_wait_test(code, WAIT, 64)
        start.record()
        call(status)
        end.record()
        torch.cuda.synchronize()
    finally:
        lib.rdl_set_wait_test(0, 0, 0)
    assert status.item() == code and name in library.FAULTS[code]
    # a call that ends with the wait takes 50,000 cycles and a few microseconds, at half of the highest clock still less than this
    assert start.elapsed_time(end) * 1e-3 >= (WAIT + DRAIN) / FASTEST
    status.zero_()
    assert all(torch.equal(a, b) for a, b in zip(call(status), want)) and status.item() == 0
