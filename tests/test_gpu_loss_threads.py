"""Host threads that run different groups of one kernel, each with its own amount of shared memory.

The ring kernels are launched with a slot count that follows from the row length, and the distillation with room for its
teacher entries: one kernel, several sizes.  A launch that asks for more than the kernel's limit at that moment is refused
with a status (nothing runs)."""
import ctypes
import threading

import pytest
import torch

import cinn_b200
from cinn_b200 import runtime as rt

pytestmark = pytest.mark.gpu

LOGPROB = """group fn_threads_{name}
input x bfloat16 {rows},{cols}
input a int64 {rows}
input w float32 {rows}
op token_logprob l = x a
op token_logprob_grad d = x a w
output l float32 {rows}
output d bfloat16 {rows},{cols}
"""
DISTILL = """group fn_threads_{name}
input x bfloat16 {rows},{cols}
input t float32 {rows},{k}
input i int64 {rows},{k}
input w float32 {rows}
op distill_loss l = x t i w
op distill_loss_grad d = x t i w
output l float32 {rows}
output d bfloat16 {rows},{cols}
"""
ROWS = 408  # a CTA of eight warps per row


def program(text, cols, k, seed):
    name = "%d_%d" % (cols, k)
    desc = text.format(name=name, rows=ROWS, cols=cols, k=k)
    fn = ctypes.c_void_p()
    assert cinn_b200.lib().cinn_b200_compile_group(desc.encode(), ctypes.byref(fn)) == 0
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(ROWS, cols, generator=g, device="cuda").bfloat16()
    w = torch.rand(ROWS, generator=g, device="cuda")
    if k:
        ins = [x, torch.randn(ROWS, k, generator=g, device="cuda"), torch.randint(0, cols, (ROWS, k), generator=g, device="cuda"), w]
    else:
        ins = [x, torch.randint(0, cols, (ROWS,), generator=g, device="cuda"), w]
    outs = [torch.empty(ROWS, device="cuda"), torch.empty_like(x)]
    bufs = [rt.make_buffer(t.data_ptr(), str(t.dtype).split(".")[1], tuple(t.shape)) for t in ins + outs]
    return ("fn_threads_" + name).encode(), rt.make_pods(bufs), len(bufs), outs, (ins, bufs)


@pytest.mark.parametrize("what", ["logprob", "distill"])
def test_groups_of_one_kernel_with_different_shared_memory_on_two_threads(what):
    L = cinn_b200.lib()
    if what == "logprob":
        progs = [program(LOGPROB, 20000, 0, 1), program(LOGPROB, 32000, 0, 2)]
    else:
        progs = [program(DISTILL, 32000, 8, 3), program(DISTILL, 32000, 1000, 4)]
    wants, errors = [], []
    for name, pods, n, outs, _ in progs:
        assert L.cinn_b200_group_run(name, pods, n, None) == 0
        torch.cuda.synchronize()
        wants.append([o.clone() for o in outs])
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    start = threading.Barrier(2)

    def loop(p, stream):
        name, pods, n, _, _ = p
        handle = ctypes.c_void_p(stream.cuda_stream)
        start.wait()
        for i in range(4000):
            rc = L.cinn_b200_group_run(name, pods, n, handle)
            if rc != 0:
                errors.append((i, rc, L.cinn_b200_last_error().decode()))
                return
    threads = [threading.Thread(target=loop, args=a) for a in zip(progs, streams)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors, errors
    for (name, _, _, outs, _), want in zip(progs, wants):
        assert all(torch.equal(o, w) for o, w in zip(outs, want))
        L.cinn_b200_release_group(name)
