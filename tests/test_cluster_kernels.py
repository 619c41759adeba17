"""Kernels whose CTAs write to each other's shared memory (a cluster's distributed shared memory).

The CTAs of a cluster are scheduled together, but one may reach its first store before another has started; only a
barrier of the whole cluster says that all of them run.  That cannot be shown by running a kernel that lacks it (the
store would go to memory that is nobody's yet), so the order is read from the source; the GPU tests then queue each of
the kernels behind another one and compare with runs that were waited for."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "cinn_b200", "csrc")
PEER = re.compile(r"map_shared_rank|\bmapa\.|ld\.shared::cluster|st\.async")
BARRIER = re.compile(r"cluster\.sync\(\)|cluster_barrier\(\)")


def kernels_with_peers():
    found = []
    for path in sorted(glob.glob(os.path.join(CSRC, "*.cu"))):
        text = re.sub(r"//[^\n]*", "", open(path).read())
        for body in text.split("__global__")[1:]:
            name = re.search(r"\b(k_\w+)\s*\(", body)
            if name and PEER.search(body):
                found.append((name.group(1), body))
    return found


def test_every_cluster_kernel_meets_before_it_touches_a_peer():
    kernels = kernels_with_peers()
    assert {"k_row_reduce_cluster", "k_rownorm_cluster", "k_row_loss", "k_expert_counts"} <= {n for n, _ in kernels}
    for name, body in kernels:
        meet = BARRIER.search(body)
        assert meet and meet.start() < PEER.search(body).start(), name + " touches a peer's shared memory before the cluster has met"


ROW_REDUCE = ("group fn_cluster_%s\ninput x float32 40,70000\nop %s y = x ; dim=1 keep_dim=false\noutput y float32 40\n")


def queued_equals_waited(group, feeds, out_shape, out_dtype):
    """Copies and runs on one stream, none waited for: each run reads what the copy kernel in front of it wrote."""
    import ctypes
    import torch
    stream = torch.cuda.Stream()
    handle = ctypes.c_void_p(stream.cuda_stream)
    buf = [torch.empty_like(t) for t in feeds[0]]
    out = torch.empty(out_shape, dtype=out_dtype, device="cuda")
    torch.cuda.synchronize()

    def go(wait):
        got = []
        with torch.cuda.stream(stream):
            for f in feeds:
                for b, t in zip(buf, f):
                    torch.add(t, 0, out=b)
                if wait:
                    torch.cuda.synchronize()
                group.run(buf + [out], handle)
                group.run(buf + [out], handle)  # and one right behind itself
                if wait:
                    torch.cuda.synchronize()
                got.append(out.clone())
        torch.cuda.synchronize()
        return got
    want = go(True)
    assert not torch.equal(want[0], want[1])
    for _ in range(20):
        assert all(torch.equal(p, q) for p, q in zip(go(False), want))
    return want


@pytest.mark.gpu
@pytest.mark.parametrize("op", ["reduce_sum", "reduce_max"])
def test_row_reductions_over_a_cluster_queued_behind_other_kernels(op):
    import torch
    import cinn_b200
    g = cinn_b200.FusedGroup(ROW_REDUCE % (op, op))
    assert any("row_reduce_cluster" in k for k in g.kernel_names())
    gen = torch.Generator(device="cuda").manual_seed(1)
    feeds = [[torch.randn(40, 70000, generator=gen, device="cuda") + s] for s in range(4)]
    for f, got in zip(feeds, queued_equals_waited(g, feeds, (40,), torch.float32)):
        x = f[0].double()
        if op == "reduce_max":
            assert torch.equal(got, f[0].amax(1))
        else:  # 70000 terms in a tree of at most 70000 / (8 * 512 * 4) + 9 + 5 + 3 levels, each half a step of the sum of magnitudes
            assert ((got - x.sum(1)).abs() <= 32 * 2.0 ** -24 * x.abs().sum(1)).all()
    g.release()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
def test_softmax_rows_over_a_cluster_queued_behind_other_kernels(dtype):
    import torch
    import cinn_b200
    rows, cols = 6, 100000
    ops = "op softmax y = x ; axis=-1\n" if dtype == "float32" else (
        "op cast a = x ; dtype=float32\nop softmax b = a ; axis=-1\nop cast y = b ; dtype=%s\n" % dtype)
    text = "group fn_cluster_softmax_%s\ninput x %s %d,%d\n%soutput y %s %d,%d\n" % (dtype, dtype, rows, cols, ops, dtype, rows, cols)
    g = cinn_b200.FusedGroup(text)
    assert any("rownorm_cluster" in k for k in g.kernel_names())
    kind = getattr(torch, dtype)
    gen = torch.Generator(device="cuda").manual_seed(2)
    feeds = [[(torch.randn(rows, cols, generator=gen, device="cuda") + s / 4).to(kind)] for s in range(4)]
    for f, got in zip(feeds, queued_equals_waited(g, feeds, (rows, cols), kind)):
        want = torch.softmax(f[0].double(), 1)
        # half steps of float32: 4 of the exponential and 4 of those in the sum, 48 + 5 + 4 + 3 of its tree (a CTA of 512 threads
        # has 25000 columns), 1 of the division; then the store's
        tol = want * (69 * 2.0 ** -24 + torch.finfo(kind).eps / 2) + torch.finfo(kind).smallest_normal * torch.finfo(kind).eps / 2
        assert ((got.double() - want).abs() <= tol * 1.001).all()
    g.release()
