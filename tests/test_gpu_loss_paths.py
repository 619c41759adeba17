"""Plans of the loss operators that a program reaches seldom: the balance loss without its gradient, teacher lists longer
than a CTA of eight warps, host buffers cut into chunks.  Formulas and tolerances as in test_gpu_loss_ops.py."""
import pytest
import torch

import cinn_b200
from cinn_b200 import common, frontend
from tests.test_gpu_loss_ops import (NAMES, POLICY, TYPES, U, check_grad, delta, distill64, distill_inputs, make, near,
                                     policy_inputs, run_program)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("rows,experts", [(1, 1), (3, 2), (64, 16), (65, 61), (1000, 128), (4099, 256), (333, 1024), (1000, 1000), (20000, 60),
                                          (513, 511), (2, 627), (300, 8), (70000, 4)])
def test_balance_loss_without_its_gradient(rows, experts, dtype):
    g, x, _ = make(rows, experts, dtype)
    counts = torch.randint(0, 100, (experts,), generator=g, device="cuda", dtype=torch.int32)
    counts[experts // 2] = 7  # at least one choice
    w = (torch.rand(rows, generator=g, device="cuda") + 0.1) / rows
    if rows > 1:
        w[1::4] = 0.0
    live = w != 0
    x[~live] = float("nan")  # a token that is out may hold anything
    f = counts.double() / int(counts.sum())
    score = (torch.softmax(x.double(), 1) * f).sum(1)
    want = experts * (w.double()[live] * score[live]).sum()
    got = run_program(lambda b, v: {"loss": b.balance_loss(v["x"], v["c"], v["w"])}, {"x": x, "c": counts, "w": w},
                      want_groups=1 if rows <= 64 else 2)
    both = run_program(lambda b, v: {"loss": b.balance_loss(v["x"], v["c"], v["w"]), "dx": b.balance_loss_grad(v["x"], v["c"], v["w"])},
                       {"x": x, "c": counts, "w": w})
    d = float(delta(x[live], 1.0).max()) + (rows / 64 / 296 / 8 + 64) * U  # and the sums over a slice, then over the slices
    near(got["loss"], want.reshape(1), d * want.abs(), "loss alone")
    near(both["loss"], want.reshape(1), d * want.abs(), "loss with the gradient")


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("rows,cols,k", [(410, 20000, 257), (420, 33001, 300), (409, 17000, 1024)])
def test_many_rows_with_more_teacher_entries_than_threads(rows, cols, k, dtype):
    tau = 1.5
    g, x, _ = make(rows, cols, dtype)
    inputs = distill_inputs(g, x, k, "int32" if k % 2 else "int64")
    want = distill64(*inputs.values(), tau)
    args = lambda v: [v[n] for n in ("x", "t", "i", "w")]  # noqa: E731
    got = run_program(lambda b, v: {"loss": b.distill_loss(*args(v), temperature=tau),
                                    "dx": b.distill_loss_grad(*args(v), temperature=tau)}, inputs, want_groups=1)
    alone = run_program(lambda b, v: {"loss": b.distill_loss(*args(v), temperature=tau)}, inputs)
    d = delta(x, tau) + delta(inputs["t"], tau) + (k // 32 + 8) * U
    for loss in (got["loss"], alone["loss"]):
        near(loss, want["loss"], 2 * d * want["size"], "loss")
    c = (inputs["w"].double() / tau)[:, None]
    check_grad(got["dx"], want["dlogits"], c * (want["q"] + want["mass"]), d[:, None], "dlogits")


HOST = {
    "distill": """group fn_host_distill
input x float32 512,4099
input t float32 512,20
input i int64 512,20
op fill_constant w = ; shape=512 value=0.25 dtype=float32
op distill_loss l = x t i w ; temperature=2
output l float32 512
""",
    "distill_grad": """group fn_host_distill_grad
input x float32 512,4099
input t float32 512,20
input i int64 512,20
op fill_constant w = ; shape=512 value=0.25 dtype=float32
op distill_loss_grad d = x t i w ; temperature=2
output d float32 512,4099
""",
    "balance_grad": """group fn_host_balance_grad
input x float32 40000,64
input c int32 64
op fill_constant w = ; shape=40000 value=0.001 dtype=float32
op balance_loss_grad d = x c w
output d float32 40000,64
""",
}


@pytest.mark.parametrize("what", sorted(HOST))
def test_host_buffers_in_chunks_of_rows(what):
    """With a constant weight all operands of such a group lie along the rows, and run_host cuts them."""
    gen = torch.Generator(device="cuda").manual_seed(9)
    group = cinn_b200.FusedGroup(HOST[what])
    if what == "balance_grad":
        ins = [torch.randn(40000, 64, generator=gen, device="cuda"), torch.randint(1, 50, (64,), generator=gen, device="cuda", dtype=torch.int32)]
        shape = (40000, 64)
    else:
        ins = [torch.randn(512, 4099, generator=gen, device="cuda"), torch.randn(512, 20, generator=gen, device="cuda"),
               torch.randint(0, 4099, (512, 20), generator=gen, device="cuda")]
        shape = (512,) if what == "distill" else (512, 4099)
    out = torch.empty(shape, device="cuda")
    group.run(ins + [out])
    host = [t.cpu().numpy() for t in ins] + [torch.zeros(shape).numpy()]
    group.run_host(host)
    torch.cuda.synchronize()
    got = torch.from_numpy(host[-1])
    assert cinn_b200.lib().cinn_b200_group_host_chunks(group.name.encode()) > 1
    # another number of rows may share a row among more CTAs: sums of magnitudes up to 1 regrouped, and a loss of at most w (ln 4099 + 8)
    assert (got - out.cpu()).abs().max() <= 200 * U * (4 if what == "distill" else 1)
    group.release()


def test_a_captured_program_of_the_row_losses_reads_the_inputs_of_each_replay():
    """Long rows on clusters, long rows one CTA each and short rows, replayed without a wait while the inputs change."""
    sizes = {"few": (6, 60000), "many": (450, 9000), "short": (70, 500)}
    net = frontend.NetBuilder("captured_losses")
    sets = [{} for _ in range(4)]
    outs, v = [], {}
    for n, (rows, cols) in sizes.items():
        for seed, s in enumerate(sets):
            g, x, a = make(rows, cols, "bfloat16", seed=seed)
            p, t = policy_inputs(g, x, a), distill_inputs(g, x, 9)
            p["w"] = p["w"].roll(seed)
            s.update({n + k: q for k, q in {**p, "t": t["t"], "i": t["i"]}.items()})
        for k in ("x", "a", "old", "ref", "adv", "w", "t", "i"):
            q = sets[0][n + k]
            v[k] = net.create_input(NAMES[q.dtype], list(q.shape), n + k)
        args = [v[k] for k in ("x", "a", "old", "ref", "adv", "w")]
        outs += [net.token_logprob(v["x"], v["a"]), net.policy_loss(*args, **POLICY), net.policy_loss_grad(*args, **POLICY),
                 net.distill_loss(v["x"], v["t"], v["i"], v["w"]), net.distill_loss_grad(v["x"], v["t"], v["i"], v["w"])]
    comp = frontend.Computation.build_and_compile(common.DefaultNVGPUTarget(), net, fetch=[str(o) for o in outs])
    feed = {k: torch.empty_like(q) for k, q in sets[0].items()}
    res = [torch.empty(o.shape, dtype=TYPES[o.type.name], device="cuda") for o in outs]
    for k, q in feed.items():
        comp.get_tensor(k).bind(q.data_ptr())
    for o, q in zip(outs, res):
        comp.get_tensor(str(o)).bind(q.data_ptr())
    stream = torch.cuda.Stream()

    def go(run, wait):
        got = []
        with torch.cuda.stream(stream):
            for s in sets:
                for k, q in feed.items():
                    q.copy_(s[k])
                run(stream.cuda_stream)
                if wait:
                    torch.cuda.synchronize()
                got.append([q.clone() for q in res])
        torch.cuda.synchronize()
        return got
    torch.cuda.synchronize()
    want = go(comp.execute, True)
    assert not torch.equal(want[0][2], want[1][2])
    go(comp.execute_graph, True)  # captures
    for _ in range(5):
        for one, two in zip(go(comp.execute_graph, False), want):
            assert all(torch.equal(p, q) for p, q in zip(one, two))
