"""Loss operators over rows of logits on the GPU, against the formulas in float64.

Tolerances count roundings.  u = 2^-24 is half a step of float32, eps_T / 2 half a step of the gradient's type T.

* z = x / temperature and z - max are rounded a few times each, the exponential to 2 units, the sum of `cols` terms by
  a tree over partial sums of at most a few hundred terms: relative error of a softmax value at most
  delta = (64 + 6 R) u with R the spread of the finite z of the row (a rounded exponent argument of size R moves the
  exponential by R u a time), and the same for a sum of such values.
* a log-probability: absolute error delta + 4 u |lp|.
* a loss or slope: its derivative by lp times that, plus a few roundings of its terms.
* the gradient is rounded to T once: eps_T / 2 of its value, or half of T's smallest subnormal.
"""
import ctypes
import math

import pytest
import torch

import cinn_b200
from cinn_b200 import common, frontend

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
NAMES = {v: k for k, v in TYPES.items()} | {torch.int32: "int32", torch.int64: "int64"}
INF = math.inf


def half_step(t):
    return torch.finfo(t).eps / 2


def tiniest(t):
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2


# ---- running a program over torch tensors ---------------------------------------------------------------------
def padded(shape, dtype, skew, fill=None):
    """A tensor `skew` elements into an allocation with 64 elements around it, which no kernel may write."""
    n = math.prod(shape)
    raw = torch.full((n + 128 + skew,), 7, dtype=dtype, device="cuda")
    view = raw[64 + skew: 64 + skew + n].view(shape)
    if fill is not None:
        view.copy_(fill)
    return view, raw


def untouched(view, raw):
    n, start = view.numel(), view.storage_offset()
    return bool((raw[:start] == 7).all()) and bool((raw[start + n:] == 7).all())


def run_program(build, inputs, skew_in=0, skew_out=0, want_groups=None):
    """build(net, variables) -> {name: variable}; inputs: {name: tensor}.  Returns {name: tensor}."""
    net = frontend.NetBuilder("loss_test")
    variables = {k: net.create_input(NAMES[t.dtype], list(t.shape), k) for k, t in inputs.items()}
    out = build(net, variables)
    comp = frontend.Computation.build_and_compile(common.DefaultNVGPUTarget(), net, fetch=[str(v) for v in out.values()])
    if want_groups is not None:
        assert len(comp.groups()) == want_groups, comp.groups()
    names = set(comp.get_all_tensor_names())
    keep = []
    for k, t in inputs.items():
        if k in names:
            view, raw = padded(t.shape, t.dtype, skew_in, t)
            keep.append((view, raw, t))
            comp.get_tensor(k).bind(view.data_ptr())
    results, guards = {}, []
    for k, v in out.items():
        kind = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16,
                "int32": torch.int32}[v.type.name]
        view, raw = padded(v.shape, kind, skew_out)
        guards.append((view, raw))
        results[k] = view
        comp.get_tensor(str(v)).bind(view.data_ptr())
    torch.cuda.synchronize()
    comp.execute(torch.cuda.current_stream().cuda_stream or 1)
    torch.cuda.synchronize()
    assert all(untouched(*g) for g in guards), "a kernel wrote outside its output"
    status = ctypes.c_uint(0)
    cinn_b200.lib().cinn_b200_device_status(ctypes.byref(status))
    assert status.value == 0
    return results


# ---- the formulas in float64 ----------------------------------------------------------------------------------
def spread(x, tau):
    z = x.double() / tau
    z = torch.where(torch.isfinite(z), z, torch.nan)
    hi = torch.nan_to_num(z, nan=-1e300).amax(-1)
    lo = torch.nan_to_num(z, nan=1e300).amin(-1)
    return torch.where(hi >= lo, hi - lo, 0.0).clamp(max=90.0) + hi.abs().clamp(max=200.0)


def delta(x, tau):
    return (64 + 6 * spread(x, tau)) * U


def logprob64(x, a, tau):
    logq = torch.log_softmax(x.double() / tau, -1)
    good = (a >= 0) & (a < x.shape[-1])
    at = torch.where(good, a, 0).long()
    return logq, torch.where(good, logq.gather(-1, at[..., None])[..., 0], 0.0), good, at


def onehot_minus_softmax(logq, at):
    d = -logq.exp()
    d.scatter_add_(-1, at[..., None], torch.ones_like(at[..., None], dtype=d.dtype))
    return d


def policy64(x, a, old, ref, adv, w, lo, hi, kl, tau):
    logq, lp, good, at = logprob64(x, a, tau)
    live = good & (w != 0)
    old, ref, adv, w = old.double(), ref.double(), adv.double(), w.double()
    r = torch.exp(lp - old)
    gap = ref - lp if kl else torch.zeros_like(lp)
    loss = kl * (torch.expm1(gap) - gap) - torch.minimum(r * adv, r.clamp(1 - lo, 1 + hi) * adv)
    cut = ((adv > 0) & (r > 1 + hi)) | ((adv < 0) & (r < 1 - lo))
    slope = -kl * torch.expm1(gap) - torch.where(cut, 0.0, adv * r)
    steep = w.abs() * (adv.abs() * r + kl * (gap.exp() + 1))           # bounds |d loss / d lp| on both branches
    terms = w.abs() * (adv.abs() * r.clamp(max=4) + kl * (gap.exp() + gap.abs() + 1))
    grad = (w * slope / tau)[..., None] * onehot_minus_softmax(logq, at)
    pick = lambda t: torch.where(live, t, 0.0)  # noqa: E731
    return {"loss": pick(w * loss), "logprob": lp, "dlogits": torch.where(live[..., None], grad, 0.0),
            "steep": pick(steep), "terms": pick(terms), "slope": pick((w * slope / tau).abs())}


def distill64(x, t, i, w, tau):
    v = x.shape[-1]
    good = (i >= 0) & (i < v)
    at = torch.where(good, i, 0).long()
    z = (t.double() / tau).masked_fill(~good, -INF)
    live = (w != 0) & (z.amax(-1) > -INF)
    logp = torch.log_softmax(z, -1)
    p = torch.where(good & (logp > -INF), logp.exp(), 0.0)
    logq = torch.log_softmax(x.double() / tau, -1)
    lq = logq.gather(-1, at)
    terms = torch.where(p > 0, p * (logp - lq), 0.0)
    loss = w.double() * terms.sum(-1)
    mass = torch.zeros_like(logq).scatter_add_(-1, at, p)
    grad = (w.double() / tau)[..., None] * (logq.exp() - mass)
    return {"loss": torch.where(live, loss, 0.0), "dlogits": torch.where(live[..., None], grad, 0.0),
            "mass": torch.where(live[..., None], mass, 0.0), "q": torch.where(live[..., None], logq.exp(), 0.0),
            "size": torch.where(live, w.double().abs() * torch.where(p > 0, p * (logp.abs() + lq.abs() + 1), 0.0).sum(-1), 0.0)}


def near(got, want, tol, what):
    got = got.double()
    same = (got == want) | (torch.isnan(got) & torch.isnan(want))
    off = torch.where(same, 0.0, (got - want).abs())
    bad = ~same & ~(off <= tol)
    assert not bad.any(), "%s: %d of %d off, worst %.3g where %.3g is allowed" % (
        what, int(bad.sum()), bad.numel(), float(torch.nan_to_num(off, nan=INF)[bad].max()),
        float(torch.broadcast_to(torch.as_tensor(tol, device=off.device), off.shape)[bad].max()))


def check_grad(got, want, parts, rel, what):
    """parts: the sum of magnitudes that the gradient is a difference of; rel: relative error of each."""
    near(got, want, half_step(got.dtype) * want.abs() * 1.001 + rel * parts + tiniest(got.dtype) * 1.001, what)


def make(rows, cols, dtype, index="int64", seed=0, scale=3.0, shape=None):
    g = torch.Generator(device="cuda").manual_seed(seed + 1000 * rows + cols)
    shape = shape or (rows,)
    x = (scale * torch.randn(shape + (cols,), generator=g, device="cuda")).to(TYPES[dtype])
    a = torch.randint(0, cols, shape, generator=g, device="cuda")
    x.scatter_add_(-1, a[..., None], (8 * torch.rand(shape + (1,), generator=g, device="cuda")).to(x.dtype))
    return g, x, a.to(torch.int32 if index == "int32" else torch.int64)


def policy_inputs(g, x, a, tau=1.0):
    lp = logprob64(x, a, tau)[1]
    shape = a.shape
    rnd = lambda: torch.randn(shape, generator=g, device="cuda")  # noqa: E731
    drift = (0.3 * rnd()).double()
    for border in (math.log(0.8), math.log(1.28)):  # either gradient is right within rounding of a border
        drift = torch.where((drift - border).abs() < 1e-3, drift + 4e-3, drift)
    w = torch.rand(shape, generator=g, device="cuda") + 0.25
    w.view(-1)[3::4] = 0.0
    return {"x": x, "a": a, "old": (lp - drift).float(), "ref": (lp + 0.3 * rnd()).float(), "adv": rnd(), "w": w}


def distill_inputs(g, x, k, index="int64", teacher="float32"):
    shape, cols = x.shape[:-1], x.shape[-1]
    t = (2 * torch.randn(shape + (k,), generator=g, device="cuda")).to(TYPES[teacher])
    i = torch.randint(0, cols, shape + (k,), generator=g, device="cuda")  # repeats some columns when there are few
    if k > 2:
        i[..., 2] = i[..., 0]
        i[..., 1] = -1
    w = torch.rand(shape, generator=g, device="cuda") + 0.25
    w.view(-1)[3::4] = 0.0
    return {"x": x, "t": t, "i": i.to(torch.int32 if index == "int32" else torch.int64), "w": w}


POLICY = dict(clip_low=0.2, clip_high=0.28, kl_coef=0.05)
SIZES = [(1, 1), (1, 2), (3, 7), (5, 31), (2, 257), (9, 1000), (3, 4097), (2, 32768), (4, 50021), (1, 131072),
         (301, 2048), (40, 20011)]


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("rows,cols", SIZES)
def test_token_logprob_and_its_gradient(rows, cols, dtype):
    index, tau = ("int32", 0.7) if rows % 2 else ("int64", 1.0)
    g, x, a = make(rows, cols, dtype, index)
    w = torch.randn(rows, generator=g, device="cuda")
    inputs = {"x": x, "a": a, "w": w}
    logq, lp, _, at = logprob64(x, a, tau)
    d = delta(x, tau)
    got = run_program(lambda b, v: {"lp": b.token_logprob(v["x"], v["a"], temperature=tau),
                                    "dx": b.token_logprob_grad(v["x"], v["a"], v["w"], temperature=tau)}, inputs, want_groups=1)
    alone = run_program(lambda b, v: {"lp": b.token_logprob(v["x"], v["a"], temperature=tau)}, inputs)
    grad_alone = run_program(lambda b, v: {"dx": b.token_logprob_grad(v["x"], v["a"], v["w"], temperature=tau)}, inputs)
    for lp_got in (got["lp"], alone["lp"]):
        near(lp_got, lp, d + 4 * U * lp.abs(), "logprob")
    c = (w.double() / tau)[:, None]
    want, parts = c * onehot_minus_softmax(logq, at), c.abs() * logq.exp()
    parts = parts.scatter_add(1, at[:, None], c.abs())
    for dx in (got["dx"], grad_alone["dx"]):
        check_grad(dx, want, parts, d[:, None], "dlogits")


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("rows,cols", SIZES)
def test_policy_loss_and_its_gradient(rows, cols, dtype):
    tau = 1.3 if rows % 2 else 1.0
    g, x, a = make(rows, cols, dtype, "int64" if rows % 2 else "int32")
    inputs = policy_inputs(g, x, a, tau)
    want = policy64(*inputs.values(), 0.2, 0.28, 0.05, tau)
    args = lambda v: [v[k] for k in ("x", "a", "old", "ref", "adv", "w")]  # noqa: E731
    got = run_program(lambda b, v: {"loss": b.policy_loss(*args(v), temperature=tau, **POLICY),
                                    "lp": b.token_logprob(v["x"], v["a"], temperature=tau),
                                    "dx": b.policy_loss_grad(*args(v), temperature=tau, **POLICY)}, inputs, want_groups=1)
    alone = run_program(lambda b, v: {"loss": b.policy_loss(*args(v), temperature=tau, **POLICY)}, inputs)
    off = delta(x, tau) + 4 * U * want["logprob"].abs() + U * (want["logprob"].abs() + 2)
    near(got["lp"], want["logprob"], off, "logprob")
    for loss in (got["loss"], alone["loss"]):
        near(loss, want["loss"], want["steep"] * off + 16 * U * want["terms"], "loss")
    # slope (1 - q) at the action, slope q elsewhere; the slope itself moves by (|A| r + kl e^gap) per unit of lp
    q = torch.softmax(x.double() / tau, -1).scatter_add(1, a.long()[:, None], torch.ones(rows, 1, dtype=torch.float64, device="cuda"))
    parts = want["slope"][:, None] * q
    wobble = ((want["steep"] * off + 16 * U * want["terms"]) / tau)[:, None] * q
    near(got["dx"], want["dlogits"], half_step(x.dtype) * want["dlogits"].abs() * 1.001 + delta(x, tau)[:, None] * parts
         + wobble * 1.01 + tiniest(x.dtype) * 1.001, "dlogits")


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("rows,cols,k", [(1, 1, 1), (3, 7, 5), (5, 31, 40), (2, 257, 64), (9, 1000, 1), (3, 4097, 33),
                                         (2, 32768, 1024), (4, 50021, 17), (1, 131072, 64), (301, 2048, 8), (40, 20011, 100), (5, 31, 300), (3, 2000, 1024),
                                         (700, 129, 128)])
def test_distill_loss_and_its_gradient(rows, cols, k, dtype):
    tau = 2.0 if rows % 2 else 1.0
    g, x, _ = make(rows, cols, dtype)
    inputs = distill_inputs(g, x, k, "int32" if rows % 2 else "int64", ["float32", "float16", "bfloat16"][k % 3])
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


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("rows,experts,k", [(1, 1, 1), (1, 2, 1), (7, 3, 3), (64, 16, 2), (65, 61, 4), (1000, 128, 8),
                                            (4099, 256, 8), (333, 1024, 2), (20000, 60, 6), (513, 511, 1), (2, 6, 5), (1, 627, 1), (2, 57, 5), (8, 4, 1)])
def test_balance_loss_its_gradient_and_the_counts(rows, experts, k, dtype):
    g, x, _ = make(rows, experts, dtype)
    i = torch.randint(0, experts, (rows, k), generator=g, device="cuda", dtype=torch.int32 if rows % 2 else torch.int64)
    i[::5, 0] = -1
    w = (torch.rand(rows, generator=g, device="cuda") + 0.1) / rows
    if rows > 1:
        w[1::4] = 0.0
    live = w != 0
    x[~live] = float("nan")  # a token that is out may hold anything
    flat = i[live].long().reshape(-1)
    counts = torch.bincount(flat[flat >= 0], minlength=experts)
    f = counts.double() / max(int(counts.sum()), 1)
    q = torch.softmax(x.double(), 1)
    score = (q * f).sum(1, keepdim=True)
    loss = experts * (w.double()[live] * score[live, 0]).sum()
    grad = torch.where(live[:, None], experts * w.double()[:, None] * q * (f - score), 0.0)

    def build(b, v):
        c = b.expert_counts(v["i"], v["w"], experts)
        return {"c": c, "loss": b.balance_loss(v["x"], c, v["w"]), "dx": b.balance_loss_grad(v["x"], c, v["w"])}
    got = run_program(build, {"x": x, "i": i, "w": w}, want_groups=2 if rows <= 64 else 3)  # one part needs no sum
    assert torch.equal(got["c"].long(), counts)
    d = float(delta(x[live], 1.0).max()) + (rows / 64 / 296 / 8 + 64) * U  # and the sums over a slice, then over the slices
    near(got["loss"], loss.reshape(1), d * loss.abs(), "loss")
    parts = torch.where(live[:, None], experts * w.double()[:, None] * q * (f + 1.0 / experts + score.abs() + 1.0 / experts), 0.0)
    check_grad(got["dx"], grad, parts, d, "dlogits")


@pytest.mark.parametrize("shape", [(1, 1), (4096, 1), (4097, 1), (1, 5000), (1025, 4), (32767, 1), (16384, 4), (9363, 7), (3, 32771),
                                   (131071, 2), (2, 50, 33, 3), (90001, 8)])
@pytest.mark.parametrize("experts", [1, 7, 1000])
def test_counts_on_one_cta_a_cluster_and_a_grid(shape, experts):
    g = torch.Generator(device="cuda").manual_seed(experts + shape[0])
    for dtype in (torch.int32, torch.int64):
        i = torch.randint(-2, experts + 2, shape, generator=g, device="cuda", dtype=dtype)
        if dtype == torch.int64:
            i[i == -2] = 2 ** 32  # an expert only in its low half
        w = torch.randn(shape[:-1], generator=g, device="cuda")
        w[torch.rand(shape[:-1], generator=g, device="cuda") < 0.3] = 0.0
        flat = i[w != 0].reshape(-1).long()
        want = torch.bincount(flat[(flat >= 0) & (flat < experts)], minlength=experts)
        got = run_program(lambda b, v: {"c": b.expert_counts(v["i"], v["w"], experts)}, {"i": i, "w": w})
        assert torch.equal(got["c"].long(), want)


@pytest.mark.parametrize("rows,cols", [(60, 131072), (2, 1000003), (20, 150001)])
def test_few_rows_too_long_for_the_rings_of_their_ctas(rows, cols):
    """Several CTAs share such a row, and each brings its part in twice."""
    g, x, a = make(rows, cols, "bfloat16")
    p, t = policy_inputs(g, x, a), distill_inputs(g, x, 70)
    inputs = {**p, "t": t["t"], "i": t["i"]}
    want, second = policy64(*p.values(), 0.2, 0.28, 0.05, 1.0), distill64(x, t["t"], t["i"], p["w"], 1.0)

    def build(b, v):
        args = [v[k] for k in ("x", "a", "old", "ref", "adv", "w")]
        return {"lp": b.token_logprob(v["x"], v["a"]), "dx": b.policy_loss_grad(*args, **POLICY),
                "dl": b.distill_loss(v["x"], v["t"], v["i"], v["w"]), "ddx": b.distill_loss_grad(v["x"], v["t"], v["i"], v["w"])}
    got = run_program(build, inputs)
    alone = run_program(lambda b, v: {"lp": b.token_logprob(v["x"], v["a"])}, inputs)
    d = delta(x, 1.0)
    off = d + 8 * U * (want["logprob"].abs() + 1)
    near(got["lp"], want["logprob"], off, "logprob")
    near(alone["lp"], want["logprob"], off, "logprob alone")
    hot = torch.softmax(x.double(), -1).scatter_add(1, a.long()[:, None], torch.ones(rows, 1, dtype=torch.float64, device="cuda"))
    tol = (d * want["slope"] + want["steep"] * off + 16 * U * want["terms"])[:, None] * hot
    near(got["dx"], want["dlogits"], half_step(x.dtype) * want["dlogits"].abs() * 1.001 + 1.01 * tol + tiniest(x.dtype), "dlogits")
    d = d + delta(t["t"], 1.0) + 16 * U
    near(got["dl"], second["loss"], 2 * d * second["size"], "distill")
    check_grad(got["ddx"], second["dlogits"], p["w"].double()[:, None] * (second["q"] + second["mass"]), d[:, None], "distill dlogits")


# ---- rows that are out, masks, borders ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("cols", [37, 4096, 40009])
def test_rows_without_weight_or_target_are_zero_whatever_they_hold(dtype, cols):
    g, x, a = make(8, cols, dtype)
    inputs = policy_inputs(g, x, a)
    inputs["w"][:] = 1.0
    clean = {k: t.clone() for k, t in inputs.items()}
    for row, (what, value) in enumerate([("w", 0.0), ("a", -1), ("a", cols), ("a", 2 ** 40 + 1), ("w", -0.0)]):
        inputs[what][row] = value
        x[row] = [float("nan"), INF, float("nan"), -INF, INF][row]
        for other in ("old", "ref", "adv"):
            inputs[other][row] = float("nan")
    args = lambda v: [v[k] for k in ("x", "a", "old", "ref", "adv", "w")]  # noqa: E731
    build = lambda b, v: {"loss": b.policy_loss(*args(v), **POLICY), "dx": b.policy_loss_grad(*args(v), **POLICY)}  # noqa: E731
    got, ref = run_program(build, inputs), run_program(build, clean)
    assert (got["loss"][:5] == 0).all() and (got["dx"][:5] == 0).all()
    assert torch.equal(got["loss"][5:], ref["loss"][5:]) and torch.equal(got["dx"][5:], ref["dx"][5:])
    lp = run_program(lambda b, v: {"lp": b.token_logprob(v["x"], v["a"])}, inputs)["lp"]
    assert (lp[1:4] == 0).all()
    dx = run_program(lambda b, v: {"dx": b.token_logprob_grad(v["x"], v["a"], v["w"])}, inputs)["dx"]
    assert (dx[:5] == 0).all() and not (dx[5:] == 0).all()


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("mask", ["-inf", "lowest"])
@pytest.mark.parametrize("cols,kept", [(50, 3), (4096, 17), (33000, 1), (33000, 32000)])
def test_masked_columns(dtype, mask, cols, kept):
    g, x, a = make(6, cols, dtype)
    value = -INF if mask == "-inf" else torch.finfo(x.dtype).min
    x[:3, kept:] = value            # the tail of the vocabulary
    x[3:, : cols - kept] = value    # all but the tail
    a[:3] %= kept
    a[3:] = cols - kept + a[3:] % kept
    inputs = {"x": x, "a": a, "w": torch.ones(6, device="cuda")}
    logq, lp, _, at = logprob64(x, a, 1.0)
    got = run_program(lambda b, v: {"lp": b.token_logprob(v["x"], v["a"]),
                                    "dx": b.token_logprob_grad(v["x"], v["a"], v["w"])}, inputs)
    finite = torch.where(x == value, torch.zeros_like(x), x)
    d = delta(finite, 1.0)
    near(got["lp"], lp, d + 4 * U * lp.abs(), "logprob")
    want = onehot_minus_softmax(logq, at)
    check_grad(got["dx"], want, logq.exp().scatter_add(1, at[:, None], torch.ones(6, 1, dtype=torch.float64, device="cuda")), d[:, None], "dlogits")
    assert (got["dx"][:3, kept:] == 0).all()


@pytest.mark.parametrize("cols", [40, 5000])
def test_a_live_row_with_nan_or_infinity_gives_nan_in_that_row_alone(cols):
    g, x, a = make(6, cols, "float32")
    x[1, cols // 2] = float("nan")
    x[2, cols - 1] = INF
    x[3] = -INF
    got = run_program(lambda b, v: {"lp": b.token_logprob(v["x"], v["a"]), "dx": b.token_logprob_grad(v["x"], v["a"], v["w"])},
                      {"x": x, "a": a, "w": torch.ones(6, device="cuda")})
    assert torch.isnan(got["lp"][1:4]).all() and torch.isfinite(got["lp"][[0, 4, 5]]).all()
    assert torch.isnan(got["dx"][1:4]).all() and torch.isfinite(got["dx"][[0, 4, 5]]).all()


def test_large_logits_do_not_overflow():
    for dtype, big in (("float16", 6e4), ("bfloat16", 1e30), ("float32", 1e30)):
        x = torch.full((2, 5000), -big, dtype=TYPES[dtype], device="cuda")
        x[0, 1234] = big
        x[1, 7:9] = big
        a = torch.tensor([1234, 7], device="cuda")
        got = run_program(lambda b, v: {"lp": b.token_logprob(v["x"], v["a"]), "dx": b.token_logprob_grad(v["x"], v["a"], v["w"])},
                          {"x": x, "a": a, "w": torch.ones(2, device="cuda")})
        near(got["lp"], torch.tensor([0.0, -math.log(2.0)], dtype=torch.float64, device="cuda"), 8 * U, "logprob")
        want = torch.zeros(2, 5000, dtype=torch.float64, device="cuda")
        want[1, 7], want[1, 8] = 0.5, -0.5
        near(got["dx"], want, 8 * U, "dlogits")


def test_teacher_entries_outside_repeated_or_masked():
    g, x, _ = make(7, 6000, "float32")
    inputs = distill_inputs(g, x, 40)
    inputs["w"][:] = 0.5
    i, t = inputs["i"], inputs["t"]
    i[0] = -1                     # nothing kept: the row is out
    i[1] = 4321                   # one column 40 times: p is 1 there
    t[2, ::2] = -INF              # a teacher that masks
    t[3] = -INF                   # nothing left
    i[4, 5:] = 6000               # outside above
    i[5, :20], i[5, 20:] = i[5, 20:].clone(), i[5, 20:].clone()  # every column twice
    x[6, i[6].clamp(min=0).long()] = -INF  # the student excludes what the teacher keeps
    want = distill64(*inputs.values(), 1.0)
    got = run_program(lambda b, v: {"loss": b.distill_loss(v["x"], v["t"], v["i"], v["w"]),
                                    "dx": b.distill_loss_grad(v["x"], v["t"], v["i"], v["w"])}, inputs)
    for row in (0, 3):
        assert got["loss"][row] == 0 and (got["dx"][row] == 0).all()
    assert got["loss"][6] == INF and torch.isfinite(got["dx"]).all()
    d = delta(torch.where(torch.isfinite(x), x, torch.zeros_like(x)), 1.0) + 64 * U
    near(got["loss"][:6], want["loss"][:6], (2 * d * want["size"])[:6], "loss")
    check_grad(got["dx"], want["dlogits"], 0.5 * (want["q"] + want["mass"]), d[:, None], "dlogits")


@pytest.mark.parametrize("cols,k", [(40, 1), (40, 5), (3000, 33), (3000, 200), (40000, 1), (40000, 5), (40000, 300)])
@pytest.mark.parametrize("bad", [float("nan"), INF])
def test_a_teacher_of_nan_or_infinity_gives_nan_in_its_row_alone(cols, k, bad):
    g, x, _ = make(5, cols, "float32")
    inputs = distill_inputs(g, x, k)
    inputs["w"][:] = 1.0
    i, t = inputs["i"], inputs["t"]
    i[:] = torch.randperm(cols, generator=g, device="cuda")[:k] if k <= cols else i
    t[1, k - 1] = bad             # among other entries
    t[2], i[2] = -INF, -1         # alone: the others are unused
    t[2, 0], i[2, 0] = bad, 3
    t[3, k // 2], i[3, k // 2] = bad, cols  # outside: not used
    got = run_program(lambda b, v: {"loss": b.distill_loss(v["x"], v["t"], v["i"], v["w"]),
                                    "dx": b.distill_loss_grad(v["x"], v["t"], v["i"], v["w"])}, inputs)
    used = torch.zeros(5, cols, dtype=torch.bool, device="cuda")
    used[1, i[1].long()] = True
    used[2, 3] = True
    assert torch.isnan(got["loss"]).tolist() == [False, True, True, False, False]
    assert torch.equal(torch.isnan(got["dx"]), used)


def test_policy_without_kl_reads_no_reference():
    g, x, a = make(5, 3001, "float32")
    inputs = policy_inputs(g, x, a)
    inputs["ref"][:] = float("nan")
    got = run_program(lambda b, v: {"loss": b.policy_loss(v["x"], v["a"], v["old"], v["ref"], v["adv"], v["w"]),
                                    "dx": b.policy_loss_grad(v["x"], v["a"], v["old"], v["ref"], v["adv"], v["w"])}, inputs)
    assert torch.isfinite(got["loss"]).all() and torch.isfinite(got["dx"]).all()


@pytest.mark.parametrize("cols", [301, 3001, 40000])
def test_a_constant_in_place_of_a_reference_that_is_not_read(cols):
    g, x, a = make(5, cols, "float32")
    inputs = policy_inputs(g, x, a)

    def build(constant):
        def f(b, v):
            ref = b.fill_constant([5], 0.0) if constant else v["ref"]
            args = [v["x"], v["a"], v["old"], ref, v["adv"], v["w"]]
            return {"loss": b.policy_loss(*args), "dx": b.policy_loss_grad(*args)}
        return f
    one, two = run_program(build(False), inputs, want_groups=1), run_program(build(True), inputs, want_groups=1)
    assert torch.equal(one["loss"], two["loss"]) and torch.equal(one["dx"], two["dx"])


def test_balance_without_any_choice_and_without_any_token():
    x = torch.randn(9, 12, device="cuda")
    i = torch.full((9, 2), -1, device="cuda")

    def build(b, v):
        c = b.expert_counts(v["i"], v["w"], 12)
        return {"c": c, "loss": b.balance_loss(v["x"], c, v["w"]), "dx": b.balance_loss_grad(v["x"], c, v["w"])}
    for w in (torch.ones(9, device="cuda"), torch.zeros(9, device="cuda")):
        got = run_program(build, {"x": x, "i": i, "w": w})
        assert (got["c"] == 0).all() and (got["loss"] == 0).all() and (got["dx"] == 0).all()


# ---- alignment, constants, streams, graphs, size -----------------------------------------------------------------
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("skew_in,skew_out", [(1, 0), (0, 1), (1, 1), (3, 5), (8, 8)])
@pytest.mark.parametrize("cols", [333, 8192, 40010])
def test_any_alignment_gives_the_same_values(dtype, skew_in, skew_out, cols):
    g, x, a = make(5, cols, dtype)
    p, t = policy_inputs(g, x, a), distill_inputs(g, x, 12)
    inputs = {**p, "t": t["t"], "i": t["i"]}

    def build(b, v):
        args = [v[k] for k in ("x", "a", "old", "ref", "adv", "w")]
        return {"loss": b.policy_loss(*args, **POLICY), "dx": b.policy_loss_grad(*args, **POLICY),
                "dloss": b.distill_loss(v["x"], v["t"], v["i"], v["w"]), "ddx": b.distill_loss_grad(v["x"], v["t"], v["i"], v["w"])}
    one, two = run_program(build, inputs), run_program(build, inputs, skew_in, skew_out)
    d = float(delta(x, 1.0).max())
    for k in ("loss", "dloss"):
        near(two[k], one[k].double(), 4 * d * (one[k].double().abs() + 4), k)
    for k in ("dx", "ddx"):  # the sums may be grouped differently: two roundings to T of values that close
        near(two[k], one[k].double(), 2.002 * half_step(x.dtype) * one[k].double().abs() + 8 * d * (one[k].double().abs() + 1e-3 * d) + 2 * tiniest(x.dtype), k)


def test_a_constant_weight_equals_a_tensor_of_it():
    g, x, a = make(11, 5003, "bfloat16")
    inputs = {"x": x, "a": a, "w": torch.full((11,), -0.125, device="cuda")}
    one = run_program(lambda b, v: {"dx": b.token_logprob_grad(v["x"], v["a"], v["w"])}, inputs)
    two = run_program(lambda b, v: {"dx": b.token_logprob_grad(v["x"], v["a"], b.fill_constant([11], -0.125))}, inputs)
    assert torch.equal(one["dx"], two["dx"])


def test_inputs_that_change_between_runs_without_a_wait():
    """Runs and copies queued on one stream, none waited for: each run sees the inputs copied in front of it."""
    rows, cols, experts = 200, 3000, 40
    sets = []
    for seed in range(6):
        g, x, a = make(rows, cols, "bfloat16", seed=seed)
        p, t = policy_inputs(g, x, a), distill_inputs(g, x, 12)
        p["w"] = p["w"].roll(seed)
        router = torch.randn(rows, experts, generator=g, device="cuda")
        sets.append({**p, "t": t["t"], "i": t["i"], "g": router, "gi": router.topk(3, 1).indices})
    net = frontend.NetBuilder("changing")
    v = {k: net.create_input(NAMES[t.dtype], list(t.shape), k) for k, t in sets[0].items()}
    w = net.scale(v["w"], 0.5)  # computed in the program, by a kernel in front of the losses
    args = [v[k] for k in ("x", "a", "old", "ref", "adv")] + [w]
    c = net.expert_counts(v["gi"], w, experts)
    out = [net.token_logprob(v["x"], v["a"]), net.policy_loss(*args, **POLICY), net.policy_loss_grad(*args, **POLICY),
           net.distill_loss(v["x"], v["t"], v["i"], w), net.distill_loss_grad(v["x"], v["t"], v["i"], w), c,
           net.balance_loss(v["g"], c, w), net.balance_loss_grad(v["g"], c, w)]
    comp = frontend.Computation.build_and_compile(common.DefaultNVGPUTarget(), net, fetch=[str(o) for o in out])
    kinds = {"float32": torch.float32, "bfloat16": torch.bfloat16, "int32": torch.int32}
    feed = {k: torch.empty_like(t) for k, t in sets[0].items()}
    res = [torch.empty(o.shape, dtype=kinds[o.type.name], device="cuda") for o in out]
    for k, t in feed.items():
        comp.get_tensor(k).bind(t.data_ptr())
    for o, t in zip(out, res):
        comp.get_tensor(str(o)).bind(t.data_ptr())
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()

    def run_all(wait):
        got = []
        with torch.cuda.stream(stream):
            for s in sets:
                for k, t in feed.items():
                    t.copy_(s[k])
                if wait:
                    torch.cuda.synchronize()
                comp.execute(stream.cuda_stream)
                if wait:
                    torch.cuda.synchronize()
                got.append([t.clone() for t in res])
        torch.cuda.synchronize()
        return got
    want = run_all(True)
    assert not torch.equal(want[0][5], want[1][5]) and not torch.equal(want[0][1], want[1][1])
    for _ in range(5):
        for one, two in zip(run_all(False), want):
            assert all(torch.equal(p, q) for p, q in zip(one, two))


def test_constant_weights_of_the_other_losses():
    g, x, a = make(13, 777, "float32")
    p, t = policy_inputs(g, x, a), distill_inputs(g, x, 9)
    i = torch.randint(0, 20, (13, 3), generator=g, device="cuda")
    router = torch.randn(13, 20, generator=g, device="cuda")
    inputs = {**p, "t": t["t"], "i": t["i"], "g": router, "gi": i}
    inputs["w"] = torch.full((13,), 0.375, device="cuda")

    def build(weight):
        def f(b, v):
            w = v["w"] if weight is None else b.fill_constant([13], weight)
            args = [v[k] for k in ("x", "a", "old", "ref", "adv")] + [w]
            c = b.expert_counts(v["gi"], w, 20)
            return {"pl": b.policy_loss(*args, **POLICY), "pg": b.policy_loss_grad(*args, **POLICY), "c": c,
                    "dl": b.distill_loss(v["x"], v["t"], v["i"], w), "dg": b.distill_loss_grad(v["x"], v["t"], v["i"], w),
                    "bl": b.balance_loss(v["g"], c, w), "bg": b.balance_loss_grad(v["g"], c, w)}
        return f
    one, two = run_program(build(None), inputs), run_program(build(0.375), inputs)
    assert all(torch.equal(one[k], two[k]) for k in one)
    none = run_program(build(0.0), inputs)
    assert all((none[k] == 0).all() for k in none)


def test_a_group_on_host_buffers():
    rows, cols = 70, 3001
    g, x, a = make(rows, cols, "float32")
    w = torch.randn(rows, generator=g, device="cuda")
    group = cinn_b200.FusedGroup("""group fn_host_logprob
input x float32 %d,%d
input a int64 %d
input w float32 %d
op token_logprob l = x a
op token_logprob_grad d = x a w
output l float32 %d
output d float32 %d,%d
""" % (rows, cols, rows, rows, rows, rows, cols))
    lp, dx = torch.empty(rows, device="cuda"), torch.empty_like(x)
    group.run([x, a, w, lp, dx])
    host = [t.cpu().numpy() for t in (x, a, w)] + [torch.zeros(rows).numpy(), torch.zeros(rows, cols).numpy()]
    group.run_host(host)
    torch.cuda.synchronize()
    assert (host[3] == lp.cpu().numpy()).all() and (host[4] == dx.cpu().numpy()).all()
    group.release()


def test_an_exported_program_gives_the_same_bits():
    g, x, a = make(9, 2500, "float16")
    inputs = policy_inputs(g, x, a)
    net = frontend.NetBuilder("exported")
    v = {k: net.create_input(NAMES[t.dtype], list(t.shape), k) for k, t in inputs.items()}
    args = [v[k] for k in ("x", "a", "old", "ref", "adv", "w")]
    out = [net.policy_loss(*args, temperature=0.7, **POLICY), net.policy_loss_grad(*args, temperature=0.7, **POLICY)]
    comp = frontend.Computation.build_and_compile(common.DefaultNVGPUTarget(), net, fetch=[str(o) for o in out])
    results = []
    for c in (comp, frontend.Computation.load(comp.export(), common.DefaultNVGPUTarget())):
        res = [torch.empty(9, device="cuda"), torch.empty_like(x)]
        for k, t in inputs.items():
            c.get_tensor(k).bind(t.data_ptr())
        for o, t in zip(out, res):
            c.get_tensor(str(o)).bind(t.data_ptr())
        c.execute(None)
        results.append(res)
    assert all(torch.equal(p, q) for p, q in zip(*results)) and results[0][1].abs().sum() > 0


def test_leading_axes_are_rows():
    g, x, a = make(1, 1234, "float16", shape=(3, 5))
    inputs = policy_inputs(g, x, a)
    args = lambda v: [v[k] for k in ("x", "a", "old", "ref", "adv", "w")]  # noqa: E731
    build = lambda b, v: {"loss": b.policy_loss(*args(v), **POLICY), "dx": b.policy_loss_grad(*args(v), **POLICY)}  # noqa: E731
    got = run_program(build, inputs)
    flat = run_program(build, {k: t.reshape((15,) + t.shape[2:]) for k, t in inputs.items()})
    assert torch.equal(got["loss"].reshape(-1), flat["loss"]) and torch.equal(got["dx"].reshape(15, -1), flat["dx"])


def test_the_same_call_twice_gives_the_same_bits():
    g, x, a = make(700, 7001, "bfloat16")
    p, t = policy_inputs(g, x, a), distill_inputs(g, x, 30)
    i = torch.randint(0, 7001, (700, 8), device="cuda")

    def build(b, v):
        args = [v[k] for k in ("x", "a", "old", "ref", "adv", "w")]
        return {"loss": b.policy_loss(*args, **POLICY), "dx": b.policy_loss_grad(*args, **POLICY),
                "dloss": b.distill_loss(v["x"], v["t"], v["i"], v["w"]), "ddx": b.distill_loss_grad(v["x"], v["t"], v["i"], v["w"])}
    inputs = {**p, "t": t["t"], "i": t["i"]}
    one, two = run_program(build, inputs), run_program(build, inputs)
    for k in one:
        assert torch.equal(one[k], two[k]), k


def logprob_group(rows, cols, name):
    return cinn_b200.FusedGroup("""group fn_%s
input x bfloat16 %d,%d
input a int64 %d
input w float32 %d
op token_logprob l = x a
op token_logprob_grad d = x a w
output l float32 %d
output d bfloat16 %d,%d
""" % (name, rows, cols, rows, rows, rows, rows, cols))


def test_one_group_on_two_streams_at_once():
    rows, cols = 64, 40000
    group = logprob_group(rows, cols, "two_streams")
    sets = []
    for seed in (1, 2):
        g, x, a = make(rows, cols, "bfloat16", seed=seed)
        w = torch.randn(rows, generator=g, device="cuda")
        sets.append([x, a, w, torch.empty(rows, device="cuda"), torch.empty_like(x)])
    wants = []
    for s in sets:
        group.run(s)
        torch.cuda.synchronize()
        wants.append([s[3].clone(), s[4].clone()])
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in sets:
        s[3].zero_(), s[4].zero_()
    torch.cuda.synchronize()
    for _ in range(20):
        for s, st in zip(sets, streams):
            group.run(s, ctypes.c_void_p(st.cuda_stream))
    torch.cuda.synchronize()
    for s, want in zip(sets, wants):
        assert torch.equal(s[3], want[0]) and torch.equal(s[4], want[1])
    group.release()


def test_two_captured_graphs_replayed_side_by_side():
    rows, experts = 5000, 96

    def program(seed):
        g, x, _ = make(rows, experts, "float32", seed=seed)
        i = torch.randint(0, experts, (rows, 4), generator=g, device="cuda")
        w = torch.rand(rows, generator=g, device="cuda") / rows
        net = frontend.NetBuilder("graph")
        v = {k: net.create_input(NAMES[t.dtype], list(t.shape), k) for k, t in (("x", x), ("i", i), ("w", w))}
        c = net.expert_counts(v["i"], v["w"], experts)
        out = [c, net.balance_loss(v["x"], c, v["w"]), net.balance_loss_grad(v["x"], c, v["w"])]
        comp = frontend.Computation.build_and_compile(common.DefaultNVGPUTarget(), net, fetch=[str(o) for o in out])
        res = [torch.empty(experts, dtype=torch.int32, device="cuda"), torch.empty(1, device="cuda"), torch.empty_like(x)]
        for k, t in (("x", x), ("i", i), ("w", w)):
            comp.get_tensor(k).bind(t.data_ptr())
        for o, t in zip(out, res):
            comp.get_tensor(str(o)).bind(t.data_ptr())
        return comp, res, (x, i, w)
    progs, streams = [program(1), program(2)], [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    wants = []
    for comp, res, _ in progs:
        comp.execute(None)
        wants.append([t.clone() for t in res])
    for (comp, res, _), s in zip(progs, streams):
        comp.execute_graph(s.cuda_stream)
    torch.cuda.synchronize()
    for _, res, _ in progs:
        for t in res:
            t.zero_()
    torch.cuda.synchronize()
    for _ in range(25):
        for (comp, res, _), s in zip(progs, streams):
            comp.execute_graph(s.cuda_stream)
    torch.cuda.synchronize()
    for (_, res, _), want in zip(progs, wants):
        assert all(torch.equal(t, u) for t, u in zip(res, want))


def test_offsets_beyond_32_bits():
    rows, cols = 16450, 131073  # 2.16e9 logits: the last rows start beyond 2^31 elements and 2^32 bytes
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device="cuda").normal_(0, 2)
    a = torch.randint(0, cols, (rows,), device="cuda")
    w = torch.full((rows,), 0.5, device="cuda")
    lp, dx = torch.empty(rows, device="cuda"), torch.empty_like(x)
    group = logprob_group(rows, cols, "far")
    group.run([x, a, w, lp, dx])
    torch.cuda.synchronize()
    group.release()
    for r in (0, 1, 8191, 16383, 16384, rows - 2, rows - 1):
        logq, want, _, at = logprob64(x[r:r + 1], a[r:r + 1], 1.0)
        d = delta(x[r:r + 1], 1.0)
        near(lp[r:r + 1], want, d + 4 * U * want.abs(), "logprob")
        check_grad(dx[r:r + 1], 0.5 * onehot_minus_softmax(logq, at), 0.5 * logq.exp().scatter_add(1, at[:, None], torch.ones(1, 1, dtype=torch.float64, device="cuda")), d[:, None], "dlogits")


# ---- gradients against differences, and the set as it is used ----------------------------------------------------
def test_gradients_against_differences():
    """Central differences of the losses themselves: step h = 0.05 leaves h^2 / 6 times a third derivative of at most
    4 |w| (|A| r + kl e^gap + 1), and the losses' own errors over 2 h."""
    rows, cols, h = 4, 24, 0.05
    g, x, a = make(rows, cols, "float32", scale=1.0)
    p = policy_inputs(g, x, a)
    p["w"][:] = 0.7
    p["adv"] = p["adv"].abs() + 0.1
    p["old"] = p["old"] + 0.8  # ratios well below the upper border: smooth everywhere the differences reach
    t = distill_inputs(g, x, 6)
    i = torch.randint(0, cols, (rows, 2), generator=g, device="cuda")
    inputs = {**p, "t": t["t"], "ti": t["i"], "gi": i}
    inputs["w"][:] = 0.7

    def losses(b, v):
        args = [v[k] for k in ("x", "a", "old", "ref", "adv", "w")]
        c = b.expert_counts(v["gi"], v["w"], cols)
        return {"lp": b.token_logprob(v["x"], v["a"]), "pl": b.policy_loss(*args, **POLICY),
                "dl": b.distill_loss(v["x"], v["t"], v["ti"], v["w"]), "bl": b.balance_loss(v["x"], c, v["w"])}

    def grads(b, v):
        args = [v[k] for k in ("x", "a", "old", "ref", "adv", "w")]
        c = b.expert_counts(v["gi"], v["w"], cols)
        return {"lp": b.token_logprob_grad(v["x"], v["a"], b.fill_constant([rows], 1.0)), "pl": b.policy_loss_grad(*args, **POLICY),
                "dl": b.distill_loss_grad(v["x"], v["t"], v["ti"], v["w"]), "bl": b.balance_loss_grad(v["x"], c, v["w"])}
    exact = run_program(grads, inputs)
    for j in range(0, cols, 5):
        for r in range(rows):
            sides = []
            for sign in (1, -1):
                moved = dict(inputs, x=x.clone())
                moved["x"][r, j] += sign * h
                sides.append(run_program(losses, moved))
            for k in ("lp", "pl", "dl", "bl"):
                diff = (sides[0][k].double() - sides[1][k].double()).sum() / (2 * h)
                near(exact[k][r, j], diff, 4 * 4 * h * h / 6 + 100 * 64 * U, "%s at %d, %d" % (k, r, j))


def test_a_training_step_of_all_of_them():
    """Scoring under a reference, the policy step with its mean loss, a distillation term added to the gradient and the
    router's loss, in one program, against the same by hand."""
    rows, cols, experts, k = 96, 5001, 32, 4
    g, x, a = make(rows, cols, "float32")
    _, ref_x, _ = make(rows, cols, "bfloat16", seed=5)
    p, t = policy_inputs(g, x, a), distill_inputs(g, x, 20)
    router = torch.randn(rows, experts, generator=g, device="cuda")
    choice = router.topk(k, 1).indices
    w = p["w"] / p["w"].sum()
    inputs = {"x": x, "xr": ref_x, "a": a, "old": p["old"], "adv": p["adv"], "w": w, "t": t["t"], "i": t["i"], "g": router, "gi": choice}

    def build(b, v):
        ref = b.token_logprob(v["xr"], v["a"])
        args = [v["x"], v["a"], v["old"], ref, v["adv"], v["w"]]
        kl = dict(POLICY, kl_coef=1e-3)
        total = b.add(b.policy_loss(*args, **kl), b.distill_loss(v["x"], v["t"], v["i"], v["w"]))
        dx = b.add(b.policy_loss_grad(*args, **kl), b.distill_loss_grad(v["x"], v["t"], v["i"], v["w"]))
        c = b.expert_counts(v["gi"], v["w"], experts)
        return {"loss": b.reduce_sum(total), "dx": dx, "ref": ref, "bl": b.balance_loss(v["g"], c, v["w"]), "dg": b.balance_loss_grad(v["g"], c, v["w"])}
    got = run_program(build, inputs)
    ref = logprob64(ref_x, a, 1.0)[1]
    near(got["ref"], ref, delta(ref_x, 1.0) + 4 * U * ref.abs(), "reference")
    one = policy64(x, a, p["old"], got["ref"], p["adv"], w, 0.2, 0.28, 1e-3, 1.0)
    two = distill64(x, t["t"], t["i"], w, 1.0)
    off = (delta(x, 1.0) + 8 * U * one["logprob"].abs() + delta(t["t"], 1.0) + 64 * U)
    near(got["loss"], (one["loss"] + two["loss"]).sum().reshape(1), (one["steep"] * off + 32 * U * one["terms"] + 4 * off * two["size"]).sum(), "loss")
    q = torch.softmax(x.double(), 1)
    hot = q.scatter_add(1, a.long()[:, None], torch.ones(rows, 1, dtype=torch.float64, device="cuda"))
    tol = (off * one["slope"] + one["steep"] * off + 32 * U * one["terms"])[:, None] * hot + (off * w)[:, None] * (two["q"] + two["mass"])
    near(got["dx"], one["dlogits"] + two["dlogits"], tol * 1.01 + 4 * U * (one["dlogits"].abs() + two["dlogits"].abs()), "dlogits")
    live = w != 0
    counts = torch.bincount(choice[live].reshape(-1), minlength=experts)
    f = counts.double() / counts.sum()
    qg = torch.softmax(router.double(), 1)
    score = (qg * f).sum(1, keepdim=True)
    near(got["bl"], (experts * (w.double() * score[:, 0]).sum()).reshape(1), 256 * U, "balance")
    near(got["dg"], experts * w.double()[:, None] * qg * (f - score), 256 * U * experts * (w.double()[:, None] * qg * (f + score + 2 / experts)), "router")
