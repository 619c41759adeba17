"""Tokens that a model is sure of: log-probabilities near 0 keep their digits.

The chosen column a holds the row's largest logit, far above the others and behind them all.  With M = z_a and e = the sum of
exp(z_j - M) over the other columns, lp = -log(1 + e) and the gradient at a is w e / (1 + e).  u = 2^-24 is half a step
of float32 at 1.  Roundings of S = 1 + e in float32, with the reference at M:

* e is a sum of exponentials that is off by (64 + 6 R + N) u relative, R the spread of the row and N the terms that a lane adds
  up (the bound that the other tests of these operators take for any softmax value, and a plain sum);
* the 1 is exact, and few values are added to it, each time half a step: the lane's other partial sums (2), the 31
  other lanes (5 levels), the other warps (2 values per lane for 64 of them, and 5 levels): 14 u;
* the logarithm of S, near 0, is right to 2 steps of itself: 4 u e;
* 1 - q = (S - 1) / S, the difference exact: 14 u, and 4 u of itself.
"""
import pytest
import torch

from tests.test_gpu_loss_ops import TYPES, U, half_step, near, run_program, tiniest

pytestmark = pytest.mark.gpu

SIZES = [(64, 256), (200, 2048), (64, 4096), (16, 32768), (700, 20000), (450, 32768)]


def sure(rows, cols, dtype, tau=1.0):
    g = torch.Generator(device="cuda").manual_seed(rows + cols)
    x = torch.randn(rows, cols, generator=g, device="cuda").to(TYPES[dtype])
    x[:, -1] = (15 + 3 * torch.rand(rows, generator=g, device="cuda")).to(x.dtype)  # at most 2^24 above what a lane has seen
    x *= tau
    a = torch.full((rows,), cols - 1, device="cuda")
    z = x.double() / tau
    e = torch.exp(z[:, :-1] - z[:, -1:]).sum(1)
    spread = z.amax(1) - z.amin(1)
    lanes = 32 * max(1, min(64, cols // 256))
    tol = (14 + (64 + 6 * spread + cols / lanes / 4 + 4) * e) * U
    assert float(e.max()) < 0.02
    return g, x, a, e, tol


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("rows,cols", SIZES)
def test_logprob_and_gradient_of_a_sure_token(rows, cols, dtype):
    g, x, a, e, tol = sure(rows, cols, dtype)
    w = torch.ones(rows, device="cuda")
    got = run_program(lambda b, v: {"lp": b.token_logprob(v["x"], v["a"]), "dx": b.token_logprob_grad(v["x"], v["a"], v["w"])},
                      {"x": x, "a": a, "w": w}, want_groups=1)
    alone = run_program(lambda b, v: {"lp": b.token_logprob(v["x"], v["a"])}, {"x": x, "a": a})
    near(got["lp"], -torch.log1p(e), tol, "logprob with the gradient")
    near(alone["lp"], -torch.log1p(e), tol, "logprob alone")
    want = e / (1 + e)
    near(got["dx"][:, -1], want, tol + (4 * U + half_step(x.dtype)) * want + tiniest(x.dtype), "gradient at the token")


@pytest.mark.parametrize("rows,cols", SIZES)
def test_policy_and_distillation_of_a_sure_token(rows, cols):
    """At the old policy's own log-probability, ratio 1: the loss is off by its slopes times lp's error and a few roundings;
    a teacher with that token alone gives -lp."""
    g, x, a, e, tol = sure(rows, cols, "float32", tau=2.0)
    lp = -torch.log1p(e)
    adv, w = torch.randn(rows, generator=g, device="cuda"), torch.ones(rows, device="cuda")
    old, kl = lp.float(), 0.5
    ref = (lp + 0.1 * torch.randn(rows, generator=g, device="cuda", dtype=torch.float64)).float()
    t = torch.zeros(rows, 1, device="cuda")
    inputs = {"x": x, "a": a, "old": old, "ref": ref, "adv": adv, "w": w, "t": t, "i": a[:, None].contiguous()}
    got = run_program(lambda b, v: {"pl": b.policy_loss(*[v[k] for k in ("x", "a", "old", "ref", "adv", "w")], kl_coef=kl, temperature=2.0),
                                    "dl": b.distill_loss(v["x"], v["t"], v["i"], v["w"], temperature=2.0)}, inputs)
    gap, r = ref.double() - lp, torch.exp(lp - old.double())
    want = kl * (torch.expm1(gap) - gap) - r * adv.double()
    tol = tol + 4 * U * lp.abs()
    near(got["pl"], want, (adv.abs() * r + kl * gap.exp().sub(1).abs()) * tol + 8 * U * (adv.abs() * r + kl * (gap.abs() + 1e-2)), "policy loss")
    near(got["dl"], -lp, tol, "distillation")
