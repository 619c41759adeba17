"""Loss operators over rows of logits, on the CPU: result types and shapes, refusals, and which ops share a kernel."""
import os
import shutil
import subprocess

import pytest

import cinn_b200
from cinn_b200 import frontend
from cinn_b200._lib import CinnB200Error


def net_with(rows=(6,), cols=40, dtype="float32", index="int64", k=3, experts=8):
    rows = list(rows)
    b = frontend.NetBuilder("losses")
    v = {"x": b.create_input(dtype, rows + [cols], "x"), "a": b.create_input(index, rows, "a"),
         "t": b.create_input("float16", rows + [k], "t"), "i": b.create_input(index, rows + [k], "i"),
         "g": b.create_input(dtype, rows + [experts], "g"), "c": b.create_input("int32", [experts], "c")}
    for n in ("old", "ref", "adv", "w"):
        v[n] = b.create_input("float32", rows, n)
    return b, v


def policy_args(v):
    return [v["x"], v["a"], v["old"], v["ref"], v["adv"], v["w"]]


def plan(b, fetch=None):
    comp = frontend.Computation.build_and_compile(None, b, fetch=fetch, plan_only=True)
    return [p.split()[0] for _, p in comp.groups()]


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("rows", [(6,), (2, 3)])
def test_result_types_and_shapes(dtype, rows):
    b, v = net_with(rows, dtype=dtype)
    for out in (b.token_logprob(v["x"], v["a"]), b.policy_loss(*policy_args(v)),
                b.distill_loss(v["x"], v["t"], v["i"], v["w"])):
        assert out.type.name == "float32" and out.shape == list(rows)
    for out in (b.token_logprob_grad(v["x"], v["a"], v["w"]), b.policy_loss_grad(*policy_args(v)),
                b.distill_loss_grad(v["x"], v["t"], v["i"], v["w"])):
        assert out.type.name == dtype and out.shape == list(rows) + [40]
    c = b.expert_counts(v["i"], v["w"], 8)
    assert c.type.name == "int32" and c.shape == [8]
    assert b.balance_loss(v["g"], c, v["w"]).shape == [1]
    out = b.balance_loss_grad(v["g"], c, v["w"])
    assert out.type.name == dtype and out.shape == list(rows) + [8]


def test_ops_over_one_tensor_of_logits_share_a_kernel():
    b, v = net_with()
    b.policy_loss(*policy_args(v), kl_coef=0.1)
    b.token_logprob(v["x"], v["a"])
    b.policy_loss_grad(*policy_args(v), kl_coef=0.1)
    assert plan(b) == ["row_loss"]
    b, v = net_with()
    b.token_logprob(v["x"], v["a"], temperature=0.5)
    b.token_logprob_grad(v["x"], v["a"], v["w"], temperature=0.5)
    assert plan(b) == ["row_loss"]
    b, v = net_with()
    b.distill_loss_grad(v["x"], v["t"], v["i"], v["w"])
    b.distill_loss(v["x"], v["t"], v["i"], v["w"])
    assert plan(b) == ["row_loss"]
    for rows, groups in ((65,), ["expert_counts", "router_loss", "row_reduce"]), ((64,), ["expert_counts", "router_loss"]):
        b, v = net_with(rows)
        c = b.expert_counts(v["i"], v["w"], 8)
        b.balance_loss(v["g"], c, v["w"])
        b.balance_loss_grad(v["g"], c, v["w"])
        assert sorted(plan(b)) == groups


@pytest.mark.parametrize("given", [{}, {"clip_low": 0.2}, {"kl_coef": 0, "clip_high": "2e-1"}, {"temperature": "1.00"}])
def test_parameters_are_compared_by_value(given):
    """One op on defaults or with numbers written another way, the other with the values spelled out."""
    b, v = net_with()
    b.policy_loss(*policy_args(v))
    b._op("policy_loss_grad", policy_args(v), **given)
    assert plan(b) == ["row_loss"]
    b, v = net_with()
    b._op("distill_loss", [v["x"], v["t"], v["i"], v["w"]])
    b.distill_loss_grad(v["x"], v["t"], v["i"], v["w"], temperature=1)
    assert plan(b) == ["row_loss"]


@pytest.mark.parametrize("one,two,good", [("temperature=1", "temperature=1.0", True), ("", "temperature=1", True),
                                          ("kl_coef=0.5", "kl_coef=5e-1", True), ("temperature=1", "temperature=2", False),
                                          ("", "kl_coef=0.1", False)])
def test_parameters_of_a_group_description_are_compared_by_value(one, two, good):
    text = """group fn_by_value
input x float32 4,50
input a int64 4
input w float32 4
op policy_loss l = x a w w w w ; %s
op policy_loss_grad d = x a w w w w ; %s
output l float32 4
output d float32 4,50
""" % (one, two)
    if good:
        cinn_b200.FusedGroup(text).release()
    else:
        with pytest.raises(CinnB200Error, match="differ in an operand or an attribute"):
            cinn_b200.FusedGroup(text)


def test_ops_that_differ_stay_apart():
    b, v = net_with()
    b.policy_loss(*policy_args(v), kl_coef=0.1)
    b.policy_loss_grad(*policy_args(v), kl_coef=0.2)
    assert plan(b) == ["row_loss", "row_loss"]
    b, v = net_with()
    b.token_logprob(v["x"], v["a"], temperature=0.5)
    b.policy_loss(*policy_args(v))
    assert plan(b) == ["row_loss", "row_loss"]
    b, v = net_with()
    b.distill_loss(v["x"], v["t"], v["i"], v["w"])
    b.policy_loss(*policy_args(v))
    assert plan(b) == ["row_loss", "row_loss"]


def test_a_gradient_scaled_by_the_loss_it_shares_logits_with_is_not_merged():
    # the upstream gradient is computed from the log-probability: one kernel cannot do both
    b, v = net_with()
    lp = b.token_logprob(v["x"], v["a"])
    b.token_logprob_grad(v["x"], v["a"], b.multiply(lp, v["w"]))
    assert plan(b) == ["row_loss", "ew_chain", "row_loss"]
    b, v = net_with()
    lp = b.token_logprob(v["x"], v["a"])
    b.token_logprob_grad(v["x"], v["a"], lp)
    assert plan(b) == ["row_loss", "row_loss"]


def test_a_loss_takes_its_place_in_a_program():
    b, v = net_with()
    w = b.multiply(v["adv"], v["w"])
    loss = b.policy_loss(v["x"], v["a"], v["old"], v["ref"], v["adv"], w)
    b.policy_loss_grad(v["x"], v["a"], v["old"], v["ref"], v["adv"], w)
    b.reduce_sum(b.scale(loss, 2.0))
    got = plan(b)
    assert got.count("row_loss") == 1 and len(got) <= 4


def test_a_constant_weight_is_taken_and_other_constants_are_refused():
    b, v = net_with()
    one = b.fill_constant([6], 1.0 / 6)
    b.token_logprob_grad(v["x"], v["a"], one)
    assert plan(b) == ["row_loss"]
    b, v = net_with()
    one = b.fill_constant([6], 1.0 / 6)
    b.policy_loss(v["x"], v["a"], one, v["ref"], v["adv"], v["w"])
    with pytest.raises(CinnB200Error, match="only the per-row weight"):
        plan(b)


def test_a_reference_that_is_not_read_may_be_a_constant():
    for kl in (0.0, 1e-60):  # the kernel's weight of the term is a float32
        b, v = net_with()
        args = policy_args(v)
        args[3] = b.fill_constant([6], 0.0)
        b.policy_loss(*args, kl_coef=kl)
        b.policy_loss_grad(*args, kl_coef=kl)
        assert plan(b) == ["row_loss"]
    b, v = net_with()
    b.policy_loss(v["x"], v["a"], v["old"], b.fill_constant([6], 0.0), v["adv"], v["w"], kl_coef=0.1)
    with pytest.raises(CinnB200Error, match="only the per-row weight"):
        plan(b)
    b, v = net_with()  # its shape and type are still checked
    with pytest.raises(CinnB200Error, match="one value per row"):
        b.policy_loss(v["x"], v["a"], v["old"], b.fill_constant([7], 0.0), v["adv"], v["w"])


def test_export_and_load_keep_the_plan():
    b, v = net_with(dtype="bfloat16")
    b.policy_loss(*policy_args(v), kl_coef=0.1, clip_high=0.28)
    b.policy_loss_grad(*policy_args(v), kl_coef=0.1, clip_high=0.28)
    comp = frontend.Computation.build_and_compile(None, b, plan_only=True)
    again = frontend.Computation.load(comp.export(), plan_only=True)
    assert [p for _, p in again.groups()] == [p for _, p in comp.groups()]


def test_program_passes_leave_the_loss_ops_alone():
    b, v = net_with(dtype="float16")
    loss, grad = b.policy_loss(*policy_args(v)), b.policy_loss_grad(*policy_args(v))
    assert b.apply_pass([loss, grad]) == 1


REFUSALS = [
    ("rank", lambda b, v: b.token_logprob(v["a"], v["a"]), "float32, float16 or bfloat16"),
    ("index type", lambda b, v: b.token_logprob(v["x"], v["w"]), "int32 or int64"),
    ("rows of the target", lambda b, v: b.token_logprob(v["x"], v["i"]), "one value per row"),
    ("weight type", lambda b, v: b.token_logprob_grad(v["x"], v["a"], v["a"]), "must be float32"),
    ("temperature 0", lambda b, v: b.token_logprob(v["x"], v["a"], temperature=0.0), "temperature"),
    ("temperature nan", lambda b, v: b.token_logprob(v["x"], v["a"], temperature=float("nan")), "temperature"),
    ("clip_low", lambda b, v: b.policy_loss(*policy_args(v), clip_low=1.5), "clip_low"),
    ("clip_high", lambda b, v: b.policy_loss(*policy_args(v), clip_high=-0.1), "clip_high"),
    ("kl_coef", lambda b, v: b.policy_loss_grad(*policy_args(v), kl_coef=float("inf")), "kl_coef"),
    ("teacher rows", lambda b, v: b.distill_loss(v["x"], v["w"], v["a"], v["w"]), "entries"),
    ("teacher index", lambda b, v: b.distill_loss(v["x"], v["t"], v["t"], v["w"]), "int32 or int64"),
    ("experts", lambda b, v: b.expert_counts(v["i"], v["w"], 0), "num_experts"),
    ("too many experts", lambda b, v: b.expert_counts(v["i"], v["w"], 1025), "num_experts"),
    ("counts type", lambda b, v: b.balance_loss_grad(v["g"], v["old"], v["w"]), "counts"),
    ("counts of another router", lambda b, v: b.balance_loss(v["x"], v["c"], v["w"]), "counts"),
    ("index without slots", lambda b, v: b.expert_counts(v["a"], v["w"], 8), "slots"),
    ("operand count", lambda b, v: b._op("policy_loss", [v["x"], v["a"]]), "takes 6 inputs"),
]


@pytest.mark.parametrize("name,call,message", REFUSALS, ids=[r[0] for r in REFUSALS])
def test_refusals(name, call, message):
    b, v = net_with()
    with pytest.raises(CinnB200Error, match=message):
        call(b, v)


@pytest.mark.parametrize("text,good", [("0.0001", True), ("9.99999975e-05", True), ("10000", True), ("9e-05", False), ("10002", False),
                                       ("-1", False), ("inf", False), ("1x", False)])
def test_borders_of_the_temperature(text, good):
    """9.99999975e-05 is 1e-4 as a float, which the C++ front end passes on."""
    b, v = net_with()
    if good:
        b._op("token_logprob", [v["x"], v["a"]], temperature=text)
        assert plan(b) == ["row_loss"]
    else:
        with pytest.raises(CinnB200Error, match="temperature"):
            b._op("token_logprob", [v["x"], v["a"]], temperature=text)


def test_too_many_teacher_entries_or_columns_are_refused():
    b, v = net_with(k=1025, cols=4000)
    with pytest.raises(CinnB200Error, match="1024 teacher entries"):
        b.distill_loss(v["x"], v["t"], v["i"], v["w"])
    b, v = net_with(experts=1025)
    with pytest.raises(CinnB200Error, match="1024 experts"):
        b.balance_loss_grad(v["g"], v["c"], v["w"])


GROUP = """group fn_{name}
input x float32 4,50
input a int64 4
input w float32 4
op token_logprob_grad d = x a w ; temperature=1.0
output d {dtype} {shape}
"""


@pytest.mark.parametrize("dtype,shape,good", [("float32", "4,50", True), ("float16", "4,50", False),
                                              ("float32", "4,51", False), ("float32", "200", False)])
def test_a_group_description_must_declare_the_result(dtype, shape, good):
    text = GROUP.format(name="d_%s_%s" % (dtype, shape.replace(",", "_")), dtype=dtype, shape=shape)
    if good:
        g = cinn_b200.FusedGroup(text)
        assert g.pattern == "row_loss" and g.launches == 1 and g.scratch_bytes == 0
        g.release()
    else:
        with pytest.raises(CinnB200Error, match="not what token_logprob_grad gives"):
            cinn_b200.FusedGroup(text)


def test_a_group_in_which_two_ops_write_one_result_is_refused():
    text = """group fn_one_result
input x float32 4,50
input a int64 4
input w float32 4
op policy_loss l = x a w w w w
op token_logprob l = x a
output l float32 4
output p float32 4
"""  # p would be written by no op
    with pytest.raises(CinnB200Error, match="two ops write 'l'"):
        cinn_b200.FusedGroup(text)


def test_a_group_that_mixes_a_loss_with_another_op_is_refused():
    text = GROUP.format(name="mixed", dtype="float32", shape="4,50").replace(
        "output d", "op relu r = d\noutput d").replace("output d float32 4,50", "output d float32 4,50\noutput r float32 4,50")
    with pytest.raises(CinnB200Error, match="no common kernel"):
        cinn_b200.FusedGroup(text)


@pytest.mark.parametrize("rows,cols", [("1", "4294967296"), ("2147483647", "2147483647,2147483647,9")])
def test_extents_beyond_what_a_buffer_describes_are_refused(rows, cols):
    text = GROUP.format(name="huge", dtype="float32", shape="4,50").replace("4,50", rows + "," + cols).replace("int64 4", "int64 " + rows).replace("w float32 4", "w float32 " + rows)
    with pytest.raises(CinnB200Error, match="too large"):
        cinn_b200.FusedGroup(text)


def test_a_group_whose_operand_has_no_rows_is_refused():
    text = GROUP.format(name="empty", dtype="float32", shape="0,50").replace("4,50", "0,50").replace("int64 4", "int64 0").replace("w float32 4", "w float32 0")
    with pytest.raises(CinnB200Error, match="non-positive extent"):
        cinn_b200.FusedGroup(text)


def test_every_per_row_weight_may_be_a_constant():
    for build in (lambda b, v, w: b.policy_loss(*policy_args(v)[:5], w), lambda b, v, w: b.distill_loss_grad(v["x"], v["t"], v["i"], w),
                  lambda b, v, w: b.balance_loss_grad(v["g"], v["c"], w), lambda b, v, w: b.expert_counts(v["i"], w, 8)):
        b, v = net_with()
        build(b, v, b.fill_constant([6], 0.25))
        assert len(plan(b)) == 1
    b, v = net_with()
    with pytest.raises(CinnB200Error, match="one value per row"):
        b.policy_loss(*policy_args(v)[:5], b.fill_constant([7], 0.25))


@pytest.fixture(scope="module")
def cpp_program(tmp_path_factory):
    cinn_b200.lib()
    gxx = shutil.which("g++")
    if not gxx:
        pytest.skip("no g++")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    exe, libdir = str(tmp_path_factory.mktemp("cpp") / "loss_test"), os.path.join(root, "cinn_b200")
    subprocess.run([gxx, "-std=c++17", "-O1", "-Wall", "-I" + os.path.join(root, "include"), os.path.join(root, "tests", "cpp", "loss_test.cc"),
                    "-o", exe, "-L" + libdir, "-lcinn_b200", "-Wl,-rpath," + libdir], check=True)
    return exe


def test_cpp_front_end_plans_the_losses(cpp_program):
    out = subprocess.run([cpp_program, "plan"], capture_output=True, text=True)
    assert out.returncode == 0 and "PLANNED" in out.stdout, out.stdout + out.stderr


@pytest.mark.gpu
def test_cpp_front_end_runs_the_losses(cpp_program):
    out = subprocess.run([cpp_program, "run"], capture_output=True, text=True)
    assert out.returncode == 0 and "PASSED" in out.stdout, out.stdout + out.stderr
