"""The loss operators over rows of logits, as timed cases: inputs, a plain form, and the calls a user makes.

Four operators: the log-probability of a chosen token, the clipped policy loss with a KL term, distillation from a
teacher's top logits, and the router's balance loss with its per-expert counts.  `direction` "loss" is the forward pass
alone, "step" the forward pass and the gradient of the summed loss with respect to the logits.
"""
import math

import torch

own = False

DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
INDEX = {"int32": torch.int32, "int64": torch.int64}
LARGEST = 4096 * 131072 * 2  # bytes of logits of the largest listed case


def _row_case(op, rows, cols, dtype, direction, **more):
    case = {"op": op, "rows": rows, "cols": cols, "dtype": dtype, "direction": direction, "index": "int64",
            "temperature": 1.0, "pad": 0}
    case.update(more)
    return case


def listed():
    cases = [
        # the log-probability of one generated token, as a server returns it: latency
        _row_case("logprob", 1, 32768, "bfloat16", "loss"),
        # scoring a batch of rollouts under the old or the reference policy
        _row_case("logprob", 4096, 131072, "bfloat16", "loss", index="int32"),
        # a cross-entropy step on float32 logits, odd sizes (no row starts on a vector boundary)
        _row_case("logprob", 777, 50021, "float32", "step"),
        # a micro-batch of a policy step, sampled at a temperature
        _row_case("policy", 16, 32768, "float16", "step", temperature=0.7),
        # a full policy step over packed rollouts
        _row_case("policy", 4096, 131072, "bfloat16", "step", index="int32"),
        # the policy loss evaluated without a gradient, odd vocabulary padded with masked columns
        _row_case("policy", 2048, 100003, "bfloat16", "loss", pad=35),
        # distillation into a small student
        _row_case("distill", 8, 8192, "float32", "step", k=8),
        # distillation from stored top logits at a temperature
        _row_case("distill", 2048, 131072, "bfloat16", "step", k=64, temperature=2.0, index="int32"),
        # the same at odd sizes in half precision
        _row_case("distill", 1000, 50021, "float16", "step", k=17),
        # the router of one decoding batch
        {"op": "balance", "rows": 64, "cols": 16, "dtype": "float32", "direction": "step", "index": "int64", "k": 2},
        # the router of a training batch with many experts
        {"op": "balance", "rows": 65536, "cols": 256, "dtype": "float32", "direction": "step", "index": "int32", "k": 8},
        # a ragged batch, 16-bit router logits
        {"op": "balance", "rows": 16383, "cols": 61, "dtype": "bfloat16", "direction": "step", "index": "int64", "k": 4},
    ]
    for c in cases:
        c["name"] = "%s %s %dx%d %s" % (c["op"], c["direction"], c["rows"], c["cols"], c["dtype"])
    return cases


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["logprob", "policy", "distill", "balance"])
    dtype, index = rng.choice(sorted(DTYPES)), rng.choice(sorted(INDEX))
    direction = rng.choice(["loss", "step", "step"])
    size = 4 if dtype == "float32" else 2
    if op == "balance":
        cols = spread(4, 512)
        rows = min(spread(1, 65536), LARGEST // (cols * size))
        return {"op": op, "rows": rows, "cols": cols, "dtype": dtype, "direction": direction, "index": index,
                "k": rng.randint(1, min(8, cols))}
    cols = spread(1000, 160000)
    rows = min(spread(1, 4096), LARGEST // (cols * size))
    more = {"index": index, "temperature": rng.choice([1.0, 1.0, 0.7, 2.0]), "pad": rng.choice([0, 0, rng.randint(1, 64)])}
    if op == "distill":
        more["k"] = spread(1, 128)
    return _row_case(op, rows, cols, dtype, direction, **more)


def _out_tokens(rows):
    """Which tokens carry no weight: the prompt in front of each packed sequence, or the padding at a short batch's end."""
    t = torch.arange(rows)
    return (t % 512) < 128 if rows >= 512 else t >= rows - rows // 8


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rows, cols, dtype = case["rows"], case["cols"], DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    live = ~_out_tokens(rows).cuda()
    # the mean over the tokens that count; float16 gradients come with the loss scale such training keeps
    scale = 16384.0 if case["dtype"] == "float16" else 1.0
    weight = live.float() * (scale / max(int(live.sum()), 1))
    logits = torch.empty(rows, cols, dtype=dtype, device="cuda").normal_(0.0, 2.0, generator=gen)
    state = {"case": case, "logits": logits, "weight": weight}
    if case["op"] == "balance":
        order = (logits.float() + 0.1 * randn(rows, cols)).topk(case["k"], dim=1).indices
        state["index"] = order.to(INDEX[case["index"]])
    else:
        pad = case["pad"]
        if pad:
            logits[:, cols - pad:] = -math.inf  # columns beyond the vocabulary
        vocab = cols - pad
        chosen = torch.randint(0, vocab, (rows,), generator=gen, device="cuda")
        peak = 12.0 * torch.rand(rows, generator=gen, device="cuda")
        line = torch.arange(rows, device="cuda")
        logits[line, chosen] = (logits[line, chosen].float() + peak).to(dtype)  # the model knows some tokens well
        tau = case["temperature"]
        if case["op"] == "distill":
            k = case["k"]
            # some overlap between what the teacher keeps and what the student favours; one short list per 16 rows
            kept = torch.rand(rows, vocab if vocab < 4096 else 4096, generator=gen, device="cuda").topk(k, dim=1).indices
            kept = kept * (vocab // kept.new_tensor(min(vocab, 4096)))
            kept[:, 0] = torch.where((kept[:, 1:] == chosen[:, None]).any(1), kept[:, 0], chosen)
            if k > 2:
                kept[::16, k - 1] = -1
            state["teacher_index"] = kept.to(INDEX[case["index"]])
            state["teacher"] = (2.0 * randn(rows, k)).sort(dim=1, descending=True).values + 4.0
        else:
            state["target"] = chosen.to(INDEX[case["index"]])
        if case["op"] == "policy":
            lp = torch.cat([(x[torch.arange(len(x), device="cuda"), a].double() / tau
                             - torch.logsumexp(x.float() / tau, 1).double())
                            for x, a in zip(logits.split(256), chosen.split(256))])
            drift = 0.15 * randn(rows).double()
            # a ratio within rounding of the clip's border has two right gradients: keep a little away from it
            for border in (math.log(1 - 0.2), math.log(1 + 0.28)):
                drift = torch.where((drift - border).abs() < 1e-3, drift + 4e-3, drift)
            state["old"] = (lp - drift).float()
            state["ref"] = (lp + 0.2 * randn(rows).double()).float()
            state["advantage"] = randn(rows)
    if own:
        state["program"] = _program(state)  # the compiled computation that such a program keeps
    return state


POLICY = {"clip_low": 0.2, "clip_high": 0.28, "kl_coef": 0.04}


def _program(s):
    """The operators as a user builds them: one computation over tensors that the caller owns."""
    from cinn_b200 import common, frontend
    case, step = s["case"], s["case"]["direction"] == "step"
    net = frontend.NetBuilder("losses")
    bound, out = [], {}

    def feed(name, tensor):
        kind = str(tensor.dtype).split(".")[1]
        bound.append((name, tensor))
        return net.create_input(kind, list(tensor.shape), name)

    x, w = feed("logits", s["logits"]), feed("weight", s["weight"])
    if case["op"] == "logprob":
        a = feed("target", s["target"])
        out["logprob"] = net.token_logprob(x, a, temperature=case["temperature"])
        if step:
            out["dlogits"] = net.token_logprob_grad(x, a, w, temperature=case["temperature"])
    elif case["op"] == "policy":
        args = [x, feed("action", s["target"]), feed("old", s["old"]), feed("ref", s["ref"]),
                feed("advantage", s["advantage"]), w]
        out["loss"] = net.policy_loss(*args, temperature=case["temperature"], **POLICY)
        if step:
            out["dlogits"] = net.policy_loss_grad(*args, temperature=case["temperature"], **POLICY)
    elif case["op"] == "distill":
        args = [x, feed("teacher", s["teacher"]), feed("teacher_index", s["teacher_index"]), w]
        out["loss"] = net.distill_loss(*args, temperature=case["temperature"])
        if step:
            out["dlogits"] = net.distill_loss_grad(*args, temperature=case["temperature"])
    else:
        out["counts"] = net.expert_counts(feed("index", s["index"]), w, num_experts=case["cols"])
        out["loss"] = net.balance_loss(x, out["counts"], w)
        if step:
            out["dlogits"] = net.balance_loss_grad(x, out["counts"], w)
    results = {}
    fetch = [str(v) for v in out.values()]
    computation = frontend.Computation.build_and_compile(common.DefaultNVGPUTarget(), net, fetch=fetch)
    for name, v in out.items():
        kind = {"counts": torch.int32, "dlogits": s["logits"].dtype}.get(name, torch.float32)
        results[name] = torch.empty(v.shape, dtype=kind, device="cuda")
        bound.append((str(v), results[name]))
    names = computation.get_all_tensor_names()
    for name, tensor in bound:
        if name in names:  # the forward pass of token_logprob takes no weight
            computation.get_tensor(name).bind(tensor.data_ptr())
    return {"computation": computation, "results": results}


def run(state):
    if own:
        # a null stream handle would make execute() wait for the device: 1 names the same (default) stream without that
        state["program"]["computation"].execute(torch.cuda.current_stream().cuda_stream or 1)
        return state["program"]["results"]
    return _plain(state)


def _plain(s):
    case, x, w = s["case"], s["logits"], s["weight"]
    step = case["direction"] == "step"
    z = x.float()
    if case["op"] != "balance" and case["temperature"] != 1.0:
        z = z / case["temperature"]
    z = z - z.amax(1, keepdim=True)
    e = torch.exp(z)
    total = e.sum(1, keepdim=True)
    logq0 = torch.log(total)
    live = w != 0
    if case["op"] == "balance":
        q = e / total
        counts = torch.zeros(case["cols"], dtype=torch.int32, device=x.device)
        hits = live[:, None].expand_as(s["index"]).reshape(-1).int()
        counts.scatter_add_(0, s["index"].reshape(-1).long(), hits)
        f = counts.float() / counts.sum().clamp(min=1)
        kept = torch.where(live[:, None], q, 0.0)
        load = (w[:, None] * kept).sum(0)
        out = {"counts": counts, "loss": (case["cols"] * (f * load).sum()).reshape(1)}
        if step:
            inner = f - (kept * f).sum(1, keepdim=True)
            out["dlogits"] = ((case["cols"] * w)[:, None] * kept * inner).to(x.dtype)
        return out
    if case["op"] == "distill":
        index = s["teacher_index"].long()
        there = index >= 0
        t = torch.where(there, s["teacher"] / case["temperature"], -math.inf)
        t = t - t.amax(1, keepdim=True)
        pt = torch.exp(t)
        mass = pt.sum(1, keepdim=True)
        pt, logp = pt / mass, t - torch.log(mass)
        at = index.clamp(min=0)
        logq = z.gather(1, at) - logq0
        loss = (pt * torch.where(there, logp - logq, 0.0)).sum(1)
        out = {"loss": torch.where(live, w * loss, 0.0)}
        if step:
            diff = (e / total).scatter_add_(1, at, -pt)
            coef = (w / case["temperature"])[:, None]
            out["dlogits"] = torch.where(live[:, None], coef * diff, 0.0).to(x.dtype)
        return out
    a = s["target"].long()[:, None]
    lp = z.gather(1, a) - logq0
    if case["op"] == "logprob":
        out = {"logprob": lp[:, 0]}
        slope = w[:, None]
    else:
        lp64 = lp[:, 0].double()
        ratio = torch.exp(lp64 - s["old"].double())
        adv = s["advantage"].double()
        free, held = ratio * adv, ratio.clamp(1 - POLICY["clip_low"], 1 + POLICY["clip_high"]) * adv
        gap = s["ref"].double() - lp64
        kl = torch.expm1(gap) - gap
        loss = POLICY["kl_coef"] * kl - torch.minimum(free, held)
        out = {"loss": torch.where(live, w * loss, 0.0).float()}
        slope = w * (-POLICY["kl_coef"] * torch.expm1(gap) - torch.where(free <= held, free, 0.0))
        slope = torch.where(live, slope, 0.0).float()[:, None]
    if step:
        slope = slope / case["temperature"]
        grad = (e / total) * -slope
        grad.scatter_add_(1, a, slope)
        out["dlogits"] = torch.where(live[:, None], grad, 0.0).to(x.dtype)
    return out


def work(case):
    rows, cols = case["rows"], case["cols"]
    size = 4 if case["dtype"] == "float32" else 2
    index = 4 if case["index"] == "int32" else 8
    out = int(_out_tokens(rows).sum())
    step = case["direction"] == "step"
    # a token without weight has a loss and a gradient of zero: written, but its logits need not be read
    reads = rows if case["op"] == "logprob" else rows - out
    each = {"logprob": index + 4 + (4 if step else 0), "policy": index + 6 * 4,
            "distill": case.get("k", 0) * (index + 4) + 8, "balance": case.get("k", 0) * index + 4}[case["op"]]
    total = reads * cols * size + (rows * cols * size if step else 0) + rows * each
    if case["op"] == "balance":
        total += 4 * cols + 4
    return {"bytes": total, "flops": reads * cols * (8 if step else 4)}


def exact(case, seed):
    s = prepare(case, seed)
    x, w, step = s["logits"], s["weight"].double(), case["direction"] == "step"
    rows, cols = x.shape
    on = w != 0
    out = {}
    grad = torch.zeros(rows, cols, dtype=torch.float64, device=x.device) if step else None
    if case["op"] == "balance":
        picked = s["index"].long()[on].reshape(-1)
        counts = torch.bincount(picked, minlength=cols)
        f = counts.double() / max(int(counts.sum()), 1)
        q = torch.softmax(x.double(), 1)
        score = (q * f).sum(1)
        out["counts"] = counts.int()
        out["loss"] = (cols * score[on] @ w[on]).reshape(1)
        if step:
            grad = cols * w[:, None] * q * (f[None] - score[:, None])
            grad[~on] = 0
            out["dlogits"] = grad
        return out
    tau = case["temperature"]
    lp_all = torch.zeros(rows, dtype=torch.float64, device=x.device)
    loss_all = torch.zeros_like(lp_all)
    for first in range(0, rows, 256):
        r = slice(first, min(first + 256, rows))
        logq = torch.log_softmax(x[r].double() / tau, 1)
        n = torch.arange(logq.shape[0], device=x.device)
        sparse = torch.zeros_like(logq) if step else None
        if case["op"] == "distill":
            index, slots = s["teacher_index"][r].long(), s["teacher"][r].double() / tau
            logp = torch.log_softmax(slots.masked_fill(index < 0, -math.inf), 1)
            for j in range(index.shape[1]):
                i = index[:, j].clamp(min=0)
                p = torch.where(index[:, j] < 0, 0.0, logp[:, j].exp())
                loss_all[r] += torch.where(p > 0, p * (logp[:, j] - logq[n, i]), 0.0)
                if step:
                    sparse[n, i] += p
            slope = -w[r] / tau
            loss_all[r] *= w[r]
            if step:
                grad[r] = -slope[:, None] * (logq.exp() - sparse)
        else:
            a = s["target"][r].long()
            lp = logq[n, a]
            lp_all[r] = lp
            slope = w[r]
            if case["op"] == "policy":
                adv, gap = s["advantage"][r].double(), s["ref"][r].double() - lp
                ratio = torch.exp(lp - s["old"][r].double())
                low, high, beta = 1 - POLICY["clip_low"], 1 + POLICY["clip_high"], POLICY["kl_coef"]
                surrogate = torch.minimum(ratio * adv, torch.clamp(ratio, low, high) * adv)
                loss_all[r] = w[r] * (beta * (torch.exp(gap) - gap - 1) - surrogate)
                cut = ((adv > 0) & (ratio > high)) | ((adv < 0) & (ratio < low))
                slope = w[r] * (beta * (1 - torch.exp(gap)) - torch.where(cut, 0.0, adv * ratio))
            if step:
                sparse[n, a] = 1.0
                grad[r] = (slope / tau)[:, None] * (sparse - logq.exp())
    if case["op"] == "logprob":
        out["logprob"] = lp_all
    else:
        out["loss"] = torch.where(on, loss_all, 0.0)
    if step:
        grad[~on] = 0
        out["dlogits"] = grad
    return out
