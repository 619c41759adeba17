// Loss operators over rows of logits: operand checks and launch plans (kernels: row_loss.cu, router_loss.cu).
#include "loss_ops.h"

#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <set>

namespace cinn_b200 {

namespace {

constexpr int64_t kMaxTeacherEntries = 1024;  // entries per row that distill_loss takes
constexpr int64_t kMaxExperts        = 1024;  // a warp keeps a router row of this length in registers

int64_t CeilDiv(int64_t a, int64_t b) { return (a + b - 1) / b; }
int64_t RoundUp(int64_t a, int64_t b) { return CeilDiv(a, b) * b; }

bool IsLogits(DType t) { return t == DType::kFloat32 || t == DType::kFloat16 || t == DType::kBFloat16; }
bool IsIndex(DType t) { return t == DType::kInt32 || t == DType::kInt64; }
const char* ShortName(DType t) {
  return t == DType::kFloat32 ? "f32" : t == DType::kFloat16 ? "f16" : "bf16";
}
// How the kernels are told an operand's type at run time.
int64_t FloatCode(DType t) { return t == DType::kFloat32 ? 0 : t == DType::kFloat16 ? 1 : 2; }

bool ReadNumber(const std::map<std::string, std::string>& attrs, const char* key, double* v) {
  auto it = attrs.find(key);
  if (it == attrs.end()) return false;
  char* end = nullptr;
  *v        = strtod(it->second.c_str(), &end);
  return end != it->second.c_str() && *end == 0 && std::isfinite(*v);
}

struct Spec {
  const char* name;
  size_t inputs;
  int weight;  // which operand is the per-row factor, the one that may be a fill_constant; -1: none
  const char* args;
};
const Spec kSpecs[] = {
    {"token_logprob", 2, -1, "(logits, target)"},
    {"token_logprob_grad", 3, 2, "(logits, target, dlogprob)"},
    {"policy_loss", 6, 5, "(logits, action, old_logprob, ref_logprob, advantage, weight)"},
    {"policy_loss_grad", 6, 5, "(logits, action, old_logprob, ref_logprob, advantage, weight)"},
    {"distill_loss", 4, 3, "(logits, teacher_logits, teacher_index, weight)"},
    {"distill_loss_grad", 4, 3, "(logits, teacher_logits, teacher_index, weight)"},
    {"expert_counts", 2, 1, "(index, weight)"},
    {"balance_part", 3, 2, "(logits, counts, weight)"},
    {"balance_loss_grad", 3, 2, "(logits, counts, weight)"},
};
const Spec* FindSpec(const std::string& op) {
  for (const Spec& s : kSpecs)
    if (op == s.name) return &s;
  return nullptr;
}

bool EndsWith(const std::string& s, const char* tail) {
  const std::string t = tail;
  return s.size() >= t.size() && s.compare(s.size() - t.size(), t.size(), t) == 0;
}

// In how many sums over tokens balance_part leaves the loss: one per CTA of its kernel, at least 64 tokens each, two CTAs
// per SM of a B200 at most.  It is the extent of the op's result, so it depends on the shape alone.
int64_t BalanceParts(int64_t rows) { return std::min<int64_t>(CeilDiv(rows, 64), 296); }

}  // namespace

bool IsLossOp(const std::string& op_type) { return FindSpec(op_type) != nullptr; }

bool InferLossOp(const std::string& op, const std::vector<TensorDesc>& in, std::map<std::string, std::string>* attrs,
                 TensorDesc* out, std::string* err) {
  auto fail = [&](const std::string& m) {
    if (err) *err = m;
    return false;
  };
  const Spec* spec = FindSpec(op);
  if (!spec) return fail("unknown loss op");
  if (in.size() != spec->inputs) return fail("takes " + std::to_string(spec->inputs) + " inputs " + spec->args);
  for (auto& t : in) {
    if (t.shape.empty()) return fail("operands need at least one dimension");
    int64_t n = 1;
    for (auto d : t.shape) {
      if (d <= 0) return fail("operand '" + t.name + "' has a non-positive extent");
      if (d > 2147483647 || n > (int64_t{1} << 58) / d) return fail("operand '" + t.name + "' is too large");
      n *= d;
    }
  }
  // One value per row of `like` (every axis but the last).
  auto per_row = [&](const TensorDesc& t, const TensorDesc& like, const char* what, DType want) {
    if (t.dtype != want) return fail(std::string(what) + " must be " + DTypeName(want));
    if (t.shape != std::vector<int64_t>(like.shape.begin(), like.shape.end() - 1))
      return fail(std::string(what) + " must have one value per row (the first operand's shape without its last axis)");
    return true;
  };
  // The parameters that scale or bound something, with their defaults and the values they may take.
  auto number = [&](const char* key, double dflt, bool (*ok)(double), const char* rule) {
    double v = dflt;
    if (attrs->count(key)) {
      if (!ReadNumber(*attrs, key, &v) || !ok(v)) return fail(std::string("'") + key + "' must be " + rule);
    } else {
      char text[64];
      snprintf(text, sizeof(text), "%.17g", dflt);
      (*attrs)[key] = text;
    }
    return true;
  };
  auto positive     = [](double v) { return (float)v >= 1e-4f && (float)v <= 1e4f; };  // (1e-4f lies below 1e-4)
  auto non_negative = [](double v) { return v >= 0.0; };
  auto fraction     = [](double v) { return v >= 0.0 && v <= 1.0; };

  if (op == "expert_counts") {
    double e = 0;
    if (!IsIndex(in[0].dtype)) return fail("index must be int32 or int64");
    if (in[0].shape.size() < 2) return fail("index must be [tokens..., slots]");
    if (!per_row(in[1], in[0], "weight", DType::kFloat32)) return false;
    if (!ReadNumber(*attrs, "num_experts", &e) || e < 1 || e > kMaxExperts || e != std::floor(e))
      return fail("'num_experts' must be a whole number from 1 to " + std::to_string(kMaxExperts));
    out->dtype = DType::kInt32;
    out->shape = {(int64_t)e};
    int64_t n  = in[0].numel();
    if (n > 2147483647) return fail("more than 2^31 - 1 choices: the counts are int32");
    return true;
  }
  const TensorDesc& x = in[0];
  if (!IsLogits(x.dtype)) return fail("logits must be float32, float16 or bfloat16");
  if (x.shape.size() < 2) return fail("logits must be [rows..., columns]");
  const int64_t cols = x.shape.back(), rows = x.numel() / cols;
  const std::vector<int64_t> row_shape(x.shape.begin(), x.shape.end() - 1);
  if (op == "balance_part" || op == "balance_loss_grad") {
    if (cols > kMaxExperts) return fail("at most " + std::to_string(kMaxExperts) + " experts");
    if (in[1].dtype != DType::kInt32 || in[1].shape != std::vector<int64_t>{cols}) return fail("counts must be int32 [experts]");
    if (!per_row(in[2], x, "weight", DType::kFloat32)) return false;
    const bool grad = op == "balance_loss_grad";
    out->dtype = grad ? x.dtype : DType::kFloat32;
    out->shape = grad ? x.shape : std::vector<int64_t>{BalanceParts(rows)};
    return true;
  }
  if (!number("temperature", 1.0, positive, "a number from 1e-4 to 1e4")) return false;
  if (op == "distill_loss" || op == "distill_loss_grad") {
    const TensorDesc &t = in[1], &i = in[2];
    if (!IsLogits(t.dtype)) return fail("teacher_logits must be float32, float16 or bfloat16");
    if (!IsIndex(i.dtype)) return fail("teacher_index must be int32 or int64");
    if (t.shape != i.shape || t.shape.size() != x.shape.size() ||
        !std::equal(row_shape.begin(), row_shape.end(), t.shape.begin()))
      return fail("teacher_logits and teacher_index must both be [rows..., entries] over the rows of the logits");
    if (t.shape.back() > kMaxTeacherEntries)
      return fail("at most " + std::to_string(kMaxTeacherEntries) + " teacher entries per row");
    if (!per_row(in[3], x, "weight", DType::kFloat32)) return false;
  } else {
    if (!IsIndex(in[1].dtype)) return fail("the token ids must be int32 or int64");
    if (!per_row(in[1], x, "the token ids", in[1].dtype)) return false;
    if (op == "token_logprob_grad" && !per_row(in[2], x, "dlogprob", DType::kFloat32)) return false;
    if (op == "policy_loss" || op == "policy_loss_grad") {
      if (!per_row(in[2], x, "old_logprob", DType::kFloat32) || !per_row(in[3], x, "ref_logprob", DType::kFloat32) ||
          !per_row(in[4], x, "advantage", DType::kFloat32) || !per_row(in[5], x, "weight", DType::kFloat32))
        return false;
      if (!number("clip_low", 0.2, fraction, "a number from 0 to 1") ||
          !number("clip_high", 0.2, non_negative, "zero or more") || !number("kl_coef", 0.0, non_negative, "zero or more"))
        return false;
    }
  }
  if (EndsWith(op, "_grad")) {
    out->dtype = x.dtype;
    out->shape = x.shape;
  } else {
    out->dtype = DType::kFloat32;
    out->shape = row_shape;
  }
  return true;
}

namespace {

struct LossMatcher {
  const GroupDesc& g;
  const DeviceInfo& dev;
  std::string* err;
  std::map<std::string, int> input_index, output_index;
  std::map<std::string, double> constants;

  LossMatcher(const GroupDesc& g_, const DeviceInfo& d, std::string* e) : g(g_), dev(d), err(e) {
    for (size_t i = 0; i < g.inputs.size(); ++i) input_index[g.inputs[i].name] = (int)i;
    for (size_t i = 0; i < g.outputs.size(); ++i) output_index[g.outputs[i].name] = (int)i;
  }
  std::unique_ptr<CompiledGroup> Fail(const std::string& m) {
    if (err) *err = "group '" + g.name + "': " + m;
    return nullptr;
  }
  std::unique_ptr<CompiledGroup> NewPlan(const char* pattern) {
    auto p     = std::make_unique<CompiledGroup>();
    p->name    = g.name;
    p->pattern = pattern;
    p->inputs  = g.inputs;
    p->outputs = g.outputs;
    for (auto& t : g.inputs) p->algorithmic_bytes += t.numel() * DTypeBytes(t.dtype);
    for (auto& t : g.outputs) p->algorithmic_bytes += t.numel() * DTypeBytes(t.dtype);
    p->elements = 0;
    for (auto& t : g.outputs) p->elements = std::max<int64_t>(p->elements, t.numel());
    return p;
  }
  // A group input, a group output, or (for an operand or result that this group does not have) a null pointer.
  ArgSpec In(const std::string& value) const {
    ArgSpec a;
    auto it = input_index.find(value);
    if (it == input_index.end()) return a;
    a.kind  = ArgSpec::kInput;
    a.index = it->second;
    return a;
  }
  ArgSpec Out(const OpDesc* op) const {
    ArgSpec a;
    if (!op) return a;
    a.kind  = ArgSpec::kOutput;
    a.index = output_index.at(op->output);
    return a;
  }
  static ArgSpec I(int64_t v) {
    ArgSpec a;
    a.ivalue = v;
    return a;
  }
  static ArgSpec F(double v) {
    ArgSpec a;
    a.kind   = ArgSpec::kFloat;
    a.fvalue = v;
    return a;
  }
  static double Attr(const OpDesc& op, const char* key) { return atof(op.attrs.at(key).c_str()); }
  // Whether two ops were given the same parameters, by value: one may spell out a default, or write 1 as 1.0.
  static bool SameParameters(const OpDesc& a, const OpDesc& b) {
    for (const char* key : {"temperature", "clip_low", "clip_high", "kl_coef"}) {
      if (a.attrs.count(key) != b.attrs.count(key)) return false;
      if (a.attrs.count(key) && Attr(a, key) != Attr(b, key)) return false;
    }
    return true;
  }
  const TensorDesc& Input(const std::string& value) const { return g.inputs[input_index.at(value)]; }
  // The value of a per-row factor that is one constant (its pointer is null then).
  ArgSpec Constant(const std::string& value) const {
    auto it = constants.find(value);
    return F(it == constants.end() ? 0.0 : it->second);
  }

  // The reference policy's log-probabilities where there is no KL term: they are not read (the kernel gets a null pointer
  // for a constant, and its weight of the term as float32).
  static bool IsPlaceholder(const OpDesc& op, size_t operand) {
    if (operand != 3 || (op.type != "policy_loss" && op.type != "policy_loss_grad")) return false;
    double kl = 0.0;
    return !op.attrs.count("kl_coef") || (ReadNumber(op.attrs, "kl_coef", &kl) && (float)kl == 0.0f);
  }

  std::unique_ptr<CompiledGroup> Run() {
    std::map<std::string, OpDesc> ops;  // by type, attributes completed
    std::map<std::string, TensorDesc> fills;
    std::set<std::string> written;
    for (auto& op : g.ops) {
      if (op.type != "fill_constant") continue;
      TensorDesc t;
      double v = 0;
      t.name   = op.output;
      auto dt = op.attrs.find("dtype"), sh = op.attrs.find("shape");
      t.dtype = dt == op.attrs.end() ? DType::kFloat32 : DTypeFromName(dt->second);
      if (sh == op.attrs.end() || !ReadNumber(op.attrs, "value", &v)) return Fail("fill_constant needs a shape and a finite value");
      for (size_t at = 0; at < sh->second.size();) {
        t.shape.push_back(atoll(sh->second.c_str() + at));
        const size_t comma = sh->second.find(',', at);
        at = comma == std::string::npos ? sh->second.size() : comma + 1;
      }
      fills[op.output]     = t;
      constants[op.output] = v;
    }
    for (auto& op : g.ops) {
      if (op.type == "fill_constant") continue;
      if (!IsLossOp(op.type)) return Fail("a loss op and '" + op.type + "' have no common kernel");
      if (ops.count(op.type)) return Fail("two " + op.type + " ops have no common kernel");
      if (!written.insert(op.output).second) return Fail("two ops write '" + op.output + "'");
      std::vector<TensorDesc> in;
      for (size_t k = 0; k < op.inputs.size(); ++k) {
        const std::string& v = op.inputs[k];
        if (fills.count(v)) {
          if ((int)k != FindSpec(op.type)->weight && !IsPlaceholder(op, k))
            return Fail(op.type + ": operand '" + v + "' is a constant, which only the per-row weight may be (and ref_logprob while kl_coef is 0)");
          in.push_back(fills[v]);
          continue;
        }
        if (!input_index.count(v)) return Fail("operand '" + v + "' of " + op.type + " is not an input of the group");
        in.push_back(Input(v));
      }
      OpDesc full = op;
      TensorDesc out;
      std::string why;
      if (!InferLossOp(op.type, in, &full.attrs, &out, &why)) return Fail(op.type + ": " + why);
      auto it = output_index.find(op.output);
      if (it == output_index.end()) return Fail("the result of " + op.type + " is not an output of the group");
      const TensorDesc& declared = g.outputs[it->second];
      if (declared.dtype != out.dtype || declared.shape != out.shape)
        return Fail("output '" + op.output + "' is not what " + op.type + " gives");
      ops[op.type] = full;
    }
    if (g.outputs.size() != ops.size()) return Fail("an output is produced by no op");
    auto get = [&](const char* type) -> const OpDesc* {
      auto it = ops.find(type);
      return it == ops.end() ? nullptr : &it->second;
    };
    auto only = [&](std::set<std::string> types) {
      for (auto& kv : ops)
        if (!types.count(kv.first)) return false;
      return true;
    };
    if (const OpDesc* op = get("expert_counts")) {
      if (ops.size() != 1) return Fail("expert_counts has a kernel of its own");
      return PlanCounts(*op);
    }
    if (only({"balance_part", "balance_loss_grad"})) return PlanRouter(get("balance_part"), get("balance_loss_grad"));
    if (only({"distill_loss", "distill_loss_grad"})) return PlanRows(2, get("distill_loss"), get("distill_loss_grad"), nullptr);
    if (only({"policy_loss", "policy_loss_grad", "token_logprob"}) && (get("policy_loss") || get("policy_loss_grad")))
      return PlanRows(1, get("policy_loss"), get("policy_loss_grad"), get("token_logprob"));
    if (only({"token_logprob", "token_logprob_grad"}))
      return PlanRows(0, nullptr, get("token_logprob_grad"), get("token_logprob"));
    return Fail("these loss ops have no common kernel");
  }

  // kind 0 token_logprob, 1 policy, 2 distill; any of the three results may be absent.
  std::unique_ptr<CompiledGroup> PlanRows(int kind, const OpDesc* loss, const OpDesc* grad, const OpDesc* logprob) {
    const OpDesc& main = grad ? *grad : loss ? *loss : *logprob;
    if (loss && grad && (loss->inputs != grad->inputs || !SameParameters(*loss, *grad)))
      return Fail("the loss and its gradient differ in an operand or an attribute");
    if (logprob && (logprob->inputs[0] != main.inputs[0] || logprob->inputs[1] != main.inputs[1] ||
                    Attr(*logprob, "temperature") != Attr(main, "temperature")))
      return Fail("the log-probability is not the one the other ops use");
    const TensorDesc& x = Input(main.inputs[0]);
    const int64_t cols = x.shape.back(), rows = x.numel() / cols;
    const char* kinds[] = {"logprob", "policy", "distill"};
    auto p = NewPlan("row_loss");
    LaunchStep s;
    const std::string name = std::string("row_loss_") + kinds[kind] + (grad ? "_grad_" : "_") + ShortName(x.dtype);
    s.kernel = FindKernel(name);
    if (!s.kernel) return Fail("kernel " + name + " is missing");
    auto arg = [&](size_t k) { return In(main.inputs[k]); };
    const int weight        = FindSpec(main.type)->weight;
    const TensorDesc& index = Input(main.inputs[kind == 2 ? 2 : 1]);
    const int64_t wide      = index.dtype == DType::kInt64 ? 1 : 0;
    int64_t entries = 0, teacher = 0;
    // logits, ids, three operands of the kind, the per-row factor
    if (kind == 0) {
      s.args = {arg(0), arg(1), ArgSpec(), ArgSpec(), ArgSpec()};
    } else if (kind == 1) {
      s.args = {arg(0), arg(1), arg(2), arg(3), arg(4)};
    } else {
      s.args  = {arg(0), arg(2), arg(1), ArgSpec(), ArgSpec()};
      entries = index.shape.back();
      teacher = FloatCode(Input(main.inputs[1]).dtype);
    }
    s.args.push_back(weight < 0 ? ArgSpec() : arg(weight));
    s.args.push_back(Out(loss));
    s.args.push_back(Out(logprob));
    s.args.push_back(Out(grad));
    for (int64_t v : {rows, cols, entries, wide, teacher}) s.args.push_back(I(v));
    s.args.push_back(weight < 0 ? F(0.0) : Constant(main.inputs[weight]));
    const double t = Attr(main, "temperature"), c = 1.4426950408889634 / t;  // exp(z / t) = 2^(c z)
    for (double v : {1.0 / t, c}) s.args.push_back(F(v));
    s.args.push_back(F(kind == 1 ? 1.0 - Attr(main, "clip_low") : 0.0));
    s.args.push_back(F(kind == 1 ? 1.0 + Attr(main, "clip_high") : 0.0));
    s.args.push_back(F(kind == 1 ? Attr(main, "kl_coef") : 0.0));
    return ShapeRows(std::move(p), s, rows, cols * DTypeBytes(x.dtype), entries, grad != nullptr);
  }

  // Warps per CTA, CTAs per row and ring slots of the row kernels (row_loss.cu says what was measured).
  std::unique_ptr<CompiledGroup> ShapeRows(std::unique_ptr<CompiledGroup> p, LaunchStep s, int64_t rows, int64_t row_bytes,
                                           int64_t entries, bool grad) {
    const int64_t vecs = row_bytes / 16;
    int64_t warps = 1, ctas = 1;
    if (rows > 2147483647) return Fail("more than 2^31 - 1 rows");
    // Short rows stay in registers: with the gradient up to 8 KiB (32768 x 4096 bf16 114 us, through a ring 128; 16 KiB 114
    // against 113), without it up to 16 KiB (55 against 68).  Eight vectors per thread in one warp, or without the
    // gradient; otherwise four, in more warps (114 us against 118).
    const int64_t most_per = grad ? 4 : 8;
    int64_t per            = 8;  // vectors per thread
    if (vecs > 256) {
      per = most_per;
      while (warps < 4 && warps * 32 * per < vecs) warps *= 2;
    }
    if (warps * 32 * per >= vecs && entries <= 128) {
      while (per > 2 && warps * 16 * per >= vecs) per /= 2;
      const std::string name = std::string(s.kernel->name) + "_n" + std::to_string(per);
      s.kernel = FindKernel(name);
      if (!s.kernel) return Fail("kernel " + name + " is missing");
      s.args.push_back(I(warps == 4 ? 2 : warps / 2));
      s.dyn_smem = (size_t)(8 / warps * 16 * RoundUp(entries, 4));
      s.block[0] = 256;
      s.grid[0]  = (unsigned)CeilDiv(rows, 8 / warps);
      p->steps.push_back(s);
      return p;
    }
    // Few rows: smaller CTAs, and several of them for a row.  With the gradient 5.5 CTAs per SM in all (89 x 131072 bf16: 16 us
    // with 8 CTAs per row, 24 with one), without it 2 (more of them wait for each other: 128 rows 11 us with 2, 13 with 4).
    const int64_t most = dev.sm_count * (grad ? 11 : 4) / 2;
    for (warps = 1; warps < 4 && warps * 256 < vecs;) warps *= 2;
    if (rows * 2 <= most) {
      while (ctas < 8 && rows * ctas * 2 <= most && vecs > 128 * warps * ctas) ctas *= 2;
    } else {
      if (vecs > 2048) warps = 8;  // (8192 x 16384 bf16: 93 us with 4 warps, 123 with 8; from 64 KiB on 8 are level or better)
    }
    const int64_t slots = std::min<int64_t>(4, CeilDiv(vecs + 1, 128 * warps));
    s.args.push_back(I(slots));
    s.cluster  = ctas > 1 ? (unsigned)ctas : 0;
    s.dyn_smem = (size_t)(slots * (warps * 2048 + 16) + 8 + 8 * warps * ctas + 16 * RoundUp(entries, 4));
    s.block[0] = (unsigned)(32 * warps + 32);
    s.grid[0]  = (unsigned)(ctas * rows);
    p->steps.push_back(s);
    return p;
  }

  std::unique_ptr<CompiledGroup> PlanRouter(const OpDesc* part, const OpDesc* grad) {
    if (part && grad && part->inputs != grad->inputs) return Fail("the loss and its gradient differ in an operand");
    const OpDesc& main  = grad ? *grad : *part;
    const TensorDesc& x = Input(main.inputs[0]);
    const int64_t cols = x.shape.back(), rows = x.numel() / cols;
    auto p = NewPlan("router_loss");
    // Vector loads need rows that start on 16-byte boundaries; other rows, and buffers that do not, go by elements.
    const int64_t vec = 16 / DTypeBytes(x.dtype);
    if (!RouterStep(part, grad, rows, cols, 1, cols % vec == 0 ? &p->steps_unaligned : &p->steps)) return nullptr;
    if (cols % vec == 0) {
      if (!RouterStep(part, grad, rows, cols, vec, &p->steps)) return nullptr;
      p->aligned_inputs = {In(main.inputs[0]).index};
      if (grad) p->aligned_outputs = {Out(grad).index};
    }
    return p;
  }
  bool RouterStep(const OpDesc* part, const OpDesc* grad, int64_t rows, int64_t cols, int64_t vec, std::vector<LaunchStep>* steps) {
    const OpDesc& main  = grad ? *grad : *part;
    const TensorDesc& x = Input(main.inputs[0]);
    const int64_t vecs  = cols / vec;
    // A token's row over as many lanes as give each about eight elements: the reductions over the lanes, 15 shuffles over
    // 32 of them, then weigh little (65536 x 256 fp32: 32 us in all; with sixteen elements 34, fewer warps fit an SM).
    int64_t lanes = 1, per = 1;
    while (per < 8 / vec && per < vecs) per *= 2;
    while (lanes < 32 && lanes * per < vecs) lanes *= 2;
    while (lanes * per < vecs) per *= 2;
    LaunchStep s;
    const std::string name = std::string("router_loss_") + ShortName(x.dtype) + (vec > 1 ? "_v" : "_s") + "_n" + std::to_string(per);
    s.kernel = FindKernel(name);
    if (!s.kernel) return Fail("kernel " + name + " is missing") != nullptr;
    s.args = {In(main.inputs[0]), In(main.inputs[2]), In(main.inputs[1]), Out(part), Out(grad), I(rows), I(cols),
              Constant(main.inputs[2]), I(lanes)};
    // A CTA per part of the loss, in warps enough for its tokens.
    const int64_t parts = BalanceParts(rows), most = per * vec > 16 ? 8 : 16;
    int64_t warps = 1;
    while (warps < most && warps * (32 / lanes) * parts < rows) warps *= 2;
    s.block[0] = (unsigned)(32 * warps);
    s.grid[0]  = (unsigned)parts;
    steps->push_back(s);
    return true;
  }

  std::unique_ptr<CompiledGroup> PlanCounts(const OpDesc& op) {
    const TensorDesc& index = Input(op.inputs[0]);
    auto p = NewPlan("expert_counts");
    LaunchStep s, zero;
    s.kernel    = FindKernel("expert_counts");
    zero.kernel = FindKernel("expert_zero");
    if (!s.kernel || !zero.kernel) return Fail("kernel expert_counts is missing");
    const int64_t choices = index.numel();
    s.args = {In(op.inputs[0]), In(op.inputs[1]), Out(&op), I(choices), I(index.shape.back()),
              I((int64_t)Attr(op, "num_experts")), I(index.dtype == DType::kInt64 ? 1 : 0), Constant(op.inputs[1])};
    s.block[0] = (unsigned)std::min<int64_t>(1024, RoundUp(choices, 32));
    // One CTA up to 4096 choices; a cluster of 8, which needs no cleared counts, up to 65536; then CTAs of 4096 choices each,
    // 128 at most (level with 8192).  The cluster saves the host a launch, which is what counts, loss and gradient called one
    // after the other wait for: 12.1 us against 14.7 from 8192 to 65536 choices.  On the device it is level or slower: the
    // counts alone 3.4 us against 3.2 at 16384 choices, 4.0 against 3.3 at 65536; the three ops replayed as a graph 10.3
    // against 10.3 up to 32768 and 12.3 against 10.3 (64 experts) beyond; at 131072 choices it loses 1.7 us.
    int64_t ctas = 1;
    if (choices > 4096) ctas = choices <= 65536 ? 8 : std::min<int64_t>(128, CeilDiv(choices, 4096));
    if (ctas > 1 && choices <= 65536) s.cluster = (unsigned)ctas;
    s.grid[0] = (unsigned)ctas;
    if (ctas > 1 && !s.cluster) {
      zero.args     = {Out(&op), I((int64_t)Attr(op, "num_experts"))};
      zero.block[0] = 256;
      p->steps.push_back(zero);
    }
    p->steps.push_back(s);
    return p;
  }
};

}  // namespace

std::unique_ptr<CompiledGroup> MatchLossGroup(const GroupDesc& g, const DeviceInfo& dev, std::string* err) {
  std::string local;
  return LossMatcher(g, dev, err ? err : &local).Run();
}

}  // namespace cinn_b200
