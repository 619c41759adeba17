// The loss operators through include/cinn_b200_frontend.hpp: a policy step with a distillation term and a router's loss.
//   argv[1] = "plan": no GPU is touched, prints the groups
//   argv[1] = "run" : executes on device 0 and checks the losses and one gradient row against doubles
#include <cmath>
#include <cstdio>
#include <cstring>
#include <random>
#include <vector>

#include "cinn_b200_frontend.hpp"

using cinn_b200::frontend::CinnComputation;
using cinn_b200::frontend::NetBuilder;

int main(int argc, char** argv) {
  const bool run = argc > 1 && !strcmp(argv[1], "run");
  const int R = 5, V = 301, K = 4, E = 6;
  try {
    NetBuilder b("losses");
    auto x = b.CreateInput("float32", {R, V}, "x");
    auto a = b.CreateInput("int64", {R}, "a");
    auto w = b.CreateInput("float32", {R}, "w"), old = b.CreateInput("float32", {R}, "old"), adv = b.CreateInput("float32", {R}, "adv");
    auto t = b.CreateInput("float32", {R, K}, "t");
    auto i = b.CreateInput("int32", {R, K}, "i");
    auto g = b.CreateInput("float32", {R, E}, "g");
    auto gi = b.CreateInput("int32", {R, 2}, "gi");
    auto lp   = b.TokenLogprob(x, a);
    auto loss = b.PolicyLoss(x, a, old, old, adv, w, 0.2f, 0.28f, 0.1f);
    auto dx   = b.PolicyLossGrad(x, a, old, old, adv, w, 0.2f, 0.28f, 0.1f);
    auto dl   = b.DistillLoss(x, t, i, w, 2.0f);
    auto ddx  = b.DistillLossGrad(x, t, i, w, 2.0f);
    auto c    = b.ExpertCounts(gi, w, E);
    auto bl   = b.BalanceLoss(g, c, w);
    auto dg   = b.BalanceLossGrad(g, c, w);
    auto dlp  = b.TokenLogprobGrad(x, a, w, 0.5f);
    auto comp = CinnComputation::BuildAndCompile(run ? 0 : -1, b, {lp, loss, dx, dl, ddx, c, bl, dg, dlp});
    int rows = 0;
    for (auto& p : comp->GroupPatterns()) {
      printf("group: %s\n", p.c_str());
      rows += p.find("row_loss") == 0;
    }
    if (rows != 3 || comp->GroupPatterns().size() != 5) {
      printf("FAILED: the loss ops were not merged as expected\n");
      return 1;
    }
    try {
      b.PolicyLoss(x, a, old, old, adv, w, 2.0f);
      printf("FAILED: clip_low = 2 was accepted\n");
      return 1;
    } catch (const std::exception&) {
    }
    if (!run) {
      printf("PLANNED\n");
      return 0;
    }
    std::mt19937 rng(3);
    std::normal_distribution<float> n01;
    std::vector<float> hx(R * V), hw(R, 0.5f), hold(R), hadv(R), ht(R * K), hg(R * E);
    std::vector<long long> ha(R);
    std::vector<int> hi(R * K), hgi(R * 2);
    for (auto& v : hx) v = 2.0f * n01(rng);
    for (auto& v : ht) v = n01(rng);
    for (auto& v : hg) v = n01(rng);
    for (auto& v : hadv) v = n01(rng);
    for (int r = 0; r < R; ++r) ha[r] = rng() % V;
    for (auto& v : hi) v = rng() % V;
    for (auto& v : hgi) v = rng() % E;
    hw[R - 1] = 0.0f;
    std::vector<double> lse(R);
    for (int r = 0; r < R; ++r) {
      double s = 0;
      for (int j = 0; j < V; ++j) s += std::exp((double)hx[r * V + j]);
      lse[r]  = std::log(s);
      hold[r] = (float)(hx[r * V + ha[r]] - lse[r] - 0.1);  // ratio e^0.1: inside the clip
    }
    comp->SetTensorData("x", hx.data(), hx.size() * 4);
    comp->SetTensorData("a", ha.data(), ha.size() * 8);
    comp->SetTensorData("w", hw.data(), hw.size() * 4);
    comp->SetTensorData("old", hold.data(), hold.size() * 4);
    comp->SetTensorData("adv", hadv.data(), hadv.size() * 4);
    comp->SetTensorData("t", ht.data(), ht.size() * 4);
    comp->SetTensorData("i", hi.data(), hi.size() * 4);
    comp->SetTensorData("g", hg.data(), hg.size() * 4);
    comp->SetTensorData("gi", hgi.data(), hgi.size() * 4);
    comp->Execute();
    std::vector<float> rl(R), rlp(R), rdx(R * V), rbl(1);
    std::vector<int> rc(E);
    comp->GetTensorData(lp.id, rlp.data(), R * 4);
    comp->GetTensorData(loss.id, rl.data(), R * 4);
    comp->GetTensorData(dx.id, rdx.data(), rdx.size() * 4);
    comp->GetTensorData(c.id, rc.data(), E * 4);
    comp->GetTensorData(bl.id, rbl.data(), 4);
    for (int r = 0; r < R; ++r) {
      const double l = hx[r * V + ha[r]] - lse[r], ratio = std::exp(l - hold[r]), gap = hold[r] - l;
      const double want = hw[r] * (0.1 * (std::exp(gap) - gap - 1) - ratio * hadv[r]);
      const double slope = hw[r] * (0.1 * (1 - std::exp(gap)) - ratio * hadv[r]);
      if (std::fabs(rlp[r] - l) > 1e-5 || std::fabs(rl[r] - want) > 1e-5) {
        printf("FAILED: row %d: log-probability %g for %g, loss %g for %g\n", r, rlp[r], l, rl[r], want);
        return 1;
      }
      for (int j = 0; j < V; ++j) {
        const double d = slope * ((j == ha[r]) - std::exp(hx[r * V + j] - lse[r]));
        if (std::fabs(rdx[r * V + j] - d) > 1e-5) {
          printf("FAILED: gradient (%d, %d): %g for %g\n", r, j, rdx[r * V + j], d);
          return 1;
        }
      }
    }
    std::vector<int> want_c(E, 0);
    for (int r = 0; r < R - 1; ++r)
      for (int k = 0; k < 2; ++k) ++want_c[hgi[r * 2 + k]];
    double want_bl = 0;
    for (int r = 0; r < R; ++r) {
      double s = 0, f = 0;
      for (int e = 0; e < E; ++e) s += std::exp((double)hg[r * E + e]);
      for (int e = 0; e < E; ++e) f += want_c[e] * std::exp((double)hg[r * E + e]) / s;
      want_bl += E * hw[r] * f / (2.0 * (R - 1));
    }
    if (rc != want_c || std::fabs(rbl[0] - want_bl) > 1e-5) {
      printf("FAILED: balance loss %g for %g\n", rbl[0], want_bl);
      return 1;
    }
    printf("PASSED\n");
    return 0;
  } catch (const std::exception& e) {
    printf("FAILED: %s\n", e.what());
    return 1;
  }
}
