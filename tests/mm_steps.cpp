// Every order in which the warps of an FP8 product that quantises its tokens inside
// (wohper_b200/csrc/fp8_gemm.cu) can take their steps, on a model of its barriers: a
// wait by parity passes when the barrier's phase in progress has the other parity.
//
//   mm_steps RULE TILES FOLD   (tests/test_fp8_gemm_steps.py)
//
// RULE: "kernel" (mm_steps.cuh), or a planted one on a barrier a stage: "both" waits for
// the fill before the last and then for the last, "last" for the last alone.  Prints
// "ok", "stuck" (no warp can go on) or "overwritten" (a fill of a stage that still has to be read).
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <string>
#include <unordered_set>
#include <vector>

#include "../wohper_b200/csrc/mm_steps.cuh"

namespace {

constexpr int kStages = 4, kWarps = 8, kAcc = 2;
using Free = wh::MmFree<kStages, 2 * kStages>;

enum Kind { kWait, kWeight, kTokens, kFull, kFree, kTaken, kSum, kTake };
// kWait: free[bar] has left parity; kWeight/kTokens: fill tile at; kFull: tile at is whole; kFree: its products arrive on free[bar];
// kTaken: sum at - kAcc has been taken; kSum: sum at is complete; kTake: wait for sum at, arrive
struct Op {
  Kind kind;
  int at, bar, parity;
};

struct State {
  int free[2 * kStages], full[kStages][2], acc_full[kAcc], taken[kAcc][kWarps];
  int consumed;  // tiles whose products have arrived
};

std::vector<std::vector<Op>> agents;
int tiles, fold;

bool fill_is_safe(const State& s, int tile) { return tile < kStages || s.consumed > tile - kStages; }

// Runs op; 0: it waits, 1: done, 2: overwrites
int step(State& s, const Op& op, int agent) {
  const int st = op.at % kStages;
  switch (op.kind) {
    case kWait:
      return (s.free[op.bar] & 1) != op.parity;
    case kWeight:
      if (!fill_is_safe(s, op.at)) return 2;
      ++s.full[st][0];
      return 1;
    case kTokens:
      if (!fill_is_safe(s, op.at)) return 2;
      ++s.full[st][1];
      return 1;
    case kFull: {  // a phase ends when both have arrived
      const int phase = s.full[st][0] < s.full[st][1] ? s.full[st][0] : s.full[st][1];
      return (phase & 1) != ((op.at / kStages) & 1);
    }
    case kFree:
      ++s.free[op.bar];
      s.consumed = op.at + 1;
      return 1;
    case kTaken: {
      int n = 1 << 20;
      for (int w = 0; w < kWarps; ++w) n = s.taken[op.at % kAcc][w] < n ? s.taken[op.at % kAcc][w] : n;
      return (n & 1) != ((op.at / kAcc - 1) & 1);
    }
    case kSum:
      ++s.acc_full[op.at % kAcc];
      return 1;
    case kTake:
      if ((s.acc_full[op.at % kAcc] & 1) == ((op.at / kAcc) & 1)) return 0;
      ++s.taken[op.at % kAcc][agent];
      return 1;
  }
  return 0;
}

struct Node {  // the places in the programs; the barriers follow from them
  State s;
  unsigned char pc[kWarps + 2];
};

}  // namespace

int main(int argc, char** argv) {
  if (argc != 4) return 2;
  const std::string rule = argv[1];
  tiles = std::atoi(argv[2]);
  fold = std::atoi(argv[3]);
  auto waits = [&](std::vector<Op>& p, int g, bool own) {
    if (rule == "kernel") {
      if (g >= kStages) p.push_back({kWait, g, Free::bar(g - kStages), (int)Free::parity(g - kStages)});
      return;
    }
    if (own && rule == "both" && g >= 2 * kStages) p.push_back({kWait, g, g % kStages, (g / kStages) & 1});
    if (g >= kStages) p.push_back({kWait, g, g % kStages, (g / kStages - 1) & 1});
  };
  // the quantising warps: tile by tile, sums taken where the products would wait for it
  for (int w = 0; w < kWarps; ++w) {
    std::vector<Op> p;
    int c0 = 0, sum = 0;
    for (int g = w; g < tiles; g += kWarps) {
      for (; g - c0 >= kAcc * fold; c0 += fold) p.push_back({kTake, sum++, 0, 0});
      waits(p, g, true);
      p.push_back({kTokens, g, 0, 0});
    }
    for (; c0 < tiles; c0 += fold) p.push_back({kTake, sum++, 0, 0});
    agents.push_back(p);
  }
  // the weight's warp
  std::vector<Op> p;
  for (int g = 0; g < tiles; ++g) {
    waits(p, g, false);
    p.push_back({kWeight, g, 0, 0});
  }
  agents.push_back(p);
  // the products
  p.clear();
  for (int c0 = 0, sum = 0; c0 < tiles; c0 += fold, ++sum) {
    if (sum >= kAcc) p.push_back({kTaken, sum, 0, 0});
    for (int g = c0; g < tiles && g < c0 + fold; ++g) {
      p.push_back({kFull, g, 0, 0});
      p.push_back({kFree, g, rule == "kernel" ? Free::bar(g) : g % kStages, 0});
    }
    p.push_back({kSum, sum, 0, 0});
  }
  agents.push_back(p);

  std::unordered_set<std::string> seen;
  std::vector<Node> todo(1);
  std::memset(&todo[0], 0, sizeof(Node));
  while (!todo.empty()) {
    Node n = todo.back();
    todo.pop_back();
    bool any = false, done = true;
    for (size_t a = 0; a < agents.size(); ++a) {
      if (n.pc[a] == agents[a].size()) continue;
      done = false;
      Node m = n;
      const int r = step(m.s, agents[a][m.pc[a]], (int)a);
      if (r == 2) return std::puts("overwritten"), 0;
      if (r == 0) continue;
      any = true;
      ++m.pc[a];
      if (seen.insert(std::string(reinterpret_cast<char*>(m.pc), sizeof(m.pc))).second) todo.push_back(m);
    }
    if (!any && !done) return std::puts("stuck"), 0;
  }
  std::puts("ok");
  return 0;
}
