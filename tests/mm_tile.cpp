// Four epilogue warps of an FP8 product (wohper_b200/csrc/fp8_gemm.cu) as threads: every
// one takes its tiles by mm_tile (mm_steps.cuh), and at tile BAD the wait of WARP runs out.
//
//   mm_tile AGREE BAD WARP   (tests/test_fp8_gemm_steps.py)
//
// AGREE: "kernel", or "alone" (planted): each warp goes by its own wait.  The barriers give
// up after a second here.  Prints "left after N" (all four stored N tiles and returned) or
// "waits" (one waited at a barrier that the others never came to).
#include <atomic>
#include <chrono>
#include <condition_variable>
#include <cstdio>
#include <cstdlib>
#include <mutex>
#include <string>
#include <thread>
#include <vector>

#include "../wohper_b200/csrc/mm_steps.cuh"

constexpr int kWarps = 4, kTiles = 5, kSums = 3;

struct Barrier {
  std::mutex mu;
  std::condition_variable cv;
  int here = 0, phase = 0;
  bool all = true, result = true;
  std::atomic<bool> lost{false};
  bool vote(bool ok) {
    std::unique_lock<std::mutex> lock(mu);
    const int mine = phase;
    all = all && ok;
    if (++here == kWarps) {
      result = all;
      all = true;
      here = 0;
      ++phase;
      cv.notify_all();
    } else if (!cv.wait_for(lock, std::chrono::seconds(1), [&] { return phase != mine || lost; }) || phase == mine) {
      lost = true;
      cv.notify_all();
    }
    return result;
  }
};

int main(int argc, char** argv) {
  if (argc != 4) return 2;
  const bool alone = std::string(argv[1]) == "alone";
  const int bad = std::atoi(argv[2]), who = std::atoi(argv[3]);
  Barrier bar;
  int stored[kWarps] = {};
  std::vector<std::thread> warps;
  for (int w = 0; w < kWarps; ++w)
    warps.emplace_back([&, w] {
      bool ok = true;
      for (int tile = 0; ok && tile < kTiles && !bar.lost; ++tile) {
        int sums = 0;
        ok = wh::mm_tile(
            8 * kSums - 1, 8, [&](bool first) { const bool fine = first == (sums == 0); return ++sums, fine && !(tile == bad && w == who && sums == 2); },
            [&](bool fine) { return alone ? fine : bar.vote(fine); },
            [&] {
              bar.vote(true);
              bar.vote(true);
              ++stored[w];
            });
      }
    });
  for (auto& t : warps) t.join();
  bool same = true;
  for (int w = 1; w < kWarps; ++w) same = same && stored[w] == stored[0];
  if (bar.lost || !same)
    std::puts("waits");
  else
    std::printf("left after %d\n", stored[0]);
  return 0;
}
