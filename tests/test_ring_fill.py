"""A ring that a warp fills, one lane waiting for room: all lanes leave when that wait gives up.  On the CPU."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
#include <condition_variable>
#include <cstdio>
#include <mutex>
#include <thread>
#include <utility>
#include <vector>
#include "ring_drain.cuh"
constexpr int LANES = 4;
// a call that every lane of a warp has to make: stuck if one has left while others wait in it
struct Warp {
  std::mutex m;
  std::condition_variable cv;
  int waiting = 0, gone = 0, round = 0, value = 0, result = 0;
  bool stuck = false;
  void pass() { waiting = 0; ++round; result = value; cv.notify_all(); }
  int shuffle(int lane, int from, int v) {
    std::unique_lock<std::mutex> l(m);
    if (stuck) return -1;
    if (lane == from) value = v;
    const int mine = round;
    if (++waiting + gone == LANES) { stuck |= gone > 0; pass(); }
    cv.wait(l, [&] { return round != mine; });
    return stuck ? -1 : result;
  }
  void leave() {
    std::unique_lock<std::mutex> l(m);
    ++gone;
    if (waiting && waiting + gone == LANES) { stuck = true; pass(); }
  }
};
// `tiles` tiles, the copying lane's wait for fill `fails` giving up; `told`: the other lanes learn of it.
// Whether every lane came out with the fills asked for, in order.
static bool run(int tiles, int fails, bool told) {
  Warp w;
  std::vector<std::pair<bool, int>> fills;
  std::vector<int> asked(LANES, -1);
  std::vector<std::thread> lanes;
  for (int lane = 0; lane < LANES; ++lane)
    lanes.emplace_back([&, lane] {
      int c = 0;
      asked[lane] = ring_keys_values(
          tiles, [&](int n) { return w.shuffle(lane, n % LANES, 100 + n); },
          [&](bool is_value, int page) {
            bool ok = !w.stuck;
            if (lane == 0 && c++ == fails) ok = false;
            if (lane == 0 && ok) fills.push_back({is_value, page});
            return told ? w.shuffle(lane, 0, ok) == 1 : ok;
          });
      w.leave();
    });
  for (auto& t : lanes) t.join();
  std::vector<std::pair<bool, int>> want;
  for (int n = 0; n < tiles; ++n) {
    want.push_back({false, 100 + n});
    if (n) want.push_back({true, 99 + n});
  }
  if (tiles) want.push_back({true, 99 + tiles});
  if (fails >= 0 && fails < (int)want.size()) want.resize(fails);
  bool right = !w.stuck && fills == want;
  for (int a : asked) right &= a == (int)want.size();
  return right;
}
int main() {
  int cases = 0;
  for (int tiles = 0; tiles < 8; ++tiles)
    for (int fails = -1; fails < 2 * tiles; ++fails) {
      if (!run(tiles, fails, true)) { std::printf("%d %d\n", tiles, fails); return 1; }
      // (the model sees a lane that leaves alone)
      if (fails >= 0 && run(tiles, fails, false)) { std::printf("unseen %d %d\n", tiles, fails); return 1; }
      ++cases;
    }
  std::printf("%d\n", cases);
}
"""


def test_every_lane_leaves_with_the_one_that_waits(tmp_path):
    src, exe = tmp_path / "fill.cpp", tmp_path / "fill"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-pthread", "-I", os.path.join(ROOT, "binfer_b200", "csrc"), str(src),
                    "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert out.returncode == 0 and int(out.stdout) > 60, out.stdout
