// The waits of csrc/linear/waits.cuh by the 32 lanes of a warp, a host thread each (SOURCE: its text without its include).
//   lanes  lanes see the ends of two barriers' phases at different looks: all of them come through, together
//   limit  a phase that does not come is reported after the limit, and every wait behind it is over after one poll
//   sent   what other CTAs send is waited for by lanes of a CTA that gave up, too, and no longer than four limits
// Exit status 0: right; 2: wrong; 3: a whole-warp operation meets lanes that are elsewhere.
#include <atomic>
#include <chrono>
#include <condition_variable>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <mutex>
#include <string>
#include <thread>
#include <vector>

#define __device__
#define __forceinline__ inline
struct Index { unsigned x; };
static Index blockIdx{7};
static uint32_t atomicCAS(uint32_t* p, uint32_t want, uint32_t v) {
  __atomic_compare_exchange_n(p, &want, v, false, __ATOMIC_ACQ_REL, __ATOMIC_ACQUIRE);
  return want;
}
static void __nanosleep(unsigned) {}
static uint64_t globaltimer_ns() { return std::chrono::steady_clock::now().time_since_epoch().count(); }

// ---- the warp
static std::mutex g_m;
static std::condition_variable g_cv;
static int g_here, g_left;
static uint64_t g_round;
static uint32_t g_votes, g_result;
static std::string g_op;
static thread_local unsigned lane_;
static void stuck(const std::string& op) { printf("%s meets lanes that are elsewhere\n", op.c_str()); fflush(stdout); _Exit(3); }
static uint32_t meet(const char* op, bool vote) {
  std::unique_lock<std::mutex> l(g_m);
  if (g_here == 0) { g_op = op; g_votes = 0; }
  if (g_op != op || g_left > 0) stuck(op);
  if (vote) g_votes |= 1u << lane_;
  const uint64_t round = g_round;
  if (++g_here == 32) {
    g_here = 0;
    g_result = g_votes;
    ++g_round;
    g_cv.notify_all();
  } else {
    g_cv.wait(l, [&] { return g_round != round; });
  }
  return g_result;
}
static void leave() {
  std::lock_guard<std::mutex> l(g_m);
  ++g_left;
  if (g_here > 0) stuck(g_op);
}
static void __syncwarp() { meet("__syncwarp", false); }
static bool __all_sync(uint32_t, bool v) { return meet("__all_sync", v) == 0xFFFFFFFFu; }
static bool __any_sync(uint32_t, bool v) { return meet("__any_sync", v) != 0; }

// ---- barriers: one whose phase ends at a lane's look number `at`
struct Bar { std::atomic<unsigned> at[32], looks[32]; };
static Bar* bar_of(uint64_t* b) { return reinterpret_cast<Bar*>(b); }
static bool look(uint64_t* b) { return ++bar_of(b)->looks[lane_] >= bar_of(b)->at[lane_]; }
static bool mbar_test(uint64_t* b, uint32_t) { return look(b); }
static bool mbar_try_wait(uint64_t* b, uint32_t) { return look(b); }

#include SOURCE

using namespace mono::lin;

template <typename F>
static void warp(F f) {
  g_left = g_here = 0;
  std::vector<std::thread> lanes;
  for (unsigned i = 0; i < 32; ++i) lanes.emplace_back([&, i] { lane_ = i; f(); leave(); });
  for (auto& t : lanes) t.join();
}

int main(int, char** argv) {
  const std::string name = argv[1];
  uint32_t stop = 0, status[2] = {0, 0};
  const Waits waits{&stop, status};
  static Bar a, b;
  uint64_t *pa = reinterpret_cast<uint64_t*>(&a), *pb = reinterpret_cast<uint64_t*>(&b);
  if (name == "lanes") {
    // looks at which even and odd lanes see the first and the second barrier's phase end
    const unsigned at[][4] = {{1, 1, 1, 1}, {1, 2, 1, 1}, {1, 1, 1, 2}, {3, 1, 1, 1}, {1, 2, 2, 1}, {2, 1, 2, 1}, {2, 2, 1, 4}, {5, 1, 1, 9}};
    for (const auto& t : at)
      for (int form = 0; form < 2; ++form) {
        for (int i = 0; i < 32; ++i) {
          a.looks[i] = b.looks[i] = 0;
          a.at[i] = t[i & 1];
          b.at[i] = t[2 + (i & 1)];
        }
        std::atomic<int> unseen{0};
        warp([&] {
          if (form == 0) waits.wait(pa, 0, pb, 0);
          else waits.wait_warp(pa, 0, pb, 0);
          if (a.looks[lane_] < a.at[lane_] || b.looks[lane_] < b.at[lane_]) ++unseen;
          meet("what follows", false);
        });
        if (unseen || stop || status[0]) { printf("came through early\n"); return 2; }
      }
    return 0;
  }
  if (name == "limit") {
    const Waits brief{&stop, status, 20000000};
    for (int i = 0; i < 32; ++i) {
      a.looks[i] = b.looks[i] = 0;
      a.at[i] = b.at[i] = ~0u;
    }
    const uint64_t t0 = globaltimer_ns();
    warp([&] {
      brief.wait(pa, 0);
      meet("what follows", false);
      if (lane_ == 0) for (int i = 0; i < 32; ++i) a.looks[i] = 0;
      meet("the next", false);
      for (int i = 0; i < 100; ++i) {
        brief.wait(pa, i & 1);
        brief.wait(pa, i & 1, pb, i & 1);
        brief.wait_warp(pa, i & 1);
        brief.wait_warp(pa, i & 1, pb, i & 1);
        brief.wait_lane(pb, i & 1);
      }
    });
    const uint64_t t = globaltimer_ns() - t0;
    if (t < 20000000 || !stop || status[0] != kWaitTimeout || status[1] != blockIdx.x) { printf("not reported: %u, %u\n", status[0], status[1]); return 2; }
    for (int i = 0; i < 32; ++i)             // a poll each, and a look in front of it where there are two barriers
      if (a.looks[i] > 600 || b.looks[i] > 500) { printf("%u and %u looks\n", unsigned(a.looks[i]), unsigned(b.looks[i])); return 2; }
    return 0;
  }
  if (name == "sent") {
    const Waits brief{&stop, status, 5000000};
    stop = 1;
    for (int i = 0; i < 32; ++i) {
      a.at[i] = 1000 + 7 * i;
      b.at[i] = ~0u;
    }
    std::atomic<int> unseen{0};
    uint64_t t = 0;
    warp([&] {
      brief.wait_sent(pa, 0);
      if (a.looks[lane_] < a.at[lane_]) ++unseen;
      meet("what follows", false);
      const uint64_t t0 = globaltimer_ns();
      brief.wait_sent(pb, 0);
      if (lane_ == 0) t = globaltimer_ns() - t0;
    });
    if (unseen) { printf("not waited for\n"); return 2; }
    return t >= 20000000 && status[0] == kWaitTimeout ? 0 : 2;
  }
  return 2;
}
