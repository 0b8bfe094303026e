// san_nn.cpp -- argument checks of the operators on ciphertexts (csrc/api_nn.cpp) under sanitizers: random calls on a context without a device, which
// are refused or say that there is no device.  Built by `make -C oracle asan_nn` and `tsan_nn` from the host pass of the product's sources; one thread, then four,
// each with a context of its own.
#include <cstdio>
#include <random>
#include <thread>
#include <vector>

#include "acehip.h"

static int calls(uint32_t N, unsigned seed, int rounds) {
  acehip_ctx* c = acehip_ctx_create_host(N, 4, 60, 50, 2);
  if (!c) return 1;
  std::mt19937_64 rng(seed);
  int bad = 0, ran = 0;
  const auto one_of = [&](std::initializer_list<uint64_t> v) { return v.begin()[rng() % v.size()]; };
  const auto count = [&] { return (uint32_t)one_of({0, 1, 1, 2, 2, 3, 4, 5, 17, 64, rng() % 8, rng() % 8, rng() % 2000, 1ull << 20, 1ull << 31, (1ull << 32) - 1}); };
  const uint64_t poly = 3ull * N;
  const auto at = [&] { return (uint64_t*)one_of({0, 1 << 20, (1 << 20) + 4, (1 << 20) + 8 * (rng() % 4096), (1ull << 40) + 8 * poly * (rng() % 64), 1ull << 50, ~0ull - 7}); };
  const auto mat = [&] {
    const auto stride = [&] { return (size_t)one_of({0, poly, poly * 2, poly * 3, poly * (rng() % 100), poly * 5000, rng() % 5000, 1ull << 40, 1ull << 61, ~0ull}); };
    return acehip_mat{at(), stride(), stride(), stride(), stride()};
  };
  const auto stride = [&] { return (size_t)one_of({0, poly, 10, 17, 100, rng() % 10000, 1ull << 61, ~0ull}); };
  for (int i = 0; i < rounds; ++i) {
    if (i % 64 == 0) {  // an arena or none, and a selection of its replicas
      const acehip_arena_cfg cfg{(void*)(1ull << 40), 1ull << 30, 1ull << 31, 3, (void*)(1ull << 40), (void*)((1ull << 40) + (1 << 28)), 8};
      if (rng() % 2 && acehip_ctx_set_arena(c, &cfg) == 0) acehip_ctx_select(c, rng() % 3, 1);
    }
    const acehip_mat m[5] = {mat(), mat(), mat(), mat(), mat()};
    const auto some = [&](int k) { return rng() % 16 ? &m[k] : nullptr; };
    const uint32_t level = rng() % 6, pos0 = one_of({0, 0, 0, 1, 2, 5, ~0u}), n = one_of({0, 1, 1, 2, 3, 6, ~0u});
    std::vector<double> freq(64, 0.5);
    std::vector<uint32_t> axis(64);
    for (auto& a : axis) a = rng() % 3;
    int rc = 0;
    switch (rng() % 6) {
      case 0: rc = acehip_linear_i8(c, some(0), some(1), (const int8_t*)at(), stride(), count(), count(), count(), count(), (const int64_t*)at(), at(), stride(), level, pos0, n, nullptr); break;
      case 1: rc = acehip_rope_messages(c, (double*)at(), (double*)at(), stride(), (const double*)at(), stride(), count(), freq.data(), axis.data(), rng() % 65, rng() % 10, nullptr); break;
      case 2: rc = acehip_rope(c, some(0), some(1), at(), at(), stride(), stride(), count(), count(), count(), count(), rng() % 2, level, pos0, n, nullptr); break;
      case 3: rc = acehip_linattn_scores(c, some(0), some(1), some(2), count(), count(), count(), count(), count(), rng() % 2, level, pos0, n, nullptr); break;
      case 4: rc = acehip_linattn_out(c, some(0), some(1), some(2), some(3), some(4), count(), count(), count(), count(), count(), count(), (const int64_t*)at(), (const int64_t*)at(), rng() % 2, level, pos0, n, nullptr); break;
      case 5: rc = acehip_linattn_state(c, some(0), some(1), some(2), some(3), count(), count(), count(), count(), count(), (const int64_t*)at(), (const int64_t*)at(), level, pos0, n, nullptr); break;
    }
    ran += rc == ACEHIP_ENODEV;
    if (rc != ACEHIP_EINVAL && rc != ACEHIP_ENODEV) {
      fprintf(stderr, "call %d of seed %u returned %d: %s\n", i, seed, rc, acehip_last_error());
      ++bad;
    }
  }
  if (ran == 0 || ran == rounds) ++bad;
  acehip_ctx_destroy(c);
  return bad;
}

int main() {
  int bad = calls(64, 1, 60000);
  int of[4] = {};
  std::vector<std::thread> threads;
  for (int t = 0; t < 4; ++t) threads.emplace_back([&of, t] { of[t] = calls(t % 2 ? 64 : 1024, 2 + t, 20000); });
  for (auto& t : threads) t.join();
  for (int b : of) bad += b;
  printf(bad ? "san_nn: %d failures\n" : "san_nn: OK\n", bad);
  return bad != 0;
}
