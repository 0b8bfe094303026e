// linear_parts.cpp -- how a layer's weights are packed in parts (csrc/linear.hip), on the CPU: the launches of launch_linear are recorded in place of
// being made, and every 16 bytes that the packing reads have to lie in the array of weights.
#include <hip/hip_runtime.h>

#include <cstdio>
#include <cstdlib>
#undef hipLaunchKernelGGL
#define hipLaunchKernelGGL(kernel, grid, block, lds, stream, ...) record(grid, __VA_ARGS__)

#include "nn.hpp"

namespace acehip {
static const int8_t* g_weights;
static u64 g_bytes;                      // of the array
static u32 g_packs, g_products, g_outputs, g_bad;
static u64 linear_pack_from_of(u64 at, u32 n_out, u64 ld_w, u32 n_in);
// linear_pack_kernel
template <class V>
static void record(dim3 grid, const int8_t* w, u64 ld_w, u32 n_in, u32 n_out, u32 steps, u32 n_frags, V*) {
  ++g_packs;
  const u64 start = w - g_weights;
  if (grid.x * 4 < n_frags || n_frags != (n_out + 15) / 16 * steps || steps * 64 < n_in) ++g_bad;
  for (u32 f = 0; f < n_frags; ++f)
    for (u32 lane = 0; lane < 64; ++lane) {
      const u32 j = (f / steps) * 16 + (lane & 15u), k = (f % steps) * 64 + 16 * (lane >> 4);
      if (j >= n_out || k >= n_in) continue;
      const u64 at = j * ld_w + k, from = linear_pack_from_of(at, n_out, ld_w, n_in);
      if (from > at || at - from > 15 || start + from + 16 > g_bytes) ++g_bad;
    }
}
// the kernels of the product, either form
template <class... Rest>
static void record(dim3, const DevCtx&, const LinearArgs& a, Rest...) {
  ++g_products;
  if (a.w != g_weights + (u64)g_outputs * a.ld_w || a.out.d != (u64*)0 + (u64)g_outputs * a.out.col) ++g_bad;
  g_outputs += a.n_out;
}
}  // namespace acehip
#include "linear.hip"
namespace acehip {
static u64 linear_pack_from_of(u64 at, u32 n_out, u64 ld_w, u32 n_in) { return linear_pack_from(at, n_out, ld_w, n_in); }
}  // namespace acehip

int main(int argc, char** argv) {
  using namespace acehip;
  if (argc != 7) return 2;
  const auto number = [&](int i) { return (u32)strtoul(argv[i], nullptr, 10); };
  DevCtx c{};
  c.N = number(1);
  LinearArgs a{};
  a.rows = number(2), a.n_in = number(3), a.n_out = number(4), a.n_comp = 3, a.level = a.n_limbs = 2;
  a.ld_w = number(5);
  a.out.col = a.in.col = 2 * c.N;
  a.wide_primes = true;
  g_bytes = (a.n_out - 1) * a.ld_w + a.n_in;
  a.w = g_weights = (const int8_t*)malloc(1);
  int ws;
  launch_linear(c, &c, 1, a, &ws, number(6), nullptr);
  printf("packs %u products %u outputs %u bad %u\n", g_packs, g_products, g_outputs, g_bad);
  return g_bad != 0 || g_outputs != a.n_out;
}
