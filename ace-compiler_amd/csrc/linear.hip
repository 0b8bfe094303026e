// linear.hip -- int8 linear layers on ciphertexts: y_j = tok * mul_j * sum_i w_ji x_i mod q on every limb and coefficient.
#include "nn.hpp"

namespace acehip {

// One coefficient per lane, kJ outputs: residues split at 31 bits, so that each half times a weight is one multiply-add into a signed
// 64-bit sum (|sum| <= 2^31 * 2^7 * 2^16 inputs).
constexpr u32 kJ = 8;
__global__ __launch_bounds__(256) void linear_i8_kernel(DevCtx c, LinearArgs a, u32 n_blocks, u32 j_blocks) {
  u32 b = blockIdx.x;
  const u32 nb = b % n_blocks;
  b /= n_blocks;
  const u32 jb = b % j_blocks;
  b /= j_blocks;
  const u32 comp = b % a.n_comp, row = b / a.n_comp, rep = c.rep0 + blockIdx.z;
  const u32 pos = a.pos0 + blockIdx.y, gi = limb_prime(pos, a.level, c.L);
  const u32 n = nb * 256 + threadIdx.x;
  if (!owns(c, gi) || n >= c.N) return;
  const DevPrime P = c.primes[gi];
  const u64 off = (u64)pos * c.N + n;
  const u64* x = reb(c, a.in.d, rep) + row * a.in.row + comp * a.in.comp + off;
  const int8_t* w = reb(c, a.w, rep);
  const int64_t* mul = reb(c, a.mul, rep);
  const u32 j0 = jb * kJ;
  int64_t lo[kJ] = {}, hi[kJ] = {};
  for (u32 i = 0; i < a.n_in; ++i) {
    const u64 v = x[i * a.in.col];
    const int32_t vl = (int32_t)(v & 0x7fffffffu), vh = (int32_t)(v >> 31);
#pragma unroll
    for (u32 t = 0; t < kJ; ++t) {
      const int32_t wv = w[(u64)min(j0 + t, a.n_out - 1) * a.ld_w + i];
      lo[t] += (int64_t)vl * wv;
      hi[t] += (int64_t)vh * wv;
    }
  }
  u64* y = reb(c, a.out.d, rep) + row * a.out.row + comp * a.out.comp + off;
  const u64 tok = a.tok ? reb(c, a.tok, rep)[row * a.tok_stride + off] : 0;
  const u64 c31 = signed_mod(1ll << 31, P.q, P.prec128_hi);
  for (u32 t = 0; t < kJ && j0 + t < a.n_out; ++t) {
    u64 v = add_mod(mul_mod(signed_mod(hi[t], P.q, P.prec128_hi), c31, P), signed_mod(lo[t], P.q, P.prec128_hi), P.q);
    if (mul) v = mul_mod(v, signed_mod(mul[j0 + t], P.q, P.prec128_hi), P);
    if (a.tok) v = mul_mod(v, tok, P);
    y[(j0 + t) * a.out.col] = v;
  }
}

void launch_linear_i8(const DevCtx& c, const LinearArgs& a, hipStream_t s) {
  const u32 n_blocks = (c.N + 255) / 256, j_blocks = (a.n_out + kJ - 1) / kJ;
  hipLaunchKernelGGL(linear_i8_kernel, dim3(n_blocks * j_blocks * a.n_comp * a.rows, a.n_limbs, c.nrep), dim3(256), 0, s, c, a, n_blocks, j_blocks);
}

}  // namespace acehip
