// rope.hip -- rotary positions with several axes: the messages (angles) and the rotation of encrypted features.
#include "nn.hpp"

namespace acehip {

// The angle is one rounded product of doubles; cos and sin of that double (positions far out lose nothing more).
__global__ __launch_bounds__(256) void rope_messages_kernel(double* cos_out, double* sin_out, u64 out_stride, const double* pos, u64 pos_stride, u32 n_pos,
                                                            RopeAngles a) {
  const u32 t = blockIdx.x * 256 + threadIdx.x, i = blockIdx.y;
  if (t >= n_pos) return;
  double s, c;
  sincos(pos[a.axis[i] * pos_stride + t] * a.freq[i], &s, &c);
  cos_out[i * out_stride + t] = c;
  sin_out[i * out_stride + t] = s;
}

void launch_rope_messages(double* cos_out, double* sin_out, u64 out_stride, const double* pos, u64 pos_stride, u32 n_pos, const RopeAngles& a, u32 n_pairs,
                          hipStream_t s) {
  hipLaunchKernelGGL(rope_messages_kernel, dim3((n_pos + 255) / 256, n_pairs), dim3(256), 0, s, cos_out, sin_out, out_stride, pos, pos_stride, n_pos, a);
}

__global__ __launch_bounds__(256) void rope_kernel(DevCtx c, RopeArgs a, u32 n_blocks) {
  u32 b = blockIdx.x;
  const u32 nb = b % n_blocks;
  b /= n_blocks;
  const u32 half = a.dim / 2;
  const u32 i = b % half, row = b / half, rep = c.rep0 + blockIdx.z;
  const u32 pos = a.pos0 + blockIdx.y, gi = limb_prime(pos, a.level, c.L);
  const u32 n = nb * 256 + threadIdx.x;
  if (!owns(c, gi) || n >= c.N) return;
  const DevPrime P = c.primes[gi];
  const u64 off = (u64)pos * c.N + n;
  const u64 tab = row * a.row_stride + i * a.pair_stride + off;
  const u64 C = reb(c, a.cosp, rep)[tab], S = reb(c, a.sinp, rep)[tab], nS = S ? P.q - S : 0;
  const u32 f0 = a.interleaved ? 2 * i : i, f1 = a.interleaved ? 2 * i + 1 : i + half;
  const u64* in = reb(c, a.in.d, rep) + row * a.in.row + off;
  u64* out = reb(c, a.out.d, rep) + row * a.out.row + off;
  for (u32 h = 0; h < a.n_heads; ++h)
    for (u32 k = 0; k < a.n_comp; ++k) {
      const u64* p = in + h * a.in.head + k * a.in.comp;
      u64* y = out + h * a.out.head + k * a.out.comp;
      const u64 x0 = p[f0 * a.in.col], x1 = p[f1 * a.in.col];
      U128 s0{0, 0}, s1{0, 0};
      mac128(s0, x0, C);
      mac128(s0, x1, nS);
      mac128(s1, x0, S);
      mac128(s1, x1, C);
      y[f0 * a.out.col] = reduce128(s0, P.q, P.prec128_lo, P.prec128_hi);
      y[f1 * a.out.col] = reduce128(s1, P.q, P.prec128_lo, P.prec128_hi);
    }
}

void launch_rope(const DevCtx& c, const RopeArgs& a, hipStream_t s) {
  const u32 n_blocks = (c.N + 255) / 256;
  hipLaunchKernelGGL(rope_kernel, dim3(n_blocks * (a.dim / 2) * a.rows, a.n_limbs, c.nrep), dim3(256), 0, s, c, a, n_blocks);
}

}  // namespace acehip
