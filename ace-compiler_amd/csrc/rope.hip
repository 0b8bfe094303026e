// rope.hip -- rotary positions with several axes: the messages (angles) and the rotation of encrypted features.
#include "nn.hpp"

namespace acehip {

// The angle is one rounded product of doubles; cos and sin of that double (positions far out lose nothing more).  Two positions a lane, whose
// latencies overlap.  Bound by its stores and its launch: 32768 positions of 64 pairs, 34 MB, in 8.5 us (4.0 TB/s); replayed in a graph 9.7 us, 10.4 with
// one position a lane, 8.3 without the functions.
__global__ __launch_bounds__(256) void rope_messages_kernel(double* cos_out, double* sin_out, u64 out_stride, const double* pos, u64 pos_stride, u32 n_pos,
                                                            RopeAngles a) {
  const u32 i = blockIdx.y, t0 = blockIdx.x * 512 + threadIdx.x;
  const double* p = pos + a.axis[i] * pos_stride;
  double s[2], c[2];
#pragma unroll
  for (u32 u = 0; u < 2; ++u) sincos(p[min(t0 + 256 * u, n_pos - 1)] * a.freq[i], &s[u], &c[u]);
#pragma unroll
  for (u32 u = 0; u < 2; ++u) {
    const u32 t = t0 + 256 * u;
    if (t >= n_pos) return;
    cos_out[i * out_stride + t] = c[u];
    sin_out[i * out_stride + t] = s[u];
  }
}

void launch_rope_messages(double* cos_out, double* sin_out, u64 out_stride, const double* pos, u64 pos_stride, u32 n_pos, const RopeAngles& a, u32 n_pairs,
                          hipStream_t s) {
  hipLaunchKernelGGL(rope_messages_kernel, dim3((n_pos + 511) / 512, n_pairs), dim3(256), 0, s, cos_out, sin_out, out_stride, pos, pos_stride, n_pos, a);
}

// A lane: one coefficient of a pair, whose table it reads once for up to `per` polynomials (heads and components); `parts` workgroups share a
// pair's polynomials.  Two products a result with 128-bit sums, reduced once: bound by memory, each word read and written once (16 heads of 64 at
// N = 16384, four limbs: 2.2 GB in 0.441 ms, 5.0 TB/s).
__global__ __launch_bounds__(256) void rope_kernel(DevCtx c, RopeArgs a, u32 n_blocks, u32 parts, u64 per) {
  u32 b = blockIdx.x;
  const u32 nb = b % n_blocks;
  b /= n_blocks;
  const u64 first = b % parts * per, end = min(first + per, (u64)a.n_heads * a.n_comp);
  b /= parts;
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
  u32 h = first / a.n_comp, k = first % a.n_comp;
  for (u64 p = first; p < end; ++p) {
    const u64* x = in + h * a.in.head + k * a.in.comp;
    u64* y = out + h * a.out.head + k * a.out.comp;
    const u64 x0 = x[f0 * a.in.col], x1 = x[f1 * a.in.col];
    U128 s0{0, 0}, s1{0, 0};
    mac128(s0, x0, C);
    mac128(s0, x1, nS);
    mac128(s1, x0, S);
    mac128(s1, x1, C);
    y[f0 * a.out.col] = reduce128(s0, P.q, P.prec128_lo, P.prec128_hi);
    y[f1 * a.out.col] = reduce128(s1, P.q, P.prec128_lo, P.prec128_hi);
    if (++k == a.n_comp) k = 0, ++h;
  }
}

void launch_rope(const DevCtx& c, const RopeArgs& a, hipStream_t s) {
  const u32 n_blocks = (c.N + 255) / 256;
  const u64 blocks = (u64)n_blocks * (a.dim / 2) * a.rows, polys = (u64)a.n_heads * a.n_comp;
  // four workgroups for each of 256 CUs, where there are that many polynomials: 15 heads of 10 at N = 2048 take 8.1 us in place of 22 (one part),
  // 16 heads of 16 at 8192 29 in place of 34; more parts than that read the tables again for nothing
  u32 parts = 1;
  while (parts < polys && blocks * a.n_limbs * c.nrep * parts < 1024) parts *= 2;
  const u64 per = (polys + parts - 1) / parts;
  hipLaunchKernelGGL(rope_kernel, dim3(blocks * parts, a.n_limbs, c.nrep), dim3(256), 0, s, c, a, n_blocks, parts, per);
}

}  // namespace acehip
