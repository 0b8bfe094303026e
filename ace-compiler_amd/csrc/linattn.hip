// linattn.hip -- linear attention with a decay per head on ciphertexts: products of matrices of ciphertexts, not relinearised.
#include "nn.hpp"

namespace acehip {

// Sums of products of residues, exact: the residues are split at hb = ceil(bits / 2), and the three 64-bit sums of
//   x*y = ll + ((xl + xh)(yl + yh) - ll - hh) 2^hb + hh 2^(2 hb)
// take one 32x32 multiply-add each.  mm may wrap on the way: only the difference mm - ll - hh counts.  For primes of n bits a product's
// middle part is below 2^(n+1), and an accumulator takes at most two products a term, so 2^(62-n) terms stay below 2^64 (the exact bound
// 2^(64-n) (2^hb - 1)(2^(n-hb) - 1) leaves room for the residue that the sums start from); then the sums are brought back to one residue.
struct Half {
  u32 l, h, s;
};
__device__ __forceinline__ Half halves(u64 x, u32 hb) {
  const u32 l = (u32)x & ((1u << hb) - 1), h = (u32)(x >> hb);
  return Half{l, h, l + h};
}
struct Acc {
  u64 ll = 0, mm = 0, hh = 0;
  __device__ __forceinline__ void mac(const Half& x, const Half& y) {
    ll += (u64)x.l * y.l;
    mm += (u64)x.s * y.s;
    hh += (u64)x.h * y.h;
  }
  __device__ __forceinline__ u64 value(u32 hb, const DevPrime& P) const {
    unsigned __int128 v = ll;
    v += (unsigned __int128)(mm - ll - hh) << hb;
    v += (unsigned __int128)hh << (2 * hb);
    return reduce128(U128{(u64)v, (u64)(v >> 64)}, P.q, P.prec128_lo, P.prec128_hi);
  }
  __device__ __forceinline__ void fold(u32 hb, const DevPrime& P) {
    const Half v = halves(value(hb, P), hb);
    ll = v.l;
    hh = 0;
    mm = (u64)v.l + v.h;
  }
};

__global__ __launch_bounds__(256) void linattn_kernel(DevCtx c, LinattnArgs a, u32 n_blocks) {
  u32 b = blockIdx.x;
  const u32 nb = b % n_blocks;
  b /= n_blocks;
  const u32 j = b % a.Nn;
  b /= a.Nn;
  const u32 m = b % a.M, h = b / a.M, rep = c.rep0 + blockIdx.z;
  const u32 pos = a.pos0 + blockIdx.y, gi = limb_prime(pos, a.level, c.L);
  const u32 n = nb * 256 + threadIdx.x;
  if (!owns(c, gi) || n >= c.N) return;
  const int64_t last = (int64_t)m + a.off;  // last column / key that row m sees
  if (a.skip_above && (int64_t)j > last) return;
  const DevPrime P = c.primes[gi];
  const u64 q = P.q, mh = P.prec128_hi;
  const u32 hb = (P.nbits + 1) / 2;
  const u32 period = 1u << min(62 - P.nbits, 24u);
  const u64 off = (u64)pos * c.N + n;
  u64 r[3] = {0, 0, 0};
  auto term = [&](const LinattnTerm& t, u32 K, bool weighted) {
    const u64* A = reb(c, t.a.d, rep) + (h / t.a_group) * t.a.head + m * t.a.row + off;
    const u64* B = reb(c, t.b.d, rep) + (h / t.b_group) * t.b.head + j * t.b.col + off;
    const int64_t* w = weighted ? reb(c, a.decay, rep) + h * a.decay_ld : nullptr;
    Acc s0, s1, s2;
    u32 left = period;
    for (u32 k = 0; k < K; ++k) {
      u64 a0 = A[k * t.a.col], a1 = A[k * t.a.col + t.a.comp];
      const Half b0 = halves(B[k * t.b.row], hb), b1 = halves(B[k * t.b.row + t.b.comp], hb);
      if (w) {
        const u64 d = signed_mod(w[a.decay_by_k ? (u64)(t.K - 1 - k) : (u64)(last - k)], q, mh);
        a0 = mul_mod(a0, d, P);
        a1 = mul_mod(a1, d, P);
      }
      const Half h0 = halves(a0, hb), h1 = halves(a1, hb);
      if (left == 0) {
        s0.fold(hb, P);
        s1.fold(hb, P);
        s2.fold(hb, P);
        left = period;
      }
      --left;
      s0.mac(h0, b0);
      s1.mac(h0, b1);
      s1.mac(h1, b0);
      s2.mac(h1, b1);
    }
    return ulong3{s0.value(hb, P), s1.value(hb, P), s2.value(hb, P)};
  };
  if (a.t1.K) {
    const ulong3 v = term(a.t1, a.t1.K, false);
    r[0] = v.x;
    r[1] = v.y;
    r[2] = v.z;
    if (a.scale) {
      const u64 g = signed_mod(reb(c, a.scale, rep)[h * a.M + m], q, mh);
      for (int p = 0; p < 3; ++p) r[p] = mul_mod(r[p], g, P);
    }
  }
  const u32 K2 = a.causal ? (u32)min((int64_t)a.t2.K, max(last + 1, (int64_t)0)) : a.t2.K;
  if (K2) {
    const ulong3 v = term(a.t2, K2, a.decay != nullptr);
    r[0] = add_mod(r[0], v.x, q);
    r[1] = add_mod(r[1], v.y, q);
    r[2] = add_mod(r[2], v.z, q);
  }
  if (a.base.d) {
    const u64* s = reb(c, a.base.d, rep) + h * a.base.head + m * a.base.row + j * a.base.col + off;
    const u64 g = a.keep ? signed_mod(reb(c, a.keep, rep)[h], q, mh) : 1;
    for (int p = 0; p < 2; ++p) r[p] = add_mod(r[p], a.keep ? mul_mod(s[p * a.base.comp], g, P) : s[p * a.base.comp], q);
  }
  u64* y = reb(c, a.out.d, rep) + h * a.out.head + m * a.out.row + j * a.out.col + off;
  for (int p = 0; p < 3; ++p) y[p * a.out.comp] = r[p];
}

void launch_linattn(const DevCtx& c, const LinattnArgs& a, hipStream_t s) {
  const u32 n_blocks = (c.N + 255) / 256;
  hipLaunchKernelGGL(linattn_kernel, dim3(n_blocks * a.Nn * a.M * a.n_heads, a.n_limbs, c.nrep), dim3(256), 0, s, c, a, n_blocks);
}

}  // namespace acehip
