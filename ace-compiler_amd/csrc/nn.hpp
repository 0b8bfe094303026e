// nn.hpp -- operators of a transformer on ciphertexts (api_nn.cpp -> linear.hip, rope.hip, linattn.hip).
#pragma once
#include "kernels.hpp"

namespace acehip {

// Matrix of ciphertexts in device memory (acehip_mat of include/acehip.h, strides in words): polynomial `comp` of element (head, row, col) starts
// at d + head*head_stride + row*row_stride + col*col_stride + comp*comp_stride, limb position pos of it N*pos further.
struct CtMat {
  u64* d = nullptr;
  u64 head = 0, row = 0, col = 0, comp = 0;
};

// w mod q for a signed word; mh = floor(2^64 / q) (DevPrime::prec128_hi), so the quotient is at most one too small
__device__ __forceinline__ u64 signed_mod(int64_t w, u64 q, u64 mh) {
  const u64 a = w < 0 ? 0 - (u64)w : (u64)w;
  u64 r = a - mulhi64(a, mh) * q;
  r = r >= q ? r - q : r;
  return w < 0 && r != 0 ? q - r : r;
}

// global address space spelled out: FLAT loads would count as LDS accesses too, and every wait for LDS would wait for them
#define GLOBAL __attribute__((address_space(1)))
// a word that is the same for the wave, kept on the scalar unit
__device__ __forceinline__ u64 uniform64(u64 v) {
  return ((u64)(u32)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32) | (u32)__builtin_amdgcn_readfirstlane((int)v);
}
// LDS writes of the workgroup are visible, requests to memory stay in flight
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}
// a * w mod q up to multiples of q, with nq = -q and a companion wp of w that is at most two units of 2^-64 too small: below 5q, below 4q for a < 2^63
// (the quotient leaves out the low product and two carries, less than 3; a w / q - a wp / 2^64 is below 2, for a < 2^63 below 1)
__device__ __forceinline__ u64 mul_near(u64 a, u64 w, u64 wp, u64 nq) {
  const u64 h = (u64)(u32)(a >> 32) * (u32)(wp >> 32) + __umulhi((u32)(a >> 32), (u32)wp) + __umulhi((u32)a, (u32)(wp >> 32));
  return a * w + h * nq;
}

// y[r][j] = tok[r] * mul[j] * sum_i w[j][i] x[r][i], every polynomial of the ciphertexts (linear.hip)
struct LinearArgs {
  CtMat out, in;
  const int8_t* w;     // [n_out][ld_w]
  u64 ld_w;
  const int64_t* mul;  // [n_out] or null
  const u64* tok;      // plaintext polynomial of row r at tok + r*tok_stride, or null
  u64 tok_stride;
  u32 rows, n_in, n_out, n_comp, level, pos0, n_limbs;
  bool wide_primes;    // every prime of the call is above 2^40
  const void* packed = nullptr;  // the weights as linear_pack_kernel left them
};
// on every one of the launch sets; ws: memory for packed weights, or null: they are read as they lie
void launch_linear(const DevCtx& c, const DevCtx* launches, u32 n_launches, LinearArgs a, void* ws, size_t ws_bytes, hipStream_t s);

// cos and sin of pos[axis[i]][t] * freq[i] (rope.hip)
constexpr u32 ROPE_PAIRS_MAX = 256;  // pairs per launch: a kernel argument
struct RopeAngles {
  double freq[ROPE_PAIRS_MAX];
  uint8_t axis[ROPE_PAIRS_MAX];
};
constexpr u32 ROPE_AXES_MAX = 8;
void launch_rope_messages(double* cos_out, double* sin_out, u64 out_stride, const double* pos, u64 pos_stride, u32 n_pos, const RopeAngles& a, u32 n_pairs,
                          hipStream_t s);
// (x0, x1) -> (x0 C - x1 S, x0 S + x1 C) for the pairs of features (i, i + dim/2) or (2i, 2i + 1)
struct RopeArgs {
  CtMat out, in;
  const u64 *cosp, *sinp;  // plaintext polynomials of (row, pair) at + row*row_stride + pair*pair_stride
  u64 pair_stride, row_stride;
  u32 n_heads, rows, dim, interleaved, n_comp, level, pos0, n_limbs;
};
void launch_rope(const DevCtx& c, const RopeArgs& a, hipStream_t s);

// out[h][m][n] = keep[h] * base[h][m][n] + scale[h][m] * sum_k A1[h][m][k] (x) B1[h][k][n] + sum_k decay[h][..] * A2[h][m][k] (x) B2[h][k][n]  (linattn.hip)
// (x): product of two ciphertexts before relinearisation, three polynomials.  Strides of A: row = m, col = k; of B: row = k, col = n.
struct LinattnTerm {
  CtMat a, b;
  u32 K = 0;            // 0: the term is absent
  u32 b_group = 1;      // head h reads head h / group of a or b (keys, values shared by groups of heads)
  u32 a_group = 1;
};
struct LinattnArgs {
  CtMat out, base;             // base.d == null: absent
  LinattnTerm t1, t2;
  const int64_t* keep = nullptr;   // [n_heads] or null: 1
  const int64_t* scale = nullptr;  // [n_heads][M] or null: 1; of term 1
  const int64_t* decay = nullptr;  // [n_heads][decay_ld] or null: 1; of term 2: entry m + off - k (causal form), or K - 1 - k (decay_by_k)
  u64 decay_ld = 0;
  u32 n_heads, M, Nn;
  // causal: term 2 takes k <= m + off only (off may be negative); skip_above: results with n > m + off are not computed and not written
  int32_t off = 0;
  u32 causal = 0, decay_by_k = 0, skip_above = 0;
  u32 level, pos0, n_limbs;
  bool wide_primes = false;        // every prime of the call is above 2^32 and up to 2^64 / 9
};
bool linattn_fits(const DevCtx& c, const LinattnArgs& a);  // the launch has less than 2^32 lanes along x
void launch_linattn(const DevCtx& c, const LinattnArgs& a, hipStream_t s);

}  // namespace acehip
