// linattn.hip -- linear attention with a decay per head on ciphertexts: products of matrices of ciphertexts, not relinearised.
#include <algorithm>

#include "nn.hpp"

namespace acehip {

// Sums of products of residues, exact: the residues are split at hb = ceil(bits / 2), and the three 64-bit sums of
//   x*y = ll + ((xl + xh)(yl + yh) - ll - hh) 2^hb + hh 2^(2 hb)
// take one 32x32 multiply-add each.  mm may wrap on the way: only the difference mm - ll - hh counts.  For primes of n bits a product's
// middle part is below 2^(n+1), so 2^(63-n) products stay below 2^64 (the exact bound 2^(64-n) (2^hb - 1)(2^(n-hb) - 1) leaves room for what carry()
// leaves in the sums); then carry() makes room again: after 2^(62-n) terms for the results' middle polynomial, which takes two products a term, and
// after twice as many for the others.
struct Half {
  u32 l, h, s;
};
__device__ __forceinline__ Half halves(u64 x, u32 hb) {
  const u32 l = (u32)x & ((1u << hb) - 1), h = (u32)(x >> hb);
  return Half{l, h, l + h};
}
// What the sums of one prime need.  WIDE: primes above 2^32 and up to 2^64 / 9.
template <bool WIDE>
struct Reduce {
  u64 q, nq, mh, ml;   // the prime, its negative, floor(2^128 / q)
  u64 w, wp;           // 2^(2 hb) mod q and its companion, at most two units of 2^-64 too small
  float near_q;        // 2^32 / q, a little too small
  u32 hb, mask;
  __device__ __forceinline__ explicit Reduce(const DevPrime& P) : q(P.q), nq(0 - P.q), mh(P.prec128_hi), ml(P.prec128_lo) {
    hb = (P.nbits + 1) / 2;
    mask = (1u << hb) - 1;
    w = signed_mod(1ll << (2 * hb), q, mh);
    wp = w * mh + mulhi64(w, ml);
    near_q = __builtin_fmaf((float)(u32)(ml >> 32), 0x1p-32f, (float)mh) * (0x1p-32f * 0.999999f);
  }
};
struct Acc {
  u64 ll, mm, hh;
  __device__ __forceinline__ void mac(const Half& x, const Half& y) {
    ll += (u64)x.l * y.l;
    mm += (u64)x.s * y.s;
    hh += (u64)x.h * y.h;
  }
  // carries brought up and hh reduced below 3q (WIDE: the quotient by floor(2^64 / q), below 2^32, of hh's upper word: less than three too small):
  // room for as many terms again
  template <bool WIDE>
  __device__ __forceinline__ void carry(const Reduce<WIDE>& r) {
    u64 mid = mm - ll - hh + (ll >> r.hb);
    ll = (u32)ll & r.mask;
    hh += mid >> r.hb;
    mid = (u32)mid & r.mask;
    if (WIDE) hh += __umulhi((u32)(hh >> 32), (u32)r.mh) * r.nq;
    else      hh -= mulhi64(hh, r.mh) * r.q;
    mm = mid + ll + hh;
  }
  template <bool WIDE>
  __device__ __forceinline__ u64 value(const Reduce<WIDE>& r) const {
    const u64 mid = mm - ll - hh + (ll >> r.hb);
    if (!WIDE) {
      const unsigned __int128 v = ((unsigned __int128)hh << (2 * r.hb)) + ((unsigned __int128)mid << r.hb) + ((u32)ll & r.mask);
      return reduce128_generic(U128{(u64)v, (u64)(v >> 64)}, r.q, r.ml, r.mh);
    }
    // low part below 2^(2 hb) <= 4q, the rest times 2^(2 hb) below 5q; then the quotient, below 9, from single precision: not too large, at most
    // one too small
    const u64 v = mul_near(hh + (mid >> r.hb), r.w, r.wp, r.nq) + (((u64)((u32)mid & r.mask) << r.hb) | ((u32)ll & r.mask));
    const u64 x = v + (u64)(u32)((float)(u32)(v >> 32) * r.near_q) * r.nq;
    return x >= r.q ? x - r.q : x;
  }
  // times f, as the start of further sums at primes of up to 60 bits: below 10q, whose part above 2^hb fits the room that the exact bound leaves.
  // fp: companion of f; g = f w mod q with its companion gp
  __device__ __forceinline__ Acc times(const Reduce<true>& r, u64 f, u64 fp, u64 g, u64 gp) const {
    const u64 mid = mm - ll - hh + (ll >> r.hb);
    const u64 v = mul_near(hh + (mid >> r.hb), g, gp, r.nq) + mul_near(((u64)((u32)mid & r.mask) << r.hb) | ((u32)ll & r.mask), f, fp, r.nq);
    const u32 l = (u32)v & r.mask;
    return Acc{l, l + (v >> r.hb), 0};
  }
};

// a pointer that is the same for the wave (lanes add their coefficient as a 32-bit offset)
__device__ __forceinline__ const GLOBAL char* uniform(const u64* p) { return (const GLOBAL char*)uniform64((u64)p); }

// One row of results.  A wave: 64 coefficients, NT results (3 sums of 3 words each) over every KW-th term; a workgroup: WN waves along the columns, KW along
// the terms, whose sums are joined through LDS.  Per term of the sums a lane reads 2 (1 + NT) residues and makes 12 NT multiply-adds.
// WIDE: primes above 2^32 (the reduction's quotient from three partial products).
// In use for one row of results, where nothing but the row is read twice: bound by memory (48 x 48 states read by one token, four heads, three limbs at
// N = 8192: 3.8 GB in 0.72 ms, 5.3 TB/s); for launches that leave the card empty; and for the chains and rings that the form below does not take.
template <int NT, int WN, int KW, bool WIDE>
__global__ __launch_bounds__(64 * WN * KW, 2) void linattn_kernel(DevCtx c, LinattnArgs a, u32 n_blocks, u32 n_tiles) {
  constexpr u32 KC = 64;  // terms whose factors are prepared at a time
  static_assert(KC % KW == 0 && (KW == 1 || WN == 1), "a wave keeps its place among the terms, a workgroup of several ends as one");
  __shared__ ulong2 factor[KC];
  __shared__ u64 joined[KW == 1 ? 1 : KW - 1][NT * 9][64];
  u32 b = blockIdx.x;
  // tiles of the same coefficients follow each other on one XCD (ids congruent mod 8): its L2 keeps their operands
  const u32 tiles = a.M * n_tiles, groups = gridDim.x / tiles;
  u32 g, t;
  if ((groups & 7u) == 0) {
    const u32 x = b >> 3;
    t = x % tiles;
    g = (x / tiles) * 8 + (b & 7u);
  } else {
    t = b % tiles;
    g = b / tiles;
  }
  t = __builtin_amdgcn_readfirstlane(t);
  g = __builtin_amdgcn_readfirstlane(g);
  const u32 nb = g & (n_blocks - 1), h = g >> __builtin_ctz(n_blocks), rep = c.rep0 + blockIdx.z;
  const u32 lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wk = wave / WN;
  const u32 row = t / n_tiles, j0 = ((t % n_tiles) * WN + wave % WN) * NT;
  const u32 pos = a.pos0 + blockIdx.y, gi = limb_prime(pos, a.level, c.L);
  if (!owns(c, gi)) return;
  const int64_t last = (int64_t)row + a.off;  // column / key that the row sees
  if (a.skip_above && (int64_t)j0 > last) return;  // (scores: no factors, so no barrier to meet before the joint one)
  const DevPrime P = c.primes[gi];
  const Reduce<WIDE> red(P);
  const u64 q = P.q, mh = P.prec128_hi;
  const u32 hb = red.hb;
  const u32 n = nb * 64 + lane, at = 8 * min(n, c.N - 1);  // (rings below 64: the lanes behind the ring repeat its last coefficient and store nothing)
  const u64 limb = (u64)pos * c.N;
  u32 col[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i) col[i] = min(j0 + i, a.Nn - 1);
  auto read = [&](const u64* p) { return *(const GLOBAL u64*)(uniform(p) + at); };

  Acc s[NT][3];
  const u32 period = 1u << min(62 - P.nbits, 24u);
  u32 left = period;  // terms that the sums still take
  bool second = false;
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int p = 0; p < 3; ++p) s[j][p] = Acc{0, 0, 0};
  if (a.base.d && wk == 0) {  // one term: keep * base
    const u64* S = reb(c, a.base.d, rep) + h * a.base.head + limb;
    const Half f = halves(a.keep ? signed_mod(reb(c, a.keep, rep)[h], q, mh) : 1, hb);
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int p = 0; p < 2; ++p) s[j][p].mac(halves(read(S + row * a.base.row + col[j] * a.base.col + p * a.base.comp), hb), f);
    --left;
  }
  struct Raw {
    u64 a[2], b[NT][2];
  };
#pragma unroll 1
  for (u32 part = 0; part < 2; ++part) {
    const LinattnTerm& t = part ? a.t2 : a.t1;
    const bool weighted = part ? a.decay != nullptr : a.scale != nullptr;
    const u32 K = part && a.causal ? (u32)min((int64_t)t.K, max(last + 1, (int64_t)0)) : t.K;  // a causal sum ends with the last key that the row sees
    if (K == 0) continue;
    const u32 k_first = min(wk, K - 1);
    const u64* A = reb(c, t.a.d, rep) + (t.a_group == 1 ? h : h / t.a_group) * t.a.head + limb + row * t.a.row + k_first * t.a.col;
    const u64* B = reb(c, t.b.d, rep) + (t.b_group == 1 ? h : h / t.b_group) * t.b.head + limb + k_first * t.b.row;
    const u64 a_next = KW * t.a.col, b_next = KW * t.b.row;
    const u64 *pa[2], *pb[NT][2];  // where the wave's next term's residues lie
#pragma unroll
    for (int p = 0; p < 2; ++p) pa[p] = A + p * t.a.comp;
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int p = 0; p < 2; ++p) pb[i][p] = B + col[i] * t.b.col + p * t.b.comp;
    auto load = [&](Raw& r, bool more) {
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        r.a[p] = read(pa[p]);
        pa[p] += more ? a_next : 0;
      }
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          r.b[i][p] = read(pb[i][p]);
          pb[i][p] += more ? b_next : 0;
        }
    };
    Raw next;
    load(next, wk + KW < K);
    for (u32 k0 = 0; k0 < K; k0 += KC) {
      if (weighted) {  // factors of the terms from k0 on: term 1's of the row, term 2's by term or by distance
        __syncthreads();
        for (u32 e = threadIdx.x; e < KC; e += 64 * WN * KW) {
          const int64_t d = part == 0 ? (int64_t)row : a.decay_by_k ? (int64_t)t.K - 1 - k0 - e : last - k0 - e;
          const bool there = d >= 0 && d < (int64_t)(part ? t.K : a.M);
          const u64 f = there ? signed_mod(part ? reb(c, a.decay, rep)[h * a.decay_ld + d] : reb(c, a.scale, rep)[h * a.M + d], q, mh) : 0;
          factor[e] = ulong2{f, f * mh + mulhi64(f, P.prec128_lo)};
        }
        __syncthreads();
      }
      const u32 k1 = min(k0 + KC, K);
#pragma unroll 1
      for (u32 k = k0 + wk; k < k1; k += KW) {
        Raw r = next;
        load(next, k + 2 * KW < K);
        if (left == 0) {
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            s[j][1].carry(red);
            if (second) s[j][0].carry(red), s[j][2].carry(red);
          }
          second = !second;
          left = period;
        }
        --left;
        if (weighted) {
          const ulong2 f = factor[k - k0];
#pragma unroll
          for (int p = 0; p < 2; ++p) {
            u64 v = r.a[p] * f.x - mulhi64(r.a[p], f.y) * q;  // (the companion is at most one too small: below 3q)
            v = v >= 2 * q ? v - 2 * q : v;
            r.a[p] = v >= q ? v - q : v;
          }
        }
        const Half h0 = halves(r.a[0], hb), h1 = halves(r.a[1], hb);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const Half b0 = halves(r.b[j][0], hb), b1 = halves(r.b[j][1], hb);
          s[j][0].mac(h0, b0);
          s[j][1].mac(h0, b1);
          s[j][1].mac(h1, b0);
          s[j][2].mac(h1, b1);
        }
      }
    }
  }
  if (KW > 1) {  // joint sums: below 3q from each wave after a carry, so three fit at primes of up to 2^64 / 9
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int p = 0; p < 3; ++p) {
        s[j][p].carry(red);
        if (wk > 0) {
          u64(*to)[64] = &joined[wk - 1][9 * j + 3 * p];
          to[0][lane] = s[j][p].ll;
          to[1][lane] = s[j][p].mm;
          to[2][lane] = s[j][p].hh;
        }
      }
    __syncthreads();
    if (wk > 0) return;
#pragma unroll
    for (int w = 0; w < KW - 1; ++w)
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int p = 0; p < 3; ++p) {
          const u64(*from)[64] = &joined[w][9 * j + 3 * p];
          if (w % 2 == 0 && w) s[j][p].carry(red);
          s[j][p].ll += from[0][lane];
          s[j][p].mm += from[1][lane];
          s[j][p].hh += from[2][lane];
        }
  }
  u64* y = reb(c, a.out.d, rep) + h * a.out.head + limb;
#pragma unroll
  for (int j = 0; j < NT; ++j)
    if (j0 + j < a.Nn && n < c.N && (!a.skip_above || (int64_t)(j0 + j) <= last))
#pragma unroll
      for (int p = 0; p < 3; ++p) *(GLOBAL u64*)((GLOBAL char*)uniform(y + row * a.out.row + col[j] * a.out.col + p * a.out.comp) + at) = s[j][p].value(red);
}

// The same with the operands of a workgroup's waves shared through LDS: every row of A and column of B is read by one wave, has its factor and mask
// applied and its residues split in halves there, KS terms at a time and one stage ahead.
// Bound by the integer instructions, at about four cycles each: 100 for a wave's term of 4 x 64 results without factors (48 multiply-adds, 10 to add halves and
// read LDS, 14 staging, up to 36 of carries at primes of 60 bits, the rest start and end of a sum of 32 terms), 60 in place of 14 where the staged
// residues have factors.  32 x 32 causal scores of 32 features, four heads of two, three limbs at N = 4096: 0.90 ms, 10^10 multiply-adds (38 % of the
// rate they reach alone), 1.8 GB.  A chunk of 16 with a state of 24 x 32, two heads, three limbs at 8192: 1.01 ms, the vector units busy for 87 % of it.
// One token into 32 x 32 states, four heads and limbs at 8192: 1.27 ms for 5.5 GB (4.3 TB/s), bound by memory.
// Sums of int8 products on the matrix cores, as in linear.hip, cost as many instructions: tiles of 16 x 16 leave a byte 16 uses for its transposition,
// and the reductions at the end weigh more at sums this short; that form took 1.63 ms.
// Tiles of 2 x 2 results in 2 x 2 waves: 2 x 4 results (half the waves) 1.56 ms, 2 x 4 waves 1.52, two terms a stage 1.16.
// The tiles of a launch, row by row, without those of causal scores that no query sees (workgroups that end at once come in a pattern that leaves some
// of the shader engines, which take workgroups in turn, without work: 32 x 32 scores 1.01 ms in place of 0.90).  Row tm of tiles has
// tm + lead of them, between 0 and n: rows r0 .. r0 + grow - 1 have c0, c0 + 1, ..; the rows behind all n.
struct Tiles {
  u32 all, n, r0 = 0, c0 = 0, grow = 0;
  Tiles(const LinattnArgs& a, u32 m, u32 nn) {
    const u32 rows = (a.M + m - 1) / m;
    n = (a.Nn + nn - 1) / nn;
    if (a.skip_above && m == nn) {
      const int64_t last = (int64_t)m - 1 + a.off, lead = 1 + (last >= 0 ? last / m : -((-last + m - 1) / (int64_t)m));
      r0 = (u32)std::min((int64_t)rows, std::max((int64_t)0, 1 - lead));
      c0 = (u32)std::min((int64_t)n, r0 + lead);
      grow = std::min(rows - r0, n - c0);
    }
    all = grow * c0 + (u32)((u64)grow * (grow - 1) / 2) + (rows - r0 - grow) * n;
  }
  __device__ __forceinline__ void place(u32 t, u32& tm, u32& tj) const {
    const u32 sum = grow * c0 + (u32)((u64)grow * (grow - 1) / 2);
    if (t >= sum) {
      tm = r0 + grow + (t - sum) / n;
      tj = (t - sum) % n;
      return;
    }
    // the largest i with i c0 + i (i - 1) / 2 <= t, from its root in single precision
    const float h = (float)c0 - 0.5f;
    u32 i = (u32)max(0.0f, sqrtf(h * h + 2.0f * (float)t) - h);
    const auto before = [&](u32 i) { return i * c0 + (u32)((u64)i * (i - 1) / 2); };
    while (i > 0 && before(i) > t) --i;
    while (before(i + 1) <= t) ++i;
    tm = r0 + i;
    tj = t - before(i);
  }
};
template <int MT, int NT, int WM, int WN, int KS, int MIN_WAVES>
__global__ __launch_bounds__(64 * WM * WN, MIN_WAVES) void linattn_shared_kernel(DevCtx c, LinattnArgs a, u32 n_blocks, Tiles tiles) {
  constexpr u32 M = MT * WM, N = NT * WN, W = WM * WN, R = (M + N) / W;  // rows and columns of the workgroup's tile; its waves; rows that a wave stages
  static_assert((M + N) % W == 0, "the waves stage equal shares");
  constexpr u32 KC = 64;  // terms whose factors are prepared at a time
  __shared__ uint4 operand[2][KS][M + N][64];  // halves of both polynomials: {l0, h0, l1, h1} of A's rows, then of B's columns
  __shared__ ulong2 factor[KC + M];
  u32 b = blockIdx.x;
  const u32 groups = gridDim.x / tiles.all;
  u32 g, t, tm, tj;
  if ((groups & 7u) == 0) {
    const u32 x = b >> 3;
    t = x % tiles.all;
    g = (x / tiles.all) * 8 + (b & 7u);
  } else {
    t = b % tiles.all;
    g = b / tiles.all;
  }
  tiles.place(t, tm, tj);
  tm = __builtin_amdgcn_readfirstlane(tm);
  tj = __builtin_amdgcn_readfirstlane(tj);
  g = __builtin_amdgcn_readfirstlane(g);
  const u32 nb = g & (n_blocks - 1), h = g >> __builtin_ctz(n_blocks), rep = c.rep0 + blockIdx.z;
  const u32 lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const u32 wg_m = tm * M, wg_j = tj * N;
  const u32 wm = (wave / WN) * MT, wn = (wave % WN) * NT, m0 = wg_m + wm, j0 = wg_j + wn;
  const u32 pos = a.pos0 + blockIdx.y, gi = limb_prime(pos, a.level, c.L);
  if (!owns(c, gi)) return;
  const int64_t off = a.off;
  // last column / key that the rows of the workgroup and of this wave's results see (rows past M: the last one's)
  const int64_t wg_last = (int64_t)min(wg_m + M, a.M) - 1 + off, last = (int64_t)min(m0 + MT, a.M) - 1 + off;
  if (a.skip_above && (int64_t)wg_j > wg_last) return;
  const bool idle = m0 >= a.M || j0 >= a.Nn || (a.skip_above && (int64_t)j0 > last);  // stages operands for the others
  const DevPrime P = c.primes[gi];
  const Reduce<true> red(P);
  const u64 q = P.q, mh = P.prec128_hi;
  const u32 hb = red.hb;
  const u32 n = nb * 64 + lane, at = 8 * n;
  const u64 limb = (u64)pos * c.N;
  auto read = [&](const u64* p) {
    u32 o = at;
    asm("" : "+v"(o));  // (opaque: a load takes the uniform base and 32-bit offset as they are)
    return *(const GLOBAL u64*)(uniform(p) + o);
  };

  Acc s[MT][NT][3];
  // Factors of rows (term 1) are applied to long sums at their end (chunks of 16, 32 columns, two heads, three limbs at N = 8192: 8 terms 670 us, 662 staged;
  // 12 terms 753 and 761, 48 terms 1.51 and 1.74 ms).  What is staged with a factor stays below 3q at primes of up to 56 bits: the upper halves and the
  // middle parts have two bits more, so a quarter of the terms between carries.
  const bool late = a.scale != nullptr && a.t1.K >= 12 && P.nbits <= 60, lazy = P.nbits <= 56;
  const u32 period = 1u << min(62 - P.nbits - (lazy && (a.decay || (a.scale && !late)) ? 2 : 0), 24u);
  u32 left = period;  // terms that the sums still take
  bool second = false;
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int p = 0; p < 3; ++p) s[i][j][p] = Acc{0, 0, 0};
  if (a.base.d) {  // one term: keep * base
    const u64* S = reb(c, a.base.d, rep) + h * a.base.head + limb;
    const Half f = halves(a.keep ? signed_mod(reb(c, a.keep, rep)[h], q, mh) : 1, hb);
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int p = 0; p < 2; ++p)
          s[i][j][p].mac(halves(read(S + min(m0 + i, a.M - 1) * a.base.row + min(j0 + j, a.Nn - 1) * a.base.col + p * a.base.comp), hb), f);
    --left;
  }
  u32 buf = 0;
#pragma unroll 1
  for (u32 part = 0; part < 2; ++part) {
    const LinattnTerm& t = part ? a.t2 : a.t1;
    const bool causal = part && a.causal, weighted = part ? a.decay != nullptr : a.scale && !late;
    const u32 K = causal ? (u32)min((int64_t)t.K, max(wg_last + 1, (int64_t)0)) : t.K;  // of the workgroup; K_own: of this wave's results
    const u32 K_own = idle ? 0 : causal ? (u32)min((int64_t)t.K, max(last + 1, (int64_t)0)) : t.K;
    if (K == 0) continue;
    const u64* A = reb(c, t.a.d, rep) + (t.a_group == 1 ? h : h / t.a_group) * t.a.head + limb;
    const u64* B = reb(c, t.b.d, rep) + (t.b_group == 1 ? h : h / t.b_group) * t.b.head + limb;
    // the wave's share: row wave + r*W of the tile's rows, then columns
    const u64* from[R][2];
    u64 next[R];
#pragma unroll
    for (u32 r = 0; r < R; ++r) {
      const u32 x = wave + r * W;
      from[r][0] = x < M ? A + min(wg_m + x, a.M - 1) * t.a.row : B + min(wg_j + x - M, a.Nn - 1) * t.b.col;
      from[r][1] = from[r][0] + (x < M ? t.a.comp : t.b.comp);
      next[r] = x < M ? t.a.col : t.b.row;
    }
    u64 raw[KS][R][2];
    u32 k_load = 0;
    auto load = [&] {  // the next KS terms (behind the last one it is read again, and staged as zeros)
#pragma unroll
      for (int e = 0; e < KS; ++e) {
        const bool more = ++k_load < K;
#pragma unroll
        for (u32 r = 0; r < R; ++r)
#pragma unroll
          for (int p = 0; p < 2; ++p) {
            raw[e][r][p] = read(from[r][p]);
            from[r][p] += more ? next[r] : 0;
          }
      }
    };
    auto factors = [&](u32 k0) {  // of the terms from k0 on, as in linattn_kernel
      lds_barrier();
      for (u32 e = threadIdx.x; e < KC + M; e += 64 * W) {
        const int64_t d = part == 0 ? (int64_t)min(wg_m + e, a.M - 1) : a.decay_by_k ? (int64_t)t.K - 1 - k0 - e : (int64_t)wg_m + off - (k0 + KC - 1) + e;
        const bool there = d >= 0 && d < (int64_t)(part ? t.K : a.M);
        const u64 f = there ? signed_mod(part ? reb(c, a.decay, rep)[h * a.decay_ld + d] : reb(c, a.scale, rep)[h * a.M + d], q, mh) : 0;
        factor[e] = ulong2{f, f * mh + mulhi64(f, P.prec128_lo)};
      }
      lds_barrier();
    };
    auto stage = [&](u32 k0, u32 to) {
#pragma unroll
      for (int e = 0; e < KS; ++e) {
        const u32 k = k0 + e;
#pragma unroll
        for (u32 r = 0; r < R; ++r) {
          const u32 x = wave + r * W;
          u64 v[2] = {raw[e][r][0], raw[e][r][1]};
          u32 mask = red.mask, there = ~0u;
          if (x < M) {
            const u32 m = min(wg_m + x, a.M - 1);
            there = (int64_t)k < (causal ? min((int64_t)K, (int64_t)m + off + 1) : (int64_t)K) ? ~0u : 0;
            mask &= there;
            if (weighted) {
              const u32 kc = k % KC;
              const ulong2 f = factor[part == 0 ? m - wg_m : a.decay_by_k ? kc : KC - 1 - kc + (m - wg_m)];
#pragma unroll
              for (int p = 0; p < 2; ++p) {
                v[p] = v[p] * f.x - mulhi64(v[p], f.y) * q;  // (the companion is at most one too small: below 3q)
                if (lazy) continue;
                v[p] = v[p] >= 2 * q ? v[p] - 2 * q : v[p];
                v[p] = v[p] >= q ? v[p] - q : v[p];
              }
            }
          }
          operand[to][e][x][lane] = uint4{(u32)v[0] & mask, (u32)(v[0] >> hb) & there, (u32)v[1] & mask, (u32)(v[1] >> hb) & there};
        }
      }
    };
    load();
    if (weighted) factors(0);
    else          lds_barrier();  // (the part before has read its last operands)
    stage(0, buf);
    load();
#pragma unroll 1
    for (u32 k0 = 0; k0 < K; k0 += KS) {
      if (weighted && (k0 + KS) % KC == 0 && k0 + KS < K) factors(k0 + KS);
      else                                                lds_barrier();
      if (k0 + KS < K) {
        stage(k0 + KS, buf ^ 1u);
        load();
      }
#pragma unroll
      for (int e = 0; e < KS; ++e) {
        if (k0 + e >= K_own) continue;
        if (left == 0) {
#pragma unroll
          for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j) {
              s[i][j][1].carry(red);
              if (second) s[i][j][0].carry(red), s[i][j][2].carry(red);
            }
          second = !second;
          left = period;
        }
        --left;
        uint4 xa[MT], xb[NT];
#pragma unroll
        for (int i = 0; i < MT; ++i) xa[i] = operand[buf][e][wm + i][lane];
#pragma unroll
        for (int j = 0; j < NT; ++j) xb[j] = operand[buf][e][M + wn + j][lane];
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          const Half h0{xa[i].x, xa[i].y, xa[i].x + xa[i].y}, h1{xa[i].z, xa[i].w, xa[i].z + xa[i].w};
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            const Half b0{xb[j].x, xb[j].y, xb[j].x + xb[j].y}, b1{xb[j].z, xb[j].w, xb[j].z + xb[j].w};
            s[i][j][0].mac(h0, b0);
            s[i][j][1].mac(h0, b1);
            s[i][j][1].mac(h1, b0);
            s[i][j][2].mac(h1, b1);
          }
        }
      }
      buf ^= 1u;
    }
    if (part == 0 && late) {
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const u64 f = signed_mod(reb(c, a.scale, rep)[h * a.M + min(m0 + i, a.M - 1)], q, mh), fp = f * mh + mulhi64(f, P.prec128_lo);
        u64 g = f * red.w - mulhi64(f, red.wp) * q;  // (below 4q)
        g = g >= 2 * q ? g - 2 * q : g;
        g = g >= q ? g - q : g;
        const u64 gp = g * mh + mulhi64(g, P.prec128_lo);
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int p = 0; p < 3; ++p) s[i][j][p] = s[i][j][p].times(red, f, fp, g, gp);
      }
      left = period;
      second = false;
    }
  }
  u64* y = reb(c, a.out.d, rep) + h * a.out.head + limb;
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j)
      if (m0 + i < a.M && j0 + j < a.Nn && (!a.skip_above || (int64_t)(j0 + j) <= (int64_t)(m0 + i) + off))
#pragma unroll
        for (int p = 0; p < 3; ++p)
          *(GLOBAL u64*)((GLOBAL char*)uniform(y + (m0 + i) * a.out.row + (j0 + j) * a.out.col + p * a.out.comp) + at) = s[i][j][p].value(red);
}

// Lanes along x of the launches below.
template <int NT, int WN, int KW>
static u64 lanes_rows(const DevCtx& c, const LinattnArgs& a) {
  return (u64)((c.N + 63) / 64) * a.M * ((a.Nn + NT * WN - 1) / (NT * WN)) * a.n_heads * (64 * WN * KW);
}
template <int MT, int NT, int WM, int WN>
static u64 lanes_shared(const DevCtx& c, const LinattnArgs& a) {
  return (u64)(c.N / 64) * Tiles(a, MT * WM, NT * WN).all * a.n_heads * (64 * WM * WN);
}
template <int NT, int WN, int KW, bool WIDE>
static void launch_rows(const DevCtx& c, const LinattnArgs& a, hipStream_t s) {
  const u32 n_blocks = (c.N + 63) / 64, n_tiles = (a.Nn + NT * WN - 1) / (NT * WN), block = 64 * WN * KW;
  hipLaunchKernelGGL((linattn_kernel<NT, WN, KW, WIDE>), dim3(lanes_rows<NT, WN, KW>(c, a) / block, a.n_limbs, c.nrep), dim3(block), 0, s, c, a, n_blocks, n_tiles);
}

template <int MT, int NT, int WM, int WN, int KS, int MIN_WAVES>
static void launch_shared(const DevCtx& c, const LinattnArgs& a, hipStream_t s) {
  const Tiles tiles(a, MT * WM, NT * WN);
  const u32 n_blocks = c.N / 64, block = 64 * WM * WN;
  if (tiles.all == 0) return;  // (no query sees a key)
  hipLaunchKernelGGL((linattn_shared_kernel<MT, NT, WM, WN, KS, MIN_WAVES>), dim3(lanes_shared<MT, NT, WM, WN>(c, a) / block, a.n_limbs, c.nrep), dim3(block), 0, s, c, a,
                     n_blocks, tiles);
}

// Up to 2048 workgroups of a result each (1792 have a place at once, seven on each of 256 CUs), the sums are cut over a workgroup's waves: 4 x 4 scores of 64
// features at N = 1024 8.3 us, 21 by the next form; a 64 x 64 state read by one token 15 and 25; with more of them it loses (16 x 16 states, 16 tokens: 24
// us, 20).  Tiles of 2 x 2 results, two terms a stage, up to 1024 workgroups of them (9 x 9 scores of 51 features at 2048: 25 us, 38 by 4 x 4; with 1280
// workgroups, 8 x 8 scores of 24 features at 4096, 27 and 24), or where 4 x 4 leave more idle than they save: one takes as long as 2.15 of 2 x 2 (2 x 2
// scores of 40 features, eight heads, three limbs at 8192: 100 us, 124 by 4 x 4; 6 x 6 states, 20 tokens: 359 and 336).
// One row: its operands are read once whatever the form, and waiting for each other costs (48 x 48 state at N = 8192: 0.72 ms, 0.86 shared) unless half the
// places stay empty (48 x 48 at 1024, three limbs: 31 us, 27 shared).  Two rows or more share (2 x 40 x 4 scores at 8192: 53 us, 91 unshared by tiles of
// 4 x 8; 64 x 2 state of four tokens 0.55 ms, 1.09).
enum class Form { GENERAL, JOINT, SMALL_TILES, TILES, ROWS };
static Form form(const DevCtx& c, const LinattnArgs& a) {
  const bool row = a.M == 1;
  const u64 blocks = (u64)((c.N + 63) / 64) * a.n_heads * a.n_limbs * c.nrep, small = Tiles(a, 2, 2).all, large = Tiles(a, 4, 4).all;
  const bool spare = row ? blocks * ((a.Nn + 15) / 16) < 512 : blocks * small <= 1024 || small * 20 < large * 43;
  if (!a.wide_primes) return Form::GENERAL;
  if (blocks * a.M * a.Nn <= 2048 && (u64)a.t1.K + a.t2.K >= 16) return Form::JOINT;
  if (c.N >= 64 && spare) return Form::SMALL_TILES;
  return c.N >= 64 && !row ? Form::TILES : Form::ROWS;
}
bool linattn_fits(const DevCtx& c, const LinattnArgs& a) {
  if ((unsigned __int128)((c.N + 63) / 64) * a.M * a.Nn * a.n_heads >> 30) return false;  // (counts of tiles stay in 32 bits; more than any form takes)
  u64 lanes = 0;
  switch (form(c, a)) {
    case Form::GENERAL: lanes = lanes_rows<1, 1, 1>(c, a); break;
    case Form::JOINT: lanes = lanes_rows<1, 1, 4>(c, a); break;
    case Form::SMALL_TILES: lanes = lanes_shared<1, 1, 2, 2>(c, a); break;
    case Form::TILES: lanes = lanes_shared<2, 2, 2, 2>(c, a); break;
    case Form::ROWS: lanes = lanes_rows<4, 4, 1>(c, a); break;
  }
  return lanes >> 32 == 0;
}
void launch_linattn(const DevCtx& c, const LinattnArgs& a, hipStream_t s) {
  switch (form(c, a)) {
    case Form::GENERAL: return launch_rows<1, 1, 1, false>(c, a, s);
    case Form::JOINT: return launch_rows<1, 1, 4, true>(c, a, s);
    case Form::SMALL_TILES: return launch_shared<1, 1, 2, 2, 2, 4>(c, a, s);
    case Form::TILES: return launch_shared<2, 2, 2, 2, 1, 4>(c, a, s);
    case Form::ROWS: return launch_rows<4, 4, 1, true>(c, a, s);
  }
}

}  // namespace acehip
