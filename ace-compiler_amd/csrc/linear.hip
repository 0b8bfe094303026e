// linear.hip -- int8 linear layers on ciphertexts: y_j = tok * mul_j * sum_i w_ji x_i mod q on every limb and coefficient.
#include <algorithm>
#include <type_traits>

#include "nn.hpp"

namespace acehip {

// ------------------------------------------------------------------------------------------------
// Matrix-core form.  For one limb the layer is a product of an int8 matrix W by a matrix X of residues, columns = coefficients.  A residue is
// NP signed bytes d_p (x = sum d_p 256^p: the bytes of (x + C) ^ C, C = 0x80 in every byte), so
//   sum_i w_ji x_i = sum_p 256^p (W D_p)_j ,
// NP int8 matrix products with exact 32-bit sums (|sum| <= 2^14 * 2^16 inputs), joined in 64-bit parts and reduced once.
// Layout: a workgroup of four waves takes 16 WN columns and 16 MT WJ outputs, WJ waves along the outputs and WN along the columns.  A step is 64
// inputs: the residues are read once by the workgroup, their bytes transposed in registers (four inputs of a column by v_perm_b32) and left in LDS
// as the B fragments of v_mfma_i32_16x16x64_i8 (1 KiB each, read without bank conflicts); the weights are the A fragments, packed by a kernel of
// their own (or, up to 32 outputs, as their rows lie in memory).  Residues are requested three steps ahead and staged one ahead, weights one.
// Bound: up to 128 outputs by memory (800 -> 32, N = 16384, two rows, three limbs: 0.28 ms, 4.7 TB/s; 333 -> 77, N = 4096, three rows: 62 us, 3.9 TB/s, of
// which the packing takes 5); above by parts that follow each other (768 -> 2304 at N = 16384: 1.67 ms, 2.78 * 10^12 int8 operations, 1.67 POP/s, matrix
// cores busy for 43 % of it at 1.94 GHz: the product with its LDS reads alone takes 1.02 ms, staging adds 0.12, the loads 0.32 and the reduction 0.19;
// a library's int8 product of 8192^3 reaches 2.07 POP/s on this card).
// ------------------------------------------------------------------------------------------------
typedef int v4i_t __attribute__((ext_vector_type(4)));
typedef int v4i_any_t __attribute__((ext_vector_type(4), aligned(1)));
template <class T>
__device__ __forceinline__ GLOBAL T* global(T* p) { return (GLOBAL T*)(uintptr_t)p; }
constexpr u64 kBytes7 = 0x7f7f7f7f7f7f7full;  // the largest residue of seven signed bytes

__device__ __forceinline__ u32 perm(u32 hi, u32 lo, u32 sel) { return __builtin_amdgcn_perm(hi, lo, sel); }
// a pointer that is the same for the wave
template <class T>
__device__ __forceinline__ T* uniform(T* p) { return (T*)uniform64((u64)p); }
// bytes of four dwords transposed: o[b] = byte b of l[0..3]
__device__ __forceinline__ void transpose4(const u32 (&l)[4], u32 (&o)[4]) {
  const u32 a01 = perm(l[1], l[0], 0x05010400u), a23 = perm(l[3], l[2], 0x05010400u);
  const u32 b01 = perm(l[1], l[0], 0x07030602u), b23 = perm(l[3], l[2], 0x07030602u);
  o[0] = perm(a23, a01, 0x05040100u);
  o[1] = perm(a23, a01, 0x07060302u);
  o[2] = perm(b23, b01, 0x05040100u);
  o[3] = perm(b23, b01, 0x07060302u);
}

// The first of 16 bytes that hold the weights from byte `at` of the array on, as far as they are there; of an array of 16 bytes at least.
__host__ __device__ __forceinline__ u64 linear_pack_from(u64 at, u32 n_out, u64 ld_w, u32 n_in) {
  const u64 last = (n_out - 1) * ld_w + n_in - 16;
  return at < last ? at : last;
}

// Weights as A fragments, [tile of 16 outputs][step][lane] of 16 bytes, zero past the matrix.  In memory a fragment's lanes read 16 bytes from each of
// 16 rows, which costs the L1 cache 64 look-ups (four waves a fragment long: the product waits for them); packed, a fragment is 1 KiB in a row:
// 2.62 -> 1.91 ms (768 -> 2304 at N = 16384), with the launch.  Up to 32 outputs one wave reads each fragment and the launch costs what it saves
// (333 -> 30, three rows at 2048: 19.6 us unpacked, 20.3 packed; one row at 1024: 8.9 and 11.6; 800 -> 32 at 16384: 276 and 268).
__global__ __launch_bounds__(256) void linear_pack_kernel(const int8_t* w, u64 ld_w, u32 n_in, u32 n_out, u32 steps, u32 n_frags, v4i_t* out) {
  const u32 f = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63u;
  if (f >= n_frags) return;
  const u32 j = (f / steps) * 16 + (lane & 15u), k = (f % steps) * 64 + 16 * (lane >> 4);
  // 16 bytes from the array, the last ones of it at most (linear_fits asks for 16 of every part), moved to their place; those past the row are cleared
  unsigned __int128 v = 0;
  if (j < n_out && k < n_in) {
    const u64 at = j * ld_w + k, from = linear_pack_from(at, n_out, ld_w, n_in);
    v = __builtin_bit_cast(unsigned __int128, (v4i_t) * (const GLOBAL v4i_any_t*)(global(w) + from)) >> (8 * (u32)(at - from));
    if (n_in - k < 16) v &= ((unsigned __int128)1 << (8 * (n_in - k))) - 1;
  }
  out[(u64)f * 64 + lane] = __builtin_bit_cast(v4i_t, v);
}

// Column blocks of a launch: 16 WN columns of one polynomial of one row.
struct Columns {
  u32 first, n;    // of a workgroup
  u32 log_blocks;  // column blocks of a polynomial
};

template <int NP, int MT, int WJ, int WN, bool PACKED, bool ODD>
__device__ __forceinline__ void linear_tiles(const DevCtx& c, const LinearArgs& a, v4i_t* frag, ulong2* factor, const DevPrime& P, u32 rep, u32 pos, const Columns& cols,
                                             u32 j0) {
  constexpr int G = 4 / WJ;  // column blocks of 16 that a thread stages
  static_assert(4 % WJ == 0 && WJ * WN % 4 == 0, "all of a step's 256 WN groups of inputs are staged");
  const u32 t = threadIdx.x, lane = t & 63u, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const u32 wj = wave % WJ, wn = wave / WJ;
  const u32 last = (a.n_in - 1) / 64;  // step (n_in > 0)
  const u64 q = P.q, mh = P.prec128_hi;
  // where a column block starts in a matrix (uniform)
  auto block = [&](u32 i, const CtMat& m, u64* base, u32& row, u64& off) {
    const u32 cb = cols.first + i, rc = cb >> cols.log_blocks;
    row = __builtin_amdgcn_readfirstlane(rc / a.n_comp);
    const u32 comp = rc - row * a.n_comp;
    off = (u64)pos * c.N + (cb & ((1u << cols.log_blocks) - 1)) * (16 * WN);
    return uniform(base + row * m.row + comp * m.comp + off);
  };
  u64* const x_base = reb(c, a.in.d, rep);
  u64* const y_base = reb(c, a.out.d, rep);
  // addresses: a uniform 64-bit base that moves with the step plus 32-bit offsets of the lanes that stay (linear_fits)
  const u64 xs = a.in.col;
  const u32 k4 = (t >> 4) & 15u, u0 = t >> 8;  // this thread stages inputs 4 k4 .. 4 k4 + 3 of a step in column blocks u0, u0 + WN / G ..
  const u32 k_wave = 16 * (wave & 3u);         // the first of its wave's 16 inputs: the base is the wave's
  u32 x_at[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) x_at[i] = 8 * ((4 * (lane >> 4) + i) * (u32)xs + u0 * 16 + (t & 15u));
  const GLOBAL char* w = (const GLOBAL char*)global(uniform(PACKED ? (const int8_t*)a.packed : reb(c, a.w, rep) + (u64)j0 * a.ld_w));
  u32 w_at[MT];  // of the lane's row; packed: of the fragments' tile, in steps
#pragma unroll
  for (int m = 0; m < MT; ++m)
    w_at[m] = PACKED ? min(j0 / 16 + wj * MT + m, (a.n_out - 1) / 16) * (last + 1)
                     : min((wj * MT + m) * 16 + (lane & 15u), a.n_out - 1 - j0) * (u32)a.ld_w + 16 * (lane >> 4);

  struct Raw {
    u64 v[G][4];
  };
  // the inputs of (tile, step) in their order, through a buffer descriptor that ends behind the last of them: those past n_in read as zero, and
  // behind the last tile nothing is read.  No branch (the steps are one block of code): x_next is made ready once a tile.
  u32 x_tile = 0, x_step = 0, any_row;
  u64 any_off;
  const int x_all = (int)a.n_in - (int)k_wave;
  int x_rest = x_all;
  const int limb16 = (int)xs * 128;
  const u64* x = block(0, a.in, x_base, any_row, any_off) + k_wave * xs;
  const u64* x_next = block(1, a.in, x_base, any_row, any_off) + k_wave * xs;
  auto load_x = [&](Raw& r) {
    const int bytes = x_rest >= 16 ? limb16 : x_rest > 0 ? x_rest * (int)xs * 8 : 0;
    const auto d = __builtin_amdgcn_make_buffer_rsrc((void*)x, 0, bytes, 0x00027000);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int u = 0; u < G; ++u) r.v[u][i] = __builtin_bit_cast(u64, __builtin_amdgcn_raw_buffer_load_b64(d, (int)x_at[i] + u * (WN / G * 128), 0, 0));
    const bool wrap = x_step == (ODD ? last : last | 1u);
    x_step = wrap ? 0 : x_step + 1;
    x_tile += wrap;
    x_rest = wrap ? (x_tile < cols.n ? x_all : 0) : x_rest - 64;
    x = wrap ? x_next : x + 64 * xs;
  };
  auto stage = [&](const Raw& r, v4i_t* buf) {
    constexpr u64 C = NP == 8 ? 0x8080808080808080ull : 0x80808080808080ull;
#pragma unroll
    for (int u = 0; u < G; ++u) {
      u32 lo[4], hi[4], o[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const u64 v = r.v[u][i] + C;
        lo[i] = (u32)v ^ (u32)C;
        hi[i] = (u32)(v >> 32) ^ (u32)(C >> 32);
      }
      transpose4(lo, *(u32(*)[4])o);
      transpose4(hi, *(u32(*)[4])(o + 4));
      u32* d = (u32*)(buf + (u0 + u * (WN / G)) * NP * 64) + ((k4 >> 2) * 16 + (t & 15u)) * 4 + (k4 & 3u);
#pragma unroll
      for (int p = 0; p < NP; ++p) d[p * 256] = o[p];
    }
  };
  const auto packed = __builtin_amdgcn_make_buffer_rsrc((void*)uniform(a.packed), 0, PACKED ? (int)((a.n_out + 15) / 16 * (last + 1) * 1024) : 0, 0x00027000);
  auto load_w = [&](u32 s, v4i_t (&aw)[MT]) {
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      if (PACKED) {
        aw[m] = __builtin_bit_cast(v4i_t, __builtin_amdgcn_raw_buffer_load_b128(packed, (int)lane * 16, __builtin_amdgcn_readfirstlane((w_at[m] + s) * 1024), 0));
      } else {
        u32 at = w_at[m];
        asm("" : "+v"(at));  // (opaque: the loads stay one uniform base and a 32-bit offset each, not a running 64-bit pointer per lane)
        aw[m] = *(const GLOBAL v4i_any_t*)(w + s * 64 + at);
      }
    }
  };
  // the last step's (s = last; a function of s, so that nothing of it is kept over the loop): nothing is read past the array, and the weights
  // past n_in may be any
  auto load_w_last = [&](u32 s, v4i_t (&aw)[MT]) {
    if (PACKED || a.n_in - 64 * s == 64) return load_w(s, aw);
    const u64 end = (u64)(a.n_out - 1 - j0) * a.ld_w + a.n_in - 64 * s;  // of the array, seen from this step
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      u32 at = w_at[m];
      asm volatile("" : "+v"(at));
      const int64_t from = at + 16ull <= end ? (int64_t)at : (int64_t)end - 16;  // (may lie before this step: the array has 16 bytes)
      const u32 skip = 8 * (u32)min((int64_t)at - from, (int64_t)15);
      unsigned __int128 v = __builtin_bit_cast(unsigned __int128, (v4i_t) * (const GLOBAL v4i_any_t*)(w + s * 64 + from));
      aw[m] = __builtin_bit_cast(v4i_t, v >> skip);
    }
  };

  v4i_t acc[MT][NP];
  auto clear = [&] {
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int p = 0; p < NP; ++p) acc[m][p] = v4i_t{0, 0, 0, 0};
  };
  // the B fragments of a step four planes ahead of their use: one LDS latency a step, 16 registers
  constexpr int AHEAD = 4;
  auto fragments = [&](const v4i_t* buf, v4i_t (&b)[AHEAD]) {
#pragma unroll
    for (int p = 0; p < AHEAD; ++p) b[p] = buf[(wn * NP + p) * 64 + lane];
    __builtin_amdgcn_sched_barrier(0);
  };
  auto multiply = [&](const v4i_t (&aw)[MT], const v4i_t* buf, v4i_t (&b)[AHEAD]) {
#pragma unroll
    for (int p = 0; p < NP; ++p) {
#pragma unroll
      for (int m = 0; m < MT; ++m) acc[m][p] = __builtin_amdgcn_mfma_i32_16x16x64_i8(aw[m], b[p % AHEAD], acc[m][p], 0, 0, 0);
      if (p + AHEAD < NP) b[p % AHEAD] = buf[(wn * NP + p + AHEAD) * 64 + lane];
      __builtin_amdgcn_sched_barrier(0x36);  // (arithmetic and requests to memory may cross, LDS reads and matrix instructions not)
    }
  };

  // ---- a tile's results.  Lane: column lane % 16, outputs 4 (lane / 16) + r of each tile.  V = sum_p acc_p 256^p is reduced by its rounded quotient in
  // floating point: |V / q| <= 2^7 n_in <= 2^23, and what the doubles leave out of V (its low 32 bits, roundings of two units of 2^32) is below
  // 2^-6 q at primes above 2^40.  V - round(V / q) q is then within (1/2 + 2^-5) q of zero, so its low 64 bits tell it.
  const u32 g4 = 4 * (lane >> 4), n = wn * 16 + (lane & 15u);
  const u32 y_at = 8 * (g4 * (u32)a.out.col + n);
  const u32 left = a.n_out - j0 - min(a.n_out - j0, wj * MT * 16);  // outputs of this wave that are there
  const u64 nq = 0 - q;
  const double inv = __builtin_bit_cast(double, (u64)uniform((char*)__builtin_bit_cast(u64, 4294967296.0 / (double)q)));
  if (a.mul && t < 16 * MT * WJ) {  // channel factors and their companions (read behind the first barrier of the steps)
    const u64 m = signed_mod(global(reb(c, a.mul, rep))[min(j0 + t, a.n_out - 1)], q, mh);
    factor[t] = ulong2{m, m * mh + mulhi64(m, P.prec128_lo)};
  }
  u32 tile = 0, row;
  u64 off, tok = 0;
  GLOBAL char* y;
  auto begin = [&] {
    x_next = block(x_tile + 1, a.in, x_base, any_row, any_off) + k_wave * xs;
    y = (GLOBAL char*)global(block(tile, a.out, y_base, row, off) + (u64)(j0 + wj * MT * 16) * a.out.col);
    y = (GLOBAL char*)uniform((char*)y);
    if (a.tok) tok = global(uniform(reb(c, a.tok, rep) + row * a.tok_stride + off))[n];
    clear();
  };
  auto finish = [&](auto with_mul, auto with_tok) {
    const u64 tokp = tok * mh + mulhi64(tok, P.prec128_lo);
    double magic = 6755399441055744.0;  // 1.5 * 2^52: the sum's low bits are the rounded integer, plus those of the constant
    u64 start = __builtin_bit_cast(u64, magic) * q, col = a.out.col * 8;
    int weight[4] = {1, 1 << 8, 1 << 16, 1 << 24};
    // (opaque: each byte's sum joins by ONE v_mad_i64_i32, and nothing made of these is kept over the steps)
    asm volatile("" : "+s"(magic), "+s"(start), "+s"(col), "+s"(weight[0]), "+s"(weight[1]), "+s"(weight[2]), "+s"(weight[3]));
    GLOBAL char* at = y;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        int64_t lo = 0;
#pragma unroll
        for (int p = 0; p < 4; ++p) lo += (int64_t)acc[m][p][r] * weight[p];
        u32 hi = 0;
        double f = 0;
#pragma unroll
        for (int p = NP - 1; p >= 4; --p) {
          hi = (hi << 8) + (u32)acc[m][p][r];
          f = __builtin_fma(f, 256.0, (double)acc[m][p][r]);
        }
        f += (double)(int)(lo >> 32);
        const u64 quot = __builtin_bit_cast(u64, __builtin_fma(f, inv, magic));
        u64 v = (u64)lo + ((u64)hi << 32) + start + quot * nq;
        if (with_mul || with_tok) {
          v += q;
          if (with_mul) {
            const ulong2 f = factor[(wj * MT + m) * 16 + g4 + r];
            v = mul_near(v, f.x, f.y, nq);
          }
          if (with_tok) v = mul_near(v, tok, tokp, nq);
          v = v >= 2 * q ? v - 2 * q : v;
          v = v >= q ? v - q : v;
        } else {
          v += q & (u64)((int64_t)v >> 63);
        }
        if (m * 16 + r + g4 < left) *(GLOBAL u64*)(at + y_at) = v;
        at += r == 3 ? 13 * col : col;
      }
  };
  auto store = [&] {
    using T = std::true_type;
    using F = std::false_type;
    if (a.mul) a.tok ? finish(T{}, T{}) : finish(T{}, F{});
    else       a.tok ? finish(F{}, T{}) : finish(F{}, F{});
  };

  // ---- the steps of all tiles in one pipeline: inputs are requested three steps ahead and staged one ahead, across the tiles' borders, so that
  // a tile's first inputs are under way while the one before it is reduced.  Steps go in pairs (registers and buffers in turn); ODD, an odd number of
  // steps: so do tiles (an empty step in place of that: 14 -> 11 at N = 32768, three limbs, 37 us, 30 in pairs of tiles; 180 -> 128 at 16384 57 and
  // 53).  Behind the last step weights are read again and inputs as zeros, never to be used: without a branch around the requests the compiler counts
  // them exactly and waits for the oldest only.
  v4i_t *buf0 = frag, *buf1 = frag + WN * NP * 64;
  Raw raw0, raw1;
  v4i_t aw0[MT], aw1[MT];
  load_x(raw0);
  if (ODD) x_next = block(x_tile + 1, a.in, x_base, any_row, any_off) + k_wave * xs;  // (a tile of one step)
  load_x(raw1);
  if (ODD) x_next = block(x_tile + 1, a.in, x_base, any_row, any_off) + k_wave * xs;
  if (!PACKED && last == 0) load_w_last(0, aw0);
  else                      load_w(0, aw0);
  stage(raw0, buf0);
  load_x(raw0);
  auto step = [&](u32 ahead, const v4i_t* buf, const v4i_t (&aw)[MT], Raw& raw, v4i_t* buf_next, v4i_t (&aw_next)[MT]) {
    v4i_t b[AHEAD];
    lds_barrier();
    fragments(buf, b);
    if (!PACKED && ahead == last) load_w_last(ahead, aw_next);
    else                          load_w(ahead, aw_next);
    __builtin_amdgcn_sched_barrier(0);  // (weights first: the next step waits for them and not for the inputs behind them)
    stage(raw, buf_next);
    load_x(raw);
    multiply(aw, buf, b);
  };
  auto even = [&](u32 ahead) { step(ahead, buf0, aw0, raw1, buf1, aw1); };
  auto odd = [&](u32 ahead) { step(ahead, buf1, aw1, raw0, buf0, aw0); };
  if (!ODD) {
    for (tile = 0; tile < cols.n; ++tile) {
      begin();
      for (u32 s = 0; s < last; s += 2) {
        even(s + 1);
        odd(s + 2 > last ? 0 : s + 2);
      }
      store();
    }
  } else {
    for (tile = 0; tile < cols.n; ++tile) {
      begin();
      for (u32 s = 0; s < last; s += 2) {
        even(s + 1);
        odd(s + 2);
      }
      even(0);
      store();
      if (++tile == cols.n) break;
      begin();
      for (u32 s = 0; s < last; s += 2) {
        odd(s + 1);
        even(s + 2);
      }
      odd(0);
      store();
    }
  }
}

// A workgroup takes `tiles` column blocks that follow each other (the last workgroup what is left).
template <int MT, int WJ, int WN, bool PACKED, bool ODD>
__global__ __launch_bounds__(64 * WJ * WN, 2) void linear_i8_mfma_kernel(DevCtx c, LinearArgs a, u32 j_blocks, u32 log_blocks, u32 tiles) {
  __shared__ v4i_t frag[2 * WN * 8 * 64];
  __shared__ ulong2 factor[16 * MT * WJ];
  // workgroups that read the same columns run side by side on one XCD (ids congruent mod 8): its L2 keeps the residues for all outputs
  const u32 groups = gridDim.x / j_blocks;
  u32 jb, g;
  if ((groups & 7u) == 0) {
    const u32 b = blockIdx.x >> 3;
    jb = b % j_blocks;
    g = (b / j_blocks) * 8 + (blockIdx.x & 7u);
  } else {
    jb = blockIdx.x % j_blocks;
    g = blockIdx.x / j_blocks;
  }
  jb = __builtin_amdgcn_readfirstlane(jb);
  g = __builtin_amdgcn_readfirstlane(g);
  const u32 pos = a.pos0 + blockIdx.y, gi = limb_prime(pos, a.level, c.L), rep = c.rep0 + blockIdx.z;
  if (!owns(c, gi)) return;
  const DevPrime P = c.primes[gi];
  const u32 all = (a.rows * a.n_comp) << log_blocks;
  const Columns cols{g * tiles, min(tiles, all - g * tiles), log_blocks};
  const u32 j0 = jb * (16 * MT * WJ);
  if (P.q <= kBytes7) linear_tiles<7, MT, WJ, WN, PACKED, ODD>(c, a, frag, factor, P, rep, pos, cols, j0);
  else                linear_tiles<8, MT, WJ, WN, PACKED, ODD>(c, a, frag, factor, P, rep, pos, cols, j0);
}

// What the matrix-core form does not take (linear_fits: rings below 64, primes below 2^40, inputs that share words or lie 128 MiB apart): one
// coefficient per lane, kJ outputs, residues split at 31 bits, so that each half times a weight is one multiply-add into a signed 64-bit sum
// (|sum| <= 2^31 * 2^7 * 2^16 inputs).
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

// the matrix-core form: rings and primes that it takes, inputs that lie apart (a descriptor that ends behind the last one reads zeros for those past
// it), lane offsets below 2^32, and an array of weights that holds a fragment of 16 bytes
static bool linear_fits(const DevCtx& c, const LinearArgs& a) {
  return c.N >= 64 && a.wide_primes && a.in.col >= c.N && a.in.col < (1u << 24) && a.out.col < (1u << 25) && a.ld_w <= (1u << 24) && a.n_in != 0 &&
         (u64)(a.n_out - 1) * a.ld_w + a.n_in >= 16;
}

template <int MT, int WJ, int WN>
static void launch_mfma(const DevCtx& c, const LinearArgs& a, hipStream_t s) {
  u32 log_blocks = 0;
  while ((16u * WN << log_blocks) < c.N) ++log_blocks;
  const u32 all = (a.rows * a.n_comp) << log_blocks, j_blocks = (a.n_out + 16 * MT * WJ - 1) / (16 * MT * WJ);
  // several column blocks to a workgroup while two for each place are left (two workgroups on each of 256 CUs): one block each takes 1.81 ms in place
  // of 1.64 (768 -> 2304 at N = 16384, three limbs), 235 us in place of 206 (512 -> 512 at 8192, four limbs); fewer workgroups leave places empty at
  // the end (77 outputs of 333 at 4096: 68 us in place of 61)
  const u64 blocks = (u64)all * j_blocks * a.n_limbs * c.nrep;
  u32 tiles = 1;
  while (tiles < 8 && blocks / (2 * tiles) >= 1024) tiles *= 2;
  const dim3 grid((all + tiles - 1) / tiles * j_blocks, a.n_limbs, c.nrep), block(64 * WJ * WN);
  const auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, block, 0, s, c, a, j_blocks, log_blocks, tiles); };
  const bool odd = (a.n_in + 63) / 64 % 2 != 0;
  if constexpr (MT * WJ > 2) {  // (linear_pack_outputs)
    if (a.packed) return odd ? launch(linear_i8_mfma_kernel<MT, WJ, WN, true, true>) : launch(linear_i8_mfma_kernel<MT, WJ, WN, true, false>);
  }
  odd ? launch(linear_i8_mfma_kernel<MT, WJ, WN, false, true>) : launch(linear_i8_mfma_kernel<MT, WJ, WN, false, false>);
}

// Outputs of a workgroup.  Waves along the outputs first, then along the columns: a thread then stages one or two column blocks, and what it holds of the
// inputs in flight stays in registers (four blocks, <4, 1, 4> for 33 .. 64 outputs, spill: 141 -> 48 at N = 16384 237 us in place of 81; 141 -> 20 by
// <2, 1, 4> 80 in place of 58).  Above 128 outputs three or four tiles a wave, whichever leaves fewer idle: 333 -> 300 at 2048 64 us by three, 76 by
// four.  Two for all widths read the inputs more often (768 -> 2304: 2.0 ms), five do not fit the registers.
static u32 linear_width(u32 n_out) {
  return n_out <= 32 ? 32 : n_out <= 64 ? 64 : n_out <= 128 ? 128 : n_out <= 192 * ((n_out + 255) / 256) ? 192 : 256;
}
// Outputs whose packed weights fit the workspace at a time (all of them unless the layer is large); 0: the weights are read as they lie, also where
// every workgroup has a place at once (two on each of 256 CUs) and packing is one launch more: 700 -> 1000 at N = 1024 22 us, 32 packed; 92 -> 103 at 2048,
// two limbs, 8.7 and 11.1; at twice as many workgroups 17 -> 244 at 2048, two rows and limbs: 22.7 and 20.3.  Rows that do not lie on words of four bytes
// cost more each time they are read: 1151 -> 211 at 1024, two rows, 39 us, 22 packed (1148 inputs: 21 and 21); 301 -> 250 at 2048 16.3 and 13.7; few
// inputs are worth no launch then either (151 -> 50 at 1024: 8.6 and 11.2)
static bool linear_takes_packed(const DevCtx& c, const LinearArgs& a) { return linear_fits(c, a) && a.n_out > 32; }
static u32 linear_pack_outputs(const DevCtx& c, const LinearArgs& a, size_t ws_bytes) {
  if (!linear_takes_packed(c, a)) return 0;
  const u32 width = linear_width(a.n_out), columns = width == 64 ? 32 : 16;
  const bool words = (((u64)(uintptr_t)a.w | a.ld_w) & 3) == 0;
  if ((words || a.n_in <= 256) && (u64)a.rows * a.n_comp * a.n_limbs * c.nrep * (c.N / columns) * ((a.n_out + width - 1) / width) <= 512) return 0;
  const u64 tile = (u64)((a.n_in + 63) / 64) * 1024, tiles = std::min(ws_bytes, (size_t)1 << 31) / tile;  // (32-bit offsets)
  if (tiles * 16 >= a.n_out) return a.n_out;
  return (u32)(tiles / 16 * 256);  // whole workgroups
}
static void launch_linear_pack(const LinearArgs& a, void* out, hipStream_t s) {
  const u32 steps = (a.n_in + 63) / 64, n_frags = (a.n_out + 15) / 16 * steps;
  hipLaunchKernelGGL(linear_pack_kernel, dim3((n_frags + 3) / 4), dim3(256), 0, s, a.w, a.ld_w, a.n_in, a.n_out, steps, n_frags, (v4i_t*)out);
}

static void launch_linear_i8(const DevCtx& c, const LinearArgs& a, hipStream_t s) {
  if (!linear_fits(c, a)) {
    const u32 n_blocks = (c.N + 255) / 256, j_blocks = (a.n_out + kJ - 1) / kJ;
    hipLaunchKernelGGL(linear_i8_kernel, dim3(n_blocks * j_blocks * a.n_comp * a.rows, a.n_limbs, c.nrep), dim3(256), 0, s, c, a, n_blocks, j_blocks);
    return;
  }
  switch (linear_width(a.n_out)) {
    case 32: return launch_mfma<1, 2, 2>(c, a, s);
    case 64: return launch_mfma<2, 2, 2>(c, a, s);
    case 128: return launch_mfma<2, 4, 1>(c, a, s);
    case 192: return launch_mfma<3, 4, 1>(c, a, s);
    default: return launch_mfma<4, 4, 1>(c, a, s);
  }
}

// A last part may be one that the packed form does not take: up to 32 outputs, or weights of fewer bytes than a fragment's 16.
void launch_linear(const DevCtx& c, const DevCtx* launches, u32 n_launches, LinearArgs a, void* ws, size_t ws_bytes, hipStream_t s) {
  const LinearArgs all = a;
  const u32 part = ws ? linear_pack_outputs(c, a, ws_bytes) : 0;
  for (u32 j = 0; j < all.n_out; j += part ? part : all.n_out) {
    a.out.d = all.out.d + (u64)j * all.out.col;
    a.w = all.w + (u64)j * all.ld_w;
    a.mul = all.mul ? all.mul + j : nullptr;
    a.n_out = part ? std::min(part, all.n_out - j) : all.n_out;
    a.packed = part && linear_takes_packed(c, a) ? ws : nullptr;
    if (a.packed) launch_linear_pack(a, ws, s);
    for (u32 l = 0; l < n_launches; ++l) launch_linear_i8(launches[l], a, s);
  }
}

}  // namespace acehip
