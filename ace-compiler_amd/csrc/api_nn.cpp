// api_nn.cpp -- C ABI (include/acehip.h): operators of a transformer on ciphertexts -- int8 linear layers, rotary positions, linear attention.
#include "api_internal.hpp"
#include "nn.hpp"

static_assert(sizeof(acehip_mat) == sizeof(CtMat), "acehip_mat / CtMat layout mismatch");

namespace {
using i128 = __int128;

// A matrix argument with its counts: words it spans, and the checks that every entry point makes of it.
struct View {
  CtMat m;
  u64 n[4];  // heads, rows, cols, comps
  u64 lo = 0, hi = 0;  // byte addresses of its first word and behind its last one (the limbs of the call)
  u64 limb0 = 0, span = 0;  // bytes from a polynomial's start to the first limb, bytes of the limbs
  bool empty() const { return n[0] == 0 || n[1] == 0 || n[2] == 0 || n[3] == 0 || span == 0; }
  u64 stride(int k) const { return k == 0 ? m.head : k == 1 ? m.row : k == 2 ? m.col : m.comp; }
};

struct Call {
  acehip_ctx* c;
  const char* name;
  u32 level, pos0, n_limbs;
  int bad(const char* what) const { return fail(ACEHIP_EINVAL, std::string(name) + ": " + what); }

  // arguments first, the device last (check_dev where the launch is due): what a call refuses does not hang on a GPU being there
  int range() const {
    if (!c) return fail(ACEHIP_EINVAL, "null context");
    if (level > c->hp.L) return bad("level exceeds the number of q primes");
    if (pos0 > level + c->hp.K || n_limbs > level + c->hp.K - pos0) return bad("limb range exceeds level + K");
    return ACEHIP_OK;
  }
  // every prime of the call is above 2^bits and up to 2^64 / 9 (all but those of chosen test chains)
  bool primes_above(u32 bits) const {
    for (u32 p = pos0; p < pos0 + n_limbs; ++p) {
      const u64 q = c->hp.q(limb_prime(p, level, c->hp.L));
      if (q >> bits == 0 || q > ~0ull / 9) return false;
    }
    return true;
  }
  int view(View& v, const acehip_mat* a, u64 heads, u64 rows, u64 cols, u64 comps) const {
    v.n[0] = heads, v.n[1] = rows, v.n[2] = cols, v.n[3] = comps;
    v.limb0 = 8ull * pos0 * c->hp.N;
    v.span = 8ull * n_limbs * c->hp.N;
    if (v.empty()) return ACEHIP_OK;
    if (!a || !a->data) return bad("null matrix");
    v.m = CtMat{a->data, a->head_stride, a->row_stride, a->col_stride, a->comp_stride};
    i128 far = (i128)v.limb0 + v.span;
    for (int k = 0; k < 4; ++k) far += (i128)(v.n[k] - 1) * v.stride(k) * 8;
    const u64 at = (u64)(uintptr_t)a->data;
    if (at % 8) return bad("a matrix is not aligned to 8 bytes");
    if (far > ((i128)1 << 62) || at > ~0ull - (u64)far) return bad("the strides of a matrix leave the address space");
    v.lo = at + v.limb0;
    v.hi = at + (u64)far;
    return memory(at, v.hi, false);
  }
  // operands inside the arena have to lie in one replica of it; with several replicas (or simulated ranks) selected a result has to lie there
  int memory(u64 lo, u64 hi, bool result) const {
    if (c->dc.rep_span == 0) return ACEHIP_OK;
    const u64 a0 = c->dc.rep_lo, a1 = a0 + c->dc.rep_span;
    const bool inside = lo >= a0 && hi <= a1;
    if (!inside && lo < a1 && hi > a0) return bad("an operand crosses the end of the arena");
    const DcList l = launch_dcs(c);
    if (result && !inside && l.n * l.d[0].nrep > 1) return bad("a result outside the arena under several replicas");
    return ACEHIP_OK;
  }
};

// Ranges of bytes [lo + sum_k i_k stride_k, .. + span), 0 <= i_k < n_k: the polynomials of a matrix (the limbs of the call), the rows of a table.
struct Ranges {
  u64 lo, span, stride[4] = {}, n[4] = {1, 1, 1, 1};
};
Ranges ranges(const View& v) {
  Ranges r{v.lo, v.span};
  for (int k = 0; k < 4; ++k) r.stride[k] = 8 * v.stride(k), r.n[k] = v.n[k];
  return r;
}
// Whether two ranges of two sets meet (or two of one set), by the differences of their starts, d + sum_k c_k stride_k: the axes are gone through from
// the widest stride on, and of each only the c_k are followed with which the axes behind it can still bring the difference near zero -- a few of them
// where the strides are nested (two interleaved matrices of 2^19 polynomials: 3 us a call in place of 42 ms, listed and sorted).
enum Meet { APART, MEET, UNKNOWN };
class Differences {
  struct Axis {
    i128 stride, lo, hi;
  };
  Axis axis_[8];
  int n_ = 0;
  i128 below_[9], above_[9];  // what the axes from k on add
  i128 from_, to_;            // of ranges that meet: from < difference < to
  u32 steps_ = 0;

 public:
  static constexpr u32 kSteps = 1u << 14;  // (some milliseconds)
  Differences(i128 from, i128 to) : from_(from), to_(to) {}
  // c in [lo, hi]; false: there was an axis of this stride
  bool axis(u64 stride, i128 lo, i128 hi) {
    for (int k = 0; k < n_; ++k)
      if (axis_[k].stride == (i128)stride) {
        axis_[k].lo += lo;
        axis_[k].hi += hi;
        return false;
      }
    axis_[n_++] = Axis{(i128)stride, lo, hi};
    return true;
  }
  // but_zero: the difference of all c = 0 does not count
  Meet find(i128 d, bool but_zero) {
    std::sort(axis_, axis_ + n_, [](const Axis& x, const Axis& y) { return x.stride > y.stride; });
    below_[n_] = above_[n_] = 0;
    for (int k = n_ - 1; k >= 0; --k) {
      below_[k] = below_[k + 1] + axis_[k].lo * axis_[k].stride;
      above_[k] = above_[k + 1] + axis_[k].hi * axis_[k].stride;
    }
    return step(0, d, but_zero);
  }

 private:
  static i128 floor_div(i128 a, i128 b) { return a / b - (a % b < 0); }
  Meet step(int k, i128 d, bool zero) {
    if (k == n_) return zero || d <= from_ || d >= to_ ? APART : MEET;
    if (++steps_ > kSteps) return UNKNOWN;
    const Axis& a = axis_[k];
    const i128 lo = std::max(a.lo, floor_div(from_ - above_[k + 1] - d, a.stride) + 1), hi = std::min(a.hi, -floor_div(d + below_[k + 1] - to_, a.stride) - 1);
    for (i128 c = lo; c <= hi; ++c)
      if (const Meet m = step(k + 1, d + c * a.stride, zero && c == 0)) return m;
    return APART;
  }
};

// Strides that cross too often for that: the ranges one by one.
constexpr u64 kListed = 1ull << 20;
u64 count(const Ranges& r) {  // (no n is 0; 2^64 - 1 where there are more)
  u64 c = 1;
  for (u64 n : r.n) c = c > ~0ull / n ? ~0ull : c * n;
  return c;
}
bool starts(const Ranges& r, std::vector<u64>& s) try {
  if (count(r) > kListed) return false;
  for (u64 i = 0; i < r.n[0]; ++i)
    for (u64 j = 0; j < r.n[1]; ++j)
      for (u64 k = 0; k < r.n[2]; ++k)
        for (u64 l = 0; l < r.n[3]; ++l) s.push_back(r.lo + i * r.stride[0] + j * r.stride[1] + k * r.stride[2] + l * r.stride[3]);
  std::sort(s.begin(), s.end());
  return true;
} catch (const std::bad_alloc&) {
  return false;
}
bool apart(const Ranges& x) {
  Differences d(-(i128)x.span, x.span);
  for (int k = 0; k < 4; ++k)
    if (x.n[k] > 1 && (x.stride[k] == 0 || !d.axis(x.stride[k], -(i128)(x.n[k] - 1), x.n[k] - 1))) return false;
  const Meet m = d.find(0, true);
  if (m != UNKNOWN) return m == APART;
  std::vector<u64> s;
  if (!starts(x, s)) return false;
  for (size_t i = 1; i < s.size(); ++i)
    if (s[i] - s[i - 1] < x.span) return false;
  return true;
}
bool apart(const Ranges& x, const Ranges& y) {
  Differences d(-(i128)x.span, y.span);
  for (int k = 0; k < 4; ++k) {
    if (x.n[k] > 1 && x.stride[k]) d.axis(x.stride[k], 0, x.n[k] - 1);
    if (y.n[k] > 1 && y.stride[k]) d.axis(y.stride[k], -(i128)(y.n[k] - 1), 0);
  }
  const Meet m = d.find((i128)x.lo - y.lo, false);
  if (m != UNKNOWN) return m == APART;
  std::vector<u64> s, t;
  if (!starts(x, s) || !starts(y, t)) return false;
  for (u64 at : t) {  // the last range of x that starts up to there, and the one behind it
    const auto it = std::upper_bound(s.begin(), s.end(), at);
    if ((it != s.begin() && at - *(it - 1) < x.span) || (it != s.end() && *it - at < y.span)) return false;
  }
  return true;
}

// every polynomial of a result has words of its own
int check_result(const Call& k, const View& v) {
  if (v.empty()) return ACEHIP_OK;
  if (int e = k.memory(v.lo, v.hi, true)) return e;
  return apart(ranges(v)) ? ACEHIP_OK : k.bad("the polynomials of a result overlap");
}
int check_apart(const Call& k, const View& out, const View& in) {
  return out.empty() || in.empty() || apart(ranges(out), ranges(in)) ? ACEHIP_OK : k.bad("a result overlaps an operand");
}
// a table of plaintexts, of rows and of columns
int check_table(const Call& k, const View& out, const u64* p, u64 rows, u64 row_stride, u64 cols, u64 col_stride) {
  const acehip_mat m{const_cast<u64*>(p), 0, row_stride, col_stride, 0};
  View t;
  if (int e = k.view(t, &m, 1, rows, cols, 1)) return e;
  return check_apart(k, out, t);
}
// a plain array argument: alignment, arena, distance from the result
int check_array(const Call& k, const View& out, const void* p, i128 bytes, u32 align) {
  if (!p || bytes <= 0) return ACEHIP_OK;
  const u64 at = (u64)(uintptr_t)p;
  if (at % align) return k.bad("an array is not aligned to its type");
  if (bytes > ((i128)1 << 62) || at > ~0ull - (u64)bytes) return k.bad("the strides of an array leave the address space");
  if (int e = k.memory(at, at + (u64)bytes, false)) return e;
  return out.empty() || apart(ranges(out), Ranges{at, (u64)bytes}) ? ACEHIP_OK : k.bad("a result overlaps an operand");
}
// a launch takes less than 2^32 lanes along x: workgroups of 256 there (limbs and replicas are its y and z)
int check_blocks(const Call& k, i128 blocks) {
  return blocks >= ((i128)1 << 24) || k.n_limbs > 65535 ? k.bad("too many results for one call") : ACEHIP_OK;
}
}  // namespace

extern "C" {

int acehip_linear_i8(acehip_ctx* c, const acehip_mat* out, const acehip_mat* in, const int8_t* d_w, size_t ld_w, uint32_t rows, uint32_t n_in,
                     uint32_t n_out, uint32_t n_comp, const int64_t* d_mul, const uint64_t* d_tok, size_t tok_stride, uint32_t level, uint32_t pos0,
                     uint32_t n_limbs, acehip_stream s) {
  const Call k{c, "acehip_linear_i8", level, pos0, n_limbs};
  if (int e = k.range()) return e;
  if (n_in > ACEHIP_LINEAR_MAX_IN) return k.bad("more than ACEHIP_LINEAR_MAX_IN inputs");
  View y, x;
  if (int e = k.view(y, out, 1, rows, n_out, n_comp)) return e;
  if (y.empty()) return check_dev(c);
  if (int e = k.view(x, in, 1, rows, n_in, n_comp)) return e;
  if (n_in && !d_w) return k.bad("null weights");
  if (n_in && ld_w < n_in && n_out > 1) return k.bad("a row of weights is shorter than n_in");
  if (int e = check_result(k, y)) return e;
  if (int e = check_apart(k, y, x)) return e;
  if (n_in)
    if (int e = check_array(k, y, d_w, (i128)(n_out - 1) * ld_w + n_in, 1)) return e;
  if (int e = check_array(k, y, d_mul, (i128)8 * n_out, 8)) return e;
  if (d_tok)
    if (int e = check_table(k, y, d_tok, rows, tok_stride, 1, 0)) return e;
  const i128 polys = (i128)rows * n_comp;
  if (int e = check_blocks(k, polys * ((c->hp.N + 255) / 256) * (((u64)n_out + 7) / 8))) return e;
  if (int e = check_dev(c)) return e;
  LinearArgs a;
  a.out = y.m;
  a.in = x.m;
  a.w = d_w;
  a.ld_w = ld_w;
  a.mul = d_mul;
  a.tok = d_tok;
  a.tok_stride = tok_stride;
  a.rows = rows, a.n_in = n_in, a.n_out = n_out, a.n_comp = n_comp;
  a.level = level, a.pos0 = pos0, a.n_limbs = n_limbs;
  a.wide_primes = k.primes_above(40);
  // (weights inside the arena differ from replica to replica: they are read as they lie)
  const bool shared = c->dc.rep_span == 0 || (u64)(uintptr_t)d_w - c->dc.rep_lo >= c->dc.rep_span;
  const DcList l = launch_dcs(c);
  // one copy for all replicas of the call, in the workspace of the first: what is not selected stays as it is
  const bool moved = (u64)(uintptr_t)c->ws - c->dc.rep_lo < c->dc.rep_span;
  u64* const ws = c->ws + (moved ? l.d[0].rep0 * (c->dc.rep_stride / sizeof(u64)) : 0);
  launch_linear(c->dc, l.d, l.n, a, shared ? ws : nullptr, c->ws_words * sizeof(u64), (hipStream_t)s);
  const u64 limb = 8ull * c->hp.N * n_limbs * rows;
  stat(ST_LINEAR, (u64)rows * n_out, limb * ((u64)n_comp * n_in + (u64)n_comp * n_out + (d_tok ? 1 : 0)) + (u64)n_in * n_out);
  return post_launch();
}

int acehip_rope_messages(acehip_ctx* c, double* d_cos, double* d_sin, size_t out_stride, const double* d_pos, size_t pos_stride, uint32_t n_pos,
                         const double* h_freq, const uint32_t* h_axis, uint32_t n_pairs, uint32_t n_axes, acehip_stream s) {
  const Call k{c, "acehip_rope_messages", 0, 0, 0};
  if (!c) return fail(ACEHIP_EINVAL, "null context");
  if (n_axes > ROPE_AXES_MAX) return k.bad("more than eight axes");
  if (n_pairs > 65535) return k.bad("more than 65535 pairs");
  if (n_pos >> 31) return k.bad("2^31 or more positions");
  if (n_pos == 0 || n_pairs == 0) return check_dev(c);
  if (!d_cos || !d_sin || !d_pos || !h_freq || !h_axis) return k.bad("null argument");
  for (u32 i = 0; i < n_pairs; ++i)
    if (h_axis[i] >= n_axes) return k.bad("an axis index is not below n_axes");
  if (n_pairs > 1 && out_stride < n_pos) return k.bad("the messages of the pairs overlap");
  const i128 out_bytes = (i128)8 * (n_pairs - 1) * out_stride + 8ull * n_pos, pos_bytes = (i128)8 * (n_axes - 1) * pos_stride + 8ull * n_pos;
  for (const void* p : {(const void*)d_cos, (const void*)d_sin, (const void*)d_pos})
    if ((uintptr_t)p % 8) return k.bad("an array is not aligned to its type");
  if (out_bytes > ((i128)1 << 62) || pos_bytes > ((i128)1 << 62)) return k.bad("the strides of an array leave the address space");
  const u64 co = (u64)(uintptr_t)d_cos, si = (u64)(uintptr_t)d_sin, po = (u64)(uintptr_t)d_pos, ob = (u64)out_bytes, pb = (u64)pos_bytes;
  const Ranges vc{co, 8ull * n_pos, {8 * out_stride}, {n_pairs, 1, 1, 1}}, vs{si, 8ull * n_pos, {8 * out_stride}, {n_pairs, 1, 1, 1}},
      vp{po, 8ull * n_pos, {8 * pos_stride}, {n_axes, 1, 1, 1}};
  if (!apart(vc, vs) || !apart(vc, vp) || !apart(vs, vp)) return k.bad("a result overlaps an operand");
  // (shared by all replicas like the plaintexts made of them: the arena is for polynomials)
  for (const auto& [p, b] : {std::pair<u64, u64>{co, ob}, {si, ob}, {po, pb}})
    if (c->dc.rep_span && p < c->dc.rep_lo + c->dc.rep_span && p + b > c->dc.rep_lo) return k.bad("positions and messages do not lie in the arena");
  if (int e = check_dev(c)) return e;
  for (u32 i0 = 0; i0 < n_pairs; i0 += ROPE_PAIRS_MAX) {
    RopeAngles a;
    const u32 n = std::min(ROPE_PAIRS_MAX, n_pairs - i0);
    for (u32 i = 0; i < n; ++i) {
      a.freq[i] = h_freq[i0 + i];
      a.axis[i] = (uint8_t)h_axis[i0 + i];
    }
    launch_rope_messages(d_cos + i0 * out_stride, d_sin + i0 * out_stride, out_stride, d_pos, pos_stride, n_pos, a, n, (hipStream_t)s);
  }
  return post_launch();
}

int acehip_rope(acehip_ctx* c, const acehip_mat* out, const acehip_mat* in, const uint64_t* d_cos, const uint64_t* d_sin, size_t pair_stride,
                size_t row_stride, uint32_t n_heads, uint32_t rows, uint32_t dim, uint32_t n_comp, int interleaved, uint32_t level, uint32_t pos0,
                uint32_t n_limbs, acehip_stream s) {
  const Call k{c, "acehip_rope", level, pos0, n_limbs};
  if (int e = k.range()) return e;
  if (dim % 2) return k.bad("the features of a head come in pairs");
  View y, x;
  if (int e = k.view(y, out, n_heads, rows, dim, n_comp)) return e;
  if (y.empty()) return check_dev(c);
  if (int e = k.view(x, in, n_heads, rows, dim, n_comp)) return e;
  if (!d_cos || !d_sin) return k.bad("null table");
  if (int e = check_result(k, y)) return e;
  // in place: every pair is read and written by the same lanes
  const bool same = x.m.d == y.m.d && x.m.head == y.m.head && x.m.row == y.m.row && x.m.col == y.m.col && x.m.comp == y.m.comp;
  if (!same)
    if (int e = check_apart(k, y, x)) return e;
  for (const u64* table : {d_cos, d_sin})
    if (int e = check_table(k, y, table, rows, row_stride, dim / 2, pair_stride)) return e;
  if (int e = check_blocks(k, (i128)((c->hp.N + 255) / 256) * (dim / 2) * rows)) return e;
  if (int e = check_dev(c)) return e;
  RopeArgs a;
  a.out = y.m;
  a.in = x.m;
  a.cosp = d_cos, a.sinp = d_sin;
  a.pair_stride = pair_stride, a.row_stride = row_stride;
  a.n_heads = n_heads, a.rows = rows, a.dim = dim, a.interleaved = interleaved != 0, a.n_comp = n_comp;
  a.level = level, a.pos0 = pos0, a.n_limbs = n_limbs;
  for (const DevCtx& dc : launch_dcs(c)) launch_rope(dc, a, (hipStream_t)s);
  const u64 limb = 8ull * c->hp.N * n_limbs * rows;
  stat(ST_ROPE, (u64)n_heads * rows * dim, limb * dim * (2ull * n_heads * n_comp + 1));
  return post_launch();
}

// the counts of a linear attention call that its entry points share
static int check_heads(const Call& k, u32 n_heads, u32 n_kv_heads, u32 n_q, u32 n_k, u32 dim) {
  if (n_heads && (n_kv_heads == 0 || n_heads % n_kv_heads)) return k.bad("n_heads is not a multiple of n_kv_heads");
  if ((n_q | n_k | dim) >> 31) return k.bad("2^31 or more tokens or features");
  return ACEHIP_OK;
}
// pairs (query, key) of a call: of a causal one, the last query sees all keys, each one before it one key less
static u64 seen(u64 n_q, u64 n_k, int causal) {
  const u64 r = std::min(n_q, n_k);
  return causal ? r * n_k - r * (r - 1) / 2 : n_q * n_k;
}
static int run_linattn(const Call& k, LinattnArgs& a, const View& y, u64 polys, acehip_stream s) {
  acehip_ctx* c = k.c;
  a.out = y.m;
  a.level = k.level, a.pos0 = k.pos0, a.n_limbs = k.n_limbs;
  a.wide_primes = k.primes_above(32);
  DcList l = launch_dcs(c);
  for (u32 i = 0; i < l.n; ++i) {
    l.d[i].N = c->hp.N;  // (a context without a device has none there)
    if (!linattn_fits(l.d[i], a) || a.n_limbs > 65535) return k.bad("too many results for one call");
  }
  if (int e = check_dev(c)) return e;
  for (const DevCtx& dc : l) launch_linattn(dc, a, (hipStream_t)s);
  stat(ST_LINATTN, (u64)a.n_heads * a.M * a.Nn, polys * 8ull * c->hp.N * k.n_limbs);
  return post_launch();
}

int acehip_linattn_scores(acehip_ctx* c, const acehip_mat* p3, const acehip_mat* q, const acehip_mat* key, uint32_t n_heads, uint32_t n_kv_heads, uint32_t n_q,
                          uint32_t n_k, uint32_t dim, int causal, uint32_t level, uint32_t pos0, uint32_t n_limbs, acehip_stream s) {
  const Call k{c, "acehip_linattn_scores", level, pos0, n_limbs};
  if (int e = k.range()) return e;
  if (int e = check_heads(k, n_heads, n_kv_heads, n_q, n_k, dim)) return e;
  View y, vq, vk;
  if (int e = k.view(y, p3, n_heads, n_q, n_k, 3)) return e;
  if (y.empty()) return check_dev(c);
  if (int e = k.view(vq, q, n_heads, n_q, dim, 2)) return e;
  if (int e = k.view(vk, key, n_kv_heads, n_k, dim, 2)) return e;
  if (int e = check_result(k, y)) return e;
  if (int e = check_apart(k, y, vq)) return e;
  if (int e = check_apart(k, y, vk)) return e;
  LinattnArgs a;
  a.n_heads = n_heads, a.M = n_q, a.Nn = n_k;
  a.t1.K = dim;
  a.t1.a = vq.m;
  a.t1.b = CtMat{vk.m.d, vk.m.head, vk.m.col, vk.m.row, vk.m.comp};  // transposed: the sum runs over the features
  a.t1.b_group = n_heads / n_kv_heads;
  a.off = (int32_t)((int64_t)n_k - n_q);
  a.skip_above = causal != 0;
  return run_linattn(k, a, y, 2ull * dim * ((u64)n_heads * n_q + (u64)n_kv_heads * n_k) + 3ull * n_heads * seen(n_q, n_k, causal), s);
}

int acehip_linattn_out(acehip_ctx* c, const acehip_mat* o3, const acehip_mat* q, const acehip_mat* state, const acehip_mat* p, const acehip_mat* v,
                       uint32_t n_heads, uint32_t n_kv_heads, uint32_t n_q, uint32_t n_k, uint32_t dim_k, uint32_t dim_v, const int64_t* d_in,
                       const int64_t* d_decay, int causal, uint32_t level, uint32_t pos0, uint32_t n_limbs, acehip_stream s) {
  const Call k{c, "acehip_linattn_out", level, pos0, n_limbs};
  if (int e = k.range()) return e;
  if (int e = check_heads(k, n_heads, n_kv_heads, n_q, n_k, dim_k)) return e;
  if (!p != !v) return k.bad("scores and values come together");
  if (!q != !state) return k.bad("queries and state come together");
  View y, vq, vs, vp, vv;
  if (int e = k.view(y, o3, n_heads, n_q, dim_v, 3)) return e;
  if (y.empty()) return check_dev(c);
  if (int e = check_result(k, y)) return e;
  LinattnArgs a;
  a.n_heads = n_heads, a.M = n_q, a.Nn = dim_v;
  u64 polys = 3ull * n_heads * n_q * dim_v;
  if (state && dim_k) {
    if (int e = k.view(vq, q, n_heads, n_q, dim_k, 2)) return e;
    if (int e = k.view(vs, state, n_heads, dim_k, dim_v, 2)) return e;
    if (int e = check_apart(k, y, vq)) return e;
    if (int e = check_apart(k, y, vs)) return e;
    if (int e = check_array(k, y, d_in, (i128)8 * n_heads * n_q, 8)) return e;
    a.t1.K = dim_k;
    a.t1.a = vq.m;
    a.t1.b = vs.m;
    a.scale = d_in;
    polys += 2ull * n_heads * dim_k * ((u64)n_q + dim_v);
  }
  if (p && n_k) {
    if (int e = k.view(vp, p, n_heads, n_q, n_k, 2)) return e;
    if (int e = k.view(vv, v, n_kv_heads, n_k, dim_v, 2)) return e;
    if (int e = check_apart(k, y, vp)) return e;
    if (int e = check_apart(k, y, vv)) return e;
    // distances of a causal call: 0 .. n_k - 1; without the mask a later key has none
    if (d_decay && !causal) return k.bad("decays by distance need the causal form");
    if (int e = check_array(k, y, d_decay, (i128)8 * n_heads * n_k, 8)) return e;
    a.t2.K = n_k;
    a.t2.a = vp.m;
    a.t2.b = vv.m;
    a.t2.b_group = n_heads / n_kv_heads;
    a.decay = d_decay;
    a.decay_ld = n_k;
    a.causal = causal != 0;
    a.off = (int32_t)((int64_t)n_k - n_q);
    polys += 2ull * n_heads * seen(n_q, n_k, causal) + 2ull * n_kv_heads * n_k * dim_v;
  }
  return run_linattn(k, a, y, polys, s);
}

int acehip_linattn_state(acehip_ctx* c, const acehip_mat* s3, const acehip_mat* state, const acehip_mat* key, const acehip_mat* v, uint32_t n_heads,
                         uint32_t n_kv_heads, uint32_t n_k, uint32_t dim_k, uint32_t dim_v, const int64_t* d_keep, const int64_t* d_decay, uint32_t level,
                         uint32_t pos0, uint32_t n_limbs, acehip_stream s) {
  const Call k{c, "acehip_linattn_state", level, pos0, n_limbs};
  if (int e = k.range()) return e;
  if (int e = check_heads(k, n_heads, n_kv_heads, 1, n_k, dim_k)) return e;
  View y, vs, vk, vv;
  if (int e = k.view(y, s3, n_heads, dim_k, dim_v, 3)) return e;
  if (y.empty()) return check_dev(c);
  if (int e = k.view(vk, key, n_kv_heads, n_k, dim_k, 2)) return e;
  if (int e = k.view(vv, v, n_kv_heads, n_k, dim_v, 2)) return e;
  if (int e = check_result(k, y)) return e;
  if (int e = check_apart(k, y, vk)) return e;
  if (int e = check_apart(k, y, vv)) return e;
  LinattnArgs a;
  a.n_heads = n_heads, a.M = dim_k, a.Nn = dim_v;
  u64 polys = 3ull * n_heads * dim_k * dim_v + 2ull * n_kv_heads * n_k * ((u64)dim_k + dim_v);
  if (state) {
    if (int e = k.view(vs, state, n_heads, dim_k, dim_v, 2)) return e;
    // in place: polynomials 0 and 1 of the new state over those of the old one, each word read and written by the same lane
    const bool same = vs.m.d == y.m.d && vs.m.head == y.m.head && vs.m.row == y.m.row && vs.m.col == y.m.col && vs.m.comp == y.m.comp;
    if (!same)
      if (int e = check_apart(k, y, vs)) return e;
    if (int e = check_array(k, y, d_keep, (i128)8 * n_heads, 8)) return e;
    a.base = vs.m;
    a.keep = d_keep;
    polys += 2ull * n_heads * dim_k * dim_v;
  }
  if (n_k) {
    if (int e = check_array(k, y, d_decay, (i128)8 * n_heads * n_k, 8)) return e;
    a.t2.K = n_k;
    a.t2.a = CtMat{vk.m.d, vk.m.head, vk.m.col, vk.m.row, vk.m.comp};  // transposed: the sum runs over the tokens
    a.t2.b = vv.m;
    a.t2.a_group = a.t2.b_group = n_heads / n_kv_heads;
    a.decay = d_decay;
    a.decay_ld = n_k;
    a.decay_by_k = 1;
  }
  return run_linattn(k, a, y, polys, s);
}

}  // extern "C"
