// attn_mod.hip — attention with modified scores for gfx950: forward, backward, and the short-query form split over the keys.
//
//   t_ij = cap * tanh(scale q_i . k_j / cap)   (or scale q_i . k_j)   - slope_h |j - i'| + table_h[clip(j - i', -R, R)]
//   o_i  = sum_j softmax_j(t_ij) v_j   over the keys that query i may see;  zeros where it may see none
// i' = i + (len - Sq): the queries are the last Sq positions of the len = kv_len[b] keys.  A query sees key j iff j < bound_i and their
// documents agree; bound_i = len, or min(len, max(i' + 1, prefix_i)) for a causal mask: every mask that depends on positions is ONE
// integer per query, compared once per score and only in tiles that cross it.
//
// Layout.  Lane = query in the forward and dQ kernels (S^T = K Q^T: the row maximum and sum stay in the lane, one exchange between the
// two halves of a wave), lane = key in the dK / dV kernel.  P^T (dS^T) goes from the accumulator registers into the next product
// as its B operand; the transposed operand comes from the staged LDS tile through ds_read_b64_tr_b16, with the accumulators' row order
// applied to both.  64-row tiles of the streamed pair (K|V, or Q|dO) are staged once per workgroup, double-buffered; see
// Stage for how their rows lie.
// Grouped heads: the gp query heads that share a K/V head are packed into the row index (row r = query r / gp, head r % gp), so K and V
// are read once for all of them; with a table each head is a unit of its own (gp = 1: the table of one head lives in LDS).
// Statistics, the running maximum and sum, lse, delta and all accumulators are fp32; P and dS are rounded to the input type for the
// matrix cores (one rounding of a factor in [0, 1], and of a gradient, the same size as the output's own rounding).  delta_i = dO_i . O_i
// wants more of O than its type holds: an error of delta stands in every dS of the row and does not average out.  A forward pass that is
// to be differentiated stores what O's rounding left behind too (o_rest), in the same type.
#include <type_traits>

#include "common.h"

namespace {

constexpr int TILE = 64;                        // staged rows
constexpr float LOG2E = 1.44269504088896341f;
constexpr float LOWEST = -3.0e38f;              // running maximum before the first visible key: finite, below every score
constexpr float FAREST = 2.9e38f;               // finite table entries in base-2 units are held inside +-FAREST, above LOWEST
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2_t;
typedef __attribute__((ext_vector_type(4))) unsigned u32x4;

__device__ __attribute__((aligned(16))) const unsigned zero_chunk[4] = {0, 0, 0, 0};

template <typename T>
struct El;
template <>
struct El<bf16_t> {
  static __device__ __forceinline__ f32x16 mfma(const bf16x8& a, const bf16x8& b, const f32x16& c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ unsigned pack2(float a, float b) { return pack2bf(a, b); }
  static __device__ __forceinline__ float add2(unsigned ab, float c) {    // a + b + c in fp32, one instruction
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, ab), __builtin_bit_cast(bf16x2_t, 0x3f803f80u), c, false);
  }
  static __device__ __forceinline__ float up(short v) { return bf2f((unsigned short)v); }
};
template <>
struct El<_Float16> {
  static __device__ __forceinline__ f32x16 mfma(const bf16x8& a, const bf16x8& b, const f32x16& c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ unsigned pack2(float a, float b) {
    const t2v_f32x2 v = {a, b};
    return __builtin_bit_cast(unsigned, __builtin_convertvector(v, f16x2));
  }
  static __device__ __forceinline__ float add2(unsigned ab, float c) {
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, ab), __builtin_bit_cast(f16x2, 0x3c003c00u), c, false);
  }
  static __device__ __forceinline__ float up(short v) { return (float)__builtin_bit_cast(_Float16, v); }
};
template <typename T>
__device__ __forceinline__ bf16x8 pack8(const f32x16& v, int kk) {
  const u32x4 q = {El<T>::pack2(v[8 * kk], v[8 * kk + 1]), El<T>::pack2(v[8 * kk + 2], v[8 * kk + 3]),
                   El<T>::pack2(v[8 * kk + 4], v[8 * kk + 5]), El<T>::pack2(v[8 * kk + 6], v[8 * kk + 7])};
  return __builtin_bit_cast(bf16x8, q);
}

// accumulator register r of lane half hi holds row crow(r, hi) of the 32 x 32 tile
__device__ __forceinline__ constexpr int crow(int r, int hi) { return (r & 3) + 8 * (r >> 2) + 4 * hi; }
// maximum / sum of the two halves' values of a lane pair (l, l + 32), in both (v_permlane32_swap: no trip through LDS)
__device__ __forceinline__ float half_max(float v) {
  const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1]));
}
__device__ __forceinline__ float half_sum(float v) {
  const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(x[0]) + __uint_as_float(x[1]);
}

struct QMeta {      // of 64 rows: smallest and largest bound, smallest and largest document >= 0, whether some row has none
  int bmin, bmax, dmin, dmax, neg;
};
struct KMeta {
  int dmin, dmax, neg;
};
// A tile's entry through the scalar cache: the index is the same in all lanes, and a vector load that is waited for would wait for the next
// tile's copies too, which were issued in front of it (the counter is in order)
template <typename M>
__device__ __forceinline__ M tile_entry(const M* table, int t) {
  const __attribute__((address_space(4))) int* p = (const __attribute__((address_space(4))) int*)(table + __builtin_amdgcn_readfirstlane(t));
  M m;
#pragma unroll
  for (int i = 0; i < (int)(sizeof(M) / 4); ++i) ((int*)&m)[i] = p[i];
  return m;
}

struct Args {
  T2VAttnMod p;
  int gp, nunit, M;                 // heads per unit, units per batch, rows per unit (Sq * gp)
  unsigned magic;                   // r / gp = r * magic >> 32 (gp > 1)
  int ntile, splits;                // row (or key) tiles of a unit, splits of the other axis
  int chunk, wgs;                   // dK / dV: row tiles a split is meant to take, workgroups of a K / V head (see kv_runs)
  int fold;                         // where the order of the row tiles turns (see row_tile)
  const int* qorder;                // [nbatch * row tiles], [nbatch * key tiles]: (batch, tile) pairs by falling work, or NULL
  const int* korder;
  int to_part;                      // dK / dV go to `part` as fp32 (several splits, or several batches that share K / V)
  const QMeta* qmeta;               // [nbatch][ceil(M / 64)] or NULL
  const KMeta* kmeta;               // [nbatch][ceil(Sk / 64)] or NULL
  float* lsum;                      // second plane of lse (slopes or a bias), or NULL
  float* part;                      // partial results of the splits
  float* part_ml;
  float* part_bias;                 // [nbatch * ntile (* parts)][heads][2R + 1]
};

__device__ __forceinline__ long long op_base(const T2VAttnOperand& o, int b) {
  return (long long)(b / o.bdiv) * o.bstride_hi + (long long)(b % o.bdiv) * o.bstride_lo;
}
__device__ __forceinline__ int div_gp(const Args& a, int r) { return a.gp == 1 ? r : (int)__umulhi((unsigned)r, a.magic); }
// what a workgroup knows of its sequence
struct Seq {
  int b, len, off, prefix;          // off = len - Sq: the first query's place among the keys; prefix of the whole sequence
  const int* per_query;             // or one per query
  bool causal;
};
__device__ __forceinline__ Seq load_seq(const Args& a, int b) {
  Seq s;
  s.b = b;
  s.len = a.p.kv_len ? max(0, min(a.p.kv_len[b], a.p.Sk)) : a.p.Sk;
  s.off = s.len - a.p.Sq;
  s.causal = a.p.causal != 0;
  s.per_query = s.causal && a.p.prefix && a.p.prefix_per_query ? a.p.prefix + (long long)b * a.p.Sq : nullptr;
  s.prefix = s.causal && a.p.prefix && !a.p.prefix_per_query ? a.p.prefix[b] : 0;
  return s;
}
// keys [0, bound) are candidates of query i
__device__ __forceinline__ int bound_of(const Seq& s, int i, int prefix) {
  return s.causal ? max(0, min(max(i + s.off + 1, prefix), s.len)) : s.len;
}
__device__ __forceinline__ int row_bound(const Seq& s, int i) { return bound_of(s, i, s.per_query ? s.per_query[i] : s.prefix); }

// the first of a unit's row tiles that may see key wk0 or a later one (0 where the meta table tells it tile by tile)
__device__ __forceinline__ int first_tile(const Args& a, const Seq& s, int wk0) {
  return a.qmeta || !s.causal || s.prefix > wk0 ? 0 : min((a.M + TILE - 1) / TILE, max(0, wk0 - s.off) * a.gp / TILE);
}

// dK / dV: how many workgroups share the rows of key tile k.  It is fixed by sizes alone (a causal mask, no prefix, whole lengths), so that the
// grid has no workgroup without work where those hold: 43 % of idle ones put the busy ones unevenly on the shader engines, and the
// launch took two rounds where one was enough (193 -> 128 us).  What the mask really leaves is divided evenly among them.
__host__ __device__ __forceinline__ int kv_runs(const Args& a, int k, int keys, int tiles) {
  if (a.chunk >= tiles) return 1;
  const long long first = a.p.causal && !a.qmeta ? ((long long)k * keys - (a.p.Sk - a.p.Sq)) * a.gp / TILE : 0;
  const int run = tiles - (int)(first > 0 ? first : 0) * (a.p.heads / a.p.kv_heads / a.gp);
  return run > a.chunk ? (run + a.chunk - 1) / a.chunk : 1;
}
// forward, dQ: the row tile of rank r.  Under a causal mask the last tiles are the longest: they come first (they then end first come, first
// served).  Where all workgroups are resident at once, two on some CUs, the order turns at rank `fold`, behind the first workgroup of every CU:
// the second of a CU is then short where the first is long (264 workgroups over 2112 keys: 56 us where it turned in the middle, 53 at fold).
__device__ __forceinline__ int row_tile(const Args& a, int r) {
  return r >= a.fold ? r - a.fold : a.ntile - 1 - r;
}

// workgroup id -> (batch, unit): workgroups go round-robin over the eight XCDs, so units that share a K/V head are placed a multiple of
// nbatch * kv_heads apart, which is the same XCD (and L2) where that is a multiple of eight
struct Unit {
  int b, kv, h0, x;                 // x: number of the unit, as unit_of counts them
};
__device__ __forceinline__ Unit unit_of(const Args& a, int x) {
  const int kvb = a.p.nbatch * a.p.kv_heads, gu = x / kvb, y = x - gu * kvb;
  Unit u;
  u.b = y / a.p.kv_heads;
  u.kv = y - u.b * a.p.kv_heads;
  u.h0 = u.kv * (a.p.heads / a.p.kv_heads) + gu * a.gp;
  u.x = x;
  return u;
}
// Which rows (keys) of a tile are a workgroup's own: all of them, or those of its entry (see attn_mod_order_kernel)
struct Part {
  int first, part;                  // part 0: documents <= first, and rows that see nothing, 1: documents > first, -1: all
  bool none;                        // an entry without rows
  __device__ __forceinline__ bool owns(int doc) const { return part < 0 || (doc > first) == (part == 1); }
};
template <typename M>
__device__ __forceinline__ Part part_of(const M* table, int t, int per, int n, int part) {
  int lo = 0x7fffffff, hi = -1;
  for (int i = t * per; i < min((t + 1) * per, n); ++i) {
    const M m = tile_entry(table, i);
    lo = min(lo, m.dmin);
    hi = max(hi, m.dmax);
  }
  return Part{lo, part, part == 1 && hi <= lo};
}
// the unit, row tile and part of workgroup `id` (of one split)
__device__ __forceinline__ Unit work_of(const Args& a, int id, int& tile, Part& part) {
  if (a.qorder) {
    const int e = a.qorder[id / a.nunit], v = id % a.nunit, b = (e >> 1) / a.ntile, gus = a.nunit / a.p.kv_heads, nqt = (a.M + TILE - 1) / TILE;
    tile = (e >> 1) - b * a.ntile;
    part = part_of(a.qmeta + (long long)b * nqt, tile, 2, nqt, e & 1);
    return unit_of(a, (v % gus) * a.p.nbatch * a.p.kv_heads + b * a.p.kv_heads + v / gus);
  }
  const int NU = a.p.nbatch * a.nunit;
  tile = row_tile(a, id / NU);
  part = Part{0, -1, false};
  return unit_of(a, id % NU);
}

// ------------------------------------------------------------------------------------------------ staging
// Two 64-row tiles (A | B) of 2 DP bytes a row, double-buffered.  They go from memory to LDS without passing registers: 16 bytes per lane,
// and a wave's instruction fills 1 KB of consecutive LDS addresses, a GROUP.  A group holds the rows of a 32-row block (DP = 128; of the
// tile: DP = 64) with one row & 7, and groups lie 1056 bytes apart: eight lanes that read eight consecutive rows (ds_read_b128), and the
// eight rows of a transposed read, start 32 bytes apart modulo the banks.  Every fragment is a lane's constant address plus an
// immediate: an XOR swizzle needed a register per fragment and stage (136 spills in dQ), row padding cannot be had with these loads.
constexpr int GROUP = 512 + 16;                 // elements
template <int DP>
struct __attribute__((aligned(16))) Stage {
  bf16_t a[TILE * DP / 512 * GROUP];
  bf16_t b[TILE * DP / 512 * GROUP];
};
template <int DP>
__device__ __forceinline__ constexpr int row_off(int row) {
  return DP == 128 ? ((row >> 5) * 8 + (row & 7)) * GROUP + ((row >> 3) & 3) * 128 : (row & 7) * GROUP + (row >> 3) * 64;
}

// What a lane loads: instruction i of a wave fills group NW i + wave.  Columns behind the head dim come from a chunk of zeros (row stride 0).
template <int DP, int NW>
struct Lane {
  static constexpr int NI = TILE * DP / 512 / NW;                       // instructions per wave
  int wave, sub, ch;
  bool ok;
  __device__ __forceinline__ Lane(int w, int lane, int D) {
    wave = w;
    sub = 8 * (lane / (DP / 8));
    ch = lane % (DP / 8);
    ok = ch * 8 < D;
  }
  __device__ __forceinline__ int row_of(int i) const {
    const int g = NW * i + wave;
    return (DP == 128 ? 32 * (g >> 3) + (g & 7) : g) + sub;
  }
  __device__ __forceinline__ int group(int i) const { return (NW * i + wave) * GROUP; }
};
__device__ __forceinline__ void copy16(const void* src, void* lds) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src, (__attribute__((address_space(3))) void*)lds, 16, 0, 0);
}
// (the builtin and not inline asm: the compiler then knows that nothing is in flight behind it, and does not wait again, for the next tile's
// copies, at the first use of what was loaded in front of the loop)
__device__ __forceinline__ void copies_done() { __builtin_amdgcn_s_waitcnt(0x0f70); }      // vmcnt(0)
// zero the staged rows for which `dead(row)`: rows that nobody sees may hold inf / NaN, which must not meet a zero weight
template <int DP, int NT, bool BOTH, typename F>
__device__ __forceinline__ void clear_rows(Stage<DP>& st, int tid, F dead) {
  const bf16x8 z = {0, 0, 0, 0, 0, 0, 0, 0};
  for (int i = tid; i < TILE * DP / 8; i += NT) {
    const int row = i / (DP / 8), o = row_off<DP>(row) + (i % (DP / 8)) * 8;
    if (dead(row)) {
      if (BOTH) *(bf16x8*)(st.a + o) = z;
      *(bf16x8*)(st.b + o) = z;
    }
  }
}

// lane's part of the address of a row fragment (32 staged rows as an MFMA operand: row = lane & 31, k = the 16 columns of step kd) and of a
// transposed fragment (rows = columns [32 fm, 32 fm + 32), k = the 16 staged rows of step kk in the accumulators' order)
template <int DP>
__device__ __forceinline__ int lane_row(int lane) { return row_off<DP>(lane & 31) + 8 * (lane >> 5); }
template <int DP>
__device__ __forceinline__ int lane_tr(int lane) {
  const int gq = lane >> 4, li = lane & 15;
  return row_off<DP>(4 * (gq >> 1) + (li >> 2)) + 16 * (gq & 1) + 4 * (li & 3);
}
template <int DP>
__device__ __forceinline__ bf16x8 rowfrag(const bf16_t* s, int blk, int kd) {
  return *(const bf16x8*)(s + row_off<DP>(32 * blk) + 16 * kd);
}
template <int DP>
__device__ __forceinline__ bf16x8 trfrag(const bf16_t* s, int blk, int fm, int kk) {
  const bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_bf16x4*)(s + row_off<DP>(32 * blk + 16 * kk) + 32 * fm));
  const bf16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_bf16x4*)(s + row_off<DP>(32 * blk + 16 * kk + 8) + 32 * fm));
  return bf16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
}

// 32 FM columns of the lane's row from the accumulators, times mul, 16 bytes per store: the halves of a wave hold columns 4 hi .. 4 hi + 3 of
// every eight and exchange them first (v_permlane32_swap), so that the lower half stores eight columns and the upper the next eight.
// To `rest`, where there is one, goes what the rounding to T left behind
template <typename T, int FM>
__device__ __forceinline__ void store_row(bf16_t* row, const f32x16 (&v)[FM], float mul, int hi, int D, bool ok, bf16_t* rest = nullptr) {
  const auto store = [&](bf16_t* to, const unsigned (&w)[4], int f, int h) {
    const auto x = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false);
    const auto y = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
    const int col = 32 * f + 16 * h + 8 * hi;
    if (ok && col < D) *(u32x4*)(to + col) = u32x4{x[0], y[0], x[1], y[1]};
  };
#pragma unroll
  for (int f = 0; f < FM; ++f)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      unsigned w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = El<T>::pack2(v[f][8 * h + 2 * e] * mul, v[f][8 * h + 2 * e + 1] * mul);
      store(row, w, f, h);
      if (rest) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          w[e] = El<T>::pack2(fmaf(v[f][8 * h + 2 * e], mul, -El<T>::up((short)(w[e] & 0xffffu))),
                              fmaf(v[f][8 * h + 2 * e + 1], mul, -El<T>::up((short)(w[e] >> 16))));
        store(rest, w, f, h);
      }
    }
}
// the accumulators as they are, a wave's registers one after the other (1 KB per instruction): partial sums of the splits
template <int FM>
__device__ __forceinline__ void store_part(float* wave_part, const f32x16 (&v)[FM], int lane, bool ok) {
#pragma unroll
  for (int f = 0; f < FM; ++f)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      if (ok) *(float4*)(wave_part + ((f * 4 + g) * 64 + lane) * 4) = float4{v[f][4 * g], v[f][4 * g + 1], v[f][4 * g + 2], v[f][4 * g + 3]};
}

__device__ __forceinline__ const bf16x8* chunk_ptr(const bf16_t* p, bool ok) { return ok ? (const bf16x8*)p : (const bf16x8*)zero_chunk; }

// ------------------------------------------------------------------------------------------------ scores
// t (in base-2 exponent units) of one lane's 16 scores.  `d0`: distance j - i' of accumulator row 0 (of the lane's half)
struct Mod {
  float c;            // scale * log2e
  float k1, capl;     // cap: 2 log2e scale / cap, cap * log2e
  float k;            // cap: scale / cap
  bool slope, table;
  int R;
};
__device__ __forceinline__ Mod make_mod(const Args& a) {
  Mod m;
  const bool cap = a.p.softcap > 0.f;
  m.slope = a.p.slopes != nullptr;
  m.table = a.p.bias != nullptr;
  m.c = a.p.scale * LOG2E;
  m.k1 = cap ? 2.f * LOG2E * a.p.scale / a.p.softcap : 0.f;
  m.k = cap ? a.p.scale / a.p.softcap : 0.f;
  m.capl = a.p.softcap * LOG2E;
  m.R = a.p.radius;
  return m;
}
// cap * tanh(x / cap) = cap (1 - 2 / (1 + e^(2 x / cap))): one exp, one reciprocal; exact at +-inf.  Returns it in base-2 units and
// leaves w = 1 / (1 + e^(..)): the derivative is 4 w (1 - w).
// The difference cancels: it is good to 4e-7 of the cap, 4e-5 at a cap of 100, where it costs nothing beside the weights' own rounding.  A larger cap
// (WIDE, kernels of their own: nothing is added to those of ordinary caps) takes the odd series x (1 - y^2 / 3 + 2 y^4 / 15 - ..), y = x / cap, where
// |y| < 1/4; its first term left out is 9e-9 there, and the exponential's error is 2e-6 of the score above.  (2 x 2011 rows, forward and backward: 16 / 4
// heads of 128 303 -> 355 us, 16 heads of 64 299 -> 406 us.)
constexpr float WIDE_CAP = 100.f;
template <bool WIDE>
__device__ __forceinline__ float capped(const Mod& m, float s, float& w) {
  w = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(s * m.k1));
  float t = fmaf(w, -2.f * m.capl, m.capl);
  if (WIDE) {
    const float y = s * m.k, z = y * y;
    const float p = fmaf(z, fmaf(z, fmaf(z, fmaf(z, 62.f / 2835, -17.f / 315), 2.f / 15), -1.f / 3), 1.f);
    t = z < 0.0625f ? s * m.c * p : t;
  }
  return t;
}

// table of head h in base-2 units in LDS; an entry at or below the type's lowest finite value hides its distance (-inf)
template <typename T>
__device__ __forceinline__ void load_table(const Args& a, int h, float* tab, int tid, int nt) {
  const int n = 2 * a.p.radius + 1;
  const auto units = [](float v) {                                      // (NaN stays NaN)
    const float w = v * LOG2E;
    return w < -FAREST ? -FAREST : w > FAREST && v < INFINITY ? FAREST : w;
  };
  for (int i = tid; i < n; i += nt) {
    const long long at = (long long)h * n + i;
    float v;
    if (a.p.bias_f32) {
      v = ((const float*)a.p.bias)[at];
      v = v <= -3.4028234e38f ? -INFINITY : units(v);
    } else {
      v = El<T>::up(((const short*)a.p.bias)[at]);
      v = v <= (std::is_same<T, bf16_t>::value ? -3.3895313e38f : -65504.f) ? -INFINITY : units(v);
    }
    tab[i] = v;
  }
}

// The tiles in [t, end) that may matter, in order: `active` is evaluated for 64 tiles at once, one per lane, and kept as a mask; without
// `filter` every tile counts.  All waves of a workgroup walk the same tiles.
struct TileIter {
  unsigned long long m;
  int base, end;
  bool filter;
};
template <typename F>
__device__ __forceinline__ int tile_next(TileIter& it, F active) {
  if (!it.filter) return it.base < it.end ? it.base++ : it.end;
  while (it.m == 0) {
    if (it.base >= it.end) return it.end;
    const int c = it.base + (int)(threadIdx.x & 63);
    it.m = __ballot(c < it.end && active(min(c, it.end - 1)));
    it.base += 64;
  }
  const int t = it.base - 64 + __builtin_ctzll(it.m);
  it.m &= it.m - 1;
  return t;
}

// The tiles [tbeg, tend) of split sp of [0, nt): equal numbers of those that count.  (Equal ranges of packed documents are mostly empty: 1839 tokens in
// seven documents, 8 heads of 80, four splits: 42 us, so 34, unsplit 31; but the one document of a step over 4000 keys: 69 us unsplit, 17 split.)
template <typename F>
__device__ __forceinline__ void split_tiles(int nt, int splits, int sp, bool filter, F active, int& tbeg, int& tend) {
  if (!filter || splits == 1) {
    const int per = (nt + splits - 1) / splits;
    tbeg = min(nt, sp * per);
    tend = min(nt, tbeg + per);
    return;
  }
  const int lane = threadIdx.x & 63;
  int total = 0, seen = 0;
  for (int base = 0; base < nt; base += 64) total += __popcll(__ballot(base + lane < nt && active(min(base + lane, nt - 1))));
  const int per = (total + splits - 1) / splits, first = min(total, sp * per), last = first + per;
  tbeg = tend = nt;
  for (int base = 0; base < nt; base += 64) {
    const unsigned long long m = __ballot(base + lane < nt && active(min(base + lane, nt - 1)));
    const int n = __popcll(m), number = seen + __popcll(m & ((1ull << lane) - 1));       // of the lane's tile among those that count
    const unsigned long long b = __ballot((m >> lane & 1) && number == first), e = __ballot((m >> lane & 1) && number == last);
    if (b) tbeg = base + __builtin_ctzll(b);
    if (e) tend = base + __builtin_ctzll(e);
    seen += n;
  }
}

// minimum / maximum over the wave as a scalar
__device__ __forceinline__ int wave_min_i(int v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = min(v, __shfl_xor(v, o));
  return __builtin_amdgcn_readfirstlane(v);
}
__device__ __forceinline__ int wave_max_i(int v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = max(v, __shfl_xor(v, o));
  return __builtin_amdgcn_readfirstlane(v);
}

// What the backward pass forms a row's weights from: the base-2 log-sum-exp; with a distance bias the exponent of the row's largest weight and, in
// a second plane, the logarithm of the sum behind it.  Beside an entry of 1e9 that every key of a row carries, one fp32 number would lose the sum
// (all gradients too large by the number of keys), and 2^(s - m) / l does not.  +inf marks a row that saw nothing: every weight is then 0.
__device__ __forceinline__ void store_lse(const Args& a, long long at, float m2, float l) {
  const float ll = __builtin_amdgcn_logf(l);
  a.p.lse[at] = l > 0.f ? (a.lsum ? m2 : m2 + ll) : INFINITY;
  if (a.lsum) a.lsum[at] = l > 0.f ? ll : 0.f;
}

// What a wave knows about the 32 query rows of its lanes (lane & 31 = row of the block)
struct Rows {
  int r, i, h;                      // row in the unit, query, head
  bool ok;                          // the row exists
  int bound, pos, doc;              // bound 0: sees nothing
  float slope;                      // in base-2 units
  int bmin, bmax, dmin, dmax, pmin; // over the wave
  bool neg;
};
__device__ __forceinline__ void load_rows(Rows& R, const Args& a, const Unit& u, const Seq& sq, const Part& part, int r0, int lane) {
  int lo = 0x7fffffff, hi = 0, dlo = 0x7fffffff, dhi = -1, ng = 0;
  R.r = r0 + (lane & 31);
  R.ok = R.r < a.M;
  const int rc = min(R.r, a.M - 1);
  R.i = div_gp(a, rc);
  R.h = u.h0 + rc - R.i * a.gp;
  R.doc = a.p.q_docs ? a.p.q_docs[(long long)u.b * a.p.Sq + R.i] : 0;
  R.bound = R.ok && R.doc >= 0 ? row_bound(sq, R.i) : 0;
  // (The tiles' entries hold the documents of rows that see something, and by them a second part may be empty: a row that sees nothing is of
  // the first part, whatever its document.)
  R.ok = R.ok && part.owns(R.bound > 0 ? R.doc : -1);
  if (!R.ok) R.bound = 0;
  R.pos = R.i + sq.off;
  R.slope = a.p.slopes ? a.p.slopes[R.h] * LOG2E : 0.f;
  if (R.ok) lo = min(lo, R.bound);
  hi = max(hi, R.bound);
  if (R.bound > 0) {
    dlo = min(dlo, R.doc);
    dhi = max(dhi, R.doc);
  } else if (R.ok) {
    ng = 1;
  }
  R.bmin = wave_min_i(lo);
  R.pmin = __builtin_amdgcn_readfirstlane(div_gp(a, min(r0, a.M - 1)) + sq.off);      // rows are in the queries' order
  R.bmax = wave_max_i(hi);
  R.dmin = wave_min_i(dlo);
  R.dmax = wave_max_i(dhi);
  R.neg = wave_max_i(ng) != 0;
}

// ------------------------------------------------------------------------------------------------ forward
// MOD: bit 0 cap, bit 1 distance bias (slopes / table), bit 2 a cap above WIDE_CAP, compile-time so that a tile is straight-line code.
// A workgroup is 128 rows (four waves of 32) and walks the key tiles its rows may see.  64 rows a wave instead (K and V fragments read once for
// both halves) leave one wave per SIMD: 656 -> 801 us at head dim 128, no change at 64.
// Measured, bf16, 8192 x 8192, 16 heads, first launch to sustained load: head dim 128 580 to 700 us, 785 to 950 TFLOP/s where a library product of
// 8192^3 reaches 1243 (causal 310 to 340, capped 790 to 890 us); head dim 64 362 to 423 us, 650 to 760 TFLOP/s.  At 128, causal with slopes, the matrix cores
// are busy for 0.38 of the time and vector instructions for about 0.58 (four cycles each, sixteen for an exponential): together the whole launch, so
// that what bounds it is that the two waves of a SIMD do both at the same times.  At 64 a score's exponential, maximum, sum and conversion take
// longer than its columns in the two products.  Without the tile copies it would be 10 % faster at most.
// One new token for 8 sequences of up to 16384 keys (165 MB of them), 16 / 4 heads of 128: 38 us, 4.4 TB/s, and 6 us for the join.
// Registers: no vectors spill but 4 at <64, 0>, held to three waves per SIMD, 4 at <128, 3>, and 13 / 16 at <128, 5 / 7>.
template <typename T, int DP, int MOD>
__global__ __launch_bounds__(256, DP == 64 && MOD < 2 ? 3 : 2) void attn_mod_fwd_kernel(const Args a) {
  warm_kernargs<(int)sizeof(Args)>();
  constexpr int NT = 256, KD = DP / 16, FM = DP / 32;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  Stage<DP>* st = (Stage<DP>*)smem;
  int* sdoc = (int*)(smem + 2 * sizeof(Stage<DP>));                     // [2][TILE]
  int* swg = sdoc + 2 * TILE;                                           // [4 waves][4]
  float* tab = (float*)(swg + 16);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), hi = lane >> 5;
  const int NU = a.p.nbatch * a.nunit;
  const int sp = blockIdx.x / NU % a.splits;
  int tile;
  Part part;
  const Unit u = work_of(a, blockIdx.x / (NU * a.splits) * NU + blockIdx.x % NU, tile, part);
  if (part.none) return;                                                // workgroup-uniform
  const Seq seq = load_seq(a, u.b);
  const int len = seq.len, D = a.p.D, Sk = a.p.Sk;
  const bf16_t* Q = (const bf16_t*)a.p.q.ptr + op_base(a.p.q, u.b);
  const bool docs = a.kmeta && a.p.kv_docs;
  const int* kdoc = docs ? a.p.kv_docs + (long long)u.b * Sk : nullptr;
  const Mod mod = make_mod(a);

  Rows R;
  load_rows(R, a, u, seq, part, (tile * 4 + wave) * 32, lane);
  bf16x8 qf[KD];
  const bf16_t* qp = Q + (long long)R.i * a.p.q.sstride + (long long)R.h * D;
#pragma unroll
  for (int kd = 0; kd < KD; ++kd) qf[kd] = *chunk_ptr(qp + 16 * kd + 8 * hi, R.bound > 0 && 16 * kd + 8 * hi < D);
  if ((MOD & 2) && mod.table) load_table<T>(a, u.h0, tab, tid, NT);
  if (lane == 0) {
    swg[wave * 4] = R.bmax;
    swg[wave * 4 + 1] = R.dmin;
    swg[wave * 4 + 2] = R.dmax;
  }
  __syncthreads();
  int bmax = 0, dmin = 0x7fffffff, dmax = -1;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    bmax = max(bmax, swg[w * 4]);
    dmin = min(dmin, swg[w * 4 + 1]);
    dmax = max(dmax, swg[w * 4 + 2]);
  }
  bmax = __builtin_amdgcn_readfirstlane(bmax);
  const KMeta* km = docs ? a.kmeta + (long long)u.b * ((Sk + TILE - 1) / TILE) : nullptr;
  auto active = [&](int c) { return km[c].dmax >= dmin && km[c].dmin <= dmax; };
  int tbeg, tend;
  split_tiles((bmax + TILE - 1) / TILE, a.splits, sp, docs, active, tbeg, tend);
  TileIter it = {0ull, tbeg, tend, docs};
  const Lane<DP, 4> ln(wave, lane, D);
  const int lrow = lane_row<DP>(lane), ltr = lane_tr<DP>(lane);
  const bf16_t* kp = ln.ok ? (const bf16_t*)a.p.k.ptr + op_base(a.p.k, u.b) + (long long)u.kv * D + ln.ch * 8 : (const bf16_t*)zero_chunk;
  const bf16_t* vp = ln.ok ? (const bf16_t*)a.p.v.ptr + op_base(a.p.v, u.b) + (long long)u.kv * D + ln.ch * 8 : (const bf16_t*)zero_chunk;
  const unsigned ks = ln.ok ? (unsigned)a.p.k.sstride : 0u, vs = ln.ok ? (unsigned)a.p.v.sstride : 0u;
  // Iteration n works on tile n: its scores were formed in iteration n - 1, so that the matrix products of tile n + 1's scores run under the
  // exponentials of tile n in the same wave.  K is fetched two tiles ahead and V one: stage halves n & 1 hold K(n + 2) and V(n).
  int nd = 0;
  auto fetch_k = [&](int t, int sidx) {                                 // rows behind the last key repeat it (masked by the bounds)
#pragma unroll
    for (int i = 0; i < Lane<DP, 4>::NI; ++i)
      copy16(kp + (unsigned long long)(unsigned)min(t * TILE + ln.row_of(i), len - 1) * ks, st[sidx].a + ln.group(i));
  };
  auto fetch_v = [&](int t, int sidx) {
#pragma unroll
    for (int i = 0; i < Lane<DP, 4>::NI; ++i)
      copy16(vp + (unsigned long long)(unsigned)min(t * TILE + ln.row_of(i), len - 1) * vs, st[sidx].b + ln.group(i));
    if (docs && tid < TILE) nd = kdoc[min(t * TILE + tid, len - 1)];
  };
  auto landed = [&](int t, int sidx, int neg) {                         // what was fetched is there for all waves; V (and documents) in stage sidx
    if (docs && tid < TILE) sdoc[sidx * TILE + tid] = t * TILE + tid < len ? nd : -1;
    copies_done();
    __syncthreads();
    if (neg) {                                                          // (K may hold what it likes there: its scores are masked by selects)
      clear_rows<DP, NT, false>(st[sidx], tid, [&](int r) { return sdoc[sidx * TILE + r] < 0; });
      __syncthreads();
    }
  };

  const float defer = a.p.o_rest ? 0.f : 6.f;
  float m = LOWEST, l = 0.f;
  f32x16 o[FM], s[2];
#pragma unroll
  for (int f = 0; f < FM; ++f)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[f][r] = 0.f;
  auto scores = [&](f32x16 (&x)[2], const bf16_t* sk) {                 // K Q^T of a tile
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
#pragma unroll
      for (int r = 0; r < 16; ++r) x[kb][r] = 0.f;
#pragma unroll
      for (int kd = 0; kd < KD; ++kd) {
        const bf16x8 kf = rowfrag<DP>(sk + lrow, kb, kd);
        x[kb] = El<T>::mfma(kf, qf[kd], x[kb]);
      }
    }
  };
  int t = tile_next(it, active), t1 = tend, cur = 0;
  KMeta kn = {0, 0, 0}, k1 = {0, 0, 0};                                 // of the tile at hand and the next (documents)
  if (t < tend) {
    t1 = tile_next(it, active);
    if (docs) kn = tile_entry(km, t);
    fetch_k(t, 0);
    fetch_v(t, 0);
    if (t1 < tend) fetch_k(t1, 1);
    landed(t, 0, kn.neg);
    scores(s, st[0].a);
    __syncthreads();                                                    // all waves have read K of stage 0
  }
  while (t < tend) {
    const int t2 = t1 < tend ? tile_next(it, active) : tend;
    if (t2 < tend) fetch_k(t2, cur);
    if (t1 < tend) {
      fetch_v(t1, cur ^ 1);
      if (docs) k1 = tile_entry(km, t1);
    }
    const int k0 = t * TILE;
    if (k0 < R.bmax) {                                                  // (tiles rise: a wave that is through stays so)
      bool some = k0 + TILE > R.bmin;
      if (docs) some |= (kn.neg != 0) | (kn.dmin != kn.dmax) | (R.dmin != R.dmax) | R.neg | (kn.dmin != R.dmin);
      const bool partial = __builtin_amdgcn_readfirstlane(some);
      const bf16_t* sv = st[cur].b;
      f32x16 n[2];
      const float c = MOD ? 1.f : mod.c;
      float off[2];                                                     // score = s + off[kb]
      if (MOD & 1) {                                                    // the cap's exponentials run beside the next tile's scores
        scores(n, st[cur ^ 1].a);
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            float w;
            s[kb][r] = capped<(MOD & 4) != 0>(mod, s[kb][r], w);
          }
      }
      off[0] = off[1] = 0.f;
      if (MOD & 2) {
        const int d0 = k0 + 4 * hi - R.pos;
        const float cc = (MOD & 1) ? 1.f : mod.c;
        if (mod.slope) {
          if (k0 + TILE - 1 <= R.pmin) {                              // every key at or before every query: |d| = -d, linear in the row
            const float sl = R.slope;
            off[0] = sl * (float)d0;
            off[1] = sl * (float)(d0 + 32);
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              const float b = sl * (float)crow(r, 0);
              s[0][r] = fmaf(s[0][r], cc, b);
              s[1][r] = fmaf(s[1][r], cc, b);
            }
          } else {
            const float f0 = (float)d0;
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
              for (int r = 0; r < 16; ++r)
                s[kb][r] = fmaf(-R.slope, fabsf(f0 + (32 * kb + crow(r, 0))), s[kb][r] * cc);
          }
        } else if (!(MOD & 1)) {
#pragma unroll
          for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int r = 0; r < 16; ++r) s[kb][r] *= cc;
        }
        if (mod.table) {
#pragma unroll
          for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int r = 0; r < 16; ++r) s[kb][r] += tab[max(-mod.R, min(mod.R, d0 + 32 * kb + crow(r, 0))) + mod.R];
        }
      }
      if (partial) {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
          const int lim = R.bound - k0 - 32 * kb - 4 * hi;
#pragma unroll
          for (int r = 0; r < 16; ++r) s[kb][r] = crow(r, 0) < lim ? s[kb][r] : -INFINITY;
          if (docs) {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              const int4 dv = *(const int4*)(sdoc + cur * TILE + 32 * kb + 8 * g + 4 * hi);
              s[kb][4 * g] = dv.x == R.doc ? s[kb][4 * g] : -INFINITY;
              s[kb][4 * g + 1] = dv.y == R.doc ? s[kb][4 * g + 1] : -INFINITY;
              s[kb][4 * g + 2] = dv.z == R.doc ? s[kb][4 * g + 2] : -INFINITY;
              s[kb][4 * g + 3] = dv.w == R.doc ? s[kb][4 * g + 3] : -INFINITY;
            }
          }
        }
      }
      float mx0 = s[0][0], mx1 = s[1][0];
#pragma unroll
      for (int r = 1; r < 16; ++r) {
        mx0 = fmaxf(mx0, s[0][r]);
        mx1 = fmaxf(mx1, s[1][r]);
      }
      const float mx = half_max(fmaxf(mx0 + off[0], mx1 + off[1]));
      // The running maximum is raised only when some row of the wave grew by more than `defer` exponent units: p <= 2^defer instead of
      // <= 1, and the common tile skips the rescale of O (8192 x 8192, 16 heads: 678 us, with defer = 0 702).  A pass that is to be differentiated
      // raises it at once: the weight of a key that dominates its row is then 1, which P's type holds exactly, and delta comes out closer
      // (dQ 0.0025 -> 0.0024 of its norm off where scores have a deviation of 4; dS's and the result's own rounding are 0.0023).
      if (!__all((mx - m) * c <= defer)) {
        const float mn = fmaxf(m, mx);
        const float alpha = __builtin_amdgcn_exp2f((m - mn) * c);
        m = mn;
        l *= alpha;
#pragma unroll
        for (int f = 0; f < FM; ++f)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[f][r] *= alpha;
      }
      // one straight block: the next tile's scores, this tile's exponentials, P V  (behind the last tile the scores are of stale rows, unused)
      if (!(MOD & 1)) scores(n, st[cur ^ 1].a);
      bf16x8 pb[4];
      float rs[2] = {0.f, 0.f};
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        const float mc = MOD ? m - off[kb] : fmaxf(m * c, LOWEST);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float pv = __builtin_amdgcn_exp2f(MOD ? s[kb][r] - mc : fmaf(s[kb][r], c, -mc));
          s[kb][r] = pv;
        }
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
          pb[2 * kb + kk] = pack8<T>(s[kb], kk);
          // The sum is of the rounded weights, those that multiply V: O is a mean of V with slightly other weights, never off by a factor.  Two
          // weights are added by one instruction (D = 64, 8192 x 8192, 16 heads: 400 -> 370 us)
          const u32x4 w = __builtin_bit_cast(u32x4, pb[2 * kb + kk]);
#pragma unroll
          for (int e = 0; e < 4; ++e) rs[e & 1] = El<T>::add2(w[e], rs[e & 1]);
        }
      }
      l += rs[0] + rs[1];
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int kk = 0; kk < 2; ++kk)
#pragma unroll
          for (int f = 0; f < FM; ++f) {
            const bf16x8 vf = trfrag<DP>(sv + ltr, kb, f, kk);
            o[f] = El<T>::mfma(vf, pb[2 * kb + kk], o[f]);
          }
      s[0] = n[0];
      s[1] = n[1];
    }
    if (t1 < tend) landed(t1, cur ^ 1, docs ? k1.neg : 0);
    cur ^= 1;
    t = t1;
    t1 = t2;
    kn = k1;
  }
  const float lt = half_sum(l);
  const float m2 = MOD ? m : fmaxf(m * mod.c, LOWEST);
  if (a.splits > 1) {
    const long long block = (((long long)sp * NU + u.x) * a.ntile + tile) * 4 + wave;       // of 32 rows
    store_part<FM>(a.part + block * (32 * DP), o, lane, R.ok);
    if (R.ok && hi == 0) *(float2*)(a.part_ml + (block * 32 + lane) * 2) = float2{m2, lt};
  } else {
    const long long at = op_base(a.p.o, u.b) + (long long)R.i * a.p.o.sstride + (long long)R.h * D;
    store_row<T, FM>((bf16_t*)a.p.o.ptr + at, o, lt > 0.f ? 1.f / lt : 0.f, hi, D, R.ok, a.p.o_rest ? (bf16_t*)a.p.o_rest + at : nullptr);
    if (R.ok && hi == 0 && a.p.lse) store_lse(a, ((long long)u.b * a.p.heads + u.h0) * a.p.Sq + R.r, m2, lt);
  }
}

// joins the splits: a workgroup per 32 rows and 32 columns, laid out like the accumulators.  It is as long as its chain of loads, so more
// than eight splits are dealt out to W = 8 waves, each has four in flight, and the eight results meet in LDS, in order; up to eight are all in
// flight in one wave.  One row, 32 / 8 heads of 128 over 32768 keys (64 splits): 48 -> 31 us with the forward kernel; 16 rows of 8 heads of 64 over 4096
// keys (4 splits): 28 us by one wave, 31 by eight.
template <typename T, int DP, int W>
__global__ __launch_bounds__(64 * W) void attn_mod_join_kernel(const Args a) {
  constexpr int FM = DP / 32, AT = W == 1 ? 8 : 4, ROW = 16 + 4;        // (16-byte aligned rows, 80 bytes apart)
  __shared__ __attribute__((aligned(16))) float meet[W > 1 ? W : 1][W > 1 ? 64 : 1][ROW];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), hi = lane >> 5, D = a.p.D;
  const int f = blockIdx.x % FM;
  const long long block = blockIdx.x / FM;                              // over (unit x, tile, 32 rows)
  const int NU = a.p.nbatch * a.nunit, per = a.ntile * 4, x = (int)(block / per);
  const int r = (int)(block - (long long)x * per) * 32 + (lane & 31);
  const bool ok = r < a.M;
  const long long stride = (long long)NU * per;                         // blocks of a split
  if (r - (lane & 31) >= a.M) return;                                   // workgroup-uniform
  const long long at = block * 32 + (lane & 31);
  // (Lanes behind the last row read their part of the padded buffer, whatever it holds, and store nothing: a branch around the loads would
  // put a wait behind each.)
  float m = -INFINITY, l = 0.f;                                         // (every split's m is finite)
  f32x16 acc[1];
#pragma unroll
  for (int e = 0; e < 16; ++e) acc[0][e] = 0.f;
  const auto add = [&](float ms, float ls, const f32x4 (&v)[4]) {       // one more partial result; m is not below ms
    const float w = __builtin_amdgcn_exp2f(ms - m);
    l = fmaf(w, ls, l);
#pragma unroll
    for (int g = 0; g < 4; ++g)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[0][4 * g + e] = fmaf(w, v[g][e], acc[0][4 * g + e]);
  };
  for (int s0 = wave; s0 < a.splits; s0 += AT * W) {
    float2 ml[AT];
    f32x4 v[AT][4];
#pragma unroll
    for (int k = 0; k < AT; ++k) {
      const long long s = min(s0 + k * W, a.splits - 1);
      ml[k] = *(const float2*)(a.part_ml + (s * stride * 32 + at) * 2);
#pragma unroll
      for (int g = 0; g < 4; ++g) v[k][g] = *(const f32x4*)(a.part + (s * stride + block) * (32 * DP) + (f * 256 + lane) * 4 + g * 256);
    }
    float mn = m;
#pragma unroll
    for (int k = 0; k < AT; ++k) mn = fmaxf(mn, ml[k].x);
    const float alpha = __builtin_amdgcn_exp2f(m - mn);
    m = mn;
    l *= alpha;
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[0][e] *= alpha;
#pragma unroll
    for (int k = 0; k < AT; ++k) {
      if (s0 + k * W >= a.splits) break;                       // wave-uniform
      add(ml[k].x, ml[k].y, v[k]);
    }
  }
  if constexpr (W > 1) {
    float* mine = meet[wave][lane];
#pragma unroll
    for (int g = 0; g < 4; ++g) *(f32x4*)(mine + 4 * g) = f32x4{acc[0][4 * g], acc[0][4 * g + 1], acc[0][4 * g + 2], acc[0][4 * g + 3]};
    *(float2*)(mine + 16) = float2{m, l};
    __syncthreads();
    if (wave) return;
    float ms[W], ls[W], mn = m;
#pragma unroll
    for (int k = 0; k < W; ++k) {
      const float2 ml = *(const float2*)(meet[k][lane] + 16);
      ms[k] = ml.x;
      ls[k] = ml.y;
      mn = fmaxf(mn, ml.x);
    }
    const float own = __builtin_amdgcn_exp2f(m - mn);
    m = mn;
    l *= own;
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[0][e] *= own;
#pragma unroll
    for (int k = 1; k < W; ++k) {
      f32x4 v[4];
#pragma unroll
      for (int g = 0; g < 4; ++g) v[g] = *(const f32x4*)(meet[k][lane] + 4 * g);
      add(ms[k], ls[k], v);
    }
  }
  const Unit u = unit_of(a, x);
  const int i = div_gp(a, min(r, a.M - 1)), h = u.h0 + min(r, a.M - 1) - i * a.gp;
  const long long col = op_base(a.p.o, u.b) + (long long)i * a.p.o.sstride + (long long)h * D + 32 * f;
  store_row<T, 1>((bf16_t*)a.p.o.ptr + col, acc, l > 0.f ? 1.f / l : 0.f, hi, D - 32 * f, ok, a.p.o_rest ? (bf16_t*)a.p.o_rest + col : nullptr);
  if (ok && f == 0 && hi == 0 && a.p.lse) store_lse(a, ((long long)u.b * a.p.heads + u.h0) * a.p.Sq + r, m, l);
}

// bounds and documents of every 64 rows / keys (launched where a mask has documents or one prefix per query): one wave per tile (5 us at 8200
// rows and keys: a launch and a chain of three loads)
__global__ __launch_bounds__(64) void attn_mod_meta_kernel(const Args a, QMeta* qm, KMeta* km, int nq, int nk) {
  const int lane = threadIdx.x, b = blockIdx.y, t = blockIdx.x;
  const Seq seq = load_seq(a, b);
  const int len = seq.len;
  if (t < nq) {
    const int r = t * TILE + lane;
    int lo = 0x7fffffff, hi = 0, dlo = 0x7fffffff, dhi = -1, ng = 0;
    if (r < a.M) {
      const int i = div_gp(a, r), d = a.p.q_docs ? a.p.q_docs[(long long)b * a.p.Sq + i] : 0;
      const int bd = d < 0 ? 0 : row_bound(seq, i);
      lo = hi = bd;
      if (bd > 0) dlo = dhi = d;
      else ng = 1;
    }
    const QMeta q = {wave_min_i(lo), wave_max_i(hi), wave_min_i(dlo), wave_max_i(dhi), wave_max_i(ng)};
    if (lane == 0) qm[(long long)b * nq + t] = q;
  } else {
    const int j = (t - nq) * TILE + lane;
    int dlo = 0x7fffffff, dhi = -1, ng = 0;
    if (j < len) {
      const int d = a.p.kv_docs ? a.p.kv_docs[(long long)b * a.p.Sk + j] : 0;
      if (d >= 0) dlo = dhi = d;
      else ng = 1;
    }
    const KMeta k = {wave_min_i(dlo), wave_max_i(dhi), wave_max_i(ng)};
    if (lane == 0) km[(long long)b * nk + t - nq] = k;
  }
}

// With documents the work of a row tile (and of a key tile) depends on them, and with about as many workgroups as the card holds at once the
// launch takes as long as its longest workgroup.  A tile across the border of two documents would visit both: it becomes two entries, one
// for the rows of its first document (and those of none), one for the others.  Entries (batch, tile, part) are sorted by the tiles they
// will visit, the longest first; equal ones stay in order, and second parts of tiles with one document come last and end at once.
// Block 0: row tiles of 128; block 1: key tiles.  One thread counts an entry and its rank among the others.
// (Nine clips, 8200 tokens, 10 heads of 64: forward 93 -> 54 us, dQ 102 -> 64 us, dK / dV 149 -> 105 us for the 9 us of this launch, once per
// mask and step.)
constexpr int ORDER_MAX = 1024, ORDER_TILES = 4096;
__global__ __launch_bounds__(1024) void attn_mod_order_kernel(const Args a, int* qorder, int* korder, int nq, int nk, int keys) {
  __shared__ unsigned long long key[ORDER_MAX];
  __shared__ int slo[ORDER_TILES], shi[ORDER_TILES], sbound[ORDER_TILES];     // of the other side's 64-row tiles
  const int tid = threadIdx.x, side = blockIdx.x;
  const int ntile = side ? nk : nq, n = 2 * a.p.nbatch * ntile, per = side ? keys / TILE : 2;
  const int nqt = (a.M + TILE - 1) / TILE, nkt = (a.p.Sk + TILE - 1) / TILE, nown = side ? nkt : nqt, nother = side ? nqt : nkt;
  const int e = min(tid, n - 1), part = e & 1, b = (e >> 1) / ntile, t = (e >> 1) - b * ntile;
  int lo = 0x7fffffff, hi = -1, bmax = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k) {                                         // (all loads in flight; one that is met twice changes nothing)
    const long long at = (long long)b * nown + min(t * per + min(k, per - 1), nown - 1);
    lo = min(lo, side ? a.kmeta[at].dmin : a.qmeta[at].dmin);
    hi = max(hi, side ? a.kmeta[at].dmax : a.qmeta[at].dmax);
    if (!side) bmax = max(bmax, a.qmeta[at].bmax);
  }
  for (int i = tid; i < a.p.nbatch * nother; i += 1024) {
    slo[i] = side ? a.qmeta[i].dmin : a.kmeta[i].dmin;
    shi[i] = side ? a.qmeta[i].dmax : a.kmeta[i].dmax;
    sbound[i] = side ? a.qmeta[i].bmax : 0x7fffffff;
  }
  if (part) lo = lo == 0x7fffffff ? lo : lo + 1;
  else hi = min(lo, hi);
  const int end = lo > hi || tid >= n ? 0 : side ? nqt : (bmax + TILE - 1) / TILE, floor = side ? t * keys : 0;
  __syncthreads();
  int count = 0;
#pragma unroll 8
  for (int c = 0; c < end; ++c) {
    const int i = b * nother + c;
    count += (sbound[i] > floor) & (shi[i] >= lo) & (slo[i] <= hi);
  }
  const unsigned long long mine = ((unsigned long long)(2 * count + 2 - part) << 32) | (unsigned)(~e);
  if (tid < n) key[tid] = mine;
  __syncthreads();
  if (tid >= n) return;
  int rank = 0;
#pragma unroll 8
  for (int k = 0; k < n; ++k) rank += key[k] > mine;
  (side ? korder : qorder)[rank] = tid;
}

// ------------------------------------------------------------------------------------------------ backward: dQ, delta, table gradient
// Three products per score, Q, dO and dQ of the wave's 32 rows in registers.  8192 x 8192, 16 heads of 128, bf16: 780 to 814 us,
// 1013 to 1057 TFLOP/s.  Scalars spill to vector lanes where there is a distance bias (88 to 102 of them), vectors at <128, 7> alone (8).  At <64, 2> three
// waves per SIMD are asked for: without that the allocator takes one register more than they leave.
template <typename T, int DP, int MOD>
__global__ __launch_bounds__(256, DP == 64 && MOD < 3 ? 3 : 2) void attn_mod_dq_kernel(const Args a) {
  warm_kernargs<(int)sizeof(Args)>();
  constexpr int NT = 256, KD = DP / 16, FM = DP / 32;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  Stage<DP>* st = (Stage<DP>*)smem;
  int* sdoc = (int*)(smem + 2 * sizeof(Stage<DP>));
  int* swg = sdoc + 2 * TILE;
  float* tab = (float*)(swg + 16);                                      // [2R + 1], then [4 waves][2R + 1] sums
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), hi = lane >> 5;
  const int NU = a.p.nbatch * a.nunit, sp = blockIdx.x / NU % a.splits;
  int tile;
  Part part;
  const Unit u = work_of(a, blockIdx.x / (NU * a.splits) * NU + blockIdx.x % NU, tile, part);
  float* dtable = a.part_bias;                                          // of this workgroup (its head's 2R + 1 sums)
  if (a.p.dbias)
    dtable += ((((long long)u.b * a.ntile + tile) * (a.qorder ? 2 : a.splits) + max(part.part, 0) + sp) * a.p.heads + u.h0) * (2 * a.p.radius + 1);
  if (part.none) {                                                      // workgroup-uniform
    if (a.p.dbias)
      for (int i = threadIdx.x; i < 2 * a.p.radius + 1; i += 256) dtable[i] = 0.f;
    return;
  }
  const Seq seq = load_seq(a, u.b);
  const int len = seq.len, D = a.p.D, Sk = a.p.Sk;
  const bool docs = a.kmeta && a.p.kv_docs;
  const int* kdoc = docs ? a.p.kv_docs + (long long)u.b * Sk : nullptr;
  const Mod mod = make_mod(a);
  const int ntab = 2 * a.p.radius + 1;
  float* sums = tab + ntab + wave * ntab;
  const bool dtab = (MOD & 2) && mod.table && a.p.dbias != nullptr;

  Rows R;
  load_rows(R, a, u, seq, part, (tile * 4 + wave) * 32, lane);
  bf16x8 qf[KD], gf[KD];
  const bf16_t* qp = (const bf16_t*)a.p.q.ptr + op_base(a.p.q, u.b) + (long long)R.i * a.p.q.sstride + (long long)R.h * D;
  const bf16_t* gp = (const bf16_t*)a.p.d_o.ptr + op_base(a.p.d_o, u.b) + (long long)R.i * a.p.d_o.sstride + (long long)R.h * D;
  const bf16_t* op = (const bf16_t*)a.p.o.ptr + op_base(a.p.o, u.b) + (long long)R.i * a.p.o.sstride + (long long)R.h * D;
  const bool rest = a.p.o_rest != nullptr;
  const bf16_t* orest = rest ? (const bf16_t*)a.p.o_rest + (op - (const bf16_t*)a.p.o.ptr) : op;
  bf16x8 of[KD], og[KD];
#pragma unroll
  for (int kd = 0; kd < KD; ++kd) {
    const bool ok = R.bound > 0 && 16 * kd + 8 * hi < D;
    qf[kd] = *chunk_ptr(qp + 16 * kd + 8 * hi, ok);
    gf[kd] = *chunk_ptr(gp + 16 * kd + 8 * hi, ok);
    of[kd] = *chunk_ptr(op + 16 * kd + 8 * hi, ok);
    og[kd] = *chunk_ptr(orest + 16 * kd + 8 * hi, ok && rest);
  }
  const long long sidx = ((long long)u.b * a.p.heads + u.h0) * a.p.Sq + min(R.r, a.M - 1);
  const float lse = R.ok ? a.p.lse[sidx] : INFINITY;
  const float lsum = (MOD & 2) && R.ok ? a.lsum[sidx] : 0.f;
  if ((MOD & 2) && mod.table) load_table<T>(a, u.h0, tab, tid, NT);
  if (dtab)
    for (int i = lane; i < ntab; i += 64) sums[i] = 0.f;
  if (lane == 0) {
    swg[wave * 4] = R.bmax;
    swg[wave * 4 + 1] = R.dmin;
    swg[wave * 4 + 2] = R.dmax;
  }
  __syncthreads();
  int bmax = 0, dmin = 0x7fffffff, dmax = -1;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    bmax = max(bmax, swg[w * 4]);
    dmin = min(dmin, swg[w * 4 + 1]);
    dmax = max(dmax, swg[w * 4 + 2]);
  }
  bmax = __builtin_amdgcn_readfirstlane(bmax);
  const KMeta* km = docs ? a.kmeta + (long long)u.b * ((Sk + TILE - 1) / TILE) : nullptr;
  auto active = [&](int c) { return km[c].dmax >= dmin && km[c].dmin <= dmax; };
  int tbeg, tend;
  split_tiles((bmax + TILE - 1) / TILE, a.splits, sp, docs, active, tbeg, tend);
  TileIter it = {0ull, tbeg, tend, docs};
  const Lane<DP, 4> ln(wave, lane, D);
  const int lrow = lane_row<DP>(lane), ltr = lane_tr<DP>(lane);
  const bf16_t* kp = ln.ok ? (const bf16_t*)a.p.k.ptr + op_base(a.p.k, u.b) + (long long)u.kv * D + ln.ch * 8 : (const bf16_t*)zero_chunk;
  const bf16_t* vp = ln.ok ? (const bf16_t*)a.p.v.ptr + op_base(a.p.v, u.b) + (long long)u.kv * D + ln.ch * 8 : (const bf16_t*)zero_chunk;
  const unsigned ks = ln.ok ? (unsigned)a.p.k.sstride : 0u, vs = ln.ok ? (unsigned)a.p.v.sstride : 0u;
  int nd = 0;
  auto fetch = [&](int t, int sidx) {                                   // rows behind the last key repeat it (masked by the bounds)
#pragma unroll
    for (int i = 0; i < Lane<DP, 4>::NI; ++i) {
      const unsigned row = (unsigned)min(t * TILE + ln.row_of(i), len - 1);
      copy16(kp + (unsigned long long)row * ks, st[sidx].a + ln.group(i));
      copy16(vp + (unsigned long long)row * vs, st[sidx].b + ln.group(i));
    }
    if (docs && tid < TILE) nd = kdoc[min(t * TILE + tid, len - 1)];
  };
  auto landed = [&](int t, int sidx, int neg) {                         // tile t, fetched into stage sidx, is there for all waves
    if (docs && tid < TILE) sdoc[sidx * TILE + tid] = t * TILE + tid < len ? nd : -1;
    copies_done();
    __syncthreads();
    if (neg) {
      clear_rows<DP, NT, true>(st[sidx], tid, [&](int r) { return sdoc[sidx * TILE + r] < 0; });
      __syncthreads();
    }
  };
  f32x16 acc[FM];
#pragma unroll
  for (int f = 0; f < FM; ++f)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[f][r] = 0.f;
  float below = 0.f, above = 0.f;                                       // gradient of the table's two ends, per lane
  int t = tile_next(it, active), cur = 0;
  KMeta kn = {0, 0, 0};                                                 // of the tile at hand (documents)
  if (t < tend) {
    if (docs) kn = tile_entry(km, t);
    fetch(t, 0);
  }
  float dl = 0.f;                                                       // delta, while the first tile is on its way
#pragma unroll
  for (int kd = 0; kd < KD; ++kd)
#pragma unroll
    for (int e = 0; e < 8; ++e) dl = fmaf(El<T>::up(of[kd][e]) + El<T>::up(og[kd][e]), El<T>::up(gf[kd][e]), dl);
  dl = half_sum(dl);
  if (R.ok && hi == 0 && sp == 0) a.p.delta[sidx] = dl;
  if (t < tend) landed(t, 0, kn.neg);
  auto math = [&](bool partial, int t) {
    const int k0 = t * TILE;
    const bf16_t* sk = st[cur].a;
    const bf16_t* sv = st[cur].b;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      f32x16 s, dp;
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = dp[r] = 0.f;
#pragma unroll
      for (int kd = 0; kd < KD; ++kd) {
        const bf16x8 kf = rowfrag<DP>(sk + lrow, kb, kd), vf = rowfrag<DP>(sv + lrow, kb, kd);
        s = El<T>::mfma(kf, qf[kd], s);
        dp = El<T>::mfma(vf, gf[kd], dp);
      }
      bf16x8 db[2];
      const int d0 = k0 + 32 * kb + 4 * hi - R.pos;
      f32x16 w;                                                         // derivative of the cap
      if (MOD & 1) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          float y;
          s[r] = capped<(MOD & 4) != 0>(mod, s[r], y);
          w[r] = 4.f * y * (1.f - y);
        }
      } else if (MOD & 2) {
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] *= mod.c;
      }
      if (MOD & 2) {
        if (mod.slope) {
          const float f0 = (float)d0;
#pragma unroll
          for (int r = 0; r < 16; ++r) s[r] = fmaf(-R.slope, fabsf(f0 + crow(r, 0)), s[r]);
        }
        if (mod.table) {
#pragma unroll
          for (int r = 0; r < 16; ++r) s[r] += tab[max(-mod.R, min(mod.R, d0 + crow(r, 0))) + mod.R];
        }
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float pv = __builtin_amdgcn_exp2f((MOD & 2) ? (s[r] - lse) - lsum : MOD ? s[r] - lse : fmaf(s[r], mod.c, -lse));
        s[r] = pv * (dp[r] - dl);
      }
      if (partial) {
        const int lim = R.bound - k0 - 32 * kb - 4 * hi;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = crow(r, 0) < lim ? s[r] : 0.f;
        if (docs) {
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const int4 dv = *(const int4*)(sdoc + cur * TILE + 32 * kb + 8 * g + 4 * hi);
            s[4 * g] = dv.x == R.doc ? s[4 * g] : 0.f;
            s[4 * g + 1] = dv.y == R.doc ? s[4 * g + 1] : 0.f;
            s[4 * g + 2] = dv.z == R.doc ? s[4 * g + 2] : 0.f;
            s[4 * g + 3] = dv.w == R.doc ? s[4 * g + 3] : 0.f;
          }
        }
      }
      if ((MOD & 2) && dtab) {
        // sums over diagonals, in the wave's own table, by LDS additions that complete in program order: a register's 32 lanes of one
        // half hold 32 different distances, so one half at a time meets no address twice and the order of the additions is fixed
        // (the wave barriers keep the compiler from joining the two halves); the clipped ends are summed per lane
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int d = d0 + crow(r, 0);
          const float v = s[r];
          const bool in = d > -mod.R && d < mod.R;
          below += d <= -mod.R ? v : 0.f;
          above += (d >= mod.R && d > -mod.R) ? v : 0.f;
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            if (in && hi == half) __builtin_amdgcn_ds_atomic_fadd_f32((__attribute__((address_space(3))) float*)(sums + d + mod.R), v);
            __builtin_amdgcn_wave_barrier();
          }
        }
      }
      if (MOD & 1) {
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] *= w[r];
      }
      db[0] = pack8<T>(s, 0);
      db[1] = pack8<T>(s, 1);
#pragma unroll
      for (int kk = 0; kk < 2; ++kk)
#pragma unroll
        for (int f = 0; f < FM; ++f) {
          const bf16x8 kT = trfrag<DP>(sk + ltr, kb, f, kk);
          acc[f] = El<T>::mfma(kT, db[kk], acc[f]);
        }
    }
  };
  while (t < tend) {
    const int tn = tile_next(it, active);
    const KMeta kt = kn;
    if (tn < tend) {
      fetch(tn, cur ^ 1);
      if (docs) kn = tile_entry(km, tn);
    }
    const int k0 = t * TILE;
    if (k0 < R.bmax) {
      bool partial = k0 + TILE > R.bmin;
      if (docs) partial |= (kt.neg != 0) | (kt.dmin != kt.dmax) | (R.dmin != R.dmax) | R.neg | (kt.dmin != R.dmin);
      math(__builtin_amdgcn_readfirstlane(partial), t);
    }
    if (tn < tend) landed(tn, cur ^ 1, docs ? kn.neg : 0);
    cur ^= 1;
    t = tn;
  }
  if (a.splits > 1) {
    const long long block = (((long long)sp * NU + u.x) * a.ntile + tile) * 4 + wave;                          // of 32 rows
    store_part<FM>(a.part + block * (32 * DP), acc, lane, R.ok);
  } else {
    bf16_t* dqp = (bf16_t*)a.p.dq.ptr + op_base(a.p.dq, u.b) + (long long)R.i * a.p.dq.sstride + (long long)R.h * D;
    store_row<T, FM>(dqp, acc, a.p.scale, hi, D, R.ok);
  }
  if (dtab) {
    below = wave_sum(below);
    above = wave_sum(above);
    if (lane == 0) {
      sums[0] += below;
      sums[ntab - 1] += above;
    }
    __syncthreads();
    for (int i = tid; i < ntab; i += NT) {
      const float* w0 = tab + ntab + i;
      dtable[i] = (w0[0] + w0[ntab]) + (w0[2 * ntab] + w0[3 * ntab]);
    }
  }
}

// dQ = sum of the splits' partial sums, in order: one wave per 32 rows and 32 columns (8 us at 15 row tiles of 8 heads of 128 in four splits)
template <typename T, int DP>
__global__ __launch_bounds__(64) void attn_mod_dq_join_kernel(const Args a) {
  constexpr int FM = DP / 32;
  const int lane = threadIdx.x, hi = lane >> 5, D = a.p.D;
  const int f = blockIdx.x % FM;
  const long long block = blockIdx.x / FM;                              // over (unit x, tile, 32 rows)
  const int NU = a.p.nbatch * a.nunit, per = a.ntile * 4, x = (int)(block / per);
  const int r0 = (int)(block - (long long)x * per) * 32, r = min(r0 + (lane & 31), a.M - 1);
  if (r0 >= a.M) return;                                                // workgroup-uniform
  f32x16 acc[1];
#pragma unroll
  for (int e = 0; e < 16; ++e) acc[0][e] = 0.f;
#pragma unroll 4
  for (int s = 0; s < a.splits; ++s) {
    const float* p = a.part + ((long long)s * NU * per + block) * (32 * DP) + (f * 256 + lane) * 4;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const f32x4 v = *(const f32x4*)(p + g * 256);
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[0][4 * g + e] += v[e];
    }
  }
  const Unit u = unit_of(a, x);
  const int i = div_gp(a, r), h = u.h0 + r - i * a.gp;
  bf16_t* dqp = (bf16_t*)a.p.dq.ptr + op_base(a.p.dq, u.b) + (long long)i * a.p.dq.sstride + (long long)h * D + 32 * f;
  store_row<T, 1>(dqp, acc, a.p.scale, hi, D - 32 * f, r0 + (lane & 31) < a.M);
}

// dtable[h][d] = sum over (batch, row tile, split), in order (4 us, a launch); entries that hide their distance get 0 by construction (P = 0 there)
template <typename T>
__global__ __launch_bounds__(256) void attn_mod_dbias_kernel(const Args a) {
  const long long n = (long long)a.p.heads * (2 * a.p.radius + 1), i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  float s = 0.f;
#pragma unroll 4
  for (int k = 0; k < a.p.nbatch * a.ntile * (a.qorder ? 2 : a.splits); ++k) s += a.part_bias[(long long)k * n + i];
  if (a.p.bias_f32) ((float*)a.p.dbias)[i] = s;
  else ((unsigned short*)a.p.dbias)[i] = (unsigned short)(El<T>::pack2(s, 0.f) & 0xffffu);
}

// ------------------------------------------------------------------------------------------------ backward: dK, dV
constexpr int INFO = 7;             // numbers of a staged query row
struct RowInfo {                    // of one query row, as loaded
  float lse, lsum, delta, slope;
  int doc, prefix;
};
// A wave owns 32 keys and streams the rows that see them.  K, V, dK and dV of 32 keys of 128 columns are 192 registers: with the score and
// gradient tiles a wave would need more than half of a SIMD's file, and one wave per SIMD has nothing to run under its exponentials
// (301 us at 2 x 2011 rows, 16 / 4 heads; this form 144 us).  So at DP = 128 the workgroup is eight waves, its V rows stay in LDS, and two
// waves share a SIMD.  LDS bounds it then: at full matrix rate it would deliver 156 bytes per clock, against its 128.  8192 x 8192, 16 heads of 128:
// 1.36 to 1.42 ms, 775 to 808 TFLOP/s.  It does not fit its 256 registers at DP = 128: 31 / 39 / 60 / 63 vectors spill for the four score forms
// (44 / 68 with caps above WIDE_CAP; 88 to 172 bytes of scratch a lane), because the 48 registers of scores, weights and dP live through a whole row block.
template <typename T, int DP, int MOD>
__global__ __launch_bounds__(DP == 128 ? 512 : 256, 2) void attn_mod_dkdv_kernel(const Args a) {
  warm_kernargs<(int)sizeof(Args)>();
  constexpr int NW = DP == 128 ? 8 : 4, NT = 64 * NW, KD = DP / 16, FM = DP / 32, KEYS = 32 * NW;
  constexpr bool VLDS = DP == 128;
  constexpr int HALF = TILE * DP / 512 * GROUP;                         // elements of 64 staged rows
  extern __shared__ __attribute__((aligned(16))) char smem[];
  Stage<DP>* st = (Stage<DP>*)smem;
  float* sinfo = (float*)(smem + 2 * sizeof(Stage<DP>));                // [2][INFO][TILE]: lse, delta, slope, bound, pos, doc, lsum
  float* tab = sinfo + 2 * INFO * TILE;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), hi = lane >> 5;
  const int NKV = a.p.nbatch * a.p.kv_heads, G = a.p.heads / a.p.kv_heads, GU = G / a.gp, ntr = (a.M + TILE - 1) / TILE;
  Part part = {0, -1, false};
  int y = blockIdx.x % NKV, ktile = blockIdx.x / NKV, sp = 0, runs = 1; // early keys are seen by the most rows of a causal mask: first
  const int w = ktile;
  if (a.korder) {
    const int e = a.korder[blockIdx.x / a.p.kv_heads], bt = (e >> 1) / a.ntile, nkt = (a.p.Sk + TILE - 1) / TILE;
    ktile = (e >> 1) - bt * a.ntile;
    y = bt * a.p.kv_heads + blockIdx.x % a.p.kv_heads;
    part = part_of(a.kmeta + (long long)bt * nkt, ktile, KEYS / TILE, nkt, e & 1);
    if (part.none) return;                                              // workgroup-uniform
  } else if (a.to_part) {
    sp = ktile;
    for (ktile = 0; sp >= (runs = kv_runs(a, ktile, KEYS, ntr * GU)); ++ktile) sp -= runs;
  }
  const int b = y / a.p.kv_heads, kv = y - b * a.p.kv_heads;
  const Seq seq = load_seq(a, b);
  const int len = seq.len, D = a.p.D, Sk = a.p.Sk;
  const bool docs = a.kmeta && a.p.kv_docs;
  const Mod mod = make_mod(a);
  const bf16_t* Q = (const bf16_t*)a.p.q.ptr + op_base(a.p.q, b);
  const bf16_t* dO = (const bf16_t*)a.p.d_o.ptr + op_base(a.p.d_o, b);
  bf16_t* sV = (bf16_t*)(tab + (a.p.bias ? (2 * a.p.radius + 1 + 3) / 4 * 4 : 0)) + (wave >> 1) * HALF;      // VLDS: the wave's 64-key tile
  const int wk0 = ktile * KEYS, kw0 = wk0 + wave * 32;                  // the first key of the workgroup, of the wave
  const int key = kw0 + (lane & 31);
  // does the key exist, and may some query see it
  auto key_doc = [&](int j) { return j < len ? (docs ? a.p.kv_docs[(long long)b * Sk + j] : 0) : -1; };
  const int kdoc = key_doc(key);
  const bool own = key < Sk && part.owns(kdoc);                         // its gradients are written here
  const int kd_ = own ? kdoc : -1;
  const bool kok = kd_ >= 0;
  const bf16_t* K = (const bf16_t*)a.p.k.ptr + op_base(a.p.k, b) + (long long)kv * D;
  const bf16_t* V = (const bf16_t*)a.p.v.ptr + op_base(a.p.v, b) + (long long)kv * D;
  bf16x8 kf[KD], vf[VLDS ? 1 : KD];
#pragma unroll
  for (int kd = 0; kd < KD; ++kd) {
    const bool ok = kok && 16 * kd + 8 * hi < D;
    kf[kd] = *chunk_ptr(K + (long long)key * a.p.k.sstride + 16 * kd + 8 * hi, ok);
    if constexpr (!VLDS) vf[kd] = *chunk_ptr(V + (long long)key * a.p.v.sstride + 16 * kd + 8 * hi, ok);
  }
  const int lrow = lane_row<DP>(lane), ltr = lane_tr<DP>(lane);
  if constexpr (VLDS) {                                                 // each wave loads, and reads, its own 32 rows
#pragma unroll
    for (int g = 0; g < 8; ++g) {
      const int j = kw0 + g + 8 * (lane >> 4), ch = lane & 15;
      copy16(chunk_ptr(V + (long long)j * a.p.v.sstride + ch * 8, key_doc(j) >= 0 && ch * 8 < D), sV + ((wave & 1) * 8 + g) * GROUP);
    }
  }
  auto vfrag = [&](int kd) {
    if constexpr (VLDS) return rowfrag<DP>(sV + lrow + row_off<DP>(32 * (wave & 1)), 0, kd);
    else return vf[kd];
  };
  int dlo = kok ? kd_ : 0x7fffffff, dhi = kd_, ng = !kok;
  const int wdmin = wave_min_i(dlo), wdmax = wave_max_i(dhi);
  const bool wneg = wave_max_i(ng) != 0;
  // over the workgroup's own keys
  int gdmin = 0x7fffffff, gdmax = -1;
  if (docs) {
    const KMeta* km = a.kmeta + (long long)b * ((Sk + TILE - 1) / TILE);
    for (int t = wk0 / TILE; t < min((Sk + TILE - 1) / TILE, (wk0 + KEYS) / TILE); ++t) {
      const KMeta m = tile_entry(km, t);
      gdmin = min(gdmin, m.dmin);
      gdmax = max(gdmax, m.dmax);
    }
    if (part.part == 0) gdmax = min(gdmax, part.first);
    if (part.part == 1) gdmin = part.first + 1;
  }
  f32x16 ka[FM], va[FM];
#pragma unroll
  for (int f = 0; f < FM; ++f)
#pragma unroll
    for (int r = 0; r < 16; ++r) ka[f][r] = va[f][r] = 0.f;

  // The row tiles that matter, of all units of the K / V head, are numbered through and divided among the `runs` workgroups.  With the meta table
  // those are all tiles, filtered on the way; without it bounds grow with the query, and only the last tiles of a unit see key wk0 or a later one.
  const QMeta* qm = a.qmeta ? a.qmeta + (long long)b * ntr : nullptr;
  const int first = first_tile(a, seq, wk0), run = ntr - first, total = wk0 < len ? run * GU : 0;
  const int per = (total + runs - 1) / runs, tbeg = min(total, sp * per), tend = min(total, tbeg + per);
  auto tile_meta = [&](int t) {
    if (qm) return tile_entry(qm, t);
    return QMeta{t * TILE + TILE > a.M ? 0 : row_bound(seq, div_gp(a, t * TILE)), row_bound(seq, div_gp(a, min(a.M, t * TILE + TILE) - 1)), 0, 0, 0};
  };
  auto active = [&](int c) {
    const QMeta m = qm[c % ntr];
    return m.bmax > wk0 && (!docs || (m.dmax >= gdmin && m.dmin <= gdmax));
  };
  TileIter it = {0ull, tbeg, tend, qm != nullptr};
  const Lane<DP, NW> ln(wave, lane, D);
  const bf16_t* qp = ln.ok ? Q + ln.ch * 8 : (const bf16_t*)zero_chunk;
  const bf16_t* gp = ln.ok ? dO + ln.ch * 8 : (const bf16_t*)zero_chunk;
  const unsigned qs = ln.ok ? (unsigned)a.p.q.sstride : 0u, gs = ln.ok ? (unsigned)a.p.d_o.sstride : 0u, hs = ln.ok ? (unsigned)D : 0u;
  RowInfo ni = {0.f, 0.f, 0.f, 0.f, 0, 0};
  auto fetch = [&](int c, int sidx) {                                   // rows behind the last repeat it (their weights are masked to 0)
    const int gu = c / run, t = first + c - gu * run, h0 = kv * G + gu * a.gp;
#pragma unroll
    for (int n = 0; n < Lane<DP, NW>::NI; ++n) {
      const int rc = min(t * TILE + ln.row_of(n), a.M - 1), i = div_gp(a, rc);
      const unsigned h = (unsigned)(h0 + rc - i * a.gp) * hs;
      copy16(qp + (unsigned long long)(unsigned)i * qs + h, st[sidx].a + ln.group(n));
      copy16(gp + (unsigned long long)(unsigned)i * gs + h, st[sidx].b + ln.group(n));
    }
    if (tid < TILE) {                                                   // (raw values only: what is computed from them waits for them)
      const int rc = min(t * TILE + tid, a.M - 1), i = div_gp(a, rc);
      const long long at = ((long long)b * a.p.heads + h0) * a.p.Sq + rc;
      ni.lse = a.p.lse[at];
      if (MOD & 2) ni.lsum = a.lsum[at];
      ni.delta = a.p.delta[at];
      if (docs) ni.doc = a.p.q_docs[(long long)b * a.p.Sq + i];
      if ((MOD & 2) && a.p.slopes) ni.slope = a.p.slopes[h0 + rc - i * a.gp];
      if (seq.per_query) ni.prefix = seq.per_query[i];
    }
  };
  auto landed = [&](int c, int sidx, bool dead) {
    float* in = sinfo + sidx * INFO * TILE;
    if (tid < TILE) {
      const int r = (first + c % run) * TILE + tid, i = div_gp(a, min(r, a.M - 1));
      const int bound = (r < a.M && ni.doc >= 0) ? bound_of(seq, i, seq.per_query ? ni.prefix : seq.prefix) : 0;
      in[tid] = bound > 0 ? ni.lse : INFINITY;
      in[TILE + tid] = bound > 0 ? ni.delta : 0.f;
      in[2 * TILE + tid] = ni.slope * LOG2E;
      in[3 * TILE + tid] = __int_as_float(bound);
      in[4 * TILE + tid] = __int_as_float(i + seq.off);
      in[5 * TILE + tid] = __int_as_float(ni.doc);
      if (MOD & 2) in[6 * TILE + tid] = ni.lsum;
    }
    copies_done();
    __syncthreads();
    if (dead) {
      clear_rows<DP, NT, true>(st[sidx], tid, [&](int r) { return __float_as_int(in[3 * TILE + r]) <= 0; });
      __syncthreads();
    }
  };
  int c = tile_next(it, active), cur = 0, gu_tab = -1;
  QMeta mn = {0, 0, 0, 0, 0};
  if (c < tend) {
    mn = tile_meta(first + c % run);
    fetch(c, 0);
    landed(c, 0, mn.bmin <= 0);
  }
  auto math = [&](bool partial) {
    const bf16_t* sq = st[cur].a;
    const bf16_t* sg = st[cur].b;
    const float* in = sinfo + cur * INFO * TILE;
#pragma unroll
    for (int qb = 0; qb < 2; ++qb) {
      f32x16 s, dp, pr;
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = dp[r] = 0.f;
#pragma unroll
      for (int kd = 0; kd < KD; ++kd) s = El<T>::mfma(rowfrag<DP>(sq + lrow, qb, kd), kf[kd], s);
#pragma unroll
      for (int kd = 0; kd < KD; ++kd) dp = El<T>::mfma(rowfrag<DP>(sg + lrow, qb, kd), vfrag(kd), dp);
      bf16x8 pb[2], db[2];
      __builtin_amdgcn_sched_barrier(0);
      {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int o = 32 * qb + 8 * g + 4 * hi;
          const f32x4 L = *(const f32x4*)(in + o), E = *(const f32x4*)(in + TILE + o);
          f32x4 W = {1.f, 1.f, 1.f, 1.f}, Z = {0.f, 0.f, 0.f, 0.f};
          if (MOD & 2) Z = *(const f32x4*)(in + 6 * TILE + o);
          if (MOD & 1) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float w;
              s[4 * g + e] = capped<(MOD & 4) != 0>(mod, s[4 * g + e], w);
              W[e] = 4.f * w * (1.f - w);
            }
          } else if (MOD & 2) {
#pragma unroll
            for (int e = 0; e < 4; ++e) s[4 * g + e] *= mod.c;
          }
          if (MOD & 2) {
            const int4 pos = *(const int4*)(in + 4 * TILE + o);
            const int ps[4] = {pos.x, pos.y, pos.z, pos.w};
            if (mod.slope) {
              const f32x4 sl = *(const f32x4*)(in + 2 * TILE + o);
#pragma unroll
              for (int e = 0; e < 4; ++e) s[4 * g + e] = fmaf(-sl[e], fabsf((float)(key - ps[e])), s[4 * g + e]);
            }
            if (mod.table) {
#pragma unroll
              for (int e = 0; e < 4; ++e) s[4 * g + e] += tab[max(-mod.R, min(mod.R, key - ps[e])) + mod.R];
            }
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            pr[4 * g + e] = __builtin_amdgcn_exp2f((MOD & 2) ? (s[4 * g + e] - L[e]) - Z[e] : MOD ? s[4 * g + e] - L[e] : fmaf(s[4 * g + e], mod.c, -L[e]));
            const float d = pr[4 * g + e] * (dp[4 * g + e] - E[e]);
            s[4 * g + e] = (MOD & 1) ? d * W[e] : d;
          }
        }
        if (partial) {
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const int o = 32 * qb + 8 * g + 4 * hi;
            const int4 bd = *(const int4*)(in + 3 * TILE + o);
            const int bs[4] = {bd.x, bd.y, bd.z, bd.w};
            int4 dc = {0, 0, 0, 0};
            if (docs) dc = *(const int4*)(in + 5 * TILE + o);
            const int ds[4] = {dc.x, dc.y, dc.z, dc.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const bool live = (key < bs[e]) & (!docs | (kd_ == ds[e]));
              pr[4 * g + e] = live ? pr[4 * g + e] : 0.f;
              s[4 * g + e] = live ? s[4 * g + e] : 0.f;
            }
          }
        }
        pb[0] = pack8<T>(pr, 0);
        pb[1] = pack8<T>(pr, 1);
        db[0] = pack8<T>(s, 0);
        db[1] = pack8<T>(s, 1);
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int kk = 0; kk < 2; ++kk)
#pragma unroll
        for (int f = 0; f < FM; ++f) {
          const bf16x8 gt = trfrag<DP>(sg + ltr, qb, f, kk), qt = trfrag<DP>(sq + ltr, qb, f, kk);
          va[f] = El<T>::mfma(gt, pb[kk], va[f]);
          ka[f] = El<T>::mfma(qt, db[kk], ka[f]);
        }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  while (c < tend) {
    const int cn = tile_next(it, active);
    const QMeta mt = mn;
    if (cn < tend) {
      fetch(cn, cur ^ 1);
      mn = tile_meta(first + cn % run);
    }
    if ((MOD & 2) && mod.table) {                                       // workgroup-uniform: the next head's table
      const int gu = c / run;
      if (gu != gu_tab) {
        if (gu_tab >= 0) __syncthreads();
        load_table<T>(a, kv * G + gu, tab, tid, NT);
        gu_tab = gu;
        __syncthreads();
      }
    }
    if (kw0 < mt.bmax) {
      bool partial = kw0 + 32 > mt.bmin;
      if (docs) partial |= wneg | (wdmin != wdmax) | (mt.dmin != mt.dmax) | (mt.neg != 0) | (mt.dmin != wdmin);
      math(__builtin_amdgcn_readfirstlane(partial));
    }
    if (cn < tend) landed(cn, cur ^ 1, mn.bmin <= 0);
    cur ^= 1;
    c = cn;
  }
  if (a.to_part) {
    const long long block = ((long long)y * a.wgs + w) * NW + wave;       // of 32 keys
    store_part<FM>(a.part + block * (64 * DP), ka, lane, true);
    store_part<FM>(a.part + block * (64 * DP) + 32 * DP, va, lane, true);
  } else {
    store_row<T, FM>((bf16_t*)a.p.dk.ptr + op_base(a.p.dk, b) + (long long)key * a.p.dk.sstride + (long long)kv * D, ka, a.p.scale, hi, D, own);
    store_row<T, FM>((bf16_t*)a.p.dv.ptr + op_base(a.p.dv, b) + (long long)key * a.p.dv.sstride + (long long)kv * D, va, 1.f, hi, D, own);
  }
}

// dK, dV = sum of the partial sums of the splits and of the batches that share a K / V head, in order: one wave per 32 keys, 32 columns and side
// (67 MB of partial sums in 13.6 us, 4.9 TB/s)
template <typename T, int DP>
__global__ __launch_bounds__(64) void attn_mod_dkdv_join_kernel(const Args a) {
  constexpr int FM = DP / 32, NW = DP == 128 ? 8 : 4, KEYS = 32 * NW;
  const int lane = threadIdx.x, hi = lane >> 5, D = a.p.D, share = a.p.kv_share, KV = a.p.kv_heads;
  const int f = blockIdx.x % FM, side = blockIdx.x / FM % 2;
  const int blk = blockIdx.x / (2 * FM), wave = blk % NW, ktile = blk / NW % a.ntile, yk = blk / NW / a.ntile;
  const int b0 = yk / KV * share, kv = yk % KV;
  const int key = ktile * KEYS + wave * 32 + (lane & 31);
  const int tiles = (a.M + TILE - 1) / TILE * (a.p.heads / KV / a.gp), runs = kv_runs(a, ktile, KEYS, tiles);
  int w0 = 0;
  for (int k = 0; k < ktile; ++k) w0 += kv_runs(a, k, KEYS, tiles);
  f32x16 acc[1];
#pragma unroll
  for (int e = 0; e < 16; ++e) acc[0][e] = 0.f;
  for (int b = b0; b < min(b0 + share, a.p.nbatch); ++b) {
#pragma unroll 4
    for (int s = 0; s < runs; ++s) {
      const float* p = a.part + (((long long)(b * KV + kv) * a.wgs + w0 + s) * NW + wave) * (64 * DP) + side * 32 * DP + (f * 256 + lane) * 4;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 v = *(const f32x4*)(p + g * 256);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[0][4 * g + e] += v[e];
      }
    }
  }
  const T2VAttnOperand& o = side ? a.p.dv : a.p.dk;
  bf16_t* op = (bf16_t*)o.ptr + op_base(o, b0) + (long long)key * o.sstride + (long long)kv * D + 32 * f;
  store_row<T, 1>(op, acc, side ? 1.f : a.p.scale, hi, D - 32 * f, key < a.p.Sk);
}

// ------------------------------------------------------------------------------------------------ host
struct Layout {
  Args a;
  int dp;
  int fwd_tiles, fwd_splits, dq_tiles, dq_splits, kv_tiles;
  bool kv_split, meta;
  long long o_qmeta, o_kmeta, o_qorder, o_korder, meta_bytes, o_part, o_ml, o_bias, bytes;
  bool order;
};

long long align256(long long n) { return (n + 255) & ~255ll; }

int check_mod(const char* fn, const T2VAttnMod* p, bool bwd) {
  T2V_CHECK_ARG(p && p->nbatch > 0 && p->heads > 0 && p->kv_heads > 0 && p->Sq > 0 && p->Sk > 0, "%s: bad dims", fn);
  T2V_CHECK_ARG(p->heads % p->kv_heads == 0, "%s: %d heads cannot share %d key / value heads evenly", fn, p->heads, p->kv_heads);
  T2V_CHECK_ARG(p->D >= 8 && p->D <= 128 && p->D % 8 == 0, "%s: the head dim must be a multiple of 8 up to 128 (got %d)", fn, p->D);
  T2V_CHECK_ARG(p->dtype == 0 || p->dtype == 1, "%s: bf16 (0) or fp16 (1) operands are wanted", fn);
  T2V_CHECK_ARG(p->scale >= 1e-15f && p->scale <= 1e6f && (p->softcap == 0.f || (p->softcap >= 1e-6f && p->softcap <= 1e4f)),
                "%s: the scale must lie in [1e-15, 1e6], the cap be 0 or lie in [1e-6, 1e4]", fn);
  T2V_CHECK_ARG((p->q_docs == nullptr) == (p->kv_docs == nullptr), "%s: documents of queries and keys come together", fn);
  T2V_CHECK_ARG(!p->prefix || p->causal, "%s: a prefix opens a causal mask: set causal", fn);
  T2V_CHECK_ARG(!p->bias || (p->radius >= 0 && p->radius <= 1024), "%s: the table's radius must be 0..1024 (got %d)", fn, p->radius);
  T2V_CHECK_ARG((long long)p->Sq * p->heads < (1ll << 26) && p->Sk < (1 << 26), "%s: too many rows (Sq * heads and Sk below 2^26)", fn);
  T2V_CHECK_ARG((long long)p->Sq * (p->heads / p->kv_heads) * (p->heads / p->kv_heads) < (1ll << 32),
                "%s: too many query heads of one key / value head (Sq * (heads / kv_heads)^2 below 2^32)", fn);      // (Args::magic is exact below it)
  T2V_CHECK_ARG((long long)p->nbatch * p->heads < (1 << 20), "%s: nbatch * heads below 2^20 is wanted", fn);
  const T2VAttnOperand* ops[] = {&p->q, &p->k, &p->v, &p->o, &p->d_o, &p->dq, &p->dk, &p->dv};
  const char* names[] = {"q", "k", "v", "o", "d_o", "dq", "dk", "dv"};
  for (int i = 0; i < (bwd ? 8 : 4); ++i) {
    const T2VAttnOperand& o = *ops[i];
    if (i >= 6 && !p->dk.ptr && !p->dv.ptr) continue;                   // no gradient of keys and values is asked for
    T2V_CHECK_ARG(o.ptr && o.bdiv > 0 && ((uintptr_t)o.ptr & 15) == 0 && o.sstride % 8 == 0 && o.bstride_hi % 8 == 0 && o.bstride_lo % 8 == 0 &&
                      o.sstride >= 0 && o.sstride < (1ll << 31),
                  "%s: operand %s: 16-byte aligned rows, less than 2^31 elements apart, are wanted (ptr %p, row stride %lld)", fn, names[i], o.ptr, o.sstride);
  }
  T2V_CHECK_ARG(((uintptr_t)p->o_rest & 15) == 0, "%s: o_rest must be 16-byte aligned", fn);
  T2V_CHECK_ARG(!bwd || (p->lse && p->delta), "%s: lse and delta are required", fn);
  T2V_CHECK_ARG(!bwd || p->kv_share >= 1, "%s: kv_share is the number of batches that share a K / V (1: none do)", fn);
  return T2V_OK;
}

Layout make_layout(const T2VAttnMod* p, bool bwd) {
  Layout L{};
  Args& a = L.a;
  a.p = *p;
  const int G = p->heads / p->kv_heads;
  a.gp = p->bias ? 1 : G;
  a.nunit = p->heads / a.gp;
  a.M = p->Sq * a.gp;
  a.magic = a.gp > 1 ? (unsigned)(((1ull << 32) + a.gp - 1) / a.gp) : 0;
  L.dp = p->D <= 64 ? 64 : 128;
  const long long NU = (long long)p->nbatch * a.nunit;
  L.fwd_tiles = (a.M + 127) / 128;
  L.fwd_splits = 1;
  if (!bwd) {
    // Few workgroups and a long key axis: the keys are split until ~512 workgroups exist, at least four 64-key tiles each (8 steps over up to 16384
    // keys, 16 / 4 heads of 128: 45 us; with 256 or 1024 workgroups 61 and 58).  A little more than one workgroup per CU leaves most CUs with one
    // and a few with two: three splits fill both places about twice (264 workgroups, 6731 keys: 214 -> 173 us, 320: 214 -> 201, 264 causal ones of 2112
    // keys: 53 -> 50; at 400 they lose, 228 -> 246, and below 32 tiles of keys their join takes what they gain).
    const long long wgs = NU * L.fwd_tiles;
    const int kt = (p->Sk + TILE - 1) / TILE;
    if (wgs < 256) {
      const int s = (int)(512 / wgs);
      L.fwd_splits = s < kt / 4 ? s : kt / 4;
      if (L.fwd_splits < 1) L.fwd_splits = 1;
    } else if (wgs <= 1024 / 3 && kt >= 32 && !p->q_docs) {
      L.fwd_splits = 3;
    }
  }
  L.dq_tiles = (a.M + 127) / 128;
  const int keys = L.dp == 64 ? 128 : 256;      // of a dK / dV workgroup
  L.kv_tiles = (p->Sk + keys - 1) / keys;
  L.meta = p->q_docs || (p->prefix && p->prefix_per_query);
  a.chunk = 1 << 30;
  if (bwd) {
    // Few K / V heads and keys: the row tiles are split.  A split costs what about four row tiles do (its prologue, and 256 KB of partial sums
    // written and read), and one workgroup runs per CU (two at DP = 64): the run length is the one with the least rounds * (length + 4).
    const long long tiles = (long long)((a.M + TILE - 1) / TILE) * (G / a.gp), heads = (long long)p->nbatch * p->kv_heads;
    const int slots = L.dp == 64 ? 512 : 256;
    a.qmeta = L.meta ? (const QMeta*)1 : nullptr;                          // (kv_runs asks whether it is there)
    // (with documents most tiles are passed over: only very few workgroups are worth a split)
    if (heads * L.kv_tiles < (L.meta ? slots / 4 : 2 * slots) && tiles > 4 && tiles < (1 << 24)) {
      double best = 1e30;
      int chunk = (int)tiles;
      for (long long c = tiles; c >= 4 && c * 16 >= tiles; c = c > 64 ? c * 15 / 16 : c - 1) {
        long long wgs = 0;
        a.chunk = (int)c;
        for (int k = 0; k < L.kv_tiles; ++k) wgs += kv_runs(a, k, keys, (int)tiles);
        const double cost = (double)((heads * wgs + slots - 1) / slots) * (double)(c + (c < tiles ? 4 : 0));
        if (cost < best) {
          best = cost;
          chunk = (int)c;
        }
      }
      a.chunk = chunk;
      L.kv_split = chunk < tiles;
    }
    a.wgs = L.kv_tiles;
    if (L.kv_split) {
      a.wgs = 0;
      for (int k = 0; k < L.kv_tiles; ++k) a.wgs += kv_runs(a, k, keys, (int)tiles);
    }
  }
  long long at = 0;
  if (L.meta) {
    L.o_qmeta = at;
    at = align256(at + (long long)sizeof(QMeta) * p->nbatch * ((a.M + TILE - 1) / TILE));
    L.o_kmeta = at;
    at = align256(at + (long long)sizeof(KMeta) * p->nbatch * ((p->Sk + TILE - 1) / TILE));
    // sorted where a launch is a few workgroups per CU (more than a few are dealt out evenly by their number) and sorting is short
    const int key_tiles = (p->Sk + (L.dp == 64 ? 127 : 255)) / (L.dp == 64 ? 128 : 256);
    const long long nq = 2ll * p->nbatch * L.dq_tiles, nk = 2ll * p->nbatch * key_tiles;
    L.order = p->q_docs && nq <= ORDER_MAX && nk <= ORDER_MAX && nq * a.nunit > 512 && (long long)p->nbatch * (a.M + TILE) <= ORDER_TILES * TILE &&
              (long long)p->nbatch * (p->Sk + TILE) <= ORDER_TILES * TILE;
    if (L.order) {
      L.o_qorder = at;
      at = align256(at + 4 * nq);
      L.o_korder = at;
      at = align256(at + 4 * nk);
    }
  }
  L.meta_bytes = at;
  at = 0;
  if (!bwd && L.fwd_splits > 1) {
    L.o_part = at;
    at = align256(at + 4ll * L.fwd_splits * NU * L.fwd_tiles * 128 * L.dp);
    L.o_ml = at;
    at = align256(at + 8ll * L.fwd_splits * NU * L.fwd_tiles * 128);
  }
  if (bwd) {
    // dQ: as the forward pass where there are few workgroups (backward of 4096 tokens, 2 heads of 64: 129 -> 83 us, 2500 causal, 4 heads of 128: 128 -> 94,
    // 1024 tokens, 10 heads of 64: 58 -> 54)
    const long long wgs = NU * L.dq_tiles;
    const int kt = (p->Sk + TILE - 1) / TILE;
    L.dq_splits = 1;
    if (wgs < 256 && !L.order) {
      const int s = (int)(512 / wgs);
      L.dq_splits = s < kt / 4 ? s : kt / 4;
      if (L.dq_splits < 1) L.dq_splits = 1;
    }
    // (the partial sums of dQ are joined before those of dK / dV are written)
    const long long q = L.dq_splits > 1 ? 4ll * L.dq_splits * wgs * 128 * L.dp : 0;
    const long long kv = L.kv_split || p->kv_share > 1 ? 8ll * p->nbatch * p->kv_heads * a.wgs * keys * L.dp : 0;
    L.o_part = at;
    at = align256(at + (q > kv ? q : kv));
    if (p->dbias) {
      L.o_bias = at;
      at = align256(at + 4ll * p->nbatch * L.dq_tiles * (L.order ? 2 : L.dq_splits) * p->heads * (2 * p->radius + 1));
    }
  }
  L.bytes = at;
  char* w = (char*)p->meta;
  a.qmeta = L.meta ? (const QMeta*)(w + L.o_qmeta) : nullptr;
  a.kmeta = L.meta ? (const KMeta*)(w + L.o_kmeta) : nullptr;
  a.qorder = L.order ? (const int*)(w + L.o_qorder) : nullptr;
  a.korder = L.order && !L.kv_split && p->kv_share <= 1 ? (const int*)(w + L.o_korder) : nullptr;
  a.lsum = p->lse && (p->slopes || p->bias) ? p->lse + (long long)p->nbatch * p->heads * p->Sq : nullptr;
  w = (char*)p->workspace;
  a.part = (float*)(w + L.o_part);
  a.part_ml = (float*)(w + L.o_ml);
  a.part_bias = (float*)(w + L.o_bias);
  return L;
}

size_t smem_bytes(const Layout& L, int tables, bool kv) {
  if (kv) {
    const size_t tab = L.a.p.bias ? 4 * ((2 * (size_t)L.a.p.radius + 1 + 3) / 4 * 4) : 0;
    return (L.dp == 64 ? 2 * sizeof(Stage<64>) : 2 * sizeof(Stage<128>) + 4 * sizeof(Stage<128>) / 2) + 2 * INFO * TILE * 4 + tab;
  }
  return 2 * (L.dp == 64 ? sizeof(Stage<64>) : sizeof(Stage<128>)) + 2 * TILE * 4 + 64 + (L.a.p.bias ? tables * 4 * (2 * (size_t)L.a.p.radius + 1) : 0);
}
template <typename K>
int launch(int which, K kern, long long grid, size_t smem, hipStream_t st, const Args& a, int threads = 256) {
  if (smem > 64 * 1024) {
    const hipError_t e = hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != hipSuccess) {
      t2v_set_error("t2v_attn_mod: %zu bytes of shared memory: %s", smem, hipGetErrorString(e));
      return T2V_ELAUNCH;
    }
  }
  t2v_launch_timed(which, kern, dim3((unsigned)grid), dim3(threads), (unsigned)smem, st, a);
  return T2V_OK;
}
// f(integral constant MOD)
template <typename F>
int with_mod(const T2VAttnMod& p, F f) {
  const bool bias = p.slopes || p.bias;
  if (p.softcap > WIDE_CAP) return bias ? f(std::integral_constant<int, 7>()) : f(std::integral_constant<int, 5>());
  if (p.softcap > 0.f) return bias ? f(std::integral_constant<int, 3>()) : f(std::integral_constant<int, 1>());
  return bias ? f(std::integral_constant<int, 2>()) : f(std::integral_constant<int, 0>());
}

// the rank at which the order turns: where all workgroups are resident, two on some CUs, the 256 longest come first
int fold(const Layout& L, int tiles, int splits) {
  const long long row = (long long)L.a.p.nbatch * L.a.nunit * splits, wgs = row * tiles;
  return L.a.p.causal && wgs > 256 && wgs <= 512 ? (int)((256 + row - 1) / row) : 1 << 30;
}

template <typename T, int DP>
int run_fwd(Layout& L, hipStream_t st) {
  Args& a = L.a;
  a.ntile = L.fwd_tiles;
  a.splits = L.fwd_splits;
  a.fold = fold(L, L.fwd_tiles, L.fwd_splits);
  const long long grid = (long long)a.p.nbatch * a.nunit * L.fwd_tiles * L.fwd_splits * (a.qorder ? 2 : 1);
  const size_t sm = smem_bytes(L, 1, false);
  const int which = L.fwd_splits > 1 ? 1 : 3;
  const int e = with_mod(a.p, [&](auto mod) { return launch(which, attn_mod_fwd_kernel<T, DP, decltype(mod)::value>, grid, sm, st, a); });
  if (e) return e;
  T2V_CHECK_LAUNCH();
  if (L.fwd_splits > 1) {
    const long long blocks = (long long)a.p.nbatch * a.nunit * a.ntile * 4 * (DP / 32);
    if (a.splits > 8) T2V_LAUNCH_LAST((attn_mod_join_kernel<T, DP, 8>), dim3((unsigned)blocks), dim3(512), 0, st, a);
    else T2V_LAUNCH_LAST((attn_mod_join_kernel<T, DP, 1>), dim3((unsigned)blocks), dim3(64), 0, st, a);
    T2V_CHECK_LAUNCH();
  }
  return T2V_OK;
}
template <typename T, int DP>
int run_bwd(Layout& L, hipStream_t st) {
  Args& a = L.a;
  a.ntile = L.dq_tiles;
  a.splits = L.dq_splits;
  a.fold = fold(L, L.dq_tiles, L.dq_splits);
  const size_t sm = smem_bytes(L, a.p.dbias ? 5 : 1, false);
  const long long gq = (long long)a.p.nbatch * a.nunit * L.dq_tiles * L.dq_splits * (a.qorder ? 2 : 1);
  const bool kv = a.p.dk.ptr != nullptr;
  int which = kv || a.splits > 1 || a.p.dbias ? 1 : 3;
  int e = with_mod(a.p, [&](auto mod) { return launch(which, attn_mod_dq_kernel<T, DP, decltype(mod)::value>, gq, sm, st, a); });
  if (e) return e;
  T2V_CHECK_LAUNCH();
  if (a.splits > 1) {
    const long long blocks = (long long)a.p.nbatch * a.nunit * a.ntile * 4 * (DP / 32);
    t2v_launch_timed(kv || a.p.dbias ? 0 : 2, attn_mod_dq_join_kernel<T, DP>, dim3((unsigned)blocks), dim3(64), 0, st, a);
    T2V_CHECK_LAUNCH();
  }
  if (a.p.dbias) {
    const long long n = (long long)a.p.heads * (2 * a.p.radius + 1);
    t2v_launch_timed(kv ? 0 : 2, attn_mod_dbias_kernel<T>, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, a);
    T2V_CHECK_LAUNCH();
  }
  if (!kv) return T2V_OK;
  a.ntile = L.kv_tiles;
  const long long gk = (long long)a.p.nbatch * a.p.kv_heads * a.wgs * (a.korder ? 2 : 1);
  const size_t smk = smem_bytes(L, 1, true);
  a.to_part = L.kv_split || a.p.kv_share > 1;
  which = a.to_part ? 0 : 2;
  e = with_mod(a.p, [&](auto mod) { return launch(which, attn_mod_dkdv_kernel<T, DP, decltype(mod)::value>, gk, smk, st, a, DP == 128 ? 512 : 256); });
  if (e) return e;
  T2V_CHECK_LAUNCH();
  if (a.to_part) {
    const long long blocks = (long long)((a.p.nbatch + a.p.kv_share - 1) / a.p.kv_share) * a.p.kv_heads * a.ntile * (DP == 128 ? 8 : 4) * 2 * (DP / 32);
    T2V_LAUNCH_LAST((attn_mod_dkdv_join_kernel<T, DP>), dim3((unsigned)blocks), dim3(64), 0, st, a);
    T2V_CHECK_LAUNCH();
  }
  return T2V_OK;
}
int check_grids(const char* fn, const Layout& L, bool bwd) {
  // the largest launches, in threads: rows (256 a tile, two entries a tile with a work list), the joins (512 or 64 per 32 x 32 block), dK / dV (512 or 256)
  const long long row_wgs = (long long)L.a.p.nbatch * L.a.nunit * L.fwd_tiles * L.fwd_splits, join = 4 * (L.dp / 32) * 512ll;
  const long long kv_wgs = bwd ? (long long)L.a.p.nbatch * L.a.p.kv_heads * L.a.wgs * (L.dp == 64 ? 1 : 2) : 0;
  T2V_CHECK_ARG(row_wgs * (join > 512 ? join : 512) < (1ll << 32) && kv_wgs * (2 * join) < (1ll << 32), "%s: too many workgroups (%lld, %lld)", fn, row_wgs, kv_wgs);
  return T2V_OK;
}
int run(const char* fn, const T2VAttnMod* p, bool bwd, hipStream_t st) {
  if (int e = check_mod(fn, p, bwd)) return e;
  Layout L = make_layout(p, bwd);
  T2V_CHECK_ARG(L.bytes == 0 || (p->workspace && ((uintptr_t)p->workspace & 255) == 0 && p->workspace_bytes >= L.bytes),
                "%s: a 256-byte aligned workspace of %lld bytes is wanted (got %p, %lld)", fn, L.bytes, p->workspace, p->workspace_bytes);
  if (int e = check_grids(fn, L, bwd)) return e;
  T2V_CHECK_ARG(!L.meta || (p->meta && ((uintptr_t)p->meta & 255) == 0 && p->meta_bytes >= L.meta_bytes),
                "%s: documents and prefixes per query want a 256-byte aligned meta buffer of %lld bytes (got %p, %lld)", fn, L.meta_bytes, p->meta,
                p->meta_bytes);
  if (L.meta && !p->meta_ready) {
    const int nq = (L.a.M + TILE - 1) / TILE, nk = (p->Sk + TILE - 1) / TILE;
    T2V_CHECK_ARG(p->nbatch <= 65535, "%s: at most 65535 batches with documents or one prefix per query", fn);
    hipLaunchKernelGGL(attn_mod_meta_kernel, dim3(nq + nk, p->nbatch), dim3(64), 0, st, L.a, (QMeta*)L.a.qmeta, (KMeta*)L.a.kmeta, nq, nk);
    T2V_CHECK_LAUNCH();
    if (L.order) {
      const int keys = L.dp == 64 ? 128 : 256;
      char* w = (char*)p->meta;
      hipLaunchKernelGGL(attn_mod_order_kernel, dim3(2), dim3(1024), 0, st, L.a, (int*)(w + L.o_qorder), (int*)(w + L.o_korder), L.dq_tiles,
                         (p->Sk + keys - 1) / keys, keys);
      T2V_CHECK_LAUNCH();
    }
  }
  if (p->dtype == 0) {
    if (L.dp == 64) return bwd ? run_bwd<bf16_t, 64>(L, st) : run_fwd<bf16_t, 64>(L, st);
    return bwd ? run_bwd<bf16_t, 128>(L, st) : run_fwd<bf16_t, 128>(L, st);
  }
  if (L.dp == 64) return bwd ? run_bwd<_Float16, 64>(L, st) : run_fwd<_Float16, 64>(L, st);
  return bwd ? run_bwd<_Float16, 128>(L, st) : run_fwd<_Float16, 128>(L, st);
}
}  // namespace

extern "C" long long t2v_attn_mod_workspace(const T2VAttnMod* p, int backward) {
  if (check_mod("t2v_attn_mod_workspace", p, false)) return -1;
  const Layout L = make_layout(p, backward != 0);
  return check_grids("t2v_attn_mod_workspace", L, backward != 0) ? -1 : L.bytes;
}
extern "C" long long t2v_attn_mod_meta_bytes(const T2VAttnMod* p) {
  if (check_mod("t2v_attn_mod_meta_bytes", p, false)) return -1;
  return make_layout(p, false).meta_bytes;
}
extern "C" int t2v_attn_mod_fwd(const T2VAttnMod* p, t2v_stream_t stream) { return run("t2v_attn_mod_fwd", p, false, (hipStream_t)stream); }
extern "C" int t2v_attn_mod_bwd(const T2VAttnMod* p, t2v_stream_t stream) { return run("t2v_attn_mod_bwd", p, true, (hipStream_t)stream); }
