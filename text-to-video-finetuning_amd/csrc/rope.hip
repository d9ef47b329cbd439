// rope.hip — rotary positions with several axes, and the per-head norm of queries and keys in the same pass (forward + backward).
//
//   y = R(pos) (w * xhat + b),   xhat = x r (RMS: r = (mean x^2 + eps)^-1/2) or (x - mean) r (layer norm), or y = R(pos) x
//   backward, d = R(pos)^T dy, e = d w:   dx = r (e - [mean e] - xhat mean(e xhat)),  dw = sum d xhat,  db = sum d
// R turns pair p of a head (columns 2p, 2p+1, or p, p + rot/2) by pos[axis(p)] * freq(p).  The angle is formed in 64 bits, in turns
// (multiples of 2 pi are dropped exactly at positions of 10^6 and beyond), and rounded to 32 bits only inside half a turn.
//
// HBM-bound: an element is read once and written once (backward with a norm: two reads).  A group of LPH lanes owns one row of one
// block of heads, eight columns per lane; the angles of a row are formed once and used for all heads of the block, and UNROLL heads
// are in flight per lane.  The statistics live in registers (two passes over them for the layer norm, none over memory) and are
// recomputed in the backward pass, which saves their round trip.  Parameter gradients: per-lane fp32 sums over the rows a group
// visits, one fixed-order sum over the groups of a workgroup in LDS, one partial row per workgroup, one fixed-order reduction
// kernel: no atomics, repeated runs are bit-equal.
// Measured, bf16, norm + rotation of 69120 rows, 2 x 20 heads of 64: forward 161 us (4.4 TB/s; a large copy reaches 4.9), forward and backward
// 400 us (1.77 GB: 4.4 TB/s with the gaps between launches).  Few rows are launch-bound: 8 rows of 16 heads of 128 take 3.9 us a launch in a captured chain,
// 5.3 us traced singly.
#include "common.h"

namespace {

constexpr int UNROLL = 4;

struct RopeSide {
  const void* x;
  long long ldx;
  const void* dy;
  long long lddy;
  void* y;
  long long ldy;
  int heads;
  const float* w;
  const float* b;
};
struct RopeArgs {
  RopeSide s[2];
  long long rows;
  int D, rot, naxes, nq, hb;             // nq: blocks of heads of the first side; hb: heads per block
  const void* pos;
  long long ldpos;
  int pos_type;
  int dims[4];
  double pw[4][7];                       // of each axis: r, r^2, r^4, ... r^64, the ratio of one frequency to the one before it
  double first[4];                       // frequency of the axis' first pair, in turns per unit of position (scale / 2 pi)
  int shared;
  const double* freqs;
  float eps;
  float* partial;
};

template <typename T>
struct Quad;
template <>
struct Quad<bf16_t> {
  typedef uint2 V;
  static __device__ __forceinline__ void get(const V& v, float* o) {
    o[0] = __uint_as_float(v.x << 16);
    o[1] = __uint_as_float(v.x & 0xffff0000u);
    o[2] = __uint_as_float(v.y << 16);
    o[3] = __uint_as_float(v.y & 0xffff0000u);
  }
  static __device__ __forceinline__ V put(const float* o) { return uint2{pack2bf(o[0], o[1]), pack2bf(o[2], o[3])}; }
};
template <>
struct Quad<_Float16> {
  typedef __attribute__((ext_vector_type(4))) _Float16 V;
  static __device__ __forceinline__ void get(const V& v, float* o) {
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = (float)v[e];
  }
  static __device__ __forceinline__ V put(const float* o) { return V{(_Float16)o[0], (_Float16)o[1], (_Float16)o[2], (_Float16)o[3]}; }
};
template <>
struct Quad<float> {
  typedef float4 V;
  static __device__ __forceinline__ void get(const V& v, float* o) {
    o[0] = v.x;
    o[1] = v.y;
    o[2] = v.z;
    o[3] = v.w;
  }
  static __device__ __forceinline__ V put(const float* o) { return float4{o[0], o[1], o[2], o[3]}; }
};

template <int LPH>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = LPH / 2; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

// the lane's four frequencies in turns per unit of position, and the axis of each pair.  theta^(-2 i / d) = r^i comes from the bits of i
// and the host's powers of r in 64 bits: at most ten products (a relative error of 1e-15, at 10^6 turns 1e-9 of a turn) in the place of
// four 64-bit exponentials, which took longer than the rest of a launch of few rows (5.4 -> 3.6 us at 8 rows).
__device__ __forceinline__ void lane_freqs(const RopeArgs& p, int c, double (&f)[4], int (&ax)[4]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int pr = 4 * c + e;
    int a = 0, first = 0, end = p.dims[0] / 2;
#pragma unroll
    for (int n = 1; n < 4; ++n)
      if (n < p.naxes) {
        const bool on = pr >= end;
        a = on ? n : a;
        first = on ? end : first;
        end += p.dims[n] / 2;
      }
    ax[e] = a;
    if (p.freqs) {
      f[e] = pr < p.rot / 2 ? p.freqs[pr] * p.first[a] : 0.0;
    } else {
      const int i = p.shared ? pr : pr - first;
      double v = p.first[a];
#pragma unroll
      for (int n = 0; n < 7; ++n) v *= (i >> n) & 1 ? p.pw[a][n] : 1.0;
      f[e] = v;
    }
  }
}
__device__ __forceinline__ double load_pos(const RopeArgs& p, long long row, int a) {
  const long long at = row * p.ldpos + a;
  return p.pos_type == 0 ? (double)((const int*)p.pos)[at] : p.pos_type == 1 ? (double)((const long long*)p.pos)[at] : (double)((const float*)p.pos)[at];
}

template <bool HALF>
__device__ __forceinline__ void turn(float (&v)[8], const float (&cs)[4], const float (&sn)[4], bool turns, float sign) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int i = HALF ? e : 2 * e, j = HALF ? e + 4 : 2 * e + 1;
    // (columns behind the turned ones carry cos = 1, sin = 0 in the interleaved form; the halves form keeps its chunk as it is)
    const float a = v[i], b = v[j], s = sn[e] * sign;
    v[i] = turns ? fmaf(a, cs[e], -b * s) : a;
    v[j] = turns ? fmaf(b, cs[e], a * s) : b;
  }
}

// NORM 0 none, 1 RMS, 2 layer norm.  BWD: x is read only where NORM needs it.
template <typename T, int NORM, bool HALF, bool BWD, int LPH>
__global__ __launch_bounds__(256) void rope_kernel(const RopeArgs p) {
  typedef typename Quad<T>::V V;
  __shared__ float sred[BWD && NORM ? 2 * 8 * 256 : 1];
  const int tid = threadIdx.x, c = tid % LPH;
  constexpr int GPB = 256 / LPH;
  const bool second = (int)blockIdx.y >= p.nq;                       // workgroup-uniform
  const RopeSide& s = p.s[second ? 1 : 0];
  const int h0 = ((int)blockIdx.y - (second ? p.nq : 0)) * p.hb, h1 = min(h0 + p.hb, s.heads);
  const int D = p.D, R = p.rot;
  const bool live = c < D / 8, turns = c < R / 8;
  // the lane's two quads of columns
  const int ca = !live ? 0 : (HALF && turns) ? 4 * c : 8 * c, cb = !live ? 4 : (HALF && turns) ? R / 2 + 4 * c : 8 * c + 4;
  double f[4];
  int ax[4];
  lane_freqs(p, c, f, ax);
  float w[8], b[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int col = e < 4 ? ca + e : cb + e - 4;
    w[e] = NORM && s.w ? s.w[col] : 1.f;
    b[e] = NORM && s.b && !BWD ? s.b[col] : 0.f;
  }
  float dw[8], db[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) dw[e] = db[e] = 0.f;
  const float inv = 1.f / D;
  const long long stride = (long long)gridDim.x * GPB;
  for (long long row0 = (long long)blockIdx.x * GPB; row0 < p.rows; row0 += stride) {
    const long long row = row0 + tid / LPH;
    const bool here = row < p.rows;
    const long long r = here ? row : p.rows - 1;
    float cs[4], sn[4];
    if (turns) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        double t = load_pos(p, r, ax[e]) * f[e];
        t -= rint(t);
        if (sizeof(T) == 2) {
          // the hardware's sine of an angle in turns: at most 1.3e-7 off over a turn (measured), far below half a
          // step of 16 bits (2^-12)
          sn[e] = __builtin_amdgcn_sinf((float)t);
          cs[e] = __builtin_amdgcn_cosf((float)t);
        } else {
          sincospif(2.f * (float)t, &sn[e], &cs[e]);
        }
      }
    }
    for (int h = h0; h < h1; h += UNROLL) {
      V xa[UNROLL], xb[UNROLL], ga[UNROLL], gb[UNROLL];
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) {
        const int hh = min(h + u, h1 - 1);
        if (!BWD || NORM) {
          const T* x = (const T*)s.x + r * s.ldx + (long long)hh * D;
          xa[u] = *(const V*)(x + ca);
          xb[u] = *(const V*)(x + cb);
        }
        if (BWD) {
          const T* g = (const T*)s.dy + r * s.lddy + (long long)hh * D;
          ga[u] = *(const V*)(g + ca);
          gb[u] = *(const V*)(g + cb);
        }
      }
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) {
        if (h + u >= h1) break;                                      // workgroup-uniform
        float v[8], g[8], rs = 1.f;
        if (!BWD || NORM) {
          Quad<T>::get(xa[u], v);
          Quad<T>::get(xb[u], v + 4);
        }
        if (NORM) {
          if (NORM == 2) {
            float m = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) m += v[e];
            m = group_sum<LPH>(live ? m : 0.f) * inv;
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] -= m;
          }
          float q = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) q = fmaf(v[e], v[e], q);
          rs = rsqrtf(group_sum<LPH>(live ? q : 0.f) * inv + p.eps);
        }
        if (!BWD) {
          if (NORM) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = fmaf(v[e] * rs, w[e], b[e]);
          }
          turn<HALF>(v, cs, sn, turns, 1.f);
        } else {
          Quad<T>::get(ga[u], g);
          Quad<T>::get(gb[u], g + 4);
          turn<HALF>(g, cs, sn, turns, -1.f);
          if (NORM) {
            float m1 = 0.f, m2 = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              v[e] *= rs;
              if (here) {
                dw[e] = fmaf(g[e], v[e], dw[e]);
                db[e] += g[e];
              }
              g[e] *= w[e];
              m1 = fmaf(g[e], v[e], m1);
              m2 += g[e];
            }
            m1 = group_sum<LPH>(live ? m1 : 0.f) * inv;
            m2 = NORM == 2 ? group_sum<LPH>(live ? m2 : 0.f) * inv : 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = rs * (g[e] - m2 - v[e] * m1);
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = g[e];
          }
        }
        if (here && live) {
          T* y = (T*)s.y + row * s.ldy + (long long)(h + u) * D;
          *(V*)(y + ca) = Quad<T>::put(v);
          *(V*)(y + cb) = Quad<T>::put(v + 4);
        }
      }
    }
  }
  if (BWD && NORM && p.partial) {                                    // launch-uniform
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      sred[e * 256 + tid] = dw[e];
      sred[(8 + e) * 256 + tid] = db[e];
    }
    __syncthreads();
    float* out = p.partial + ((long long)blockIdx.y * gridDim.x + blockIdx.x) * 2 * D;
    for (int i = tid; i < 16 * LPH; i += 256) {
      const int which = i / (8 * LPH), e = (i / LPH) % 8, l = i % LPH;
      if (l < D / 8) {
        float sum = 0.f;
        for (int gidx = 0; gidx < GPB; ++gidx) sum += sred[(which * 8 + e) * 256 + gidx * LPH + l];
        const bool tl = l < R / 8;
        const int a0 = (HALF && tl) ? 4 * l : 8 * l, b0 = (HALF && tl) ? R / 2 + 4 * l : 8 * l + 4;
        out[which * D + (e < 4 ? a0 + e : b0 + e - 4)] = sum;
      }
    }
  }
}

// out[side][which][col] = sum over the side's partial rows, in order within a slice and over the slices (4 us, a launch)
__global__ __launch_bounds__(1024) void rope_param_reduce_kernel(const float* __restrict__ partial, int D, int n0, int n1, float* dw0,
                                                                 float* db0, float* dw1, float* db1) {
  __shared__ float s[32][33];
  const int side = blockIdx.y >> 1, which = blockIdx.y & 1;
  float* out = side ? (which ? db1 : dw1) : (which ? db0 : dw0);
  if (!out) return;                                                  // workgroup-uniform
  const int col = blockIdx.x * 32 + (threadIdx.x & 31), sl = threadIdx.x >> 5;
  const int first = side ? n0 : 0, n = side ? n1 : n0;
  float a = 0.f;
  if (col < D)
#pragma unroll 4
    for (int r = sl; r < n; r += 32) a += partial[((long long)(first + r) * 2 + which) * D + col];
  s[sl][threadIdx.x & 31] = a;
  __syncthreads();
  if (sl == 0 && col < D) {
    float t = 0.f;
    for (int i = 0; i < 32; ++i) t += s[i][threadIdx.x];
    out[col] = t;
  }
}

struct Plan {
  int lph, gx, hb, nq, nk;
};
// Heads per block of work: as many as leave 1.5 workgroups per CU — a block shares the angles and the per-lane set-up (16384 rows, five heads of
// 64: 7.8 us with all heads in a block, 13.1 us with one; 6669 rows of five fp32 heads: 8.7 against 17.0).  Workgroups are bounded and
// visit several rows: 2048 forward (69120 rows, 2 x 20 heads of 64: 161 us, 172 unbounded; 2 x 8 heads of 128: 113 against 128 us), and 1024
// where each leaves a partial row of parameter gradients (249 us; 337 at 512, where too few loads are in flight, 247 at 2048, whose partial rows cost
// the reduction 3 us more).
Plan rope_plan(const T2VQkRope* p, bool partials) {
  Plan q;
  const int lanes = p->D / 8;
  q.lph = lanes <= 8 ? 8 : lanes <= 16 ? 16 : 32;
  const long long bx = (p->rows * q.lph + 255) / 256;
  for (q.hb = 16; q.hb > 1; q.hb /= 2) {
    const long long blocks = bx * ((p->heads[0] + q.hb - 1) / q.hb + (p->heads[1] + q.hb - 1) / q.hb);
    if (blocks >= 384) break;
  }
  q.nq = (p->heads[0] + q.hb - 1) / q.hb;
  q.nk = (p->heads[1] + q.hb - 1) / q.hb;
  const int most = partials ? 1024 : 2048;
  const long long cap = most / (q.nq + q.nk) > 1 ? most / (q.nq + q.nk) : 1;
  q.gx = (int)(bx < cap ? bx : cap);
  return q;
}

int check_rope(const char* fn, const T2VQkRope* p, bool bwd) {
  T2V_CHECK_ARG(p && p->rows > 0 && p->rows < (1ll << 31) && p->heads[0] > 0 && p->heads[1] >= 0 && p->heads[0] <= 4096 && p->heads[1] <= 4096,
                "%s: bad dims", fn);
  T2V_CHECK_ARG(p->D >= 8 && p->D <= 256 && p->D % 8 == 0, "%s: the head dim must be a multiple of 8 up to 256 (got %d)", fn, p->D);
  T2V_CHECK_ARG(p->dtype >= 0 && p->dtype <= 2 && p->norm >= 0 && p->norm <= 2 && p->style >= 0 && p->style <= 1, "%s: bad dtype / norm / style", fn);
  T2V_CHECK_ARG(p->naxes >= 0 && p->naxes <= 4, "%s: at most four axes (got %d)", fn, p->naxes);
  int rot = 0;
  for (int a = 0; a < p->naxes; ++a) {
    T2V_CHECK_ARG(p->dims[a] > 0 && p->dims[a] % 2 == 0, "%s: axis %d turns %d columns: an even number is wanted", fn, a, p->dims[a]);
    rot += p->dims[a];
  }
  T2V_CHECK_ARG(rot <= p->D && rot % 8 == 0, "%s: the axes turn %d columns: a multiple of 8, at most the head dim %d", fn, rot, p->D);
  T2V_CHECK_ARG(rot == 0 || (p->pos && p->pos_type >= 0 && p->pos_type <= 2 && p->ldpos >= p->naxes), "%s: positions missing", fn);
  T2V_CHECK_ARG(p->freqs || rot == 0 || p->theta > 0, "%s: theta must be positive", fn);
  const int es = p->dtype == 2 ? 4 : 2;
  for (int i = 0; i < 2; ++i) {
    if (p->heads[i] == 0) continue;
    const void* ptrs[3] = {p->x[i], p->y[i], bwd ? p->dy[i] : p->y[i]};
    const long long lds[3] = {p->ldx[i], p->ldy[i], bwd ? p->lddy[i] : p->ldy[i]};
    for (int n = 0; n < 3; ++n) {
      if (n == 0 && bwd && p->norm == 0) continue;
      T2V_CHECK_ARG(ptrs[n] && ((uintptr_t)ptrs[n] & 15) == 0 && (lds[n] * es) % 16 == 0 && lds[n] >= (long long)p->heads[i] * p->D,
                    "%s: operand %d of side %d: 16-byte aligned rows of at least heads * dim elements are wanted (ptr %p, row stride %lld)", fn, n, i,
                    ptrs[n], lds[n]);
    }
  }
  return T2V_OK;
}

RopeArgs rope_args(const T2VQkRope* p, const Plan& q) {
  RopeArgs a{};
  for (int i = 0; i < 2; ++i) {
    a.s[i] = RopeSide{p->x[i], p->ldx[i], p->dy[i], p->lddy[i], p->y[i], p->ldy[i], p->heads[i], p->w[i], p->b[i]};
  }
  a.rows = p->rows;
  a.D = p->D;
  a.naxes = p->naxes;
  for (int n = 0; n < p->naxes; ++n) {
    a.rot += p->dims[n];
    a.dims[n] = p->dims[n];
  }
  for (int n = 0; n < p->naxes; ++n) {
    a.first[n] = p->scale[n] * 0.15915494309189533577;
    const double step = p->freqs ? 0.0 : -2.0 * log2(p->theta) / (p->shared ? a.rot : p->dims[n]);
    for (int k = 0; k < 7; ++k) a.pw[n][k] = exp2(step * (1 << k));
  }
  a.nq = q.nq;
  a.hb = q.hb;
  a.pos = p->pos;
  a.ldpos = p->ldpos;
  a.pos_type = p->pos_type;
  a.shared = p->shared;
  a.freqs = p->freqs;
  a.eps = p->eps;
  return a;
}

template <typename T, int NORM, bool HALF, bool BWD>
void go_lph(const RopeArgs& a, const Plan& q, bool last, hipStream_t st) {
  const dim3 grid(q.gx, q.nq + q.nk);
  const int which = last ? 3 : 1;
  if (q.lph == 8) t2v_launch_timed(which, rope_kernel<T, NORM, HALF, BWD, 8>, grid, dim3(256), 0, st, a);
  else if (q.lph == 16) t2v_launch_timed(which, rope_kernel<T, NORM, HALF, BWD, 16>, grid, dim3(256), 0, st, a);
  else t2v_launch_timed(which, rope_kernel<T, NORM, HALF, BWD, 32>, grid, dim3(256), 0, st, a);
}
template <typename T, bool BWD>
void go(const T2VQkRope* p, const RopeArgs& a, const Plan& q, bool last, hipStream_t st) {
  const bool half = p->style == 1;
  if (p->norm == 0) half ? go_lph<T, 0, true, BWD>(a, q, last, st) : go_lph<T, 0, false, BWD>(a, q, last, st);
  else if (p->norm == 1) half ? go_lph<T, 1, true, BWD>(a, q, last, st) : go_lph<T, 1, false, BWD>(a, q, last, st);
  else half ? go_lph<T, 2, true, BWD>(a, q, last, st) : go_lph<T, 2, false, BWD>(a, q, last, st);
}
template <bool BWD>
void go_type(const T2VQkRope* p, const RopeArgs& a, const Plan& q, bool last, hipStream_t st) {
  if (p->dtype == 0) go<bf16_t, BWD>(p, a, q, last, st);
  else if (p->dtype == 1) go<_Float16, BWD>(p, a, q, last, st);
  else go<float, BWD>(p, a, q, last, st);
}
bool wants_partials(const T2VQkRope* p) { return p->norm && (p->dw[0] || p->db[0] || p->dw[1] || p->db[1]); }
}  // namespace

extern "C" long long t2v_qk_rope_bwd_floats(const T2VQkRope* p) {
  if (check_rope("t2v_qk_rope_bwd_floats", p, true)) return -1;
  if (!wants_partials(p)) return 0;
  const Plan q = rope_plan(p, true);
  return (long long)q.gx * (q.nq + q.nk) * 2 * p->D;
}

extern "C" int t2v_qk_rope_fwd(const T2VQkRope* p, t2v_stream_t stream) {
  if (int e = check_rope("t2v_qk_rope_fwd", p, false)) return e;
  const Plan q = rope_plan(p, false);
  const RopeArgs a = rope_args(p, q);
  go_type<false>(p, a, q, true, (hipStream_t)stream);
  T2V_CHECK_LAUNCH();
  return T2V_OK;
}

extern "C" int t2v_qk_rope_bwd(const T2VQkRope* p, t2v_stream_t stream) {
  if (int e = check_rope("t2v_qk_rope_bwd", p, true)) return e;
  const bool pg = wants_partials(p);
  T2V_CHECK_ARG(!pg || p->workspace, "t2v_qk_rope_bwd: parameter gradients need a workspace of t2v_qk_rope_bwd_floats() floats");
  const Plan q = rope_plan(p, pg);
  RopeArgs a = rope_args(p, q);
  a.partial = pg ? p->workspace : nullptr;
  go_type<true>(p, a, q, !pg, (hipStream_t)stream);
  T2V_CHECK_LAUNCH();
  if (pg) {
    T2V_LAUNCH_LAST(rope_param_reduce_kernel, dim3((p->D + 31) / 32, 4), dim3(1024), 0, (hipStream_t)stream, (const float*)p->workspace,
                    p->D, q.gx * q.nq, q.gx * q.nk, p->dw[0], p->db[0], p->dw[1], p->db[1]);
    T2V_CHECK_LAUNCH();
  }
  return T2V_OK;
}
