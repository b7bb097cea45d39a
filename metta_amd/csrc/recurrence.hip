// recurrence.hip -- gated linear recurrence over segments, its gradients and its one-step form for gfx950
// (mg_gated_recurrence, mg_gated_recurrence_backward).
//
// Per row and column, with a = sigmoid(gate):   h[t] = a[t] * (resets[t] ? 0 : h[t-1]) + (1 - a[t]) * x[t]
// and backwards, with d[t] = dh[t] + v[t+1] and v[t] = (resets[t] ? 0 : a[t] * d[t]):
//   dx[t] = (1 - a[t]) d[t]      dgate[t] = d[t] (h_before[t] - x[t]) a[t] (1 - a[t])      dstate = v[0]
//
// x, gate, h and their gradients are f32, bf16 or f16; the state, the products along time and the running gradient are
// f32 throughout, h and the gradients are rounded once when they are stored.
//
// Both directions are first-order recurrences s -> p s + q, which compose: a stretch of steps is the pair (P, Q) of its
// composition.  Columns are independent, so with many of them a thread walks its columns through all of time; with few,
// the waves of a block take REC_L steps each, compose them, exchange the pairs through LDS and go on from the state
// that enters them (tiles of REC_W * REC_L steps); with fewer still, time is cut over blocks, whose pairs a first
// launch leaves in a workspace.  The backward pass recomputes h inside a stretch from the state entering it, which the
// forward pass kept in f32 every REC_L steps ("marks"; an f32 h is its own): cheaper than reading h again, and exact.
#include <hip/hip_runtime.h>

#include <string>
#include <type_traits>

#include "../../include/mettagrid_hip.h"

#define REC_L MG_RECURRENCE_MARK_STEPS  // steps a thread holds in registers at a time
#define REC_W 8                         // waves that share a tile of time
#define REC_TILE (REC_W * REC_L)

extern int mg_fail_msg(const std::string& m);  // mettagrid_hip.hip: sets mg_last_error(), returns 1

// VEC adjacent columns of a tensor, moved as one
template <typename T, int VEC> struct RecVec { typedef T type __attribute__((ext_vector_type(VEC))); };
template <typename T, int VEC> using rec_vec = typename RecVec<T, VEC>::type;

// sigmoid(g) and sigmoid(-g) from one exponential of -|g|: neither overflows, neither is 1 minus the other (which would
// lose the small one's digits); both are exact at +-infinity.  The exponential is exp2 of a product carried in two
// parts, the quotient a reciprocal with one Newton step: 3 and 2 roundings, against 40 instructions more for the
// library's exponential and division (one wave instruction per element and load is what the memory leaves room for).
__device__ __forceinline__ void rec_gate(float g, float& a, float& w) {
  const float m = -fabsf(g);
  const float hi = m * 1.44269502f;                                     // log2(e) = 1.44269502 + 1.92596303e-8
  const float lo = fmaf(m, 1.92596303e-8f, fmaf(m, 1.44269502f, -hi));  // what the product lost
  float e = __builtin_amdgcn_exp2f(hi);
  e = hi > -126.f ? fmaf(e, lo * 0.693147182f, e) : 0.f;  // (below: smaller than every normal number; -infinity too)
  const float s = 1.0f + e;
  float r = __builtin_amdgcn_rcpf(s);
  r = fmaf(fmaf(-s, r, 1.0f), r, r);
  const float small = e * r;
  a = g >= 0.f ? r : small;
  w = g >= 0.f ? small : r;
  if (g != g) a = w = g;
}

struct RecArgs {
  const void *x, *gate;
  const float* state;           // [rows][width], or null: zeros
  const unsigned char* resets;  // [rows][steps], or null: none
  long steps;
  long x_row, x_step, g_row, g_step;  // in elements; columns are adjacent
  unsigned rows, width, groups;       // groups = rows * width / VEC
  unsigned tiles, tiles_each;         // tiles of time, and how many of them a block of the time split takes
  float* pairs;                       // [splits][2][rows * width]: compositions of the splits, in time's order
};
struct RecMarks {  // the state entering step k * REC_L, k >= 1, is p[row * row_stride + (k - 1) * stride + column]
  const float* p;
  long row_stride, stride;
};
struct RecGrads {
  const void* dh;  // or null: zeros
  const float* dlast;
  void *dx, *dgate;
  float* dstate;
  long dh_row, dh_step, dx_row, dx_step, dg_row, dg_step;
};

template <typename T, int VEC>
struct RecTile { rec_vec<T, VEC> v[REC_L]; };

// n steps (uniform over the wave) from p on; the steps behind the n-th are filled.  Candidates and gradients of 0 and gates
// of +infinity leave state and gradient as they are, so that nothing but the stores has to know where time ends.
template <typename T, int VEC>
__device__ __forceinline__ void rec_load(RecTile<T, VEC>& x, const T* p, long step, int n, float fill) {
  if (n >= REC_L) {
#pragma unroll
    for (int i = 0; i < REC_L; i++, p += step) x.v[i] = *(const rec_vec<T, VEC>*)p;
  } else {
#pragma unroll
    for (int i = 0; i < REC_L; i++, p += step) x.v[i] = i < n ? *(const rec_vec<T, VEC>*)p : rec_vec<T, VEC>((T)fill);
  }
}

template <typename T, int VEC>
__device__ __forceinline__ void rec_store(const RecTile<T, VEC>& x, T* p, long step, int n) {
  if (n >= REC_L) {
#pragma unroll
    for (int i = 0; i < REC_L; i++, p += step) *(rec_vec<T, VEC>*)p = x.v[i];
  } else {
#pragma unroll
    for (int i = 0; i < REC_L; i++, p += step)
      if (i < n) *(rec_vec<T, VEC>*)p = x.v[i];
  }
}

// bit i: step i is reset
__device__ __forceinline__ unsigned rec_resets(const unsigned char* p, int n) {
  if (!p) return 0;
  unsigned bits = 0;
  if (n >= REC_L) {
    static_assert(REC_L == 16, "one 16-byte load");
    unsigned b[4];
    __builtin_memcpy(b, p, 16);  // (unaligned where steps is odd)
    if (b[0] | b[1] | b[2] | b[3]) {
#pragma unroll
      for (int i = 0; i < 16; i++) bits |= ((b[i / 4] >> (8 * (i % 4))) & 0xFFu) ? 1u << i : 0u;
    }
  } else {
    for (int i = 0; i < n; i++) bits |= p[i] ? 1u << i : 0u;
  }
  return bits;
}

// A thread's columns.  The threads behind the last group do the last group's work once more (the same values to the same
// places): how many steps there are is then the same for a whole wave, and known to it as a scalar.
template <int VEC>
struct RecPlace {
  unsigned row, col;
  __device__ RecPlace(const RecArgs& a, unsigned group) {
    group = min(group, a.groups - 1);
    const unsigned per_row = a.width / VEC;
    row = group / per_row;
    col = (group - row * per_row) * VEC;
  }
};
__device__ __forceinline__ int rec_wave() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

// ---- many columns: a thread walks through all of time, the next REC_L steps on their way while it computes ------------
// Bound by memory: x and gate in, h and a 32nd of it in marks out.  8192 x 256 x 128 bf16: 380 us for 1.67 GB, 4.4 TB/s,
// where a copy of gigabytes reaches 4.8.
template <typename T, int VEC>
__global__ __launch_bounds__(256) void mg_recurrence_kernel(RecArgs a, T* __restrict__ h, float* __restrict__ last,
                                                            float* __restrict__ marks) {
  const RecPlace<VEC> at(a, blockIdx.x * 256 + threadIdx.x);
  const T* x = (const T*)a.x + at.row * a.x_row + at.col;
  const T* g = (const T*)a.gate + at.row * a.g_row + at.col;
  const unsigned char* rs = a.resets ? a.resets + at.row * a.steps : nullptr;
  T* out = h ? h + ((long)at.row * a.steps) * a.width + at.col : nullptr;
  float* mark = marks ? marks + (long)at.row * ((a.steps - 1) / REC_L) * a.width + at.col : nullptr;
  const long flat = (long)at.row * a.width + at.col;
  float s[VEC];
#pragma unroll
  for (int j = 0; j < VEC; j++) s[j] = a.state ? a.state[flat + j] : 0.f;

  RecTile<T, VEC> xt[2], gt[2];
  unsigned rt[2];
  auto fetch = [&](int k, long t) {
    const int n = (int)min((long)REC_L, a.steps - t);
    if (n <= 0) return;
    rec_load<T, VEC>(xt[k], x + t * a.x_step, a.x_step, n, 0.f);
    rec_load<T, VEC>(gt[k], g + t * a.g_step, a.g_step, n, INFINITY);
    rt[k] = rec_resets(rs ? rs + t : nullptr, n);
  };
  auto walk = [&](int k, long t) {
    const int n = (int)min((long)REC_L, a.steps - t);
    if (n <= 0) return;
    if (mark && t) {
      rec_vec<float, VEC> m;
#pragma unroll
      for (int j = 0; j < VEC; j++) m[j] = s[j];
      *(rec_vec<float, VEC>*)(mark + (t / REC_L - 1) * a.width) = m;
    }
    RecTile<T, VEC> o;
    auto step = [&](int i) {
#pragma unroll
      for (int j = 0; j < VEC; j++) {
        float ga, gw;
        rec_gate((float)gt[k].v[i][j], ga, gw);
        const float q = gw * (float)xt[k].v[i][j];
        s[j] = (rt[k] >> i) & 1 ? q : fmaf(ga, s[j], q);
        o.v[i][j] = (T)s[j];
      }
    };
    if (n == REC_L) {
#pragma unroll
      for (int i = 0; i < REC_L; i++) step(i);
    } else {
#pragma unroll
      for (int i = 0; i < REC_L; i++)
        if (i < n) step(i);
    }
    if (out) rec_store<T, VEC>(o, out + t * a.width, a.width, n);
  };
  fetch(0, 0);
  for (long t = 0; t < a.steps; t += 2 * REC_L) {
    fetch(1, t + REC_L);
    walk(0, t);
    fetch(0, t + 2 * REC_L);
    walk(1, t + REC_L);
  }
#pragma unroll
  for (int j = 0; j < VEC; j++) last[flat + j] = s[j];
}

// One step, no marks: a flat pass over the columns.  98304 x 128 bf16: 27 us for 176 MB, 6.5 TB/s (part of it stays in the
// caches); 24 x 128 f32: 2.6 us, the time of a launch.
template <typename T, int VEC>
__global__ __launch_bounds__(256) void mg_recurrence_step_kernel(RecArgs a, T* __restrict__ h, float* last) {
  if (blockIdx.x * 256 + threadIdx.x >= a.groups) return;  // (the state may be overwritten in place)
  const RecPlace<VEC> at(a, blockIdx.x * 256 + threadIdx.x);
  const rec_vec<T, VEC> x = *(const rec_vec<T, VEC>*)((const T*)a.x + at.row * a.x_row + at.col);
  const rec_vec<T, VEC> g = *(const rec_vec<T, VEC>*)((const T*)a.gate + at.row * a.g_row + at.col);
  const long flat = (long)at.row * a.width + at.col;
  rec_vec<float, VEC> s = a.state ? *(const rec_vec<float, VEC>*)(a.state + flat) : rec_vec<float, VEC>(0);
  const bool reset = a.resets && a.resets[at.row];
  rec_vec<T, VEC> o;
#pragma unroll
  for (int j = 0; j < VEC; j++) {
    float ga, gw;
    rec_gate((float)g[j], ga, gw);
    const float q = gw * (float)x[j];
    s[j] = reset ? q : fmaf(ga, s[j], q);
    o[j] = (T)s[j];
  }
  *(rec_vec<float, VEC>*)(last + flat) = s;
  if (h) *(rec_vec<T, VEC>*)(h + flat) = o;
}

// The walk back: a stretch's states are made again from its mark, its gradients go out in time's reverse order.  Bound by memory:
// x, gate and dh in, their gradients out.  8192 x 256 x 128 bf16: 611 us for 2.75 GB, 4.5 TB/s.
template <typename T, int VEC>
__global__ __launch_bounds__(256) void mg_recurrence_backward_kernel(RecArgs a, RecMarks m, RecGrads d) {
  const RecPlace<VEC> at(a, blockIdx.x * 256 + threadIdx.x);
  const T* x = (const T*)a.x + at.row * a.x_row + at.col;
  const T* g = (const T*)a.gate + at.row * a.g_row + at.col;
  const T* dh = d.dh ? (const T*)d.dh + at.row * d.dh_row + at.col : nullptr;
  T* dx = (T*)d.dx + at.row * d.dx_row + at.col;
  T* dg = (T*)d.dgate + at.row * d.dg_row + at.col;
  const unsigned char* rs = a.resets ? a.resets + at.row * a.steps : nullptr;
  const float* mark = m.p + at.row * m.row_stride + at.col;
  const long flat = (long)at.row * a.width + at.col;
  float v[VEC];
#pragma unroll
  for (int j = 0; j < VEC; j++) v[j] = d.dlast ? d.dlast[flat + j] : 0.f;
  for (long k = (a.steps - 1) / REC_L; k >= 0; k--) {
    const long t0 = k * REC_L;
    const int n = (int)min((long)REC_L, a.steps - t0);
    RecTile<T, VEC> xt, gt, dt;
    rec_load<T, VEC>(xt, x + t0 * a.x_step, a.x_step, n, 0.f);
    rec_load<T, VEC>(gt, g + t0 * a.g_step, a.g_step, n, INFINITY);
    if (dh) rec_load<T, VEC>(dt, dh + t0 * d.dh_step, d.dh_step, n, 0.f);
    const unsigned rt = rec_resets(rs ? rs + t0 : nullptr, n);
    float s[VEC];
#pragma unroll
    for (int j = 0; j < VEC; j++) s[j] = k ? mark[(k - 1) * m.stride + j] : a.state ? a.state[flat + j] : 0.f;
    float before[REC_L][VEC], ga[REC_L][VEC], gw[REC_L][VEC];
#pragma unroll
    for (int i = 0; i < REC_L; i++) {
#pragma unroll
      for (int j = 0; j < VEC; j++) {
        rec_gate((float)gt.v[i][j], ga[i][j], gw[i][j]);
        const float q = gw[i][j] * (float)xt.v[i][j];
        before[i][j] = (rt >> i) & 1 ? 0.f : s[j];
        s[j] = (rt >> i) & 1 ? q : fmaf(ga[i][j], s[j], q);
      }
    }
    RecTile<T, VEC> ox, og;
#pragma unroll
    for (int i = REC_L - 1; i >= 0; i--) {
#pragma unroll
      for (int j = 0; j < VEC; j++) {
        const float dd = dh ? v[j] + (float)dt.v[i][j] : v[j];
        ox.v[i][j] = (T)(gw[i][j] * dd);
        og.v[i][j] = (T)(dd * (before[i][j] - (float)xt.v[i][j]) * (ga[i][j] * gw[i][j]));
        v[j] = (rt >> i) & 1 ? 0.f : ga[i][j] * dd;
      }
    }
    rec_store<T, VEC>(ox, dx + t0 * d.dx_step, d.dx_step, n);
    rec_store<T, VEC>(og, dg + t0 * d.dg_step, d.dg_step, n);
  }
  if (d.dstate) {
#pragma unroll
    for (int j = 0; j < VEC; j++) d.dstate[flat + j] = v[j];
  }
}

// ---- few columns: REC_W waves share time ------------------------------------------------------------------------------
// One lane per group of columns, one wave per REC_L steps.  LDS holds the pairs of the current tile's waves, twice, so
// that one barrier per tile is enough.
// A pair (p, q) stands for s -> p s + q.  p is never negative, so -0 marks a stretch with a reset in it: what stood before
// it, NaN and infinity too, is gone (a product that underflowed to +0 does not hide them).  The mark is told by all its bits:
// a factor may be a NaN with its sign set, which is no reset.
__device__ __forceinline__ bool rec_marked(float p) { return __float_as_uint(p) == 0x80000000u; }
__device__ __forceinline__ float rec_apply(float p, float q, float s) { return rec_marked(p) ? q : fmaf(p, s, q); }
__device__ __forceinline__ void rec_compose(float later_p, float later_q, float& p, float& q) {
  q = rec_apply(later_p, later_q, q);
  p = rec_marked(later_p) ? -0.f : p * later_p;
}

template <int VEC>
struct RecExchange { float p[2][REC_W][VEC][64], q[2][REC_W][VEC][64]; };

// the compositions of the blocks that come before this one in the order of the pass (step = 1: forwards in time;
// -1: backwards), applied to s.  Wave w composes a share of them, then all waves compose the shares.
template <int VEC>
__device__ __forceinline__ void rec_join(const RecArgs& a, RecExchange<VEC>& ex, long flat, int first, int count,
                                         int step, int wave, int lane, float* s) {
  const long cols = (long)a.rows * a.width;
  const int each = (count + REC_W - 1) / REC_W;
  float p[VEC], q[VEC];
#pragma unroll
  for (int j = 0; j < VEC; j++) p[j] = 1.f, q[j] = 0.f;
  {
    const int end = min(count, (wave + 1) * each);
    for (int i0 = wave * each; i0 < end; i0 += 8) {  // eight pairs on their way at a time
      rec_vec<float, VEC> pw[8], qw[8];
#pragma unroll
      for (int u = 0; u < 8; u++) {
        const float* pair = a.pairs + 2 * cols * (first + min(i0 + u, end - 1) * step) + flat;
        pw[u] = *(const rec_vec<float, VEC>*)pair;
        qw[u] = *(const rec_vec<float, VEC>*)(pair + cols);
      }
#pragma unroll
      for (int u = 0; u < 8; u++)
        if (i0 + u < end) {
#pragma unroll
          for (int j = 0; j < VEC; j++) rec_compose(pw[u][j], qw[u][j], p[j], q[j]);
        }
    }
  }
#pragma unroll
  for (int j = 0; j < VEC; j++) ex.p[1][wave][j][lane] = p[j], ex.q[1][wave][j][lane] = q[j];
  __syncthreads();
  for (int w = 0; w < REC_W; w++) {
#pragma unroll
    for (int j = 0; j < VEC; j++) s[j] = rec_apply(ex.p[1][w][j][lane], ex.q[1][w][j][lane], s[j]);
  }
}

// The pair of one split of time: forwards s -> a s + w x, backwards v -> a (v + dh), 0 at a reset.  It reads what the tiles will
// read again, which is what cutting time costs: 1 x 65536 x 128 f32: 14 us for 67 MB, 4.9 TB/s.
template <typename T, int VEC, bool BACK>
__global__ __launch_bounds__(64 * REC_W) void mg_recurrence_pairs_kernel(RecArgs a, RecGrads d) {
  __shared__ RecExchange<VEC> ex;
  const int lane = threadIdx.x & 63, wave = rec_wave();
  const RecPlace<VEC> at(a, blockIdx.x * 64 + lane);
  const T* x = BACK ? (d.dh ? (const T*)d.dh + at.row * d.dh_row + at.col : nullptr) : (const T*)a.x + at.row * a.x_row + at.col;
  const long x_step = BACK ? d.dh_step : a.x_step;
  const T* g = (const T*)a.gate + at.row * a.g_row + at.col;
  const unsigned char* rs = a.resets ? a.resets + at.row * a.steps : nullptr;
  // a wave takes tiles_each stretches of REC_L steps that follow each other
  const long t_begin = ((long)blockIdx.y * REC_W + wave) * a.tiles_each * REC_L;
  float p[VEC], q[VEC];
#pragma unroll
  for (int j = 0; j < VEC; j++) p[j] = 1.f, q[j] = 0.f;
  for (unsigned kk = 0; kk < a.tiles_each; kk++) {
    const unsigned k = BACK ? a.tiles_each - 1 - kk : kk;
    const long t = t_begin + (long)k * REC_L;
    const int n = (int)min((long)REC_L, a.steps - t);
    if (n <= 0) continue;
    RecTile<T, VEC> xt, gt;
    if (x) rec_load<T, VEC>(xt, x + t * x_step, x_step, n, 0.f);
    rec_load<T, VEC>(gt, g + t * a.g_step, a.g_step, n, INFINITY);
    const unsigned rt = rec_resets(rs ? rs + t : nullptr, n);
#pragma unroll
    for (int ii = 0; ii < REC_L; ii++) {
      const int i = BACK ? REC_L - 1 - ii : ii;
#pragma unroll
      for (int j = 0; j < VEC; j++) {
        float ga, gw;
        rec_gate((float)gt.v[i][j], ga, gw);
        const bool reset = (rt >> i) & 1;
        if (BACK) {
          q[j] = reset ? 0.f : ga * (x ? q[j] + (float)xt.v[i][j] : q[j]);
        } else {
          const float b = gw * (float)xt.v[i][j];
          q[j] = reset ? b : fmaf(ga, q[j], b);
        }
        p[j] = reset ? -0.f : p[j] * ga;
      }
    }
  }
#pragma unroll
  for (int j = 0; j < VEC; j++) ex.p[0][wave][j][lane] = p[j], ex.q[0][wave][j][lane] = q[j];
  __syncthreads();
  if (wave) return;
  const long cols = (long)a.rows * a.width;
  float* pair = a.pairs + 2 * cols * blockIdx.y + (long)at.row * a.width + at.col;
#pragma unroll
  for (int j = 0; j < VEC; j++) {
    float pj = 1.f, qj = 0.f;
    for (int ww = 0; ww < REC_W; ww++) {
      const int w = BACK ? REC_W - 1 - ww : ww;
      rec_compose(ex.p[0][w][j][lane], ex.q[0][w][j][lane], pj, qj);
    }
    pair[j] = pj;
    pair[cols + j] = qj;
  }
}

// Tile after tile: the waves' pairs meet in LDS, then each wave goes on from the state that enters it.  Bound by memory where
// there are enough blocks (1 x 65536 x 128 f32 in 512 of them: 22 us for 101 MB, 4.6 TB/s), else by the way through a tile
// (250 x 129 x 100 f16, two tiles: 14 us for 19 MB).
template <typename T, int VEC>
__global__ __launch_bounds__(64 * REC_W) void mg_recurrence_tile_kernel(RecArgs a, T* __restrict__ h, float* __restrict__ last,
                                                                        float* __restrict__ marks) {
  __shared__ RecExchange<VEC> ex;
  const int lane = threadIdx.x & 63, wave = rec_wave();
  const RecPlace<VEC> at(a, blockIdx.x * 64 + lane);
  const T* x = (const T*)a.x + at.row * a.x_row + at.col;
  const T* g = (const T*)a.gate + at.row * a.g_row + at.col;
  const unsigned char* rs = a.resets ? a.resets + at.row * a.steps : nullptr;
  T* out = h ? h + ((long)at.row * a.steps) * a.width + at.col : nullptr;
  float* mark = marks ? marks + (long)at.row * ((a.steps - 1) / REC_L) * a.width + at.col : nullptr;
  const long flat = (long)at.row * a.width + at.col;
  float s[VEC];  // the state entering the tile, the same in all waves
#pragma unroll
  for (int j = 0; j < VEC; j++) s[j] = a.state ? a.state[flat + j] : 0.f;
  const unsigned k_begin = blockIdx.y * a.tiles_each, k_end = min(a.tiles, k_begin + a.tiles_each);
  RecTile<T, VEC> xt, gt;
  unsigned rt = 0;
  auto fetch = [&](unsigned k) {
    const long t = (long)k * REC_TILE + wave * REC_L;
    const int n = (int)min((long)REC_L, a.steps - t);
    if (n <= 0) return;
    rec_load<T, VEC>(xt, x + t * a.x_step, a.x_step, n, 0.f);
    rec_load<T, VEC>(gt, g + t * a.g_step, a.g_step, n, INFINITY);
    rt = rec_resets(rs ? rs + t : nullptr, n);
  };
  fetch(k_begin);
  if (gridDim.y > 1) rec_join<VEC>(a, ex, flat, 0, blockIdx.y, 1, wave, lane, s);
  for (unsigned k = k_begin; k < k_end; k++) {
    const int buf = (k - k_begin) & 1;
    const long t = (long)k * REC_TILE + wave * REC_L;
    const int n = (int)min((long)REC_L, a.steps - t);
    if (k != k_begin) fetch(k);
    float ga[REC_L][VEC], q[REC_L][VEC], p[VEC], c[VEC];
#pragma unroll
    for (int j = 0; j < VEC; j++) p[j] = 1.f, c[j] = 0.f;
    if (n > 0) {
#pragma unroll
      for (int i = 0; i < REC_L; i++) {
#pragma unroll
        for (int j = 0; j < VEC; j++) {
          float gw;
          rec_gate((float)gt.v[i][j], ga[i][j], gw);
          q[i][j] = gw * (float)xt.v[i][j];
          const bool reset = (rt >> i) & 1;
          c[j] = reset ? q[i][j] : fmaf(ga[i][j], c[j], q[i][j]);
          p[j] = reset ? -0.f : p[j] * ga[i][j];
        }
      }
    }
#pragma unroll
    for (int j = 0; j < VEC; j++) ex.p[buf][wave][j][lane] = p[j], ex.q[buf][wave][j][lane] = c[j];
    __syncthreads();
    float mine[VEC];
    for (int w = 0; w < REC_W; w++) {
#pragma unroll
      for (int j = 0; j < VEC; j++) {
        if (w == wave) mine[j] = s[j];
        s[j] = rec_apply(ex.p[buf][w][j][lane], ex.q[buf][w][j][lane], s[j]);
      }
    }
    if (n > 0) {
      if (mark && t) {
        rec_vec<float, VEC> mv;
#pragma unroll
        for (int j = 0; j < VEC; j++) mv[j] = mine[j];
        *(rec_vec<float, VEC>*)(mark + (t / REC_L - 1) * a.width) = mv;
      }
      RecTile<T, VEC> o;
#pragma unroll
      for (int i = 0; i < REC_L; i++) {
#pragma unroll
        for (int j = 0; j < VEC; j++) {
          mine[j] = (rt >> i) & 1 ? q[i][j] : fmaf(ga[i][j], mine[j], q[i][j]);
          o.v[i][j] = (T)mine[j];
        }
      }
      if (out) rec_store<T, VEC>(o, out + t * a.width, a.width, n);
    }
  }
  if (wave == 0 && k_end == a.tiles) {
#pragma unroll
    for (int j = 0; j < VEC; j++) last[flat + j] = s[j];
  }
}

// The same from the last tile to the first (1 x 65536 x 128 f32: 38 us for 169 MB, 4.5 TB/s; 250 x 129 x 100 f16: 18 us).
template <typename T, int VEC>
__global__ __launch_bounds__(64 * REC_W) void mg_recurrence_tile_backward_kernel(RecArgs a, RecMarks m, RecGrads d) {
  __shared__ RecExchange<VEC> ex;
  const int lane = threadIdx.x & 63, wave = rec_wave();
  const RecPlace<VEC> at(a, blockIdx.x * 64 + lane);
  const T* x = (const T*)a.x + at.row * a.x_row + at.col;
  const T* g = (const T*)a.gate + at.row * a.g_row + at.col;
  const T* dh = d.dh ? (const T*)d.dh + at.row * d.dh_row + at.col : nullptr;
  T* dx = (T*)d.dx + at.row * d.dx_row + at.col;
  T* dg = (T*)d.dgate + at.row * d.dg_row + at.col;
  const unsigned char* rs = a.resets ? a.resets + at.row * a.steps : nullptr;
  const float* mark = m.p + at.row * m.row_stride + at.col;
  const long flat = (long)at.row * a.width + at.col;
  float v[VEC];  // what flows into the tile from the steps behind it, the same in all waves
#pragma unroll
  for (int j = 0; j < VEC; j++) v[j] = d.dlast ? d.dlast[flat + j] : 0.f;
  const unsigned k_begin = blockIdx.y * a.tiles_each, k_end = min(a.tiles, k_begin + a.tiles_each);
  RecTile<T, VEC> xt, gt, dt;
  unsigned rt = 0;
  float s[VEC];
  auto fetch = [&](unsigned k) {
    const long t0 = (long)k * REC_TILE + wave * REC_L;
    const int n = (int)min((long)REC_L, a.steps - t0);
    if (n <= 0) return;
    rec_load<T, VEC>(xt, x + t0 * a.x_step, a.x_step, n, 0.f);
    rec_load<T, VEC>(gt, g + t0 * a.g_step, a.g_step, n, INFINITY);
    if (dh) rec_load<T, VEC>(dt, dh + t0 * d.dh_step, d.dh_step, n, 0.f);
    rt = rec_resets(rs ? rs + t0 : nullptr, n);
#pragma unroll
    for (int j = 0; j < VEC; j++) s[j] = t0 ? mark[(t0 / REC_L - 1) * m.stride + j] : a.state ? a.state[flat + j] : 0.f;
  };
  fetch(k_end - 1);
  if (gridDim.y > 1) rec_join<VEC>(a, ex, flat, gridDim.y - 1, gridDim.y - 1 - blockIdx.y, -1, wave, lane, v);
  for (unsigned k = k_end; k-- > k_begin;) {
    const int buf = (k_end - 1 - k) & 1;
    const long t0 = (long)k * REC_TILE + wave * REC_L;
    const int n = (int)min((long)REC_L, a.steps - t0);
    float ak[REC_L][VEC], gw[REC_L][VEC], e[REC_L][VEC], p[VEC], c[VEC];  // ak: a, or -0 at a reset; e: dgate / d
#pragma unroll
    for (int j = 0; j < VEC; j++) p[j] = 1.f, c[j] = 0.f;
    if (k + 1 < k_end) fetch(k);
    if (n > 0) {
#pragma unroll
      for (int i = 0; i < REC_L; i++) {
#pragma unroll
        for (int j = 0; j < VEC; j++) {
          float ga;
          rec_gate((float)gt.v[i][j], ga, gw[i][j]);
          const float xv = (float)xt.v[i][j], q = gw[i][j] * xv;
          const bool reset = (rt >> i) & 1;
          e[i][j] = ((reset ? 0.f : s[j]) - xv) * (ga * gw[i][j]);
          ak[i][j] = reset ? -0.f : ga;
          s[j] = rec_apply(ak[i][j], q, s[j]);
        }
      }
#pragma unroll
      for (int i = REC_L - 1; i >= 0; i--) {
#pragma unroll
        for (int j = 0; j < VEC; j++) {
          const float cd = dh ? c[j] + (float)dt.v[i][j] : c[j];
          c[j] = rec_apply(ak[i][j], 0.f, cd);
          p[j] = rec_marked(ak[i][j]) ? -0.f : p[j] * ak[i][j];
        }
      }
    }
#pragma unroll
    for (int j = 0; j < VEC; j++) ex.p[buf][wave][j][lane] = p[j], ex.q[buf][wave][j][lane] = c[j];
    __syncthreads();
    float mine[VEC];
    for (int w = REC_W - 1; w >= 0; w--) {
#pragma unroll
      for (int j = 0; j < VEC; j++) {
        if (w == wave) mine[j] = v[j];
        v[j] = rec_apply(ex.p[buf][w][j][lane], ex.q[buf][w][j][lane], v[j]);
      }
    }
    if (n > 0) {
      RecTile<T, VEC> ox, og;
#pragma unroll
      for (int i = REC_L - 1; i >= 0; i--) {
#pragma unroll
        for (int j = 0; j < VEC; j++) {
          const float dd = dh ? mine[j] + (float)dt.v[i][j] : mine[j];
          ox.v[i][j] = (T)(gw[i][j] * dd);
          og.v[i][j] = (T)(dd * e[i][j]);
          mine[j] = rec_apply(ak[i][j], 0.f, dd);
        }
      }
      rec_store<T, VEC>(ox, dx + t0 * d.dx_step, d.dx_step, n);
      rec_store<T, VEC>(og, dg + t0 * d.dg_step, d.dg_step, n);
    }
  }
  if (d.dstate && wave == 0 && k_begin == 0) {
#pragma unroll
    for (int j = 0; j < VEC; j++) d.dstate[flat + j] = v[j];
  }
}

// ---- host side --------------------------------------------------------------------------------------------------------

static int rec_check(const char* who, const mg_recurrence* r) {
  if (!r) return mg_fail_msg(std::string(who) + ": NULL arguments");
  if (r->rows < 0 || r->steps < 0 || r->width < 0) return mg_fail_msg(std::string(who) + ": negative shape");
  if (r->type < 0 || r->type > 2) return mg_fail_msg(std::string(who) + ": type must be MG_F32, MG_BF16 or MG_F16");
  if (r->rows && r->width && r->rows > ((int64_t)1 << 31) / r->width)
    return mg_fail_msg(std::string(who) + ": rows * width must not exceed 2^31");
  if (r->steps > (int64_t)1 << 31) return mg_fail_msg(std::string(who) + ": steps must not exceed 2^31");
  if (r->rows && r->steps && r->width && (!r->x || !r->gate)) return mg_fail_msg(std::string(who) + ": NULL tensor");
  return 0;
}

// How the work is laid out; a function of the shape alone, so that results do not depend on addresses.
struct RecPlan { bool shared; unsigned tiles, tiles_each, splits; };

static RecPlan rec_plan(const mg_recurrence* r) {
  // 4 bytes per lane and step whatever the type: with two f32 columns per lane a block's registers leave room for no second
  // one on a CU (1 x 65536 x 128: 45 us backward against 39; 2500 x 100 x 128: 154 against 138)
  const bool f32 = r->type == MG_F32;
  RecPlan p{false, (unsigned)((r->steps + REC_TILE - 1) / REC_TILE), 0, 1};
  const int64_t each = f32 ? 64 : 128, waves = (r->rows * r->width + each - 1) / each;
  // a walk through time needs five waves per CU (eight with f32's smaller loads) to keep the memory busy: 1500 x 170 x 128
  // bf16 takes 55 us that way and 66 in tiles, 1024 x 256 x 128 53 and 54
  p.shared = waves < (f32 ? 2048 : 1280) && r->steps > REC_L;
  // time is cut where there is less than a block per CU, into as many blocks as are resident at a time: two per CU (f32) or
  // one (1 x 65536 x 128 bf16: 30 us, with two 42).  The pairs are the price, of reading the inputs again: 256 x 1024 x 128
  // bf16 takes 50 us forward in one launch and 87 cut in two.  Close below 256 waves the rule costs more than it gives in 16
  // bits (250 x 1024 x 128: 84 us forward and 128 back, 256: 50 and 95), with f32 it does not (83 and 141, 81 and 144).
  if (p.shared && p.tiles >= 4 && waves < 256) {
    const int64_t want = ((f32 ? 512 : 256) + waves - 1) / waves;
    p.splits = (unsigned)(want < p.tiles ? want : p.tiles);
  }
  p.tiles_each = (p.tiles + p.splits - 1) / p.splits;
  p.splits = (p.tiles + p.tiles_each - 1) / p.tiles_each;
  return p;
}

static RecArgs rec_args(const mg_recurrence* r, const RecPlan& p, int vec) {
  return RecArgs{r->x, r->gate, r->state, r->resets, (long)r->steps, (long)r->x_row, (long)r->x_step, (long)r->gate_row,
                 (long)r->gate_step, (unsigned)r->rows, (unsigned)r->width, (unsigned)(r->rows * r->width / vec), p.tiles,
                 p.tiles_each, (float*)r->workspace};
}

// whether columns can be moved two (or four) at a time: whole groups in a row, every row start on a group's boundary
static bool rec_fits(int vec, int64_t elem, int64_t width, std::initializer_list<const void*> tensors,
                     std::initializer_list<const void*> f32, std::initializer_list<int64_t> strides) {
  if (width % vec) return false;
  for (const void* t : tensors) if ((uintptr_t)t % (vec * elem)) return false;
  for (const void* t : f32) if ((uintptr_t)t % (vec * 4)) return false;
  for (int64_t s : strides) if (s % vec) return false;
  return true;
}

template <typename F>
static int rec_by_type(int type, F f) {
  if (type == MG_F32) return f((float*)nullptr);
  if (type == MG_BF16) return f((__bf16*)nullptr);
  return f((_Float16*)nullptr);
}
template <int V> using rec_int = std::integral_constant<int, V>;

static int rec_launched(const char* who) {
  const hipError_t err = hipGetLastError();
  return err == hipSuccess ? 0 : mg_fail_msg(std::string(who) + ": " + hipGetErrorString(err));
}

static int rec_workspace(const char* who, const mg_recurrence* r, const RecPlan& p) {
  if (p.splits > 1 && (!r->workspace || r->workspace_bytes < mg_gated_recurrence_workspace(r)))
    return mg_fail_msg(std::string(who) + ": workspace smaller than mg_gated_recurrence_workspace says");
  return 0;
}

extern "C" int64_t mg_gated_recurrence_workspace(const mg_recurrence* r) {
  if (!r || r->rows <= 0 || r->steps <= 0 || r->width <= 0 || r->rows > ((int64_t)1 << 31) / r->width) return 0;
  const RecPlan p = rec_plan(r);
  return p.splits > 1 ? (int64_t)p.splits * 2 * r->rows * r->width * 4 : 0;
}

extern "C" int mg_gated_recurrence(const mg_recurrence* r, void* h, float* last, float* marks, void* stream) try {
  static const char who[] = "mg_gated_recurrence";
  if (const int rc = rec_check(who, r)) return rc;
  if (!r->rows || !r->steps || !r->width) return 0;
  if (!last) return mg_fail_msg(std::string(who) + ": NULL tensor");
  const RecPlan p = rec_plan(r);
  if (const int rc = rec_workspace(who, r, p)) return rc;
  const hipStream_t s = (hipStream_t)stream;
  return rec_by_type(r->type, [&](auto* null) {
    using T = std::remove_pointer_t<decltype(null)>;
    const int64_t e = sizeof(T);
    auto fits = [&](int vec) {
      return rec_fits(vec, e, r->width, {r->x, r->gate, h}, {r->state, last, marks}, {r->x_row, r->x_step, r->gate_row, r->gate_step});
    };
    auto step = [&](auto vec) {
      constexpr int VEC = decltype(vec)::value;
      const RecArgs a = rec_args(r, p, VEC);
      hipLaunchKernelGGL((mg_recurrence_step_kernel<T, VEC>), dim3((a.groups + 255) / 256), dim3(256), 0, s, a, (T*)h, last);
      return rec_launched(who);
    };
    if (r->steps == 1) {  // with fewer columns than that, rather more threads
      if (r->rows * r->width >= 1 << 20 && fits(4)) return step(rec_int<4>());
      return fits(2) ? step(rec_int<2>()) : step(rec_int<1>());
    }
    auto with = [&](auto vec) {
      constexpr int VEC = decltype(vec)::value;
      const RecArgs a = rec_args(r, p, VEC);
      if (!p.shared) {
        hipLaunchKernelGGL((mg_recurrence_kernel<T, VEC>), dim3((a.groups + 255) / 256), dim3(256), 0, s, a, (T*)h, last, marks);
      } else {
        const dim3 grid((a.groups + 63) / 64, p.splits);
        if (p.splits > 1)
          hipLaunchKernelGGL((mg_recurrence_pairs_kernel<T, VEC, false>), grid, dim3(64 * REC_W), 0, s, a, RecGrads{});
        hipLaunchKernelGGL((mg_recurrence_tile_kernel<T, VEC>), grid, dim3(64 * REC_W), 0, s, a, (T*)h, last, marks);
      }
      return rec_launched(who);
    };
    if constexpr (sizeof(T) == 2) {
      if (fits(2)) return with(rec_int<2>());
    }
    return with(rec_int<1>());
  });
} catch (...) {
  return 1;
}

extern "C" int mg_gated_recurrence_backward(const mg_recurrence* r, const float* marks, int64_t marks_row,
                                            int64_t marks_stride, const mg_recurrence_gradients* d, void* stream) try {
  static const char who[] = "mg_gated_recurrence_backward";
  if (const int rc = rec_check(who, r)) return rc;
  if (!r->rows || !r->steps || !r->width) return 0;
  if (!d || !d->dx || !d->dgate || (!marks && r->steps > REC_L)) return mg_fail_msg(std::string(who) + ": NULL tensor");
  const RecPlan p = rec_plan(r);
  if (const int rc = rec_workspace(who, r, p)) return rc;
  const hipStream_t s = (hipStream_t)stream;
  return rec_by_type(r->type, [&](auto* null) {
    using T = std::remove_pointer_t<decltype(null)>;
    auto with = [&](auto vec) {
      constexpr int VEC = decltype(vec)::value;
      const RecArgs a = rec_args(r, p, VEC);
      const RecMarks m{marks, (long)marks_row, (long)marks_stride};
      const RecGrads g{d->dh, d->dlast, d->dx, d->dgate, d->dstate, (long)d->dh_row, (long)d->dh_step, (long)d->dx_row,
                       (long)d->dx_step, (long)d->dgate_row, (long)d->dgate_step};
      if (!p.shared) {
        hipLaunchKernelGGL((mg_recurrence_backward_kernel<T, VEC>), dim3((a.groups + 255) / 256), dim3(256), 0, s, a, m, g);
      } else {
        const dim3 grid((a.groups + 63) / 64, p.splits);
        if (p.splits > 1)
          hipLaunchKernelGGL((mg_recurrence_pairs_kernel<T, VEC, true>), grid, dim3(64 * REC_W), 0, s, a, g);
        hipLaunchKernelGGL((mg_recurrence_tile_backward_kernel<T, VEC>), grid, dim3(64 * REC_W), 0, s, a, m, g);
      }
      return rec_launched(who);
    };
    if constexpr (sizeof(T) == 2) {
      if (rec_fits(2, 2, r->width, {r->x, r->gate, d->dh, d->dx, d->dgate}, {},
                   {r->x_row, r->x_step, r->gate_row, r->gate_step, d->dh_row, d->dh_step, d->dx_row, d->dx_step, d->dgate_row, d->dgate_step}))
        return with(rec_int<2>());
    }
    return with(rec_int<1>());
  });
} catch (...) {
  return 1;
}
