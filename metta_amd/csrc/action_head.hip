// action_head.hip -- the head between a policy's logits and its actions for gfx950: adjusted logits, sampling, and the
// log-probability and entropy of given actions, with gradients (mg_adjust_logits, mg_sample_actions,
// mg_evaluate_actions and their backward forms).
//
// Per row, with c = how often token v stands in the row's history:
//   l1 = c > 0 ? (l > 0 ? l / repetition : l * repetition) : l        l2 = l1 - frequency * c - presence * (c > 0)
//   x = allowed ? l2 + bias : -infinity      adjusted = x / temperature
//   M = max x, d = (M - x) / temperature, Z = sum exp(-d), q = exp(-d) / Z, H = log Z + sum d q
//   sampled: the first v with sum_{w <= v} exp(-d_w) > u Z;  without u: the first v with x = M
//   log q_v = -d_v - log Z;   d x_v of g_p log q_a + g_h H:  (g_p (1[v = a] - q_v) - g_h q_v (log q_v + H)) / temperature
// A row with nothing left (M = -infinity) has action -1, log-probability 0, entropy 0 and no gradient; a row with NaN
// or +infinity among its allowed tokens has action -1 and NaN.
//
// Rows of up to HEAD_NARROW columns are held in registers, E adjacent columns per lane, by as many lanes as that takes
// (one lane for five actions, a wave for a thousand), so logits are read once.  Wider rows are cut into parts of
// HEAD_PART columns, a block each; what a part found (maximum, sum, ...) goes to a workspace and a second launch joins
// the parts of a row.  A history is counted in LDS by the block that needs it, for the columns that it holds.
//
// Sampling is done in 64 bits from the exponential on: an action that falls next to a border of the distribution is then
// the definition's whatever the order of the sums, and a 64-bit multiply-add costs what a 32-bit one costs here.
// Log-probabilities and entropies of given actions need no more than 32 bits, and are computed in 32 unless a bias or a
// penalty could cancel large logits (HeadX = double).
#include <hip/hip_runtime.h>

#include <cmath>
#include <string>
#include <type_traits>

#include "../../include/mettagrid_hip.h"

#define HEAD_THREADS 256
#define HEAD_NARROW MG_EVALUATE_STATS_WIDTH
#define HEAD_CHUNK (HEAD_THREADS * 8)  // columns that a block holds as 8 per thread
#define HEAD_CHUNKS 4
#define HEAD_PART (HEAD_CHUNKS * HEAD_CHUNK)
#define HEAD_FOUND 5  // doubles per part in the workspace: M, Z, sum d exp(-d), bad, first column of M

extern int mg_fail_msg(const std::string& m);  // mettagrid_hip.hip: sets mg_last_error(), returns 1

// ---- elements: the tensors' type is a scalar branch around the loads and stores ---------------------------------------

template <int E>
__device__ __forceinline__ void head_load(const void* p, int type, long at, int n, float* out) {
  if (type == MG_F32) {
    const float* q = (const float*)p + at;
    if (n >= E) {
      __builtin_memcpy(out, q, 4 * E);  // (rows of any width: the start is aligned to an element only)
    } else {
#pragma unroll
      for (int e = 0; e < E; e++) out[e] = e < n ? q[e] : 0.f;
    }
    return;
  }
  const unsigned short* q = (const unsigned short*)p + at;
  unsigned short raw[E];
  if (n >= E) {
    __builtin_memcpy(raw, q, 2 * E);
  } else {
#pragma unroll
    for (int e = 0; e < E; e++) raw[e] = e < n ? q[e] : (unsigned short)0;
  }
#pragma unroll
  for (int e = 0; e < E; e++) out[e] = type == MG_BF16 ? __uint_as_float((unsigned)raw[e] << 16) : (float)__builtin_bit_cast(_Float16, raw[e]);
}

template <int E>
__device__ __forceinline__ void head_store(void* p, int type, long at, int n, const float* x) {
  if (type == MG_F32) {
    float* q = (float*)p + at;
    if (n >= E) {
      __builtin_memcpy(q, x, 4 * E);
    } else {
#pragma unroll
      for (int e = 0; e < E; e++) if (e < n) q[e] = x[e];
    }
    return;
  }
  unsigned short* q = (unsigned short*)p + at;
  unsigned short raw[E];
#pragma unroll
  for (int e = 0; e < E; e++) raw[e] = type == MG_BF16 ? __builtin_bit_cast(unsigned short, (__bf16)x[e]) : __builtin_bit_cast(unsigned short, (_Float16)x[e]);
  if (n >= E) {
    __builtin_memcpy(q, raw, 2 * E);
  } else {
#pragma unroll
    for (int e = 0; e < E; e++) if (e < n) q[e] = raw[e];
  }
}

// ---- arithmetic -------------------------------------------------------------------------------------------------------

// e^-d for d >= 0 (NaN: NaN).  n = rint(y log2 e) with y = -d, r = y - n ln 2 in two parts, |r| <= 0.347: the series to
// r^12 / 12! leaves 2e-16; 18 instructions, where the library's takes 40.
__device__ __forceinline__ double head_exp(double d) {
  const double n = rint(d * -1.4426950408889634);
  double r = fma(n, -0.69314718055994529, -d);  // ln 2 = 0.69314718055994529 + 2.3190468138462996e-17
  r = fma(n, -2.3190468138462996e-17, r);
  double p = 1.0 / 479001600.0;
  p = fma(p, r, 1.0 / 39916800.0);
  p = fma(p, r, 1.0 / 3628800.0);
  p = fma(p, r, 1.0 / 362880.0);
  p = fma(p, r, 1.0 / 40320.0);
  p = fma(p, r, 1.0 / 5040.0);
  p = fma(p, r, 1.0 / 720.0);
  p = fma(p, r, 1.0 / 120.0);
  p = fma(p, r, 1.0 / 24.0);
  p = fma(p, r, 1.0 / 6.0);
  p = fma(p, r, 0.5);
  p = fma(p, r, 1.0);
  p = fma(p, r, 1.0);
  return d > 746.0 ? 0.0 : ldexp(p, (int)n);  // (the smallest denormal is e^-745)
}
// the same in 32 bits: exp2 of a product carried in two parts
__device__ __forceinline__ float head_exp(float d) {
  const float hi = d * -1.44269502f;  // log2 e = 1.44269502 + 1.92596303e-8
  const float lo = fmaf(d, -1.92596303e-8f, fmaf(d, -1.44269502f, -hi));
  const float e = __builtin_amdgcn_exp2f(hi);
  return hi < -126.f ? 0.f : fmaf(e, lo * 0.693147182f, e);
}
__device__ __forceinline__ double head_log(double z) { return log(z); }
__device__ __forceinline__ float head_log(float z) { return logf(z); }

// One row's controls.
struct HeadRow {
  const float* bias;
  const void* allowed;
  int kind;
  bool counted;
  double inv_rep, rep, presence, frequency, inv_temp;
};

__device__ __forceinline__ HeadRow head_row(const mg_logits& a, long row) {
  HeadRow r;
  r.bias = a.bias ? a.bias + row * a.bias_row : nullptr;
  r.kind = a.allowed ? a.allowed_kind : 0;
  r.allowed = !a.allowed ? nullptr : r.kind == MG_ALLOWED_BOOL ? (const void*)((const unsigned char*)a.allowed + row * a.allowed_row)
                                                               : (const void*)((const int*)a.allowed + row * a.allowed_row);
  r.counted = a.history != nullptr;
  r.rep = a.repetition; r.inv_rep = 1.0 / a.repetition;
  r.presence = a.presence; r.frequency = a.frequency; r.inv_temp = 1.0 / a.temperature;
  return r;
}

// bit e: column v0 + e is allowed, e < n
template <int E>
__device__ __forceinline__ unsigned head_allowed(const HeadRow& r, int v0, int n) {
  static_assert(E <= 16, "bits of one half word");
  if (n <= 0) return 0;
  const unsigned inside = n >= E ? (1u << E) - 1 : (1u << n) - 1;
  if (r.kind == MG_ALLOWED_BITS) return (((const unsigned*)r.allowed)[v0 >> 5] >> (v0 & 31)) & inside;  // (E divides 32)
  if (r.kind == MG_ALLOWED_BOOL) {
    const unsigned char* p = (const unsigned char*)r.allowed + v0;
    unsigned bits = 0;
    if (n >= E) {
      unsigned b[(E + 3) / 4];
      __builtin_memcpy(b, p, E);
#pragma unroll
      for (int e = 0; e < E; e++) bits |= ((b[e / 4] >> (8 * (e % 4))) & 0xFFu) ? 1u << e : 0u;
    } else {
#pragma unroll
      for (int e = 0; e < E; e++) if (e < n) bits |= p[e] ? 1u << e : 0u;
    }
    return bits;
  }
  return inside;
}

// the whole factor of a gradient, from what head_columns leaves in `slope`
__device__ __forceinline__ double head_slope(const HeadRow& r, float slope) { return slope * r.inv_temp; }

// E adjacent columns from v0 on, n of them in the row: x, and (GRAD) what a gradient of x is multiplied by besides 1 /
// temperature.  counts: of these columns in the history.
template <int E, bool GRAD, typename X>
__device__ __forceinline__ void head_columns(const HeadRow& r, const void* logits, int type, long at, int v0, int n,
                                             const unsigned* counts, X* x, float* slope) {
  float l[E];
  head_load<E>(logits, type, at + v0, n, l);
  const unsigned ok = head_allowed<E>(r, v0, n);
  float b[E];
  if (std::is_same<X, double>::value && r.bias) head_load<E>(r.bias, MG_F32, v0, n, b);
#pragma unroll
  for (int e = 0; e < E; e++) {
    X y = l[e];
    if (GRAD) slope[e] = 1.f;
    if (std::is_same<X, double>::value) {
      if (r.counted) {
        const unsigned c = counts[e];
        if (c) {
          if (GRAD) slope[e] = (float)(y > 0 ? r.inv_rep : r.rep);
          y = (y > 0 ? y * r.inv_rep : y * r.rep) - r.frequency * c - r.presence;
        }
      }
      if (r.bias) y += b[e];
    }
    const bool in = (ok >> e) & 1;
    x[e] = in ? y : (X)-INFINITY;
    if (GRAD && !in) slope[e] = 0.f;
  }
}

// ---- lanes ------------------------------------------------------------------------------------------------------------

__device__ __forceinline__ double head_add(double a, double b) { return a + b; }
__device__ __forceinline__ float head_add(float a, float b) { return a + b; }
__device__ __forceinline__ int head_lane() { return threadIdx.x & 63; }

// over the `lanes` (a power of two) lanes of a group; every lane gets the result
template <typename V, typename F>
__device__ __forceinline__ V head_group(V x, int lanes, F f) {
  for (int o = 1; o < lanes; o <<= 1) x = f(x, __shfl_xor(x, o));
  return x;
}
template <typename V>
__device__ __forceinline__ V head_group_max(V x, int lanes) {
  return head_group(x, lanes, [](V a, V b) { return a > b ? a : b; });
}
template <typename V>
__device__ __forceinline__ V head_group_min(V x, int lanes) {
  return head_group(x, lanes, [](V a, V b) { return a < b ? a : b; });
}
template <typename V>
__device__ __forceinline__ V head_group_sum(V x, int lanes) {
  return head_group(x, lanes, [](V a, V b) { return a + b; });
}
// the sum of the lanes before this one in its group
__device__ __forceinline__ double head_group_before(double x, int lanes, int lane) {
  double sum = x;
  for (int o = 1; o < lanes; o <<= 1) {
    const double up = __shfl_up(sum, o);
    if (lane >= o) sum += up;
  }
  return sum - x;
}

// ---- narrow rows ------------------------------------------------------------------------------------------------------

struct HeadNarrow { int lanes, rows; };  // lanes per row (a power of two), rows per block

// counts[row * lanes + lane][e] over the block's rows, all threads together; barriers inside
template <int E>
__device__ __forceinline__ void head_count_rows(const mg_logits& a, const HeadNarrow& g, long row0, unsigned (*counts)[E + 1]) {
  __syncthreads();
#pragma unroll
  for (int e = 0; e < E; e++) counts[threadIdx.x][e] = 0;
  __syncthreads();
  const int rows = (int)min((long)g.rows, a.rows - row0);
  // entry threadIdx.x, then every 256th of the block's rows * history_len, row and place kept without a division a step
  const int len = a.history_len, skip = HEAD_THREADS / len, rest = HEAD_THREADS - skip * len;
  int row = threadIdx.x / len, place = threadIdx.x - row * len;
  while (row < rows) {
    const int v = a.history[(row0 + row) * a.history_row + place];
    if (v >= 0 && v < a.width) atomicAdd(&counts[row * g.lanes + v / E][v % E], 1u);
    row += skip;
    place += rest;
    if (place >= len) place -= len, row++;
  }
  __syncthreads();
}

// what a group of lanes knows of its row
template <int E, typename X>
struct HeadHeld {
  X x[E], d[E], e[E], m, z, s;  // d and e stay unset where the row is bad or empty
  float slope[E];
  long row;      // clamped: the groups behind the last row do that row's work once more
  int lane, v0, n;
  bool bad, empty, mine;  // mine: the row is this group's own
};

template <int E, bool GRAD, typename X>
__device__ __forceinline__ void head_hold(const mg_logits& a, const HeadNarrow& g, const HeadRow& r, const unsigned* counts, HeadHeld<E, X>& h) {
  h.v0 = h.lane * E;
  h.n = a.width - h.v0;
  head_columns<E, GRAD>(r, a.logits, a.type, h.row * a.logits_row, h.v0, h.n, counts, h.x, h.slope);
  X m = -INFINITY;
  bool bad = false;
#pragma unroll
  for (int e = 0; e < E; e++) {
    if (!(h.x[e] < (X)INFINITY)) bad = true;
    m = h.x[e] > m ? h.x[e] : m;
  }
  h.m = head_group_max(m, g.lanes);
  h.bad = head_group_max((int)bad, g.lanes) != 0;
  h.empty = !h.bad && h.m == (X)-INFINITY;
  const X top = h.bad || h.empty ? (X)0 : h.m, inv_temp = (X)r.inv_temp;
  X z = 0, s = 0;
#pragma unroll
  for (int e = 0; e < E; e++) {
    h.d[e] = (top - h.x[e]) * inv_temp;
    h.e[e] = head_exp(h.d[e]);
    z += h.e[e];
    s += h.e[e] > 0 ? h.d[e] * h.e[e] : 0;
  }
  h.z = head_group_sum(z, g.lanes);
  h.s = head_group_sum(s, g.lanes);
}

template <int E, typename X>
__device__ __forceinline__ void head_place(const mg_logits& a, const HeadNarrow& g, long row0, HeadHeld<E, X>& h) {
  const long row = row0 + threadIdx.x / g.lanes;
  h.mine = row < a.rows;
  h.row = h.mine ? row : a.rows - 1;
  h.lane = threadIdx.x & (g.lanes - 1);
}

template <int E>
__global__ __launch_bounds__(HEAD_THREADS) void mg_adjust_narrow_kernel(mg_logits a, HeadNarrow g, void* __restrict__ out,
                                                                       const void* __restrict__ dout, void* __restrict__ dlogits) {
  using X = double;
  __shared__ unsigned counts[HEAD_THREADS][E + 1];
  for (long row0 = (long)blockIdx.x * g.rows; row0 < a.rows; row0 += (long)gridDim.x * g.rows) {
    if (a.history) head_count_rows<E>(a, g, row0, counts);
    HeadHeld<E, X> h;
    head_place(a, g, row0, h);
    const HeadRow r = head_row(a, h.row);
    h.v0 = h.lane * E;
    h.n = h.mine ? a.width - h.v0 : 0;
    float y[E];
    if (out) {
      head_columns<E, false>(r, a.logits, a.type, h.row * a.logits_row, h.v0, h.n, counts[threadIdx.x], h.x, h.slope);
#pragma unroll
      for (int e = 0; e < E; e++) y[e] = (float)(h.x[e] * r.inv_temp);
      head_store<E>(out, a.type, h.row * a.width + h.v0, h.n, y);
    } else {
      float go[E];
      head_columns<E, true>(r, a.logits, a.type, h.row * a.logits_row, h.v0, h.n, counts[threadIdx.x], h.x, h.slope);
      head_load<E>(dout, a.type, h.row * a.width + h.v0, h.n, go);
#pragma unroll
      for (int e = 0; e < E; e++) y[e] = h.slope[e] == 0.f ? 0.f : (float)((double)go[e] * head_slope(r, h.slope[e]));
      head_store<E>(dlogits, a.type, h.row * a.width + h.v0, h.n, y);
    }
  }
}

template <int E>
__global__ __launch_bounds__(HEAD_THREADS) void mg_sample_narrow_kernel(mg_logits a, HeadNarrow g, const float* __restrict__ uniforms,
                                                                       int* __restrict__ actions, float* __restrict__ log_prob,
                                                                       float* __restrict__ entropy) {
  using X = double;
  __shared__ unsigned counts[HEAD_THREADS][E + 1];
  for (long row0 = (long)blockIdx.x * g.rows; row0 < a.rows; row0 += (long)gridDim.x * g.rows) {
    if (a.history) head_count_rows<E>(a, g, row0, counts);
    HeadHeld<E, X> h;
    head_place(a, g, row0, h);
    const HeadRow r = head_row(a, h.row);
    head_hold<E, false>(a, g, r, counts[threadIdx.x], h);
    int hit = a.width, last = -1;
    if (uniforms) {
      const double target = fmax((double)uniforms[h.row], 0.0) * h.z;
      double mine = 0.0;
#pragma unroll
      for (int e = 0; e < E; e++) mine += h.e[e];
      double run = head_group_before(mine, g.lanes, h.lane);
#pragma unroll
      for (int e = 0; e < E; e++) {
        run += h.e[e];
        if (run > target && hit == a.width && e < h.n) hit = h.v0 + e;
        if (h.e[e] > 0.0) last = h.v0 + e;
      }
      hit = head_group_min(hit, g.lanes);
      last = head_group_max(last, g.lanes);
      if (hit == a.width) hit = last;  // a uniform of 1 or more
    } else {
#pragma unroll
      for (int e = E - 1; e >= 0; e--)
        if (h.x[e] == h.m && e < h.n) hit = h.v0 + e;
      hit = head_group_min(hit, g.lanes);
    }
    double d = 0.0;
#pragma unroll
    for (int e = 0; e < E; e++) if (h.v0 + e == hit) d = h.d[e];
    d = __shfl(d, (head_lane() & ~(g.lanes - 1)) + (hit >= 0 && hit < a.width ? hit / E : 0));
    if (h.mine && h.lane == 0) {
      const double log_z = head_log(h.z);
      const bool none = h.bad || h.empty;
      actions[h.row] = none ? -1 : hit;
      log_prob[h.row] = h.bad ? NAN : h.empty ? 0.f : (float)(-d - log_z);
      entropy[h.row] = h.bad ? NAN : h.empty ? 0.f : (float)(log_z + h.s / h.z);
    }
  }
}

template <int E, typename X>
__global__ __launch_bounds__(HEAD_THREADS) void mg_evaluate_narrow_kernel(mg_logits a, HeadNarrow g, const int* __restrict__ actions,
                                                                         float* __restrict__ log_prob, float* __restrict__ entropy) {
  __shared__ unsigned counts[HEAD_THREADS][E + 1];
  for (long row0 = (long)blockIdx.x * g.rows; row0 < a.rows; row0 += (long)gridDim.x * g.rows) {
    if (a.history) head_count_rows<E>(a, g, row0, counts);
    HeadHeld<E, X> h;
    head_place(a, g, row0, h);
    const HeadRow r = head_row(a, h.row);
    head_hold<E, false>(a, g, r, counts[threadIdx.x], h);
    const int act = actions[h.row];
    const bool inside = act >= 0 && act < a.width;
    X d = INFINITY;
#pragma unroll
    for (int e = 0; e < E; e++) if (inside && h.v0 + e == act) d = h.d[e];
    d = head_group_min(d, g.lanes);
    if (h.mine && h.lane == 0) {
      const X log_z = head_log(h.z);
      log_prob[h.row] = h.bad ? NAN : h.empty ? 0.f : (float)(-d - log_z);
      entropy[h.row] = h.bad ? NAN : h.empty ? 0.f : (float)(log_z + h.s / h.z);
    }
  }
}

template <int E, typename X>
__global__ __launch_bounds__(HEAD_THREADS) void mg_evaluate_narrow_backward_kernel(mg_logits a, HeadNarrow g, const int* __restrict__ actions,
                                                                                  const float* __restrict__ dlog_prob,
                                                                                  const float* __restrict__ dentropy,
                                                                                  void* __restrict__ dlogits) {
  __shared__ unsigned counts[HEAD_THREADS][E + 1];
  for (long row0 = (long)blockIdx.x * g.rows; row0 < a.rows; row0 += (long)gridDim.x * g.rows) {
    if (a.history) head_count_rows<E>(a, g, row0, counts);
    HeadHeld<E, X> h;
    head_place(a, g, row0, h);
    const HeadRow r = head_row(a, h.row);
    head_hold<E, true>(a, g, r, counts[threadIdx.x], h);
    const int act = actions[h.row];
    X da = INFINITY;
#pragma unroll
    for (int e = 0; e < E; e++) if (e < h.n && h.v0 + e == act) da = h.x[e] == (X)-INFINITY ? (X)INFINITY : (X)0;
    const bool counts_for = head_group_min(da, g.lanes) == 0;  // the action is a token of the row that is left
    const X gp = dlog_prob && counts_for ? dlog_prob[h.row] : 0.f, gh = dentropy ? dentropy[h.row] : 0.f;
    const X log_z = head_log(h.z), inv_z = 1 / h.z, ent = log_z + h.s * inv_z, inv_temp = (X)r.inv_temp;
    float y[E];
#pragma unroll
    for (int e = 0; e < E; e++) {
      const X q = h.e[e] * inv_z;
      X d = gp * ((h.v0 + e == act ? (X)1 : (X)0) - q) - (h.e[e] > 0 ? gh * q * (ent - log_z - h.d[e]) : 0);
      if (h.bad) d = NAN;
      y[e] = h.empty || h.x[e] == (X)-INFINITY ? 0.f : (float)(d * inv_temp * h.slope[e]);
    }
    if (h.mine) head_store<E>(dlogits, a.type, h.row * a.width + h.v0, h.n, y);
  }
}

// ---- wide rows --------------------------------------------------------------------------------------------------------
// Thread t of a block holds columns part * HEAD_PART + chunk * HEAD_CHUNK + 8 t ... + 7 of each of the part's chunks.

// counts of the n columns from v0 on, all threads together; barriers inside
__device__ __forceinline__ void head_count_columns(const mg_logits& a, long row, unsigned* counts, long v0, int n) {
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += HEAD_THREADS) counts[i] = 0;
  __syncthreads();
  const int* h = a.history + row * a.history_row;
  for (int i = threadIdx.x; i < a.history_len; i += HEAD_THREADS) {
    const long v = (long)h[i] - v0;
    if (h[i] >= 0 && v >= 0 && v < n) atomicAdd(&counts[v], 1u);
  }
  __syncthreads();
}

// over the block; every thread gets the result
template <typename V, typename F>
__device__ __forceinline__ V head_block(V x, V* red, F f) {
  for (int o = 1; o < 64; o <<= 1) x = f(x, __shfl_xor(x, o));
  __syncthreads();
  if (head_lane() == 0) red[threadIdx.x >> 6] = x;
  __syncthreads();
  V y = red[0];
#pragma unroll
  for (int w = 1; w < HEAD_THREADS / 64; w++) y = f(y, red[w]);
  return y;
}
template <typename V>
__device__ __forceinline__ V head_block_max(V x, V* red) {
  return head_block(x, red, [](V a, V b) { return a > b ? a : b; });
}
template <typename V>
__device__ __forceinline__ V head_block_min(V x, V* red) {
  return head_block(x, red, [](V a, V b) { return a < b ? a : b; });
}
template <typename V>
__device__ __forceinline__ V head_block_sum(V x, V* red) {
  return head_block(x, red, [](V a, V b) { return a + b; });
}
// the sum of the threads before this one, and of all
__device__ __forceinline__ double head_block_before(double x, double* red, double& all) {
  const double in_wave = head_group_before(x, 64, head_lane());
  __syncthreads();
  if (head_lane() == 63) red[threadIdx.x >> 6] = in_wave + x;
  __syncthreads();
  double base = 0.0;
  all = 0.0;
#pragma unroll
  for (int w = 0; w < HEAD_THREADS / 64; w++) {
    if (w == (int)(threadIdx.x >> 6)) base = all;
    all += red[w];
  }
  return base + in_wave;
}

#define HEAD_PART_COUNTS()                                                                      \
  __shared__ unsigned counts[HEAD_PART];                                                        \
  const long part0 = (long)blockIdx.x * HEAD_PART;                                              \
  const int part_n = (int)min((long)HEAD_PART, a.width - part0);                                \
  if (a.history) head_count_columns(a, row, counts, part0, part_n);

__global__ __launch_bounds__(HEAD_THREADS) void mg_adjust_wide_kernel(mg_logits a, void* __restrict__ out, const void* __restrict__ dout,
                                                                     void* __restrict__ dlogits) {
  for (long row = blockIdx.y; row < a.rows; row += gridDim.y) {
    HEAD_PART_COUNTS()
    const HeadRow r = head_row(a, row);
#pragma unroll
    for (int c = 0; c < HEAD_CHUNKS; c++) {
      const int at = c * HEAD_CHUNK + threadIdx.x * 8, n = part_n - at;
      if (n <= 0) continue;
      const int v0 = (int)(part0 + at);
      double x[8];
      float slope[8], y[8];
      if (out) {
        head_columns<8, false>(r, a.logits, a.type, row * a.logits_row, v0, n, counts + at, x, slope);
#pragma unroll
        for (int e = 0; e < 8; e++) y[e] = (float)(x[e] * r.inv_temp);
        head_store<8>(out, a.type, row * a.width + v0, n, y);
      } else {
        float go[8];
        head_columns<8, true>(r, a.logits, a.type, row * a.logits_row, v0, n, counts + at, x, slope);
        head_load<8>(dout, a.type, row * a.width + v0, n, go);
#pragma unroll
        for (int e = 0; e < 8; e++) y[e] = slope[e] == 0.f ? 0.f : (float)((double)go[e] * head_slope(r, slope[e]));
        head_store<8>(dlogits, a.type, row * a.width + v0, n, y);
      }
    }
  }
}

// what a part knows: found[row][part] = M, Z, sum d exp(-d) (against its own M), bad, first column of M
template <typename X>
__global__ __launch_bounds__(HEAD_THREADS) void mg_head_parts_kernel(mg_logits a, double* __restrict__ found) {
  __shared__ double red[HEAD_THREADS / 64];
  __shared__ int red_int[HEAD_THREADS / 64];
  for (long row = blockIdx.y; row < a.rows; row += gridDim.y) {
    HEAD_PART_COUNTS()
    const HeadRow r = head_row(a, row);
    X x[HEAD_CHUNKS][8], m = -INFINITY;
    bool bad = false;
#pragma unroll
    for (int c = 0; c < HEAD_CHUNKS; c++) {
      const int at = c * HEAD_CHUNK + threadIdx.x * 8, n = part_n - at;
      if (n > 0) {
        head_columns<8, false>(r, a.logits, a.type, row * a.logits_row, (int)(part0 + at), n, counts + at, x[c], (float*)nullptr);
      } else {
#pragma unroll
        for (int e = 0; e < 8; e++) x[c][e] = -INFINITY;
      }
#pragma unroll
      for (int e = 0; e < 8; e++) {
        if (!(x[c][e] < (X)INFINITY)) bad = true;
        m = x[c][e] > m ? x[c][e] : m;
      }
    }
    const double top = head_block_max((double)m, red);
    const bool any_bad = head_block_max((int)bad, red_int) != 0;
    int first = a.width;
    X z = 0, s = 0;
    const X inv_temp = (X)r.inv_temp, base = any_bad || top == -INFINITY ? (X)0 : (X)top;
#pragma unroll
    for (int c = 0; c < HEAD_CHUNKS; c++) {
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const X d = (base - x[c][e]) * inv_temp, w = head_exp(d);
        z += w;
        s += w > 0 ? d * w : 0;
        if (x[c][e] == base) first = min(first, (int)(part0 + c * HEAD_CHUNK + threadIdx.x * 8 + e));
      }
    }
    const double zz = head_block_sum((double)z, red), ss = head_block_sum((double)s, red);
    first = head_block_min(first, red_int);
    if (threadIdx.x == 0) {
      double* f = found + (row * gridDim.x + blockIdx.x) * HEAD_FOUND;
      f[0] = top; f[1] = zz; f[2] = ss; f[3] = any_bad ? 1.0 : 0.0; f[4] = first;
    }
  }
}

struct HeadJoined { double m, z, s; bool bad, empty; };

// the parts of a row, by all lanes of a wave
__device__ __forceinline__ HeadJoined head_join(const double* f, int parts, double inv_temp, int lane) {
  HeadJoined j;
  double m = -INFINITY, bad = 0.0;
  for (int i = lane; i < parts; i += 64) {
    bad = fmax(bad, f[i * HEAD_FOUND + 3]);
    m = fmax(m, f[i * HEAD_FOUND]);
  }
  j.m = head_group_max(m, 64);
  j.bad = head_group_max(bad, 64) != 0.0;
  j.empty = !j.bad && j.m == -INFINITY;
  double z = 0.0, s = 0.0;
  if (!j.bad && !j.empty)
    for (int i = lane; i < parts; i += 64) {
      const double mi = f[i * HEAD_FOUND];
      if (mi == -INFINITY) continue;
      const double d = (j.m - mi) * inv_temp, w = head_exp(d), zi = f[i * HEAD_FOUND + 1];
      z += w * zi;
      s += w > 0.0 ? w * (f[i * HEAD_FOUND + 2] + d * zi) : 0.0;
    }
  j.z = head_group_sum(z, 64);
  j.s = head_group_sum(s, 64);
  return j;
}

__global__ __launch_bounds__(HEAD_THREADS) void mg_sample_join_kernel(mg_logits a, int parts, const double* __restrict__ found,
                                                                     const float* __restrict__ uniforms, int* __restrict__ actions,
                                                                     float* __restrict__ log_prob, float* __restrict__ entropy) {
  __shared__ unsigned counts[HEAD_CHUNK];
  __shared__ double red[HEAD_THREADS / 64], picked_d, picked_run;
  __shared__ int red_int[HEAD_THREADS / 64], picked;
  for (long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const HeadRow r = head_row(a, row);
    const double* f = found + row * parts * HEAD_FOUND;
    const HeadJoined j = head_join(f, parts, r.inv_temp, head_lane());
    int hit = -1;
    double d_hit = 0.0;
    if (!j.bad && !j.empty) {
      const double target = uniforms ? fmax((double)uniforms[row], 0.0) * j.z : 0.0;
      __syncthreads();
      if (threadIdx.x < 64) {  // one wave finds the part: the first whose running sum is above the target, or the last with any
        double run = 0.0, before = 0.0;
        int part = -1, last = -1, best = a.width;
        for (int i0 = 0; i0 < parts && part < 0; i0 += 64) {
          const int i = i0 + threadIdx.x;
          const double mi = i < parts ? f[i * HEAD_FOUND] : -INFINITY;
          const double w = mi == -INFINITY ? 0.0 : head_exp((j.m - mi) * r.inv_temp) * f[i * HEAD_FOUND + 1];
          const double lead = run + head_group_before(w, 64, head_lane());
          if (!uniforms && mi == j.m) best = min(best, (int)f[i * HEAD_FOUND + 4]);
          const unsigned long long over = __ballot(w > 0.0 && lead + w > target), some = __ballot(w > 0.0);
          if (uniforms && over) {
            const int k = __ffsll((unsigned long long)over) - 1;
            part = i0 + k;
            before = __shfl(lead, k);
          } else if (some) {
            const int k = 63 - __clzll((long long)some);
            last = i0 + k;
            before = __shfl(lead, k);
          }
          run = __shfl(lead + w, 63);
        }
        best = head_group_min(best, 64);
        if (threadIdx.x == 0) picked = !uniforms ? best : part >= 0 ? part : last, picked_run = before;
      }
      __syncthreads();
      if (!uniforms) {
        hit = picked;
      } else {
        const long part0 = (long)picked * HEAD_PART;
        double run = picked_run;
        int last = -1;
        double d_last = 0.0;
        hit = a.width;
        for (int c = 0; c < HEAD_CHUNKS && hit == a.width; c++) {
          const long chunk0 = part0 + c * HEAD_CHUNK;
          const int chunk_n = (int)min((long)HEAD_CHUNK, a.width - chunk0);
          if (chunk_n <= 0) break;
          if (a.history) head_count_columns(a, row, counts, chunk0, chunk_n);
          const int at = threadIdx.x * 8, n = chunk_n - at;
          double x[8], d[8], e8[8], mine = 0.0;
          head_columns<8, false>(r, a.logits, a.type, row * a.logits_row, (int)(chunk0 + at), n, counts + at, x, (float*)nullptr);
#pragma unroll
          for (int e = 0; e < 8; e++) {
            d[e] = (j.m - x[e]) * r.inv_temp;
            e8[e] = head_exp(d[e]);
            mine += e8[e];
          }
          double all;
          double sum = run + head_block_before(mine, red, all);
          int h = a.width, l = -1;
          double dh = 0.0, dl = 0.0;
#pragma unroll
          for (int e = 0; e < 8; e++) {
            sum += e8[e];
            if (sum > target && h == a.width && e < n) h = (int)(chunk0 + at + e), dh = d[e];
            if (e8[e] > 0.0) l = (int)(chunk0 + at + e), dl = d[e];
          }
          const int h_all = head_block_min(h, red_int), l_all = head_block_max(l, red_int);
          if (h_all < a.width && h == h_all) picked_d = dh;
          __syncthreads();
          if (h_all < a.width) {
            hit = h_all;
            d_hit = picked_d;
          } else if (l_all >= 0) {
            if (l == l_all) picked_run = dl;
            __syncthreads();
            last = l_all;
            d_last = picked_run;
          }
          run += all;
        }
        if (hit == a.width) hit = last, d_hit = d_last;  // a uniform of 1 or more, or one that the roundings of a border took
      }
    }
    if (threadIdx.x == 0) {
      const double log_z = head_log(j.z);
      actions[row] = j.bad || j.empty ? -1 : hit;
      log_prob[row] = j.bad ? NAN : j.empty ? 0.f : (float)(-d_hit - log_z);
      entropy[row] = j.bad ? NAN : j.empty ? 0.f : (float)(log_z + j.s / j.z);
    }
    __syncthreads();
  }
}

// one wave per row
__global__ __launch_bounds__(HEAD_THREADS) void mg_evaluate_join_kernel(mg_logits a, int parts, const double* __restrict__ found,
                                                                       const int* __restrict__ actions, float* __restrict__ log_prob,
                                                                       float* __restrict__ entropy, double* __restrict__ stats) {
  const long row = ((long)blockIdx.x * HEAD_THREADS + threadIdx.x) >> 6;
  if (row >= a.rows) return;
  const HeadRow r = head_row(a, row);
  const HeadJoined j = head_join(found + row * parts * HEAD_FOUND, parts, r.inv_temp, head_lane());
  const int act = actions[row];
  const bool inside = act >= 0 && act < a.width;
  double x = -INFINITY;
  if (inside) {
    unsigned count = 0;
    if (a.history) {
      for (int i = head_lane(); i < a.history_len; i += 64) count += a.history[row * a.history_row + i] == act;
      count = head_group_sum(count, 64);
    }
    // (one column, with the bits of its place in a word of the mask)
    HeadRow one = r;
    if (r.kind == MG_ALLOWED_BITS) one.kind = 0;
    double y[1];
    head_columns<1, false>(one, a.logits, a.type, row * a.logits_row, act, 1, &count, y, (float*)nullptr);
    const bool ok = r.kind != MG_ALLOWED_BITS || ((((const unsigned*)r.allowed)[act >> 5] >> (act & 31)) & 1);
    x = ok ? y[0] : -INFINITY;
  }
  if (head_lane() == 0) {
    const double log_z = j.bad || j.empty ? 0.0 : head_log(j.z);
    log_prob[row] = j.bad ? NAN : j.empty ? 0.f : (float)((x - j.m) * r.inv_temp - log_z);
    entropy[row] = j.bad ? NAN : j.empty ? 0.f : (float)(log_z + j.s / j.z);
    if (stats) stats[2 * row] = j.bad ? NAN : j.m, stats[2 * row + 1] = j.bad ? NAN : log_z;
  }
}

template <typename X>
__global__ __launch_bounds__(HEAD_THREADS) void mg_evaluate_wide_backward_kernel(mg_logits a, const int* __restrict__ actions,
                                                                                const float* __restrict__ entropy,
                                                                                const double* __restrict__ stats,
                                                                                const float* __restrict__ dlog_prob,
                                                                                const float* __restrict__ dentropy,
                                                                                void* __restrict__ dlogits) {
  for (long row = blockIdx.y; row < a.rows; row += gridDim.y) {
    HEAD_PART_COUNTS()
    const HeadRow r = head_row(a, row);
    const double m = stats[2 * row];
    const X log_z = (X)stats[2 * row + 1], ent = entropy[row], inv_temp = (X)r.inv_temp;
    const bool bad = m != m, empty = m == -INFINITY;
    const X top = bad || empty ? (X)0 : (X)m;
    const int act = actions[row];
    X gp = 0;
    const X gh = dentropy ? dentropy[row] : 0.f;
    if (dlog_prob && act >= 0 && act < a.width) {  // the action's token is left if it is allowed and not at -infinity
      float l[1], b[1] = {0.f};
      head_load<1>(a.logits, a.type, row * a.logits_row + act, 1, l);
      if (r.bias) b[0] = r.bias[act];
      bool ok = l[0] > -INFINITY && b[0] > -INFINITY;
      if (r.kind == MG_ALLOWED_BOOL) ok = ok && ((const unsigned char*)r.allowed)[act];
      if (r.kind == MG_ALLOWED_BITS) ok = ok && ((((const unsigned*)r.allowed)[act >> 5] >> (act & 31)) & 1);
      if (ok) gp = dlog_prob[row];
    }
#pragma unroll
    for (int c = 0; c < HEAD_CHUNKS; c++) {
      const int at = c * HEAD_CHUNK + threadIdx.x * 8, n = part_n - at;
      if (n <= 0) continue;
      const int v0 = (int)(part0 + at);
      X x[8];
      float slope[8], y[8];
      head_columns<8, true>(r, a.logits, a.type, row * a.logits_row, v0, n, counts + at, x, slope);
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const X d = (top - x[e]) * inv_temp, q = head_exp(d + log_z);
        X g = gp * ((v0 + e == act ? (X)1 : (X)0) - q) + (q > 0 ? gh * q * (d + log_z - ent) : 0);
        if (bad) g = NAN;
        y[e] = empty || x[e] == (X)-INFINITY ? 0.f : (float)(g * inv_temp * slope[e]);
      }
      head_store<8>(dlogits, a.type, row * a.width + v0, n, y);
    }
  }
}

// ---- host side --------------------------------------------------------------------------------------------------------

static int head_check(const char* who, const mg_logits* a) {
  const std::string w(who);
  if (!a) return mg_fail_msg(w + ": NULL arguments");
  if (a->rows < 0 || a->width < 1) return mg_fail_msg(w + ": a row has at least one token");
  if (a->type < 0 || a->type > 2) return mg_fail_msg(w + ": type must be MG_F32, MG_BF16 or MG_F16");
  if (!(a->temperature > 0.0 && a->temperature < INFINITY)) return mg_fail_msg(w + ": temperature must be positive and finite");
  if (!(a->repetition > 0.0 && a->repetition < INFINITY)) return mg_fail_msg(w + ": repetition must be positive and finite");
  if (!(std::abs(a->presence) < INFINITY && std::abs(a->frequency) < INFINITY)) return mg_fail_msg(w + ": penalties must be finite");
  if (a->allowed && a->allowed_kind != MG_ALLOWED_BOOL && a->allowed_kind != MG_ALLOWED_BITS)
    return mg_fail_msg(w + ": allowed_kind must be MG_ALLOWED_BOOL or MG_ALLOWED_BITS");
  if (a->history && (a->history_len < 1 || a->history_len > 1 << 30)) return mg_fail_msg(w + ": a history has 1 to 2^30 entries");
  if (a->rows && !a->logits) return mg_fail_msg(w + ": NULL tensor");
  return 0;
}

static int head_parts(const mg_logits* a) { return (int)(((int64_t)a->width + HEAD_PART - 1) / HEAD_PART); }
static dim3 head_wide_grid(const mg_logits* a) { return dim3(head_parts(a), (unsigned)(a->rows < 32768 ? a->rows : 32768)); }
static bool head_narrow(const mg_logits* a) { return a->width <= HEAD_NARROW; }

// lanes per row: as many as hold the row with E columns each
static HeadNarrow head_layout(const mg_logits* a, int e) {
  int lanes = 1;
  while (lanes * e < a->width) lanes *= 2;
  return HeadNarrow{lanes, HEAD_THREADS / lanes};
}
static unsigned head_blocks(int64_t rows, int per_block) {
  const int64_t n = (rows + per_block - 1) / per_block;
  return (unsigned)(n < (1 << 23) ? n : 1 << 23);  // (a grid has fewer than 2^32 threads; the kernels loop)
}

template <int V> using head_int = std::integral_constant<int, V>;
template <typename F>
static void head_by_width(const mg_logits* a, F f) {
  if (a->width <= 64 * 8) f(head_int<8>(), head_layout(a, 8));
  else f(head_int<16>(), head_layout(a, 16));
}
// the arithmetic of given actions: 64 bits where a bias or a penalty could cancel large logits
template <typename F>
static void head_by_controls(const mg_logits* a, F f) {
  if (a->bias || a->history) f((double*)nullptr);
  else f((float*)nullptr);
}

static int head_launched(const char* who) {
  const hipError_t err = hipGetLastError();
  return err == hipSuccess ? 0 : mg_fail_msg(std::string(who) + ": " + hipGetErrorString(err));
}
static int head_workspace(const char* who, const mg_logits* a) {
  if (!head_narrow(a) && (!a->workspace || a->workspace_bytes < mg_logits_workspace(a)))
    return mg_fail_msg(std::string(who) + ": workspace smaller than mg_logits_workspace says");
  return 0;
}

extern "C" int64_t mg_logits_workspace(const mg_logits* a) {
  if (!a || a->rows <= 0 || a->width < 1 || head_narrow(a)) return 0;
  return a->rows * head_parts(a) * HEAD_FOUND * (int64_t)sizeof(double);
}

static int head_adjust(const char* who, const mg_logits* a, void* out, const void* dout, void* dlogits, void* stream) {
  const hipStream_t s = (hipStream_t)stream;
  if (head_narrow(a))
    head_by_width(a, [&](auto e, HeadNarrow g) {
      hipLaunchKernelGGL(mg_adjust_narrow_kernel<decltype(e)::value>, dim3(head_blocks(a->rows, g.rows)), dim3(HEAD_THREADS), 0, s, *a, g, out, dout, dlogits);
    });
  else
    hipLaunchKernelGGL(mg_adjust_wide_kernel, head_wide_grid(a), dim3(HEAD_THREADS), 0, s, *a, out, dout, dlogits);
  return head_launched(who);
}

extern "C" int mg_adjust_logits(const mg_logits* a, void* out, void* stream) try {
  if (const int rc = head_check("mg_adjust_logits", a)) return rc;
  if (!a->rows) return 0;
  if (!out) return mg_fail_msg("mg_adjust_logits: NULL tensor");
  return head_adjust("mg_adjust_logits", a, out, nullptr, nullptr, stream);
} catch (...) {
  return 1;
}

extern "C" int mg_adjust_logits_backward(const mg_logits* a, const void* dout, void* dlogits, void* stream) try {
  if (const int rc = head_check("mg_adjust_logits_backward", a)) return rc;
  if (!a->rows) return 0;
  if (!dout || !dlogits) return mg_fail_msg("mg_adjust_logits_backward: NULL tensor");
  return head_adjust("mg_adjust_logits_backward", a, nullptr, dout, dlogits, stream);
} catch (...) {
  return 1;
}

extern "C" int mg_sample_actions(const mg_logits* a, const float* uniforms, int32_t* actions, float* log_prob,
                                 float* entropy, void* stream) try {
  static const char who[] = "mg_sample_actions";
  if (const int rc = head_check(who, a)) return rc;
  if (!a->rows) return 0;
  if (!actions || !log_prob || !entropy) return mg_fail_msg(std::string(who) + ": NULL tensor");
  if (const int rc = head_workspace(who, a)) return rc;
  const hipStream_t s = (hipStream_t)stream;
  if (head_narrow(a)) {
    head_by_width(a, [&](auto e, HeadNarrow g) {
      hipLaunchKernelGGL(mg_sample_narrow_kernel<decltype(e)::value>, dim3(head_blocks(a->rows, g.rows)), dim3(HEAD_THREADS), 0, s, *a, g,
                         uniforms, actions, log_prob, entropy);
    });
  } else {
    hipLaunchKernelGGL(mg_head_parts_kernel<double>, head_wide_grid(a), dim3(HEAD_THREADS), 0, s, *a, (double*)a->workspace);
    hipLaunchKernelGGL(mg_sample_join_kernel, dim3(head_blocks(a->rows, 1)), dim3(HEAD_THREADS), 0, s, *a, head_parts(a),
                       (const double*)a->workspace, uniforms, actions, log_prob, entropy);
  }
  return head_launched(who);
} catch (...) {
  return 1;
}

extern "C" int mg_evaluate_actions(const mg_logits* a, const int32_t* actions, float* log_prob, float* entropy,
                                   double* stats, void* stream) try {
  static const char who[] = "mg_evaluate_actions";
  if (const int rc = head_check(who, a)) return rc;
  if (!a->rows) return 0;
  if (!actions || !log_prob || !entropy) return mg_fail_msg(std::string(who) + ": NULL tensor");
  if (const int rc = head_workspace(who, a)) return rc;
  const hipStream_t s = (hipStream_t)stream;
  head_by_controls(a, [&](auto* null) {
    using X = std::remove_pointer_t<decltype(null)>;
    if (head_narrow(a)) {
      head_by_width(a, [&](auto e, HeadNarrow g) {
        hipLaunchKernelGGL((mg_evaluate_narrow_kernel<decltype(e)::value, X>), dim3(head_blocks(a->rows, g.rows)), dim3(HEAD_THREADS), 0, s,
                           *a, g, actions, log_prob, entropy);
      });
    } else {
      hipLaunchKernelGGL(mg_head_parts_kernel<X>, head_wide_grid(a), dim3(HEAD_THREADS), 0, s, *a, (double*)a->workspace);
    }
  });
  if (!head_narrow(a))
    hipLaunchKernelGGL(mg_evaluate_join_kernel, dim3((unsigned)((a->rows + 3) / 4)), dim3(HEAD_THREADS), 0, s, *a, head_parts(a),
                       (const double*)a->workspace, actions, log_prob, entropy, stats);
  return head_launched(who);
} catch (...) {
  return 1;
}

extern "C" int mg_evaluate_actions_backward(const mg_logits* a, const int32_t* actions, const float* entropy,
                                            const double* stats, const float* dlog_prob, const float* dentropy,
                                            void* dlogits, void* stream) try {
  static const char who[] = "mg_evaluate_actions_backward";
  if (const int rc = head_check(who, a)) return rc;
  if (!a->rows) return 0;
  if (!actions || !dlogits || (!head_narrow(a) && (!entropy || !stats))) return mg_fail_msg(std::string(who) + ": NULL tensor");
  const hipStream_t s = (hipStream_t)stream;
  head_by_controls(a, [&](auto* null) {
    using X = std::remove_pointer_t<decltype(null)>;
    if (head_narrow(a))
      head_by_width(a, [&](auto e, HeadNarrow g) {
        hipLaunchKernelGGL((mg_evaluate_narrow_backward_kernel<decltype(e)::value, X>), dim3(head_blocks(a->rows, g.rows)), dim3(HEAD_THREADS),
                           0, s, *a, g, actions, dlog_prob, dentropy, dlogits);
      });
    else
      hipLaunchKernelGGL(mg_evaluate_wide_backward_kernel<X>, head_wide_grid(a), dim3(HEAD_THREADS), 0, s, *a, actions, entropy, stats,
                         dlog_prob, dentropy, dlogits);
  });
  return head_launched(who);
} catch (...) {
  return 1;
}
