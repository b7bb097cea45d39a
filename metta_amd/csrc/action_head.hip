// action_head.hip -- the head between a policy's logits and its actions for gfx950: adjusted logits, sampling, and the
// log-probability and entropy of given actions, with gradients (mg_adjust_logits, mg_sample_actions,
// mg_evaluate_actions and their backward forms).
//
// Per row, with c = how often token v stands in the row's history:
//   l1 = c > 0 ? (l > 0 ? l / repetition : l * repetition) : l        l2 = l1 - frequency * c - presence * (c > 0)
//   l4 = allowed ? (l2 + bias) / temperature : -infinity
//   M = max l4, Z = sum exp(l4 - M), q = exp(l4 - M) / Z, H = log Z + sum (M - l4) q
//   sampled: the first v with sum_{w <= v} exp(l4_w - M) > u Z;  without u: the first v with l4 = M
// A row with nothing left (M = -infinity) has action -1, log-probability 0, entropy 0 and no gradient; a row with NaN
// or +infinity among its allowed tokens has action -1 and NaN.
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <string>

#include "../../include/mettagrid_hip.h"

#define HEAD_THREADS 256
#define HEAD_TILE 4096  // columns whose counts are held in LDS at a time

extern int mg_fail_msg(const std::string& m);  // mettagrid_hip.hip: sets mg_last_error(), returns 1

__device__ __forceinline__ float head_up(float v) { return v; }
__device__ __forceinline__ float head_up(__hip_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float head_up(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T head_down(double v);
template <> __device__ __forceinline__ float head_down<float>(double v) { return (float)v; }
template <> __device__ __forceinline__ __hip_bfloat16 head_down<__hip_bfloat16>(double v) { return __float2bfloat16((float)v); }
template <> __device__ __forceinline__ __half head_down<__half>(double v) { return __float2half((float)v); }

// One row's controls.  A value is adjusted in 64 bits: a picked action must not depend on how 32-bit roundings fall.
struct HeadRow {
  const float* bias;
  const void* allowed;
  const int* history;
  int history_len, kind;
  double inv_rep, rep, presence, frequency, inv_temp;
};

__device__ __forceinline__ HeadRow head_row(const mg_logits& a, long row) {
  HeadRow r;
  r.bias = a.bias ? a.bias + row * a.bias_row : nullptr;
  r.kind = a.allowed ? a.allowed_kind : 0;
  r.allowed = !a.allowed ? nullptr : a.allowed_kind == MG_ALLOWED_BOOL ? (const void*)((const unsigned char*)a.allowed + row * a.allowed_row)
                                                                       : (const void*)((const int*)a.allowed + row * a.allowed_row);
  r.history = a.history ? a.history + row * a.history_row : nullptr;
  r.history_len = a.history ? a.history_len : 0;
  r.rep = a.repetition; r.inv_rep = 1.0 / a.repetition;
  r.presence = a.presence; r.frequency = a.frequency; r.inv_temp = 1.0 / a.temperature;
  return r;
}

__device__ __forceinline__ bool head_allowed(const HeadRow& r, int v) {
  if (r.kind == MG_ALLOWED_BOOL) return ((const unsigned char*)r.allowed)[v] != 0;
  if (r.kind == MG_ALLOWED_BITS) return (((const unsigned*)r.allowed)[v >> 5] >> (v & 31)) & 1;
  return true;
}

__device__ __forceinline__ double head_adjust(const HeadRow& r, float l, int v, unsigned count) {
  if (!head_allowed(r, v)) return -INFINITY;
  double d = l;
  if (count) d = (d > 0 ? d * r.inv_rep : d * r.rep) - r.frequency * count - r.presence;
  if (r.bias) d += r.bias[v];
  return d * r.inv_temp;
}

__device__ __forceinline__ double head_slope(const HeadRow& r, float l, int v, unsigned count) {
  if (!head_allowed(r, v)) return 0.0;
  return count ? (l > 0 ? r.inv_temp * r.inv_rep : r.inv_temp * r.rep) : r.inv_temp;
}

// counts[v - v0] of the row's history for the tile's n columns; barriers inside
__device__ void head_count(const HeadRow& r, unsigned* counts, int v0, int n) {
  if (!r.history) return;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += HEAD_THREADS) counts[i] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < r.history_len; i += HEAD_THREADS) {
    const int v = r.history[i] - v0;
    if (r.history[i] >= 0 && v >= 0 && v < n) atomicAdd(&counts[v], 1u);
  }
  __syncthreads();
}

// over all threads of the block; every thread gets the result
template <typename F>
__device__ double head_reduce(double x, double* red, F f) {
  __syncthreads();
  red[threadIdx.x] = x;
  for (int s = HEAD_THREADS / 2; s; s /= 2) {
    __syncthreads();
    if (threadIdx.x < s) red[threadIdx.x] = f(red[threadIdx.x], red[threadIdx.x + s]);
  }
  __syncthreads();
  return red[0];
}
__device__ double head_sum(double x, double* red) {
  return head_reduce(x, red, [](double p, double q) { return p + q; });
}

#define HEAD_EACH(...)                                                                       \
  for (int v0 = 0; v0 < a.width; v0 += HEAD_TILE) {                                          \
    const int n = min(HEAD_TILE, a.width - v0);                                              \
    head_count(r, counts, v0, n);                                                            \
    for (int i = threadIdx.x; i < n; i += HEAD_THREADS) {                                    \
      const int v = v0 + i;                                                                  \
      const unsigned count = r.history ? counts[i] : 0u;                                     \
      const float l = head_up(logits[v]);                                                    \
      __VA_ARGS__                                                                            \
    }                                                                                        \
  }

template <typename T>
__global__ __launch_bounds__(HEAD_THREADS) void mg_adjust_logits_kernel(mg_logits a, T* __restrict__ out,
                                                                       const T* __restrict__ dout,
                                                                       T* __restrict__ dlogits) {
  __shared__ unsigned counts[HEAD_TILE];
  for (long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const HeadRow r = head_row(a, row);
    const T* logits = (const T*)a.logits + row * a.logits_row;
    HEAD_EACH({
      if (out) out[row * a.width + v] = head_down<T>(head_adjust(r, l, v, count));
      if (dlogits) {
        const double s = head_slope(r, l, v, count);
        dlogits[row * a.width + v] = s == 0.0 ? head_down<T>(0.0) : head_down<T>(s * head_up(dout[row * a.width + v]));
      }
    })
  }
}

struct HeadStats { double m, z, s; bool bad, empty; };  // s = sum (m - l4) exp(l4 - m)

template <typename T>
__device__ HeadStats head_stats(const mg_logits& a, const HeadRow& r, const T* logits, unsigned* counts, double* red) {
  HeadStats st;
  double m = -INFINITY, bad = 0.0;
  HEAD_EACH({
    const double x = head_adjust(r, l, v, count);
    if (!(x < INFINITY)) bad = 1.0;
    m = fmax(m, x);
  })
  st.bad = head_sum(bad, red) > 0.0;
  st.m = head_reduce(m, red, [](double p, double q) { return fmax(p, q); });
  st.empty = !st.bad && st.m == -INFINITY;
  st.z = st.s = 0.0;
  if (st.bad || st.empty) return st;
  double z = 0.0, s = 0.0;
  HEAD_EACH({
    const double d = st.m - head_adjust(r, l, v, count);
    const double e = exp(-d);
    z += e;
    if (e > 0.0) s += d * e;
  })
  st.z = head_sum(z, red);
  st.s = head_sum(s, red);
  return st;
}

template <typename T>
__global__ __launch_bounds__(HEAD_THREADS) void mg_sample_actions_kernel(mg_logits a, const float* __restrict__ uniforms,
                                                                         int* __restrict__ actions,
                                                                         float* __restrict__ log_prob,
                                                                         float* __restrict__ entropy) {
  __shared__ unsigned counts[HEAD_TILE];
  __shared__ double red[HEAD_THREADS];
  __shared__ int hit, last;
  for (long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const HeadRow r = head_row(a, row);
    const T* logits = (const T*)a.logits + row * a.logits_row;
    const HeadStats st = head_stats(a, r, logits, counts, red);
    if (threadIdx.x == 0) hit = a.width, last = -1;
    __syncthreads();
    if (!st.bad && !st.empty) {
      const double target = uniforms ? (double)uniforms[row] * st.z : 0.0;
      double base = 0.0;  // the sum before the current 256 columns
      for (int v0 = 0; v0 < a.width; v0 += HEAD_TILE) {
        const int n = min(HEAD_TILE, a.width - v0);
        head_count(r, counts, v0, n);
        for (int i0 = 0; i0 < n; i0 += HEAD_THREADS) {
          const int i = i0 + threadIdx.x, v = v0 + i;
          const double x = i < n ? head_adjust(r, head_up(logits[v]), v, r.history ? counts[i] : 0u) : -INFINITY;
          const double e = exp(x - st.m);
          if (!uniforms) {
            if (x == st.m) atomicMin(&hit, v);
            continue;
          }
          if (e > 0.0) atomicMax(&last, v);
          __syncthreads();
          red[threadIdx.x] = e;
          __syncthreads();
          double sum = base;
          for (int k = 0; k <= threadIdx.x; k++) sum += red[k];
          if (i < n && sum > target) atomicMin(&hit, v);
          __syncthreads();
          for (int k = 0; k < HEAD_THREADS; k++) base += red[k];
        }
      }
    }
    __syncthreads();
    const int v = hit < a.width ? hit : last;
    unsigned count = 0;
    if (v >= 0)
      for (int i = 0; i < r.history_len; i++) count += r.history[i] == v;
    if (threadIdx.x == 0) {
      const bool none = st.bad || st.empty || v < 0;
      actions[row] = none ? -1 : v;
      const double lp = none ? 0.0 : head_adjust(r, head_up(logits[v]), v, count) - st.m - log(st.z);
      log_prob[row] = st.bad ? NAN : (float)lp;
      entropy[row] = st.bad ? NAN : none ? 0.f : (float)(log(st.z) + st.s / st.z);
    }
    __syncthreads();
  }
}

template <typename T>
__global__ __launch_bounds__(HEAD_THREADS) void mg_evaluate_actions_kernel(mg_logits a, const int* __restrict__ actions,
                                                                           float* __restrict__ log_prob,
                                                                           float* __restrict__ entropy,
                                                                           double* __restrict__ stats) {
  __shared__ unsigned counts[HEAD_TILE];
  __shared__ double red[HEAD_THREADS];
  for (long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const HeadRow r = head_row(a, row);
    const T* logits = (const T*)a.logits + row * a.logits_row;
    const HeadStats st = head_stats(a, r, logits, counts, red);
    const int v = actions[row];
    if (threadIdx.x == 0) {
      unsigned count = 0;
      const bool inside = v >= 0 && v < a.width;
      if (inside)
        for (int i = 0; i < r.history_len; i++) count += r.history[i] == v;
      const double x = inside ? head_adjust(r, head_up(logits[v]), v, count) : -INFINITY;
      log_prob[row] = st.bad ? NAN : st.empty ? 0.f : (float)(x - st.m - log(st.z));
      entropy[row] = st.bad ? NAN : st.empty ? 0.f : (float)(log(st.z) + st.s / st.z);
      if (stats) {
        stats[2 * row] = st.bad ? NAN : st.m;
        stats[2 * row + 1] = st.bad ? NAN : st.empty ? 0.0 : log(st.z);
      }
    }
  }
}

template <typename T>
__global__ __launch_bounds__(HEAD_THREADS) void mg_evaluate_actions_backward_kernel(
    mg_logits a, const int* __restrict__ actions, const float* __restrict__ entropy, const double* __restrict__ stats,
    const float* __restrict__ dlog_prob, const float* __restrict__ dentropy, T* __restrict__ dlogits) {
  __shared__ unsigned counts[HEAD_TILE];
  for (long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const HeadRow r = head_row(a, row);
    const T* logits = (const T*)a.logits + row * a.logits_row;
    const double m = stats[2 * row], log_z = stats[2 * row + 1], h = entropy[row];
    const int act = actions[row];
    const double gh = dentropy ? dentropy[row] : 0.0;
    double gp = dlog_prob ? dlog_prob[row] : 0.0;
    if (act < 0 || act >= a.width) {
      gp = 0.0;
    } else {
      unsigned count = 0;
      for (int i = 0; i < r.history_len; i++) count += r.history[i] == act;
      if (head_adjust(r, head_up(logits[act]), act, count) == -INFINITY) gp = 0.0;
    }
    HEAD_EACH({
      const double x = head_adjust(r, l, v, count);
      double d = 0.0;
      if (!(x == -INFINITY)) {
        const double lq = (x - m) - log_z, q = exp(lq);
        d = gp * ((v == act ? 1.0 : 0.0) - q) - (q > 0.0 ? gh * q * (lq + h) : 0.0);
        if (q != q) d = NAN;
        d *= head_slope(r, l, v, count);
      }
      dlogits[row * a.width + v] = head_down<T>(d);
    })
  }
}

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
  if (a->history && a->history_len < 0) return mg_fail_msg(w + ": negative shape");
  if (a->rows && !a->logits) return mg_fail_msg(w + ": NULL tensor");
  return 0;
}

static unsigned head_blocks(const mg_logits* a) { return (unsigned)(a->rows < 65536 ? a->rows : 65536); }

template <typename F>
static int head_by_type(const char* who, int type, F f) {
  if (type == MG_F32) f((float*)nullptr);
  else if (type == MG_BF16) f((__hip_bfloat16*)nullptr);
  else f((__half*)nullptr);
  const hipError_t err = hipGetLastError();
  return err == hipSuccess ? 0 : mg_fail_msg(std::string(who) + ": " + hipGetErrorString(err));
}
#define HEAD_TYPE(p) std::remove_pointer_t<decltype(p)>

extern "C" int mg_adjust_logits(const mg_logits* a, void* out, void* stream) try {
  if (const int rc = head_check("mg_adjust_logits", a)) return rc;
  if (!a->rows) return 0;
  if (!out) return mg_fail_msg("mg_adjust_logits: NULL tensor");
  return head_by_type("mg_adjust_logits", a->type, [&](auto* p) {
    using T = HEAD_TYPE(p);
    hipLaunchKernelGGL(mg_adjust_logits_kernel<T>, dim3(head_blocks(a)), dim3(HEAD_THREADS), 0, (hipStream_t)stream, *a,
                       (T*)out, (const T*)nullptr, (T*)nullptr);
  });
} catch (...) {
  return 1;
}

extern "C" int mg_adjust_logits_backward(const mg_logits* a, const void* dout, void* dlogits, void* stream) try {
  if (const int rc = head_check("mg_adjust_logits_backward", a)) return rc;
  if (!a->rows) return 0;
  if (!dout || !dlogits) return mg_fail_msg("mg_adjust_logits_backward: NULL tensor");
  return head_by_type("mg_adjust_logits_backward", a->type, [&](auto* p) {
    using T = HEAD_TYPE(p);
    hipLaunchKernelGGL(mg_adjust_logits_kernel<T>, dim3(head_blocks(a)), dim3(HEAD_THREADS), 0, (hipStream_t)stream, *a,
                       (T*)nullptr, (const T*)dout, (T*)dlogits);
  });
} catch (...) {
  return 1;
}

extern "C" int mg_sample_actions(const mg_logits* a, const float* uniforms, int32_t* actions, float* log_prob,
                                 float* entropy, void* stream) try {
  if (const int rc = head_check("mg_sample_actions", a)) return rc;
  if (!a->rows) return 0;
  if (!actions || !log_prob || !entropy) return mg_fail_msg("mg_sample_actions: NULL tensor");
  return head_by_type("mg_sample_actions", a->type, [&](auto* p) {
    using T = HEAD_TYPE(p);
    hipLaunchKernelGGL(mg_sample_actions_kernel<T>, dim3(head_blocks(a)), dim3(HEAD_THREADS), 0, (hipStream_t)stream, *a,
                       uniforms, actions, log_prob, entropy);
  });
} catch (...) {
  return 1;
}

extern "C" int mg_evaluate_actions(const mg_logits* a, const int32_t* actions, float* log_prob, float* entropy,
                                   double* stats, void* stream) try {
  if (const int rc = head_check("mg_evaluate_actions", a)) return rc;
  if (!a->rows) return 0;
  if (!actions || !log_prob || !entropy) return mg_fail_msg("mg_evaluate_actions: NULL tensor");
  return head_by_type("mg_evaluate_actions", a->type, [&](auto* p) {
    using T = HEAD_TYPE(p);
    hipLaunchKernelGGL(mg_evaluate_actions_kernel<T>, dim3(head_blocks(a)), dim3(HEAD_THREADS), 0, (hipStream_t)stream, *a,
                       actions, log_prob, entropy, stats);
  });
} catch (...) {
  return 1;
}

extern "C" int mg_evaluate_actions_backward(const mg_logits* a, const int32_t* actions, const float* entropy,
                                            const double* stats, const float* dlog_prob, const float* dentropy,
                                            void* dlogits, void* stream) try {
  if (const int rc = head_check("mg_evaluate_actions_backward", a)) return rc;
  if (!a->rows) return 0;
  if (!actions || !entropy || !stats || !dlogits) return mg_fail_msg("mg_evaluate_actions_backward: NULL tensor");
  return head_by_type("mg_evaluate_actions_backward", a->type, [&](auto* p) {
    using T = HEAD_TYPE(p);
    hipLaunchKernelGGL(mg_evaluate_actions_backward_kernel<T>, dim3(head_blocks(a)), dim3(HEAD_THREADS), 0, (hipStream_t)stream,
                       *a, actions, entropy, stats, dlog_prob, dentropy, (T*)dlogits);
  });
} catch (...) {
  return 1;
}
