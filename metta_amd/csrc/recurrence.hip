// recurrence.hip -- gated linear recurrence over segments, its gradients and its one-step form for gfx950
// (mg_gated_recurrence, mg_gated_recurrence_backward).
//
// Per row and column, with a = sigmoid(gate):   h[t] = a[t] * (resets[t] ? 0 : h[t-1]) + (1 - a[t]) * x[t]
// and backwards, with d[t] = dh[t] + (resets[t+1] ? 0 : a[t+1] * d[t+1]):
//   dx[t] = (1 - a[t]) d[t]      dgate[t] = d[t] (h_before[t] - x[t]) a[t] (1 - a[t])      dstate = a[0] d[0]
//
// x, gate, h and their gradients are f32, bf16 or f16; the state, the products along time and the running gradient are
// f32 throughout, h and the gradients are rounded once when they are stored.
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <string>

#include "../../include/mettagrid_hip.h"

#define REC_MARK MG_RECURRENCE_MARK_STEPS  // the state entering every REC_MARK-th step is kept for the backward pass

extern int mg_fail_msg(const std::string& m);  // mettagrid_hip.hip: sets mg_last_error(), returns 1

__device__ __forceinline__ float rec_up(float v) { return v; }
__device__ __forceinline__ float rec_up(__hip_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float rec_up(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T rec_down(float v);
template <> __device__ __forceinline__ float rec_down<float>(float v) { return v; }
template <> __device__ __forceinline__ __hip_bfloat16 rec_down<__hip_bfloat16>(float v) { return __float2bfloat16(v); }
template <> __device__ __forceinline__ __half rec_down<__half>(float v) { return __float2half(v); }

// sigmoid(g) and sigmoid(-g) from one exponential of -|g|: neither overflows, neither is 1 minus the other (which would
// lose the small one's digits); both are exact at +-infinity.
__device__ __forceinline__ void rec_gate(float g, float& a, float& w) {
  const float e = expf(-fabsf(g));
  const float big = 1.0f / (1.0f + e), small = e * big;
  a = g >= 0.f ? big : small;
  w = g >= 0.f ? small : big;
  if (g != g) a = w = g;
}

struct RecArgs {
  const void *x, *gate;
  const float* state;           // [rows][width], or null: zeros
  const unsigned char* resets;  // [rows][steps], or null: none
  long rows, steps, width;
  long x_row, x_step, g_row, g_step;  // in elements; columns are adjacent
};

template <typename T>
__global__ __launch_bounds__(256) void mg_recurrence_kernel(RecArgs a, T* __restrict__ h, float* __restrict__ last,
                                                            float* __restrict__ marks) {
  const long gid = (long)blockIdx.x * 256 + threadIdx.x;
  if (gid >= a.rows * a.width) return;
  const long row = gid / a.width, col = gid - row * a.width;
  const T* x = (const T*)a.x + row * a.x_row + col;
  const T* g = (const T*)a.gate + row * a.g_row + col;
  const unsigned char* rs = a.resets ? a.resets + row * a.steps : nullptr;
  const long nmarks = (a.steps - 1) / REC_MARK;
  float s = a.state ? a.state[gid] : 0.f;
  for (long t = 0; t < a.steps; t++) {
    if (marks && t && t % REC_MARK == 0) marks[(row * nmarks + t / REC_MARK - 1) * a.width + col] = s;
    float ga, gw;
    rec_gate(rec_up(g[t * a.g_step]), ga, gw);
    const float b = gw * rec_up(x[t * a.x_step]);
    s = rs && rs[t] ? b : fmaf(ga, s, b);
    if (h) h[(row * a.steps + t) * a.width + col] = rec_down<T>(s);
  }
  last[gid] = s;
}

struct RecMarks {  // the state entering step k * REC_MARK, k >= 1, is p[row * row_stride + (k - 1) * stride + column]
  const float* p;
  long row_stride, stride;
};

template <typename T>
__global__ __launch_bounds__(256) void mg_recurrence_backward_kernel(RecArgs a, RecMarks m, const T* __restrict__ dh,
                                                                     long dh_row, long dh_step,
                                                                     const float* __restrict__ dlast, T* __restrict__ dx,
                                                                     long dx_row, long dx_step, T* __restrict__ dgate,
                                                                     long dg_row, long dg_step,
                                                                     float* __restrict__ dstate) {
  const long gid = (long)blockIdx.x * 256 + threadIdx.x;
  if (gid >= a.rows * a.width) return;
  const long row = gid / a.width, col = gid - row * a.width;
  const T* x = (const T*)a.x + row * a.x_row + col;
  const T* g = (const T*)a.gate + row * a.g_row + col;
  const unsigned char* rs = a.resets ? a.resets + row * a.steps : nullptr;
  float d = dlast ? dlast[gid] : 0.f;
  for (long k = (a.steps - 1) / REC_MARK; k >= 0; k--) {
    const long t0 = k * REC_MARK;
    const int n = (int)min((long)REC_MARK, a.steps - t0);
    float before[REC_MARK];
    float s = k ? m.p[row * m.row_stride + (k - 1) * m.stride + col] : a.state ? a.state[gid] : 0.f;
    for (int i = 0; i < n; i++) {
      float ga, gw;
      rec_gate(rec_up(g[(t0 + i) * a.g_step]), ga, gw);
      const float b = gw * rec_up(x[(t0 + i) * a.x_step]);
      before[i] = rs && rs[t0 + i] ? 0.f : s;
      s = rs && rs[t0 + i] ? b : fmaf(ga, s, b);
    }
    for (int i = n - 1; i >= 0; i--) {
      const long t = t0 + i;
      float ga, gw;
      rec_gate(rec_up(g[t * a.g_step]), ga, gw);
      if (dh) d += rec_up(dh[row * dh_row + t * dh_step + col]);
      dx[row * dx_row + t * dx_step + col] = rec_down<T>(gw * d);
      dgate[row * dg_row + t * dg_step + col] = rec_down<T>(d * (before[i] - rec_up(x[t * a.x_step])) * (ga * gw));
      d = rs && rs[t] ? 0.f : ga * d;
    }
  }
  if (dstate) dstate[gid] = d;
}

static int rec_check(const char* who, const mg_recurrence* r) {
  if (!r) return mg_fail_msg(std::string(who) + ": NULL arguments");
  if (r->rows < 0 || r->steps < 0 || r->width < 0) return mg_fail_msg(std::string(who) + ": negative shape");
  if (r->type < 0 || r->type > 2) return mg_fail_msg(std::string(who) + ": type must be MG_F32, MG_BF16 or MG_F16");
  if (r->rows && r->width && r->rows > ((int64_t)1 << 31) / r->width)
    return mg_fail_msg(std::string(who) + ": rows * width must not exceed 2^31");
  if (r->rows && r->steps && r->width && (!r->x || !r->gate)) return mg_fail_msg(std::string(who) + ": NULL tensor");
  return 0;
}

static RecArgs rec_args(const mg_recurrence* r) {
  return RecArgs{r->x,      r->gate,  r->state,     r->resets,    (long)r->rows,
                 (long)r->steps, (long)r->width, (long)r->x_row, (long)r->x_step, (long)r->gate_row, (long)r->gate_step};
}

template <typename F>
static int rec_by_type(int type, F f) {
  if (type == MG_F32) return f((float*)nullptr);
  if (type == MG_BF16) return f((__hip_bfloat16*)nullptr);
  return f((__half*)nullptr);
}

static int rec_launched(const char* who) {
  const hipError_t err = hipGetLastError();
  return err == hipSuccess ? 0 : mg_fail_msg(std::string(who) + ": " + hipGetErrorString(err));
}

extern "C" int mg_gated_recurrence(const mg_recurrence* r, void* h, float* last, float* marks, void* stream) try {
  static const char who[] = "mg_gated_recurrence";
  if (const int rc = rec_check(who, r)) return rc;
  if (!r->rows || !r->steps || !r->width) return 0;
  if (!last) return mg_fail_msg(std::string(who) + ": NULL tensor");
  const unsigned blocks = (unsigned)((r->rows * r->width + 255) / 256);
  return rec_by_type(r->type, [&](auto* p) {
    using T = std::remove_pointer_t<decltype(p)>;
    hipLaunchKernelGGL(mg_recurrence_kernel<T>, dim3(blocks), dim3(256), 0, (hipStream_t)stream, rec_args(r), (T*)h, last, marks);
    return rec_launched(who);
  });
} catch (...) {
  return 1;
}

extern "C" int mg_gated_recurrence_backward(const mg_recurrence* r, const float* marks, int64_t marks_row,
                                            int64_t marks_stride, const mg_recurrence_gradients* d, void* stream) try {
  static const char who[] = "mg_gated_recurrence_backward";
  if (const int rc = rec_check(who, r)) return rc;
  if (!r->rows || !r->steps || !r->width) return 0;
  if (!d || !d->dx || !d->dgate || (!marks && r->steps > REC_MARK)) return mg_fail_msg(std::string(who) + ": NULL tensor");
  const unsigned blocks = (unsigned)((r->rows * r->width + 255) / 256);
  return rec_by_type(r->type, [&](auto* p) {
    using T = std::remove_pointer_t<decltype(p)>;
    hipLaunchKernelGGL(mg_recurrence_backward_kernel<T>, dim3(blocks), dim3(256), 0, (hipStream_t)stream, rec_args(r),
                       RecMarks{marks, (long)marks_row, (long)marks_stride}, (const T*)d->dh, (long)d->dh_row, (long)d->dh_step,
                       d->dlast, (T*)d->dx, (long)d->dx_row, (long)d->dx_step, (T*)d->dgate, (long)d->dgate_row,
                       (long)d->dgate_step, d->dstate);
    return rec_launched(who);
  });
} catch (...) {
  return 1;
}
