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
// or +infinity among its allowed tokens, or with a u of NaN, has action -1 and NaN.
//
// Rows of up to HEAD_NARROW columns are held in registers, E adjacent columns per lane, by as many lanes as that takes
// (one lane for five actions, a wave for five hundred); rows of up to HEAD_ROW columns by a block, in chunks of eight columns
// per thread.  Their logits are read once.  Wider rows are cut into parts, a block each; what a part found (maximum, sum, ...)
// goes to a workspace and a second launch joins the parts of a row.  A history is counted in LDS by the block that needs it,
// for the columns that it holds.
//
// The logits are held in 64 bits where a bias or a penalty could cancel large ones, the differences from the largest and all
// that follows in 32 (weights, sums, logarithm: log-probabilities and entropies are some 8e-8 off where 64 bits, rounded, are
// 3e-8, in half of the time; gradients are rounded to the logits' type anyway).  A sampled action is the one that 64 bits find
// all the same, whatever the order of the sums: the error of the running sum is bounded, and a row in which the target comes
// within that bound of a token's border is done once more in 64 bits, its log-probability and entropy with it (normal logits:
// 1 row in 1000 at 157 tokens, 1 in 200 at 1024, 1 in 25 at 8192).  The parts of wide rows are summed in 64 bits from the start:
// 13 to 20 rows in 100 would be repeated at 32003 tokens and 35 to 56 at 131072, by launches of their own.
#include <hip/hip_runtime.h>

#include <cmath>
#include <string>
#include <type_traits>

#include "../../include/mettagrid_hip.h"

#define HEAD_THREADS 256
#define HEAD_NARROW (64 * 8)  // the widest row that lanes of one wave hold
#define HEAD_CHUNK (HEAD_THREADS * 8)  // columns that a block holds as 8 per thread
#define HEAD_ROW (4 * HEAD_CHUNK)  // the widest row that a block holds
static_assert(HEAD_CHUNK / 2 == MG_EVALUATE_STATS_WIDTH, "a backward pass computes again what half a block holds");
#define HEAD_FOUND 5  // doubles per part in the workspace: M, Z, sum d exp(-d), bad, first column of M

extern int mg_fail_msg(const std::string& m);  // mettagrid_hip.hip: sets mg_last_error(), returns 1

// ---- arithmetic -------------------------------------------------------------------------------------------------------

// 2^y for y <= 0: n = rint(y), and with r = y - n, |r| <= 1/2, the polynomial 1 + r q(r), q of degree 10 through
// (2^r - 1) / r at the Chebyshev points, which is 2e-17 off.  (y of less than -1075 gives 0.)  14 instructions, where the
// library's e^x takes 40.
__device__ __forceinline__ double head_exp_two(double y) {
  const double n = rint(y), r = y - n;
  double p = 4.4549605981865186e-10;
  p = fma(p, r, 7.072585949269223e-09);
  p = fma(p, r, 1.0178062445845774e-07);
  p = fma(p, r, 1.321544258792169e-06);
  p = fma(p, r, 1.525273382983612e-05);
  p = fma(p, r, 0.0001540353044173605);
  p = fma(p, r, 0.0013333558146416936);
  p = fma(p, r, 0.009618129107606888);
  p = fma(p, r, 0.0555041086648216);
  p = fma(p, r, 0.24022650695910097);
  p = fma(p, r, 0.6931471805599453);
  p = fma(p, r, 1.0);
  return ldexp(p, (int)n);
}

// 1 / z; in 32 bits by the hardware's reciprocal and one Newton step
__device__ __forceinline__ double head_inverse(double z) { return 1.0 / z; }
__device__ __forceinline__ float head_inverse(float z) {
  const float r = __builtin_amdgcn_rcpf(z);
  return fmaf(fmaf(-z, r, 1.0f), r, r);
}
__device__ __forceinline__ double head_log(double z) { return log(z); }
__device__ __forceinline__ float head_log(float z) { return logf(z); }

// The call's arguments, with the quotients that every row wants (a 64-bit division costs a wave as much as a dozen tokens).
struct HeadArgs : mg_logits {
  double inv_temp, inv_rep;
  double weight_scale;  // -log2 e / temperature
};

// One row's controls.
struct HeadRow {
  const float* bias;
  const void* allowed;
  int kind;
  bool counted;
  double inv_rep, rep, presence, frequency, inv_temp, weight_scale;
};

__device__ __forceinline__ HeadRow head_row(const HeadArgs& a, long row) {
  HeadRow r;
  r.bias = a.bias ? a.bias + row * a.bias_row : nullptr;
  r.kind = a.allowed ? a.allowed_kind : 0;
  r.allowed = !a.allowed ? nullptr : r.kind == MG_ALLOWED_BOOL ? (const void*)((const unsigned char*)a.allowed + row * a.allowed_row)
                                                               : (const void*)((const int*)a.allowed + row * a.allowed_row);
  r.counted = a.history != nullptr;
  r.rep = a.repetition; r.inv_rep = a.inv_rep;
  r.presence = a.presence; r.frequency = a.frequency; r.inv_temp = a.inv_temp; r.weight_scale = a.weight_scale;
  return r;
}

// What a row's exponentials and gradients are scaled by.  weight(t) = exp(-t / temperature) for t = M - x: the scale and
// log2 e are one factor.  In 32 bits the difference, the factor and the product round once each, 3 u t / temperature
// relative, plus the 2 u of the hardware's exp2.  In 64 bits a NaN is not handed on (the caller looks for it).
// log2() is the weight's logarithm, kept finite where t is infinite or far: the weight is 0 there (from -150 on in 32 bits, from
// -1075 on in 64), and 0 times it has to be 0.  sum() adds it times the weight; finish() turns that into sum t / temperature.
template <typename X> struct HeadScale;
template <> struct HeadScale<double> {
  double inv_temp, k;
  __device__ explicit HeadScale(const HeadRow& r) : inv_temp(r.inv_temp), k(r.weight_scale) {}
  __device__ __forceinline__ double weight(double t) const { return head_exp_two(log2(t)); }
  __device__ __forceinline__ double log2(double t) const { return fmax(t * k, -2000.0); }
  __device__ __forceinline__ double sum(double t, double w, double s) const { return fma(log2(t), w, s); }
  __device__ __forceinline__ double finish(double s) const { return s * -0.69314718055994529; }
};
template <> struct HeadScale<float> {
  float inv_temp, k;
  __device__ explicit HeadScale(const HeadRow& r) : inv_temp((float)r.inv_temp), k((float)r.weight_scale) {}
  __device__ __forceinline__ float weight(float t) const { return __builtin_amdgcn_exp2f(t * k); }
  __device__ __forceinline__ float weight(float t, float log_z) const { return __builtin_amdgcn_exp2f(fmaf(t, k, log_z * -1.44269504f)); }
  __device__ __forceinline__ float log2(float t) const { return fmaxf(t * k, -160.f); }
  __device__ __forceinline__ float sum(float t, float w, float s) const { return fmaf(log2(t), w, s); }
  __device__ __forceinline__ float finish(float s) const { return s * -0.693147182f; }
  // H + log q of a token, from `past` = H - log Z
  __device__ __forceinline__ float surprise(float t, float past) const { return fmaf(log2(t), 0.693147182f, past); }
};
// M - x in W, from values in X: in the wider of the two
template <typename W, typename X>
__device__ __forceinline__ W head_far(X m, X x) {
  if constexpr (sizeof(W) > sizeof(X)) return (W)m - (W)x;
  else return (W)(m - x);
}
// (M - x) / temperature of one token: as far as the temperature brings it back, also where M - x leaves the range of 32 bits;
// infinity for a token at -infinity
template <typename X>
__device__ __forceinline__ float head_distance(const HeadRow& r, X m, X x) {
  if (x == (X)-INFINITY) return INFINITY;
  if constexpr (sizeof(X) == 8) return (float)((m - x) * r.inv_temp);
  else return (0.5f * m - 0.5f * x) * (2.0f * (float)r.inv_temp);
}
__device__ __forceinline__ double head_max(double a, double b) { return fmax(a, b); }  // (a NaN loses)
__device__ __forceinline__ float head_max(float a, float b) { return fmaxf(a, b); }

__device__ __forceinline__ bool head_allowed(const HeadRow& r, int v) {
  if (r.kind == MG_ALLOWED_BITS) return (((const unsigned*)r.allowed)[v >> 5] >> (v & 31)) & 1;
  return r.kind != MG_ALLOWED_BOOL || ((const unsigned char*)r.allowed)[v] != 0;
}

// bit e of `bits` over a whole word
__device__ __forceinline__ unsigned head_bit(unsigned bits, int e) { return (unsigned)((int)(bits << (31 - e)) >> 31); }

// N words from (to) an address that is aligned to an element of its tensor only
typedef unsigned head_four __attribute__((ext_vector_type(4), aligned(1)));
typedef unsigned head_two __attribute__((ext_vector_type(2), aligned(1)));
typedef unsigned head_one __attribute__((aligned(1)));
template <int N>
__device__ __forceinline__ void head_words(const void* p, unsigned* out) {
#pragma unroll
  for (int i = 0; i + 4 <= N; i += 4) {
    const head_four w = ((const head_four*)p)[i / 4];
    out[i] = w.x, out[i + 1] = w.y, out[i + 2] = w.z, out[i + 3] = w.w;
  }
  constexpr int two = N & ~3, one = N & ~1;
  if constexpr (N & 2) {
    const head_two w = *(const head_two*)((const char*)p + 4 * two);
    out[two] = w.x, out[two + 1] = w.y;
  }
  if constexpr (N & 1) out[one] = *(const head_one*)((const char*)p + 4 * one);
}
template <int N>
__device__ __forceinline__ void head_put_words(void* p, const unsigned* in) {
#pragma unroll
  for (int i = 0; i + 4 <= N; i += 4) ((head_four*)p)[i / 4] = head_four{in[i], in[i + 1], in[i + 2], in[i + 3]};
  constexpr int two = N & ~3, one = N & ~1;
  if constexpr (N & 2) *(head_two*)((char*)p + 4 * two) = head_two{in[two], in[two + 1]};
  if constexpr (N & 1) *(head_one*)((char*)p + 4 * one) = in[one];
}

// E adjacent elements, n of them in the row
template <int E>
__device__ __forceinline__ void head_store(void* p, int type, long at, int n, const float* x) {
  unsigned w[E];
  if (type == MG_F32) {
    unsigned* q = (unsigned*)p + at;
#pragma unroll
    for (int e = 0; e < E; e++) w[e] = __float_as_uint(x[e]);
    if (n >= E) {
      head_put_words<E>(q, w);
    } else {
#pragma unroll
      for (int e = 0; e < E; e++) if (e < n) q[e] = w[e];
    }
    return;
  }
  unsigned short* q = (unsigned short*)p + at;
  if (type == MG_BF16) {
#pragma unroll
    for (int e = 0; e < E; e++) w[e] = __builtin_bit_cast(unsigned short, (__bf16)x[e]);
  } else {
#pragma unroll
    for (int e = 0; e < E; e++) w[e] = __builtin_bit_cast(unsigned short, (_Float16)x[e]);
  }
  if (n >= E) {
    unsigned pair[(E + 1) / 2];
#pragma unroll
    for (int e = 0; e + 1 < E; e += 2) pair[e / 2] = w[e] | w[e + 1] << 16;
    head_put_words<E / 2>(q, pair);
    if constexpr (E & 1) q[E - 1] = (unsigned short)w[E - 1];
  } else {
#pragma unroll
    for (int e = 0; e < E; e++) if (e < n) q[e] = (unsigned short)w[e];
  }
}

// E adjacent columns of a row as they lie in memory, on their way: what is fetched for several groups of columns before
// the first is looked at waits for the memory once.  FULL: all E columns are in the row, for every lane.
template <int E>
struct HeadRaw {
  static constexpr bool BORDER = 32 % E != 0 && E > 4;  // a group's mask bits may lie in two words (narrower groups start at column 0)
  unsigned logits[E], allowed[(E + 3) / 4];
  float bias[E];

  // logits of `type` (null: not wanted) at element `at` of the tensor; columns v0 ... of the row's controls.  (Every path
  // sets every word: stores to places that differ from path to path would keep the struct out of registers.)
  template <bool FULL, bool BIAS>
  __device__ __forceinline__ void fetch(const HeadRow& r, const void* p, int type, long at, int v0, int n) {
    static_assert(E <= 16, "mask bits of one half word");
#pragma unroll
    for (int e = 0; e < E; e++) logits[e] = 0;
    if (p) {
      if (type == MG_F32) words<FULL>((const unsigned*)p + at, n, logits);
      else halves<FULL>((const unsigned short*)p + at, n, logits);
    }
#pragma unroll
    for (int e = 0; e < (E + 3) / 4; e++) allowed[e] = 0;
    if (r.kind == MG_ALLOWED_BITS) {
      allowed[0] = FULL || n > 0 ? ((const unsigned*)r.allowed)[v0 >> 5] : 0u;
      if constexpr (BORDER) {
        if (!FULL && (v0 & 31) + min(n, E) > 32) allowed[1] = ((const unsigned*)r.allowed)[(v0 >> 5) + 1];
      }
    }
    if (r.kind == MG_ALLOWED_BOOL) bytes<FULL>((const unsigned char*)r.allowed + v0, n, allowed);
    if constexpr (BIAS) {
      unsigned b[E];
#pragma unroll
      for (int e = 0; e < E; e++) b[e] = 0;
      if (r.bias) words<FULL>((const unsigned*)(r.bias + v0), n, b);
#pragma unroll
      for (int e = 0; e < E; e++) bias[e] = __uint_as_float(b[e]);
    }
  }
  template <bool FULL>
  static __device__ __forceinline__ void words(const unsigned* p, int n, unsigned* out) {
    if (FULL || n >= E) {
      head_words<E>(p, out);
    } else {
#pragma unroll
      for (int e = 0; e < E; e++) out[e] = e < n ? p[e] : 0u;
    }
  }
  template <bool FULL>
  static __device__ __forceinline__ void halves(const unsigned short* p, int n, unsigned* out) {
    if (FULL || n >= E) {
      head_words<E / 2>(p, out);
      if constexpr (E & 1) out[E / 2] = p[E - 1];
    } else {
#pragma unroll
      for (int e = 0; e < E; e += 2) {
        const unsigned lo = e < n ? p[e] : 0u, hi = e + 1 < n ? p[e + 1] : 0u;
        out[e / 2] = lo | hi << 16;
      }
    }
  }
  template <bool FULL>
  static __device__ __forceinline__ void bytes(const unsigned char* p, int n, unsigned* out) {
    if (FULL || n >= E) {
      head_words<E / 4>(p, out);
      if constexpr (E % 4 != 0) {
        unsigned b = 0;
#pragma unroll
        for (int e = E / 4 * 4; e < E; e++) b |= (unsigned)p[e] << (8 * (e % 4));
        out[E / 4] = b;
      }
    } else {
#pragma unroll
      for (int w = 0; w < (E + 3) / 4; w++) {
        unsigned b = 0;
#pragma unroll
        for (int e = 4 * w; e < E && e < 4 * w + 4; e++) b |= (e < n ? (unsigned)p[e] : 0u) << (8 * (e % 4));
        out[w] = b;
      }
    }
  }

  __device__ __forceinline__ void values(int type, float* l) const {
    if (type == MG_F32) {
#pragma unroll
      for (int e = 0; e < E; e++) l[e] = __uint_as_float(logits[e]);
    } else if (type == MG_BF16) {
#pragma unroll
      for (int e = 0; e < E; e++) l[e] = __uint_as_float(e % 2 ? logits[e / 2] & 0xFFFF0000u : logits[e / 2] << 16);
    } else {
#pragma unroll
      for (int e = 0; e < E; e++) l[e] = (float)__builtin_bit_cast(_Float16, (unsigned short)(e % 2 ? logits[e / 2] >> 16 : logits[e / 2]));
    }
  }

  // bit e: column e is in the row (of which n are left) and allowed
  __device__ __forceinline__ unsigned bits(const HeadRow& r, int v0, int n) const {
    if (n <= 0) return 0;
    const unsigned inside = n >= E ? (1u << E) - 1 : (1u << n) - 1;
    if (r.kind == MG_ALLOWED_BITS) {
      if constexpr (BORDER) return (unsigned)(((unsigned long long)allowed[1] << 32 | allowed[0]) >> (v0 & 31)) & inside;
      return (allowed[0] >> (v0 & 31)) & inside;
    }
    if (r.kind != MG_ALLOWED_BOOL) return inside;
    unsigned b = 0;
#pragma unroll
    for (int e = 0; e < E; e++) b |= (allowed[e / 4] & (0xFFu << (8 * (e % 4)))) ? 1u << e : 0u;
    return b & inside;
  }

  // x, and (GRAD) what a gradient of x is multiplied by besides 1 / temperature: 0 where masked, and only where ADJUST,
  // else the bits tell.  ADJUST: whether there may be a bias or a history at all.  counts: these columns in the history.
  // Returns bits().
  template <bool FULL, bool GRAD, bool ADJUST, typename X>
  __device__ __forceinline__ unsigned columns(const HeadRow& r, int type, int v0, int n, const unsigned* counts, X* x, float* slope) const {
    float l[E];
    values(type, l);
    const unsigned ok = bits(r, v0, n);
    if (!FULL || r.kind) {  // masked, or behind the row's end: -infinity
#pragma unroll
      for (int e = 0; e < E; e++) {
        const unsigned in = head_bit(ok, e);
        l[e] = __uint_as_float((__float_as_uint(l[e]) & in) | (0xFF800000u & ~in));
      }
    }
#pragma unroll
    for (int e = 0; e < E; e++) x[e] = (X)l[e];
    if (!ADJUST) return ok;
    if (r.counted) {
#pragma unroll
      for (int e = 0; e < E; e++) {
        const unsigned c = counts[e];
        const X y = (x[e] > 0 ? x[e] * r.inv_rep : x[e] * r.rep) - r.frequency * c - r.presence;
        if (GRAD) slope[e] = !head_bit(ok, e) ? 0.f : c ? (float)(x[e] > 0 ? r.inv_rep : r.rep) : 1.f;
        x[e] = c ? y : x[e];
      }
    } else if (GRAD) {
#pragma unroll
      for (int e = 0; e < E; e++) slope[e] = head_bit(ok, e) ? 1.f : 0.f;
    }
    if (r.bias) {
#pragma unroll
      for (int e = 0; e < E; e++) x[e] += __uint_as_float(__float_as_uint(bias[e]) & head_bit(ok, e));
    }
    return ok;
  }
};

// which of the grid's blocks this is (head_grid)
__device__ __forceinline__ long head_block() { return (long)blockIdx.y * gridDim.x + blockIdx.x; }

// ---- lanes ------------------------------------------------------------------------------------------------------------

__device__ __forceinline__ int head_lane() { return threadIdx.x & 63; }

// x of the lane that DPP control C names (within 16 lanes, or from one row of 16 to others); `none` where there is none
template <int C, typename V>
__device__ __forceinline__ V head_dpp(V x, V none) {
  if constexpr (sizeof(V) == 4) {
    return __builtin_bit_cast(V, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, none), __builtin_bit_cast(int, x), C, 0xF, 0xF, false));
  } else {
    const long long xs = __builtin_bit_cast(long long, x), ns = __builtin_bit_cast(long long, none);
    const unsigned lo = __builtin_amdgcn_update_dpp((int)ns, (int)xs, C, 0xF, 0xF, false);
    const unsigned hi = __builtin_amdgcn_update_dpp((int)(ns >> 32), (int)(xs >> 32), C, 0xF, 0xF, false);
    return __builtin_bit_cast(V, (long long)hi << 32 | lo);
  }
}
// over the `lanes` (a power of two) lanes of a group; every lane gets the result.  (Pairs, quads, then mirrors within 8 and
// 16 lanes: what is mirrored is the same in each half by then.)
template <typename V, typename F>
__device__ __forceinline__ V head_group(V x, int lanes, F f) {
  if (lanes > 1) x = f(x, head_dpp<0xB1>(x, x));
  if (lanes > 2) x = f(x, head_dpp<0x4E>(x, x));
  if (lanes > 4) x = f(x, head_dpp<0x141>(x, x));
  if (lanes > 8) x = f(x, head_dpp<0x140>(x, x));
  if (lanes > 16) x = f(x, __shfl_xor(x, 16));
  if (lanes > 32) x = f(x, __shfl_xor(x, 32));
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
// the sum of the lanes before this one in its group, and of all of them
__device__ __forceinline__ double head_group_before(double x, int lanes, int lane, double& all) {
  double sum = x;
  auto add = [&](double up, int o) { sum += lane >= o ? up : 0.0; };
  if (lanes > 1) add(head_dpp<0x111>(sum, 0.0), 1);
  if (lanes > 2) add(head_dpp<0x112>(sum, 0.0), 2);
  if (lanes > 4) add(head_dpp<0x114>(sum, 0.0), 4);
  if (lanes > 8) add(head_dpp<0x118>(sum, 0.0), 8);
  // (so far within rows of 16 lanes: now the whole of the rows before)
  if (lanes > 16) {
    const double row = __shfl(sum, (head_lane() & 48) - 1);  // (read by all lanes: those that are off hold nothing to read)
    sum += lane & 16 ? row : 0.0;
  }
  if (lanes > 32) {
    const double half = __shfl(sum, 31);
    sum += lane & 32 ? half : 0.0;
  }
  all = __shfl(sum, head_lane() | (lanes - 1));
  return sum - x;
}

// adjusted logits of E columns, or their gradient, from what was fetched (for a gradient with a history: the logits and the
// outer gradient; without: the outer gradient alone, on which the logits have no influence)
template <int E>
struct HeadAdjust {
  HeadRaw<E> raw, outer;

  template <bool FULL>
  __device__ __forceinline__ void fetch(const HeadArgs& a, const HeadRow& r, long row, int v0, int n, const void* dout) {
    HeadRow plain = r;
    if (dout) plain.bias = nullptr;  // (no gradient depends on it)
    raw.template fetch<FULL, true>(plain, !dout || r.counted ? a.logits : nullptr, a.type, row * a.logits_row + v0, v0, n);
    if (dout) {
      plain.kind = 0;
      outer.template fetch<FULL, false>(plain, dout, a.type, row * a.width + v0, v0, n);
    }
  }
  __device__ __forceinline__ void store(const HeadArgs& a, const HeadRow& r, long row, int v0, int n, const unsigned* counts, void* out,
                                        const void* dout, void* dlogits) const {
    double x[E];
    float slope[E], y[E];
    if (!dout) {
      raw.template columns<false, false, true>(r, a.type, v0, n, counts, x, slope);
#pragma unroll
      for (int e = 0; e < E; e++) y[e] = (float)(x[e] * r.inv_temp);
      head_store<E>(out, a.type, row * a.width + v0, n, y);
      return;
    }
    outer.values(a.type, y);
    if (r.counted) {
      HeadRow plain = r;
      plain.bias = nullptr;
      raw.template columns<false, true, true>(plain, a.type, v0, n, counts, x, slope);
#pragma unroll
      for (int e = 0; e < E; e++) y[e] = slope[e] == 0.f ? 0.f : (float)((double)y[e] * (slope[e] * r.inv_temp));
    } else {
      const unsigned ok = raw.bits(r, v0, n);
#pragma unroll
      for (int e = 0; e < E; e++) y[e] = __uint_as_float(__float_as_uint((float)(y[e] * r.inv_temp)) & head_bit(ok, e));
    }
    head_store<E>(dlogits, a.type, row * a.width + v0, n, y);
  }
};

// ---- narrow rows ------------------------------------------------------------------------------------------------------

struct HeadNarrow { int lanes, rows; };  // lanes per row, rows per block

// counts[row * lanes + lane][e] over the block's rows, all threads together, eight entries on their way at a time;
// barriers inside
template <int E>
__device__ __forceinline__ void head_count_rows(const HeadArgs& a, const HeadNarrow& g, long row0, unsigned (*counts)[E + 1]) {
  __syncthreads();
#pragma unroll
  for (int e = 0; e < E; e++) counts[threadIdx.x][e] = 0;
  __syncthreads();
  const int rows = (int)min((long)g.rows, a.rows - row0);
  // entry threadIdx.x, then every 256th of the block's rows * history_len, row and place kept without a division a step
  const int len = a.history_len, skip = HEAD_THREADS / len, rest = HEAD_THREADS - skip * len;
  int row = threadIdx.x / len, place = threadIdx.x - row * len;
  const int* h = a.history + row0 * a.history_row;
  while (row < rows) {
    int v[8], slot[8];
#pragma unroll
    for (int u = 0; u < 8; u++) {
      v[u] = row < rows ? h[row * a.history_row + place] : -1;
      slot[u] = row * g.lanes;
      row += skip;
      place += rest;
      if (place >= len) place -= len, row++;
    }
#pragma unroll
    for (int u = 0; u < 8; u++)
      if (v[u] >= 0 && v[u] < a.width) atomicAdd(&counts[slot[u] + v[u] / E][v[u] % E], 1u);
  }
  __syncthreads();
}

// What the lanes of a row know of it.  ONE: a lane per row, of exactly E columns.  X: the type of x, W: of what comes after
// the difference from the largest (64 bits for x alone are enough where large logits and biases or penalties could cancel).
template <int E, bool ONE, typename X, typename W>
struct HeadHeld {
  X x[E], m;
  W t[E], w[E], z, s;  // t = M - x, w = its weight; t and w say nothing where the row is bad or empty
  double z_lane, before, all;  // (of a group whose running sum is wanted) z of this lane's columns, of the lanes before it, of all
  float slope[E];
  long row;         // clamped: the groups behind the last row do that row's work once more
  int lane, v0, n;  // this lane's columns, n of them (or fewer than one) in the row
  bool bad, empty, mine;  // mine: the row is this group's own

  __device__ __forceinline__ void place(const HeadArgs& a, const HeadNarrow& g, long row0) {
    const long at = row0 + (ONE ? threadIdx.x : threadIdx.x / g.lanes);
    lane = ONE ? 0 : threadIdx.x % g.lanes;
    mine = at < a.rows && (ONE || (int)threadIdx.x < g.rows * g.lanes);
    row = mine ? at : a.rows - 1;
    v0 = lane * E;
    n = ONE ? E : a.width - v0;
  }

  template <bool GRAD, bool RUN>
  __device__ __forceinline__ void hold(const HeadArgs& a, const HeadNarrow& g, const HeadRow& r, const HeadScale<W>& scale, const unsigned* counts) {
    constexpr bool adjust = std::is_same<X, double>::value;
    HeadRaw<E> raw;
    raw.template fetch<ONE, adjust>(r, a.logits, a.type, row * a.logits_row + v0, v0, n);
    raw.template columns<ONE, GRAD, adjust>(r, a.type, v0, n, counts, x, slope);
    m = x[0];
#pragma unroll
    for (int e = 1; e < E; e++) m = head_max(m, x[e]);
    if (!ONE) m = head_group(m, g.lanes, [](X p, X q) { return head_max(p, q); });
    const X top = m < (X)INFINITY && m > (X)-INFINITY ? m : (X)0;
    z = s = 0;
    bool lost = false;  // a NaN
#pragma unroll
    for (int e = 0; e < E; e++) {
      const W far = head_far<W, X>(top, x[e]);
      t[e] = far;
      w[e] = scale.weight(far);
      z += w[e];
      s = scale.sum(far, w[e], s);
      if (sizeof(W) == 8) lost = lost || far != far;
    }
    if (lost) z = NAN;
    if constexpr (RUN) z_lane = all = z, before = 0.0;
    if (!ONE) {
      if constexpr (RUN) before = head_group_before(z_lane, g.lanes, lane, all), z = (W)all;
      else z = head_group_sum(z, g.lanes);
      s = head_group_sum(s, g.lanes);
    }
    s = scale.finish(s);
    // +infinity is the largest, NaN has lost to everything but makes the sum NaN
    bad = !(m < (X)INFINITY) || z != z;
    empty = !bad && m == (X)-INFINITY;
  }
  // the lanes of this row
  __device__ __forceinline__ unsigned long long group(const HeadNarrow& g) const {
    return ONE ? 1ull << head_lane() : ~0ull >> (64 - g.lanes) << (head_lane() - lane);
  }
  // whether this lane has the token that is meant: the one at which the running sum passes the target, or (SUM false) the first
  // of the largest.  Where no lane has (a uniform of 1 or more, or one that the roundings between two lanes took): the last
  // with any weight.
  template <bool SUM>
  __device__ __forceinline__ bool picks(const HeadNarrow& g, double target) const {
    if (ONE) return true;
    bool pass = false;
    if (SUM) {
      pass = z_lane > 0.0 && before + z_lane > target;
    } else {
#pragma unroll
      for (int e = 0; e < E; e++) pass = pass || x[e] == m;
    }
    const unsigned long long over = __ballot(pass) & group(g), some = SUM ? __ballot(z_lane > 0.0) & group(g) : over;
    return head_lane() == (bad || empty ? head_lane() - lane : over ? __ffsll(over) - 1 : 63 - __clzll((long long)some));
  }
};

// Which of a thread's E tokens a running sum passes the target at, and its t: the last with any weight, if it does not.  (A
// token without weight is never picked, also where the sum of what came before is rounded up over the target.)
template <typename W>
struct HeadPick {
  int e;
  W t;
  double before, at;  // the running sum before it and with it
};
template <int E, typename W>
__device__ __forceinline__ HeadPick<W> head_pick(const W* w, const W* t, double run, double target) {
  HeadPick<W> pick{0, 0, run, run};
  bool over = false;
#pragma unroll
  for (int e = 0; e < E; e++) {
    const bool take = !over && w[e] > 0;
    pick.e = take ? e : pick.e;
    pick.t = take ? t[e] : pick.t;
    pick.before = take ? run : pick.before;
    run += w[e];
    pick.at = take ? run : pick.at;
    over = over || (take && run > target);
  }
  return pick;
}
// How far a running sum of 32-bit weights and a target made with their whole sum z may be off together.  A weight at distance d
// is off by 3 u d (difference, scale, product; u = 2^-24) and 1.43 u (the hardware's exp2, over all its arguments), a thread's
// sum of eight by 7 u more, everything else is added in 64 bits: (3 s + 8.5 z) u with s = sum of d w, and the target the
// same, where 2 (4 s + 12 z) u is taken; what is below 2^-126 does not count beside that, since z is 1 or more.
__device__ __forceinline__ double head_margin(double z, double s) { return 0x1p-23 * (4.0 * s + 12.0 * z); }
__device__ __forceinline__ bool head_sure(const HeadPick<float>& pick, double target, double margin) {
  return pick.before + margin < target && pick.at - margin > target;
}
template <int E, typename X>
__device__ __forceinline__ int head_first(const X* x, X m) {
  int first = 0;
#pragma unroll
  for (int e = E - 1; e >= 0; e--) first = x[e] == m ? e : first;
  return first;
}
// t and weights of E tokens from their x, once more: what is kept from the first time takes the registers of other waves.  (The
// empty assembly is what stops the compiler from keeping it.)
template <int E, typename W, typename X>
__device__ __forceinline__ void head_again(const X* x, X m, const HeadScale<W>& scale, W* t, W* w) {
#pragma unroll
  for (int e = 0; e < E; e++) {
    X xe = x[e];
    asm volatile("" : "+v"(xe));
    t[e] = head_far<W, X>(m, xe);
    w[e] = scale.weight(t[e]);
  }
}
template <typename W>
__device__ __forceinline__ void head_sampled(long row, bool bad, bool empty, int action, W t, W z, W s, const HeadScale<W>& scale, int* actions,
                                             float* log_prob, float* entropy) {
  const W log_z = head_log(z);
  actions[row] = bad || empty ? -1 : action;
  log_prob[row] = bad ? NAN : empty ? 0.f : (float)(-t * scale.inv_temp - log_z);
  entropy[row] = bad ? NAN : empty ? 0.f : (float)(log_z + s * head_inverse(z));
}

// Adjusted logits or their gradient, E columns per lane and no word between lanes.  Bound by memory without a history (32768 x
// 512 bf16: 14 us for 67 MB, 4.9 TB/s), by counting it with one (24576 x 157 f32, masks, 32 entries: 14 us each way for 38
// and 53 MB).
template <int E>
__global__ __launch_bounds__(HEAD_THREADS) void mg_adjust_narrow_kernel(HeadArgs a, HeadNarrow g, void* __restrict__ out,
                                                                       const void* __restrict__ dout, void* __restrict__ dlogits) {
  __shared__ unsigned counts[HEAD_THREADS][E + 1];
  const long row0 = head_block() * g.rows;
  if (row0 >= a.rows) return;
  if (a.history) head_count_rows<E>(a, g, row0, counts);
  HeadHeld<E, false, double, double> h;
  h.place(a, g, row0);
  if (!h.mine) return;
  const HeadRow r = head_row(a, h.row);
  HeadAdjust<E> it;
  it.template fetch<false>(a, r, h.row, h.v0, h.n, dout);
  it.store(a, r, h.row, h.v0, h.n, counts[threadIdx.x], out, dout, dlogits);
}

// An action per row.  Bound by the launch and the way through it (24 x 5: 2.0 us; 98304 x 5 bf16, masks, 16 entries of history:
// 6.4 us for 9 MB), from some 50 columns on by its instructions (98304 x 64 bf16: 11 us, 7.5 of them the issue of 4.6 million
// vector instructions; 32768 x 512: 25 us for 14.8 million, which take 24).  A long history over few columns is bound by its
// count: a block counts for up to 256 rows, whatever its length, and a wave's lanes add to the same words (4096 x 5, 4096
// entries: 520 us for 67 MB).
template <int E, bool ONE, typename X>
__global__ __launch_bounds__(HEAD_THREADS) void mg_sample_narrow_kernel(HeadArgs a, HeadNarrow g, const float* __restrict__ uniforms,
                                                                       int* __restrict__ actions, float* __restrict__ log_prob,
                                                                       float* __restrict__ entropy) {
  constexpr bool adjust = std::is_same<X, double>::value;
  __shared__ unsigned counts[adjust ? HEAD_THREADS : 1][E + 1];
  const long row0 = head_block() * g.rows;
  if (row0 >= a.rows) return;
  if constexpr (adjust) {
    if (a.history) head_count_rows<E>(a, g, row0, counts);
  }
  HeadHeld<E, ONE, X, float> h;
  h.place(a, g, row0);
  const HeadRow r = head_row(a, h.row);
  const HeadScale<float> scale(r);
  const unsigned* mine = counts[adjust ? threadIdx.x : 0];
  if (!uniforms) {
    h.template hold<false, false>(a, g, r, scale, mine);
    if (h.template picks<false>(g, 0.0) && h.mine)
      head_sampled(h.row, h.bad, h.empty, h.v0 + head_first<E>(h.x, h.m), 0.f, h.z, h.s, scale, actions, log_prob, entropy);
    return;
  }
  h.template hold<false, true>(a, g, r, scale, mine);
  const float uniform = uniforms[h.row];
  h.bad = h.bad || uniform != uniform;
  const double u = fmax((double)uniform, 0.0), target = u < 1.0 ? u * h.all : INFINITY;
  bool unsure = false;
  if (h.template picks<true>(g, target)) {
    const HeadPick<float> pick = head_pick<E>(h.w, h.t, h.before, target);
    unsure = !h.bad && !h.empty && !head_sure(pick, target, head_margin(h.all, h.s));
    if (h.mine && !unsure) head_sampled(h.row, h.bad, h.empty, h.v0 + pick.e, pick.t, h.z, h.s, scale, actions, log_prob, entropy);
  }
  const unsigned long long again = __ballot(unsure);
  if (!again) return;
  // the same in 64 bits
  const HeadScale<double> exact(r);
  double t[E], w[E], s = 0.0;
  head_again<E>(h.x, h.m, exact, t, w);
  h.z_lane = 0.0;
#pragma unroll
  for (int e = 0; e < E; e++) h.z_lane += w[e], s = exact.sum(t[e], w[e], s);
  h.all = h.z_lane, h.before = 0.0;
  if (!ONE) {
    h.before = head_group_before(h.z_lane, g.lanes, h.lane, h.all);
    s = head_group_sum(s, g.lanes);
  }
  const double line = u < 1.0 ? u * h.all : INFINITY;
  if (h.template picks<true>(g, line) && h.mine && (again & h.group(g))) {
    const HeadPick<double> pick = head_pick<E>(w, t, h.before, line);
    head_sampled(h.row, false, false, h.v0 + pick.e, pick.t, h.all, exact.finish(s), exact, actions, log_prob, entropy);
  }
}

// Bound by memory at few columns (2097152 x 5 bf16: 10.4 us for 46 MB, 4.4 TB/s), by its instructions at many (32768 x 512 bf16: 18
// us, as long as the issue of its 11.6 million vector instructions takes).
template <int E, bool ONE, typename X>
__global__ __launch_bounds__(HEAD_THREADS) void mg_evaluate_narrow_kernel(HeadArgs a, HeadNarrow g, const int* __restrict__ actions,
                                                                         float* __restrict__ log_prob, float* __restrict__ entropy) {
  constexpr bool adjust = std::is_same<X, double>::value;
  __shared__ unsigned counts[adjust ? HEAD_THREADS : 1][E + 1];
  const long row0 = head_block() * g.rows;
  if (row0 >= a.rows) return;
  if constexpr (adjust) {
    if (a.history) head_count_rows<E>(a, g, row0, counts);
  }
  HeadHeld<E, ONE, X, float> h;
  h.place(a, g, row0);
  const HeadRow r = head_row(a, h.row);
  const HeadScale<float> scale(r);
  const int act = actions[h.row];
  h.template hold<false, false>(a, g, r, scale, counts[adjust ? threadIdx.x : 0]);
  X at = -INFINITY;  // (behind the row's end, where an action outside of it could lie, too)
#pragma unroll
  for (int e = 0; e < E; e++) at = h.v0 + e == act ? h.x[e] : at;
  if (!ONE) at = head_group_max(at, g.lanes);
  const float d = head_distance(r, h.m, at);
  if (h.mine && h.lane == 0) {
    const float log_z = head_log(h.z);
    log_prob[h.row] = h.bad ? NAN : h.empty ? 0.f : (float)(-d - log_z);
    entropy[h.row] = h.bad ? NAN : h.empty ? 0.f : (float)(log_z + h.s * head_inverse(h.z));
  }
}

// The row's sums are computed again, which costs less than reading them (2097152 x 5 bf16: 13.6 us for 67 MB, 4.9 TB/s).
template <int E, bool ONE, typename X>
__global__ __launch_bounds__(HEAD_THREADS) void mg_evaluate_narrow_backward_kernel(HeadArgs a, HeadNarrow g, const int* __restrict__ actions,
                                                                                  const float* __restrict__ dlog_prob,
                                                                                  const float* __restrict__ dentropy,
                                                                                  void* __restrict__ dlogits) {
  constexpr bool adjust = std::is_same<X, double>::value;
  __shared__ unsigned counts[adjust ? HEAD_THREADS : 1][E + 1];
  const long row0 = head_block() * g.rows;
  if (row0 >= a.rows) return;
  if constexpr (adjust) {
    if (a.history) head_count_rows<E>(a, g, row0, counts);
  }
  HeadHeld<E, ONE, X, float> h;
  h.place(a, g, row0);
  const HeadRow r = head_row(a, h.row);
  const HeadScale<float> scale(r);
  const int act = actions[h.row];
  const float gp_row = dlog_prob ? dlog_prob[h.row] : 0.f, gh = (dentropy ? dentropy[h.row] : 0.f) * scale.inv_temp;
  h.template hold<true, false>(a, g, r, scale, counts[adjust ? threadIdx.x : 0]);
  bool left = false;  // whether the action is a token that is left
#pragma unroll
  for (int e = 0; e < E; e++) left = left || (h.v0 + e == act && e < h.n && h.x[e] > (X)-INFINITY);
  if (!ONE) left = head_group_max((int)left, g.lanes) != 0;
  // (a bad row's NaN reaches every token that is left)
  const float gp = h.bad ? NAN : left ? gp_row * scale.inv_temp : 0.f, inv_z = head_inverse(h.z);
  const float past = h.s * inv_z;  // H - log Z
  float y[E];
#pragma unroll
  for (int e = 0; e < E; e++) {
    const float q = h.w[e] * inv_z;
    float d = (h.v0 + e == act ? gp : 0.f) - q * fmaf(gh, scale.surprise(h.t[e], past), gp);
    if (adjust) d *= h.slope[e];
    y[e] = h.x[e] != (X)-INFINITY ? d : 0.f;
  }
  if (h.mine) head_store<E>(dlogits, a.type, h.row * a.width + h.v0, h.n, y);
}

// ---- wide rows --------------------------------------------------------------------------------------------------------
// Thread t of a block holds columns 8 t ... 8 t + 7 of each of its part's chunks.

// counts of the n columns from v0 on, all threads together, four entries each on their way at a time; barriers inside
__device__ __forceinline__ void head_count_columns(const HeadArgs& a, long row, unsigned* counts, long v0, int n) {
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += blockDim.x) counts[i] = 0;
  __syncthreads();
  const int* h = a.history + row * a.history_row;
  for (long i0 = threadIdx.x; i0 < a.history_len; i0 += 4L * blockDim.x) {
    int v[4];
#pragma unroll
    for (int u = 0; u < 4; u++) {
      const long i = i0 + u * (long)blockDim.x;
      v[u] = i < a.history_len ? h[i] : -1;
    }
#pragma unroll
    for (int u = 0; u < 4; u++) {
      const long at = v[u] - v0;
      if (v[u] >= 0 && at >= 0 && at < n) atomicAdd(&counts[at], 1u);
    }
  }
  __syncthreads();
}

// lane l: f over lanes 0 ... l
template <typename V, typename F>
__device__ __forceinline__ V head_scan(V x, V none, F f) {
  x = f(head_dpp<0x111>(x, none), x);
  x = f(head_dpp<0x112>(x, none), x);
  x = f(head_dpp<0x114>(x, none), x);
  x = f(head_dpp<0x118>(x, none), x);
  const V a = head_dpp<0x142>(x, none);  // rows 1 and 3 take the row before them
  x = (head_lane() & 16) ? f(a, x) : x;
  const V b = head_dpp<0x143>(x, none);  // lanes 32 ... 63 take lane 31
  return (head_lane() & 32) ? f(b, x) : x;
}
template <typename V>
__device__ __forceinline__ V head_lane_of(V x, int lane) {
  if constexpr (sizeof(V) == 4) {
    return __builtin_bit_cast(V, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), lane));
  } else {
    const long long xs = __builtin_bit_cast(long long, x);
    const unsigned lo = __builtin_amdgcn_readlane((int)xs, lane), hi = __builtin_amdgcn_readlane((int)(xs >> 32), lane);
    return __builtin_bit_cast(V, (long long)hi << 32 | lo);
  }
}

// over a block of up to 16 waves; every thread gets the result.  (Two calls with the same `red` want a barrier between them.)
template <typename V, typename F>
__device__ __forceinline__ V head_block(V x, V none, V* red, F f) {
  x = head_lane_of(head_scan(x, none, f), 63);
  if (head_lane() == 0) red[threadIdx.x >> 6] = x;
  __syncthreads();
  V y = red[0];
  for (int w = 1; w < (int)(blockDim.x >> 6); w++) y = f(y, red[w]);
  return y;
}
__device__ __forceinline__ int head_block_min(int x, int* red) {
  return head_block<int>(x, 0x7FFFFFFF, red, [](int a, int b) { return a < b ? a : b; });
}

// Where a running sum over a block passes a target: among the n sums of whole waves in `red`, which all threads look at alike,
// the first that does, or the last with anything in it; then among the lanes of that wave; then among a lane's tokens.
struct HeadSpot { int entry; double base; };  // what comes before the entry
__device__ __forceinline__ HeadSpot head_spot(const double* red, int n, double run, double target) {
  HeadSpot spot{0, run};
  bool over = false;
  for (int k = 0; k < n; k++) {
    const double x = red[k];
    const bool take = !over && x > 0.0;
    spot.entry = take ? k : spot.entry;
    spot.base = take ? run : spot.base;
    run += x;
    over = over || (take && run > target);
  }
  return spot;
}
__device__ __forceinline__ double head_total(const double* red, int n) {
  double all = 0.0;
  for (int k = 0; k < n; k++) all += red[k];
  return all;
}
// whether this lane is the one; what comes before it
__device__ __forceinline__ bool head_lane_picks(double mine, double base, double target, double& before) {
  before = base + (head_scan(mine, 0.0, [](double a, double b) { return a + b; }) - mine);
  const unsigned long long over = __ballot(mine > 0.0 && before + mine > target), some = __ballot(mine > 0.0);
  return head_lane() == (over ? __ffsll(over) - 1 : 63 - __clzll((long long)some));
}

// `fetch` for every chunk c of the part, whose columns of this thread start at `at` with n of them left; FULL says whether
// the part lies in the row as a whole
#define HEAD_PART_FETCH(fetch)                                                                  \
  if (part_n == CHUNKS * THREADS * 8) {                                                         \
    constexpr bool FULL = true;                                                                 \
    _Pragma("unroll") for (int c = 0; c < CHUNKS; c++) {                                        \
      const int at = (c * THREADS + threadIdx.x) * 8, n = 8;                                    \
      fetch;                                                                                    \
    }                                                                                           \
  } else {                                                                                      \
    constexpr bool FULL = false;                                                                \
    _Pragma("unroll") for (int c = 0; c < CHUNKS; c++) {                                        \
      const int at = (c * THREADS + threadIdx.x) * 8, n = part_n - at;                          \
      fetch;                                                                                    \
    }                                                                                           \
  }

// Bound by memory where there is enough of it (1024 x 32003 bf16: 23 us for 131 MB, 5.7 TB/s, part of it in the caches), else by
// latency (64 x 50001 bf16, all controls, 512 entries of history that every block of a row counts: 8.4 us for 13 MB).
__global__ __launch_bounds__(HEAD_THREADS) void mg_adjust_wide_kernel(HeadArgs a, void* __restrict__ out, const void* __restrict__ dout,
                                                                     void* __restrict__ dlogits) {
  __shared__ unsigned counts[HEAD_CHUNK];
  const long row = (long)blockIdx.z * gridDim.y + blockIdx.y, part0 = (long)blockIdx.x * HEAD_CHUNK;
  if (row >= a.rows) return;
  const int part_n = (int)min((long)HEAD_CHUNK, a.width - part0), at = threadIdx.x * 8, n = part_n - at, v0 = (int)(part0 + at);
  const HeadRow r = head_row(a, row);
  HeadAdjust<8> it;
  if (part_n == HEAD_CHUNK) it.fetch<true>(a, r, row, v0, 8, dout);
  else it.fetch<false>(a, r, row, v0, n, dout);
  if (a.history) head_count_columns(a, row, counts, part0, part_n);
  if (n > 0) it.store(a, r, row, v0, n, counts + at, out, dout, dlogits);
}

// What a block of THREADS knows of a part of CHUNKS * THREADS * 8 columns (X, W: as for narrow rows).
struct HeadRed {
  double m[16], z[16], s[16];
  int i[16];
};
template <int CHUNKS, int THREADS, typename X, typename W>
struct HeadPart {
  static constexpr bool adjust = std::is_same<X, double>::value;
  X x[CHUNKS][8], m;
  W w[CHUNKS][8], z, s;  // s = sum (M - x) exp(-d) / temperature
  float slope[CHUNKS][8];
  W z_lane[CHUNKS];  // (where the running sum is wanted) z of this thread's columns of a chunk
  bool bad, empty;

  __device__ __forceinline__ W far(int c, int e) const { return head_far<W, X>(top(), x[c][e]); }
  __device__ __forceinline__ X top() const { return m < (X)INFINITY && m > (X)-INFINITY ? m : (X)0; }
  static __device__ __forceinline__ int at(int c) { return (c * THREADS + threadIdx.x) * 8; }

  // RUN: red.z gets the sums of waves, chunk by chunk
  template <bool GRAD, bool RUN>
  __device__ __forceinline__ void hold(const HeadArgs& a, const HeadRow& r, const HeadScale<W>& scale, long row, long part0, int part_n,
                                       unsigned* counts, HeadRed& red) {
    HeadRaw<8> raw[CHUNKS];
    HEAD_PART_FETCH((raw[c].template fetch<FULL, adjust>(r, a.logits, a.type, row * a.logits_row + part0 + at, (int)(part0 + at), n)))
    if (adjust && a.history) head_count_columns(a, row, counts, part0, part_n);  // (while the columns are on their way)
    m = -INFINITY;
#pragma unroll
    for (int c = 0; c < CHUNKS; c++) {
      raw[c].template columns<false, GRAD, adjust>(r, a.type, (int)(part0 + at(c)), part_n - at(c), counts + at(c), x[c], slope[c]);
#pragma unroll
      for (int e = 0; e < 8; e++) m = head_max(m, x[c][e]);
    }
    m = head_block<X>(m, -INFINITY, (X*)red.m, [](X p, X q) { return head_max(p, q); });
    z = s = 0;
    bool lost = false;  // a NaN
#pragma unroll
    for (int c = 0; c < CHUNKS; c++) {
      if constexpr (RUN) z = 0;
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const W t = far(c, e);
        w[c][e] = scale.weight(t);
        z += w[c][e];
        s = scale.sum(t, w[c][e], s);
        if (sizeof(W) == 8) lost = lost || t != t;
      }
      if constexpr (RUN) z_lane[c] = z;
    }
    if (lost) z = NAN;
    auto add = [](auto p, auto q) { return p + q; };
    // (all sums before the first is stored: a branch in between, and what makes one of them is kept until after it)
    constexpr int SUMS = RUN ? CHUNKS : 1;
    double here[SUMS];
    if constexpr (RUN) {
#pragma unroll
      for (int c = 0; c < CHUNKS; c++) here[c] = head_lane_of(head_scan<double>(z_lane[c], 0.0, add), 63);
    } else {
      here[0] = head_lane_of(head_scan<W>(z, 0, add), 63);
    }
    s = head_lane_of(head_scan<W>(s, 0, add), 63);
    if (head_lane() == 0) {
#pragma unroll
      for (int c = 0; c < SUMS; c++) red.z[c * (THREADS / 64) + (threadIdx.x >> 6)] = here[c];
      red.s[threadIdx.x >> 6] = s;
    }
    __syncthreads();
    z = (W)head_total(red.z, SUMS * (THREADS / 64));
    s = (W)head_total(red.s, THREADS / 64);
    s = scale.finish(s);
    // +infinity is the largest, NaN has lost to everything but makes the sum NaN
    bad = !(m < (X)INFINITY) || z != z;
    empty = !bad && m == (X)-INFINITY;
  }
  // the first column of the largest
  __device__ __forceinline__ int first(long part0, HeadRed& red) const {
    int v = 0x7FFFFFFF;
#pragma unroll
    for (int c = CHUNKS - 1; c >= 0; c--) {
#pragma unroll
      for (int e = 7; e >= 0; e--)
        if (x[c][e] == m) v = (int)(part0 + at(c) + e);
    }
    return head_block_min(v, red.i);
  }
};

// ---- rows of up to HEAD_ROW columns: a block holds the row ---------------------------------------------------------------

// A row whose action 32 bits cannot tell, in 64: m is the row's largest, u its uniform.  It is read again.
template <int CHUNKS, int THREADS, typename X>
__device__ __forceinline__ void head_sample_again(const HeadArgs& a, const HeadRow& r, long row, X m, double u, const unsigned* counts, HeadRed& red,
                                                  int* actions, float* log_prob, float* entropy) {
  constexpr int WAVES = THREADS / 64;
  constexpr bool adjust = std::is_same<X, double>::value;
  const HeadScale<double> scale(r);
  const int wave = threadIdx.x >> 6;
  auto look = [&](int c, double* t, double* w) {
    const int at = (c * THREADS + threadIdx.x) * 8;
    X x[8];
    HeadRaw<8> raw;
    raw.template fetch<false, adjust>(r, a.logits, a.type, row * a.logits_row + at, at, a.width - at);
    raw.template columns<false, false, adjust>(r, a.type, at, a.width - at, counts + at, x, (float*)nullptr);
    head_again<8>(x, m, scale, t, w);
    double sum = 0.0;
#pragma unroll
    for (int e = 0; e < 8; e++) sum += w[e];
    return sum;
  };
  auto add = [](double p, double q) { return p + q; };
  double t[8], w[8], s = 0.0;
#pragma unroll 1
  for (int c = 0; c < CHUNKS; c++) {
    const double here = head_scan(look(c, t, w), 0.0, add);
    if (head_lane() == 63) red.z[c * WAVES + wave] = here;
#pragma unroll
    for (int e = 0; e < 8; e++) s = scale.sum(t[e], w[e], s);
  }
  s = head_scan(s, 0.0, add);
  if (head_lane() == 63) red.s[wave] = s;
  __syncthreads();
  const double z = head_total(red.z, CHUNKS * WAVES), target = u < 1.0 ? u * z : INFINITY;
  const HeadSpot spot = head_spot(red.z, CHUNKS * WAVES, 0.0, target);
  if (spot.entry % WAVES != wave) return;
  const int c = spot.entry / WAVES;
  double before;
  if (!head_lane_picks(look(c, t, w), spot.base, target, before)) return;
  const HeadPick<double> pick = head_pick<8>(w, t, before, target);
  head_sampled(row, false, false, (c * THREADS + (int)threadIdx.x) * 8 + pick.e, pick.t, z, scale.finish(head_total(red.s, WAVES)), scale, actions,
               log_prob, entropy);
}

// An action per row.  Bound by its instructions at 1024 columns (16384 rows bf16: 21 us for 34 MB, 17 of them the issue of 10.6
// million vector instructions); at 8192 these are 22 of 37 us (4096 rows), the rest is a row's barriers and its choice of a wave,
// then of a lane.  All in 64 bits: 39 and 122 us.
template <int CHUNKS, int THREADS, typename X>
__global__ __launch_bounds__(THREADS) void mg_sample_row_kernel(HeadArgs a, const float* __restrict__ uniforms, int* __restrict__ actions,
                                                               float* __restrict__ log_prob, float* __restrict__ entropy) {
  constexpr int WAVES = THREADS / 64;
  constexpr bool adjust = std::is_same<X, double>::value;
  __shared__ unsigned counts[adjust ? CHUNKS * THREADS * 8 : 1];
  __shared__ HeadRed red;
  const long row = head_block();
  if (row >= a.rows) return;
  const HeadRow r = head_row(a, row);
  const HeadScale<float> scale(r);
  HeadPart<CHUNKS, THREADS, X, float> h;
  h.template hold<false, true>(a, r, scale, row, 0, a.width, counts, red);
  if (h.bad || h.empty || !uniforms) {
    const int first = h.bad || h.empty ? -1 : h.first(0, red);
    if (threadIdx.x == 0) head_sampled(row, h.bad, h.empty, first, 0.f, h.z, h.s, scale, actions, log_prob, entropy);
    return;
  }
  const float uniform = uniforms[row];
  if (uniform != uniform) {
    if (threadIdx.x == 0) head_sampled(row, true, false, -1, 0.f, h.z, h.s, scale, actions, log_prob, entropy);
    return;
  }
  const double all = head_total(red.z, CHUNKS * WAVES), u = fmax((double)uniform, 0.0), target = u < 1.0 ? u * all : INFINITY;
  const HeadSpot spot = head_spot(red.z, CHUNKS * WAVES, 0.0, target);
  if (spot.entry % WAVES == (int)threadIdx.x >> 6) {
#pragma unroll
    for (int c = 0; c < CHUNKS; c++) {
      double before;
      if (c != spot.entry / WAVES || !head_lane_picks(h.z_lane[c], spot.base, target, before)) continue;
      float t[8], w[8];
      head_again<8>(h.x[c], h.m, scale, t, w);
      const HeadPick<float> pick = head_pick<8>(w, t, before, target);
      const bool sure = head_sure(pick, target, head_margin(all, h.s));
      if (sure) head_sampled(row, false, false, h.at(c) + pick.e, pick.t, h.z, h.s, scale, actions, log_prob, entropy);
      red.i[0] = sure;
    }
  }
  __syncthreads();
  if (!red.i[0])
    head_sample_again<CHUNKS, THREADS, X>(a, r, row, h.m, u, counts, red, actions, log_prob, entropy);
}

// Bound by its instructions: the issue of 6.8 million vector instructions is 11 of 13 us (16384 x 1024 bf16, 34 MB), of 8.7 million
// 14 of 19 (4096 x 8192, 67 MB, 3.5 TB/s).
template <int CHUNKS, int THREADS, typename X>
__global__ __launch_bounds__(THREADS) void mg_evaluate_row_kernel(HeadArgs a, const int* __restrict__ actions, float* __restrict__ log_prob,
                                                                 float* __restrict__ entropy, double* __restrict__ stats) {
  __shared__ unsigned counts[std::is_same<X, double>::value ? CHUNKS * THREADS * 8 : 1];
  __shared__ HeadRed red;
  const long row = head_block();
  if (row >= a.rows) return;
  const HeadRow r = head_row(a, row);
  const HeadScale<float> scale(r);
  const int act = actions[row];
  HeadPart<CHUNKS, THREADS, X, float> h;
  h.template hold<false, false>(a, r, scale, row, 0, a.width, counts, red);
  if ((int)threadIdx.x == (act >= 0 && act < a.width ? act / 8 % THREADS : 0)) {  // who holds the action's column
    X x = -INFINITY;
#pragma unroll
    for (int c = 0; c < CHUNKS; c++) {
#pragma unroll
      for (int e = 0; e < 8; e++) x = h.at(c) + e == act ? h.x[c][e] : x;
    }
    const float log_z = head_log(h.z), d = head_distance(r, h.m, x);
    log_prob[row] = h.bad ? NAN : h.empty ? 0.f : -d - log_z;
    entropy[row] = h.bad ? NAN : h.empty ? 0.f : log_z + h.s * head_inverse(h.z);
    if (stats) stats[2 * row] = h.bad ? NAN : (double)h.m, stats[2 * row + 1] = h.bad ? NAN : h.empty ? 0.0 : (double)log_z;
  }
}

// whether the action's token is left: allowed, and neither logit nor bias at -infinity
__device__ __forceinline__ bool head_left(const HeadArgs& a, const HeadRow& r, long row, int act) {
  if (act < 0 || act >= a.width) return false;
  HeadRow one = r;
  one.kind = 0;
  HeadRaw<1> raw;
  float l[1];
  raw.fetch<true, false>(one, a.logits, a.type, row * a.logits_row + act, act, 1);
  raw.values(a.type, l);
  return head_allowed(r, act) && l[0] > -INFINITY && (!r.bias || r.bias[act] > -INFINITY);
}

// For rows of up to MG_EVALUATE_STATS_WIDTH columns, whose sums are computed again (16384 x 1024 bf16: 20 us for 67 MB, 3.4 TB/s).
template <typename X>
__global__ __launch_bounds__(HEAD_THREADS / 2) void mg_evaluate_row_backward_kernel(HeadArgs a, const int* __restrict__ actions,
                                                                               const float* __restrict__ dlog_prob,
                                                                               const float* __restrict__ dentropy, void* __restrict__ dlogits) {
  constexpr int CHUNKS = 1, THREADS = HEAD_THREADS / 2;
  constexpr bool adjust = std::is_same<X, double>::value;
  __shared__ unsigned counts[adjust ? THREADS * 8 : 1];
  __shared__ HeadRed red;
  const long row = head_block();
  if (row >= a.rows) return;
  const HeadRow r = head_row(a, row);
  const HeadScale<float> scale(r);
  const int act = actions[row];
  const float gp_row = dlog_prob ? dlog_prob[row] : 0.f, gh = (dentropy ? dentropy[row] : 0.f) * scale.inv_temp;
  const bool left = head_left(a, r, row, act);
  HeadPart<CHUNKS, THREADS, X, float> h;
  h.template hold<true, false>(a, r, scale, row, 0, a.width, counts, red);
  // (a bad row's NaN reaches every token that is left)
  const float gp = h.bad ? NAN : left ? gp_row * scale.inv_temp : 0.f, inv_z = head_inverse(h.z), past = h.s * inv_z;
#pragma unroll
  for (int c = 0; c < CHUNKS; c++) {
    float y[8];
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const float q = h.w[c][e] * inv_z;
      float d = (h.at(c) + e == act ? gp : 0.f) - q * fmaf(gh, scale.surprise(h.far(c, e), past), gp);
      if (adjust) d *= h.slope[c][e];
      y[e] = h.x[c][e] != (X)-INFINITY ? d : 0.f;
    }
    if (h.at(c) < a.width) head_store<8>(dlogits, a.type, row * a.width + h.at(c), a.width - h.at(c), y);
  }
}

// ---- wider rows: parts, and a second launch that joins them ------------------------------------------------------------

// found[row][part] = M, Z, sum (M - x) exp(-d) / temperature (against the part's own M), bad, first column of M.  In 32 bits bound
// by memory (2048 x 32003 bf16, masks: 31 us for 139 MB, 4.4 TB/s), in 64, for sampling, by instructions (1024 x 32003 bf16 with
// its join 49 us for 66 MB; the issue of 24.3 million vector instructions is 40 of the parts' 43) or, with few rows, latency (16 x
// 131072 f16, all controls: 9.0 us).  The most likely action, which no 64-bit weight decides, takes the same way (50 us).
template <int CHUNKS, bool FIRST, typename X, typename W>
__global__ __launch_bounds__(HEAD_THREADS) void mg_head_parts_kernel(HeadArgs a, double* __restrict__ found) {
  constexpr bool ADJUST = std::is_same<X, double>::value;
  __shared__ unsigned counts[ADJUST ? CHUNKS * HEAD_CHUNK : 1];
  __shared__ HeadRed red;
  const long row = (long)blockIdx.z * gridDim.y + blockIdx.y;
  if (row >= a.rows) return;
  const long part0 = (long)blockIdx.x * (CHUNKS * HEAD_CHUNK);
  const int part_n = (int)min((long)CHUNKS * HEAD_CHUNK, a.width - part0);
  const HeadRow r = head_row(a, row);
  const HeadScale<W> scale(r);
  HeadPart<CHUNKS, HEAD_THREADS, X, W> h;
  h.template hold<false, false>(a, r, scale, row, part0, part_n, counts, red);
  const int first = FIRST ? h.first(part0, red) : 0;
  if (threadIdx.x == 0) {
    double* f = found + (row * gridDim.x + blockIdx.x) * HEAD_FOUND;
    f[0] = h.m; f[1] = h.z; f[2] = h.s; f[3] = h.bad ? 1.0 : 0.0; f[4] = first;
  }
}

struct HeadJoined { double m, z, s; bool bad, empty; };

// the parts of a row, by all lanes of a wave
__device__ __forceinline__ HeadJoined head_join(const double* f, int parts, const HeadScale<double>& scale, int lane) {
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
      const double d = (j.m - mi) * scale.inv_temp, w = scale.weight(j.m - mi), zi = f[i * HEAD_FOUND + 1];
      z += w * zi;
      s += w > 0.0 ? w * (f[i * HEAD_FOUND + 2] + d * zi) : 0.0;
    }
  j.z = head_group_sum(z, 64);
  j.s = head_group_sum(s, 64);
  return j;
}

// The part in which the running sum passes the target is looked at once more for the token (16 x 131072 f16, all controls: 6.8 us,
// a chain of memory latencies and the count of the history).
template <typename X>
__global__ __launch_bounds__(HEAD_THREADS) void mg_sample_join_kernel(HeadArgs a, int parts, const double* __restrict__ found,
                                                                const float* __restrict__ uniforms, int* __restrict__ actions,
                                                                float* __restrict__ log_prob, float* __restrict__ entropy) {
  constexpr bool adjust = std::is_same<X, double>::value;
  __shared__ unsigned counts[adjust ? HEAD_CHUNK : 1];
  __shared__ double red[16];
  const long row = head_block();
  if (row >= a.rows) return;
  const HeadRow r = head_row(a, row);
  const HeadScale<double> scale(r);
  const double* f = found + row * parts * HEAD_FOUND;
  const float uniform = uniforms ? uniforms[row] : 0.f;
  HeadJoined j = head_join(f, parts, scale, head_lane());
  j.bad = j.bad || uniform != uniform;
  const double u = fmax((double)uniform, 0.0), target = u < 1.0 ? u * j.z : INFINITY;
  HeadPick<double> pick{0, 0.0, 0.0, 0.0};
  bool picks = threadIdx.x == 0;
  int v0 = 0;
  if (!j.bad && !j.empty) {
    // every wave finds the part: the first whose running sum is above the target, or the last with any (without uniforms:
    // the first of those with the largest)
    double start = 0.0, run = 0.0;
    int part = -1, last = -1, best = a.width;
    for (int i0 = 0; i0 < parts && part < 0; i0 += 64) {
      const int i = i0 + head_lane();
      const double mi = i < parts ? f[i * HEAD_FOUND] : -INFINITY;
      const double w = mi == -INFINITY ? 0.0 : scale.weight(j.m - mi) * f[i * HEAD_FOUND + 1];
      const double to_here = run + head_scan(w, 0.0, [](double p, double q) { return p + q; });
      if (!uniforms && mi == j.m) best = min(best, (int)f[i * HEAD_FOUND + 4]);
      const unsigned long long over = __ballot(w > 0.0 && to_here > target), some = __ballot(w > 0.0);
      if (uniforms && over) {
        const int k = __ffsll(over) - 1;
        part = i0 + k;
        start = head_lane_of(to_here - w, k);
      } else if (some) {
        const int k = 63 - __clzll((long long)some);
        last = i0 + k;
        start = head_lane_of(to_here - w, k);
      }
      run = head_lane_of(to_here, 63);
    }
    if (!uniforms) {
      v0 = head_group_min(best, 64);
    } else {
      part = part >= 0 ? part : last;
      const long part0 = (long)part * HEAD_CHUNK;
      const int part_n = (int)min((long)HEAD_CHUNK, a.width - part0);
      const int at = threadIdx.x * 8, n = part_n - at;
      X x[8];
      double t[8], w[8], mine = 0.0;
      HeadRaw<8> raw;
      raw.template fetch<false, adjust>(r, a.logits, a.type, row * a.logits_row + part0 + at, (int)(part0 + at), n);
      if (adjust && a.history) head_count_columns(a, row, counts, part0, part_n);
      raw.template columns<false, false, adjust>(r, a.type, (int)(part0 + at), n, counts + at, x, (float*)nullptr);
#pragma unroll
      for (int e = 0; e < 8; e++) {
        t[e] = j.m - (double)x[e];
        w[e] = scale.weight(t[e]);
        mine += w[e];
      }
      const double here = head_scan(mine, 0.0, [](double p, double q) { return p + q; });
      if (head_lane() == 63) red[threadIdx.x >> 6] = here;
      __syncthreads();
      const HeadSpot spot = head_spot(red, HEAD_THREADS / 64, start, target);
      picks = false;
      if (spot.entry == (int)threadIdx.x >> 6) {
        double before;
        picks = head_lane_picks(mine, spot.base, target, before);
        if (picks) pick = head_pick<8>(w, t, before, target);
      }
      v0 = (int)(part0 + at);
      __syncthreads();
    }
  }
  if (picks) head_sampled(row, j.bad, j.empty, v0 + pick.e, pick.t, j.z, j.s, scale, actions, log_prob, entropy);
}

// One wave per row (2048 x 32003: 4.5 us, two memory latencies).
__global__ __launch_bounds__(HEAD_THREADS) void mg_evaluate_join_kernel(HeadArgs a, int parts, const double* __restrict__ found,
                                                                       const int* __restrict__ actions, float* __restrict__ log_prob,
                                                                       float* __restrict__ entropy, double* __restrict__ stats) {
  const long row = head_block() * (HEAD_THREADS / 64) + (threadIdx.x >> 6);
  if (row >= a.rows) return;
  const HeadRow r = head_row(a, row);
  const HeadJoined j = head_join(found + row * parts * HEAD_FOUND, parts, HeadScale<double>(r), head_lane());
  const int act = actions[row];
  const bool inside = act >= 0 && act < a.width;
  double x = -INFINITY;
  if (inside) {
    unsigned count = 0;
    if (a.history) {
      for (int i = head_lane(); i < a.history_len; i += 64) count += a.history[row * a.history_row + i] == act;
      count = head_group_sum(count, 64);
    }
    HeadRow one = r;  // (one column; its bit of the mask is not at a multiple of anything)
    one.kind = 0;
    HeadRaw<1> raw;
    double y[1];
    raw.fetch<true, true>(one, a.logits, a.type, row * a.logits_row + act, act, 1);
    raw.columns<false, false, true>(one, a.type, act, 1, &count, y, (float*)nullptr);
    x = head_allowed(r, act) ? y[0] : -INFINITY;
  }
  if (head_lane() == 0) {
    const double log_z = j.bad || j.empty ? 0.0 : head_log(j.z);
    log_prob[row] = j.bad ? NAN : j.empty ? 0.f : (float)((x - j.m) * r.inv_temp - log_z);
    entropy[row] = j.bad ? NAN : j.empty ? 0.f : (float)(log_z + j.s / j.z);
    if (stats) stats[2 * row] = j.bad ? NAN : j.m, stats[2 * row + 1] = j.bad ? NAN : log_z;
  }
}

// From the forward pass's stats, so that every block works alone.  Bound by memory: 2048 x 32003 bf16, masks: 47 us for 270 MB, 5.7
// TB/s (part of it still in the caches).
template <int CHUNKS, typename X>
__global__ __launch_bounds__(HEAD_THREADS) void mg_evaluate_wide_backward_kernel(HeadArgs a, const int* __restrict__ actions,
                                                                                const float* __restrict__ entropy,
                                                                                const double* __restrict__ stats,
                                                                                const float* __restrict__ dlog_prob,
                                                                                const float* __restrict__ dentropy,
                                                                                void* __restrict__ dlogits) {
  constexpr bool adjust = std::is_same<X, double>::value;
  __shared__ unsigned counts[adjust ? CHUNKS * HEAD_CHUNK : 1];
  const long row = (long)blockIdx.z * gridDim.y + blockIdx.y, part0 = (long)blockIdx.x * (CHUNKS * HEAD_CHUNK);
  if (row >= a.rows) return;
  const int part_n = (int)min((long)CHUNKS * HEAD_CHUNK, a.width - part0);
  const HeadRow r = head_row(a, row);
  const HeadScale<float> scale(r);
  const double m = stats[2 * row];
  const float log_z = (float)stats[2 * row + 1], past = (float)((double)entropy[row] - stats[2 * row + 1]);  // H - log Z
  const bool bad = m != m, empty = m == -INFINITY;
  const X top = bad || empty ? (X)0 : (X)m;
  const int act = actions[row];
  float gp = 0;
  const float gh = (dentropy ? dentropy[row] : 0.f) * scale.inv_temp;
  if (dlog_prob && head_left(a, r, row, act)) gp = dlog_prob[row] * scale.inv_temp;
  constexpr int THREADS [[maybe_unused]] = HEAD_THREADS;
  HeadRaw<8> raw[CHUNKS];
  HEAD_PART_FETCH((raw[c].template fetch<FULL, adjust>(r, a.logits, a.type, row * a.logits_row + part0 + at, (int)(part0 + at), n)))
  if (adjust && a.history) head_count_columns(a, row, counts, part0, part_n);
#pragma unroll
  for (int c = 0; c < CHUNKS; c++) {
    const int at = c * HEAD_CHUNK + threadIdx.x * 8, n = part_n - at, v0 = (int)(part0 + at);
    if (n <= 0) continue;
    X x[8];
    float g[8], slope[8], y[8];
    raw[c].template columns<false, true, adjust>(r, a.type, v0, n, counts + at, x, slope);
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const float t = (float)(top - x[e]);
      g[e] = -scale.weight(t, log_z) * fmaf(gh, scale.surprise(t, past), gp);
    }
    if ((unsigned)(act - v0) < 8u) {
#pragma unroll
      for (int e = 0; e < 8; e++) if (v0 + e == act) g[e] += gp;
    }
    if (bad) {
#pragma unroll
      for (int e = 0; e < 8; e++) g[e] = NAN;
    }
#pragma unroll
    for (int e = 0; e < 8; e++) {
      if (adjust) g[e] *= slope[e];
      y[e] = x[e] != (X)-INFINITY ? g[e] : 0.f;  // (masked, or no part of the row; nothing is left of an empty one)
    }
    head_store<8>(dlogits, a.type, row * a.width + v0, n, y);
  }
}

// ---- host side --------------------------------------------------------------------------------------------------------

static int head_check(const char* who, const mg_logits* a) {
  const std::string w(who);
  if (!a) return mg_fail_msg(w + ": NULL arguments");
  if (a->rows < 0 || a->width < 1) return mg_fail_msg(w + ": a row has at least one token");
  if (a->type < 0 || a->type > 2) return mg_fail_msg(w + ": type must be MG_F32, MG_BF16 or MG_F16");
  // (so that neither they nor their inverses leave the range of 32 bits)
  if (!(a->temperature >= 1e-30 && a->temperature <= 1e30)) return mg_fail_msg(w + ": temperature must be from 1e-30 to 1e30");
  if (!(a->repetition >= 1e-30 && a->repetition <= 1e30)) return mg_fail_msg(w + ": repetition must be from 1e-30 to 1e30");
  if (!(std::abs(a->presence) < INFINITY && std::abs(a->frequency) < INFINITY)) return mg_fail_msg(w + ": penalties must be finite");
  if (a->allowed && a->allowed_kind != MG_ALLOWED_BOOL && a->allowed_kind != MG_ALLOWED_BITS)
    return mg_fail_msg(w + ": allowed_kind must be MG_ALLOWED_BOOL or MG_ALLOWED_BITS");
  if (a->history && (a->history_len < 1 || a->history_len > 1 << 30)) return mg_fail_msg(w + ": a history has 1 to 2^30 entries");
  if (a->rows && !a->logits) return mg_fail_msg(w + ": NULL tensor");
  return 0;
}

static HeadArgs head_args(const mg_logits* a) {
  HeadArgs g;
  (mg_logits&)g = *a;
  g.inv_temp = 1.0 / a->temperature;
  g.inv_rep = 1.0 / a->repetition;
  g.weight_scale = g.inv_temp * -1.4426950408889634;
  return g;
}

// A part is a chunk, which is as fast as larger parts or faster (sampling 2048 x 8193 bf16: 38 us, with four chunks 86;
// adjustment 4096 x 8192: 25 and 28), but for the evaluation of large batches: 2048 x 32003 takes 31 + 47 us in parts of four
// chunks and 46 + 56 in single ones (64 x 50001: 8.9 and 8.2; 2048 x 8193, of whose parts half would be nearly empty: 22 and 19).
static int head_chunks(const mg_logits* a) { return a->width > 2 * HEAD_ROW && a->rows * (a->width / HEAD_ROW) >= 2048 ? 4 : 1; }
static int head_parts(const mg_logits* a, int chunks = 1) { return (a->width - 1) / (chunks * HEAD_CHUNK) + 1; }
// A block does one row (or, of narrow ones, as many as its lanes hold) and no loop over them: the compiler would keep what does
// not change from row to row in registers, the constants of a rare path too.
static dim3 head_wide_grid(const mg_logits* a, int chunks = 1) {
  const int64_t y = a->rows < 32768 ? a->rows : 32768;
  return dim3(head_parts(a, chunks), (unsigned)y, (unsigned)((a->rows + y - 1) / y));
}
// (a dimension of a grid has fewer than 2^32 threads)
static dim3 head_grid(int64_t blocks) {
  const int64_t x = blocks < 1 << 20 ? blocks : 1 << 20;
  return dim3((unsigned)x, (unsigned)((blocks + x - 1) / x));
}
static bool head_narrow(const mg_logits* a) { return a->width <= HEAD_NARROW; }
static bool head_remembers(const mg_logits* a) { return a->width > MG_EVALUATE_STATS_WIDTH; }  // what the forward pass found
static bool head_wide(const mg_logits* a) { return a->width > HEAD_ROW; }

// lanes per row: as many as hold the row with E columns each; a power of two where they work on it together
static HeadNarrow head_layout(const mg_logits* a, int e, bool together) {
  int lanes = together ? 1 : (a->width + e - 1) / e;
  while (lanes * e < a->width) lanes *= 2;
  return HeadNarrow{lanes, HEAD_THREADS / lanes};
}

template <int V> using head_int = std::integral_constant<int, V>;
template <bool V> using head_bool = std::integral_constant<bool, V>;
template <typename F>
static void head_by_width(const mg_logits* a, F f) {
  const head_bool<true> one;
  const HeadNarrow g{1, HEAD_THREADS};
  switch (a->width) {
    case 1: return f(head_int<1>(), one, g);
    case 2: return f(head_int<2>(), one, g);
    case 3: return f(head_int<3>(), one, g);
    case 4: return f(head_int<4>(), one, g);
    case 5: return f(head_int<5>(), one, g);
    case 6: return f(head_int<6>(), one, g);
    case 7: return f(head_int<7>(), one, g);
    case 8: return f(head_int<8>(), one, g);
  }
  // as few lanes as eight columns each allow, then as few columns as so many lanes allow (65536 x 157 bf16 in five columns each:
  // sampling 21 us, evaluation 15 and its gradient 20; in eight, 20 lanes of 32: 27, 18 and 25)
  const head_bool<false> several;
  const HeadNarrow group = head_layout(a, 8, true);
  switch ((a->width + group.lanes - 1) / group.lanes) {
    case 5: return f(head_int<5>(), several, group);
    case 6: return f(head_int<6>(), several, group);
    case 7: return f(head_int<7>(), several, group);
  }
  f(head_int<8>(), several, group);
}
// How a block holds a row: chunks of eight columns per thread, and threads.  Rather more chunks than more threads to wait for
// (4096 x 8192 bf16: evaluation 19 us and sampling 37 with 256 threads, 27 and 77 with 1024; only where there are few rows is it
// the other way round, 64 x 8192: 4.6 and 10.5 us, 3.9 and 9.0).
template <typename F>
static void head_by_row(const mg_logits* a, F f) {
  if (a->width <= HEAD_CHUNK / 2) f(head_int<1>(), head_int<HEAD_THREADS / 2>());
  else if (a->width <= HEAD_CHUNK) f(head_int<1>(), head_int<HEAD_THREADS>());
  else if (a->width <= 2 * HEAD_CHUNK) f(head_int<2>(), head_int<HEAD_THREADS>());
  else f(head_int<4>(), head_int<HEAD_THREADS>());
}
template <typename F>
static void head_by_chunks(const mg_logits* a, F f) {
  if (head_chunks(a) == 4) f(head_int<4>());
  else f(head_int<1>());
}
// the type of the logits' values: 64 bits where there is a bias or a penalty, which could cancel large logits
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
  if (head_wide(a) && (!a->workspace || a->workspace_bytes < mg_logits_workspace(a)))
    return mg_fail_msg(std::string(who) + ": workspace smaller than mg_logits_workspace says");
  return 0;
}

extern "C" int64_t mg_logits_workspace(const mg_logits* a) {
  if (!a || a->rows <= 0 || a->width < 1 || !head_wide(a)) return 0;
  return a->rows * head_parts(a) * HEAD_FOUND * (int64_t)sizeof(double);
}

static int head_adjust(const char* who, const mg_logits* a, void* out, const void* dout, void* dlogits, void* stream) {
  const hipStream_t s = (hipStream_t)stream;
  if (a->width <= HEAD_CHUNK / 2) {
    const HeadNarrow g = head_layout(a, 8, false);
    hipLaunchKernelGGL(mg_adjust_narrow_kernel<8>, head_grid((a->rows + g.rows - 1) / g.rows), dim3(HEAD_THREADS), 0, s, head_args(a), g, out, dout, dlogits);
  } else {
    hipLaunchKernelGGL(mg_adjust_wide_kernel, head_wide_grid(a), dim3(HEAD_THREADS), 0, s, head_args(a), out, dout, dlogits);
  }
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
  head_by_controls(a, [&](auto* null) {
    using X = std::remove_pointer_t<decltype(null)>;
    if (head_narrow(a)) {
      head_by_width(a, [&](auto e, auto one, HeadNarrow g) {
        hipLaunchKernelGGL((mg_sample_narrow_kernel<decltype(e)::value, decltype(one)::value, X>), head_grid((a->rows + g.rows - 1) / g.rows),
                           dim3(HEAD_THREADS), 0, s, head_args(a), g, uniforms, actions, log_prob, entropy);
      });
    } else if (!head_wide(a)) {
      head_by_row(a, [&](auto c, auto t) {
        hipLaunchKernelGGL((mg_sample_row_kernel<decltype(c)::value, decltype(t)::value, X>), head_grid(a->rows), dim3(decltype(t)::value), 0, s,
                           head_args(a), uniforms, actions, log_prob, entropy);
      });
    } else {
      if (uniforms)
        hipLaunchKernelGGL((mg_head_parts_kernel<1, false, X, double>), head_wide_grid(a), dim3(HEAD_THREADS), 0, s, head_args(a), (double*)a->workspace);
      else
        hipLaunchKernelGGL((mg_head_parts_kernel<1, true, X, double>), head_wide_grid(a), dim3(HEAD_THREADS), 0, s, head_args(a), (double*)a->workspace);
      hipLaunchKernelGGL(mg_sample_join_kernel<X>, head_grid(a->rows), dim3(HEAD_THREADS), 0, s, head_args(a), head_parts(a),
                         (const double*)a->workspace, uniforms, actions, log_prob, entropy);
    }
  });
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
      head_by_width(a, [&](auto e, auto one, HeadNarrow g) {
        hipLaunchKernelGGL((mg_evaluate_narrow_kernel<decltype(e)::value, decltype(one)::value, X>), head_grid((a->rows + g.rows - 1) / g.rows), dim3(HEAD_THREADS), 0, s,
                           head_args(a), g, actions, log_prob, entropy);
      });
    } else if (!head_wide(a)) {
      head_by_row(a, [&](auto c, auto t) {
        hipLaunchKernelGGL((mg_evaluate_row_kernel<decltype(c)::value, decltype(t)::value, X>), head_grid(a->rows), dim3(decltype(t)::value), 0,
                           s, head_args(a), actions, log_prob, entropy, stats);
      });
    } else {
      head_by_chunks(a, [&](auto c) {
        constexpr int C = decltype(c)::value;
        hipLaunchKernelGGL((mg_head_parts_kernel<C, false, X, float>), head_wide_grid(a, C), dim3(HEAD_THREADS), 0, s, head_args(a), (double*)a->workspace);
      });
    }
  });
  if (head_wide(a))
    hipLaunchKernelGGL(mg_evaluate_join_kernel, head_grid((a->rows + HEAD_THREADS / 64 - 1) / (HEAD_THREADS / 64)), dim3(HEAD_THREADS), 0, s, head_args(a),
                       head_parts(a, head_chunks(a)), (const double*)a->workspace, actions, log_prob, entropy, stats);
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
  if (!actions || !dlogits || (head_remembers(a) && (!entropy || !stats))) return mg_fail_msg(std::string(who) + ": NULL tensor");
  const hipStream_t s = (hipStream_t)stream;
  head_by_controls(a, [&](auto* null) {
    using X = std::remove_pointer_t<decltype(null)>;
    if (head_narrow(a))
      head_by_width(a, [&](auto e, auto one, HeadNarrow g) {
        hipLaunchKernelGGL((mg_evaluate_narrow_backward_kernel<decltype(e)::value, decltype(one)::value, X>), head_grid((a->rows + g.rows - 1) / g.rows), dim3(HEAD_THREADS),
                           0, s, head_args(a), g, actions, dlog_prob, dentropy, dlogits);
      });
    else if (!head_remembers(a))
      hipLaunchKernelGGL(mg_evaluate_row_backward_kernel<X>, head_grid(a->rows), dim3(HEAD_THREADS / 2), 0, s, head_args(a), actions,
                         dlog_prob, dentropy, dlogits);
    else
      head_by_chunks(a, [&](auto c) {
        constexpr int C = decltype(c)::value;
        hipLaunchKernelGGL((mg_evaluate_wide_backward_kernel<C, X>), head_wide_grid(a, C), dim3(HEAD_THREADS), 0, s, head_args(a), actions, entropy,
                           stats, dlog_prob, dentropy, dlogits);
      });
  });
  return head_launched(who);
} catch (...) {
  return 1;
}
