// mev_learn.hip -- MI355X (gfx950) kernels + C ABI of the policy operators (mev.h,
// mobile_env.learning): the clipped policy loss over categorical logits with its gradient, the
// log-probability of an action, the advantages of a rollout, and clipping to a global norm.
//
// All of them are bound by memory (a large copy reaches 4.8 to 5.1 TB/s on an MI355X) or, when
// small, by their launches; figures are of an MI355X, times here medians of the kernels' own, below
// per call unless said otherwise.
//
// Policy rows. Per row m = max x, s = sum e^(x-m), t = sum e^(x-m) (x-m) give everything:
// log p = (x - m) - ln s, the entropy H = ln s - t / s, and with c = dloss/dlog p(action) the
// gradient w (c (1[action] - p) + h p (log p + H)) = e^(x-m) (ga + gb log p) + gc 1[action], with
// 1 / s in ga and gb. A row is read once and stays in registers until its gradient is written: by
// one lane (few actions), by 2 to 64 lanes of a wavefront, or by a workgroup of up to 1,024; rows
// beyond that, and long ones that are too few for the chip, are split over workgroups and read
// twice. 23 vector instructions an element, two of them exponentials at a quarter of the rate, issue
// in 0.8 of the time that its bytes take in 16 bits. 10,240 rows of 40,000 bf16 (a quarter of them
// without weight) move 1.44 GB in 287 us: 5.0 TB/s; 8,192 rows of 4,096 f32 in 50 us, partly out
// of the memory-side cache.
// Advantages. A scan of maps over the lanes of a column; 20 steps of 262,144 columns 16.4 us
// (5.4 TB/s); rewards read from column 3 of the observations take their whole cache lines
// (20 x 32,768 x 30: 518 MB for 278 MB asked, 96 us).
// Clipping. Two passes (the norm has to be whole before anything is scaled), the second from the
// end: 1.07 GB of gradients 215 + 401 us (5.2 TB/s on read, read, write).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <new>
#include <vector>

#include "mev.h"
#include "mev_internal.h"

namespace {

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLog2eLow = 1.92596299112661746887e-8f;  // log2 e - kLog2e
constexpr float kLn2 = 0.69314718055994530942f;

// --------------------------------------------------------------------------------------
// element types: 16-byte vectors of them, widened to float and rounded back (to nearest even)
// --------------------------------------------------------------------------------------
struct alignas(16) Vec {
  uint32_t w[4];
};
struct F32 {
  using elem = float;
  static constexpr int kPer = 4;  // elements of a vector
  static constexpr uint32_t kNegInf = 0xff800000u;
  static __device__ float widen(float v) { return v; }
  static __device__ float narrow(float v) { return v; }
  static __device__ void unpack(const Vec& v, float* x) {
    for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(v.w[i]);
  }
  static __device__ Vec pack(const float* x) {
    Vec v;
    for (int i = 0; i < 4; ++i) v.w[i] = __float_as_uint(x[i]);
    return v;
  }
};
struct BF16 {
  using elem = __bf16;
  static constexpr int kPer = 8;
  static constexpr uint32_t kNegInf = 0xff80ff80u;
  static __device__ float widen(__bf16 v) { return (float)v; }
  static __device__ __bf16 narrow(float v) { return (__bf16)v; }
  static __device__ void unpack(const Vec& v, float* x) {
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(v.w[i] << 16);
      x[2 * i + 1] = __uint_as_float(v.w[i] & 0xffff0000u);
    }
  }
  static __device__ Vec pack(const float* x) {
    Vec v;
    for (int i = 0; i < 4; ++i) {
      typedef __bf16 Pair __attribute__((ext_vector_type(2)));
      const Pair p = {(__bf16)x[2 * i], (__bf16)x[2 * i + 1]};
      v.w[i] = __builtin_bit_cast(uint32_t, p);
    }
    return v;
  }
};
struct F16 {
  using elem = _Float16;
  static constexpr int kPer = 8;
  static constexpr uint32_t kNegInf = 0xfc00fc00u;
  static __device__ float widen(_Float16 v) { return (float)v; }
  static __device__ _Float16 narrow(float v) { return (_Float16)v; }
  typedef _Float16 Pair __attribute__((ext_vector_type(2)));
  static __device__ void unpack(const Vec& v, float* x) {
    for (int i = 0; i < 4; ++i) {
      const Pair p = __builtin_bit_cast(Pair, v.w[i]);
      x[2 * i] = (float)p.x;
      x[2 * i + 1] = (float)p.y;
    }
  }
  static __device__ Vec pack(const float* x) {
    Vec v;
    for (int i = 0; i < 4; ++i) {
      const Pair p = {(_Float16)x[2 * i], (_Float16)x[2 * i + 1]};
      v.w[i] = __builtin_bit_cast(uint32_t, p);
    }
    return v;
  }
};

// 16 bytes at any element: rows start where they start (an odd number of 16-bit actions), and a
// global access of this hardware needs no more than its element's alignment.
template <class E>
__device__ inline Vec load16(const E* p) {
  Vec v;
  __builtin_memcpy(&v, p, 16);
  return v;
}
template <class E>
__device__ inline void store16(E* p, const Vec& v) {
  __builtin_memcpy(p, &v, 16);
}
// The same at element i of a row: an offset of 32 bits beside the row's (scalar) address.
template <class E>
__device__ inline Vec load16(const E* row, uint32_t i) {
  return load16((const E*)((const char*)row + i * (uint32_t)sizeof(E)));
}
template <class E>
__device__ inline void store16(E* row, uint32_t i, const Vec& v) {
  store16((E*)((char*)row + i * (uint32_t)sizeof(E)), v);
}

// --------------------------------------------------------------------------------------
// policy rows
// --------------------------------------------------------------------------------------
// Of a row: the maximum m, s = sum e^(x-m), t = sum e^(x-m) (x-m). m is -inf where every logit
// is (then s = 0); a NaN logit makes s NaN.
struct Stats {
  float m, s, t;
};

// 2^x, one instruction: 1 ulp, results below 2^-126 are 0
__device__ inline float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ inline float finite_max(float m) { return m == -INFINITY ? 0.0f : m; }

// A difference that e^d turns into 0 anyway, kept where d times a sum stays finite (logits may be
// -inf or the type's lowest value).
__device__ inline float bound(float d) { return fmaxf(d, -200.0f); }

__device__ inline Stats join(const Stats& a, const Stats& b) {
  const float m = fmaxf(a.m, b.m), g = finite_max(m);
  const float da = bound(a.m - g), db = bound(b.m - g);
  const float fa = exp2_hw(da * kLog2e), fb = exp2_hw(db * kLog2e);
  return Stats{m, a.s * fa + b.s * fb, (a.t + da * a.s) * fa + (b.t + db * b.s) * fb};
}

__device__ inline void add(Stats& a, float x) {
  if (x > a.m) {
    const float d = bound(a.m - x), f = exp2_hw(d * kLog2e);
    a.t = (a.t + d * a.s) * f;
    a.s *= f;
    a.m = x;
  }
  const float d = x - finite_max(a.m), e = exp2_hw(d * kLog2e);  // (NaN where the logit is)
  a.s += e;
  a.t += e * bound(d);
}

struct PolicyRow {
  float logp, ent;   // outputs
  float m, lns;      // log p = (x - m) - lns
  float ga, gb, gc;  // gradient: e^(x - m) (ga + gb log p), plus gc at the action
  bool none;         // no distribution (every logit -inf)
};

// e^x within 2 ulp: the rounding of x log2 e is made up for behind the exponential
__device__ inline float exp_full(float x) {
  const float h = x * kLog2e;
  const float l = __builtin_fmaf(x, kLog2e, -h) + x * kLog2eLow;
  const float e = exp2_hw(h);
  // (0, infinity: l may be infinite or NaN there)
  return e > 0.0f && e < INFINITY ? __builtin_fmaf(e, l * kLn2, e) : e;
}

// e^d - d - 1 without cancellation: its series near 0 (8 terms: 2^-25 relative at |d| = 0.5)
__device__ inline float exp_rest(float d) {
  if (!(fabsf(d) < 0.5f)) {
    const float e = exp_full(d);
    return d > 64.0f ? e : (e - 1.0f) - d;
  }
  float p = 1.0f / 362880.0f;
  p = __builtin_fmaf(p, d, 1.0f / 40320.0f);
  p = __builtin_fmaf(p, d, 1.0f / 5040.0f);
  p = __builtin_fmaf(p, d, 1.0f / 720.0f);
  p = __builtin_fmaf(p, d, 1.0f / 120.0f);
  p = __builtin_fmaf(p, d, 1.0f / 24.0f);
  p = __builtin_fmaf(p, d, 1.0f / 6.0f);
  p = __builtin_fmaf(p, d, 0.5f);
  return p * d * d;
}

struct PolicyArgs {
  const void* logits;
  const void* action;
  const float *old_logp, *advantage, *weight, *ref_logp;
  float *logp, *entropy;
  double* part;  // [gridDim.x] partial losses, summed by k_sum_loss
  float* loss;   // NULL: no loss
  void* grad;
  const float* grad_scale;
  int64_t rows, inner, outer_stride, inner_stride;
  int actions, action_bytes, skip_unit_scale;
  double unit_weight, clip_lo, clip_hi, kl, ent;
  float above, below;  // a ratio is clipped beyond these: clip_lo / clip_hi rounded inwards
};

// A workgroup's part of the loss; alone it is the loss.
__device__ inline void put_loss(const PolicyArgs& a, double wl) {
  if (gridDim.x == 1) *a.loss = (float)wl;
  else a.part[blockIdx.x] = wl;
}

// What a row brings beside its logits, asked for together with them.
struct RowIn {
  int action;  // -1: out of range
  float xa;    // the action's logit, or NaN
  float old_logp, advantage, ref_logp;
};

// No branch around a load (each would be waited for where its branch ends): what is not given is
// read from the actions instead, and not used.
template <class E>
__device__ inline RowIn row_in(const PolicyArgs& a, int64_t row, const E* x) {
  RowIn in;
  const char* ap = (const char*)a.action + row * a.action_bytes;
  const uint32_t low = *(const uint32_t*)ap;
  const uint32_t high = *(const uint32_t*)(ap + (a.action_bytes & 8) / 2);  // (low again, if 4)
  const float* any = (const float*)ap;
  in.old_logp = *(a.old_logp ? a.old_logp + row : any);
  in.advantage = *(a.advantage ? a.advantage + row : any);
  in.ref_logp = *(a.ref_logp ? a.ref_logp + row : any);
  const bool ok = low < (uint32_t)a.actions && (high == 0 || a.action_bytes == 4);
  const float xa = (float)x[ok ? low : 0];
  in.action = ok ? (int)low : -1;
  in.xa = ok ? xa : NAN;
  return in;
}

// Row `row` of the logits.
template <class E>
__device__ inline const E* row_ptr(const PolicyArgs& a, int64_t row) {
  if (a.inner == a.rows) return (const E*)a.logits + row * a.inner_stride;  // (no division)
  return (const E*)a.logits + (row / a.inner) * a.outer_stride + (row % a.inner) * a.inner_stride;
}

// The row's scalars from its statistics, in 32 bits (the row's logits wait in registers).
__device__ inline PolicyRow policy_row(const PolicyArgs& a, const RowIn& in, const Stats& st,
                                       float ws) {
  PolicyRow r;
  r.none = st.s == 0.0f;
  r.m = finite_max(st.m);
  r.lns = logf(st.s);
  r.logp = (in.xa - r.m) - r.lns;
  r.ent = r.lns - st.t / st.s;
  r.ga = r.gb = r.gc = 0.0f;
  if (r.none) {
    r.logp = in.xa;  // -inf, or NaN for an action out of range
    r.ent = 0.0f;
    return r;
  }
  if (!a.old_logp) return r;
  const float ratio = exp_full(r.logp - in.old_logp);
  // (no advantage: no gradient, also where the ratio is beyond float32)
  const bool cut = (in.advantage >= 0.0f && ratio > a.above) ||
                   (in.advantage < 0.0f && ratio < a.below);
  float c = cut ? 0.0f : -ratio * in.advantage;
  if (a.ref_logp) {
    const float d = in.ref_logp - r.logp;
    c -= (float)a.kl * (exp_rest(d) + d);
  }
  r.gc = ws * c;
  r.gb = ws * (float)a.ent;
  r.ga = __builtin_fmaf(r.gb, r.ent, -r.gc);
  const float one = __builtin_amdgcn_rcpf(st.s);  // p = e^(x - m) / s
  r.ga *= one;
  r.gb *= one;
  return r;
}

// ln s of a sum 1 <= s < 2^31, to 1e-10: with s = 2^k f, f within a factor sqrt 2 of 1, and
// z = (f - 1) / (f + 1), ln f = 2 (z + z^3 / 3 + z^5 / 5 + ...), z^2 < 0.03.
__device__ inline double log_near(float s) {
  const uint32_t bits = __float_as_uint(s);
  int k = (int)(bits >> 23) - 127;
  float f = __uint_as_float((bits & 0x007fffffu) | 0x3f800000u);
  if (f > 1.41421356f) f *= 0.5f, ++k;
  const double den = 1.0 + (double)f;
  double q = __builtin_amdgcn_rcp(den);
  q = __builtin_fma(__builtin_fma(-den, q, 1.0), q, q);  // (one step from the hardware's start)
  const double z = ((double)f - 1.0) * q, y = z * z;
  double p = 1.0 / 11.0;
  p = __builtin_fma(p, y, 1.0 / 9.0);
  p = __builtin_fma(p, y, 1.0 / 7.0);
  p = __builtin_fma(p, y, 1.0 / 5.0);
  p = __builtin_fma(p, y, 1.0 / 3.0);
  p = __builtin_fma(p, y, 1.0);
  return __builtin_fma((double)k, 0.69314718055994530942, 2.0 * z * p);
}

// e^x to 1e-10: x = k ln 2 + r, |r| <= 0.35, and the series of e^r to r^9.
__device__ inline double exp_near(double x) {
  x = x > 800.0 ? 800.0 : x < -800.0 ? -800.0 : x;  // (0 and inf beyond; NaN stays)
  const double k = __builtin_rint(x * 1.44269504088896340736);
  const double r = __builtin_fma(-k, 0.69314718055994530942, x);
  double p = 1.0 / 362880.0;
  p = __builtin_fma(p, r, 1.0 / 40320.0);
  p = __builtin_fma(p, r, 1.0 / 5040.0);
  p = __builtin_fma(p, r, 1.0 / 720.0);
  p = __builtin_fma(p, r, 1.0 / 120.0);
  p = __builtin_fma(p, r, 1.0 / 24.0);
  p = __builtin_fma(p, r, 1.0 / 6.0);
  p = __builtin_fma(p, r, 0.5);
  p = __builtin_fma(p, r, 1.0);
  p = __builtin_fma(p, r, 1.0);
  return __builtin_amdgcn_ldexp(p, (int)k);
}

// Weight times the row's loss, for one lane of the row. In 64 bits from the row's sum on: the rows
// of a batch nearly cancel, and 1.2 in float32 alone moved the mean of a million rows by 1e-5 of
// its value. (It takes 4 us of a million short rows' 26; ln and exp only to what a sum needs.)
__device__ inline double row_loss(const PolicyArgs& a, const RowIn& in, const Stats& st,
                                  const PolicyRow& r, double w) {
  if (r.none) return in.action < 0 ? w * (double)NAN : 0.0;
  if (!(st.s >= 1.0f)) return w * (double)st.s;  // NaN
  const double logp = ((double)in.xa - (double)r.m) - log_near(st.s);
  const double ratio = exp_near(logp - in.old_logp);
  const double adv = in.advantage, one = ratio * adv;
  const double two = (ratio < a.clip_lo ? a.clip_lo : ratio > a.clip_hi ? a.clip_hi : ratio) * adv;
  double l = one > two ? -two : -one;  // (NaN: NaN)
  if (a.ref_logp) l += a.kl * exp_rest((float)(in.ref_logp - logp));
  l -= a.ent * r.ent;
  return w * l;
}

__device__ inline float policy_grad(const PolicyRow& r, float x) {
  const float d = x - r.m, e = exp2_hw(d * kLog2e);  // (of d, not of log p: a rounding less)
  return e * __builtin_fmaf(r.gb, bound(d - r.lns), r.ga);
}

// Sum over a workgroup in a fixed order; every thread gets it.
template <int kBlock>
__device__ inline double block_sum(double v, double* lds) {
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0.0;
  for (int i = 0; i < kBlock / 64; ++i) v += lds[i];
  return v;
}

// The statistics of W neighbouring lanes, for each of them: their maximum, every lane's sums moved
// to it once, then added.
template <int W>
__device__ inline Stats lanes_join(Stats a) {
  float m = a.m;
#pragma unroll
  for (int o = W / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
  const float d = bound(a.m - finite_max(m)), f = exp2_hw(d * kLog2e);
  float t = __builtin_fmaf(d, a.s, a.t) * f, s = a.s * f;
#pragma unroll
  for (int o = W / 2; o > 0; o >>= 1) {
    s += __shfl_xor(s, o);
    t += __shfl_xor(t, o);
  }
  return Stats{m, s, t};
}

// The vector as it is, but unknown to the compiler: what was unpacked from it before is not kept
// alive beside it (a row of bf16 would take three times its registers).
__device__ inline void forget(Vec& v) {
  asm volatile("" : "+v"(v.w[0]), "+v"(v.w[1]), "+v"(v.w[2]), "+v"(v.w[3]));
}

// A row's last vector ends with the row, and its first `again` elements are those of the one before:
// the rest of them, of each word.
template <class T>
__device__ inline void last_vector(int again, uint32_t (&keep)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int left = again - i * (T::kPer / 4);  // of this word's elements, and behind
    keep[i] = left <= 0 ? ~0u : T::kPer == 8 && left == 1 ? 0xffff0000u : 0u;
  }
}

// A row in the registers of G lanes, NV vectors of 16 bytes each, the last one ending with the row
// (it may repeat elements of the one before; they count once, and both write the same gradient):
// read once, its statistics formed relative to each lane's own maximum and joined once, the
// gradient written from the registers.
template <class T, int G, int NV>
__global__ __launch_bounds__(G < 256 ? 256 : G, 4) void k_policy_regs(PolicyArgs a) {
  constexpr int kBlock = G < 256 ? 256 : G, kRows = kBlock / G, kPer = T::kPer;
  using E = typename T::elem;
  __shared__ Stats part[2][16];
  __shared__ double lsum[4];
  float scale = 1.0f;
  if (a.grad_scale) {
    scale = *a.grad_scale;
    if (a.skip_unit_scale && scale == 1.0f) return;
  }
  const int V = a.actions, nvec = (V + kPer - 1) / kPer, last = V - kPer;
  uint32_t keep[4];
  last_vector<T>(nvec * kPer - V, keep);
  double wl = 0.0;
  int flip = 0;
  // a row of whole wavefronts is the same for each of them: its addresses and inputs stay scalar
  const int sub = kRows == 1 ? 0
                  : G == 64  ? __builtin_amdgcn_readfirstlane(threadIdx.x / G)
                             : threadIdx.x / G;
  for (int64_t row = (int64_t)blockIdx.x * kRows + sub; row < a.rows;
       row += (int64_t)gridDim.x * kRows) {
    // What a lane derives from its number is derived anew for each row, and again for the
    // gradient: kept over the loop it takes a register a vector (a row of 40,000 bf16 then fits a
    // unit once, not twice).
    int lane = threadIdx.x % G;
    asm volatile("" : "+v"(lane));
    const float w = a.weight ? a.weight[row] : (float)a.unit_weight;
    E* g = a.grad ? (E*)a.grad + row * V : nullptr;
    if (w == 0.0f) {
      if (lane == 0 && a.logp) a.logp[row] = 0.0f, a.entropy[row] = 0.0f;
      for (int i = lane; g && i < nvec; i += G) store16(g, min(i * kPer, last), Vec{});
      continue;
    }
    const E* x = row_ptr<E>(a, row);
    Vec v[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j)  // (clamped, not branched around: all loads are in flight)
      v[j] = load16(x, min((j * G + lane) * kPer, last));
    const RowIn in = row_in(a, row, x);
    const int act = in.action;
    Stats st{-INFINITY, 0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      float f[kPer];
      T::unpack(v[j], f);
#pragma unroll
      for (int k = 0; k < kPer; ++k) st.m = fmaxf(st.m, f[k]);
    }
    const float m0 = finite_max(st.m);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      float f[kPer];
      // (behind the sums so far: masked one at a time, else a copy of the whole row stays alive)
      asm volatile("" : "+v"(v[j].w[0]), "+v"(v[j].w[1]), "+v"(v[j].w[2]), "+v"(v[j].w[3]),
                   "+v"(st.s), "+v"(st.t));
      Vec once = v[j];
      if ((j + 1) * G >= nvec) {
        int i = j * G + lane;
        asm volatile("" : "+v"(i));  // (a branch: most vectors need no mask)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t mask = i < nvec - 1 ? ~0u : i < nvec ? keep[k] : 0u;
          once.w[k] = (once.w[k] & mask) | (T::kNegInf & ~mask);
        }
      }
      T::unpack(once, f);
#pragma unroll
      for (int k = 0; k < kPer; ++k) {
        const float d = f[k] - m0, e = exp2_hw(d * kLog2e);
        st.s += e;
        st.t = __builtin_fmaf(e, bound(d), st.t);
      }
    }
    st = lanes_join<(G < 64 ? G : 64)>(st);
    if (G > 64) {
      Stats* p = part[flip];
      flip ^= 1;  // (the next row's are written while this row's may still be read)
      if ((threadIdx.x & 63) == 0) p[threadIdx.x >> 6] = st;
      __syncthreads();
      st = lanes_join<(G > 64 ? G / 64 : 1)>(p[threadIdx.x & (G / 64 - 1)]);
    }
    const PolicyRow r = policy_row(a, in, st, w * scale);
    if (lane == 0 && a.logp) a.logp[row] = r.logp, a.entropy[row] = r.ent;
    if (g && r.none) {
      for (int i = lane; i < nvec; i += G) store16(g, min(i * kPer, last), Vec{});
    } else if (g) {
      int l2 = lane;
      asm volatile("" : "+v"(l2));
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int i = j * G + l2, first = min(i * kPer, last);
        forget(v[j]);
        if (i >= nvec) continue;
        float f[kPer];
        T::unpack(v[j], f);
#pragma unroll
        for (int k = 0; k < kPer; ++k) f[k] = policy_grad(r, f[k]);
        const int at = act - first;
        if (at >= 0 && at < kPer) {
#pragma unroll
          for (int k = 0; k < kPer; ++k) f[k] += k == at ? r.gc : 0.0f;
        }
        store16(g, first, T::pack(f));
      }
    }
    // (behind the gradient: the row's registers are free by then)
    if (lane == 0 && a.loss) wl += row_loss(a, in, st, r, a.weight ? (double)w : a.unit_weight);
  }
  if (!a.loss) return;
  if (G < 256) wl = block_sum<256>(wl, lsum);
  if (threadIdx.x == 0) put_loss(a, wl);
}

// Few actions: a row a lane, in NV vectors of 16 bytes, the last one ending with the row (it may
// repeat elements of the one before; they count once).
template <class T, int NV>
__global__ __launch_bounds__(256, 4) void k_policy_lane(PolicyArgs a) {
  constexpr int kPer = T::kPer;
  using E = typename T::elem;
  __shared__ double lsum[4];
  float scale = 1.0f;
  if (a.grad_scale) {
    scale = *a.grad_scale;
    if (a.skip_unit_scale && scale == 1.0f) return;
  }
  const int V = a.actions, last = V - kPer;  // (last < 0: loaded and stored by elements, NV = 1)
  // Elements that the last vector repeats (the instances are chosen at exact limits: no other does):
  // of two vectors a select each (16 bf16 actions 204 us per 0.6 GB moved, masked words 209), of
  // three masked words in vector registers, the scalar ones being full (12 f32 172 us, selects 177;
  // 24 bf16 185 either way).
  uint32_t keep[4];
  if (NV == 3) {
    last_vector<T>(NV * kPer - V, keep);
    asm volatile("" : "+v"(keep[0]), "+v"(keep[1]), "+v"(keep[2]), "+v"(keep[3]));
  }
  double wl = 0.0;
  for (int64_t row = (int64_t)blockIdx.x * 256 + threadIdx.x; row < a.rows;
       row += (int64_t)gridDim.x * 256) {
    const float w = a.weight ? a.weight[row] : (float)a.unit_weight;
    E* g = a.grad ? (E*)a.grad + row * V : nullptr;
    PolicyRow r;
    r.none = true;
    RowIn in;
    Stats st{-INFINITY, 0.0f, 0.0f};
    Vec v[NV];
    int act = -1;
    if (w != 0.0f) {
      const E* x = row_ptr<E>(a, row);
      if (NV == 1 && last < 0) {
        float f[kPer];
#pragma unroll
        for (int k = 0; k < kPer; ++k) f[k] = k < V ? T::widen(x[k]) : -INFINITY;
        v[0] = T::pack(f);
      } else {
#pragma unroll
        for (int j = 0; j < NV; ++j) v[j] = load16(x + (j * kPer < last ? j * kPer : last));
      }
      in = row_in(a, row, x);
      act = in.action;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        float f[kPer];
        T::unpack(v[j], f);
#pragma unroll
        for (int k = 0; k < kPer; ++k) st.m = fmaxf(st.m, f[k]);
      }
      const float m0 = finite_max(st.m);
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        float f[kPer];
        if (NV > 2) forget(v[j]);
        Vec once = v[j];
        for (int k = 0; NV == 3 && j == 2 && k < 4; ++k)
          once.w[k] = (once.w[k] & keep[k]) | (T::kNegInf & ~keep[k]);
        T::unpack(once, f);
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
          const float d = f[k] - m0;
          float e = exp2_hw(d * kLog2e);
          if (NV == 2 && j == 1 && last + k < kPer) e = 0.0f;
          st.s += e;
          st.t = __builtin_fmaf(e, bound(d), st.t);
        }
      }
      r = policy_row(a, in, st, w * scale);
      if (a.logp) a.logp[row] = r.logp, a.entropy[row] = r.ent;
    } else if (a.logp) {
      a.logp[row] = 0.0f, a.entropy[row] = 0.0f;
    }
#pragma unroll
    for (int j = 0; g && j < NV; ++j) {
      const int first = last < 0 ? 0 : j * kPer < last ? j * kPer : last;
      float f[kPer];
      if (NV > 2) forget(v[j]);
      T::unpack(v[j], f);
#pragma unroll
      for (int k = 0; k < kPer; ++k)
        f[k] = r.none ? 0.0f : policy_grad(r, f[k]) + (first + k == act ? r.gc : 0.0f);
      if (NV == 1 && last < 0) {
#pragma unroll
        for (int k = 0; k < kPer; ++k)
          if (k < V) g[k] = T::narrow(f[k]);
      } else {
        store16(g + first, T::pack(f));
      }
    }
    if (a.loss && w != 0.0f)
      wl += row_loss(a, in, st, r, a.weight ? (double)w : a.unit_weight);
  }
  if (!a.loss) return;
  wl = block_sum<256>(wl, lsum);
  if (threadIdx.x == 0) put_loss(a, wl);
}

// Rows beyond the registers, or too few of them for the chip: S workgroups a row, each with a
// stretch of `chunk` actions (a multiple of the vector). The first launch forms every stretch's
// statistics; the second joins a row's and writes its outputs and its gradient, the logits read
// again (from the cache, for few rows).
constexpr int kSplitVecs = 4;  // vectors a lane has in flight

template <class T>
__global__ __launch_bounds__(256) void k_policy_part(PolicyArgs a, int S, int64_t chunk,
                                                     Stats* out) {
  constexpr int kPer = T::kPer, NV = kSplitVecs;
  using E = typename T::elem;
  __shared__ Stats part[4];
  if (a.skip_unit_scale && *a.grad_scale == 1.0f) return;
  const int64_t row = blockIdx.x / S;
  if (a.weight && a.weight[row] == 0.0f) return;
  const int64_t begin = (blockIdx.x % S) * chunk;
  const int64_t end = begin + chunk < a.actions ? begin + chunk : a.actions;
  const E* x = row_ptr<E>(a, row);
  const int64_t tail = end - (end - begin) % kPer;  // the row's end, shorter than a vector
  Stats st{-INFINITY, 0.0f, 0.0f};
  for (int64_t i = begin + threadIdx.x * kPer; i < tail; i += NV * 256 * kPer) {
    Vec v[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int64_t at = i + j * 256 * kPer;
      v[j] = load16(x + (at < tail ? at : begin));
    }
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (i + j * 256 * kPer >= tail) v[j] = Vec{T::kNegInf, T::kNegInf, T::kNegInf, T::kNegInf};
    Stats n{-INFINITY, 0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      float f[kPer];
      T::unpack(v[j], f);
#pragma unroll
      for (int k = 0; k < kPer; ++k) n.m = fmaxf(n.m, f[k]);
    }
    const float m0 = finite_max(n.m);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      float f[kPer];
      T::unpack(v[j], f);
#pragma unroll
      for (int k = 0; k < kPer; ++k) {
        const float d = f[k] - m0, e = exp2_hw(d * kLog2e);
        n.s += e;
        n.t = __builtin_fmaf(e, bound(d), n.t);
      }
    }
    st = join(st, n);
  }
  if (tail + threadIdx.x < end) add(st, T::widen(x[tail + threadIdx.x]));
  st = lanes_join<64>(st);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = st;
  __syncthreads();
  if (threadIdx.x == 0)
    out[blockIdx.x] = join(join(part[0], part[1]), join(part[2], part[3]));
}

// parts: S of the row's statistics; G workgroups a row (S of them write the gradient, or one).
template <class T>
__global__ __launch_bounds__(256) void k_policy_join(PolicyArgs a, int S, int G, int64_t chunk,
                                                     const Stats* parts) {
  constexpr int kPer = T::kPer;
  using E = typename T::elem;
  __shared__ Stats part[4];
  float scale = 1.0f;
  if (a.grad_scale) {
    scale = *a.grad_scale;
    if (a.skip_unit_scale && scale == 1.0f) return;
  }
  // from the end: what the launch before read last is still in the memory-side cache
  const int block = gridDim.x - 1 - blockIdx.x;
  const int64_t row = block / G;
  const int piece = block % G, tid = threadIdx.x, V = a.actions;
  const int64_t begin = piece * chunk;
  const int64_t end = begin + chunk < V ? begin + chunk : V;
  const int64_t tail = end - (end - begin) % kPer;
  const float w = a.weight ? a.weight[row] : (float)a.unit_weight;
  E* __restrict__ g = a.grad ? (E*)a.grad + row * V : nullptr;
  const E* __restrict__ x = row_ptr<E>(a, row);
  PolicyRow r;
  r.none = true;
  r.logp = r.ent = 0.0f;
  double wl = 0.0;
  int64_t act = -1;
  if (w != 0.0f) {
    const RowIn in = row_in(a, row, x);
    act = in.action;
    Stats st{-INFINITY, 0.0f, 0.0f};
    for (int i = tid; i < S; i += 256) st = join(st, parts[row * S + i]);
    st = lanes_join<64>(st);
    if ((tid & 63) == 0) part[tid >> 6] = st;
    __syncthreads();
    st = join(join(part[0], part[1]), join(part[2], part[3]));
    r = policy_row(a, in, st, w * scale);
    if (a.loss) wl = row_loss(a, in, st, r, a.weight ? (double)w : a.unit_weight);
  }
  if (piece == 0 && tid == 0) {
    if (a.logp) a.logp[row] = r.logp, a.entropy[row] = r.ent;
    if (a.loss) {
      if (a.rows == 1) *a.loss = (float)wl;
      else a.part[row] = wl;
    }
  }
  if (!g) return;
  if (r.none) {
    for (int64_t i = begin + tid * kPer; i < tail; i += 256 * kPer) store16(g + i, Vec{});
    if (tail + tid < end) g[tail + tid] = T::narrow(0.0f);
    return;
  }
  for (int64_t i0 = begin + tid * kPer; i0 < tail; i0 += kSplitVecs * 256 * kPer) {
    Vec v[kSplitVecs];
#pragma unroll
    for (int j = 0; j < kSplitVecs; ++j) {
      const int64_t i = i0 + j * 256 * kPer;
      v[j] = load16(x + (i < tail ? i : begin));
    }
#pragma unroll
    for (int j = 0; j < kSplitVecs; ++j) {
      const int64_t i = i0 + j * 256 * kPer;
      if (i >= tail) break;
      float f[kPer];
      T::unpack(v[j], f);
#pragma unroll
      for (int k = 0; k < kPer; ++k) f[k] = policy_grad(r, f[k]);
      const int64_t at = act - i;
      if (at >= 0 && at < kPer) {
#pragma unroll
        for (int k = 0; k < kPer; ++k) f[k] += k == at ? r.gc : 0.0f;
      }
      store16(g + i, T::pack(f));
    }
  }
  if (tail + tid < end) {
    const int64_t i = tail + tid;
    g[i] = T::narrow(policy_grad(r, T::widen(x[i])) + (i == act ? r.gc : 0.0f));
  }
}

// A lane's share of n numbers; a batch of loads at once.
template <int kBlock>
__device__ inline double strided_sum(const double* part, int n) {
  constexpr int kBatch = kBlock == 1024 ? 16 : 4;
  double v = 0.0;
  for (int i = threadIdx.x; i < n; i += kBatch * kBlock) {
    double p[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) p[j] = part[i + j * kBlock < n ? i + j * kBlock : i];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) v += i + j * kBlock < n ? p[j] : 0.0;
  }
  return v;
}

__global__ __launch_bounds__(1024) void k_sum_loss(const double* part, int n, float* loss) {
  __shared__ double lds[16];
  const double v = block_sum<1024>(strided_sum<1024>(part, n), lds);
  if (threadIdx.x == 0) *loss = (float)v;
}

// --------------------------------------------------------------------------------------
// advantages
// --------------------------------------------------------------------------------------
// A_t = delta_t + c_t A_{t+1} is a map of what comes behind it, and maps compose: a stretch of
// steps is (b, p) with A = b + p (what comes behind the stretch). p = 0 only where a step of the
// stretch is cut (what lies behind must not reach it, were it NaN); elsewhere it stays a normal
// number.
struct Trace {
  float b, p;
};
__device__ inline float after(const Trace& x, float behind) {
  return x.p == 0.0f ? x.b : __builtin_fmaf(x.p, behind, x.b);
}
__device__ inline Trace compose(const Trace& first, const Trace& behind) {
  if (first.p == 0.0f) return first;
  const float p = first.p * behind.p;
  return Trace{__builtin_fmaf(first.p, behind.b, first.b),
               behind.p == 0.0f ? 0.0f : fmaxf(p, 1.17549435e-38f)};
}

constexpr int kAdvSteps = 8;  // steps of a lane, in registers

enum AdvPart { kAdvWhole, kAdvTrace, kAdvJoin };

// A workgroup has CX columns and walks their steps from the last in tiles of CY lanes x 8 steps:
// each lane reads its steps, forms their trace, a scan over the column's lanes brings what lies
// behind each, and the lane walks its steps again from there. Long rollouts of few columns are cut
// into `segs` segments of `seg` steps (whole tiles): kAdvTrace forms every segment's trace (but the
// first steps', which none needs), kAdvJoin starts each segment from those behind it.
template <class T, int CX, int CY, AdvPart kPart>
__global__ __launch_bounds__(CX * CY) void k_advantages(mev_advantages a, int segs, int64_t seg,
                                                        Trace* traces) {
  constexpr int K = kAdvSteps;
  using E = typename T::elem;
  __shared__ Trace scan[2][CY][CX];
  const int tx = threadIdx.x % CX, ty = threadIdx.x / CX;
  const int64_t cols = a.E * a.U;
  // (an uncut rollout may need a second axis of the grid; a cut one has at most 1,024 workgroups)
  const int64_t block = kPart == kAdvWhole ? (int64_t)blockIdx.y * gridDim.x + blockIdx.x
                                           : blockIdx.x / segs;
  const int64_t col = block * CX + tx;
  const int piece = kPart == kAdvWhole ? 0 : blockIdx.x % segs;  // 0: the last steps
  // (returned from, not left out of the grid: a segment's workgroup of the join then has the number
  // of its trace's, and so its L2: 2,000 steps of 1,000 columns 14.6 us, 16.4 numbered anew)
  if (kPart == kAdvTrace && piece == segs - 1) return;
  const int64_t c = col < cols ? col : cols - 1;
  const int64_t e = a.U == 1 ? c : c / a.U, u = a.U == 1 ? 0 : c % a.U;
  const float* r = a.reward + e * a.reward_stride[1] + u * a.reward_stride[2];
  const E* v = (const E*)a.value + e * a.value_stride[1] + u * a.value_stride[2];
  const E* last = (const E*)a.last_value + e * a.last_stride[0] + u * a.last_stride[1];
  const uint8_t* done = a.done + e * a.done_stride[1];
  const float gl = a.gamma * a.lam;
  int64_t hi = a.T - piece * seg;
  const int64_t lo = kPart == kAdvWhole || hi < seg ? 0 : hi - seg;
  float behind = 0.0f;            // what the steps before `hi` see
  Trace whole{0.0f, 1.0f};        // kAdvTrace: the segment's
  if (kPart == kAdvJoin)
    for (int i = 0; i < piece; i += 8) {
      Trace q[8];  // (at once: one wait a batch)
#pragma unroll
      for (int k = 0; k < 8; ++k) q[k] = traces[(i + k < piece ? i + k : i) * cols + c];
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (i + k < piece) behind = after(q[k], behind);
    }
  for (; hi > lo; hi -= CY * K) {
    // the lane's steps: t0 and those before it, `count` of them in the segment; pointers walk back
    // with them and stay on the last (clamped: no branch around a load, no product for an address)
    const int64_t left = hi - lo - ty * K;
    const int count = left < K ? (int)left : K;
    const int64_t t0 = count > 0 ? hi - 1 - ty * K : lo;
    const float* pr = r + t0 * a.reward_stride[0];
    const E* pv = v + t0 * a.value_stride[0];
    const uint8_t* pd = done + t0 * a.done_stride[0];
    float rew[K], val[K];
    uint8_t end[K];
    float next = T::widen(*(t0 + 1 < a.T ? pv + a.value_stride[0] : last));
#pragma unroll
    for (int k = 0; k < K; ++k) {
      rew[k] = *pr;
      val[k] = T::widen(*pv);
      end[k] = *pd;
      const bool more = k + 1 < count;
      pr -= more ? a.reward_stride[0] : 0;
      pv -= more ? a.value_stride[0] : 0;
      pd -= more ? a.done_stride[0] : 0;
    }
    Trace x{0.0f, 1.0f};
#pragma unroll
    for (int k = 0; k < K; ++k) {  // rew becomes delta
      const bool cut = end[k] != 0;
      const float boot = cut && !a.bootstrap_done ? 0.0f : a.gamma * next;
      rew[k] = rew[k] + boot - val[k];
      next = val[k];
      if (k < count) x = compose(Trace{rew[k], cut ? 0.0f : gl}, x);
    }
    float from = behind;
    if (CY > 1) {
      int f = 0;
#pragma unroll
      for (int o = 1; o < CY; o <<= 1, f ^= 1) {
        scan[f][ty][tx] = x;
        __syncthreads();
        if (ty >= o) x = compose(x, scan[f][ty - o][tx]);
      }
      scan[f][ty][tx] = x;  // the trace of this lane's steps and all behind them in the tile
      __syncthreads();
      if (ty > 0) from = after(scan[f][ty - 1][tx], behind);
      x = scan[f][CY - 1][tx];
      __syncthreads();
    }
    if (kPart == kAdvTrace) {
      whole = compose(x, whole);
      continue;
    }
    behind = after(x, behind);
    if (col >= cols) continue;
    // nontemporal, so that they leave the reads their cache: 20 x 65,536 5.5 us (plain stores 6.4),
    // 100 x 30,000 9.8 (11.6), 20 x 32,768 x 30 97 (101)
    float* pa = a.advantage + t0 * cols + col;
    float* pq = a.returns + t0 * cols + col;
#pragma unroll
    for (int k = 0; k < K; ++k, pa -= cols, pq -= cols) {
      if (k >= count) break;
      from = end[k] || gl == 0.0f ? rew[k] : __builtin_fmaf(gl, from, rew[k]);
      __builtin_nontemporal_store(from, pa);
      __builtin_nontemporal_store(from + val[k], pq);
    }
  }
  if (kPart == kAdvTrace && ty == 0 && col < cols) traces[piece * cols + col] = whole;
}

// --------------------------------------------------------------------------------------
// global norm and clipping
// --------------------------------------------------------------------------------------
constexpr int kClipVecs = 4;  // vectors a lane has in flight
constexpr int kClipBatch = 128;  // tensors of one launch (their table travels with the launch)
struct ClipBatch {
  const void* src[kClipBatch];
  void* dst[kClipBatch];
  int64_t numel[kClipBatch];
  int32_t first[kClipBatch + 1];  // first workgroup of each tensor
  uint8_t dtype[kClipBatch];
  int32_t count;
  int64_t chunk;
};

struct ClipPiece {
  int i;
  int64_t begin, end;
};
__device__ inline ClipPiece clip_piece(const ClipBatch& b, int block) {
  int lo = 0, hi = b.count;  // last tensor whose first workgroup is not behind this one
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (b.first[mid] <= block) lo = mid;
    else hi = mid;
  }
  const int64_t begin = (int64_t)(block - b.first[lo]) * b.chunk;
  const int64_t end = begin + b.chunk;
  return ClipPiece{lo, begin, end < b.numel[lo] ? end : b.numel[lo]};
}

template <class T>
__device__ double square_sum(const void* p, int64_t begin, int64_t end) {
  constexpr int kPer = T::kPer;
  const typename T::elem* x = (const typename T::elem*)p;
  const int64_t tail = end - (end - begin) % kPer;
  double s[4] = {0.0, 0.0, 0.0, 0.0};
  for (int64_t i0 = begin + threadIdx.x * kPer; i0 < tail; i0 += kClipVecs * 256 * kPer) {
    Vec r[kClipVecs];
#pragma unroll
    for (int j = 0; j < kClipVecs; ++j) {
      const int64_t i = i0 + j * 256 * kPer;
      r[j] = load16(x + (i < tail ? i : begin));
    }
#pragma unroll
    for (int j = 0; j < kClipVecs; ++j) {
      if (i0 + j * 256 * kPer >= tail) break;
      float f[kPer];
      T::unpack(r[j], f);
#pragma unroll
      for (int k = 0; k < kPer; ++k)
        s[k & 3] = __builtin_fma((double)f[k], (double)f[k], s[k & 3]);
    }
  }
  if (tail + threadIdx.x < end) {
    const double v = T::widen(x[tail + threadIdx.x]);
    s[0] = __builtin_fma(v, v, s[0]);
  }
  return (s[0] + s[1]) + (s[2] + s[3]);
}

__global__ __launch_bounds__(256) void k_clip_squares(ClipBatch b, double* part) {
  __shared__ double lds[4];
  const ClipPiece c = clip_piece(b, blockIdx.x);
  const void* p = b.src[c.i];
  double s = b.dtype[c.i] == MEV_F32    ? square_sum<F32>(p, c.begin, c.end)
             : b.dtype[c.i] == MEV_BF16 ? square_sum<BF16>(p, c.begin, c.end)
                                        : square_sum<F16>(p, c.begin, c.end);
  s = block_sum<256>(s, lds);
  if (threadIdx.x == 0) part[blockIdx.x] = s;
}

// The norm from the sum of squares, and what the gradients are multiplied by.
__device__ inline double clip_factor(double squares, float max_norm, float* norm) {
  const double v = sqrt(squares);
  const float f = (float)v;
  if (norm) *norm = f;
  return v > (double)max_norm && f < INFINITY ? (double)max_norm / v : 1.0;
}

// norm and factor from the n partial sums, the factor to part[n]
__global__ __launch_bounds__(1024) void k_clip_norm(double* part, int n, float max_norm,
                                                    float* norm) {
  __shared__ double lds[16];
  const double s = block_sum<1024>(strided_sum<1024>(part, n), lds);
  if (threadIdx.x == 0) part[n] = clip_factor(s, max_norm, norm);
}

// times f, then times rest
template <class T>
__device__ void scale_to(const void* src, void* dst, int64_t begin, int64_t end, float f,
                         float rest) {
  constexpr int kPer = T::kPer;
  const typename T::elem* x = (const typename T::elem*)src;
  typename T::elem* y = (typename T::elem*)dst;
  const int64_t tail = end - (end - begin) % kPer;
  for (int64_t i0 = begin + threadIdx.x * kPer; i0 < tail; i0 += kClipVecs * 256 * kPer) {
    Vec r[kClipVecs];  // (a batch of loads before its stores: dst may be src)
#pragma unroll
    for (int j = 0; j < kClipVecs; ++j) {
      const int64_t i = i0 + j * 256 * kPer;
      r[j] = load16(x + (i < tail ? i : i0));
    }
#pragma unroll
    for (int j = 0; j < kClipVecs; ++j) {
      const int64_t i = i0 + j * 256 * kPer;
      if (i >= tail) break;
      float v[kPer];
      T::unpack(r[j], v);
#pragma unroll
      for (int k = 0; k < kPer; ++k) v[k] = v[k] * f * rest;
      store16(y + i, T::pack(v));
    }
  }
  if (tail + threadIdx.x < end)
    y[tail + threadIdx.x] = T::narrow(T::widen(x[tail + threadIdx.x]) * f * rest);
}

// n > 0: the factor is still in the n partial sums, and every workgroup forms it (one writes the
// norm); n = 0: it lies at part[0].
__global__ __launch_bounds__(256) void k_clip_scale(ClipBatch b, const double* part, int n,
                                                    float max_norm, float* norm) {
  __shared__ double lds[4];
  // from the end: what the pass before read last is still in the memory-side cache
  const ClipPiece c = clip_piece(b, gridDim.x - 1 - blockIdx.x);
  double factor = n > 0 ? block_sum<256>(strided_sum<256>(part, n), lds) : *part;
  if (n > 0)
    factor = clip_factor(factor, max_norm, blockIdx.x + threadIdx.x == 0 ? norm : nullptr);
  // a factor below float32's normal numbers (gradients of 1e30 clipped to 1e-10) keeps its digits
  const bool tiny = factor < 0x1p-126;
  const float f = (float)(tiny ? factor * 0x1p100 : factor), rest = tiny ? 0x1p-100f : 1.0f;
  const void* s = b.src[c.i];
  void* d = b.dst[c.i];
  if (f == 1.0f && s == d) return;
  if (b.dtype[c.i] == MEV_F32) scale_to<F32>(s, d, c.begin, c.end, f, rest);
  else if (b.dtype[c.i] == MEV_BF16) scale_to<BF16>(s, d, c.begin, c.end, f, rest);
  else scale_to<F16>(s, d, c.begin, c.end, f, rest);
}

}  // namespace

// --------------------------------------------------------------------------------------
// C ABI
// --------------------------------------------------------------------------------------
// Workgroups of so many lanes along one axis of a grid: fewer than 2^32 lanes.
static constexpr int64_t grid_max(int lanes) { return UINT32_MAX / lanes; }

static bool dtype_ok(int32_t d) { return d == MEV_F32 || d == MEV_BF16 || d == MEV_F16; }

// How a call is launched. One launch of `kernel` (rows a workgroup each, or several), or two of
// `part` and `join` where split > 0 (workgroups a row, `chunk` actions each).
struct PolicyPlan {
  void (*kernel)(PolicyArgs) = nullptr;
  void (*part)(PolicyArgs, int, int64_t, Stats*) = nullptr;
  void (*join)(PolicyArgs, int, int, int64_t, const Stats*) = nullptr;
  int block = 256, rows_per_block = 1;
  int64_t grid = 0;   // workgroups of `kernel`: at most 16,384, a partial loss each
  int64_t split = 0, chunk = 0;
  int64_t losses = 0;                       // partial losses
};

template <class T, int NV>
static bool plan_lane(PolicyPlan* p, int V) {
  if (V > T::kPer * NV) return false;
  p->kernel = k_policy_lane<T, NV>;
  p->rows_per_block = 256;
  return true;
}

template <class T, int G, int NV>
static bool plan_regs(PolicyPlan* p, int V) {
  if (V > G * NV * T::kPer) return false;
  p->kernel = k_policy_regs<T, G, NV>;
  p->block = G < 256 ? 256 : G;
  p->rows_per_block = p->block / G;
  return true;
}

template <class T>
static PolicyPlan plan_policy(const mev_policy* a) {
  PolicyPlan p;
  const int V = a->actions;
  // Rows of 1,024 lanes, too few for the chip: split though they fit the registers, up to 160 in
  // 16 bits, 80 in f32, at any length. 32 rows of 84,000 bf16 12.3 us with their gradient (one
  // workgroup each 19.7), 160 23.1 (23.9), 200 26.2 (25.2); 32 of 49,000 f32 11.8 us (13.5), 80
  // 16.0 (15.4), 200 26.1 (20.6).
  const bool few = a->rows <= 20 * T::kPer;
  // 512 lanes while two workgroups fit a unit, one loading while the other computes (60,000 bf16
  // 133 us per 0.6 GB moved; 1,024 lanes of 8 vectors fill the unit alone, 168 us). Those for
  // longer rows (100,000 161 us, split 217 us), as far as 128 registers a lane hold them.
  // The fewest lanes that hold a row in 8 vectors each: what is done once a row (its scalars, the
  // joins) is done for as many rows at a time as a wavefront holds. Per 0.6 GB moved, 300 bf16
  // actions 133 us in 8 lanes of 5 vectors (16 of 3: 165 us), 64 158 us in 4 of 2 (8 of 1: 232 us),
  // 256 in 4 of 8 123 us; 32 of them 165 us in 2 of 2, one lane 183 us. A lane alone up to 24 bf16
  // actions (24: 182 us, 2 of 2 196 us; 16: 195 us, 2 of 1 221 us).
  if (plan_lane<T, 1>(&p, V) || plan_lane<T, 2>(&p, V) || plan_lane<T, 3>(&p, V) ||
      plan_regs<T, 2, 2>(&p, V) || plan_regs<T, 2, 3>(&p, V) ||
      plan_regs<T, 4, 2>(&p, V) || plan_regs<T, 4, 3>(&p, V) || plan_regs<T, 4, 4>(&p, V) ||
      plan_regs<T, 4, 5>(&p, V) || plan_regs<T, 4, 6>(&p, V) || plan_regs<T, 4, 7>(&p, V) ||
      plan_regs<T, 4, 8>(&p, V) || plan_regs<T, 8, 5>(&p, V) || plan_regs<T, 8, 6>(&p, V) ||
      plan_regs<T, 8, 7>(&p, V) || plan_regs<T, 8, 8>(&p, V) || plan_regs<T, 16, 5>(&p, V) ||
      plan_regs<T, 16, 6>(&p, V) || plan_regs<T, 16, 7>(&p, V) || plan_regs<T, 16, 8>(&p, V) ||
      plan_regs<T, 32, 5>(&p, V) || plan_regs<T, 32, 6>(&p, V) || plan_regs<T, 32, 7>(&p, V) ||
      plan_regs<T, 32, 8>(&p, V) || plan_regs<T, 64, 5>(&p, V) || plan_regs<T, 64, 6>(&p, V) ||
      plan_regs<T, 64, 7>(&p, V) || plan_regs<T, 64, 8>(&p, V) ||
      plan_regs<T, 256, 4>(&p, V) || plan_regs<T, 256, 6>(&p, V) ||
      plan_regs<T, 256, 8>(&p, V) || plan_regs<T, 512, 6>(&p, V) ||
      plan_regs<T, 512, 8>(&p, V) || plan_regs<T, 512, 10>(&p, V) ||
      plan_regs<T, 512, 12>(&p, V) || plan_regs<T, 512, 14>(&p, V) ||
      plan_regs<T, 512, 16>(&p, V) || (!few && (plan_regs<T, 1024, 12>(&p, V) ||
      plan_regs<T, 1024, 14>(&p, V) || plan_regs<T, 1024, 16>(&p, V)))) {
    p.grid = (a->rows + p.rows_per_block - 1) / p.rows_per_block;
    if (p.grid > 16384) p.grid = 16384;
    p.losses = p.grid;
    return p;
  }
  p.part = k_policy_part<T>;
  p.join = k_policy_join<T>;
  // about 2,048 workgroups, each with one round of its lanes' vectors or more
  constexpr int64_t round = 256 * T::kPer * kSplitVecs;
  const int64_t rounds = (V + round - 1) / round, rows = a->rows > 0 ? a->rows : 1;
  int64_t each = (rounds * rows + 2047) / 2048;
  if (each > rounds) each = rounds;
  p.chunk = each * round;
  p.split = (V + p.chunk - 1) / p.chunk;
  p.losses = a->rows;
  return p;
}

static PolicyPlan policy_plan(const mev_policy* a) {
  return a->dtype == MEV_F32    ? plan_policy<F32>(a)
         : a->dtype == MEV_BF16 ? plan_policy<BF16>(a)
                                : plan_policy<F16>(a);
}

static int64_t loss_bytes(const mev_policy* a, const PolicyPlan& p) {
  return a->loss && p.losses > 1 ? (8 * p.losses + 15) / 16 * 16 : 0;
}

int64_t mev_policy_workspace(const mev_policy* a) {
  if (!a || a->rows < 0 || a->rows > int64_t(1) << 40 || a->actions < 1 || !dtype_ok(a->dtype))
    return MEV_EINVAL;
  const PolicyPlan p = policy_plan(a);
  return loss_bytes(a, p) + a->rows * p.split * (int64_t)sizeof(Stats);
}

int mev_policy_rows(const mev_policy* a, void* stream) {
  const int64_t need = mev_policy_workspace(a);
  if (need < 0) return MEV_EINVAL;
  if (a->rows > 0 && (!a->logits || !a->action || a->inner < 1)) return MEV_EINVAL;
  if (a->action_bytes != 4 && a->action_bytes != 8) return MEV_EINVAL;
  if (!a->logp != !a->entropy || !a->old_logp != !a->advantage) return MEV_EINVAL;
  if ((a->loss || a->grad) && a->rows > 0 && !a->old_logp) return MEV_EINVAL;
  if (a->skip_unit_scale && (a->loss || a->logp || !a->grad_scale)) return MEV_EINVAL;
  if (need > 0 && (!a->workspace || a->workspace_bytes < need)) return MEV_EINVAL;
  hipStream_t st = (hipStream_t)stream;
  const PolicyPlan p = policy_plan(a);
  PolicyArgs k{};
  k.logits = a->logits;
  k.action = a->action;
  k.old_logp = a->old_logp;
  k.advantage = a->advantage;
  k.weight = a->weight;
  k.ref_logp = a->kl_coef != 0.0 ? a->ref_logp : nullptr;
  k.logp = a->logp;
  k.entropy = a->entropy;
  k.part = (double*)a->workspace;
  k.loss = a->loss;
  k.grad = a->grad;
  k.grad_scale = a->grad_scale;
  k.rows = a->rows;
  k.inner = a->inner;
  k.outer_stride = a->outer_stride;
  k.inner_stride = a->inner_stride;
  k.actions = a->actions;
  k.action_bytes = a->action_bytes;
  k.skip_unit_scale = a->skip_unit_scale;
  k.unit_weight = a->rows > 0 ? 1.0 / (double)a->rows : 0.0;
  k.clip_lo = 1.0 - a->clip_low;
  k.clip_hi = 1.0 + a->clip_high;
  k.above = (float)k.clip_hi;
  if ((double)k.above > k.clip_hi) k.above = nextafterf(k.above, -INFINITY);
  k.below = (float)k.clip_lo;
  if ((double)k.below < k.clip_lo) k.below = nextafterf(k.below, INFINITY);
  k.kl = a->kl_coef;
  k.ent = a->entropy_coef;
  if (a->rows > 0 && (a->logp || a->loss || a->grad)) {
    if (p.kernel) {
      // a launch that most likely finds nothing to do: no more workgroups than the chip holds
      // (10,240 of them that return at once take 5.5 us)
      const int64_t few = (1 << 18) / p.block;
      const int64_t grid = a->skip_unit_scale && p.grid > few ? few : p.grid;
      hipLaunchKernelGGL(p.kernel, dim3((unsigned)grid), dim3(p.block), 0, st, k);
      MEV_HIP(hipGetLastError());
    } else {
      Stats* parts = (Stats*)((char*)a->workspace + loss_bytes(a, p));
      const int64_t pieces = a->grad ? p.split : 1;
      if (a->rows > grid_max(256) / p.split) return MEV_EINVAL;
      hipLaunchKernelGGL(p.part, dim3((unsigned)(a->rows * p.split)), dim3(256), 0, st, k,
                         (int)p.split, p.chunk, parts);
      MEV_HIP(hipGetLastError());
      hipLaunchKernelGGL(p.join, dim3((unsigned)(a->rows * pieces)), dim3(256), 0, st, k,
                         (int)p.split, (int)pieces, p.chunk, (const Stats*)parts);
      MEV_HIP(hipGetLastError());
    }
  }
  if (a->loss && p.losses != 1) {  // (no rows: 0)
    hipLaunchKernelGGL(k_sum_loss, dim3(1), dim3(1024), 0, st, (const double*)a->workspace,
                       (int)p.losses, a->loss);
    MEV_HIP(hipGetLastError());
  }
  return MEV_OK;
}

// Columns and lanes a column of a workgroup, and segments of the rollout. 64 columns side by side
// fill the cache lines: from 256 columns on, though 16 would leave fewer lanes idle. A rollout of
// one tile of 256 lanes takes them (four lanes a column also where columns abound: 20 steps of
// 262,144 columns 16.5 us, a lane to itself 32 us), with more columns and fewer lanes to each while
// that is one tile too -- or two that a lane walks, where the columns still make 256 workgroups (16
// steps of 65,536 columns 4.9 us, four lanes a column 5.5; of 32,768 4.9 and 4.4 us). A longer one
// takes 1,024 lanes where that is one tile or the columns are 64 (100 steps of 30,000 columns
// 9.9 us; with plain stores 11.6, 256 lanes 19.7; 3,000 steps of 100 columns the other way, 12.7 and 10.2 us: fewer
// columns read by short stretches, and one unit does all of it). What is longer still is cut into
// segments until 256 large or 1,024 small workgroups share it (20,000 steps of 800 columns 85 us,
// 512 large ones 90 us).
struct AdvPlan {
  int cx, cy;
  int64_t blocks, segs, seg;
};
static AdvPlan adv_plan(const mev_advantages* a) {
  AdvPlan p;
  const int64_t cols = a->E * a->U;
  p.cx = cols >= 256 ? 64 : cols >= 64 ? 16 : cols >= 4 ? 4 : 1;
  int lanes = 256;
  if (a->T > 256 / p.cx * kAdvSteps &&
      (p.cx == 64 || (p.cx > 1 && a->T <= 1024 / p.cx * kAdvSteps)))
    lanes = 1024;
  while (lanes == 256 && p.cx < 256) {
    const int64_t wider = 256 / (4 * p.cx) * kAdvSteps;
    if (wider < a->T && (2 * wider < a->T || cols < int64_t(256) * 4 * p.cx)) break;
    p.cx *= 4;
  }
  p.cy = lanes / p.cx;
  p.blocks = (cols + p.cx - 1) / p.cx;
  const int64_t tile = p.cy * kAdvSteps, tiles = (a->T + tile - 1) / tile;
  int64_t want = (lanes == 1024 ? 256 : 1024) / p.blocks;
  if (want > 64) want = 64;  // (each segment walks the traces behind it)
  if (want < 1 || p.cx == 256) want = 1;  // (256 columns: a tile, or two to be walked)
  const int64_t each = (tiles + want - 1) / want;
  p.seg = each * tile;
  p.segs = (tiles + each - 1) / each;
  return p;
}

static bool adv_ok(const mev_advantages* a) {
  if (!a || a->T < 0 || a->E < 0 || a->U < 0 || !dtype_ok(a->value_dtype)) return false;
  constexpr int64_t kMax = int64_t(1) << 40;
  return a->T <= kMax && a->E <= kMax && a->U <= kMax && (a->U == 0 || a->E <= kMax / a->U);
}

int64_t mev_advantages_workspace(const mev_advantages* a) {
  if (!adv_ok(a)) return MEV_EINVAL;
  if (a->T == 0 || a->E == 0 || a->U == 0) return 0;
  const AdvPlan p = adv_plan(a);
  return (p.segs - 1) * a->E * a->U * (int64_t)sizeof(Trace);
}

template <class T, int CX, int CY>
static void launch_columns(const mev_advantages& a, const AdvPlan& p, hipStream_t st) {
  const dim3 b(CX * CY);
  Trace* t = (Trace*)a.workspace;
  if (p.segs == 1) {
    const int64_t y = (p.blocks - 1) / grid_max(CX * CY) + 1, x = (p.blocks - 1) / y + 1;
    hipLaunchKernelGGL((k_advantages<T, CX, CY, kAdvWhole>), dim3((unsigned)x, (unsigned)y), b, 0,
                       st, a, 1, (int64_t)0, t);
    return;
  }
  const dim3 g((unsigned)(p.blocks * p.segs));
  hipLaunchKernelGGL((k_advantages<T, CX, CY, kAdvTrace>), g, b, 0, st, a, (int)p.segs, p.seg, t);
  hipLaunchKernelGGL((k_advantages<T, CX, CY, kAdvJoin>), g, b, 0, st, a, (int)p.segs, p.seg, t);
}

template <class T>
static void launch_advantages(const mev_advantages& a, const AdvPlan& p, hipStream_t st) {
  const bool large = p.cx * p.cy == 1024;
  switch (p.cx) {
    case 1: launch_columns<T, 1, 256>(a, p, st); break;
    case 4: large ? launch_columns<T, 4, 256>(a, p, st) : launch_columns<T, 4, 64>(a, p, st); break;
    case 16: large ? launch_columns<T, 16, 64>(a, p, st) : launch_columns<T, 16, 16>(a, p, st); break;
    case 64: large ? launch_columns<T, 64, 16>(a, p, st) : launch_columns<T, 64, 4>(a, p, st); break;
    default: launch_columns<T, 256, 1>(a, p, st);
  }
}

int mev_advantages_run(const mev_advantages* a, void* stream) {
  const int64_t need = mev_advantages_workspace(a);
  if (need < 0) return MEV_EINVAL;
  if (a->T == 0 || a->E == 0 || a->U == 0) return MEV_OK;
  if (!a->reward || !a->value || !a->last_value || !a->done || !a->advantage || !a->returns)
    return MEV_EINVAL;
  if (need > 0 && (!a->workspace || a->workspace_bytes < need)) return MEV_EINVAL;
  const AdvPlan p = adv_plan(a);
  hipStream_t st = (hipStream_t)stream;
  if (a->value_dtype == MEV_F32) launch_advantages<F32>(*a, p, st);
  else if (a->value_dtype == MEV_BF16) launch_advantages<BF16>(*a, p, st);
  else launch_advantages<F16>(*a, p, st);
  MEV_HIP(hipGetLastError());
  return MEV_OK;
}

// Elements of one workgroup: about 32,768 workgroups over all tensors, in whole multiples of 4,096
// (400 M elements: 610 us; 2,048 workgroups, each walking 48 rounds, 707 us)
static int64_t clip_chunk(int64_t total) {
  const int64_t c = (total / 32768 + 4095) / 4096 * 4096;
  return c < 4096 ? 4096 : c;
}

// Workgroups over all tensors (negative: bad sizes)
static int64_t clip_blocks(const int64_t* numel, int32_t count, int64_t* chunk) {
  int64_t total = 0, blocks = 0;
  for (int32_t i = 0; i < count; ++i) {
    if (numel[i] < 0 || numel[i] > ((int64_t)1 << 50) - total) return MEV_EINVAL;
    total += numel[i];
  }
  *chunk = clip_chunk(total);
  for (int32_t i = 0; i < count; ++i) blocks += (numel[i] + *chunk - 1) / *chunk;
  return blocks;
}

// Whether two of the buffers that a call reads or writes share memory (in place: src[i] is dst[i]).
static int clip_overlap(const void* const* src, void* const* dst, const int64_t* numel,
                        const int32_t* dtype, int32_t count) {
  try {
    std::vector<std::pair<uintptr_t, uintptr_t>> r;
    r.reserve(2 * (size_t)count);
    for (int32_t i = 0; i < count; ++i) {
      if (numel[i] == 0) continue;
      const uintptr_t n = (uintptr_t)numel[i] * (dtype[i] == MEV_F32 ? 4 : 2);
      const uintptr_t s = (uintptr_t)src[i], d = (uintptr_t)dst[i];
      r.emplace_back(s, s + n);
      if (d != s) r.emplace_back(d, d + n);
    }
    std::sort(r.begin(), r.end());
    for (size_t i = 1; i < r.size(); ++i)
      if (r[i].first < r[i - 1].second) return MEV_EINVAL;
    return MEV_OK;
  } catch (const std::bad_alloc&) {
    return MEV_ENOMEM;
  }
}

int64_t mev_clip_norm_workspace(const int64_t* numel, int32_t count) {
  if (count < 0 || (count > 0 && !numel)) return MEV_EINVAL;
  int64_t chunk;
  const int64_t blocks = clip_blocks(numel, count, &chunk);
  return blocks < 0 ? MEV_EINVAL : 8 * (blocks + 1);
}

int mev_clip_norm(const void* const* src, void* const* dst, const int64_t* numel,
                  const int32_t* dtype, int32_t count, float max_norm, float* norm,
                  void* workspace, int64_t workspace_bytes, void* stream) {
  const int64_t need = mev_clip_norm_workspace(numel, count);
  if (need < 0 || !norm || !workspace || workspace_bytes < need) return MEV_EINVAL;
  if (!(max_norm >= 0.0f) || max_norm == INFINITY) return MEV_EINVAL;
  if (count > 0 && (!src || !dst || !dtype)) return MEV_EINVAL;
  for (int32_t i = 0; i < count; ++i)
    if (!dtype_ok(dtype[i]) || (numel[i] > 0 && (!src[i] || !dst[i]))) return MEV_EINVAL;
  const int rc = clip_overlap(src, dst, numel, dtype, count);
  if (rc) return rc;
  hipStream_t st = (hipStream_t)stream;
  int64_t chunk;
  const int64_t blocks = clip_blocks(numel, count, &chunk);
  double* part = (double*)workspace;
  // up to 1,024 partial sums are joined by every workgroup that scales: a launch less (4 of
  // 15 us for eight small gradients)
  const bool joined = blocks > 0 && blocks <= 1024;
  for (int pass = 0; pass < 2; ++pass) {
    int64_t done = 0;
    for (int32_t i = 0; i < count;) {
      ClipBatch b;
      b.count = 0;
      b.chunk = chunk;
      b.first[0] = 0;
      for (; i < count && b.count < kClipBatch; ++i) {
        if (numel[i] == 0) continue;
        const int k = b.count++;
        b.src[k] = src[i];
        b.dst[k] = dst[i];
        b.numel[k] = numel[i];
        b.dtype[k] = (uint8_t)dtype[i];
        b.first[k + 1] = b.first[k] + (int32_t)((numel[i] + chunk - 1) / chunk);
      }
      const int n = b.first[b.count];
      if (n == 0) continue;
      if (pass == 0)
        hipLaunchKernelGGL(k_clip_squares, dim3(n), dim3(256), 0, st, b, part + done);
      else
        hipLaunchKernelGGL(k_clip_scale, dim3(n), dim3(256), 0, st, b,
                           (const double*)(joined ? part : part + blocks),
                           joined ? (int)blocks : 0, max_norm, norm);
      MEV_HIP(hipGetLastError());
      done += n;
    }
    if (pass == 0 && !joined) {
      hipLaunchKernelGGL(k_clip_norm, dim3(1), dim3(1024), 0, st, part, (int)blocks, max_norm,
                         norm);
      MEV_HIP(hipGetLastError());
    }
  }
  return MEV_OK;
}
