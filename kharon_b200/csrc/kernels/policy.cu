// Losses of a policy on the head's logits, with their gradients: the clipped policy loss with a KL term (one row at a time) and the preference
// loss (pairs of sequences of whole rows).  bf16 logits [rows, ld], V of them a vocabulary; rows without a target are masked: loss 0, a gradient of
// zeros, and they are not read.
//
// Of a row x with target t, m = max x:  R = sum_{j != t} exp(x_j - m) and e_t = exp(x_t - m) are kept apart, so that 1 - p_t = R / (R + e_t) and, where
// the target is the largest, log p_t = -log(1 + R) keep their relative precision for a policy that is nearly certain.  With slope = dloss / dlog p_t the
// gradient is  dx_j = -slope exp(x_j - m) / (R + e_t)  and  dx_t = slope R / (R + e_t),  rounded once to bf16.
#include <algorithm>

#include "common.cuh"

#define KH_LAUNCH_CHECK(name)                                                     \
  do {                                                                            \
    cudaError_t e_ = cudaGetLastError();                                          \
    if (e_ != cudaSuccess) { kh_set_error(name ": %s", cudaGetErrorString(e_)); return -1; } \
  } while (0)

namespace {

constexpr uint32_t NEG2 = 0xff80ff80u;       // a pair of -inf
constexpr int TWICE = 2304, ONCE = 4096;     // columns up to which a warp takes a row; without a gradient, where there are not rows enough for the stream
constexpr int ROW_SMEM = 222 * 1024;         // shared memory of two places for a row (or its share of a cluster), at most
constexpr int ROW_PIECES = ROW_SMEM / 32 - 16;             // pieces of 8 columns in a place (rounded up to a multiple of the warps)

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float warp_max(float v) {                    // a NaN gives way to a number
  float m;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(v));
  return m;
}
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {      // a NaN gives way to a number
  const __nv_bfloat162 m = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&m);
}
// the pieces below are changed by value: an array of them whose elements' addresses are taken ends up in local memory
__device__ __forceinline__ uint32_t cut_word(uint32_t w, int k) { return k <= 0 ? NEG2 : k == 1 ? (w & 0xffffu) | 0xff800000u : w; }
// -inf in the columns k.. of an 8-column piece
__device__ __forceinline__ uint4 cut_from(const uint4& v, int k) { return make_uint4(cut_word(v.x, k), cut_word(v.y, k - 2), cut_word(v.z, k - 4), cut_word(v.w, k - 6)); }
__device__ __forceinline__ uint32_t put_word(uint32_t w, int k, uint32_t b) { return k == 0 ? (w & 0xffff0000u) | b : k == 1 ? (w & 0xffffu) | b << 16 : w; }
// the bits b in column k of it
__device__ __forceinline__ uint4 put_bits(const uint4& v, int k, uint32_t b) {
  return make_uint4(put_word(v.x, k, b), put_word(v.y, k - 2, b), put_word(v.z, k - 4, b), put_word(v.w, k - 6, b));
}
__device__ __forceinline__ uint4 cut_one(const uint4& v, int k) { return put_bits(v, k, 0xff80u); }
__device__ __forceinline__ uint4 put_one(const uint4& v, int k, float x) { return put_bits(v, k, pack_bf16(x, 0.f) & 0xffffu); }
__device__ __forceinline__ float ex2(float x) {                         // 2^x to 2^-22 of itself; results below 2^-126 are 0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Exponentials relative to one of a row's values m: exp(x - m) is taken as 2^(x a + b) in one fused step, with a = log2 e and b = -m log2 e rounded to a whole number less BELOW, so
// that it loses nothing, and another m is another power of two.  Beyond 2^20 values of bf16 lie 4096 and more apart, and any base will do: 2^(x - m).
constexpr float LOG2E = 1.44269504f, BELOW = 3.f;
struct Scale {
  float a, b;
};
__device__ __forceinline__ bool is_far(float m) { return !(fabsf(m) < 1048576.f); }
__device__ __forceinline__ Scale scale_of(float m) {
  if (is_far(m)) return m == -INFINITY ? Scale{LOG2E, 0.f} : Scale{1.f, -m};      // (nothing but -inf: terms of 0)
  return {LOG2E, -rintf(m * LOG2E) - BELOW};
}
// what a sum relative to m is to be multiplied by to be one relative to top >= m
__device__ __forceinline__ float onto(float m, float top) {
  return m == top ? 1.f : is_far(m) || is_far(top) ? 0.f : ex2(rintf(m * LOG2E) - rintf(top * LOG2E));
}
__device__ __forceinline__ f32x2 exp2x2(uint32_t w, f32x2 a, f32x2 b) {
  const f32x2 y = fma2(un2(w), a, b);
  return mk2(ex2(lo2(y)), ex2(hi2(y)));
}
// A warp's running sum of exponentials relative to one of the values, at most SLACK below the largest.
constexpr float SLACK = 1.f;
struct Sum {
  f32x2 s0 = 0, s1 = 0;
  float lim = -INFINITY, m = -INFINITY;
  Scale sc = {LOG2E, 0.f};
  __device__ __forceinline__ void see(uint32_t top2) {                      // the largest of the lane's pieces to come (by the whole warp)
    const f32x2 t = un2(top2);
    const float mx = warp_max(fmaxf(lo2(t), hi2(t)));
    if (mx > lim) {
      const float c = onto(m, mx);
      s0 = mul2(s0, mk2(c, c)); s1 = mul2(s1, mk2(c, c));
      m = mx;
      sc = scale_of(mx);
      lim = mx + SLACK;
    }
  }
  __device__ __forceinline__ void add(const uint4& v) {
    const f32x2 a = mk2(sc.a, sc.a), b = mk2(sc.b, sc.b);
    s0 = add2(s0, add2(exp2x2(v.x, a, b), exp2x2(v.y, a, b)));
    s1 = add2(s1, add2(exp2x2(v.z, a, b), exp2x2(v.w, a, b)));
  }
  __device__ __forceinline__ float sum() const { const f32x2 s = add2(s0, s1); return lo2(s) + hi2(s); }
};
__device__ __forceinline__ uint32_t top8(const uint4& v) { return max2(max2(v.x, v.y), max2(v.z, v.w)); }
// What a row's gradient is made of: k exp(x - m), k = -slope / sum.  The size of k is a further term of the exponent where that stays below 96 and so loses less than 2^-17 (of a
// result that is rounded to 2^-8), with f = 0 or -0 for its sign; else f is k, or k 2^-BELOW, and never 0.  Results below 2^-126 are 0 in the first form, exponentials in the second.
constexpr float LEAST = 0x1p-147f;             // k up to that is 0 times 2^-BELOW in fp32, and no bf16 number times an exponential
struct Shape {
  float a, b, f;
};
__device__ __forceinline__ Shape shape_of(float m, float k) {
  const Scale s = scale_of(m);
  if (fabsf(k) <= LEAST) return {s.a, -INFINITY, 0.f};
  const float b = s.b + log2f(fabsf(k));
  if (!is_far(m) && fabsf(b) <= 96.f) return {s.a, b, copysignf(0.f, k)};
  return is_far(m) ? Shape{s.a, s.b, k} : Shape{s.a, s.b + BELOW, k * exp2f(-BELOW)};
}
template <bool FUSED>
__device__ __forceinline__ uint4 grad8(const uint4& v, const Shape& g) {
  const f32x2 a = mk2(g.a, g.a), b = mk2(g.b, g.b), k = mk2(g.f, g.f);
  if (FUSED) {
    const uint32_t sign = __float_as_uint(g.f) >> 16 | __float_as_uint(g.f);
    return make_uint4(pack2(exp2x2(v.x, a, b)) ^ sign, pack2(exp2x2(v.y, a, b)) ^ sign, pack2(exp2x2(v.z, a, b)) ^ sign, pack2(exp2x2(v.w, a, b)) ^ sign);
  }
  return make_uint4(pack2(mul2(exp2x2(v.x, a, b), k)), pack2(mul2(exp2x2(v.y, a, b), k)), pack2(mul2(exp2x2(v.z, a, b), k)), pack2(mul2(exp2x2(v.w, a, b), k)));
}
__device__ __forceinline__ uint4 grad8(const uint4& v, const Shape& g) { return g.f == 0.f ? grad8<true>(v, g) : grad8<false>(v, g); }
// piece i of a gradient row of gcols columns; the last one may be cut
__device__ __forceinline__ void store8(bf16* row, int i, int gcols, const uint4& v) {
  if (8 * i + 8 <= gcols) {
    reinterpret_cast<uint4*>(row)[i] = v;
  } else {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int k = 0; k < 8; k++)
      if (8 * i + k < gcols) reinterpret_cast<unsigned short*>(row)[8 * i + k] = (unsigned short)(w[k >> 1] >> (16 * (k & 1)));
  }
}
// log p_t from the row's parts relative to m: R (the others) and e_t = 2^(x_t a + b); NaN for a row without a finite logit or with an infinite one, as by the formula.  The
// logarithm of the sum f 2^k, f about 1, is k log 2 in 64 bits and log f in 32, which is off by 2^-25 at most where a logarithm of the whole would be off by 2^-21.  The
// exponentials of arguments below -1 (as those of all that matters are, by BELOW) come out low by 5e-8 of themselves on average, which would add up over a sequence's rows.
// And the fp32 log2 e is SHORT of itself low, as if the logits were: log p, taken with the same one, is SHORT (sum p x - x_t) too high, a matter of targets far below what the row
// expects, up to 3e-6 at x_t = m - 250.  sum p x lies within log V of m: what m - x_t has beyond 16 is made up for.
constexpr double LOW = 5.0e-8, SHORT = 1.0 - (double)LOG2E / 1.4426950408889634;
__device__ __forceinline__ float exp_at(float x, float m) {
  const Scale s = scale_of(m);
  return ex2(fmaf(x, s.a, s.b));
}
__device__ __forceinline__ double log_prob(float rest, float et, float xt, float m) {
  const float sum = rest + et;
  if (isinf(m) || sum != sum) return NAN;
  if (rest < 0.5f * et) return -(double)log1pf(rest / et);
  const int bits = __float_as_int(sum), k = (bits - 0x3f3504f3) >> 23;            // f in [sqrt(1/2), sqrt(2))
  const Scale s = scale_of(m);
  double e = is_far(m) ? (double)xt - (double)m : ((double)xt * (double)LOG2E + (double)s.b) * 0.693147180559945309;
  if (!is_far(m) && m - xt > 16.f && !isinf(xt)) e -= SHORT * ((double)m - (double)xt - 16.0);
  return e - ((double)k * 0.693147180559945309 + (double)logf(__int_as_float(bits - (k << 23))) + LOW);
}

struct Rows {                                // logits in, gradient out
  const bf16* x;
  long ld;
  int V;
  const int* target;
  bf16* g;                                   // or null
  long ldg;
  int gcols, rows;
};
// A row whose slope is not finite: 0 in its columns from V on too, where the padding's exponentials of 0 times that are NaN.  By a warp, behind its stores of the row's last piece.
// (Out of line: inside the kernels it cost pair_k up to 9 %.)
__device__ __noinline__ void clear_columns(bf16* g, int from, int to) {
  __syncwarp();
  for (int c = from + (int)(threadIdx.x & 31); c < to; c += 32) g[c] = __float2bfloat16(0.f);
}
__device__ __forceinline__ void clear_behind(const Rows& q, bf16* g, const Shape& shape) {
  if (!(fabsf(shape.f) < INFINITY)) clear_columns(g, q.V, q.gcols);
}
struct Policy {
  const float *adv, *old_lp, *ref_lp, *weight;
  int adv_rows;                              // rows of an advantage
  float lo, hi, beta, uniform;
  float *loss, *logp, *kl, *clipped;
};

// What a row's terms are made of besides its log probability.
struct Terms {
  float adv, old_lp, ref_lp;
};
__device__ __forceinline__ Terms terms_of(const Policy& a, int r) {
  return {a.adv ? a.adv[r / a.adv_rows] : 0.f, a.old_lp ? a.old_lp[r] : 0.f, a.ref_lp ? a.ref_lp[r] : 0.f};
}

// exp(d) - 1 - d
__device__ __forceinline__ float k3(float d) {
  if (fabsf(d) >= 0.5f) return expm1f(d) - d;
  float s = 1.f / 362880.f;                  // the series, from d^9 / 9! down
  s = fmaf(s, d, 1.f / 40320.f);
  s = fmaf(s, d, 1.f / 5040.f);
  s = fmaf(s, d, 1.f / 720.f);
  s = fmaf(s, d, 1.f / 120.f);
  s = fmaf(s, d, 1.f / 24.f);
  s = fmaf(s, d, 1.f / 6.f);
  s = fmaf(s, d, 0.5f);
  return s * d * d;
}
// Loss terms of a row from its log probability; returns dloss / dlog p.
struct Said {
  float loss, logp, kl, clipped;
};
__device__ __forceinline__ float policy_terms(const Policy& a, const Terms& at, double lp, float w, Said& said) {
  float loss = 0.f, slope = 0.f, kl = 0.f, clipped = 0.f;
  if (a.adv) {
    const float ratio = a.old_lp ? expf((float)(lp - (double)at.old_lp)) : lp == lp ? 1.f : NAN;
    const float raw = ratio * at.adv, held = fminf(fmaxf(ratio, 1.f - a.lo), 1.f + a.hi) * at.adv;
    if (raw > held) { loss = -held; clipped = 1.f; }
    else { loss = -raw; slope = -raw; }
  }
  if (a.ref_lp) {
    const float d = (float)((double)at.ref_lp - lp);
    kl = k3(d);
    if (a.beta != 0.f) {
      loss = fmaf(a.beta, kl, loss);
      slope = fmaf(-a.beta, expm1f(d), slope);
    }
  }
  said = {w * loss, (float)lp, kl, clipped};
  return w * slope;
}
__device__ __forceinline__ void policy_say(const Policy& a, int r, const Said& said) {
  if (a.loss) a.loss[r] = said.loss;
  if (a.logp) a.logp[r] = said.logp;
  if (a.kl) a.kl[r] = said.kl;
  if (a.clipped) a.clipped[r] = said.clipped;
}
__device__ __forceinline__ float policy_terms(const Policy& a, int r, const Terms& at, double lp, float w) {
  Said said;
  const float slope = policy_terms(a, at, lp, w, said);
  policy_say(a, r, said);
  return slope;
}
__device__ __forceinline__ void policy_masked(const Policy& a, int r) { policy_say(a, r, {}); }

// global -> this CTA's shared memory, both on 16 bytes, completion on an mbarrier
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}

// the same with a policy for L2
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar, uint64_t policy) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, [%3], %4;"
               ::"r"(dst), "l"(src), "r"(bytes), "r"(bar), "l"(policy) : "memory");
}
__device__ __forceinline__ uint64_t l2_keep() {
  uint64_t p;
  asm volatile("createpolicy.fractional.L2::evict_last.b64 %0, 1.0;" : "=l"(p));
  return p;
}
__device__ __forceinline__ uint64_t l2_pass() {
  uint64_t p;
  asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(p));
  return p;
}

// Up to 1024 columns: a warp takes K rows at a time (NC pieces of 8 x 32 columns each), and a lane each the terms of a row, which cost a warp more instructions than the
// exponentials of 1024 columns.  One row stays in registers for its gradient; of several the pieces are read again, from L1 or L2 (kept in registers they cost the warps that hide
// the terms' latency).  Bound by the issue of instructions (72 % of the slots; every exponential is taken twice, for the sum and for the gradient) and by latency, not by memory:
// 60000 x 256, three quarters of the rows counting, 28.7 us with K = 4 (all counting: 31), 31.7 with 1; 20000 x 1003 24.5 us with K = 1, 29.7 with 4.
template <int NC, int K>
__global__ void __launch_bounds__(256) policy_warp_k(Rows q, Policy a) {
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, r0 = ((int)blockIdx.x * 8 + (int)(threadIdx.x >> 5)) * K;
  if (r0 >= q.rows) return;
  const int gv = q.g ? (q.gcols + 7) / 8 : 0, my_r = r0 + min(lane, K - 1);
  // the rows' own numbers, a row a lane
  int my_t = my_r < q.rows ? q.target[my_r] : -1;
  const float w = my_r < q.rows && a.weight ? a.weight[my_r] : a.uniform;
  if (my_t >= q.V || w == 0.f) my_t = -1;
  Terms at = {};
  float my_xt = 0.f;
  if (lane < K && my_t >= 0) {
    my_xt = __bfloat162float(q.x[(long)my_r * q.ld + my_t]);
    at = terms_of(a, my_r);
  }
  uint4 v[NC];
  auto fetch = [&](int r) {
    const bf16* x = q.x + (long)r * q.ld;
#pragma unroll
    for (int j = 0; j < NC; j++) {
      const int c = (j * 32 + lane) * 8;
      v[j] = c < q.V ? *reinterpret_cast<const uint4*>(x + c) : make_uint4(NEG2, NEG2, NEG2, NEG2);
      if (c + 8 > q.V) v[j] = cut_from(v[j], q.V - c);
    }
  };
  float my_m = 0.f, my_rest = 0.f;
#pragma unroll (K > 1 ? 2 : 1)
  for (int k = 0; k < K; k++) {
    const int t = __shfl_sync(0xffffffffu, my_t, k);
    if (t < 0) continue;
    fetch(r0 + k);
    uint32_t m2 = NEG2;
#pragma unroll
    for (int j = 0; j < NC; j++) m2 = max2(m2, top8(v[j]));
    const float m = warp_max(fmaxf(lo2(un2(m2)), hi2(un2(m2))));
    Sum s;
    s.m = m;
    s.sc = scale_of(m);
#pragma unroll
    for (int j = 0; j < NC; j++) {
      if ((j * 32 + lane) == t >> 3) v[j] = cut_one(v[j], t & 7);
      s.add(v[j]);
    }
    const float rest = warp_sum(s.sum());
    if (lane == k) { my_m = m; my_rest = rest; }
  }
  Shape my_shape = {0.f, 0.f, 0.f};
  float my_at = 0.f;
  if (lane < K && my_r < q.rows) {
    if (my_t < 0) {
      policy_masked(a, my_r);
    } else {
      const float et = exp_at(my_xt, my_m), slope = policy_terms(a, my_r, at, log_prob(my_rest, et, my_xt, my_m), w), inv = slope / (my_rest + et);
      my_shape = shape_of(my_m, -inv);
      my_at = inv * my_rest;
    }
  }
  if (!q.g) return;
  __syncwarp();                              // every lane has the targets' logits: the gradient may take the rows' place
#pragma unroll (K > 1 ? 2 : 1)
  for (int k = 0; k < K; k++) {
    if (r0 + k >= q.rows) return;
    bf16* g = q.g + (long)(r0 + k) * q.ldg;
    const int t = __shfl_sync(0xffffffffu, my_t, k);
    if (t >= 0) {
      const Shape shape = {__shfl_sync(0xffffffffu, my_shape.a, k), __shfl_sync(0xffffffffu, my_shape.b, k), __shfl_sync(0xffffffffu, my_shape.f, k)};
      const float at_t = __shfl_sync(0xffffffffu, my_at, k);
      if (K > 1) fetch(r0 + k);
#pragma unroll
      for (int j = 0; j < NC; j++) {
        const int i = j * 32 + lane;
        if (i >= gv) continue;
        uint4 o = grad8(v[j], shape);
        if (i == t >> 3) o = put_one(o, t & 7, at_t);
        store8(g, i, q.gcols, o);
      }
      clear_behind(q, g, shape);
    }
    for (int i = (t >= 0 ? NC * 32 : 0) + lane; i < gv; i += 32) store8(g, i, q.gcols, make_uint4(0, 0, 0, 0));
  }
}

// mbar_wait with the first look inline
__device__ __noinline__ bool wait_longer(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* err) { return mbar_wait(bar, parity, abort_flag, 1, err); }
__device__ __forceinline__ bool wait_for(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* err) {
  return mbar_try(bar, parity) || wait_longer(bar, parity, abort_flag, err);
}
// Sums of the pieces v[lane], v[lane + 32], ... below n.
__device__ __forceinline__ void sum_pieces(Sum& s, const uint4* v, int n) {
  const int lane = threadIdx.x & 31;
  int j0 = 0;
  for (; j0 + 128 <= n; j0 += 128) {
    const int j = j0 + lane;
    const uint4 x[4] = {v[j], v[j + 32], v[j + 64], v[j + 96]};
    s.see(max2(max2(top8(x[0]), top8(x[1])), max2(top8(x[2]), top8(x[3]))));
#pragma unroll
    for (int u = 0; u < 4; u++) s.add(x[u]);
  }
  for (; j0 < n; j0 += 32) {
    const uint4 x = j0 + lane < n ? v[j0 + lane] : make_uint4(NEG2, NEG2, NEG2, NEG2);
    s.see(top8(x));
    s.add(x);
  }
}
// The same pieces' gradients.
template <bool FUSED>
__device__ __forceinline__ void grad_pieces(uint4* g, const uint4* v, int n, const Shape& shape) {
  int j = threadIdx.x & 31;
  for (; j + 96 < n; j += 128) {
    const uint4 x[4] = {v[j], v[j + 32], v[j + 64], v[j + 96]};
#pragma unroll
    for (int u = 0; u < 4; u++) __stcs(g + j + 32 * u, grad8<FUSED>(x[u], shape));
  }
  for (; j < n; j += 32) __stcs(g + j, grad8<FUSED>(v[j], shape));
}
__device__ __forceinline__ void grad_pieces(uint4* g, const uint4* v, int n, const Shape& shape) {
  if (shape.f == 0.f) grad_pieces<true>(g, v, n, shape);
  else grad_pieces<false>(g, v, n, shape);
}

// Rows of up to TWICE columns: a warp per row, read twice, the second time from L1 or L2 (8192 x 2100: 22.7 us; through shared memory, as longer rows, 25.6, and at 4000 columns 32
// where a warp takes 35.5).  Without a gradient it is read once: up to ONCE columns where the rows are few (1000 x 2500: 4.2 us, the stream below 5.9; 8192 x 4000: 20.8 and 17.8).
__global__ void __launch_bounds__(256, 4) policy_twice_k(Rows q, Policy a) {
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, r = (int)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (r >= q.rows) return;
  const int t = q.target[r], nv = (q.V + 7) / 8, gv = q.g ? (q.gcols + 7) / 8 : 0;
  const float w = a.weight ? a.weight[r] : a.uniform;
  bf16* g = q.g + (long)r * q.ldg;
  uint4* const gp = reinterpret_cast<uint4*>(g);
  if (t < 0 || t >= q.V || w == 0.f) {
    if (lane == 0) policy_masked(a, r);
    for (int i = lane; i < q.gcols / 8 && q.g; i += 32) __stcs(gp + i, make_uint4(0, 0, 0, 0));
    if (gv > q.gcols / 8 && lane == 0) store8(g, gv - 1, q.gcols, make_uint4(0, 0, 0, 0));
    return;
  }
  const bf16* x = q.x + (long)r * q.ld;
  const uint4* const v = reinterpret_cast<const uint4*>(x);
  const float xt = __bfloat162float(x[t]);
  const Terms at = terms_of(a, r);
  const int tv = t >> 3, cut = q.V & 7 ? nv - 1 : -1, skip = tv & ~127;               // the target's 128 pieces and the last ones are looked at one by one
  Sum s;
  auto one = [&](int j) {
    uint4 y = j < nv ? v[j] : make_uint4(NEG2, NEG2, NEG2, NEG2);
    if (j == cut) y = cut_from(y, q.V - 8 * j);
    if (j == tv) y = cut_one(y, t & 7);
    s.see(top8(y));
    s.add(y);
  };
  int j0 = 0;
  for (; j0 + 128 <= nv - (cut >= 0); j0 += 128) {
    const int j = j0 + lane;
    if (j0 == skip) {
      for (int u = 0; u < 4; u++) one(j + 32 * u);
      continue;
    }
    const uint4 y[4] = {v[j], v[j + 32], v[j + 64], v[j + 96]};
    s.see(max2(max2(top8(y[0]), top8(y[1])), max2(top8(y[2]), top8(y[3]))));
#pragma unroll
    for (int u = 0; u < 4; u++) s.add(y[u]);
  }
  for (; j0 < nv; j0 += 32) one(j0 + lane);
  const float m = fmaxf(s.m, xt), rest = warp_sum(s.sum()) * onto(s.m, m), et = exp_at(xt, m);
  float slope = 0.f;
  if (lane == 0) slope = policy_terms(a, r, at, log_prob(rest, et, xt, m), w);
  if (!q.g) return;
  const float inv = __shfl_sync(0xffffffffu, slope, 0) / (rest + et);
  __syncwarp();                              // every lane has the row's sums: the gradient may take its place
  const Shape shape = shape_of(m, -inv);
  grad_pieces(gp, v, min(nv - (cut >= 0), q.gcols / 8), shape);
  if (cut >= 0 && lane == 0) {
    uint4 y = v[cut];
    y = cut_from(y, q.V - 8 * cut);
    store8(g, cut, q.gcols, grad8(y, shape));
  }
  clear_behind(q, g, shape);
  __syncwarp();
  if (lane == 0) g[t] = __float2bfloat16(inv * rest);      // (behind the store of the piece)
  for (int i = nv + lane; i < gv; i += 32) store8(g, i, q.gcols, make_uint4(0, 0, 0, 0));
}

// Longer rows pass through shared memory once: NS places, each for a row (or the CTA's share of it in a cluster of CL), and in each place a part for each of NP pairs of warps.
// The first warp of a pair sums its part, the second turns it into the gradient once the row's slope is known and fetches the part of the row that comes NS rows
// later, 256 pieces at a time, so that one row's exponentials, another's gradient and the copies of a third run side by side.  One more warp
// adds the pairs' sums and turns them into the row's terms (when the first of the others did, they waited: 8192 x 32003 took 196 us).  A CTA takes the rows
// blockIdx / CL + k gridDim / CL.  Three quarters of the rows counting: 16384 x 50257 470 us, 0.92 of the copy rate; 8192 x 32003 159 (0.87); in clusters 4096 x 128256 343 (0.82),
// bound by the clusters that fit and by a trip between their CTAs for each row.
constexpr int CHUNK = 256, CHUNKS = 4;                     // pieces of a copy, copies of a part at most
struct RowOut {                                            // what the gradient is made of
  Shape shape;
  float at_target;                                         // the target's column
  int t;
};
__device__ __forceinline__ void mbar_arrive_remote(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
__device__ __forceinline__ bool mbar_try_cluster(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred P;\n\t"
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 P, [%1], %2;\n\t"
      "selp.b32 %0, 1, 0, P;\n\t}"
      : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
  return ok != 0;
}
// The CTA's rows, 32 at a time: which of them count, and (per lane) their targets.
struct Block {
  int base, t;
  unsigned on;
  __device__ __forceinline__ void load(const Rows& q, const float* weight, float uniform, int first, int step, int at, int total) {
    base = at;
    const int i = at + (threadIdx.x & 31), r = first + i * step;
    t = i < total ? q.target[r] : -1;
    const float w = i < total && weight ? weight[r] : uniform;
    on = __ballot_sync(0xffffffffu, t >= 0 && t < q.V && w != 0.f);
  }
};
template <int NP>
__global__ void __launch_bounds__(64 * NP + 32, NP >= 8 ? 1 : 12 / NP) policy_row_k(Rows q, Policy a, int CL, int NS, int pw, int* err) {
  extern __shared__ __align__(16) uint4 buf[];             // [NS][NP][pw]
  __shared__ __align__(8) uint64_t s_full[4 * NP * CHUNKS], s_done[4], s_ready[4], s_peer[4];
  __shared__ float2 s_part[4][NP];
  __shared__ float4 s_all[4][2][8];                        // (by turns, so that a CTA that is ahead doesn't write over what another has yet to read)
  __shared__ RowOut s_out[4];
  __shared__ int s_abort;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, rank = CL > 1 ? (int)cluster_ctarank() : 0, step = (int)gridDim.x / CL, first = (int)blockIdx.x / CL;
  for (int i = tid; i < 4 * NP * CHUNKS; i += blockDim.x) mbar_init(smem_u32(&s_full[i]), 1);
  if (tid < 4) {
    mbar_init(smem_u32(&s_done[tid]), NP);
    mbar_init(smem_u32(&s_ready[tid]), 1);
    mbar_init(smem_u32(&s_peer[tid]), CL);
  }
  if (tid == 0) s_abort = 0;
  mbar_fence_init();
  __syncthreads();
  if (CL > 1) cluster_sync_all();
  pdl_wait();
  pdl_launch_dependents();
  const int p = warp % NP;                                                                                         // the pair
  const int nv = (q.V + 7) / 8, per = (nv + CL - 1) / CL, c0 = min(rank * per, nv), c1 = min(c0 + per, nv);        // the CTA's pieces
  const int v0 = min(c0 + p * pw, c1), n = min(v0 + pw, c1) - v0, nc = (n + CHUNK - 1) / CHUNK;                    // the pair's, in nc copies
  const int total = first < q.rows ? (q.rows - first + step - 1) / step : 0;
  bool dead = false;                                       // a wait ran out: no further ones
  auto wait = [&](uint64_t* bar, int parity) {
    if (!dead && !wait_for(smem_u32(bar), parity, &s_abort, err)) dead = true;
  };
  auto place = [&](int k) { return buf + (k * NP + p) * pw; };
  auto full = [&](int k, int c) { return &s_full[(k * NP + p) * CHUNKS + c]; };
  auto part = [&](int r) { return reinterpret_cast<const uint4*>(q.x + (long)r * q.ld) + v0; };
  auto fetch = [&](const uint4* x, int k, int c) {         // copy c of a row's part x into place k
    if (!dead && lane == 0) {
      const int m = min(CHUNK, n - c * CHUNK);
      const uint32_t bar = smem_u32(full(k, c));
      mbar_expect_tx(bar, 16 * m);
      bulk_load(smem_u32(place(k) + c * CHUNK), x + c * CHUNK, 16 * m, bar);
    }
  };
  // the rows to come that count, one after the other
  Block ahead;
  unsigned left = 0;
  ahead.base = -32;
  auto next = [&]() {
    while (left == 0) {
      if (ahead.base + 32 >= total) return -1;
      ahead.load(q, a.weight, a.uniform, first, step, ahead.base + 32, total);
      left = ahead.on;
    }
    const int b = __ffs(left) - 1;
    left &= left - 1;
    return first + (ahead.base + b) * step;
  };
  if (warp >= NP && warp < 2 * NP)
    for (int k = 0; k < NS; k++) {
      const int r = next();
      if (r < 0) break;
      for (int c = 0; c < nc; c++) fetch(part(r), k, c);
    }
  // the row's terms, from its pairs' sums (by a warp)
  auto tell = [&](int k, int phase, int r, int t, float xt, const Terms& at, float w) {
    wait(&s_done[k], phase);
    const float2 y = s_part[k][lane % NP];
    const float ym = lane < NP ? y.x : -INFINITY, ys = lane < NP ? y.y : 0.f;
    float top = warp_max(ym), rest = warp_sum(ys * onto(ym, top));
    if (CL > 1) {                                          // and the CTAs' to all of them (with the target's logit, which is so read before any CTA writes)
      if (lane < CL) {
        const uint32_t to = mapa_shared(smem_u32(&s_all[k][phase][rank]), lane);
        asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %3};" ::"r"(to), "f"(top), "f"(rest), "f"(xt) : "memory");
        mbar_arrive_remote(mapa_shared(smem_u32(&s_peer[k]), lane));
      }
      if (!dead) {
        uint64_t t0 = 0;
        for (uint32_t it = 1; !mbar_try_cluster(smem_u32(&s_peer[k]), phase); ++it)
          if ((it & 0x3ff) == 0) {
            const uint64_t now = kh_globaltimer();
            if (t0 == 0) t0 = now;
            else if (now - t0 > KH_WAIT_LIMIT_NS || *(volatile int*)&s_abort) {
              s_abort = 1;
              atomicCAS(err, 0, 1);
              dead = true;
              break;
            }
          }
      }
      __syncwarp();
      const float4 z = s_all[k][phase][lane % CL];
      const float am = lane < CL ? z.x : -INFINITY, as = lane < CL ? z.y : 0.f;
      top = warp_max(am);
      rest = warp_sum(as * onto(am, top));
    }
    if (lane == 0) {
      const float m1 = fmaxf(top, xt), et = exp_at(xt, m1);
      rest *= onto(top, m1);
      Said said;
      const float inv = policy_terms(a, at, log_prob(rest, et, xt, m1), w, said) / (rest + et);
      s_out[k] = {shape_of(m1, -inv), inv * rest, t};
      mbar_arrive(smem_u32(&s_ready[k]));
      if (rank == 0) policy_say(a, r, said);
    }
    __syncwarp();
  };
  if (warp < NP) {
    // ---- sums
    const int cut = 8 * (v0 + n) > q.V && n > 0 ? n - 1 : -1;                                                      // a piece that sticks out of the vocabulary
    int k = 0, phase = 0;
    for (int base = 0; base < total; base += 32) {
      Block b;
      b.load(q, a.weight, a.uniform, first, step, base, total);
      for (unsigned m = b.on; m; m &= m - 1) {
        const int t = __shfl_sync(0xffffffffu, b.t, __ffs(m) - 1), tv = (t >> 3) - v0;
        uint4* const here = place(k);
        Sum s;
        for (int c = 0; c < nc; c++) {
          wait(full(k, c), phase);
          if (cut >> 8 == c && (cut & 31) == lane) here[cut] = cut_from(here[cut], q.V - 8 * (v0 + cut));
          if (tv >> 8 == c && tv < n && (tv & 31) == lane) reinterpret_cast<unsigned short*>(here)[8 * tv + (t & 7)] = 0xff80;          // the others alone
          sum_pieces(s, here + c * CHUNK, min(CHUNK, n - c * CHUNK));
        }
        const float rest = warp_sum(s.sum());
        if (lane == 0) {
          s_part[k][p] = make_float2(s.m, rest);
          mbar_arrive(smem_u32(&s_done[k]));
        }
        __syncwarp();
        if (++k == NS) { k = 0; phase ^= 1; }
      }
    }
  } else if (warp == 2 * NP) {
    // ---- terms: a lane each what a row's need, 32 rows at a time
    int k = 0, phase = 0;
    for (int base = 0; base < total; base += 32) {
      Block b;
      b.load(q, a.weight, a.uniform, first, step, base, total);
      const int my_r = first + (base + lane) * step;
      const bool on = b.on >> lane & 1;
      if (rank == 0 && base + lane < total && !on) policy_masked(a, my_r);
      Terms my_at = {};
      float my_xt = 0.f, my_w = a.uniform;
      if (on) {
        my_xt = __bfloat162float(q.x[(long)my_r * q.ld + b.t]);
        my_at = terms_of(a, my_r);
        if (a.weight) my_w = a.weight[my_r];
      }
      for (unsigned m = b.on; m; m &= m - 1) {
        const int i = __ffs(m) - 1;
        auto of = [&](float x) { return __shfl_sync(0xffffffffu, x, i); };
        const Terms at = {of(my_at.adv), of(my_at.old_lp), of(my_at.ref_lp)};
        tell(k, phase, first + (base + i) * step, __shfl_sync(0xffffffffu, b.t, i), of(my_xt), at, of(my_w));
        if (++k == NS) { k = 0; phase ^= 1; }
      }
    }
  } else {
    // ---- gradients
    const int gv = (q.gcols + 7) / 8, whole = min(n, q.gcols / 8 - v0);
    const bool sticks = 8 * (v0 + n) > q.V;                // the part ends behind the vocabulary
    int k = 0, phase = 0;
    for (int base = 0; base < total; base += 32) {
      Block b;
      b.load(q, a.weight, a.uniform, first, step, base, total);
      for (int i = 0; i < min(32, total - base); i++) {
        bf16* const g = q.g + (long)(first + (base + i) * step) * q.ldg;
        uint4* const gp = reinterpret_cast<uint4*>(g) + v0;
        if (rank == CL - 1)                                // beyond the vocabulary
          for (int j = nv + p * 32 + lane; j < gv; j += 32 * NP) store8(g, j, q.gcols, make_uint4(0, 0, 0, 0));
        if (!(b.on >> i & 1)) {
          for (int j = lane; j < whole; j += 32) gp[j] = make_uint4(0, 0, 0, 0);
          if (n > 0 && whole < n && lane == 0) store8(g, v0 + whole, q.gcols, make_uint4(0, 0, 0, 0));
          continue;
        }
        const int rn = next();
        const uint4* const xn = part(rn);
        wait(&s_ready[k], phase);
        const RowOut o = s_out[k];
        const uint4* const here = place(k);
        const int tv = (o.t >> 3) - v0;
        for (int c = 0; c < nc; c++) {
          wait(full(k, c), phase);
          grad_pieces(gp + c * CHUNK, here + c * CHUNK, min(CHUNK, whole - c * CHUNK), o.shape);
          if (whole < n && c == nc - 1 && lane == 0) store8(g, v0 + whole, q.gcols, grad8(here[whole], o.shape));
          fence_proxy_async_smem();
          __syncwarp();
          if (tv >> 8 == c && tv < n && lane == 0) g[o.t] = __float2bfloat16(o.at_target);                      // (behind the store of the piece)
          if (rn >= 0) fetch(xn, k, c);
        }
        if (sticks) clear_behind(q, g, o.shape);
        if (++k == NS) { k = 0; phase ^= 1; }
      }
    }
  }
  if (dead)                                                // given up: the copies on their way come to their end first
    for (const uint64_t t0 = kh_globaltimer(); kh_globaltimer() - t0 < 1000000;) {}
  __syncwarp();
  if (CL > 1) cluster_sync_all();                          // no CTA leaves while another may still write to it
}

// ------------------------------------------------------------------------------ rows read as a stream: log probabilities, preference
// A CTA takes rows in pieces of up to CHUNK x 8 columns.  One warp (the scout) goes through the CTA's rows, 32 at a time, and finds out what is to be done with them; a second
// fetches their chunks by bulk copies into a ring of slots, from which WORKERS warps take one after the other.  Sums (S) of a row's chunks are put together by
// the warp that ends the row's last one.  The preference loss reads ranges of pairs for their sums and, LAG_BYTES of logits behind a range's end, for their gradients (G; a CTA's
// latest row first), so that a pair's margin is known when it is asked for: the warp
// that ends a pair's last row adds the pair up, in the order of its rows.  A pair's slope is known only when all its rows have been summed, so the logits are read twice: three passes
// over memory where L2 does not hold the rows in between, which it hardly does (7 % of the sectors: the gradients follow 100 MB behind the pair's end, as a smaller distance costs
// waits: 32 pairs, 6400 x 50257, with 36 MB 332 us, with 100 281).  6 pairs, 9600 x 50257: 451 us, 0.98 of the copy rate for three passes; 20 pairs, 8000 x 32003: 230 (1.02).
// Log probabilities, 8192 x 50257, three quarters counting: 111 us, 0.84; the exponentials' unit is busy for 70 % of
// the time and the issue slots for 65 %.  (Parts fixed to 16 or 24 warps that fetch for themselves took 136 and 152 us, a CTA a row with plain loads 129: better below 300 rows alone.)
struct Pairs {
  const int* starts;                         // [2 P + 1]
  int P;
  const float *ref_lp, *weight;
  float beta, smooth, uniform;
  float *loss, *margin, *ratio, *logp;
  // work.  What one CTA tells another are words that are EMPTY until written and again when read, so that no fence is needed: one waits for all the stores that an SM has on
  // their way, which took 10 us and more beside the stream of gradients.
  uint64_t* lead;                            // log p - ref of each row
  uint64_t* stat;                            // [2]: m, 1 / (R + e_t); R / (R + e_t), 0 of each row
  uint64_t* coef;                            // dloss / dlog p of each pair's chosen sequence, 0; EMPTY again at the end
  int *count, *gone;                         // rows of a pair that are done, CTAs that are: 0 before and after
  int want, lag;                             // rows of a range, about; rows whose sums are taken between a range and its gradients
};
constexpr int WORKERS = 24, SLOTS = 2 * WORKERS;           // warps that compute
constexpr int PARTS = 512;                   // sums of chunks that are kept: a row's, and those of the chunks that may be taken before they are added
constexpr int MOST_CHUNKS = PARTS - 2 * SLOTS;
constexpr int RANGE_BYTES = 18 << 20, LAG_BYTES = 100 << 20;

struct Range {                               // pairs p0 .. p1 - 1, rows lo .. hi - 1
  int p0, p1, lo, hi;
};
enum { SUMS, GRADS, FAR, ZEROS, END };       // (FAR: gradients of a row whose scale is)
template <bool PREF>
struct Walk {                                // a CTA's way through its rows, by a warp
  Range now, cur, due;                       // of now; the latest whose sums are taken; the one whose gradients are due
  int kind;
  int first, base, n;                        // rows of the CTA in the range: the first, the 32 of now, their number

  __device__ __forceinline__ Range range(const Rows& q, const Pairs& b, int p0) {
    if (!PREF) return {p0, 1, 0, p0 ? 0 : q.rows};
    Range r = {b.P, b.P, 0, 0};
    if (p0 >= b.P) return r;
    r.p0 = p0;
    r.lo = b.starts[2 * p0];
    for (int p = p0 + 1;; p += 32) {
      const int x = p + (int)(threadIdx.x & 31);
      const unsigned end = __ballot_sync(0xffffffffu, x >= b.P || b.starts[2 * x] - r.lo >= b.want);
      if (end) { r.p1 = min(b.P, p + __ffs(end) - 1); break; }
    }
    r.hi = b.starts[2 * r.p1];
    return r;
  }
  __device__ __forceinline__ void enter(int k, const Range& r) {
    const int unit = blockIdx.x, units = gridDim.x;
    kind = k; now = r; base = -32;
    first = r.lo + (unit - r.lo % units + units) % units;  // the rows that leave the CTA's number over the CTAs: as many as any other has, one more or less, over all ranges
    n = r.hi > first ? (r.hi - first + units - 1) / units : 0;
  }
  __device__ __forceinline__ void start(const Rows& q, const Pairs& b) {
    cur = due = range(q, b, 0);
    if (PREF ? cur.p0 < cur.p1 : true) enter(SUMS, cur);
    else kind = END;
  }
  __device__ __forceinline__ void advance(const Rows& q, const Pairs& b) {
    if (!PREF) { kind = END; return; }
    const bool grads = q.g && due.p0 < cur.p1;
    if (cur.p1 < b.P && !(grads && cur.hi - due.hi > b.lag)) {
      cur = range(q, b, cur.p1);
      enter(SUMS, cur);
    } else if (grads) {
      enter(GRADS, due);
      due = range(q, b, due.p1);
    } else {
      kind = END;
    }
  }
  __device__ __forceinline__ int row(int i) const { return first + (kind == GRADS ? n - 1 - i : i) * (int)gridDim.x; }
};
struct Job {                                 // what is to be done with a slot's chunk
  int kind, r, c, t;
  float b, f, at_t;                          // gradients: of the shape, the target's column; sums: the target's logit, the reference's log probability, the pair
  int order;                                 // the row's place among the CTA's that are summed
};
__device__ __forceinline__ bool mbar_test(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred P;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 P, [%1], %2;\n\t"
      "selp.b32 %0, 1, 0, P;\n\t}"
      : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
  return ok != 0;
}
constexpr uint64_t EMPTY = ~0ull;            // (as a double or as two floats a NaN that no instruction gives)
__device__ __forceinline__ uint64_t get(const uint64_t* p) {
  uint64_t v;
  asm volatile("ld.relaxed.gpu.global.b64 %0, [%1];" : "=l"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ void put(uint64_t* p, uint64_t v) { asm volatile("st.relaxed.gpu.global.b64 [%0], %1;" ::"l"(p), "l"(v) : "memory"); }
__device__ __forceinline__ uint64_t two(float a, float b) { return (uint64_t)__float_as_uint(a) | (uint64_t)__float_as_uint(b) << 32; }
__device__ __forceinline__ float first_of(uint64_t v) { return __uint_as_float((uint32_t)v); }
__device__ __forceinline__ float second_of(uint64_t v) { return __uint_as_float((uint32_t)(v >> 32)); }
// a word once it has been written; EMPTY if that does not happen (error 9)
__device__ __forceinline__ uint64_t await(const uint64_t* p, volatile int* abort_flag, int* err) {
  uint64_t t0 = 0, v;
  for (uint32_t it = 1; (v = get(p)) == EMPTY; ++it)
    if ((it & 0x3f) == 0) {
      const uint64_t time = kh_globaltimer();
      if (t0 == 0) t0 = time;
      else if (time - t0 > KH_WAIT_LIMIT_NS || *abort_flag) { *abort_flag = 1; atomicCAS(err, 0, 9); break; }
    }
  return v;
}
__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// Margin, loss and slope of a pair of weight w from its sequences' sums; returns dloss / dlog p of the chosen one.
__device__ __forceinline__ float pair_terms(const Pairs& b, int p, float w, double chosen, double rejected, bool write = true) {
  float loss = 0.f, slope = 0.f;
  const double m = (double)b.beta * (chosen - rejected);
  if (w != 0.f) {
    const double z = exp(-fabs(m)), soft = log1p(z);       // log(1 + exp(-m)) = max(-m, 0) + log(1 + exp(-|m|))
    const double lose = fmax(-m, 0.0) + soft, win = fmax(m, 0.0) + soft, big = 1.0 / (1.0 + z), small = z * big;
    loss = (float)(w * ((1.0 - b.smooth) * lose + b.smooth * win));
    slope = (float)(w * b.beta * (b.smooth * (m >= 0.0 ? big : small) - (1.0 - b.smooth) * (m >= 0.0 ? small : big)));
  }
  if (!write) return slope;
  if (b.loss) b.loss[p] = loss;
  if (b.margin) b.margin[p] = (float)m;
  if (b.ratio) { b.ratio[2 * p] = (float)chosen; b.ratio[2 * p + 1] = (float)rejected; }
  return slope;
}
// All rows of pair p are done, or about to be: its margin, loss and slope (by a warp).
__device__ __noinline__ void end_pair(const Pairs& b, int p, volatile int* abort_flag, int* err) {
  const int lane = threadIdx.x & 31;
  const float w = b.weight ? b.weight[p] : b.uniform;
  double sum[2];
#pragma unroll
  for (int k = 0; k < 2; k++) {
    double s = 0.0;
    const int hi = b.starts[2 * p + k + 1];
    for (int r = b.starts[2 * p + k] + lane; r < hi; r += 32 * 8) {           // (eight rows a lane on their way)
      uint64_t v[8];
#pragma unroll
      for (int u = 0; u < 8; u++) v[u] = r + 32 * u < hi ? get(b.lead + r + 32 * u) : 0;
#pragma unroll
      for (int u = 0; u < 8; u++) {
        if (r + 32 * u >= hi) break;
        if (v[u] == EMPTY) v[u] = await(b.lead + r + 32 * u, abort_flag, err);
        put(b.lead + r + 32 * u, EMPTY);
        s += __longlong_as_double((long long)v[u]);
      }
    }
    __syncwarp();
    sum[k] = warp_sum(s);
  }
  if (lane == 0) {
    put(b.coef + p, two(pair_terms(b, p, w, sum[0], sum[1]), 0.f));
    b.count[p] = 0;
  }
  __syncwarp();
}

// Small vocabularies and pairs: a CTA per pair, or a cluster of C where the pairs are fewer than the SMs, a warp per row (NC pieces of 8 x 32 columns in registers), read once for
// the sums and once more, from L1 or L2, for the gradients.  32 rows of a warp at a time, so that their terms are taken side by side.  64 pairs of 36 rows x 256: 6.7 us, a chain of
// dependent trips (starts, targets, rows, the pair's sums, its slope); 32 pairs, 6400 x 1003: 15 us, with a CTA a pair 52; 200 pairs, 100000 x 256: 56 us, as a stream (below) 176, but
// 50 pairs, 25000 x 2000: 78 us, 73 as a stream.  The rule goes by the average: one pair of 50000 rows among 500 of 40 has its CTA alone (3.5 ms, where the two lists by themselves take 17 and 274 us).
constexpr long PAIR_ROWS[2] = {2048, 128};   // rows of a pair, on average, for each of its CTAs, up to which that is so: with 1024 columns at most, with more
constexpr int KEPT = 1024;                   // rows of a CTA whose numbers stay in shared memory; others' go through the workspace
template <int NC>
__global__ void __launch_bounds__(512) pair_k(Rows q, Pairs b, int C, int* err) {
  __shared__ uint64_t s_lead[KEPT], s_stat[KEPT][2];
  __shared__ double s_sum[8][2];             // of each CTA's rows
  __shared__ float s_slope;
  __shared__ int s_bad;
  pdl_wait();
  pdl_launch_dependents();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, rank = C > 1 ? (int)cluster_ctarank() : 0;
  int lo, mid, hi;
  float w;
  auto load = [&](int p) {
    lo = b.starts[2 * p]; mid = b.starts[2 * p + 1]; hi = b.starts[2 * p + 2];
    w = b.weight ? b.weight[p] : b.uniform;
  };
  load((int)blockIdx.x / C);                               // (on its way while all starts are looked over)
  if (tid == 0) s_bad = 0;
  __syncthreads();
  bool bad = false;
#pragma unroll 4
  for (int i = tid; i <= 2 * b.P; i += 512) {
    const int x = b.starts[i], before = b.starts[max(i - 1, 0)];
    bad |= (x < (i ? before : 0)) | (x > q.rows);
  }
  if (bad) s_bad = 1;
  __syncthreads();
  if (s_bad) {                               // (every CTA sees the same)
    if (tid == 0) atomicCAS(err, 0, 8);
    return;
  }
  if (C > 1) cluster_sync_all();             // the others run: their shared memory is there
  const int gv = q.g ? (q.gcols + 7) / 8 : 0;
  for (int p = (int)blockIdx.x / C;;) {
    const int n = (hi - lo - rank + C - 1) / C;            // rows lo + rank, lo + rank + C, ...
    auto fetch = [&](int r, uint4 (&v)[NC]) {
      const bf16* x = q.x + (long)r * q.ld;
#pragma unroll
      for (int j = 0; j < NC; j++) {
        const int c = (j * 32 + lane) * 8;
        v[j] = c < q.V ? *reinterpret_cast<const uint4*>(x + c) : make_uint4(NEG2, NEG2, NEG2, NEG2);
        if (c + 8 > q.V) v[j] = cut_from(v[j], q.V - c);
      }
    };
    auto row = [&](int i) { return lo + rank + i * C; };
    auto lead = [&](int i) { return i < KEPT ? s_lead + i : b.lead + row(i); };
    auto stat = [&](int i) { return i < KEPT ? s_stat[i] : b.stat + 2 * (long)row(i); };
    // 32 rows of a warp at a time: a lane each the numbers and the terms of a row, and the next row's pieces come while this one's are added
    for (int i0 = warp; i0 < n; i0 += 512) {
      const int i = i0 + 16 * lane, r = row(i);
      const int my_t = i < n ? q.target[r] : -1;
      const bool mine = my_t >= 0 && my_t < q.V && w != 0.f;
      const float my_xt = mine ? __bfloat162float(q.x[(long)r * q.ld + my_t]) : 0.f, my_ref = mine && b.ref_lp ? b.ref_lp[r] : 0.f;
      float my_m = 0.f, my_rest = 0.f;
      uint4 v[NC], u[NC];
      uint32_t todo = __ballot_sync(0xffffffffu, mine);
      if (todo) fetch(row(i0 + 16 * (__ffs(todo) - 1)), u);
      while (todo) {
        const int k = __ffs(todo) - 1, t = __shfl_sync(0xffffffffu, my_t, k);
        todo &= todo - 1;
#pragma unroll
        for (int j = 0; j < NC; j++) v[j] = u[j];
        if (todo) fetch(row(i0 + 16 * (__ffs(todo) - 1)), u);
        uint32_t m2 = NEG2;
#pragma unroll
        for (int j = 0; j < NC; j++) m2 = max2(m2, top8(v[j]));
        const float m = warp_max(fmaxf(lo2(un2(m2)), hi2(un2(m2))));
        Sum s;
        s.m = m;
        s.sc = scale_of(m);
#pragma unroll
        for (int j = 0; j < NC; j++) {
          if ((j * 32 + lane) == t >> 3) v[j] = cut_one(v[j], t & 7);
          s.add(v[j]);
        }
        const float rest = warp_sum(s.sum());
        if (lane == k) my_m = m, my_rest = rest;
      }
      if (mine) {
        const float et = exp_at(my_xt, my_m);
        const double lp = log_prob(my_rest, et, my_xt, my_m);
        *lead(i) = (uint64_t)__double_as_longlong(lp - (double)my_ref);
        stat(i)[0] = two(my_m, 1.f / (my_rest + et));
        stat(i)[1] = two(my_rest / (my_rest + et), 0.f);
        if (b.logp) b.logp[r] = (float)lp;
      } else if (i < n) {
        *lead(i) = 0;
        if (b.logp) b.logp[r] = 0.f;
      }
    }
    // the first rows' targets and pieces are on their way again while the pair is added up
    uint4 v[NC], u[NC];
    int my_t;
    uint32_t on, todo;
    auto begin = [&](int i0) {
      my_t = i0 + 16 * lane < n ? q.target[row(i0 + 16 * lane)] : -1;
      on = todo = __ballot_sync(0xffffffffu, q.g && my_t >= 0 && my_t < q.V && w != 0.f);
      if (todo) fetch(row(i0 + 16 * (__ffs(todo) - 1)), u);
    };
    begin(warp);
    __syncthreads();
    if (warp < 2) {                            // the chosen sequence's rows, the rejected one's
      const int half = max(mid - lo - rank + C - 1, 0) / C, to = warp ? n : half;              // the first of the rejected sequence
      double sum = 0.0;
      for (int i = (warp ? half : 0) + lane; i < to; i += 32) sum += __longlong_as_double((long long)*lead(i));
      sum = warp_sum(sum);
      if (C == 1 && lane == 0) s_sum[0][warp] = sum;
      if (C > 1 && lane < C) asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(mapa_shared(smem_u32(&s_sum[rank][warp]), lane)), "d"(sum) : "memory");
      __syncwarp();
    }
    if (C > 1) cluster_sync_all();
    else __syncthreads();
    auto pair = [&](bool write) {
      double chosen = 0.0, rejected = 0.0;
      for (int c = 0; c < C; c++) chosen += s_sum[c][0], rejected += s_sum[c][1];
      return pair_terms(b, p, w, chosen, rejected, write);
    };
    if (tid == 0) s_slope = pair(false);       // (the loss, which nothing waits for, is left to the warp with the fewest rows)
    __syncthreads();
    const float slope = s_slope;
    if (tid == 480 && rank == 0) pair(true);
    __syncwarp();
    for (int i0 = warp; i0 < n; i0 += 512) {
      const int i = i0 + 16 * lane, end = min(32, (n - i0 + 15) / 16);
      if (i0 != warp) begin(i0);
      for (int k = 0; k < end && q.g; k++) {
        const int r = row(i0 + 16 * k), t = __shfl_sync(0xffffffffu, my_t, k);
        bf16* g = q.g + (long)r * q.ldg;
        if (!(on >> k & 1)) {
          for (int at = lane; at < gv; at += 32) store8(g, at, q.gcols, make_uint4(0, 0, 0, 0));
          continue;
        }
        todo &= todo - 1;
#pragma unroll
        for (int j = 0; j < NC; j++) v[j] = u[j];
        if (todo) fetch(row(i0 + 16 * (__ffs(todo) - 1)), u);
        __syncwarp();                          // the gradient may take the row's place
        const uint64_t* st = stat(i0 + 16 * k);
        const float f = r < mid ? slope : -slope, at_t = f * first_of(st[1]);
        const Shape shape = shape_of(first_of(st[0]), -f * second_of(st[0]));
#pragma unroll
        for (int j = 0; j < NC; j++) {
          const int at = j * 32 + lane;
          if (at >= gv) continue;
          uint4 o = grad8(v[j], shape);
          if (at == t >> 3) o = put_one(o, t & 7, at_t);
          store8(g, at, q.gcols, o);
        }
        clear_behind(q, g, shape);
        for (int at = NC * 32 + lane; at < gv; at += 32) store8(g, at, q.gcols, make_uint4(0, 0, 0, 0));
      }
      __syncwarp();
      if (i >= KEPT && i < n) b.lead[row(i)] = b.stat[2 * (long)row(i)] = b.stat[2 * (long)row(i) + 1] = EMPTY;
    }
    p += (int)gridDim.x / C;
    if (p >= b.P) break;
    load(p);
    __syncthreads();                                       // shared memory is the next pair's (clusters have one pair each)
  }
}

template <bool PREF>
__global__ void __launch_bounds__(32 * (WORKERS + 2), 1) stream_k(Rows q, Policy a, Pairs b, int nch, int cp, int* err) {
  extern __shared__ __align__(16) uint4 ring[];            // [SLOTS][CHUNK]
  __shared__ __align__(8) uint64_t s_full[SLOTS], s_free[SLOTS];
  __shared__ __align__(16) Job s_job[SLOTS], s_row[64];   // of chunks; of rows to come
  __shared__ float2 s_part[PARTS];
  __shared__ int s_have[64], s_of[SLOTS], s_next, s_head, s_tail, s_abort, s_bad, s_last;        // s_of: the chunk that a slot was last filled with
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid < SLOTS) {
    mbar_init(smem_u32(&s_full[tid]), 1);
    mbar_init(smem_u32(&s_free[tid]), 1);
    s_of[tid] = -1;
  }
  if (tid < 64) s_have[tid] = 0;
  if (tid == 0) s_abort = s_bad = s_next = s_head = s_tail = 0;
  mbar_fence_init();
  __syncthreads();
  pdl_wait();
  pdl_launch_dependents();
  if (PREF) {                                // every CTA sees to it that the sequences are in order and within the rows
    bool bad = false;
    for (int i = tid; i <= 2 * b.P; i += blockDim.x) bad |= b.starts[i] < (i ? b.starts[i - 1] : 0) || b.starts[i] > q.rows;
    if (bad) s_bad = 1;
    __syncthreads();
    if (s_bad) {
      if (tid == 0) atomicCAS(err, 0, 8);
      return;
    }
  }
  const int nv = (q.V + 7) / 8;              // pieces of a row, in nch chunks of cp
  bool dead = false;                         // a wait ran out
  if (warp == WORKERS + 1) {
    // ---- the rows
    Walk<PREF> at;
    int tail = 0;                            // rows so far
    at.start(q, b);
    bool fresh = true;                       // a range begins
    while (true) {
      if (at.kind != END) {
        if (PREF && fresh && at.kind == SUMS)              // pairs without a row
          for (int x = at.now.p0 + (int)blockIdx.x; x < at.now.p1; x += (int)gridDim.x)
            if (b.starts[2 * x] == b.starts[2 * x + 2]) end_pair(b, x, &s_abort, err);
        fresh = false;
        at.base += 32;
        if (at.base >= at.n) {
          at.advance(q, b);
          fresh = true;
          continue;
        }
      }
      // 32 rows, one a lane
      const int i = at.base + lane;
      const bool is = at.kind != END && i < at.n;
      Job job = {END, 0, 0, 0, 0.f, 0.f, 0.f};
      bool ends = false;
      int seq = 0;
      if (is) {
        job.r = at.row(i);
        job.t = q.target[job.r];
        float w;
        if (PREF) {                          // starts[seq] <= r < starts[seq + 1]
          int lo = 2 * at.now.p0, hi = 2 * at.now.p1;
          while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (b.starts[mid] <= job.r) lo = mid;
            else hi = mid;
          }
          seq = lo;
          w = b.weight ? b.weight[seq >> 1] : b.uniform;
        } else {
          w = a.weight ? a.weight[job.r] : a.uniform;
        }
        const bool on = job.t >= 0 && job.t < q.V && w != 0.f;
        if (at.kind == SUMS) {
          if (on) {
            job.kind = SUMS;
            job.b = __bfloat162float(q.x[(long)job.r * q.ld + job.t]);
            if (PREF) {
              job.f = b.ref_lp ? b.ref_lp[job.r] : 0.f;
              job.at_t = __int_as_float(seq >> 1);
            }
          } else if (PREF) {
            put(b.lead + job.r, 0);
            if (b.logp) b.logp[job.r] = 0.f;
            const int x = seq >> 1;
            ends = atomicAdd(b.count + x, 1) + 1 == b.starts[2 * x + 2] - b.starts[2 * x];
          } else {
            policy_masked(a, job.r);
          }
        } else if (on) {
          const uint64_t coef = await(b.coef + (seq >> 1), &s_abort, err), st0 = await(b.stat + 2 * (long)job.r, &s_abort, err), st1 = await(b.stat + 2 * (long)job.r + 1, &s_abort, err);
          put(b.stat + 2 * (long)job.r, EMPTY);
          put(b.stat + 2 * (long)job.r + 1, EMPTY);
          dead |= coef == EMPTY || st0 == EMPTY || st1 == EMPTY;
          const float slope = seq & 1 ? -first_of(coef) : first_of(coef);
          const Shape shape = shape_of(first_of(st0), -slope * second_of(st0));
          job.kind = is_far(first_of(st0)) ? FAR : GRADS;
          job.b = shape.b; job.f = shape.f; job.at_t = slope * first_of(st1);
        } else {
          job.kind = ZEROS;
        }
      }
      __syncwarp();
      if (PREF)
        for (unsigned e = __ballot_sync(0xffffffffu, ends); e; e &= e - 1) end_pair(b, __shfl_sync(0xffffffffu, seq >> 1, __ffs(e) - 1), &s_abort, err);
      const bool last = at.kind == END;      // (one more row then, of that kind)
      const unsigned todo = last ? 1u : __ballot_sync(0xffffffffu, job.kind != END);
      while (tail + 32 - __shfl_sync(0xffffffffu, *(volatile int*)&s_head, 0) > 64) {
        __nanosleep(100);
        if (*(volatile int*)&s_abort) dead = true;
        if (__any_sync(0xffffffffu, dead)) break;
      }
      dead = __any_sync(0xffffffffu, dead);
      if (dead) break;
      if (todo >> lane & 1) s_row[(tail + __popc(todo & ((1u << lane) - 1))) & 63] = job;
      __threadfence_block();
      __syncwarp();
      tail += __popc(todo);
      if (lane == 0) *(volatile int*)&s_tail = tail;
      if (last) break;
    }
  } else if (warp == WORKERS) {
    // ---- the copies
    int j = 0;                               // chunks so far
    const uint64_t keep = l2_keep(), pass = l2_pass();     // rows that come again; rows that do not
    for (int head = 0;;) {
      int rows = 0;
      while (true) {                         // rows that the scout has (whose waits are bounded: it says so when it gives up)
        rows = __shfl_sync(0xffffffffu, *(volatile int*)&s_tail, 0) - head;
        if (rows > 0) break;
        __nanosleep(40);
        if (*(volatile int*)&s_abort) dead = true;
        dead = __any_sync(0xffffffffu, dead);
        if (dead) break;
      }
      if (dead) break;
      __threadfence_block();
      rows = min(rows, 32);
      const bool last = s_row[(head + rows - 1) & 63].kind == END;
      const int items = last ? (rows - 1) * nch + WORKERS : rows * nch;
      // every lane goes on as its slots come free, no further than SLOTS ahead of any other: a slot's parity tells one turn from the next alone
      uint64_t t0 = 0;
      uint32_t it = 0;
      for (int k = lane;;) {
        const int least = __reduce_min_sync(0xffffffffu, min(k, items));
        if (least >= items) break;
        const int turn = (j + k) / SLOTS, slot = (j + k) - turn * SLOTS;
        const bool go = k < items && k < least + SLOTS && (turn == 0 || mbar_test(smem_u32(&s_free[slot]), (turn - 1) & 1));
        if (go) {
          const int order = head + min(k / nch, rows - 1);
          Job x = s_row[order & 63];
          x.c = k - (order - head) * nch;
          x.order = order;
          s_job[slot] = x;
          *(volatile int*)&s_of[slot] = j + k;
          const uint32_t bar = smem_u32(&s_full[slot]);
          if (x.kind < ZEROS) {
            const uint32_t bytes = 16 * min(cp, nv - x.c * cp);
            mbar_expect_tx(bar, bytes);
            bulk_load(smem_u32(ring + slot * CHUNK), reinterpret_cast<const uint4*>(q.x + (long)x.r * q.ld) + x.c * cp, bytes, bar, x.kind == SUMS && q.g ? keep : pass);
          } else {
            mbar_arrive(bar);
          }
          k += 32;
        }
        if (__any_sync(0xffffffffu, go)) {
          it = 0;
        } else {
          __nanosleep(40);
          if ((++it & 0x3ff) == 0) {
            const uint64_t time = kh_globaltimer();
            if (it == 0x400) t0 = time;
            else if (time - t0 > KH_WAIT_LIMIT_NS || *(volatile int*)&s_abort) { s_abort = 1; atomicCAS(err, 0, 1); dead = true; }
          }
        }
        dead = __any_sync(0xffffffffu, dead);
        if (dead) break;
      }
      __syncwarp();
      if (dead || last) break;
      j += items;
      head += rows;
      if (lane == 0) *(volatile int*)&s_head = head;
    }
  } else {
    // ---- sums and gradients
    const int gv = (q.gcols + 7) / 8, whole_row = q.gcols / 8;
    // every warp takes the next chunk when it has done with its last one
    auto take = [&]() {
      int j = 0;
      if (lane == 0) j = atomicAdd(&s_next, 1);
      return __shfl_sync(0xffffffffu, j, 0);
    };
    for (int j = take();; j = take()) {
      const int turn = j / SLOTS, slot = j - turn * SLOTS;
      // the slot is this chunk's (a parity alone could be that of the turn before the last, when a warp holds the slot's last chunk for long), and it has come
      uint64_t t0 = 0;
      for (uint32_t it = 1; *(volatile int*)&s_of[slot] != j; ++it) {
        __nanosleep(20);
        if ((it & 0x3ff) == 0) {
          const uint64_t time = kh_globaltimer();
          if (t0 == 0) t0 = time;
          else if (time - t0 > KH_WAIT_LIMIT_NS || *(volatile int*)&s_abort) { s_abort = 1; atomicCAS(err, 0, 1); dead = true; break; }
        }
      }
      if (!dead && !wait_for(smem_u32(&s_full[slot]), turn & 1, &s_abort, err)) dead = true;
      dead = __any_sync(0xffffffffu, dead);
      if (dead) break;
      const Job x = s_job[slot];
      if (x.kind == END) break;
      const uint4* const v = ring + slot * CHUNK;
      const int m0 = x.c * cp, n = min(cp, nv - m0);       // the chunk's pieces
      const int tv = (x.t >> 3) - m0;                      // the target's
      const int cut = 8 * (m0 + n) > q.V ? n - 1 : -1;     // one that sticks out of the vocabulary
      if (x.kind == SUMS) {
        Sum s;
        if (cut >= 0 || (tv >= 0 && tv < n)) {
          for (int i0 = 0; i0 < n; i0 += 32) {
            const int i = i0 + lane;
            uint4 y = i < n ? v[i] : make_uint4(NEG2, NEG2, NEG2, NEG2);
            if (i == cut) y = cut_from(y, q.V - 8 * (m0 + cut));
            if (i == tv) y = cut_one(y, x.t & 7);
            s.see(top8(y));
            s.add(y);
          }
        } else {
          sum_pieces(s, v, n);
        }
        float top = s.m, rest = warp_sum(s.sum());
        bool mine = true;
        if (nch > 1) {                       // the last of a row's chunks has all their sums
          int have = 0;
          if (lane == 0) {
            s_part[j & (PARTS - 1)] = make_float2(top, rest);
            __threadfence_block();
            have = atomicAdd(&s_have[x.order & 63], 1);
          }
          mine = __shfl_sync(0xffffffffu, have, 0) == nch - 1;
          if (mine) {
            __threadfence_block();
            if (lane == 0) s_have[x.order & 63] = 0;
            const int j0 = j - x.c;
            float am = -INFINITY;
            for (int i = lane; i < nch; i += 32) am = fmaxf(am, *(volatile float*)&s_part[(j0 + i) & (PARTS - 1)].x);
            top = warp_max(am);
            float as = 0.f;
            for (int i = lane; i < nch; i += 32) {
              const volatile float2* const z = &s_part[(j0 + i) & (PARTS - 1)];
              as += z->y * onto(z->x, top);
            }
            rest = warp_sum(as);
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&s_free[slot]));
        if (mine) {
          int ends = -1;                     // a pair whose last row this is
          if (lane == 0) {
            const float xt = x.b, m1 = fmaxf(top, xt), et = exp_at(xt, m1);
            rest *= onto(top, m1);
            const double lp = log_prob(rest, et, xt, m1);
            if (PREF) {
              const uint64_t lead = (uint64_t)__double_as_longlong(lp - (double)x.f);
              put(b.lead + x.r, lead == EMPTY ? lead - 1 : lead);
              if (q.g) {
                const uint64_t st = two(m1, 1.f / (rest + et));
                put(b.stat + 2 * (long)x.r, st == EMPTY ? st - 1 : st);
                put(b.stat + 2 * (long)x.r + 1, two(rest / (rest + et), 0.f));
              }
              if (b.logp) b.logp[x.r] = (float)lp;
              const int pair = __float_as_int(x.at_t);
              if (atomicAdd(b.count + pair, 1) + 1 == b.starts[2 * pair + 2] - b.starts[2 * pair]) ends = pair;
            } else {
              policy_terms(a, x.r, terms_of(a, x.r), lp, a.weight ? a.weight[x.r] : a.uniform);
            }
          }
          if (PREF) {
            ends = __shfl_sync(0xffffffffu, ends, 0);
            if (ends >= 0) end_pair(b, ends, &s_abort, err);
          }
        }
      } else if (PREF) {
        bf16* const g = q.g + (long)x.r * q.ldg;
        uint4* const gp = reinterpret_cast<uint4*>(g) + m0;
        const int whole = min(n, whole_row - m0);
        const bool end = x.c == nch - 1;
        if (x.kind == ZEROS) {
          for (int i = lane; i < whole; i += 32) __stcs(gp + i, make_uint4(0, 0, 0, 0));
          if (whole < n && lane == 0) store8(g, m0 + whole, q.gcols, make_uint4(0, 0, 0, 0));
        } else {
          const Shape shape = {x.kind == FAR ? 1.f : LOG2E, x.b, x.f};
          grad_pieces(gp, v, min(whole, cut >= 0 ? n - 1 : n), shape);
          if (cut >= 0 && lane == 0) {
            uint4 y = v[n - 1];
            y = cut_from(y, q.V - 8 * (m0 + n - 1));
            store8(g, m0 + n - 1, q.gcols, grad8(y, shape));
          }
          if (cut >= 0) clear_behind(q, g, shape);
          __syncwarp();
          if (tv >= 0 && tv < n && lane == 0) g[x.t] = __float2bfloat16(x.at_t);          // (behind the store of the piece)
        }
        if (end)                             // beyond the vocabulary
          for (int i = nv + lane; i < gv; i += 32) store8(g, i, q.gcols, make_uint4(0, 0, 0, 0));
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&s_free[slot]));
      }
    }
  }
  if (dead)                                  // given up: the copies on their way come to their end first
    for (const uint64_t t0 = kh_globaltimer(); kh_globaltimer() - t0 < 1000000;) {}
  if (PREF) {                                // the last CTA leaves the workspace as it was found
    __syncthreads();
    if (tid == 0) {
      __threadfence();
      s_last = (atomicAdd(b.gone, s_abort ? 0x10001 : 1) & 0xffff) == (int)gridDim.x - 1;
    }
    __syncthreads();
    if (s_last) {
      for (int i = tid; i < b.P; i += blockDim.x) b.coef[i] = EMPTY;
      if (__ldcg(b.gone) >> 16) {            // some CTA gave up
        for (int i = tid; i < b.P; i += blockDim.x) b.count[i] = 0;
        for (int i = tid; i < q.rows; i += blockDim.x) b.lead[i] = b.stat[2 * (long)i] = b.stat[2 * (long)i + 1] = EMPTY;
      }
      __syncthreads();
      if (tid == 0) *b.gone = 0;
    }
  }
}

Rows rows_of(const void* x, long ld, int V, const void* target, void* grad, long ldg, int gcols, int rows) {
  if (rows == 1) {                           // the pitch of a single row says nothing
    ld = ((long)V + 7) / 8 * 8;
    ldg = std::max(((long)gcols + 7) / 8 * 8, ld);
  }
  return {(const bf16*)x, ld, V, (const int*)target, (bf16*)grad, ldg, gcols, rows};
}
int check_rows(const char* name, const Rows& q) {
  if (q.rows < 0 || q.V < 1 || q.ld < q.V || q.ld % 8 || ((uintptr_t)q.x & 15)) {
    kh_set_error("%s: logits of %d rows, %d of %ld columns: the row pitch must be a multiple of 8 and the address of 16 bytes", name, q.rows, q.V, q.ld);
    return -1;
  }
  if (q.g && (q.ldg < q.gcols || q.gcols < q.V || q.ldg % 8 || ((uintptr_t)q.g & 15))) {
    kh_set_error("%s: a gradient of %d columns with row pitch %ld for %d: the pitch must be a multiple of 8 and the address of 16 bytes", name, q.gcols, q.ldg, q.V);
    return -1;
  }
  return 0;
}
int sm_count() {                             // of the current device
  int dev = 0, n = 0;
  cudaGetDevice(&dev);
  return cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess && n > 0 ? n : 148;
}
template <int NP>
cudaError_t launch_row(const Rows& q, const Policy& a, int CL, int part, int sms, cudaStream_t st) {
  cudaError_t e = cudaFuncSetAttribute(policy_row_k<NP>, cudaFuncAttributeMaxDynamicSharedMemorySize, ROW_SMEM);
  if (e != cudaSuccess) return e;
  const int T = 64 * NP + 32, last = (q.V + 7) / 8 - (CL - 1) * part, least = (part + NP - 1) / NP, even = (least + 31) / 32 * 32;
  const int pw = last > (NP - 1) * even && 32 * NP * even <= ROW_SMEM ? even : least, bytes = pw * NP * 16, more = 2304 + 256 * NP;                   // whole 32s where they fit and the last pair has some too
  if (last <= (NP - 1) * pw) return cudaErrorInvalidValue; // (every pair has a piece: one without would run ahead of the others)
  const int fit = std::max(1, std::min(NP >= 8 ? 1 : 12 / NP, 228 * 1024 / (2 * bytes + more)));             // CTAs an SM, by registers and by shared memory with two places
  const int NS = std::max(2, std::min(4, std::min(ROW_SMEM, 228 * 1024 / fit - more) / bytes));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(sms * fit / CL * CL); cfg.blockDim = dim3(T); cfg.dynamicSmemBytes = (size_t)bytes * NS; cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = CL; attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int most = sms * fit;
  if (CL > 1) {                              // clusters that the device holds at once: its groups of SMs are not multiples of every size
    e = cudaOccupancyMaxActiveClusters(&most, policy_row_k<NP>, &cfg);
    if (e != cudaSuccess) return e;
  }
  cfg.gridDim = dim3(std::min(q.rows, std::max(most, 1)) * CL);
  cfg.numAttrs = kh_pdl_enabled() ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, policy_row_k<NP>, q, a, CL, NS, pw, kh_error_word_dev());
}
// pairs of warps: parts of some 100 to 900 pieces, and as many pairs an SM as its registers and shared memory hold (8192 x 6000, 750 pieces: two pairs 44 us, four 38; 8192 x 17000,
// 2125: four 92, eight 100; 8192 x 24000, 3000: four 126, eight 118)
cudaError_t launch_rows(const Rows& q, const Policy& a, int CL, int part, int sms, cudaStream_t st) {
  return part <= 700 ? launch_row<2>(q, a, CL, part, sms, st)
         : part <= 2700 ? launch_row<4>(q, a, CL, part, sms, st) : launch_row<8>(q, a, CL, part, sms, st);
}

template <int NC>
cudaError_t launch_pair(const Rows& q, const Pairs& b, int C, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  // every CTA looks all starts over: with more pairs than this, several each (32768 pairs of 20 rows, 256 columns: with a CTA each 1.4 ms, most of it for that)
  cfg.gridDim = dim3(C > 1 ? b.P * C : std::min(b.P, 8 * sm_count())); cfg.blockDim = dim3(512); cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = C; attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = kh_pdl_enabled() ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, pair_k<NC>, q, b, C, kh_error_word_dev());
}

template <bool PREF>
cudaError_t launch_stream(const Rows& q, const Policy& a, const Pairs& b, cudaStream_t st) {
  constexpr int SMEM = SLOTS * CHUNK * 16;
  const int nv = (q.V + 7) / 8, most = (nv + CHUNK - 1) / CHUNK, cp = ((nv + most - 1) / most + 31) / 32 * 32, nch = (nv + cp - 1) / cp, sms = sm_count();
  if (nch > MOST_CHUNKS) return cudaErrorInvalidValue;
  cudaError_t e = cudaFuncSetAttribute(stream_k<PREF>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(std::max(1, std::min(sms, q.rows))); cfg.blockDim = dim3(32 * (WORKERS + 2)); cfg.dynamicSmemBytes = SMEM; cfg.stream = st;
  cudaLaunchAttribute attr[1];
  if (PREF) {                                // its CTAs wait for one another
    attr[0].id = cudaLaunchAttributeCooperative;
    attr[0].val.cooperative = 1;
    cfg.numAttrs = 1;
  } else {
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs = kh_pdl_enabled() ? 1 : 0;
  }
  cfg.attrs = attr;
  return cudaLaunchKernelEx(&cfg, stream_k<PREF>, q, a, b, nch, cp, kh_error_word_dev());
}

}  // namespace

extern "C" int kh_policy_loss(const void* x, long ld, int V, const void* target, const void* adv, int adv_rows, const void* old_lp, const void* ref_lp, float lo,
                              float hi, float beta, const void* weight, float uniform, void* loss, void* logp, void* kl, void* clipped, void* grad, long ldg,
                              int gcols, int rows, void* stream) {
  const Rows q = rows_of(x, ld, V, target, grad, ldg, gcols, rows);
  const Policy a = {(const float*)adv, (const float*)old_lp, (const float*)ref_lp, (const float*)weight, adv_rows, lo, hi, beta, uniform, (float*)loss, (float*)logp,
                    (float*)kl, (float*)clipped};
  if (check_rows("policy_loss", q)) return -1;
  if (rows == 0) return 0;
  if (adv && adv_rows < 1) { kh_set_error("policy_loss: an advantage serves %d rows", adv_rows); return -1; }
  cudaStream_t st = (cudaStream_t)stream;
  const int nv = (V + 7) / 8;
  if (V <= 1024) {
    // Four rows a warp where the vocabulary is small and the warps are many, so that the terms are taken by four lanes at once; elsewhere that only makes warps wait.
    const bool many = rows >= 128L * sm_count();
#define KH_WARPS(NC, K) KH_LAUNCH((policy_warp_k<NC, K>), (rows + 8 * K - 1) / (8 * K), 256, 0, st, q, a)
    if (V <= 256 && many) KH_WARPS(1, 4);
    else if (V <= 256) KH_WARPS(1, 1);
    else if (V <= 512) KH_WARPS(2, 1);
    else KH_WARPS(4, 1);
#undef KH_WARPS
  } else if (V <= (grad || rows > 32L * sm_count() ? TWICE : ONCE)) {
    KH_LAUNCH(policy_twice_k, (rows + 7) / 8, 256, 0, st, q, a);
  } else {
    int CL = 1;
    while (CL < 8 && (nv + CL - 1) / CL > ROW_PIECES) CL++;
    const int part = (nv + CL - 1) / CL;
    if (part > ROW_PIECES) { kh_set_error("policy_loss: %d columns are too many", V); return -1; }
    const cudaError_t e = grad ? launch_rows(q, a, CL, part, sm_count(), st) : launch_stream<false>(q, a, Pairs{}, st);
    if (e != cudaSuccess) { cudaGetLastError(); kh_set_error("policy_loss: %s", cudaGetErrorString(e)); return -1; }
  }
  KH_LAUNCH_CHECK("policy_loss");
  return 0;
}

// Bytes of the preference loss's workspace: counters in front, 0 before and after every call, and at its end words that are EMPTY (all bits set) before and after; calls of
// fewer rows and pairs find both so.
extern "C" long kh_preference_work_front(int rows, int P) { return (16 + (long)P * 4 + 15) / 16 * 16; }
extern "C" long kh_preference_work_bytes(int rows, int P) { return kh_preference_work_front(rows, P) + ((long)rows * 24 + (long)P * 8 + 15) / 16 * 16; }

extern "C" int kh_preference_loss(const void* x, long ld, int V, const void* target, const void* starts, int P, const void* ref_lp, float beta, float smooth,
                                  const void* weight, float uniform, void* loss, void* margin, void* ratio, void* logp, void* grad, long ldg, int gcols, void* work,
                                  long work_bytes, int rows, void* stream) {
  const Rows q = rows_of(x, ld, V, target, grad, ldg, gcols, rows);
  if (check_rows("preference_loss", q)) return -1;
  if (P < 0 || P > 0x3fffffff || ((uintptr_t)work & 15) || work_bytes < kh_preference_work_bytes(rows, P)) {
    kh_set_error("preference_loss: %d pairs, or a workspace that is not on 16 bytes or too small", P);
    return -1;
  }
  if (P == 0) return 0;
  Pairs b = {(const int*)starts, P, (const float*)ref_lp, (const float*)weight, beta, smooth, uniform, (float*)loss, (float*)margin, (float*)ratio, (float*)logp};
  b.gone = (int*)work;
  b.count = b.gone + 4;
  b.stat = (uint64_t*)((char*)work + (work_bytes - ((long)rows * 24 + (long)P * 8)) / 16 * 16);
  b.lead = b.stat + 2 * (long)rows;
  b.coef = b.lead + rows;
  b.want = std::max(1, RANGE_BYTES / (2 * V));
  b.lag = std::max(1, LAG_BYTES / (2 * V));
  cudaError_t e = cudaSuccess;
  int C = 1;
  if (V <= 2048)
    for (const long sms = sm_count(); C < 8 && 2L * C * P <= sms && rows > 32L * C * P;) C *= 2;
  if (V <= 2048 && (long)rows <= PAIR_ROWS[V > 1024] * C * P) {
    e = V <= 256 ? launch_pair<1>(q, b, C, (cudaStream_t)stream) : V <= 512 ? launch_pair<2>(q, b, C, (cudaStream_t)stream)
        : V <= 1024 ? launch_pair<4>(q, b, C, (cudaStream_t)stream) : launch_pair<8>(q, b, C, (cudaStream_t)stream);
  } else {
    e = launch_stream<true>(q, Policy{}, b, (cudaStream_t)stream);
  }
  if (e != cudaSuccess) { cudaGetLastError(); kh_set_error("preference_loss: %s", cudaGetErrorString(e)); return -1; }
  KH_LAUNCH_CHECK("preference_loss");
  return 0;
}
