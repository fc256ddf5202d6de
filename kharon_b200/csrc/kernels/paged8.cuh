// The 8-bit paged cache (paged8.cu): format, quantisation, page lookup, one token's attention by one warp.
#pragma once
#include "common.cuh"

#define KH_LAUNCH_CHECK(name)                                                     \
  do {                                                                            \
    cudaError_t e_ = cudaGetLastError();                                          \
    if (e_ != cudaSuccess) { kh_set_error(name ": %s", cudaGetErrorString(e_)); return -1; } \
  } while (0)

namespace {

constexpr int E_LO = 64, E_HI = 190;             // exponent bytes: 2^-63 .. 2^63

// j / bs for 0 <= j < 2^32 / bs (checked on the host)
struct Div { uint32_t inv; };
__device__ __forceinline__ int quot(Div d, int j) { return d.inv ? (int)__umulhi((uint32_t)j, d.inv) : j; }

struct Cache {
  uint8_t* kv;
  const int *pos, *slot, *btab;
  int* err;
  int n_blocks, n_slots, max_lb, bs, H, rec;
  Div div;
};

__device__ __forceinline__ uint8_t* record(const Cache& c, int blk, int h) { return c.kv + ((size_t)blk * c.H + h) * c.rec; }
__device__ __forceinline__ void report(int* err) { atomicCAS(err, 0, 8); }
// block of position p of a sequence, or -1 where the position, the sequence or the table's entry is out of range
__device__ __forceinline__ int block_of(const Cache& c, int sl, int p) {
  if (p < 0 || sl < 0 || sl >= c.n_slots) return -1;
  const int lb = quot(c.div, p);
  if (lb >= c.max_lb) return -1;
  const int b = __ldg(c.btab + (size_t)sl * c.max_lb + lb);
  return (unsigned)b < (unsigned)c.n_blocks ? b : -1;
}

__device__ __forceinline__ uint32_t max_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// largest magnitude of eight bf16, as its bits; NaN counts as nothing (max gives the other operand, and NaN for two)
__device__ __forceinline__ uint32_t amax8(const uint4& u) {
  constexpr uint32_t M = 0x7fff7fffu;
  const uint32_t m = max_bf16x2(max_bf16x2(u.x & M, u.y & M), max_bf16x2(u.z & M, u.w & M)), a = m & 0xffffu, b = m >> 16;
  return max(a > 0x7f80u ? 0u : a, b > 0x7f80u ? 0u : b);
}
// exponent byte of a row whose largest magnitude has these bf16 bits: 448 = 1.75 * 2^8
__device__ __forceinline__ uint32_t exp_byte(uint32_t a) {
  const int b = (int)(a >> 7) - 8 + ((a & 0x7fu) > 0x60u);
  return (uint32_t)min(max(b, E_LO), E_HI);
}
// eq of a query row whose largest magnitude has these bf16 bits: q = q' 2^eq with the largest |q'| in [2^14, 2^15).  Both 2^eq and 2^-eq are normal numbers; queries that
// the limit leaves smaller (below 2^-98) have scores below 2^-19 beside any key that the format holds.
__device__ __forceinline__ int q_exponent(uint32_t m) { return m == 0 ? 0 : max((int)(m >> 7) - 127 - 14, -112); }
__device__ __forceinline__ float pow2_of(uint32_t byte) { return __uint_as_float(byte << 23); }
__device__ __forceinline__ uint32_t to_e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint2 encode8(const uint4& u, float inv) {
  const float2 a = unpack_bf16(u.x), b = unpack_bf16(u.y), c = unpack_bf16(u.z), d = unpack_bf16(u.w);
  return make_uint2(to_e4m3x2(a.x * inv, a.y * inv) | to_e4m3x2(b.x * inv, b.y * inv) << 16,
                    to_e4m3x2(c.x * inv, c.y * inv) | to_e4m3x2(d.x * inv, d.y * inv) << 16);
}
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// 2^d of a part of a row, as two factors: references hold exponents of values too, so a part whose values are small may have weight although 2^d is below fp32's range.
struct Weight {
  float a, b;                                      // b = 1 down to 2^-120
  __device__ __forceinline__ explicit Weight(float d) : a(ex2(fmaxf(d, -120.f))), b(ex2(fminf(d + 120.f, 0.f))) {}
  __device__ __forceinline__ float operator*(float x) const { return b * (a * x); }
};
// two codes -> two f16 (exact)
__device__ __forceinline__ uint32_t half2_of(uint32_t codes) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)codes));
  return r;
}
__device__ __forceinline__ f32x2 f32x2_of(uint32_t h) {
  f32x2 r;
  asm("{\n\t.reg .b16 l, h;\n\t.reg .f32 a, b;\n\tmov.b32 {l, h}, %1;\n\tcvt.f32.f16 a, l;\n\tcvt.f32.f16 b, h;\n\tmov.b64 %0, {a, b};\n\t}" : "=l"(r) : "r"(h));
  return r;
}

}  // namespace

// Checks that every entry point makes; fills the kernels' view of the cache.
inline int make_cache(Cache& c, const char* name, const void* kv, int n_blocks, int rec, const void* pos, const void* slot, const void* btab,
                      int n_slots, int max_lb, int bs, int H, int hd) {
  if (hd != 16 && hd != 32 && hd != 64 && hd != 128) { kh_set_error("%s: head dim %d is not supported", name, hd); return -1; }
  if (bs < 1 || H < 1 || H > 65535 || n_blocks < 1 || max_lb < 1 || n_slots < 1) { kh_set_error("%s: empty cache", name); return -1; }
  if (rec < 2 * bs * hd + 2 * bs || rec % 32 || ((uintptr_t)kv & 31)) { kh_set_error("%s: records of %d bytes do not fit block size %d", name, rec, bs); return -1; }
  if ((unsigned long long)max_lb * bs * bs >= 1ull << 32 || (long long)max_lb * bs > 1ll << 30) { kh_set_error("%s: block table of %d x %d positions is too long", name, max_lb, bs); return -1; }
  if ((unsigned long long)n_blocks * H * rec >> 36) { kh_set_error("%s: a cache of %d blocks x %d heads x %d bytes is larger than 64 GB", name, n_blocks, H, rec); return -1; }
  c = Cache{(uint8_t*)kv, (const int*)pos, (const int*)slot, (const int*)btab, kh_error_word_dev(), n_blocks, n_slots, max_lb, bs, H, rec,
            Div{bs == 1 ? 0u : (uint32_t)(((1ull << 32) + bs - 1) / bs)}};
  return 0;
}
namespace {

// One token and head by one warp, a position per HD / 16 lanes at a time, in fp32: for the few rows that the tensor cores' formats do not suit.
// Adds positions first .. first + 31, first + step .. first + step + 31 ... below end to the sums of the lane's group of HD / 16 lanes (o: lane's sixteen dims).
template <int HD>
__device__ __forceinline__ void plain_sums8(const Cache& c, const bf16* row, int h, int sl, float scale, int first, int end, int step, float& m, float& l, f32x2 (&o)[8]) {
  constexpr int LPK = HD / 16, KPW = 32 / LPK;
  constexpr float DOWN = 0x1p-24f, UP = 0x1p24f;   // q 2^-24: a sum of codes times the largest q stays finite
  const int lane = threadIdx.x & 31, g = lane / LPK, e0 = lane % LPK * 16, bs = c.bs;
  f32x2 q[8];
  {
    const uint4 u0 = *reinterpret_cast<const uint4*>(row + e0), u1 = *reinterpret_cast<const uint4*>(row + e0 + 8);
    const uint32_t w[8] = {u0.x, u0.y, u0.z, u0.w, u1.x, u1.y, u1.z, u1.w};
#pragma unroll
    for (int i = 0; i < 8; i++) q[i] = mul2(un2(w[i]), mk2(scale * DOWN, scale * DOWN));
  }
#pragma unroll 1
  for (int j0 = first, k = KPW; j0 < end; j0 += k & 31 ? KPW : step - 32 + KPW, k += KPW) {
    const int j = j0 + g, jj = min(j, end - 1), lb = quot(c.div, jj), at = jj - lb * bs;
    const int b = __ldg(c.btab + (size_t)sl * c.max_lb + lb);
    const uint8_t* rc = record(c, (unsigned)b < (unsigned)c.n_blocks ? b : 0, h);
    const uint4 k4 = *reinterpret_cast<const uint4*>(rc + at * HD + e0), v = *reinterpret_cast<const uint4*>(rc + (bs + at) * HD + e0);
    const uint32_t e = *reinterpret_cast<const uint16_t*>(rc + 2 * bs * HD + 2 * at), kw[4] = {k4.x, k4.y, k4.z, k4.w}, vw[4] = {v.x, v.y, v.z, v.w};
    f32x2 a = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) a = fma2(f32x2_of(half2_of(kw[i >> 1] >> (i & 1) * 16)), q[i], a);
    float s = lo2(a) + hi2(a);
#pragma unroll
    for (int x = LPK / 2; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
    if (j < end) {
      s *= pow2_of(e & 0xffu) * UP;
      const float mn = fmaxf(m, s), ref = mn == -INFINITY ? 0.f : mn, sc = ex2(m - ref), pr = ex2(s - ref), pv = pr * pow2_of(e >> 8);
      m = mn;
      l = fmaf(l, sc, pr);
#pragma unroll
      for (int i = 0; i < 8; i++) o[i] = fma2(f32x2_of(half2_of(vw[i >> 1] >> (i & 1) * 16)), mk2(pv, pv), mul2(o[i], mk2(sc, sc)));
    }
  }
}
// The groups' sums together, in every group.
template <int HD>
__device__ __forceinline__ void plain_join8(float& m, float& l, f32x2 (&o)[8]) {
#pragma unroll
  for (int x = HD / 16; x < 32; x <<= 1) {
    const float m2 = __shfl_xor_sync(0xffffffffu, m, x), l2 = __shfl_xor_sync(0xffffffffu, l, x);
    const float mn = fmaxf(m, m2), ref = mn == -INFINITY ? 0.f : mn, c1 = ex2(m - ref), c2 = ex2(m2 - ref);
    m = mn;
    l = l * c1 + l2 * c2;
#pragma unroll
    for (int i = 0; i < 8; i++) o[i] = fma2(o[i], mk2(c1, c1), mul2((f32x2)__shfl_xor_sync(0xffffffffu, o[i], x), mk2(c2, c2)));
  }
}
// A whole row: positions 0 .. p.
template <int HD>
__device__ __forceinline__ void attend_row8(const Cache& c, const bf16* row, int h, int p, int sl, float scale, bf16* dst) {
  constexpr int LPK = HD / 16;
  const int lane = threadIdx.x & 31;
  float m = -INFINITY, l = 0.f;
  f32x2 o[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  plain_sums8<HD>(c, row, h, sl, scale, 0, p + 1, 32, m, l, o);
  plain_join8<HD>(m, l, o);
  const float inv = 1.f / l;
  if (lane < LPK) {
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 8; i++) w[i] = pack_bf16(lo2(o[i]) * inv, hi2(o[i]) * inv);
    *reinterpret_cast<uint4*>(dst + lane * 16) = make_uint4(w[0], w[1], w[2], w[3]);
    *reinterpret_cast<uint4*>(dst + lane * 16 + 8) = make_uint4(w[4], w[5], w[6], w[7]);
  }
}

}  // namespace
