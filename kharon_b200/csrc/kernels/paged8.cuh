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

// largest magnitude of eight bf16, as its bits; NaN counts as nothing
__device__ __forceinline__ uint32_t amax8(const uint4& u) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const uint32_t a = w[i] & 0x7fffu, b = w[i] >> 16 & 0x7fffu;
    m = max(m, max(a > 0x7f80u ? 0u : a, b > 0x7f80u ? 0u : b));
  }
  return m;
}
// exponent byte of a row whose largest magnitude has these bf16 bits: 448 = 1.75 * 2^8
__device__ __forceinline__ uint32_t exp_byte(uint32_t a) {
  const int b = (int)(a >> 7) - 8 + ((a & 0x7fu) > 0x60u);
  return (uint32_t)min(max(b, E_LO), E_HI);
}
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
  if ((unsigned long long)max_lb * bs * bs >= 1ull << 32 || (long long)max_lb * bs > 0x7fffffffll) { kh_set_error("%s: block table of %d x %d positions is too long", name, max_lb, bs); return -1; }
  c = Cache{(uint8_t*)kv, (const int*)pos, (const int*)slot, (const int*)btab, kh_error_word_dev(), n_blocks, n_slots, max_lb, bs, H, rec,
            Div{bs == 1 ? 0u : (uint32_t)(((1ull << 32) + bs - 1) / bs)}};
  return 0;
}
namespace {

template <int HD>
__device__ __forceinline__ void decode_partial(const Cache& c, const bf16* row, int d, int h, int p, int sl, float scale, int wi, int nw, int append,
                                               float& m, float& l, f32x2 (&o)[8], bool& bad) {
  constexpr int LPK = HD / 16, KPW = 32 / LPK, U = 4, CH = U * KPW;
  const int lane = threadIdx.x & 31, g = lane / LPK, e0 = lane % LPK * 16, bs = c.bs, exps = 2 * bs * HD;
  const int* bt = c.btab + (size_t)sl * c.max_lb;
  const int n = append ? p : p + 1;                // positions read from the cache
  const size_t head = (size_t)h * c.rec, block = (size_t)c.H * c.rec;
  uint4 k4[U], v4[U], kn, vn;
  uint32_t e4[U], en = 0;
  const uint8_t* a4[U];                            // K row of a position; V row and exponents lie at fixed distances
  uint32_t x4[U];
  kn = vn = make_uint4(0, 0, 0, 0);
  auto rows = [&](int j0) {
#pragma unroll
    for (int i = 0; i < U; i++) {
      const int j = j0 + i * KPW;
      if (j < n) {
        const int lb = quot(c.div, j), at = j - lb * bs;
        int b = __ldg(bt + lb);
        if ((unsigned)b >= (unsigned)c.n_blocks) { bad = true; b = 0; }
        const uint8_t* rc = c.kv + (size_t)b * block + head;
        a4[i] = rc + at * HD + e0;
        x4[i] = (uint32_t)(exps + 2 * at) - (uint32_t)(at * HD + e0);
      }
    }
  };
  auto fetch_k = [&](int j0) {
#pragma unroll
    for (int i = 0; i < U; i++)
      if (j0 + i * KPW < n) {
        k4[i] = *reinterpret_cast<const uint4*>(a4[i]);
        e4[i] = *reinterpret_cast<const uint16_t*>(a4[i] + x4[i]);
      }
  };
  auto fetch_v = [&](int j0) {
#pragma unroll
    for (int i = 0; i < U; i++)
      if (j0 + i * KPW < n) v4[i] = *reinterpret_cast<const uint4*>(a4[i] + bs * HD);
  };
  const int step = nw * CH;
  int j0 = wi * CH + g;
  rows(j0);
  fetch_k(j0);
  fetch_v(j0);
  const bool owner = append && (p / CH) % nw == wi;                // uniform over the warp
  if (owner) {
    uint4 s[4];
#pragma unroll
    for (int i = 0; i < 4; i++) s[i] = *reinterpret_cast<const uint4*>(row + d * (1 + i / 2) + e0 + (i & 1) * 8);
    uint32_t mk = max(amax8(s[0]), amax8(s[1])), mv = max(amax8(s[2]), amax8(s[3]));
#pragma unroll
    for (int x = LPK / 2; x > 0; x >>= 1) {
      mk = max(mk, __shfl_xor_sync(0xffffffffu, mk, x));
      mv = max(mv, __shfl_xor_sync(0xffffffffu, mv, x));
    }
    const uint32_t ek = exp_byte(mk), ev = exp_byte(mv);
    const uint2 k0 = encode8(s[0], pow2_of(254u - ek)), k1 = encode8(s[1], pow2_of(254u - ek));
    const uint2 v0 = encode8(s[2], pow2_of(254u - ev)), v1 = encode8(s[3], pow2_of(254u - ev));
    kn = make_uint4(k0.x, k0.y, k1.x, k1.y);
    vn = make_uint4(v0.x, v0.y, v1.x, v1.y);
    en = ek | ev << 8;
    const int b = block_of(c, sl, p);
    if (b < 0) bad = true;
    else if (g == 0) {
      uint8_t* rc = c.kv + (size_t)b * block + head;
      const int at = p - quot(c.div, p) * bs;
      *reinterpret_cast<uint4*>(rc + at * HD + e0) = kn;
      *reinterpret_cast<uint4*>(rc + (bs + at) * HD + e0) = vn;
      if (e0 == 0) *reinterpret_cast<uint16_t*>(rc + exps + 2 * at) = (uint16_t)en;
    }
  }
  f32x2 q[8];
  {
    const uint4 u0 = *reinterpret_cast<const uint4*>(row + e0), u1 = *reinterpret_cast<const uint4*>(row + e0 + 8);
    const uint32_t w[8] = {u0.x, u0.y, u0.z, u0.w, u1.x, u1.y, u1.z, u1.w};
    const f32x2 s2 = mk2(scale, scale);
#pragma unroll
    for (int i = 0; i < 8; i++) q[i] = mul2(un2(w[i]), s2);
  }
  for (; j0 - g <= p; j0 += step) {                                // uniform over the warp
    float s[U];
    uint32_t ev[U];
#pragma unroll
    for (int i = 0; i < U; i++) {
      if (j0 + i * KPW >= n) { k4[i] = kn; v4[i] = vn; e4[i] = en; }        // the appended position, or past the end (masked below)
      const uint32_t w[4] = {k4[i].x, k4[i].y, k4[i].z, k4[i].w};
      f32x2 a = 0, b = 0;
#pragma unroll
      for (int x = 0; x < 4; x++) {
        a = fma2(f32x2_of(half2_of(w[x])), q[2 * x], a);
        b = fma2(f32x2_of(half2_of(w[x] >> 16)), q[2 * x + 1], b);
      }
      a = add2(a, b);
      s[i] = lo2(a) + hi2(a);
      ev[i] = e4[i];
    }
    rows(j0 + step);
    fetch_k(j0 + step);
#pragma unroll
    for (int x = LPK / 2; x > 0; x >>= 1)
#pragma unroll
      for (int i = 0; i < U; i++) s[i] += __shfl_xor_sync(0xffffffffu, s[i], x);
    float mn = m;
#pragma unroll
    for (int i = 0; i < U; i++) {
      s[i] = j0 + i * KPW > p ? -INFINITY : s[i] * pow2_of(ev[i] & 0xffu);
      mn = fmaxf(mn, s[i]);
    }
    const float ref = mn == -INFINITY ? 0.f : mn, sc = ex2(m - ref);
    const f32x2 sc2 = mk2(sc, sc);
    m = mn;
    l *= sc;
#pragma unroll
    for (int x = 0; x < 8; x++) o[x] = mul2(o[x], sc2);
#pragma unroll
    for (int i = 0; i < U; i++) {
      const float pr = ex2(s[i] - ref);
      l += pr;
      const float pv = pr * pow2_of(ev[i] >> 8);
      const f32x2 w2 = mk2(pv, pv);
      if (j0 + i * KPW > p) v4[i] = make_uint4(0, 0, 0, 0);          // (a NaN there would count)
      const uint32_t w[4] = {v4[i].x, v4[i].y, v4[i].z, v4[i].w};
#pragma unroll
      for (int x = 0; x < 4; x++) {
        o[2 * x] = fma2(f32x2_of(half2_of(w[x])), w2, o[2 * x]);
        o[2 * x + 1] = fma2(f32x2_of(half2_of(w[x] >> 16)), w2, o[2 * x + 1]);
      }
    }
    fetch_v(j0 + step);
  }
#pragma unroll
  for (int x = LPK; x < 32; x <<= 1) {                             // merge the lane groups of the warp
    const float m2 = __shfl_xor_sync(0xffffffffu, m, x), l2 = __shfl_xor_sync(0xffffffffu, l, x);
    const float mn = fmaxf(m, m2), ref = mn == -INFINITY ? 0.f : mn;
    const float c1 = ex2(m - ref), c2 = ex2(m2 - ref);
    m = mn;
    l = l * c1 + l2 * c2;
    const f32x2 c1v = mk2(c1, c1), c2v = mk2(c2, c2);
#pragma unroll
    for (int k = 0; k < 8; k++) o[k] = fma2(o[k], c1v, mul2((f32x2)__shfl_xor_sync(0xffffffffu, o[k], x), c2v));
  }
}

// One token and head by one warp.
template <int HD>
__device__ __forceinline__ void attend_row8(const Cache& c, const bf16* row, int d, int h, int p, int sl, float scale, bf16* dst) {
  float m = -INFINITY, l = 0.f;
  f32x2 o[8];
  bool bad = false;
#pragma unroll
  for (int k = 0; k < 8; k++) o[k] = 0;
  decode_partial<HD>(c, row, d, h, p, sl, scale, 0, 1, 0, m, l, o, bad);
  const float inv = 1.f / l;
  const int lane = threadIdx.x & 31;
  if (lane < HD / 16) {
    uint32_t w[8];
#pragma unroll
    for (int k = 0; k < 8; k++) w[k] = pack_bf16(lo2(o[k]) * inv, hi2(o[k]) * inv);
    *reinterpret_cast<uint4*>(dst + lane * 16) = make_uint4(w[0], w[1], w[2], w[3]);
    *reinterpret_cast<uint4*>(dst + lane * 16 + 8) = make_uint4(w[4], w[5], w[6], w[7]);
  }
}
}  // namespace
