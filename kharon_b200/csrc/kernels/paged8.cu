// Paged KV cache in 8 bits: keys and values quantised as they are written, read back, and attended to.
//
// Cache of one layer: uint8 [n_blocks, H, record].  The record of a (block, head) is one contiguous piece:
//   bs x hd e4m3 codes of K | bs x hd codes of V | bs pairs of exponent bytes (K, V) | padding to a multiple of 32 bytes,
// so a (sequence, head) reads its pages with consecutive addresses, and a block of all heads is copied as one piece.  A decode step with
// long contexts is bound by these bytes: 2 hd + 2 per position and head where the bf16 cache has 4 hd.
//
// A row x of hd numbers is kept as code_i * 2^e with e = min { e : max |x_i| <= 448 2^e }, -63 <= e <= 63 (448 is e4m3's largest
// number), and code_i = x_i 2^-e rounded to e4m3, nearest even.  The scale is a power of two: x_i 2^-e is exact, so the only
// rounding is the one to e4m3 (half a step, 2^-4 of the value at most, or 2^-10 2^e for values below 2^-6 2^e), and the stored value is exact in bf16.  Magnitudes above 448 2^63
// and infinities become the largest code, NaN stays NaN and does not count for the maximum.
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
static int make_cache(Cache& c, const char* name, const void* kv, int n_blocks, int rec, const void* pos, const void* slot, const void* btab,
                      int n_slots, int max_lb, int bs, int H, int hd) {
  if (hd != 16 && hd != 32 && hd != 64 && hd != 128) { kh_set_error("%s: head dim %d is not supported", name, hd); return -1; }
  if (bs < 1 || H < 1 || H > 65535 || n_blocks < 1 || max_lb < 1 || n_slots < 1) { kh_set_error("%s: empty cache", name); return -1; }
  if (rec < 2 * bs * hd + 2 * bs || rec % 32 || ((uintptr_t)kv & 31)) { kh_set_error("%s: records of %d bytes do not fit block size %d", name, rec, bs); return -1; }
  if ((unsigned long long)max_lb * bs * bs >= 1ull << 32 || (long long)max_lb * bs > 0x7fffffffll) { kh_set_error("%s: block table of %d x %d positions is too long", name, max_lb, bs); return -1; }
  c = Cache{(uint8_t*)kv, (const int*)pos, (const int*)slot, (const int*)btab, kh_error_word_dev(), n_blocks, n_slots, max_lb, bs, H, rec,
            Div{bs == 1 ? 0u : (uint32_t)(((1ull << 32) + bs - 1) / bs)}};
  return 0;
}
extern "C" int kh_kv8_record_bytes(int bs, int hd) { return (2 * bs * hd + 2 * bs + 31) / 32 * 32; }

// ------------------------------------------------------------------------------- append
// A lane per eight elements: HD / 8 lanes of a warp hold one k or v row of a head and find its largest magnitude with shuffles.
template <int HD>
__global__ void __launch_bounds__(256) append_kv8_k(const Cache c, const bf16* __restrict__ qkv, int ld, int ntok) {
  constexpr int LPR = HD / 8;
  pdl_wait();
  pdl_launch_dependents();
  const int per = 2 * c.H * LPR;                                            // lanes of a token
  const long i = (long)blockIdx.x * blockDim.x + threadIdx.x;
  const int t = (int)(i / per), r = (int)(i % per), row = r / LPR, e0 = r % LPR * 8;   // row: heads of k, then heads of v
  const bool live = t < ntok;
  const uint4 u = live ? *reinterpret_cast<const uint4*>(qkv + (size_t)t * ld + c.H * HD + row * HD + e0) : make_uint4(0, 0, 0, 0);
  uint32_t m = amax8(u);
#pragma unroll
  for (int x = LPR / 2; x > 0; x >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, x));
  if (!live) return;
  const int p = c.pos[t], blk = block_of(c, c.slot[t], p);
  if (blk < 0) { report(c.err); return; }                                   // recorded (status code 8), its store skipped
  const int which = row >= c.H, h = row - which * c.H, at = p - quot(c.div, p) * c.bs;
  const uint32_t eb = exp_byte(m);
  uint8_t* rc = record(c, blk, h);
  *reinterpret_cast<uint2*>(rc + ((size_t)which * c.bs + at) * HD + e0) = encode8(u, pow2_of(254u - eb));
  if (e0 == 0) rc[2 * c.bs * HD + 2 * at + which] = (uint8_t)eb;
}
extern "C" int kh_append_kv8(const void* qkv, int ld, void* kv, int n_blocks, int rec, const void* pos, const void* slot, const void* btab,
                             int n_slots, int max_lb, int bs, int H, int hd, int ntok, void* stream) {
  Cache c;
  if (make_cache(c, "append_kv8", kv, n_blocks, rec, pos, slot, btab, n_slots, max_lb, bs, H, hd)) return -1;
  if (((uintptr_t)qkv & 15) || ld % 8 || ld < 3 * H * hd) { kh_set_error("append_kv8: qkv rows must be 16-byte aligned"); return -1; }
  if (ntok <= 0) return 0;
  const long grid = ((long)ntok * 2 * H * (hd / 8) + 255) / 256;
  if (grid > 0x7fffffffl) { kh_set_error("append_kv8: %d tokens are too many", ntok); return -1; }
#define LAUNCH(HD) KH_LAUNCH(append_kv8_k<HD>, (unsigned)grid, 256, 0, stream, c, (const bf16*)qkv, ld, ntok)
  if (hd == 128) LAUNCH(128); else if (hd == 64) LAUNCH(64); else if (hd == 32) LAUNCH(32); else LAUNCH(16);
#undef LAUNCH
  KH_LAUNCH_CHECK("append_kv8");
  return 0;
}

// ------------------------------------------------------------------------------- read back
// A lane per eight elements, as in the append; out [ntok, H * hd] in bf16 (exact) or fp32.
template <int HD, typename T>
__global__ void __launch_bounds__(256) read_kv8_k(const Cache c, T* __restrict__ k, T* __restrict__ v, int ldo, int ntok) {
  constexpr int LPR = HD / 8;
  pdl_wait();
  pdl_launch_dependents();
  const int per = 2 * c.H * LPR;
  const long i = (long)blockIdx.x * blockDim.x + threadIdx.x;
  const int t = (int)(i / per), r = (int)(i % per), row = r / LPR, e0 = r % LPR * 8;
  if (t >= ntok) return;
  const int p = c.pos[t], blk = block_of(c, c.slot[t], p);
  if (blk < 0) { report(c.err); return; }
  const int which = row >= c.H, h = row - which * c.H, at = p - quot(c.div, p) * c.bs;
  const uint8_t* rc = record(c, blk, h);
  const uint2 u = *reinterpret_cast<const uint2*>(rc + ((size_t)which * c.bs + at) * HD + e0);
  const float s = pow2_of(rc[2 * c.bs * HD + 2 * at + which]);
  const f32x2 s2 = mk2(s, s);
  f32x2 x[4];
#pragma unroll
  for (int q = 0; q < 4; q++) x[q] = mul2(f32x2_of(half2_of((q < 2 ? u.x : u.y) >> (q & 1) * 16)), s2);
  T* dst = (which ? v : k) + (size_t)t * ldo + h * HD + e0;
  if constexpr (sizeof(T) == 2) *reinterpret_cast<uint4*>(dst) = make_uint4(pack2(x[0]), pack2(x[1]), pack2(x[2]), pack2(x[3]));
  else {
    *reinterpret_cast<float4*>(dst) = make_float4(lo2(x[0]), hi2(x[0]), lo2(x[1]), hi2(x[1]));
    *reinterpret_cast<float4*>(dst + 4) = make_float4(lo2(x[2]), hi2(x[2]), lo2(x[3]), hi2(x[3]));
  }
}
extern "C" int kh_read_kv8(const void* kv, int n_blocks, int rec, void* k, void* v, int ldo, int f32, const void* pos, const void* slot,
                           const void* btab, int n_slots, int max_lb, int bs, int H, int hd, int ntok, void* stream) {
  Cache c;
  if (make_cache(c, "read_kv8", kv, n_blocks, rec, pos, slot, btab, n_slots, max_lb, bs, H, hd)) return -1;
  if (((uintptr_t)k & 15) || ((uintptr_t)v & 15) || ldo % (f32 ? 4 : 8) || ldo < H * hd) { kh_set_error("read_kv8: rows must be 16-byte aligned"); return -1; }
  if (ntok <= 0) return 0;
  const long grid = ((long)ntok * 2 * H * (hd / 8) + 255) / 256;
  if (grid > 0x7fffffffl) { kh_set_error("read_kv8: %d positions are too many", ntok); return -1; }
#define LAUNCH(HD)                                                                                                      \
  {                                                                                                                     \
    if (f32) KH_LAUNCH((read_kv8_k<HD, float>), (unsigned)grid, 256, 0, stream, c, (float*)k, (float*)v, ldo, ntok);    \
    else KH_LAUNCH((read_kv8_k<HD, bf16>), (unsigned)grid, 256, 0, stream, c, (bf16*)k, (bf16*)v, ldo, ntok);           \
  }
  if (hd == 128) LAUNCH(128) else if (hd == 64) LAUNCH(64) else if (hd == 32) LAUNCH(32) else LAUNCH(16)
#undef LAUNCH
  KH_LAUNCH_CHECK("read_kv8");
  return 0;
}

// ------------------------------------------------------------------------------- single-token attention
// o = sum_j p_j v_j / sum_j p_j, p_j = exp(q k_j / sqrt(hd) - max), over positions j = 0 .. pos of the token's sequence.
// W warps of a CTA and the S CTAs of a cluster share a (token, head).  A position is read by HD / 16 lanes in 16-byte pieces, so a warp holds
// KPW = 512 / HD groups of lanes; it takes chunks of U * KPW consecutive positions, chunk i goes to warp i mod (S W).  Each group keeps a running
// fp32 softmax of its own; the groups are merged once at the end: shuffles in the warp, shared memory in warp order across warps,
// the cluster's shared memory in rank order across CTAs (no scratch in global memory, one launch).  The next chunk's K and V replace the current
// ones in their registers as soon as those are used.
// With `append` != 0 the warp that owns position pos quantises the token's k and v, writes them into the cache and uses what it wrote.
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

__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

}  // namespace

template <int HD, int W>
__global__ void __launch_bounds__(W == 1 ? 128 : 32 * W)
paged_attn8_k(const Cache c, const bf16* __restrict__ qkv, int ld, bf16* __restrict__ out, int ldo, int ntok, float scale, int max_ctx, int append, int S) {
  constexpr int LPK = HD / 16, IPC = W == 1 ? 4 : 1;
  __shared__ float s_part[W > 1 ? W * (HD + 2) : 1], s_cta[HD + 2];       // per warp, per CTA: HD sums, maximum, normaliser
  pdl_wait();
  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, d = c.H * HD;
  const int rank = W > 1 ? (int)(blockIdx.x % S) : 0, t = W > 1 ? (int)(blockIdx.x / S) : (int)blockIdx.x * IPC + warp, h = blockIdx.y;
  const int wi = W > 1 ? rank * W + warp : 0;
  const bool live = t < ntok;
  const int p = live ? c.pos[t] : -1, sl = live ? c.slot[t] : -1;
  // index guard: a context longer than the caller's limit or the block table is recorded (status code 8) and the token skipped
  const bool valid = live && p >= 0 && p < max_ctx && quot(c.div, p) < c.max_lb && sl >= 0 && sl < c.n_slots;      // uniform over the item
  bool bad = live && !valid;
  float m = -INFINITY, l = 0.f;
  f32x2 o[8];
#pragma unroll
  for (int k = 0; k < 8; k++) o[k] = 0;
  if (valid) decode_partial<HD>(c, qkv + (size_t)t * ld + h * HD, d, h, p, sl, scale, wi, W * S, append, m, l, o, bad);
  if (bad) report(c.err);
  if constexpr (W == 1) {
    if (!valid || lane >= LPK) return;
    const float inv = 1.f / l;
    bf16* dst = out + (size_t)t * ldo + h * HD + lane * 16;
    uint32_t w[8];
#pragma unroll
    for (int k = 0; k < 8; k++) w[k] = pack_bf16(lo2(o[k]) * inv, hi2(o[k]) * inv);
    *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
    *reinterpret_cast<uint4*>(dst + 8) = make_uint4(w[4], w[5], w[6], w[7]);
  } else {
    float* part = s_part + warp * (HD + 2);
    if (lane < LPK) {
#pragma unroll
      for (int k = 0; k < 8; k++) { part[lane * 16 + 2 * k] = lo2(o[k]); part[lane * 16 + 2 * k + 1] = hi2(o[k]); }
      if (lane == 0) { part[HD] = m; part[HD + 1] = l; }
    }
    __syncthreads();
    const int tid = threadIdx.x;
    bf16* dst = out + (size_t)t * ldo + h * HD;
    if (tid < HD) {                                                // the CTA's warps, in order
      float mx = -INFINITY, num = 0.f, den = 0.f;
#pragma unroll
      for (int w = 0; w < W; w++) mx = fmaxf(mx, s_part[w * (HD + 2) + HD]);
      const float ref = mx == -INFINITY ? 0.f : mx;
#pragma unroll
      for (int w = 0; w < W; w++) {
        const float f = ex2(s_part[w * (HD + 2) + HD] - ref);
        den += f * s_part[w * (HD + 2) + HD + 1];
        num += f * s_part[w * (HD + 2) + tid];
      }
      if (S == 1) { if (valid) dst[tid] = __float2bfloat16(num / den); }
      else {
        s_cta[tid] = num;
        if (tid == 0) { s_cta[HD] = mx; s_cta[HD + 1] = den; }
      }
    }
    if (S == 1) return;
    __syncwarp();
    cluster_sync_all();
    if (valid && tid < HD / S) {                                   // rank r joins and writes columns [r HD / S, (r + 1) HD / S)
      const int col = rank * (HD / S) + tid;
      const uint32_t base = smem_u32(s_cta);
      float mx = -INFINITY, num = 0.f, den = 0.f, pm[8], pl[8], po[8];
#pragma unroll
      for (int r = 0; r < 8; r++)
        if (r < S) {
          const uint32_t a = mapa_shared(base, r);
          pm[r] = ld_cluster_f32(a + HD * 4);
          pl[r] = ld_cluster_f32(a + (HD + 1) * 4);
          po[r] = ld_cluster_f32(a + col * 4);
        }
#pragma unroll
      for (int r = 0; r < 8; r++)
        if (r < S) mx = fmaxf(mx, pm[r]);
      const float ref = mx == -INFINITY ? 0.f : mx;
#pragma unroll
      for (int r = 0; r < 8; r++)
        if (r < S) {
          const float f = ex2(pm[r] - ref);
          den += f * pl[r];
          num += f * po[r];
        }
      dst[col] = __float2bfloat16(num / den);
    }
    __syncwarp();
    cluster_sync_all();                                            // the others' partials are read until here
  }
}

template <int HD, int W>
static int launch_attn8(const Cache& c, const void* qkv, int ld, void* out, int ldo, int ntok, float scale, int max_ctx, int append, int S, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (kh_pdl_enabled()) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (S > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = S; attr[n].val.clusterDim.y = 1; attr[n++].val.clusterDim.z = 1;
  }
  cfg.gridDim = W == 1 ? dim3((ntok + 3) / 4, c.H) : dim3((unsigned)ntok * S, c.H);
  cfg.blockDim = dim3(W == 1 ? 128 : 32 * W); cfg.stream = st; cfg.attrs = attr; cfg.numAttrs = n;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, paged_attn8_k<HD, W>, c, (const bf16*)qkv, ld, (bf16*)out, ldo, ntok, scale, max_ctx, append, S);
  if (e != cudaSuccess) { cudaGetLastError(); kh_set_error("paged_attn8: %s", cudaGetErrorString(e)); return -1; }
  return 0;
}
extern "C" int kh_paged_attn8(const void* qkv, int ld, void* kv, int n_blocks, int rec, void* out, int ldo, const void* pos, const void* slot,
                              const void* btab, int n_slots, int max_lb, int bs, int H, int hd, float scale, int ntok, int max_ctx, int append, void* stream) {
  Cache c;
  if (make_cache(c, "paged_attn8", kv, n_blocks, rec, pos, slot, btab, n_slots, max_lb, bs, H, hd)) return -1;
  if (((uintptr_t)qkv & 15) || ld % 8 || ld < 3 * H * hd || ((uintptr_t)out & 15) || ldo % 8 || ldo < H * hd) { kh_set_error("paged_attn8: rows must be 16-byte aligned"); return -1; }
  if (ntok <= 0) return 0;
  if (ntok > (1 << 27)) { kh_set_error("paged_attn8: %d tokens are too many", ntok); return -1; }
  const float sl2 = scale * 1.4426950408889634f;
  cudaStream_t st = (cudaStream_t)stream;
  // warps to an item: one where the items alone give every SM some sixteen, else four; sixteen and a cluster of up to eight CTAs where four to an
  // item would still leave the SMs with few bytes in flight, as far as the longest context has a chunk of 2048 / hd positions for each
  const long items = (long)ntok * H, want = 148 * 16;
  const int chunks = (max_ctx + 2048 / hd - 1) / (2048 / hd);
  int W = items >= want || chunks <= 1 ? 1 : items * 4 >= want || chunks <= 4 ? 4 : 16, S = 1;
  while (W > 1 && S < 8 && items * W * S < want && chunks >= 2 * W * S) S *= 2;
#define LAUNCH(HD)                                                                                                      \
  return W == 1 ? launch_attn8<HD, 1>(c, qkv, ld, out, ldo, ntok, sl2, max_ctx, append, 1, st)                          \
       : W == 4 ? launch_attn8<HD, 4>(c, qkv, ld, out, ldo, ntok, sl2, max_ctx, append, S, st)                          \
                : launch_attn8<HD, 16>(c, qkv, ld, out, ldo, ntok, sl2, max_ctx, append, S, st);
  if (hd == 128) { LAUNCH(128) }
  if (hd == 64) { LAUNCH(64) }
  if (hd == 32) { LAUNCH(32) }
  LAUNCH(16)
#undef LAUNCH
}

// ------------------------------------------------------------------------------- attention of pieces of prompts
// CTA = (up to 64 consecutive tokens of a sequence, head), a warp per 16 tokens, mma.sync on K and V tiles of 64 positions that are
// turned into bf16 (exact) on their way into shared memory; fp32 probabilities, which enter P V as three bf16 terms.
namespace {
constexpr int P8_ROWS = 64, P8_MAX_TILES = 1024;
struct Pieces { int row0[P8_MAX_TILES]; uint8_t n[P8_MAX_TILES]; };

__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// x = hi + mid + lo, each bf16 (pairs packed)
__device__ __forceinline__ void terms3(float x, float y, uint32_t& hi, uint32_t& mid, uint32_t& lo) {
  hi = pack_bf16(x, y);
  const float2 h = unpack_bf16(hi);
  mid = pack_bf16(x - h.x, y - h.y);
  const float2 m = unpack_bf16(mid);
  lo = pack_bf16(x - h.x - m.x, y - h.y - m.y);
}
// sixteen codes times s (exact), as bf16
__device__ __forceinline__ void decode16(const uint4& u, float s, uint4& a, uint4& b) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
  const f32x2 s2 = mk2(s, s);
  uint32_t r[8];
#pragma unroll
  for (int i = 0; i < 8; i++) r[i] = pack2(mul2(f32x2_of(half2_of(w[i >> 1] >> (i & 1) * 16)), s2));
  a = make_uint4(r[0], r[1], r[2], r[3]);
  b = make_uint4(r[4], r[5], r[6], r[7]);
}
// One token and head by one warp.
template <int HD>
__device__ __noinline__ void attend_row8(const Cache& c, const bf16* row, int d, int h, int p, int sl, float scale, bf16* dst) {
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

template <int HD>
__global__ void __launch_bounds__(128)
paged_prefill8_k(const __grid_constant__ Pieces tiles, const Cache c, const bf16* __restrict__ qkv, int ld, bf16* __restrict__ out, int ldo, float scale, int max_ctx) {
  constexpr int PITCH = HD * 2 + 16, TILE = P8_ROWS * PITCH, PC = HD / 16, NL = P8_ROWS * PC / 128;     // bytes per row, per tile; 16-code pieces per row, per thread
  extern __shared__ __align__(16) uint8_t smem[];                               // [K, V][64 rows]
  pdl_wait();
  pdl_launch_dependents();
  const uint32_t sK = smem_u32(smem), sV = sK + TILE;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c4 = lane & 3, h = blockIdx.y, d = c.H * HD;
  const int r0 = tiles.row0[blockIdx.x], p0 = c.pos[r0], sl = c.slot[r0];
  int n = tiles.n[blockIdx.x];
  // index guard: tokens beyond the limits are recorded (status code 8) and skipped; they are the last of the run
  const int ok = sl < 0 || sl >= c.n_slots || p0 < 0 ? 0 : (int)min((long)n, min((long)max_ctx, (long)c.max_lb * c.bs) - p0);
  bool bad = ok < n;
  if (bad && tid == 0) report(c.err);
  if (ok <= 0) return;
  n = ok;
  bad = false;
  const int ctx = p0 + n, bs = c.bs;
  const int* bt = c.btab + (size_t)sl * c.max_lb;
  constexpr int NLR = NL > 0 ? NL : 1;
  uint4 kr[NLR], vr[NLR];
  uint32_t er[NLR];
  auto fetch = [&](int kt) {
#pragma unroll
    for (int x = 0; x < NLR; x++) {
      const int i = tid + x * 128, r = i / PC, j = kt * P8_ROWS + r;
      kr[x] = vr[x] = make_uint4(0, 0, 0, 0);
      er[x] = 0;
      if (r < P8_ROWS && j < ctx) {
        const int lb = quot(c.div, j), at = j - lb * bs;
        int b = __ldg(bt + lb);
        if ((unsigned)b >= (unsigned)c.n_blocks) { bad = true; b = 0; }
        const uint8_t* rc = record(c, b, h);
        kr[x] = *reinterpret_cast<const uint4*>(rc + at * HD + i % PC * 16);
        vr[x] = *reinterpret_cast<const uint4*>(rc + (bs + at) * HD + i % PC * 16);
        er[x] = *reinterpret_cast<const uint16_t*>(rc + 2 * bs * HD + 2 * at);
      }
    }
  };
  auto store = [&]() {
#pragma unroll
    for (int x = 0; x < NLR; x++) {
      const int i = tid + x * 128, r = i / PC;
      if (r >= P8_ROWS) continue;
      uint4 a, b;
      uint8_t* at = smem + r * PITCH + i % PC * 32;
      decode16(kr[x], pow2_of(er[x] & 0xffu), a, b);
      *reinterpret_cast<uint4*>(at) = a;
      *reinterpret_cast<uint4*>(at + 16) = b;
      decode16(vr[x], pow2_of(er[x] >> 8), a, b);
      *reinterpret_cast<uint4*>(at + TILE) = a;
      *reinterpret_cast<uint4*>(at + TILE + 16) = b;
    }
  };
  fetch(0);
  const int w0 = warp * 16;                                                     // this warp's first token of the run
  uint4 q[HD / 32][2];                                                          // rows g and g + 8, piece c4 of every 32-wide block
#pragma unroll
  for (int j = 0; j < HD / 32; j++)
#pragma unroll
    for (int i = 0; i < 2; i++) {
      q[j][i] = make_uint4(0, 0, 0, 0);
      if (w0 + g + 8 * i < n) q[j][i] = *reinterpret_cast<const uint4*>(qkv + (size_t)(r0 + w0 + g + 8 * i) * ld + h * HD + j * 32 + c4 * 8);
    }
  float o[HD / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
  for (int t = 0; t < HD / 8; t++)
#pragma unroll
    for (int i = 0; i < 4; i++) o[t][i] = 0.f;
  const int n_kt = (ctx + P8_ROWS - 1) / P8_ROWS;
#pragma unroll 1
  for (int kt = 0; kt < n_kt; kt++) {
    __syncthreads();                                                            // the tile before has been read
    store();
    __syncthreads();
    if (kt + 1 < n_kt) fetch(kt + 1);
    const int k0 = kt * P8_ROWS;
    if (w0 < n && k0 <= p0 + w0 + 15) {                                         // uniform over the warp
      float s[8][4];
#pragma unroll
      for (int t = 0; t < 8; t++) {
#pragma unroll
        for (int i = 0; i < 4; i++) s[t][i] = 0.f;
#pragma unroll
        for (int j = 0; j < HD / 32; j++) {
          uint4 k;
          asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(k.x), "=r"(k.y), "=r"(k.z), "=r"(k.w)
                       : "r"(sK + (t * 8 + g) * PITCH + j * 64 + c4 * 16) : "memory");
          mma_bf16(s[t], q[j][0].x, q[j][1].x, q[j][0].y, q[j][1].y, k.x, k.y);
          mma_bf16(s[t], q[j][0].z, q[j][1].z, q[j][0].w, q[j][1].w, k.z, k.w);
        }
      }
      float mx[2] = {m[0], m[1]};
#pragma unroll
      for (int t = 0; t < 8; t++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
          s[t][i] *= scale;
          if (k0 + t * 8 + c4 * 2 + (i & 1) > p0 + w0 + g + 8 * (i >> 1)) s[t][i] = -INFINITY;
          mx[i >> 1] = fmaxf(mx[i >> 1], s[t][i]);
        }
      float ref[2];
#pragma unroll
      for (int i = 0; i < 2; i++) {
        mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 1));
        mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 2));
        ref[i] = mx[i] == -INFINITY ? 0.f : mx[i];
        const float sc = ex2(m[i] - ref[i]);
        m[i] = mx[i];
        l[i] *= sc;
#pragma unroll
        for (int t = 0; t < HD / 8; t++) { o[t][2 * i] *= sc; o[t][2 * i + 1] *= sc; }
      }
#pragma unroll
      for (int t = 0; t < 8; t++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
          s[t][i] = ex2(s[t][i] - ref[i >> 1]);
          l[i >> 1] += s[t][i];
        }
#pragma unroll
      for (int t = 0; t < 4; t++) {                                             // sixteen keys at a time
        uint32_t hi[4], mid[4], lo[4];
        terms3(s[2 * t][0], s[2 * t][1], hi[0], mid[0], lo[0]);
        terms3(s[2 * t][2], s[2 * t][3], hi[1], mid[1], lo[1]);
        terms3(s[2 * t + 1][0], s[2 * t + 1][1], hi[2], mid[2], lo[2]);
        terms3(s[2 * t + 1][2], s[2 * t + 1][3], hi[3], mid[3], lo[3]);
#pragma unroll
        for (int e = 0; e < HD; e += 16) {
          uint32_t b[4];
          asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(b[0]), "=r"(b[1]), "=r"(b[2]), "=r"(b[3])
                       : "r"(sV + (t * 16 + (lane & 15)) * PITCH + (e + (lane >> 4) * 8) * 2) : "memory");
#pragma unroll
          for (int x = 0; x < 2; x++) {
            mma_bf16(o[e / 8 + x], hi[0], hi[1], hi[2], hi[3], b[2 * x], b[2 * x + 1]);
            mma_bf16(o[e / 8 + x], mid[0], mid[1], mid[2], mid[3], b[2 * x], b[2 * x + 1]);
            mma_bf16(o[e / 8 + x], lo[0], lo[1], lo[2], lo[3], b[2 * x], b[2 * x + 1]);
          }
        }
      }
    }
  }
  if (bad) report(c.err);
  // A NaN in V reaches the rows that see its position and no others.  The products above multiply it with the zeros of masked
  // positions too, which leaves a NaN in every row of the warp: such a warp does its rows anew.
  uint32_t top = 0;
#pragma unroll
  for (int t = 0; t < HD / 8; t++)
#pragma unroll
    for (int i = 0; i < 4; i++) top = max(top, __float_as_uint(o[t][i]) & 0x7fffffffu);
  if (__any_sync(0xffffffffu, top >= 0x7f800000u)) {
#pragma unroll 1
    for (int r = w0; r < min(n, w0 + 16); r++)
      attend_row8<HD>(c, qkv + (size_t)(r0 + r) * ld + h * HD, d, h, p0 + r, sl, scale, out + (size_t)(r0 + r) * ldo + h * HD);
    return;
  }
#pragma unroll
  for (int i = 0; i < 2; i++) {
    l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
    l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
    if (w0 + g + 8 * i < n) {
      const float inv = 1.f / l[i];
      bf16* dst = out + (size_t)(r0 + w0 + g + 8 * i) * ldo + h * HD + c4 * 2;
#pragma unroll
      for (int t = 0; t < HD / 8; t++) *reinterpret_cast<uint32_t*>(dst + t * 8) = pack_bf16(o[t][2 * i] * inv, o[t][2 * i + 1] * inv);
    }
  }
}
// Runs of tokens: `row0`, `len` (host arrays) give each run's first row in qkv / pos / slot / out and its length; the positions of a run
// are consecutive and belong to one sequence, and its K / V are in the cache already.
extern "C" int kh_paged_prefill8(const void* qkv, int ld, const void* kv, int n_blocks, int rec, void* out, int ldo, const void* pos, const void* slot,
                                 const void* btab, int n_slots, int max_lb, int bs, int H, int hd, float scale, int max_ctx, const void* row0,
                                 const void* len, int n_runs, void* stream) {
  Cache c;
  if (make_cache(c, "paged_prefill8", kv, n_blocks, rec, pos, slot, btab, n_slots, max_lb, bs, H, hd)) return -1;
  if (hd == 16) { kh_set_error("paged_prefill8: head dim %d is not supported", hd); return -1; }
  if (((uintptr_t)qkv & 15) || ld % 8 || ld < 3 * H * hd || ((uintptr_t)out & 15) || ldo % 8 || ldo < H * hd) { kh_set_error("paged_prefill8: rows must be 16-byte aligned"); return -1; }
  const float sl2 = scale * 1.4426950408889634f;
  const int smem = 2 * P8_ROWS * (hd * 2 + 16);
  Pieces tiles;
  int nt = 0;
  auto flush = [&]() -> int {
    if (nt == 0) return 0;
#define LAUNCH(HD) KH_LAUNCH(paged_prefill8_k<HD>, dim3(nt, H), 128, smem, stream, tiles, c, (const bf16*)qkv, ld, (bf16*)out, ldo, sl2, max_ctx)
    if (hd == 128) LAUNCH(128); else if (hd == 64) LAUNCH(64); else LAUNCH(32);
#undef LAUNCH
    KH_LAUNCH_CHECK("paged_prefill8");
    nt = 0;
    return 0;
  };
  for (int i = 0; i < n_runs; i++) {
    const int r = ((const int*)row0)[i], n = ((const int*)len)[i];
    if (r < 0 || n < 1) { kh_set_error("paged_prefill8: run %d is empty", i); return -1; }
    for (int at = (n - 1) / P8_ROWS * P8_ROWS; at >= 0; at -= P8_ROWS) {          // the pieces that see the most keys first
      tiles.row0[nt] = r + at;
      tiles.n[nt] = (uint8_t)(n - at < P8_ROWS ? n - at : P8_ROWS);
      if (++nt == P8_MAX_TILES && flush()) return -1;
    }
  }
  return flush();
}

// ------------------------------------------------------------------------------- block copies
// Whole blocks (all heads' records) src -> dst in every layer: the device half of copy-on-write.
__global__ void __launch_bounds__(128) copy_blocks8_k(uint8_t* __restrict__ kv, const int* __restrict__ pairs, size_t block_bytes, size_t layer_bytes,
                                                      int n_blocks, int* err) {
  pdl_wait();
  pdl_launch_dependents();
  const int s = pairs[2 * blockIdx.x], d = pairs[2 * blockIdx.x + 1];
  if ((unsigned)s >= (unsigned)n_blocks || (unsigned)d >= (unsigned)n_blocks) { if (threadIdx.x == 0) report(err); return; }
  const uint4* src = reinterpret_cast<const uint4*>(kv + blockIdx.y * layer_bytes + s * block_bytes);
  uint4* dst = reinterpret_cast<uint4*>(kv + blockIdx.y * layer_bytes + d * block_bytes);
  for (size_t i = threadIdx.x; i < block_bytes / 16; i += blockDim.x) dst[i] = src[i];
}
extern "C" int kh_copy_blocks8(void* kv, const void* pairs, int npairs, int n_layer, int n_blocks, long block_bytes, long layer_bytes, void* stream) {
  if (npairs <= 0 || n_layer <= 0) return 0;
  if (((uintptr_t)kv & 15) || block_bytes % 16 || layer_bytes % 16 || n_layer > 65535) { kh_set_error("copy_blocks8: blocks must be multiples of 16 bytes"); return -1; }
  KH_LAUNCH(copy_blocks8_k, dim3(npairs, n_layer), 128, 0, stream, (uint8_t*)kv, (const int*)pairs, (size_t)block_bytes, (size_t)layer_bytes, n_blocks,
            kh_error_word_dev());
  KH_LAUNCH_CHECK("copy_blocks8");
  return 0;
}
