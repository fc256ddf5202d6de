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
#include "paged8.cuh"

// ------------------------------------------------------------------------------- append and read back
// A lane takes sixteen elements of a k row and of the v row beside it: HD / 16 lanes of a warp hold both and find their largest magnitudes with
// shuffles; the exponents leave as one pair.  The lanes of a token (H HD / 16 of them) lie side by side; a CTA covers 256 of them, of several tokens
// where one has fewer.  Bound by memory: 6018 tokens of 16 heads of 128 appended in 14.6 us (4.5 TB/s), 39800 positions read back in 74.5 us (5.8 TB/s), as fp32 in 183 (4.5).
// With k and v in different lanes (two byte stores for the exponents of a row) 23.6 and 132 us; the largest magnitude element by element instead of by packed
// maxima 17.0; then two or four tokens a lane, fetched together: 16.7 and 80, 21.0 and 81.
namespace {

struct Lanes { int per, tpc; };                      // lanes of a token; tokens side by side in a CTA
// the thread's token and lane of it, or false
__device__ __forceinline__ bool lane_of(const Lanes q, int ntok, int& t, int& r) {
  const int x = q.per <= 256 ? (int)threadIdx.x / q.per : 0;
  r = q.per <= 256 ? (int)threadIdx.x - x * q.per : (int)(blockIdx.y * 256 + threadIdx.x);
  t = (int)blockIdx.x * q.tpc + x;
  return x < q.tpc && r < q.per && t < ntok;
}
static dim3 lanes_grid(int H, int hd, int ntok, Lanes& q) {
  q.per = H * (hd / 16);                             // at most 65535 * 8
  q.tpc = q.per <= 256 ? 256 / q.per : 1;
  return dim3((unsigned)((ntok + q.tpc - 1) / q.tpc), (unsigned)((q.per + 255) / 256));
}

}  // namespace

template <int HD>
__global__ void __launch_bounds__(256) append_kv8_k(const Cache c, const bf16* __restrict__ qkv, int ld, int ntok, const Lanes q) {
  constexpr int LPR = HD / 16;
  pdl_wait();
  pdl_launch_dependents();
  int t, r;
  const bool live = lane_of(q, ntok, t, r);
  const int h = r / LPR, e0 = r % LPR * 16, d = c.H * HD;
  uint4 x[4];                                        // k, k, v, v
  const bf16* src = qkv + (size_t)t * ld + d + h * HD + e0;
#pragma unroll
  for (int i = 0; i < 4; i++) x[i] = live ? *reinterpret_cast<const uint4*>(src + (i >> 1) * d + (i & 1) * 8) : make_uint4(0, 0, 0, 0);
  const int p = live ? c.pos[t] : 0, blk = live ? block_of(c, c.slot[t], p) : -1;
  uint32_t m[2];
#pragma unroll
  for (int i = 0; i < 2; i++) {
    m[i] = max(amax8(x[2 * i]), amax8(x[2 * i + 1]));
#pragma unroll
    for (int y = LPR / 2; y > 0; y >>= 1) m[i] = max(m[i], __shfl_xor_sync(0xffffffffu, m[i], y));
    m[i] = exp_byte(m[i]);
  }
  if (blk < 0) {
    if (live) report(c.err);                         // recorded (status code 8), its store skipped
    return;
  }
  const int at = p - quot(c.div, p) * c.bs;
  uint8_t* rc = record(c, blk, h);
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const float inv = pow2_of(254u - m[i]);
    const uint2 a = encode8(x[2 * i], inv), b = encode8(x[2 * i + 1], inv);
    *reinterpret_cast<uint4*>(rc + ((size_t)i * c.bs + at) * HD + e0) = make_uint4(a.x, a.y, b.x, b.y);
  }
  if (e0 == 0) *reinterpret_cast<uint16_t*>(rc + 2 * c.bs * HD + 2 * at) = (uint16_t)(m[0] | m[1] << 8);
}
extern "C" int kh_append_kv8(const void* qkv, int ld, void* kv, int n_blocks, int rec, const void* pos, const void* slot, const void* btab,
                             int n_slots, int max_lb, int bs, int H, int hd, int ntok, void* stream) {
  Cache c;
  if (make_cache(c, "append_kv8", kv, n_blocks, rec, pos, slot, btab, n_slots, max_lb, bs, H, hd)) return -1;
  if (((uintptr_t)qkv & 15) || ld % 8 || ld < 3 * H * hd) { kh_set_error("append_kv8: qkv rows must be 16-byte aligned"); return -1; }
  if (ntok <= 0) return 0;
  Lanes q;
  const dim3 grid = lanes_grid(H, hd, ntok, q);
#define LAUNCH(HD) KH_LAUNCH(append_kv8_k<HD>, grid, 256, 0, stream, c, (const bf16*)qkv, ld, ntok, q)
  if (hd == 128) LAUNCH(128); else if (hd == 64) LAUNCH(64); else if (hd == 32) LAUNCH(32); else LAUNCH(16);
#undef LAUNCH
  KH_LAUNCH_CHECK("append_kv8");
  return 0;
}

// out [ntok, H * hd] in bf16 (exact) or fp32
template <int HD, typename T>
__global__ void __launch_bounds__(256) read_kv8_k(const Cache c, T* __restrict__ k, T* __restrict__ v, int ldo, int ntok, const Lanes q) {
  constexpr int LPR = HD / 16;
  pdl_wait();
  pdl_launch_dependents();
  int t, r;
  if (!lane_of(q, ntok, t, r)) return;
  const int h = r / LPR, e0 = r % LPR * 16, p = c.pos[t], blk = block_of(c, c.slot[t], p);
  if (blk < 0) { report(c.err); return; }
  const int at = p - quot(c.div, p) * c.bs;
  const uint8_t* rc = record(c, blk, h);
  uint4 x[2];
#pragma unroll
  for (int i = 0; i < 2; i++) x[i] = *reinterpret_cast<const uint4*>(rc + ((size_t)i * c.bs + at) * HD + e0);
  const uint32_t e = *reinterpret_cast<const uint16_t*>(rc + 2 * c.bs * HD + 2 * at);
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const float s = pow2_of(e >> 8 * i & 0xffu);
    const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
    f32x2 y[8];
#pragma unroll
    for (int j = 0; j < 8; j++) y[j] = mul2(f32x2_of(half2_of(w[j >> 1] >> (j & 1) * 16)), mk2(s, s));
    T* dst = (i ? v : k) + (size_t)t * ldo + h * HD + e0;
    if constexpr (sizeof(T) == 2) {
      reinterpret_cast<uint4*>(dst)[0] = make_uint4(pack2(y[0]), pack2(y[1]), pack2(y[2]), pack2(y[3]));
      reinterpret_cast<uint4*>(dst)[1] = make_uint4(pack2(y[4]), pack2(y[5]), pack2(y[6]), pack2(y[7]));
    } else
#pragma unroll
      for (int j = 0; j < 4; j++) reinterpret_cast<float4*>(dst)[j] = make_float4(lo2(y[2 * j]), hi2(y[2 * j]), lo2(y[2 * j + 1]), hi2(y[2 * j + 1]));
  }
}
extern "C" int kh_read_kv8(const void* kv, int n_blocks, int rec, void* k, void* v, int ldo, int f32, const void* pos, const void* slot,
                           const void* btab, int n_slots, int max_lb, int bs, int H, int hd, int ntok, void* stream) {
  Cache c;
  if (make_cache(c, "read_kv8", kv, n_blocks, rec, pos, slot, btab, n_slots, max_lb, bs, H, hd)) return -1;
  if (((uintptr_t)k & 15) || ((uintptr_t)v & 15) || ldo % (f32 ? 4 : 8) || ldo < H * hd) { kh_set_error("read_kv8: rows must be 16-byte aligned"); return -1; }
  if (ntok <= 0) return 0;
  Lanes q;
  const dim3 grid = lanes_grid(H, hd, ntok, q);
#define LAUNCH(HD)                                                                                            \
  {                                                                                                           \
    if (f32) KH_LAUNCH((read_kv8_k<HD, float>), grid, 256, 0, stream, c, (float*)k, (float*)v, ldo, ntok, q); \
    else KH_LAUNCH((read_kv8_k<HD, bf16>), grid, 256, 0, stream, c, (bf16*)k, (bf16*)v, ldo, ntok, q);        \
  }
  if (hd == 128) LAUNCH(128) else if (hd == 64) LAUNCH(64) else if (hd == 32) LAUNCH(32) else LAUNCH(16)
#undef LAUNCH
  KH_LAUNCH_CHECK("read_kv8");
  return 0;
}

// ------------------------------------------------------------------------------- single-token attention
// o = sum_j 2^(s_j) v_j / sum_j 2^(s_j), s_j = q k_j log2(e) / sqrt(hd), over positions j = 0 .. pos of the token's sequence.
//
// A warp takes chunks of 32 consecutive positions; W warps of a CTA and the S CTAs of a cluster share a (token, head), chunk i goes to warp
// i mod (S W).  The products run on mma.sync (f16, fp32 sums), because what bounds a plain loop is not memory but its 4.8 instructions per code (conversion to fp32,
// multiply, reduction): 313 us for 128 sequences of 1000 to 4096 positions, 16 heads of 128.  Codes become f16 with one instruction for two:
//   S:  A = K, B = q in every column: lanes 4 g + i hold 1/4 of the codes of position g of each eight, and get its score;
//   O:  A = V^T, B = P: lanes 4 g + i hold 1/8 of the dims, of positions 2 i, 2 i + 1 of each eight; two positions' codes are interleaved by byte permutation.
// What f16 cannot hold is taken out as powers of two and put back in fp32: q = q' 2^eq (largest |q'| in [2^14, 2^15)), scores times 2^ek, and
// P' = 2^(s + ev - R + 14) with R the running maximum of s + ev, so that V's codes enter as they are.  P' goes in as two f16 terms, in the even and
// the odd columns of B (22 bits; 2^-39 of the largest term): nothing is rounded to fewer bits than a sum of the same length in fp32 as long as the exponents of V
// of positions with weight are not far below the largest, and as q' is exact.  Otherwise (value rows whose sizes differ by 2^10 and more, rows of zeros among them, with the
// weight on the small ones; a query with an element 2^-29 times its largest) the warp takes its positions again, one by one in fp32: 1.2 ms for the 0.225 below, 38 us for the 16.
// A score shares its fp32 number with ev, 63 at most: it is off by 2^-18 of a log2 unit at most.  Scores beyond fp32's range give NaN, as they do in a plain evaluation in fp32.
// The block table and the exponents of a chunk are read by one lane per position and passed on by shuffles; the next chunk's K and V replace the
// current ones in their registers as soon as those are used.
// With `append` != 0 the item's first warp quantises the token's k and v, writes them into the cache and starts its sums with them.
// The warps are merged once at the end: shared memory in warp order, then the cluster's shared memory in rank order (no scratch in global
// memory, one launch).  Bound by memory for wide heads: 128 sequences of 1000 to 4096 positions, 16 heads of 128, 225 us (5.8 TB/s); by
// issue slots and latency for narrower ones (128 sequences of 3000, 16 heads of 64: 149 us, 5.4 TB/s; of 32: 106 us, 3.8 TB/s; of 16: 92 us, 2.3 TB/s); few items by three dependent trips to memory and
// the join (16 heads of 64 at 16300 positions: 16.3 us, 2.1 TB/s).
namespace {

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  return r;
}
// the codes of a word's lower / upper half as two f16
__device__ __forceinline__ void halves(uint32_t w, uint32_t& a, uint32_t& b) {
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}" : "=r"(a), "=r"(b) : "r"(w));
}
// (volatile: the compiler would move loads for the next turn down to their use)
template <int BYTES, int WORDS>
__device__ __forceinline__ void ld_codes(uint32_t (&r)[WORDS], const uint8_t* p) {
  if constexpr (BYTES == 16) asm volatile("ld.global.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "l"(p));
  else if constexpr (BYTES == 8) asm volatile("ld.global.v2.b32 {%0, %1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "l"(p));
  else if constexpr (BYTES == 4) asm volatile("ld.global.b32 %0, [%1];" : "=r"(r[0]) : "l"(p));
  else asm volatile("{\n\t.reg .b16 h;\n\tld.global.b16 h, [%1];\n\tcvt.u32.u16 %0, h;\n\t}" : "=r"(r[0]) : "l"(p));
}
__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

// What a lane notes of its positions, as a minimum: ev, in the upper of two bytes; 0 for a query of which f16 loses bits.
constexpr uint32_t NOTHING = 0xffffu;

// A warp's share of one token and head: R, l (the whole warp's) and o[t] = sums of dims g HD / 8 + t (in every lane of a group of four).
template <int HD>
__device__ __forceinline__ void decode_partial(const Cache& c, const bf16* row, int d, int h, int p, int sl, float scale, int wi, int nw, int append,
                                               float& R, float& l, float (&out)[HD / 8], bool& bad, uint32_t& marks) {
  constexpr int KS = HD == 128 ? 2 : 1, KW = HD / 16 / KS, VW = HD >= 32 ? HD / 32 : 1, NM = HD / 16;       // K: slabs of 64 codes, words per lane; V: words per lane; MMAs across hd
  const int lane = threadIdx.x & 31, g = lane >> 2, i4 = lane & 3, bs = c.bs;
  const int* bt = c.btab + (size_t)sl * c.max_lb;
  const int n = append ? p : p + 1;                // positions read from the cache
  // A lane looks up one position of a chunk (lanes past the end of the context: its last position, or one of the same eight; masked below): its block, two chunks before the
  // chunk's K is fetched; its exponents and its K row (in units of 16 bytes from the cache's start) one chunk before.  No load stands behind a condition:
  // its registers would be copied, and waited for, at once.
  const int step = nw * 32;
  int j0 = wi * 32;
  const bool by8 = bs % 8 == 0;                    // then eight positions from a multiple of eight lie in one record
  const int last = max(n - 1, 0);
  struct Look { int blk, at; };
  auto look = [&](int j0) {
    const int j = min(j0 + lane, by8 ? (last & ~7) + (lane & 7) : last), lb = quot(c.div, j);
    Look k;
    k.at = j - lb * bs;
    asm volatile("ld.global.nc.b32 %0, [%1];" : "=r"(k.blk) : "l"(bt + lb));
    return k;
  };
  uint32_t e_n, ko[4], vo[8];                      // of the next chunk to be fetched: exponents, rows of the positions whose K and V the lane takes
  auto place = [&](Look k) {
    bad |= (unsigned)k.blk >= (unsigned)c.n_blocks;
    const uint32_t rc = ((uint32_t)min((unsigned)k.blk, (unsigned)c.n_blocks - 1) * c.H + h) * (uint32_t)(c.rec >> 4), off = rc + k.at * (HD / 16);
    uint16_t e;
    asm volatile("ld.global.b16 %0, [%1];" : "=h"(e) : "l"(c.kv + (size_t)rc * 16 + 2 * bs * HD + 2 * k.at));
    e_n = e;
    if (by8) {
#pragma unroll
      for (int q = 0; q < 4; q++) {
        const uint32_t first = __shfl_sync(0xffffffffu, off, q * 8);
        ko[q] = first + g * (HD / 16);
        vo[2 * q] = first + 2 * i4 * (HD / 16);
        vo[2 * q + 1] = first + (2 * i4 + 1) * (HD / 16);
      }
    } else {
#pragma unroll
      for (int q = 0; q < 4; q++) {
        ko[q] = __shfl_sync(0xffffffffu, off, q * 8 + g);
        vo[2 * q] = __shfl_sync(0xffffffffu, off, q * 8 + 2 * i4);
        vo[2 * q + 1] = __shfl_sync(0xffffffffu, off, q * 8 + 2 * i4 + 1);
      }
    }
  };
  uint32_t k[4][KS][KW], v[2][4][VW], e;           // [eight positions][slab][word]; [sixteen positions][one of a lane's four][word]; lane's position
  const uint8_t* const kb = c.kv + i4 * KW * 4;
  const uint8_t* const vb = c.kv + bs * HD + g * (HD / 8);
  auto fetch_k = [&]() {
#pragma unroll
    for (int q = 0; q < 4; q++)
#pragma unroll
      for (int s = 0; s < KS; s++) ld_codes<KW * 4>(k[q][s], kb + (size_t)ko[q] * 16 + s * 64);
  };
  auto fetch_v = [&]() {
#pragma unroll
    for (int q = 0; q < 8; q++) ld_codes<HD / 8>(v[q >> 2][q & 3], vb + (size_t)vo[q] * 16);
  };
  Look n0 = look(j0), n1 = look(j0 + step), n2 = look(j0 + 2 * step);
  place(n0);
  fetch_k();
  fetch_v();
  e = e_n;
  // q: lane's dims (of slab s: 64 s + 16 i4 ..; narrower heads: HD / 4 from HD / 4 i4) as f16 pairs, rows alike
  uint32_t qa[NM][2];
  float sc, qf;
  {
    constexpr uint32_t MAG = 0x7fff7fffu, EXP = 0x7c007c00u;
    uint32_t lost = 0;                             // sign bits: an element of q that is not 0, and below f16's normal numbers as q'
    constexpr int PER = HD / 4 / KS;               // dims of a lane and slab
    uint32_t w[KS][PER / 2], m = 0;
#pragma unroll
    for (int s = 0; s < KS; s++)
#pragma unroll
      for (int x = 0; x < PER / 2; x++) {
        w[s][x] = reinterpret_cast<const uint32_t*>(row + s * 64 + i4 * PER)[x];
        const uint32_t a = w[s][x] & 0x7fffu, b = w[s][x] >> 16 & 0x7fffu;
        m = max(m, max(a > 0x7f80u ? 0u : a, b > 0x7f80u ? 0u : b));
      }
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
    const int eq = q_exponent(m);
    qf = pow2_of((uint32_t)(127 - eq));
    sc = scale * pow2_of((uint32_t)(127 + eq));
#pragma unroll
    for (int s = 0; s < KS; s++)
#pragma unroll
      for (int x = 0; x < PER / 2; x++) {
        const float2 a = unpack_bf16(w[s][x]);
        const uint32_t y = pack_f16(a.x * qf, a.y * qf);
        qa[s * (PER / 4) + x / 2][x & 1] = y;
        lost |= ((w[s][x] & MAG) + MAG) & ~((y & EXP) + EXP);
      }
    if (lost & ~MAG) marks = 0;
  }
  float o[NM][4];
#pragma unroll
  for (int t = 0; t < NM; t++)
#pragma unroll
    for (int x = 0; x < 4; x++) o[t][x] = 0.f;
  R = -INFINITY;
  l = 0.f;
  if (append && wi == 0) {
    // the token's own position: lane's HD / 8 dims of q, k, v; groups of eight lanes of the same i4 hold a row
    constexpr int PER = HD / 8;
    uint32_t kw[PER / 2], vw[PER / 2], qw[PER / 2], mk = 0, mv = 0;
    const uint32_t* src = reinterpret_cast<const uint32_t*>(row + g * PER);
#pragma unroll
    for (int x = 0; x < PER / 2; x++) {
      qw[x] = src[x];
      kw[x] = src[d / 2 + x];
      vw[x] = src[d + x];
      const uint32_t a = kw[x] & 0x7fffu, b = kw[x] >> 16 & 0x7fffu, aa = vw[x] & 0x7fffu, bb = vw[x] >> 16 & 0x7fffu;
      mk = max(mk, max(a > 0x7f80u ? 0u : a, b > 0x7f80u ? 0u : b));
      mv = max(mv, max(aa > 0x7f80u ? 0u : aa, bb > 0x7f80u ? 0u : bb));
    }
#pragma unroll
    for (int x = 4; x < 32; x <<= 1) {
      mk = max(mk, __shfl_xor_sync(0xffffffffu, mk, x));
      mv = max(mv, __shfl_xor_sync(0xffffffffu, mv, x));
    }
    const uint32_t ek = exp_byte(mk), ev = exp_byte(mv);
    const float fk = pow2_of(254u - ek), fv = pow2_of(254u - ev);
    uint32_t kc[PER / 2], vc[PER / 2];             // codes, two in a word
    float s = 0.f;
#pragma unroll
    for (int x = 0; x < PER / 2; x++) {
      const float2 a = unpack_bf16(kw[x]), b = unpack_bf16(vw[x]), q = unpack_bf16(qw[x]);
      kc[x] = to_e4m3x2(a.x * fk, a.y * fk);
      vc[x] = to_e4m3x2(b.x * fv, b.y * fv);
      const f32x2 kk = f32x2_of(half2_of(kc[x])), vv = f32x2_of(half2_of(vc[x]));
      s = fmaf(q.x * qf, lo2(kk), fmaf(q.y * qf, hi2(kk), s));
      o[x][0] = lo2(vv) * 16384.f;
      o[x][2] = hi2(vv) * 16384.f;
    }
#pragma unroll
    for (int x = 4; x < 32; x <<= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
    R = fmaf(s, sc * pow2_of(ek), (float)((int)ev - 127));
    l = g == 0 ? 16384.f * fv : 0.f;
    marks = min(marks, ev << 8);
    if (R == -INFINITY) {                          // (an infinity in q: the position has no weight ..
      l = 0.f;
#pragma unroll
      for (int x = 0; x < PER / 2; x++) o[x][0] = o[x][2] = 0.f;
    } else if (!(R < INFINITY)) l = __int_as_float(0x7fffffff);      // .. or all of it, inf - inf; or a NaN in q or k)
    const int b = block_of(c, sl, p);
    if (b < 0) bad = true;
    else {
      uint8_t* rc = record(c, b, h);
      const int a = p - quot(c.div, p) * bs;
      if (i4 < 2) {                                // lanes 0 write k, lanes 1 v
        uint8_t* dst = rc + (size_t)(i4 * bs + a) * HD + g * PER;
        uint32_t cw[PER / 2];
#pragma unroll
        for (int x = 0; x < PER / 2; x++) cw[x] = i4 ? vc[x] : kc[x];
        if constexpr (PER == 16) *reinterpret_cast<uint4*>(dst) = make_uint4(cw[0] | cw[1] << 16, cw[2] | cw[3] << 16, cw[4] | cw[5] << 16, cw[6] | cw[7] << 16);
        else if constexpr (PER == 8) *reinterpret_cast<uint2*>(dst) = make_uint2(cw[0] | cw[1] << 16, cw[2] | cw[3] << 16);
        else if constexpr (PER == 4) *reinterpret_cast<uint32_t*>(dst) = cw[0] | cw[1] << 16;
        else *reinterpret_cast<uint16_t*>(dst) = (uint16_t)cw[0];
      } else if (lane == 2) *reinterpret_cast<uint16_t*>(rc + 2 * bs * HD + 2 * a) = (uint16_t)(ek | ev << 8);
    }
  }
  const uint32_t term = g & 1 ? 0x7632 : 0x5410;   // which f16 of two (first term, second term) words the lane's column of B takes
  place(n1);
#pragma unroll 1
  for (; j0 < n; j0 += step) {                     // uniform over the warp
    if (j0 + lane < n) marks = min(marks, e);
    n1 = n2;
    n2 = look(j0 + 3 * step);
    float s[4];                                    // of positions 8 q + g
#pragma unroll
    for (int x = 0; x < 2; x++) {
      float a[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int t = 0; t < NM; t++) {
        uint32_t a0, a1, a2, a3;
        halves(k[2 * x][t / KW][t % KW], a0, a2);
        halves(k[2 * x + 1][t / KW][t % KW], a1, a3);
        mma_f16(a, a0, a1, a2, a3, qa[t][0], qa[t][1]);
      }
      s[2 * x] = a[0];
      s[2 * x + 1] = a[2];
    }
    fetch_k();
    float nev[4], tm = -INFINITY;                  // 2^-ev
#pragma unroll
    for (int q = 0; q < 4; q++) {
      const uint32_t x = __shfl_sync(0xffffffffu, e, q * 8 + g), ev = x >> 8;
      s[q] = fmaf(s[q], sc * pow2_of(x & 0xffu), (float)((int)ev - 127));      // (both powers first: of opposite size they meet)
      nev[q] = pow2_of(254u - ev);
    }
    if (j0 + 32 > n) {                             // the last chunk: scores past the end are -inf, values zero (a NaN there would count)
#pragma unroll
      for (int q = 0; q < 4; q++) {
        if (j0 + q * 8 + g >= n) { s[q] = -INFINITY; nev[q] = 0.f; }
#pragma unroll
        for (int x = 0; x < 2; x++)
          if (j0 + q * 8 + 2 * i4 + x >= n)
#pragma unroll
            for (int w = 0; w < VW; w++) v[q >> 1][(q & 1) * 2 + x][w] = 0;
      }
    }
#pragma unroll
    for (int q = 0; q < 4; q++) tm = fmaxf(tm, s[q]);
#pragma unroll
    for (int x = 4; x < 32; x <<= 1) tm = fmaxf(tm, __shfl_xor_sync(0xffffffffu, tm, x));
    if (tm > R) {                                  // uniform over the warp
      const float al = ex2(R - tm);
      l *= al;
#pragma unroll
      for (int t = 0; t < NM; t++)
#pragma unroll
        for (int x = 0; x < 4; x++) o[t][x] *= al;
      R = tm;
    }
    const float ref = R == -INFINITY ? 0.f : R;      // (the difference before the 14: of large scores 14 - R is off by whole numbers, and P' would pass f16's end)
    uint32_t pb[4];
#pragma unroll
    for (int x = 0; x < 2; x++) {
      const float p0 = ex2(s[2 * x] - ref + 14.f), p1 = ex2(s[2 * x + 1] - ref + 14.f);
      l = fmaf(p0, nev[2 * x], fmaf(p1, nev[2 * x + 1], l));
      const uint32_t hi = pack_f16(p0, p1);
      const f32x2 hf = f32x2_of(hi);
      const uint32_t lo = pack_f16(p0 - lo2(hf), p1 - hi2(hf)), w0 = __byte_perm(hi, lo, 0x5410), w1 = __byte_perm(hi, lo, 0x7632);
      pb[2 * x] = __byte_perm(__shfl_sync(0xffffffffu, w0, i4 * 8), __shfl_sync(0xffffffffu, w0, i4 * 8 + 4), term);
      pb[2 * x + 1] = __byte_perm(__shfl_sync(0xffffffffu, w1, i4 * 8), __shfl_sync(0xffffffffu, w1, i4 * 8 + 4), term);
    }
#pragma unroll
    for (int q = 0; q < 2; q++)
#pragma unroll
      for (int w = 0; w < VW; w++) {
        // dims 4 w .. of the lane: (position 2 i4, 2 i4 + 1) pairs of each, for the lower and the upper eight positions
        uint32_t x0, x1, x2, x3, y0, y1, y2, y3;
        halves(__byte_perm(v[q][0][w], v[q][1][w], 0x5140), x0, x1);
        halves(__byte_perm(v[q][2][w], v[q][3][w], 0x5140), y0, y1);
        mma_f16(o[2 * w], x0, x1, y0, y1, pb[2 * q], pb[2 * q + 1]);
        if constexpr (HD >= 32) {
          halves(__byte_perm(v[q][0][w], v[q][1][w], 0x7362), x2, x3);
          halves(__byte_perm(v[q][2][w], v[q][3][w], 0x7362), y2, y3);
          mma_f16(o[2 * w + 1], x2, x3, y2, y3, pb[2 * q], pb[2 * q + 1]);
        }
      }
    fetch_v();
    e = e_n;
    place(n1);
  }
#pragma unroll
  for (int x = 4; x < 32; x <<= 1) l += __shfl_xor_sync(0xffffffffu, l, x);
#pragma unroll
  for (int t = 0; t < NM; t++) {
    out[2 * t] = o[t][0] + o[t][1];
    out[2 * t + 1] = o[t][2] + o[t][3];
  }
}

// The same share in fp32, for exponents that f16 does not suit.
template <int HD>
__device__ __forceinline__ void plain_partial(const Cache& c, const bf16* row, int h, int p, int sl, float scale, int wi, int nw, int append, float& R, float& l, float (&out)[HD / 8]) {
  constexpr int PER = HD / 8;
  const int g = (threadIdx.x & 31) >> 2;
  R = -INFINITY;
  l = 0.f;
  f32x2 o[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  plain_sums8<HD>(c, row, h, sl, scale, wi * 32, append ? p : p + 1, nw * 32, R, l, o);
  if (append && wi == 0 && block_of(c, sl, p) >= 0) {       // the token's own position, which this warp has just written
    __syncwarp();
    plain_sums8<HD>(c, row, h, sl, scale, p, p + 1, 32, R, l, o);
  }
  plain_join8<HD>(R, l, o);
  l *= 16384.f;
#pragma unroll
  for (int i = 0; i < 16; i++) {                   // dims g PER .. of the row are a piece of the sixteen that lane g PER / 16 has
    const float y = __shfl_sync(0xffffffffu, i & 1 ? hi2(o[i >> 1]) : lo2(o[i >> 1]), g * PER >> 4) * 16384.f;
    if (i / PER == (g * PER & 15) / PER) out[i % PER] = y;
  }
}

}  // namespace

template <int HD, int W>
__global__ void __launch_bounds__(W == 8 ? 256 : 128, W == 8 ? 2 : HD == 128 ? 3 : 4)
paged_attn8_k(const Cache c, const bf16* __restrict__ qkv, int ld, bf16* __restrict__ out, int ldo, int ntok, float scale, int max_ctx, int append, int S) {
  constexpr int IPC = W == 1 ? 4 : 1, PER = HD / 8;
  __shared__ float s_part[W > 1 ? W * (HD + 2) : 1], s_cta[HD + 2];       // per warp, per CTA: HD sums, reference, normaliser
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
  uint32_t marks = NOTHING;
  float R = -INFINITY, l = 0.f, o[PER];
#pragma unroll
  for (int k = 0; k < PER; k++) o[k] = 0.f;
  if (valid) {
    decode_partial<HD>(c, qkv + (size_t)t * ld + h * HD, d, h, p, sl, scale, wi, W * S, append, R, l, o, bad, marks);
    // 2^-25 in P' moves o by 2^-39 sum |v| 2^-ev over sum 2^(s - R): where that may be more than 2^-29 sum |v|, or is not a number, the warp takes its positions again.
    const uint32_t least = __reduce_min_sync(0xffffffffu, marks);
    if (least != NOTHING && !(l * pow2_of(least >> 8) >= 16.f)) {
      const volatile int* pos = c.pos;             // (read again: seldom used, and not kept in registers for it)
      const volatile int* slot = c.slot;
      if constexpr (W == 1) {                      // (the row's output at once: fewer registers, 7.6 us for 8.1 at 704 heads of 128 and 40 positions)
        __syncwarp();                              // (with `append` the token's own position has just been written)
        attend_row8<HD>(c, qkv + (size_t)t * ld + h * HD, h, pos[t], slot[t], scale, out + (size_t)t * ldo + h * HD);
        if (bad) report(c.err);
        return;
      } else
        plain_partial<HD>(c, qkv + (size_t)t * ld + h * HD, h, pos[t], slot[t], scale, wi, W * S, append, R, l, o);
    }
  }
  if (bad) report(c.err);
  if constexpr (W == 1) {
    if (!valid || (lane & 3)) return;
    const float inv = 1.f / l;
    uint32_t* dst = reinterpret_cast<uint32_t*>(out + (size_t)t * ldo + h * HD + (lane >> 2) * PER);
    uint32_t w[PER / 2];
#pragma unroll
    for (int k = 0; k < PER / 2; k++) w[k] = pack_bf16(o[2 * k] * inv, o[2 * k + 1] * inv);
    if constexpr (PER >= 8)
#pragma unroll
      for (int k = 0; k < PER / 8; k++) reinterpret_cast<uint4*>(dst)[k] = make_uint4(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
    else
#pragma unroll
      for (int k = 0; k < PER / 2; k++) dst[k] = w[k];
  } else {
    float* part = s_part + warp * (HD + 2);
    if ((lane & 3) == 0) {
#pragma unroll
      for (int k = 0; k < PER; k++) part[(lane >> 2) * PER + k] = o[k];
      if (lane == 0) { part[HD] = R; part[HD + 1] = l; }
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
        const Weight f(s_part[w * (HD + 2) + HD] - ref);
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
    if (valid && tid < HD / S) {                                  // rank r joins and writes columns [r HD / S, (r + 1) HD / S)
      const int col = rank * (HD / S) + tid;
      const uint32_t base = smem_u32(s_cta);
      float mx = -INFINITY, num = 0.f, den = 0.f;
#pragma unroll 4
      for (int r = 0; r < S; r++) mx = fmaxf(mx, ld_cluster_f32(mapa_shared(base, r) + HD * 4));
      const float ref = mx == -INFINITY ? 0.f : mx;
#pragma unroll 4
      for (int r = 0; r < S; r++) {
        const uint32_t a = mapa_shared(base, r);
        const Weight f(ld_cluster_f32(a + HD * 4) - ref);
        den += f * ld_cluster_f32(a + (HD + 1) * 4);
        num += f * ld_cluster_f32(a + col * 4);
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
  if (S > 8 && cudaFuncSetAttribute(paged_attn8_k<HD, W>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) {
    cudaGetLastError();
    S = 8;
  }
  if (S > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = S; attr[n].val.clusterDim.y = 1; attr[n++].val.clusterDim.z = 1;
  }
  cfg.gridDim = W == 1 ? dim3((ntok + 3) / 4, c.H) : dim3((unsigned)ntok * S, c.H);
  cfg.blockDim = dim3(W == 8 ? 256 : 128); cfg.stream = st; cfg.attrs = attr; cfg.numAttrs = n;
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
  max_ctx = max_ctx < max_lb * bs ? max_ctx : max_lb * bs;
  if (ntok > (1 << 27)) { kh_set_error("paged_attn8: %d tokens are too many", ntok); return -1; }
  const float sl2 = scale * 1.4426950408889634f;
  cudaStream_t st = (cudaStream_t)stream;
  // One warp to an item or four: by rounds of the warps that the SMs hold (some 3 us each) and chunks of 32 positions per warp (some 1 us each) of the longest
  // context.  us, one / four: 704 heads of 128 at 40 positions 7.0 / 9.9, 2400 of 64 at 60 9.2 / 16.1, at 200 24.8 / 28.8, 512 of 64 at 20 to 1000 34 / 13.
  // Where four leave SMs idle: eight (heads of up to 64; wider ones have no registers for two such CTAs per SM), then a cluster of up to eight CTAs, as
  // long as they fit the chip together (16 warps per SM) and the longest context has a chunk for each warp; sixteen CTAs of four warps for wide heads
  // beyond 8192 positions.  us, warps x CTAs:
  //   16 heads of 64, 16300 positions: 4 x 4 45.6, 4 x 8 21.2, 4 x 16 16.9, 8 x 8 15.8;  4000: 4 x 4 10.9, 8 x 4 7.5, 8 x 8 8.8;  200: 4 x 2 5.0, 8 x 1 3.8
  //   512 heads of 64, 20 to 1000 positions: 4 x 1 12.7, 8 x 1 14.5;  72 at 960: 4 x 4 7.2, 8 x 2 5.7;  256 heads of 32 at 700: 4 x 2 7.5, 8 x 1 5.8
  //   16 heads of 128, 16300: 4 x 8 28.5, 4 x 16 22.8;  64 at 4000: 4 x 8 27.9, 4 x 16 40.7
  const long items = (long)ntok * H;
  const int chunks = (max_ctx + 31) / 32;
  const long held = 148 * (hd == 128 ? 12 : 16);
  auto cost = [&](int w) { return 3 * ((items * w + held - 1) / held) + (chunks + w - 1) / w; };
  int W = cost(1) <= cost(4) ? 1 : 4, S = 1;
  if (W == 4 && hd <= 64 && items * 8 <= 148 * 16 && chunks >= 8) W = 8;
  while (W > 1 && S < (W == 4 ? 16 : 8) && items * W * S * 2 <= 148 * 16 && chunks >= (S == 8 ? 256 : 2 * W * S)) S *= 2;
#define ARGS c, qkv, ld, out, ldo, ntok, sl2, max_ctx, append
#define LAUNCH(HD) return W == 1 ? launch_attn8<HD, 1>(ARGS, 1, st) : W == 4 ? launch_attn8<HD, 4>(ARGS, S, st) : launch_attn8<HD, HD == 128 ? 4 : 8>(ARGS, S, st);
  if (hd == 128) { LAUNCH(128) }
  if (hd == 64) { LAUNCH(64) }
  if (hd == 32) { LAUNCH(32) }
  LAUNCH(16)
#undef LAUNCH
#undef ARGS
}

// ------------------------------------------------------------------------------- block copies
// Whole blocks (all heads' records) src -> dst in every layer: the device half of copy-on-write.  A CTA a block and layer, bound by memory for many pairs: 24 layers, blocks of
// 16 positions and 16 heads of 64, one pair 4.7 us, 256 pairs 72 us (5.7 TB/s).
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
