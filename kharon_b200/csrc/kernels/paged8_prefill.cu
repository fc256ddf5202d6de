// Attention of runs of new tokens over the 8-bit paged cache (paged8.cu).
#include "paged8.cuh"
#include <stdlib.h>

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
// ------------------------------------------------------------------------------- runs of new tokens on tcgen05
// A work item is (up to 256 consecutive tokens of a run, head).  Warps 0-3 and 4-7 are two groups of one thread per query row, warps 8-11 fetch the
// codes of 128 positions at a time through the block table and turn them into bf16 tiles (exact: four bits of mantissa, a power-of-two
// scale) in the swizzled layout that the tensor core reads, one lane of warp 12 issues every tcgen05.mma:
//   S_w = Q_w K_j^T -> TMEM;  group w: online softmax, P_w -> TMEM over S_w as bf16;  O_w += P_w V_j in TMEM.
// Items of more than 128 tokens: group w has query rows 128 w .. and every key tile.  Items of up to 128: both groups have the same
// rows and alternate key tiles.  While one group works on its scores, the tensor core does the other's products.  The key tiles of an item
// are shared by the S CTAs of a cluster, in contiguous ranges, where the items alone would leave SMs idle.  Groups and CTAs that share
// rows leave (maximum, normaliser, O) in shared memory and join them in a fixed order.
// A row is rescaled only when its maximum grows by more than 2^8 (the older maximum stays the reference of its exponentials).
namespace {
constexpr int CH_ROWS = 256, CH_MAX = 1024, CH_THREADS = 416;
struct Runs { int row0[CH_MAX]; uint16_t n[CH_MAX]; };

template <int HD>
struct Chunk {
  static constexpr int HP = HD < 64 ? 64 : HD;               // columns of a tile in shared memory (slabs of 64)
  static constexpr int TILE = 128 * HP * 2, NS = 2;
  static constexpr int DATA = 2 * TILE + NS * 2 * TILE;      // Q of both groups, NS stages of K and V
  static constexpr int PITCH = HD + 4;                       // floats per row of a group's O when it is shared
  static constexpr int ML = DATA, BARS = ML + 2 * 128 * 8, SMEM = BARS + 256;
  static_assert(2 * 128 * PITCH * 4 <= DATA, "the shared O takes the tiles' place");
};
__device__ __forceinline__ uint32_t tile_chunk(uint32_t base, int row, int ch) {      // 16-byte chunk `ch` of a row of a [128 x HP] tile
  return base + (ch >> 3) * 16384 + row * 128 + (((ch & 7) ^ (row & 7)) << 4);
}
__device__ __forceinline__ void st_shared_16(uint32_t addr, const uint4& v) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ float4 ld_cluster_f32x4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float2 ld_cluster_f32x2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float ld_cluster_1(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void rows_barrier() { asm volatile("bar.sync 1, 256;" ::: "memory"); }      // the two groups
}  // namespace

template <int HD>
__global__ void __launch_bounds__(CH_THREADS, 1)
paged_chunk8_k(const __grid_constant__ Runs runs, const Cache c, const bf16* __restrict__ qkv, int ld, bf16* __restrict__ out, int ldo, float sl2, int max_ctx, int S) {
  using C = Chunk<HD>;
  constexpr int NS = C::NS;
  extern __shared__ __align__(1024) uint8_t chunk_smem[];
  uint8_t* const smem = chunk_smem;
  const uint32_t base = smem_u32(smem), sQ = base, sKV = base + 2 * C::TILE, b0 = base + C::BARS;
  const uint32_t bar_q = b0, bar_kfull = b0 + 8, bar_kfree = bar_kfull + 8 * NS, bar_vfull = bar_kfree + 8 * NS, bar_vfree = bar_vfull + 8 * NS,
                 bar_s = bar_vfree + 8 * NS, bar_p = bar_s + 16, bar_o = bar_p + 16;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + C::BARS + 8 * (1 + 4 * NS + 6));
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::BARS + 8 * (1 + 4 * NS + 6) + 4);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    mbar_init(bar_q, 8);
    for (int s = 0; s < NS; s++) {
      mbar_init(bar_kfull + 8 * s, 4); mbar_init(bar_kfree + 8 * s, 1);
      mbar_init(bar_vfull + 8 * s, 4); mbar_init(bar_vfree + 8 * s, 1);
    }
    for (int w = 0; w < 2; w++) { mbar_init(bar_s + 8 * w, 1); mbar_init(bar_p + 8 * w, 4); mbar_init(bar_o + 8 * w, 1); }
    *abort_flag = (base & 1023u) ? 6 : 0;         // swizzled tiles need the 1024-byte alignment
    if (base & 1023u) atomicCAS(c.err, 0, 6);
    mbar_fence_init();
  }
  if (warp == 12) { tmem_alloc(smem_u32(tmem_slot), 512); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();
  pdl_launch_dependents();

  const int rank = (int)(blockIdx.x % S), item = (int)(blockIdx.x / S), h = item % c.H, piece = item / c.H, d = c.H * HD;
  const int r0 = runs.row0[piece], p0 = c.pos[r0], sl = c.slot[r0], listed = runs.n[piece];
  // index guard: tokens beyond the limits are recorded (status code 8) and skipped; they are the last of the run
  const int ok = sl < 0 || sl >= c.n_slots || p0 < 0 ? 0 : (int)min((long)listed, min((long)max_ctx, (long)c.max_lb * c.bs) - p0);
  if (ok < listed && tid == 0 && rank == 0) report(c.err);
  const int n = max(ok, 0), nq = n > 128 ? 2 : 1, ctx = p0 + n;
  const int tiles = n > 0 ? (ctx + 127) >> 7 : 0, kt0 = (int)((long)tiles * rank / S), kt1 = (int)((long)tiles * (rank + 1) / S);
  const int lim0 = nq == 2 ? (p0 + 128 + 127) >> 7 : tiles;      // key tiles that group 0's rows see
  auto has = [&](int w, int j) { return nq == 2 ? w == 1 || j < lim0 : ((j - kt0) & 1) == w; };
  const bool live = *abort_flag == 0 && n > 0;

  if (warp >= 8 && warp < 12) {
    // ------------------------------------------------------------------ codes -> bf16 tiles
    constexpr int LPR = HD / 16, RPP = 128 / LPR;          // lanes per row, rows per pass; LPR passes per tile
    const int t2 = tid - 256, l = t2 % LPR, r1 = t2 / LPR, bs = c.bs;
    const int* bt = c.btab + (size_t)sl * c.max_lb;
    bool bad = false;
    uint4 kr[LPR], vr[LPR];
    uint32_t er[LPR];
    const uint8_t* ad[LPR];
    auto rows = [&](int j) {
#pragma unroll
      for (int x = 0; x < LPR; x++) {
        const int p = j * 128 + x * RPP + r1;
        ad[x] = nullptr;
        er[x] = 0;
        if (p < ctx) {
          const int lb = quot(c.div, p), at = p - lb * bs;
          int b = __ldg(bt + lb);
          if ((unsigned)b >= (unsigned)c.n_blocks) { bad = true; b = 0; }
          const uint8_t* rc = record(c, b, h);
          ad[x] = rc + at * HD + l * 16;
          er[x] = *reinterpret_cast<const uint16_t*>(rc + 2 * bs * HD + 2 * at);
        }
      }
    };
    auto fetch = [&](uint4 (&r)[LPR], int off) {
#pragma unroll
      for (int x = 0; x < LPR; x++) r[x] = ad[x] ? *reinterpret_cast<const uint4*>(ad[x] + off) : make_uint4(0, 0, 0, 0);
    };
    auto store = [&](const uint4 (&r)[LPR], const uint32_t (&e)[LPR], int sh, uint32_t dst) {
#pragma unroll
      for (int x = 0; x < LPR; x++) {
        uint4 a, b;
        decode16(r[x], pow2_of(e[x] >> sh & 0xffu), a, b);
        const int row = x * RPP + r1, odd = l >> 2 & 1;      // lanes 4-7 of a wide row store their halves the other way round: eight lanes, eight bank groups
        st_shared_16(tile_chunk(dst, row, 2 * l + odd), odd ? b : a);
        st_shared_16(tile_chunk(dst, row, 2 * l + 1 - odd), odd ? a : b);
      }
      fence_proxy_async_smem();
      __syncwarp();
    };
    if (live && kt0 < kt1) {
      rows(kt0);
      fetch(kr, 0);
      fetch(vr, bs * HD);
      for (int j = kt0; j < kt1; j++) {
        const int it = j - kt0, s = it % NS;
        const uint32_t par = ((it / NS) & 1) ^ 1, sk = sKV + s * 2 * C::TILE;
        uint32_t e[LPR];
#pragma unroll
        for (int x = 0; x < LPR; x++) e[x] = er[x];
        if (!mbar_wait(bar_kfree + 8 * s, par, abort_flag, 6, c.err)) break;
        store(kr, e, 0, sk);
        if (lane == 0) mbar_arrive(bar_kfull + 8 * s);
        if (j + 1 < kt1) { rows(j + 1); fetch(kr, 0); }
        if (!mbar_wait(bar_vfree + 8 * s, par, abort_flag, 6, c.err)) break;
        store(vr, e, 8, sk + C::TILE);
        if (lane == 0) mbar_arrive(bar_vfull + 8 * s);
        if (j + 1 < kt1) fetch(vr, bs * HD);
      }
    }
    if (bad) report(c.err);
  } else if (warp == 12) {
    // ------------------------------------------------------------------ MMA issuer
    if (live && elect_one()) {
      constexpr uint32_t idesc_s = umma_idesc_bf16(128, 128, 0, 0), idesc_o = umma_idesc_bf16(128, HD, 0, 1);
      int last[2] = {-1, -1}, np[2] = {0, 0};      // the tile whose P V is due, products P V so far
      bool fine = mbar_wait(bar_q, 0, abort_flag, 6, c.err);
      auto pv = [&](int w) {
        const int it = last[w], s = it % NS, j = kt0 + it;
        if (!mbar_wait(bar_vfull + 8 * s, (it / NS) & 1, abort_flag, 6, c.err) || !mbar_wait(bar_p + 8 * w, np[w] & 1, abort_flag, 6, c.err)) { fine = false; return; }
        tc_fence_after();
        const uint64_t dv = umma_desc_sw128(sKV + s * 2 * C::TILE + C::TILE, 16384, 1024);
#pragma unroll
        for (int kk = 0; kk < 8; kk++)
          umma_f16_ts(tmem + 256 + w * HD, tmem + w * 128 + kk * 8, dv + (uint64_t)((kk * 2048) >> 4), idesc_o, np[w] > 0 || kk > 0);
        np[w]++;
        last[w] = -1;
        if (w == 1 || !has(1, j)) umma_commit(bar_vfree + 8 * s);       // the tile's last reader
      };
      for (int j = kt0; fine && j < kt1; j++) {
        const int it = j - kt0, s = it % NS;
        for (int w = 0; fine && w < 2; w++) {
          if (last[w] >= 0 && (nq == 2 || has(w, j))) pv(w);
          if (!fine || !has(w, j)) continue;
          if (!mbar_wait(bar_kfull + 8 * s, (it / NS) & 1, abort_flag, 6, c.err)) { fine = false; break; }
          tc_fence_after();
          const uint64_t dq = umma_desc_sw128(sQ + (nq == 2 ? w * C::TILE : 0), 16, 1024), dk = umma_desc_sw128(sKV + s * 2 * C::TILE, 16, 1024);
#pragma unroll
          for (int kk = 0; kk < HD / 16; kk++) {
            const uint64_t step = (uint64_t)(((kk >> 2) * 16384 + (kk & 3) * 32) >> 4);
            umma_f16_ss(tmem + w * 128, dq + step, dk + step, idesc_s, kk > 0);
          }
          umma_commit(bar_s + 8 * w);
          if (w == 1 || !has(1, j)) umma_commit(bar_kfree + 8 * s);
          last[w] = it;
        }
      }
      for (int w = 0; fine && w < 2; w++) {
        if (last[w] >= 0) pv(w);
        if (fine && np[w] > 0) umma_commit(bar_o + 8 * w);
      }
    }
    __syncwarp();
  } else if (live) {
    // ------------------------------------------------------------------ query rows
    const int w = warp >> 2, row = tid & 127, lrow = nq == 2 ? tid : row, qpos = p0 + lrow, wpos = qpos - lane;      // wpos: the warp's first row
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16, tS = tmem + w * 128 + lanes, tO = tmem + 256 + w * HD + lanes;
    for (int i = tid; i < nq * 128 * (HD / 8); i += 256) {
      const int r = i / (HD / 8), ch = i % (HD / 8);
      const uint4 u = r < n ? *reinterpret_cast<const uint4*>(qkv + (size_t)(r0 + r) * ld + h * HD + ch * 8) : make_uint4(0, 0, 0, 0);
      st_shared_16(tile_chunk(sQ + (r >> 7) * C::TILE, r & 127, ch), u);
    }
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(bar_q);
    float m = -INFINITY, l = 0.f;                // reference maximum (scaled, log2 units) and normaliser
    int cnt = 0;
    for (int j = kt0; j < kt1; j++) {
      if (!has(w, j)) continue;
      if (!mbar_wait(bar_s + 8 * w, cnt & 1, abort_flag, 6, c.err)) break;
      tc_fence_after();
      const int k0 = j * 128;
      uint32_t r[32], pk[16];
      if (k0 > wpos + 31) {                      // every key comes after the warp's queries
#pragma unroll
        for (int i = 0; i < 16; i++) pk[i] = 0u;
#pragma unroll
        for (int q = 0; q < 4; q++) tmem_st16(tS + q * 16, pk);
      } else {
        const bool edge = k0 + 127 > wpos;       // masks keys after the query
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int q = 0; q < 4; q++) {
          tmem_ld32(tS + q * 32, r);
          tmem_ld_wait();
          if (edge) {
#pragma unroll
            for (int i = 0; i < 32; i++)
              if (k0 + q * 32 + i > qpos) r[i] = 0xff800000u;
          }
#pragma unroll
          for (int i = 0; i < 32; i++) mx[i & 3] = fmaxf(mx[i & 3], __uint_as_float(r[i]));
        }
        const float mt = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * sl2;
        const bool grow = mt > m + 8.f;          // (from -inf too)
        if (cnt > 0 && __any_sync(0xffffffffu, grow)) {       // S_j is there, so P V of the tile before is done: O can be rescaled in place
          const float al = grow ? ex2(m - mt) : 1.f;
#pragma unroll 1
          for (int q = 0; q < HD; q += 32) {
            tmem_ld32(tO + q, r);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; i++) r[i] = __float_as_uint(__uint_as_float(r[i]) * al);
            tmem_st32(tO + q, r);
          }
          l *= al;
        }
        if (grow) m = mt;
        const float ref = m == -INFINITY ? 0.f : m;
        const f32x2 sl = mk2(sl2, sl2), nm = mk2(-ref, -ref);
        f32x2 rs0 = 0, rs1 = 0;
#pragma unroll
        for (int q = 0; q < 4; q++) {
          tmem_ld32(tS + q * 32, r);
          tmem_ld_wait();
          if (edge) {
#pragma unroll
            for (int i = 0; i < 32; i++)
              if (k0 + q * 32 + i > qpos) r[i] = 0xff800000u;
          }
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            const f32x2 e0 = fma2(mk2(__uint_as_float(r[i]), __uint_as_float(r[i + 1])), sl, nm);
            const f32x2 e1 = fma2(mk2(__uint_as_float(r[i + 2]), __uint_as_float(r[i + 3])), sl, nm);
            const f32x2 x0 = mk2(ex2(lo2(e0)), ex2(hi2(e0))), x1 = mk2(ex2(lo2(e1)), ex2(hi2(e1)));
            rs0 = add2(rs0, x0);
            rs1 = add2(rs1, x1);
            pk[i >> 1] = pack2(x0);
            pk[(i >> 1) + 1] = pack2(x1);
          }
          tmem_st16(tS + q * 16, pk);            // over scores that have been read
        }
        l += (lo2(rs0) + hi2(rs0)) + (lo2(rs1) + hi2(rs1));
      }
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_p + 8 * w);
      cnt++;
    }
    if (cnt > 0) mbar_wait(bar_o + 8 * w, 0, abort_flag, 6, c.err);
    tc_fence_after();
    const bool intact = *abort_flag == 0;
    // A NaN in V reaches the rows that see its position and no others.  P V multiplies it with the zeros of masked positions too, which leaves a
    // NaN in every row of the tile: such rows are done anew, one by one.
    if (S == 1 && nq == 2) {
      const float inv = 1.f / l;
      bf16* dst = out + (size_t)(r0 + lrow) * ldo + h * HD;
      uint32_t top = 0;
#pragma unroll 1
      for (int q = 0; q < HD; q += 32) {
        uint32_t r[32];
        tmem_ld32(tO + q, r);
        tmem_ld_wait();
        uint32_t o[16];
#pragma unroll
        for (int i = 0; i < 32; i++) top = max(top, r[i] & 0x7fffffffu);
#pragma unroll
        for (int i = 0; i < 16; i++) o[i] = pack_bf16(__uint_as_float(r[2 * i]) * inv, __uint_as_float(r[2 * i + 1]) * inv);
        if (lrow < n && intact)
#pragma unroll
          for (int i = 0; i < 4; i++) *reinterpret_cast<uint4*>(dst + q + 8 * i) = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
      }
      uint32_t again = __ballot_sync(0xffffffffu, top >= 0x7f800000u && lrow < n && intact);
      while (again) {
        const int i = __ffs(again) - 1;
        again &= again - 1;
        const int t = r0 + lrow - lane + i;
        __syncwarp();
        attend_row8<HD>(c, qkv + (size_t)t * ld + h * HD, d, h, wpos + i, sl, sl2, out + (size_t)t * ldo + h * HD);
      }
    } else {
      rows_barrier();                            // no tile is read any more
      float* part = reinterpret_cast<float*>(smem) + (w * 128 + row) * C::PITCH;
#pragma unroll 1
      for (int q = 0; q < HD; q += 32) {
        uint32_t r[32];
        if (cnt > 0) { tmem_ld32(tO + q, r); tmem_ld_wait(); }
        else {
#pragma unroll
          for (int i = 0; i < 32; i++) r[i] = 0u;
        }
#pragma unroll
        for (int i = 0; i < 32; i += 4)
          *reinterpret_cast<uint4*>(part + q + i) = make_uint4(r[i], r[i + 1], r[i + 2], r[i + 3]);
      }
      *reinterpret_cast<float2*>(smem + C::ML + (w * 128 + row) * 8) = make_float2(m, l);
    }
  }
  // ------------------------------------------------------------------ groups and CTAs that share rows join
  if (S > 1) { __syncwarp(); cluster_sync_all(); }
  if (live && warp < 8 && (S > 1 || nq == 1)) {
    if (S == 1) rows_barrier();
    const int parts = nq == 2 ? S : 2 * S;       // of a row: part i is group i % 2 (or the row's own) of CTA i / 2 (or i)
#pragma unroll 1
    for (int r = rank * 8 + warp; r < n; r += 8 * S) {
      const int row = r & 127;
      auto where = [&](int i) {                  // (CTA, group row) of part i
        const uint32_t off = nq == 2 ? (uint32_t)(r >> 7) * 128 + row : (uint32_t)(i & 1) * 128 + row;
        return make_uint2(S > 1 ? mapa_shared(base, nq == 2 ? i : i >> 1) : base, off);
      };
      float pm = -INFINITY, pl = 0.f;
      if (lane < parts) {
        const uint2 at = where(lane);
        const float2 v = ld_cluster_f32x2(at.x + C::ML + at.y * 8);
        pm = v.x;
        pl = v.y;
      }
      float mx = pm;
#pragma unroll
      for (int x = 8; x > 0; x >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
      const float ref = mx == -INFINITY ? 0.f : mx;
      const float f = ex2(pm - ref);
      float den = f * pl;
#pragma unroll
      for (int x = 8; x > 0; x >>= 1) den += __shfl_xor_sync(0xffffffffu, den, x);
      constexpr int E = HD / 32;
      float o[E];
#pragma unroll
      for (int e = 0; e < E; e++) o[e] = 0.f;
#pragma unroll 4
      for (int i = 0; i < parts; i++) {
        const uint2 at = where(i);
        const uint32_t a = at.x + (at.y * C::PITCH + lane * E) * 4;
        const float fi = __shfl_sync(0xffffffffu, f, i);
        if constexpr (E == 4) { const float4 v = ld_cluster_f32x4(a); o[0] += fi * v.x; o[1] += fi * v.y; o[2] += fi * v.z; o[3] += fi * v.w; }
        else if constexpr (E == 2) { const float2 v = ld_cluster_f32x2(a); o[0] += fi * v.x; o[1] += fi * v.y; }
        else o[0] += fi * ld_cluster_1(a);
      }
      const float inv = 1.f / __shfl_sync(0xffffffffu, den, 0);
      bool nan = false;
#pragma unroll
      for (int e = 0; e < E; e++) nan |= (__float_as_uint(o[e]) & 0x7fffffffu) >= 0x7f800000u;
      if (*abort_flag) break;
      bf16* dst = out + (size_t)(r0 + r) * ldo + h * HD;
      if (__any_sync(0xffffffffu, nan)) attend_row8<HD>(c, qkv + (size_t)(r0 + r) * ld + h * HD, d, h, p0 + r, sl, sl2, dst);
      else if constexpr (E == 4) *reinterpret_cast<uint2*>(dst + lane * 4) = make_uint2(pack_bf16(o[0] * inv, o[1] * inv), pack_bf16(o[2] * inv, o[3] * inv));
      else if constexpr (E == 2) *reinterpret_cast<uint32_t*>(dst + lane * 2) = pack_bf16(o[0] * inv, o[1] * inv);
      else dst[lane] = __float2bfloat16(o[0] * inv);
    }
  }
  if (S > 1) { __syncwarp(); cluster_sync_all(); }          // the others' parts are read until here
  tc_fence_before();
  __syncthreads();
  if (warp == 12) { tc_fence_after(); tmem_dealloc(tmem, 512); }
}

template <int HD>
static int launch_chunks(const Runs& runs, int n_runs, const Cache& c, const bf16* qkv, int ld, bf16* out, int ldo, float sl2, int max_ctx, int S, cudaStream_t st) {
  using C = Chunk<HD>;
  if (cudaFuncSetAttribute(paged_chunk8_k<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM) != cudaSuccess) {
    cudaGetLastError();
    kh_set_error("paged_prefill8: shared memory opt-in failed");
    return -1;
  }
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
  cfg.gridDim = dim3((unsigned)n_runs * c.H * S); cfg.blockDim = dim3(CH_THREADS); cfg.dynamicSmemBytes = C::SMEM; cfg.stream = st; cfg.attrs = attr; cfg.numAttrs = n;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, paged_chunk8_k<HD>, runs, c, qkv, ld, out, ldo, sl2, max_ctx, S);
  if (e != cudaSuccess) { cudaGetLastError(); kh_set_error("paged_prefill8: %s", cudaGetErrorString(e)); return -1; }
  return 0;
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
  static const int force = getenv("KH_CHUNK") ? atoi(getenv("KH_CHUNK")) : 1;
  if (force) {
    Runs runs;
    int nt = 0;
    const int S = getenv("KH_S") ? atoi(getenv("KH_S")) : 1;
    auto flush = [&]() -> int {
      if (nt == 0) return 0;
      const int n = nt;
      nt = 0;
#define LAUNCH(HD) return launch_chunks<HD>(runs, n, c, (const bf16*)qkv, ld, (bf16*)out, ldo, sl2, max_ctx, S, (cudaStream_t)stream);
      if (hd == 128) { LAUNCH(128) }
      if (hd == 64) { LAUNCH(64) }
      LAUNCH(32)
#undef LAUNCH
    };
    for (int i = 0; i < n_runs; i++) {
      const int r = ((const int*)row0)[i], n = ((const int*)len)[i];
      if (r < 0 || n < 1) { kh_set_error("paged_prefill8: run %d is empty", i); return -1; }
      for (int at = (n - 1) / CH_ROWS * CH_ROWS; at >= 0; at -= CH_ROWS) {
        runs.row0[nt] = r + at;
        runs.n[nt] = (uint16_t)(n - at < CH_ROWS ? n - at : CH_ROWS);
        if (++nt == CH_MAX && flush()) return -1;
      }
    }
    return flush();
  }
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
