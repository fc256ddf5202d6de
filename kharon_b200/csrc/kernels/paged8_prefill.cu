// Attention of runs of new tokens over the 8-bit paged cache (paged8.cu).
#include <type_traits>

#include "paged8.cuh"

// ------------------------------------------------------------------------------- short runs
// CTA = (a run of up to 64 tokens, head), a warp per 16 tokens, mma.sync on K and V tiles of 64 positions that are turned into bf16 (exact) on
// their way into shared memory; fp32 probabilities, which enter P V as three bf16 terms.  The key tiles are shared by the S CTAs of a cluster, in
// contiguous ranges, where the runs leave SMs idle.  Bound by the trips to memory of a tile (some 1 us each): few instructions, small tiles and several
// CTAs per SM, where the tcgen05 kernel below has 2 us more to set up (16 heads of 64, us, this / that: a fresh run of 16 3.6 / 6.0, of 64 4.1 / 6.0, thirty of
// 64 9.4 / 14.0).
namespace {
constexpr int P8_ROWS = 64, P8_MAX = 1024;
struct Pieces { int row0[P8_MAX]; uint8_t n[P8_MAX]; };
template <int N>
__device__ __forceinline__ void ld_cluster(uint32_t addr, float (&v)[N]) {
  if constexpr (N == 4) asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]) : "r"(addr) : "memory");
  else if constexpr (N == 2) asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v[0]), "=f"(v[1]) : "r"(addr) : "memory");
  else asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v[0]) : "r"(addr) : "memory");
}

// Joins `parts` partial results of NR rows: (reference, normaliser) at ml, four columns of the sums at data, in the cluster's shared memory.  Four parts
// of all rows are on their way together: a trip takes some 300 cycles.
template <int NR, typename A>
__device__ __forceinline__ void join_parts(int parts, A place, float (&den)[NR], float (&o)[NR][4]) {
  float mx[NR];
#pragma unroll
  for (int k = 0; k < NR; k++) {
    mx[k] = -INFINITY;
    den[k] = 0.f;
#pragma unroll
    for (int e = 0; e < 4; e++) o[k][e] = 0.f;
  }
#pragma unroll 1
  for (int i0 = 0; i0 < parts; i0 += 4) {
    float v[NR][4][2], y[NR][4][4];
#pragma unroll
    for (int k = 0; k < NR; k++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        uint32_t ml, data;
        place(k, min(i0 + i, parts - 1), ml, data);
        ld_cluster(ml, v[k][i]);
        ld_cluster(data, y[k][i]);
      }
#pragma unroll
    for (int k = 0; k < NR; k++) {
      const float m = fmaxf(fmaxf(fmaxf(v[k][0][0], v[k][1][0]), fmaxf(v[k][2][0], v[k][3][0])), mx[k]), ref = m == -INFINITY ? 0.f : m;
      const Weight al(mx[k] - ref);
      mx[k] = m;
      den[k] = al * den[k];
#pragma unroll
      for (int e = 0; e < 4; e++) o[k][e] = al * o[k][e];
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const Weight f(i0 + i < parts ? v[k][i][0] - ref : -INFINITY);
        den[k] += f * v[k][i][1];
#pragma unroll
        for (int e = 0; e < 4; e++) o[k][e] += f * y[k][i][e];
      }
    }
  }
}

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
paged_short8_k(const __grid_constant__ Pieces tiles, const __grid_constant__ Cache c, const bf16* __restrict__ qkv, int ld, bf16* __restrict__ out, int ldo, float scale, int max_ctx, int S) {
  constexpr int PITCH = HD * 2 + 16, TILE = P8_ROWS * PITCH, PC = HD / 16, NL = P8_ROWS * PC / 128;     // bytes per row, per tile; 16-code pieces per row, per thread
  constexpr int OP = HD + 4, ML = P8_ROWS * OP * 4;                             // joining: floats per row of O; where (maximum, normaliser) and the rows to do anew lie
  extern __shared__ __align__(16) uint8_t smem[];                               // [K, V][64 rows]
  pdl_wait();
  pdl_launch_dependents();
  const int rank = (int)(blockIdx.x % S), piece = (int)(blockIdx.x / S);
  const uint32_t sK = smem_u32(smem), sV = sK + TILE;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c4 = lane & 3, h = blockIdx.y;
  const int r0 = tiles.row0[piece], p0 = c.pos[r0], sl = c.slot[r0];
  int n = tiles.n[piece];
  // index guard: tokens beyond the limits are recorded (status code 8) and skipped; they are the last of the run
  const int ok = sl < 0 || sl >= c.n_slots || p0 < 0 ? 0 : (int)min((long)n, min((long)max_ctx, (long)c.max_lb * c.bs) - p0);
  bool bad = ok < n;
  if (bad && tid == 0 && rank == 0) report(c.err);
  if (ok <= 0) return;                                                          // (the whole cluster)
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
  const int n_kt = (ctx + P8_ROWS - 1) / P8_ROWS, kt0 = (int)((long)n_kt * rank / S), kt1 = (int)((long)n_kt * (rank + 1) / S);
  if (kt0 < kt1) fetch(kt0);
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
#pragma unroll 1
  for (int kt = kt0; kt < kt1; kt++) {
    __syncthreads();                                                            // the tile before has been read
    store();
    __syncthreads();
    if (kt + 1 < kt1) fetch(kt + 1);
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
#pragma unroll
  for (int i = 0; i < 2; i++) {
    l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
    l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
  }
  // A NaN in V reaches the rows that see its position and no others.  The products above multiply it with the zeros of masked positions
  // too, which leaves a NaN in every row of the warp: such rows are done anew.
  if (S == 1) {
    uint32_t top = 0;
#pragma unroll
    for (int t = 0; t < HD / 8; t++)
#pragma unroll
      for (int i = 0; i < 4; i++) top = max(top, __float_as_uint(o[t][i]) & 0x7fffffffu);
    if (__any_sync(0xffffffffu, top >= 0x7f800000u)) {
#pragma unroll 1
      for (int r = w0; r < min(n, w0 + 16); r++)
        attend_row8<HD>(c, qkv + (size_t)(r0 + r) * ld + h * HD, h, p0 + r, sl, scale, out + (size_t)(r0 + r) * ldo + h * HD);
      return;
    }
#pragma unroll
    for (int i = 0; i < 2; i++)
      if (w0 + g + 8 * i < n) {
        const float inv = 1.f / l[i];
        bf16* dst = out + (size_t)(r0 + w0 + g + 8 * i) * ldo + h * HD + c4 * 2;
#pragma unroll
        for (int t = 0; t < HD / 8; t++) *reinterpret_cast<uint32_t*>(dst + t * 8) = pack_bf16(o[t][2 * i] * inv, o[t][2 * i + 1] * inv);
      }
    return;
  }
  __syncthreads();                                                              // no tile is read any more
  uint32_t* s_again = reinterpret_cast<uint32_t*>(smem + ML + P8_ROWS * 8);
  if (tid < 2) s_again[tid] = 0;
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const int row = w0 + g + 8 * i;
    float* part = reinterpret_cast<float*>(smem) + row * OP + c4 * 2;
#pragma unroll
    for (int t = 0; t < HD / 8; t++) *reinterpret_cast<float2*>(part + t * 8) = make_float2(o[t][2 * i], o[t][2 * i + 1]);
    if (c4 == 0) *reinterpret_cast<float2*>(smem + ML + row * 8) = make_float2(m[i], l[i]);
  }
  __syncwarp();
  cluster_sync_all();
  constexpr int TPR = HD / 4;                                                   // CTA `rank` joins rows rank, rank + S ...; a thread four columns of a row
  const int ch = tid % TPR;
#pragma unroll 1
  for (int r = rank + tid / TPR * S; r < n; r += 128 / TPR * S) {
    float dens[1], sums[1][4];
    join_parts<1>(S, [&](int, int i, uint32_t& ml, uint32_t& data) {
      const uint32_t a = mapa_shared(sK, i);
      ml = a + ML + r * 8;
      data = a + (r * OP + ch * 4) * 4;
    }, dens, sums);
    const float den = dens[0], (&y)[4] = sums[0];
    const float inv = 1.f / den;
    bool anew = false;
#pragma unroll
    for (int e = 0; e < 4; e++) anew |= (__float_as_uint(y[e]) & 0x7fffffffu) >= 0x7f800000u;
    if (anew) atomicOr(s_again + (r >> 5), 1u << (r & 31));
    else *reinterpret_cast<uint2*>(out + (size_t)(r0 + r) * ldo + h * HD + ch * 4) = make_uint2(pack_bf16(y[0] * inv, y[1] * inv), pack_bf16(y[2] * inv, y[3] * inv));
  }
  __syncwarp();
  cluster_sync_all();                                                           // the others' parts are read until here
#pragma unroll 1
  for (uint32_t m = s_again[warp >> 1] >> (warp & 1) * 16 & 0xffffu; m; m &= m - 1) {
    const int r = w0 + __ffs(m) - 1;
    attend_row8<HD>(c, qkv + (size_t)(r0 + r) * ld + h * HD, h, p0 + r, sl, scale, out + (size_t)(r0 + r) * ldo + h * HD);
  }
}

// ------------------------------------------------------------------------------- runs of new tokens on tcgen05
// A work item is (up to 128 G consecutive tokens of a run, head): G = 2 groups of four warps, one thread per query row, or one group (heads of up to 64,
// two CTAs per SM).  Four more warps fetch the codes of K, 128 positions at a time, through the block table and turn them into f16 tiles in the swizzled
// layout that the tensor core reads, four those of V.  One lane issues the products, half a tile (64 positions) at a time:
//   S_w = Q_w K_j^T -> TMEM;  group w: online softmax, P_w -> TMEM over S_w as f16;  O_w += P_w V_j in TMEM.
// One group, and two with more than 128 tokens: group w has query rows 128 w .. and every key tile.  Two groups, up to 128 tokens: both have the same
// rows and alternate key tiles.  While one group works on its scores, the tensor core does the other's products.  The key tiles of an item are shared
// by the S CTAs of a cluster, in contiguous ranges, where the items alone would leave SMs idle.  Groups and CTAs that share rows leave (reference,
// normaliser, O) in shared memory and join them in a fixed order.
//
// Why f16: a code times a power of two is one conversion and one half2 product for two numbers, where bf16 with its own scale takes five instructions, and
// P keeps 11 bits.  f16 has few exponents, so every power of two that is common to a row or a tile is taken out and put back in fp32:
//   q = q' 2^eq (row; largest |q'| in [2^14, 2^15)),  k = k' 2^(EK - 7),  v = v' 2^(EV - 7)  with EK, EV the tile's largest exponents,
//   P' = 2^(s + EV - R),  O = sum P' v' = 2^(7 - R) sum 2^s v,  l = sum over tiles of 2^(EB - EV) sum P' = 2^(EB - R) sum 2^s,
// where R + 7 is the row's running maximum of (largest score + EV), in log2 units (so the largest P' is 2^7 to 2^15), and EB the first tile's EV.  What f16 rounds:
//   q', k' below 2^-14: off by 2^-25, and by up to 448 * 2^-25 where a key's exponent is more than 31 below the tile's largest: a score by at most HD times
//   q' times that.  From 22 below on (until there k' is exact) the fetching warps note the tile's exponent, and rows for which that bound is more than
//   2^-12 of a log2 unit are done anew in fp32 (typical sizes stay 11 octaves below it, so keys of nearly nothing cost nothing);
//   v' of positions whose exponent is more than 22 below the tile's largest (but for rows of zeros): the item's rows are done anew, one by one, in fp32;
//   P': half a step of 11 bits; below 2^-14, 2^-25, which moves o by 2^-25 sum |v| 2^(EB - EV) / l.  Where that may be more than 2^-9 of the mean |v| (largest scores
//   beside values that are small compared with other tiles') the row is done anew.
// Rows whose |q| |k| may give scores beyond 2^23 (HD 2^15 448 2^7 of the products' units) are done anew too: R is off by more than one half there, which P' would have in its
// exponent, and elements of q' below 2^-14 may be what the score is made of, where a larger one meets zeros.
// A row is rescaled only when R would grow by more than 8 (the older R stays the reference).  A row to be done anew leaves NaN as its normaliser, which passes through every
// join.
//
// Heads of 128 are bound by the tensor core (its operands' trips through shared memory) and the exponentials together, each two thirds of the
// time on the SMs in use: 2048 tokens behind 14300 positions, 16 heads, 273 us (942 TFLOP/s; 128 items on 148 SMs), four turns of 384 to 640 tokens behind 1500 to 4000
// 82.5 us (765).  Narrower heads are bound by the exponentials and by the latency of a tile's way through the roles: eight prompts of 1024 tokens, 16
// heads of 64, 58 us (296 TFLOP/s); short prompts by an item's set-up, some 4 us: six of 403 to 1001 tokens 33.4 us, 1024 (run of 128, head) items 33.5 us.
// Rows done anew cost a warp each over their whole context: all rows of the first example 91 ms, of the second 19, of the prompts 2.
namespace {
constexpr int CH_MAX = 1024;
struct Runs { int row0[CH_MAX]; uint16_t n[CH_MAX]; };

template <int HD, int G>
struct Chunk {
  static constexpr int GW = 4 * G, ROWS = 128 * G, THREADS = ROWS + 384;      // warps of the groups; query rows
  static constexpr int HP = HD < 64 ? 64 : HD;               // columns of a tile in shared memory (slabs of 64)
  static constexpr int TILE = 128 * HP * 2, NS = 2;
  static constexpr int DATA = G * TILE + NS * 2 * TILE;      // Q of the groups, NS stages of K and V
  static constexpr int PITCH = HD + 4;                       // floats per row of a group's O when it is shared
  static constexpr int ML = DATA;                            // (R, normaliser) of the groups' rows
  static constexpr int QE = ML + ROWS * 8;                   // 2^eq of the rows
  static constexpr int ADDR = QE + ROWS * 4;                 // [K, V][2 tiles][128] addresses, then as many factors
  static constexpr int FAC = ADDR + 2 * 2 * 128 * 8;
  static constexpr int WMAX = FAC + 2 * 2 * 128 * 4;            // [K, V][2 tiles][4 warps] largest exponents, of K and of V
  static constexpr int TMAX = WMAX + 2 * 2 * 4 * 4;          // [4 tiles] of the tile
  static constexpr int AGAIN = TMAX + 4 * 4;                 // rows to be done anew, as bits
  static constexpr int BARS = AGAIN + 8 * 4, SMEM = BARS + 8 * (4 * NS + 13) + 16;
  static_assert(G == 1 || ROWS * PITCH * 4 <= DATA, "the shared O takes the tiles' place");
};
__device__ __forceinline__ uint32_t tile_chunk(uint32_t base, int row, int ch) {      // 16-byte chunk `ch` of a row of a [128 x HP] tile
  return base + (ch >> 3) * 16384 + row * 128 + (((ch & 7) ^ (row & 7)) << 4);
}
__device__ __forceinline__ void st_shared_16(uint32_t addr, const uint4& v) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
template <int ID, int N>
__device__ __forceinline__ void named_barrier() { asm volatile("bar.sync %0, %1;" ::"n"(ID), "n"(N) : "memory"); }
__device__ __forceinline__ void pair_barrier(int id) { asm volatile("bar.sync %0, 128;" ::"r"(id) : "memory"); }
__device__ __forceinline__ uint32_t pack_f16(f32x2 v) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi2(v)), "f"(lo2(v)));
  return r;
}
// loads whose value is used a turn later, and which the compiler would move down to that use
__device__ __forceinline__ int ld_early_i32(const int* p) {
  int r;
  asm volatile("ld.global.nc.b32 %0, [%1];" : "=r"(r) : "l"(p));
  return r;
}
__device__ __forceinline__ uint32_t ld_early_u16(const uint8_t* p) {
  uint16_t r;
  asm volatile("ld.global.b16 %0, [%1];" : "=h"(r) : "l"(p));
  return r;
}
__device__ __forceinline__ uint4 ld_early_16(uint64_t p) {
  uint4 r;
  asm volatile("ld.global.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
  return r;
}
// four codes times f (twice in a word), as f16
__device__ __forceinline__ void scale4(uint32_t codes, uint32_t f, uint32_t& a, uint32_t& b) {
  asm("{\n\t.reg .b16 l, h;\n\t.reg .b32 x, y;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 x, l;\n\tcvt.rn.f16x2.e4m3x2 y, h;\n\t"
      "mul.rn.f16x2 %0, x, %3;\n\tmul.rn.f16x2 %1, y, %3;\n\t}" : "=r"(a), "=r"(b) : "r"(codes), "r"(f));
}
// 2^x as f16, for x <= 7
__device__ __forceinline__ uint32_t f16_pow2(int x) { return x >= -14 ? (uint32_t)(x + 15) << 10 : x >= -24 ? 1u << (x + 24) : 0u; }
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// A warp's rows of O times al.
template <int HD>
__device__ __forceinline__ void rescale(uint32_t tO, float al) {
  uint32_t r[16];
#pragma unroll 1
  for (int i = 0; i < HD; i += 16) {
    tmem_ld16(tO + i, r);
    tmem_ld_wait();
#pragma unroll
    for (int k = 0; k < 16; k++) r[k] = __float_as_uint(__uint_as_float(r[k]) * al);
    tmem_st16(tO + i, r);
  }
}
// The MMAs with descriptors given by their low words (the high word is the same for all tiles: groups of 8 rows 1024 bytes apart, 128-byte swizzle).
constexpr uint32_t DESC_HI = 64u | 1u << 14 | 2u << 29;
__device__ __forceinline__ void mma_f16_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tsetp.ne.b32 p, %4, 0;\n\tmov.b64 a, {%1, %5};\n\tmov.b64 b, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}" ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "n"(DESC_HI) : "memory");
}
__device__ __forceinline__ void mma_f16_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\tsetp.ne.b32 p, %4, 0;\n\tmov.b64 b, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}" ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "n"(DESC_HI) : "memory");
}
// f16 x f16 -> fp32
__host__ __device__ constexpr uint32_t idesc_f16(int M, int N, int b_mn_major) {
  return umma_idesc_bf16(M, N, 0, b_mn_major) & ~((1u << 7) | (1u << 10));
}
}  // namespace

template <int HD, int G>
__global__ void __launch_bounds__(Chunk<HD, G>::THREADS, G == 1 ? 2 : 1)
paged_chunk8_k(const __grid_constant__ Runs runs, const __grid_constant__ Cache c, const bf16* __restrict__ qkv, int ld, bf16* __restrict__ out, int ldo, float sl2, int max_ctx, int S) {
  using C = Chunk<HD, G>;
  constexpr int NS = C::NS, GW = C::GW, COLS = G == 1 ? 256 : 512;     // TMEM: 128 columns of scores and HD of O a group
  extern __shared__ __align__(1024) uint8_t chunk_smem[];
  uint8_t* const smem = chunk_smem;
  const uint32_t base = smem_u32(smem), sQ = base, sKV = base + G * C::TILE, b0 = base + C::BARS;
  const uint32_t bar_kfull = b0, bar_kfree = bar_kfull + 8 * NS, bar_vfull = bar_kfree + 8 * NS, bar_vfree = bar_vfull + 8 * NS, bar_s = bar_vfree + 8 * NS, bar_p = bar_s + 32, bar_pv = bar_p + 32, bar_o = bar_pv + 16, bar_q = bar_o + 16;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + C::BARS + 8 * (4 * NS + 13));
  // Rows to be done anew: none (0), all, or those whose q is large beside the keys of a tile with this largest exponent byte (see above).
  constexpr int REDO_ALL = 256;
  int* redo = const_cast<int*>(abort_flag) + 1;
  auto lost = [](int redo, float rq) { return redo >= REDO_ALL || (redo && !(rq * pow2_of(redo - 7) * HD <= 0x1p-11f)); };
  uint32_t* reach = reinterpret_cast<uint32_t*>(redo) + 2;       // of the tiles: largest EK, largest 255 - EV
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::BARS + 8 * (4 * NS + 13) + 8);
  uint32_t* s_again = reinterpret_cast<uint32_t*>(smem + C::AGAIN);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid < 8) s_again[tid] = 0;
  if (warp == 0) { tmem_alloc(smem_u32(tmem_slot), COLS); tmem_relinquish(); }
  // What needs no other kernel's results comes first: barriers, TMEM, the roles' registers.  (Grid: heads times S, pieces; S is a power of two.)
  // What every thread knows alike goes through a shuffle where the compiler is to keep it in uniform registers, which is what tcgen05 instructions take;
  // h for the opposite reason: as a uniform value it made the inner loops spill (heads of 128: 276 us for 271).
  auto uniform = [](int x) { return __shfl_sync(0xffffffffu, x, 0); };
  const int ls = 31 - __clz(S), rank = (int)blockIdx.x & (S - 1), h = uniform((int)blockIdx.x >> ls), piece = (int)blockIdx.y;
  const int r0 = runs.row0[piece], listed = runs.n[piece], nq = G == 2 && listed > 128 ? 2 : 1;
  const bool apart = G == 1 || nq == 2;          // every group has rows of its own
  if (tid == 0) {
    // a stage is read by both groups, or by one of them: with NS = 2 and alternating tiles always by the same.  (The last tile may lack group 0:
    // nothing is fetched over it.)
    static_assert(NS == 2, "stages go with groups");
    for (int s = 0; s < NS; s++) {
      mbar_init(bar_kfull + 8 * s, 4); mbar_init(bar_kfree + 8 * s, nq);
      mbar_init(bar_vfull + 8 * s, 4); mbar_init(bar_vfree + 8 * s, nq);
    }
    for (int i = 0; i < 4; i++) { mbar_init(bar_s + 8 * i, 1); mbar_init(bar_p + 8 * i, 4); }      // [group][half]
    mbar_init(bar_pv, 1); mbar_init(bar_pv + 8, 1); mbar_init(bar_o, 1); mbar_init(bar_o + 8, 1); mbar_init(bar_q, GW);
    *redo = 0;
    *reach = 0;
    *abort_flag = (base & 1023u) ? 6 : 0;         // swizzled tiles need the 1024-byte alignment
    if (base & 1023u) atomicCAS(c.err, 0, 6);
    mbar_fence_init();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_wait();
  pdl_launch_dependents();

  const int p0 = uniform(c.pos[r0]), sl = uniform(c.slot[r0]);
  // index guard: tokens beyond the limits are recorded (status code 8) and skipped; they are the last of the run
  const int n = sl < 0 || sl >= c.n_slots || p0 < 0 ? 0 : max(0, min(listed, max_ctx - p0)), ctx = p0 + n;
  if (n < listed && tid == 0 && rank == 0) report(c.err);
  const int tiles = n > 0 ? (ctx + 127) >> 7 : 0, kt0 = tiles * rank >> ls, kt1 = tiles * (rank + 1) >> ls;
  // tiles of group w: all, where it has its own rows (the first of two groups maybe without the last one); every second, where both have the same
  const int lim0 = min(kt1, (p0 + 128 + 127) >> 7);
  auto tiles_of = [&](int w) { return w >= G ? 0 : apart ? max(0, (w ? kt1 : lim0) - kt0) : (kt1 - kt0 + 1 - w) >> 1; };
  const uint32_t tmem = (uint32_t)uniform((int)*tmem_slot);
  const bool live = *abort_flag == 0 && n > 0;
  // After a wait that ran out the roles go through their loops without waiting, so that the named barriers match and the kernel ends.
  bool dead = false;
  auto wait = [&](uint32_t bar, uint32_t parity) { if (!dead && !mbar_wait(bar, parity, abort_flag, 6, c.err)) dead = true; };

  // 640 threads of 96 registers: 128 to the groups, 80 to the fetching warps, 64 to the rest; 512 of 64: 128, 48 and 32.  What follows a role's loop
  // stays in its branch.
  if (warp < GW) asm volatile("setmaxnreg.inc.sync.aligned.u32 128;");
  else if (warp < GW + 8) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(G == 1 ? 48 : 80));
  else asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(G == 1 ? 32 : 64));

  if (warp >= GW + 8) {
    // ------------------------------------------------------------------ MMA issuer
    if (warp == GW + 8 && live && elect_one()) {
      constexpr uint32_t idesc_s = idesc_f16(128, 64, 0), idesc_o = idesc_f16(128, HD, 1);
      const int tiles_w[2] = {tiles_of(0), tiles_of(1)};
      const uint32_t dq0 = (uint32_t)umma_desc_sw128(sQ, 16, 1024), dk0 = (uint32_t)umma_desc_sw128(sKV, 16, 1024), dv0 = (uint32_t)umma_desc_sw128(sKV + C::TILE, 16384, 1024);
      auto scores = [&](int w, int half, int t) {          // S of half a tile, the group's t-th
        const int it = apart ? t : 2 * t + w, s = it & 1;
        if (half == 0) wait(bar_kfull + 8 * s, (it / NS) & 1);
        if (dead) return;
        tc_fence_after();
        const uint32_t dq = dq0 + (nq == 2 && w ? C::TILE >> 4 : 0), dk = dk0 + s * (2 * C::TILE >> 4) + half * 512;
#pragma unroll
        for (int kk = 0; kk < HD / 16; kk++) {
          const uint32_t step = ((kk >> 2) * 16384 + (kk & 3) * 32) >> 4;
          mma_f16_ss(tmem + w * 128 + half * 64, dq + step, dk + step, idesc_s, kk > 0);
        }
        umma_commit(bar_s + 16 * w + 8 * half);
        if (half) umma_commit(bar_kfree + 8 * s);
      };
      wait(bar_q, 0);
#pragma unroll
      for (int i = 0; i < 4; i++)
        if (tiles_w[i & 1] > 0) scores(i & 1, i >> 1, 0);
      const int most = max(tiles_w[0], tiles_w[1]);
#pragma unroll 1
      for (int t = 0; t < most; t++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const int w = i & 1, half = i >> 1;
          if (t >= tiles_w[w]) continue;
          const int it = apart ? t : 2 * t + w, s = it & 1;
          if (half == 0) wait(bar_vfull + 8 * s, (it / NS) & 1);
          wait(bar_p + 16 * w + 8 * half, t & 1);
          if (dead) continue;
          tc_fence_after();
          const uint32_t dv = dv0 + s * (2 * C::TILE >> 4) + half * 512;
#pragma unroll
          for (int kk = 0; kk < 4; kk++)
            mma_f16_ts(tmem + 128 * G + w * HD, tmem + w * 128 + half * 64 + kk * 8, dv + (kk * 2048 >> 4), idesc_o, half > 0 || kk > 0 ? 1 : t > 0);
          umma_commit(half && t + 1 == tiles_w[w] ? bar_o + 8 * w : bar_pv + 8 * w);
          if (half) umma_commit(bar_vfree + 8 * s);
          if (t + 1 < tiles_w[w]) scores(w, half, t + 1);      // behind P V in the tensor core: these scores take P's place
        }
    }
    __syncwarp();
    if (G == 2 && S > 1) { cluster_sync_all(); cluster_sync_all(); }
  } else if (warp >= GW) {
    // ------------------------------------------------------------------ codes -> f16 tiles: K by four warps, V by four
    // A lane takes 16 codes (two 16-byte chunks of a tile) at a time; LPR lanes cover a row of a slab, so eight lanes of a store lie in rows whose
    // numbers differ in the lowest bit, i.e. in eight bank groups.
    constexpr int LPR = HD < 64 ? HD / 16 : 4, RPP = 128 / LPR, SLABS = HD / (16 * LPR), NP = 128 / RPP * SLABS;
    const int vr = warp >= GW + 4, t = tid & 127, l = t % LPR, r1 = t / LPR, bs = c.bs;
    const uint32_t full = vr ? bar_vfull : bar_kfull, free = vr ? bar_vfree : bar_kfree;
    const int* bt = c.btab + (size_t)sl * c.max_lb;
    uint64_t* s_addr = reinterpret_cast<uint64_t*>(smem + C::ADDR) + vr * 256;
    uint32_t* s_fac = reinterpret_cast<uint32_t*>(smem + C::FAC) + vr * 256;
    uint32_t* s_tmax = reinterpret_cast<uint32_t*>(smem + C::TMAX);
    const uint32_t off0 = tile_chunk(0, r1, 2 * l);
    uint32_t* s_wmax = reinterpret_cast<uint32_t*>(smem + C::WMAX) + vr * 8;
    bool bad = false;
    // A thread looks up one position of a tile (t of 128; past the end of the context: its last position, with a factor of zero): block two tiles ahead,
    // exponents one tile ahead, and passes address and exponent on.  No loaded value is looked at before the next turn, and no load stands
    // behind a condition: its registers would be copied, and waited for, at once.
    int blk, blk_at;
    uint32_t e_next = 0, e_now = 0;
    uint64_t a_next = 0;
    auto look = [&](int j) {                               // block of position 128 j + t
      const int p = min(j * 128 + t, ctx - 1), lb = quot(c.div, p);
      blk_at = p - lb * bs;
      blk = ld_early_i32(bt + lb);
    };
    auto exponent = [&]() {                                // ... its address and exponents
      bad |= (unsigned)blk >= (unsigned)c.n_blocks;
      const uint8_t* rc = record(c, (int)min((unsigned)blk, (unsigned)c.n_blocks - 1), h);
      e_next = ld_early_u16(rc + 2 * bs * HD + 2 * blk_at);
      a_next = (uint64_t)(rc + (vr * bs + blk_at) * HD);
    };
    uint4 x[NP];
    auto publish = [&](int b) {                            // tile -> buffer b; then its codes are on their way
      s_addr[b * 128 + t] = a_next;
      pair_barrier(4 + vr);
#pragma unroll
      for (int i = 0; i < NP / SLABS; i++) {
        const uint64_t a = s_addr[b * 128 + i * RPP + r1] + l * 16;
#pragma unroll
        for (int q = 0; q < SLABS; q++) x[i * SLABS + q] = ld_early_16(a + q * 64);
      }
      e_now = e_next;
    };
    auto any_code = [&](uint64_t row) {                    // rows of the smallest exponent: whether it holds numbers or zeros
      uint32_t any = 0;
#pragma unroll 1
      for (int i = 0; i < HD; i += 16) {
        const uint4 w = ld_early_16(row + i);
        any |= (w.x | w.y | w.z | w.w) & 0x7f7f7f7fu;
      }
      return any != 0;
    };
    auto factors = [&](int b, int it) {                    // 2^(e - E + 7) of its positions, E the tile's largest exponent
      if ((kt0 + it) * 128 + t >= ctx) e_now = 0;
      const uint32_t mk = __reduce_max_sync(0xffffffffu, e_now & 0xffu), mv = __reduce_max_sync(0xffffffffu, e_now >> 8);
      if (lane == 0) s_wmax[b * 4 + (warp & 3)] = mk | mv << 16;
      pair_barrier(4 + vr);
      const uint32_t tops = __vmaxu2(__vmaxu2(s_wmax[b * 4], s_wmax[b * 4 + 1]), __vmaxu2(s_wmax[b * 4 + 2], s_wmax[b * 4 + 3]));
      const int e = (int)(e_now >> 8 * vr & 0xffu), off = e - (int)(tops >> 16 * vr & 0xffffu);
      if (off < -22 && e > 0) {                            // (e: 0 past the end)
        if (!vr) atomicMax(redo, (int)(tops & 0xffffu));
        else if (e > E_LO || any_code(s_addr[b * 128 + t])) atomicMax(redo, REDO_ALL);
      }
      s_fac[b * 128 + t] = f16_pow2(off + 7) * 0x10001u;
      // K's warps tell the groups both exponents: scores that are there have passed bar_kfull.  (Of four slots this one was last read for the tile
      // four before, whose scores both groups have used: K's stage of the tile two before this one has been freed.)
      if (t == 0 && !vr) s_tmax[it & 3] = tops;
      pair_barrier(4 + vr);
      if (t == 0 && !vr) *reach = __vmaxu2(*reach, (tops & 0xffffu) | (255u - (tops >> 16)) << 16);
    };
    if (live && kt0 < kt1) {
      look(kt0);
      exponent();
      look(kt0 + 1);
      publish(0);
      exponent();
      look(kt0 + 2);
      for (int j = kt0; j < kt1; j++) {
        const int it = j - kt0, s = it % NS, b = it & 1;
        wait(free + 8 * s, ((it / NS) & 1) ^ 1);
        factors(b, it);
        // chunks 2 l and 2 l + 1 of rows r1, r1 + RPP ...: RPP is a multiple of 8, the swizzle is the same for all of them
        const uint32_t dst0 = sKV + s * 2 * C::TILE + vr * C::TILE + off0, dst1 = dst0 ^ 16u;
#pragma unroll
        for (int i = 0; i < NP / SLABS; i++) {
          const uint32_t f = s_fac[b * 128 + i * RPP + r1];
#pragma unroll
          for (int q = 0; q < SLABS; q++) {
            const uint4 w = x[i * SLABS + q];
            uint4 u, v;
            scale4(w.x, f, u.x, u.y);
            scale4(w.y, f, u.z, u.w);
            scale4(w.z, f, v.x, v.y);
            scale4(w.w, f, v.z, v.w);
            st_shared_16(dst0 + i * RPP * 128 + q * 16384, u);
            st_shared_16(dst1 + i * RPP * 128 + q * 16384, v);
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(full + 8 * s);
        publish(b ^ 1);                                    // (once more than there are tiles)
        exponent();
        look(j + 3);
      }
    }
    if (bad) report(c.err);
    __syncwarp();
    if (G == 2 && S > 1) { cluster_sync_all(); cluster_sync_all(); }
  } else {
    // ------------------------------------------------------------------ query rows
    if (live) {
    const int w = warp >> 2, row = tid & 127, lrow = nq == 2 ? tid : row, qpos = p0 + lrow, wpos = qpos - lane;      // wpos: the warp's first row
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16, tO = tmem + 128 * G + w * HD + lanes;
    const float* s_qe = reinterpret_cast<const float*>(smem + C::QE);
    const uint32_t* s_tmax = reinterpret_cast<const uint32_t*>(smem + C::TMAX);
    {
      constexpr int LQ = HD / 8, NQ = LQ;        // lanes per row of q; loads of a thread, all on their way together
      uint4 u[NQ];
#pragma unroll
      for (int i = 0; i < NQ; i++) {
        const int r = (tid + i * C::ROWS) / LQ;
        u[i] = r < n ? *reinterpret_cast<const uint4*>(qkv + (size_t)(r0 + r) * ld + h * HD + tid % LQ * 8) : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < NQ; i++) {
        const int r = (tid + i * C::ROWS) / LQ, ch = tid % LQ;
        uint32_t m = amax8(u[i]);
#pragma unroll
        for (int y = LQ / 2; y > 0; y >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, y));
        const int eq = q_exponent(m);
        const float f = pow2_of((uint32_t)(127 - eq));
        const f32x2 f2 = mk2(f, f);
        st_shared_16(tile_chunk(sQ + (r >> 7) * C::TILE, r & 127, ch),
                     make_uint4(pack_f16(mul2(un2(u[i].x), f2)), pack_f16(mul2(un2(u[i].y), f2)), pack_f16(mul2(un2(u[i].z), f2)), pack_f16(mul2(un2(u[i].w), f2))));
        if (ch == 0) reinterpret_cast<float*>(smem + C::QE)[r] = pow2_of((uint32_t)(127 + eq));
      }
    }
    fence_proxy_async_smem();
    named_barrier<1, C::ROWS>();
    if (lane == 0) mbar_arrive(bar_q);
    const float rq = sl2 * s_qe[lrow];
    float R = -INFINITY, l = 0.f;
    uint32_t eb = 127;
    const int mine = tiles_of(w);
#pragma unroll 1
    for (int cnt = 0; cnt < mine; cnt++) {
      const int it = apart ? cnt : 2 * cnt + w, j = kt0 + it;
#pragma unroll 1
      for (int half = 0; half < 2; half++) {
        const int k0 = j * 128 + half * 64;
        const uint32_t tS = tmem + w * 128 + half * 64 + lanes;
        // (never on bar_kfull here: its stage may hold the tile after next by now, and a parity that has come round again would not be seen)
        wait(bar_s + 16 * w + 8 * half, cnt & 1);
        tc_fence_after();
        const uint32_t ek = s_tmax[it & 3] & 0xffffu, ev = s_tmax[it & 3] >> 16;
        if (cnt == 0) eb = ev;
        const float sl = rq * pow2_of(ek - 7), fev = (float)((int)ev - 127);
        const f32x2 slv = mk2(sl, sl);
        bool done = false;
        // Optimistic: exponentials with the reference R as it stands, the next scores on their way; the largest score beside them.  Where that would have
        // moved R (seldom after the first tile) what follows does it again.
        auto optimistic = [&](auto masked) {
          constexpr int W = 16;
          const float c0 = fev - R;
          const f32x2 c2 = mk2(c0, c0);
          f32x2 rs0 = 0, rs1 = 0;
          uint32_t r[2][W], pk[32];
          float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
          tmem_ld16(tS, r[0]);
#pragma unroll
          for (int q = 0; q < 64 / W; q++) {
            uint32_t (&x)[W] = r[q & 1];
            tmem_ld_wait();
            if (q + 1 < 64 / W) tmem_ld16(tS + (q + 1) * W, r[(q + 1) & 1]);
            if constexpr (decltype(masked)::value) {
#pragma unroll
              for (int i = 0; i < W; i++)
                if (k0 + q * W + i > qpos) x[i] = 0xff800000u;
            }
#pragma unroll
            for (int i = 0; i < W; i += 4) {
              const f32x2 e0 = fma2(mk2(__uint_as_float(x[i]), __uint_as_float(x[i + 1])), slv, c2);
              const f32x2 e1 = fma2(mk2(__uint_as_float(x[i + 2]), __uint_as_float(x[i + 3])), slv, c2);
              const f32x2 y0 = mk2(ex2(lo2(e0)), ex2(hi2(e0))), y1 = mk2(ex2(lo2(e1)), ex2(hi2(e1)));
              mx[i & 4 ? 2 : 0] = max3(mx[i & 4 ? 2 : 0], __uint_as_float(x[i]), __uint_as_float(x[i + 1]));
              mx[i & 4 ? 3 : 1] = max3(mx[i & 4 ? 3 : 1], __uint_as_float(x[i + 2]), __uint_as_float(x[i + 3]));
              rs0 = add2(rs0, y0);
              rs1 = add2(rs1, y1);
              pk[(q * W + i) >> 1] = pack_f16(y0);
              pk[((q * W + i) >> 1) + 1] = pack_f16(y1);
            }
          }
          const float mt = fmaf(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])), sl, fev);
          done = !__any_sync(0xffffffffu, mt > R + 15.f);
          if (done) {
            tmem_st16(tS, pk);                   // over the scores
            tmem_st16(tS + 16, pk + 16);
            l = fmaf((lo2(rs0) + hi2(rs0)) + (lo2(rs1) + hi2(rs1)), pow2_of(127 + eb - ev), l);
          }
        };
        if (k0 <= wpos + 31 && !__any_sync(0xffffffffu, R == -INFINITY)) {
          if (k0 + 63 <= wpos) optimistic(std::false_type{}); else optimistic(std::true_type{});
        }
        if (done) {
        } else if (k0 > wpos + 31) {             // every key comes after the warp's queries
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 16; i++) pk[i] = 0u;
          tmem_st16(tS, pk);
          tmem_st16(tS + 16, pk);
        } else {
          float mx = -INFINITY;
          auto half_of = [&](int q, uint32_t (&r)[32]) {       // 32 scores, masked
            tmem_ld32(tS + q * 32, r);
            tmem_ld_wait();
            if (k0 + q * 32 + 31 > wpos)         // masks keys after the query
#pragma unroll
              for (int i = 0; i < 32; i++)
                if (k0 + q * 32 + i > qpos) r[i] = 0xff800000u;
          };
#pragma unroll 1
          for (int q = 0; q < 2; q++) {
            uint32_t r[32];
            half_of(q, r);
            float m0 = mx, m1 = -INFINITY;
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
              m0 = max3(m0, __uint_as_float(r[i]), __uint_as_float(r[i + 1]));
              m1 = max3(m1, __uint_as_float(r[i + 2]), __uint_as_float(r[i + 3]));
            }
            mx = fmaxf(m0, m1);
          }
          const float mt = fmaf(mx, sl, fev);
          const bool grow = mt > R + 15.f;       // (from -inf too)
          if (__any_sync(0xffffffffu, grow)) {
            const float al = grow ? ex2(R - (mt - 7.f)) : 1.f;
            if (cnt + half > 0) {                // O is there, once the last P V is done (the one before it is: these scores came after it)
              wait(bar_pv + 8 * w, (half ^ 1) & 1);
              tc_fence_after();
              rescale<HD>(tO, al);
            }
            l *= al;
            if (grow) R = mt - 7.f;
          }
          const float c0 = fev - (R == -INFINITY ? 0.f : R);
          const f32x2 c2 = mk2(c0, c0);
          f32x2 rs0 = 0, rs1 = 0;
#pragma unroll 1
          for (int q = 0; q < 2; q++) {
            uint32_t r[32], pk[16];
            half_of(q, r);
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
              const f32x2 e0 = fma2(mk2(__uint_as_float(r[i]), __uint_as_float(r[i + 1])), slv, c2);
              const f32x2 e1 = fma2(mk2(__uint_as_float(r[i + 2]), __uint_as_float(r[i + 3])), slv, c2);
              const f32x2 x0 = mk2(ex2(lo2(e0)), ex2(hi2(e0))), x1 = mk2(ex2(lo2(e1)), ex2(hi2(e1)));
              rs0 = add2(rs0, x0);
              rs1 = add2(rs1, x1);
              pk[i >> 1] = pack_f16(x0);
              pk[(i >> 1) + 1] = pack_f16(x1);
            }
            tmem_st16(tS + q * 16, pk);          // over scores that have been used
          }
          l = fmaf((lo2(rs0) + hi2(rs0)) + (lo2(rs1) + hi2(rs1)), pow2_of(127 + eb - ev), l);
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_p + 16 * w + 8 * half);
      }
    }
    if (mine > 0) wait(bar_o + 8 * w, 0);      // (on a barrier of its own: the P V before the last may not be done, and its parity would be taken for the last one's)
    tc_fence_after();
    float den = l * pow2_of(261u - eb);          // l 2^(7 - EB)
    // A NaN in V reaches the rows that see its position and no others.  P V multiplies it with the zeros of masked positions too, which leaves a
    // NaN in every row of the tile: such rows are done anew, one by one.
    auto leave = [&]() {                         // (R, normaliser, O) of the group's rows in shared memory, over the tiles
      float* part = reinterpret_cast<float*>(smem) + (w * 128 + row) * C::PITCH;
      *reinterpret_cast<float2*>(smem + C::ML + (w * 128 + row) * 8) = make_float2(R, den);
      if (lrow - lane >= n) return;              // (a warp without rows)
#pragma unroll 1
      for (int q = 0; q < HD; q += 32) {
        uint32_t r[32];
        if (mine > 0) { tmem_ld32(tO + q, r); tmem_ld_wait(); }
        else {
#pragma unroll
          for (int i = 0; i < 32; i++) r[i] = 0u;
        }
#pragma unroll
        for (int i = 0; i < 32; i += 4)
          *reinterpret_cast<uint4*>(part + q + i) = make_uint4(r[i], r[i + 1], r[i + 2], r[i + 3]);
      }
    };
    named_barrier<1, C::ROWS>();                     // no tile is read any more; `redo` and `reach` are written
    // (l beyond 2^100: a first tile of values 2^85 times the later ones', and no weight)
    const uint32_t far = *reach;
    if (R > -INFINITY && (lost(*redo, rq) || !(rq * pow2_of((far & 0xffffu) - 7) * HD <= 0x1p-8f) || !(l * pow2_of(382u - (far >> 16) - eb) * 0x1p16f >= ctx) || l > 0x1p100f))
      den = __int_as_float(0x7fffffff);
    if (G == 2 && S > 1) leave();
    else {
      float own = 1.f, other = 0.f, sum = den;   // weights of the group's sums and of the second group's for the same rows
      if (!apart) {
        if (w == 1) leave();
        named_barrier<1, C::ROWS>();
        if (w == 0) {
          const float2 v = *reinterpret_cast<const float2*>(smem + C::ML + (128 + row) * 8);
          const float mx = fmaxf(R, v.x), ref = mx == -INFINITY ? 0.f : mx;
          own = ex2(R - ref);
          other = ex2(v.x - ref);
          sum = fmaf(own, den, other * v.y);
        }
      }
      if (apart || w == 0) {
        const bool intact = *abort_flag == 0 && lrow < n;
        const float inv = 1.f / sum;
        const float* part = reinterpret_cast<const float*>(smem) + (128 + row) * C::PITCH;
        bf16* dst = out + (size_t)(r0 + lrow) * ldo + h * HD;
        uint32_t top = sum > 0.f ? __float_as_uint(inv) & 0x7fffffffu : 0x7f800000u;
        if (lrow - lane < n)
#pragma unroll 1
          for (int q = 0; q < HD; q += 32) {
            uint32_t r[32], o[16];
            tmem_ld32(tO + q, r);
            tmem_ld_wait();
            if (!apart)
#pragma unroll
              for (int i = 0; i < 32; i += 4) {
                const float4 v = *reinterpret_cast<const float4*>(part + q + i);
                r[i] = __float_as_uint(fmaf(other, v.x, own * __uint_as_float(r[i])));
                r[i + 1] = __float_as_uint(fmaf(other, v.y, own * __uint_as_float(r[i + 1])));
                r[i + 2] = __float_as_uint(fmaf(other, v.z, own * __uint_as_float(r[i + 2])));
                r[i + 3] = __float_as_uint(fmaf(other, v.w, own * __uint_as_float(r[i + 3])));
              }
#pragma unroll
            for (int i = 0; i < 32; i++) top = max(top, r[i] & 0x7fffffffu);
#pragma unroll
            for (int i = 0; i < 16; i++) o[i] = pack_bf16(__uint_as_float(r[2 * i]) * inv, __uint_as_float(r[2 * i + 1]) * inv);
            if (intact)
#pragma unroll
              for (int i = 0; i < 4; i++) *reinterpret_cast<uint4*>(dst + q + 8 * i) = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
          }
        const uint32_t again = __ballot_sync(0xffffffffu, intact && top >= 0x7f800000u);
        if (lane == 0) s_again[warp] = again;
      }
    }
    }
  // ------------------------------------------------------------------ the cluster's CTAs join
  if (G == 2 && S > 1) { __syncwarp(); cluster_sync_all(); }
  if (G == 2 && live && S > 1) {
    const int parts = nq == 2 ? S : 2 * S;       // of a row: part i is group i % 2 (or the row's own) of CTA i / 2 (or i)
    // CTA `rank` joins rows rank, rank + S ...; a thread four columns of a row
    constexpr int TPR = HD / 4;
    const int ch = tid % TPR;
    constexpr int NR = 2, STEP = 256 / TPR;
#pragma unroll 1
    for (int r1 = rank + tid / TPR * S; r1 < n; r1 += NR * STEP * S) {
      float den[NR], o[NR][4];
      join_parts<NR>(parts, [&](int k, int i, uint32_t& ml, uint32_t& data) {
        const int r = min(r1 + k * STEP * S, n - 1), line = nq == 2 ? r : (i & 1) * 128 + (r & 127);
        const uint32_t a = mapa_shared(base, nq == 2 ? i : i >> 1);
        ml = a + C::ML + line * 8;
        data = a + (line * C::PITCH + ch * 4) * 4;
      }, den, o);
      if (*abort_flag) break;
#pragma unroll
      for (int k = 0; k < NR; k++) {
        const int r = r1 + k * STEP * S;
        if (r >= n) break;
        const float inv = 1.f / den[k];
        bool anew = !(den[k] > 0.f) || (__float_as_uint(inv) & 0x7fffffffu) >= 0x7f800000u;
#pragma unroll
        for (int e = 0; e < 4; e++) anew |= (__float_as_uint(o[k][e]) & 0x7fffffffu) >= 0x7f800000u;
        if (anew) atomicOr(s_again + (r >> 5), 1u << (r & 31));
        else *reinterpret_cast<uint2*>(out + (size_t)(r0 + r) * ldo + h * HD + ch * 4) = make_uint2(pack_bf16(o[k][0] * inv, o[k][1] * inv), pack_bf16(o[k][2] * inv, o[k][3] * inv));
      }
    }
  }
  if (G == 2 && S > 1) { __syncwarp(); cluster_sync_all(); }          // the others' parts are read until here
  if (live) {                                    // (after the join: a row's other columns may have been stored)
    named_barrier<1, C::ROWS>();
#pragma unroll 1
    for (uint32_t m = s_again[warp]; m; m &= m - 1) {      // (over the set bits: a turn costs some 140 cycles even where it does nothing)
      const int r = warp * 32 + __ffs(m) - 1;
      attend_row8<HD>(c, qkv + (size_t)(r0 + r) * ld + h * HD, h, p0 + r, sl, sl2, out + (size_t)(r0 + r) * ldo + h * HD);
    }
  }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) { tc_fence_after(); tmem_dealloc(tmem, COLS); }
}

// Launch in clusters of S CTAs along x.
template <typename... P, typename... A>
static int launch_clusters(void (*kernel)(P...), dim3 grid, int threads, int smem, int S, cudaStream_t st, A... args) {
  if (smem > 48 * 1024 && cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) {
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
  cfg.gridDim = grid; cfg.blockDim = dim3(threads); cfg.dynamicSmemBytes = smem; cfg.stream = st; cfg.attrs = attr; cfg.numAttrs = n;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, P(args)...);
  if (e != cudaSuccess) { cudaGetLastError(); kh_set_error("paged_prefill8: %s", cudaGetErrorString(e)); return -1; }
  return 0;
}
// Clusters of S = 2, 4, 8 CTAs of the tcgen05 kernel (one per SM) that the chip holds at once: a cluster lies in one group of SMs.
template <int HD>
static int chunk_clusters(int S) {
  static int known[4] = {0, 0, 0, 0};
  int& n = known[S == 2 ? 1 : S == 4 ? 2 : 3];
  if (n == 0) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = S; attr.val.clusterDim.y = 1; attr.val.clusterDim.z = 1;
    cfg.gridDim = dim3(S * 148); cfg.blockDim = dim3(Chunk<HD, 2>::THREADS); cfg.dynamicSmemBytes = Chunk<HD, 2>::SMEM; cfg.attrs = &attr; cfg.numAttrs = 1;
    int got = 0;
    if (cudaFuncSetAttribute(paged_chunk8_k<HD, 2>, cudaFuncAttributeMaxDynamicSharedMemorySize, Chunk<HD, 2>::SMEM) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&got, paged_chunk8_k<HD, 2>, &cfg) != cudaSuccess || got < 1) {
      cudaGetLastError();
      got = -1;                                      // not available
    }
    n = got;
  }
  return n;
}
template <int HD>
static int launch_runs(const Cache& c, const bf16* qkv, int ld, bf16* out, int ldo, float sl2, int max_ctx, const int* row0, const int* len, int n_runs, cudaStream_t st) {
  int n_short = 0, most = 0;
  for (int i = 0; i < n_runs; i++) {
    if (row0[i] < 0 || len[i] < 1) { kh_set_error("paged_prefill8: run %d is empty", i); return -1; }
    n_short += len[i] <= P8_ROWS;
    most = len[i] > most ? len[i] : most;
  }
  // Runs of up to 64 tokens take the kernel of short runs where a CTA has up to four tiles of the longest context, counting rounds of two CTAs per SM.  us, that kernel / the
  // one below, 16 heads of 64: 30 fresh runs of 64 9.4 / 14.0, behind 200 positions 26.6 / 22.2; one of 32 behind 1000 9.3 / 10.1, behind 2000 12.8 / 11.9; 8 behind
  // 500 16.9 / 12.4; 20 behind 2000 88 / 64 (heads of 128: 225 / 103).
  const int tiles64 = (max_ctx + P8_ROWS - 1) / P8_ROWS;
  int S_short = 1;                                   // two CTAs per SM, two tiles of the longest context for each
  while (S_short < 8 && (long)n_short * c.H * S_short * 2 <= 2 * 148 && tiles64 >= 4 * S_short) S_short *= 2;
  const bool split_short = (tiles64 + S_short - 1) / S_short * (((long)n_short * c.H * S_short + 295) / 296) <= 4;
  int nt = 0;
  if (split_short && n_short) {
    Pieces tiles;
    auto flush = [&]() -> int {
      const int n = nt;
      nt = 0;
      return n ? launch_clusters(paged_short8_k<HD>, dim3((unsigned)n * S_short, c.H), 128, 2 * P8_ROWS * (HD * 2 + 16) + P8_ROWS * 8 + 16, S_short, st, tiles, c, qkv, ld, out, ldo, sl2, max_ctx, S_short) : 0;
    };
    for (int i = 0; i < n_runs; i++)
      if (len[i] <= P8_ROWS) {
        tiles.row0[nt] = row0[i];
        tiles.n[nt] = (uint8_t)len[i];
        if (++nt == P8_MAX && flush()) return -1;
      }
    if (flush()) return -1;
  }
  // Clusters where all their CTAs are on the chip at once: of eight from 24 key tiles, of four from 4, of two from 8 (8 heads, us in clusters of 1 / 2 / 4 / 8.
  // Of 64: 384 fresh tokens 10.2 / 12.3 / 11.3 / -, 700 14.7 / 15.7 / 13.1 / -, 2048 31.7 / 27.0 / 29.6 / -, 100 behind 2000 24.7 / 18.0 / 14.6 / 15.0, behind
  // 4000 42.6 / 26.8 / 18.7 / 16.8.  Of 128: 512 fresh 18.5 / 20.5 / 15.6 / -, 200 behind 14000 256 / 142 / 77 / 48).
  long items = 0, halves = 0;                        // pieces of 256 and of 128 tokens
  for (int i = 0; i < n_runs; i++)
    if (!split_short || len[i] > P8_ROWS) { items += (len[i] + 255) / 256; halves += (len[i] + 127) / 128; }
  items *= c.H;
  halves *= c.H;
  const int kt = (max_ctx + 127) / 128;
  int S = 8;
  while (S > 1 && (items > chunk_clusters<HD>(S) || kt < (S == 8 ? 24 : S == 4 ? 4 : 8))) S /= 2;
  // Without a cluster, heads of up to 64: items of 128 tokens, two CTAs per SM, unless items of 256 fill the SMs in whole rounds (three quarters at least)
  // and see more than three tiles: those fetch the keys once for twice the rows.  us, items of 128 / of 256, heads of 64: 1024 runs of 128 fresh tokens and heads 35.7 / 56.2,
  // 320 of 300 20.9 / 28.6, 192 of 200 behind 500 positions 32.5 / 36.8, 128 of 150 behind 1000 29.1 / 25.6, 192 of 500 behind 4000 256 / 230.
  const long rounds = (items + 147) / 148;
  const bool one = HD <= 64 && S == 1 && (kt <= 3 || halves * 2 < 3 * 148 * rounds);
  const int rows = one ? 128 : 256;
  Runs runs;
  auto flush = [&]() -> int {
    const int n = nt;
    nt = 0;
    if (n == 0) return 0;
    if constexpr (HD <= 64)
      if (one) return launch_clusters(paged_chunk8_k<HD, 1>, dim3((unsigned)c.H, n), Chunk<HD, 1>::THREADS, Chunk<HD, 1>::SMEM, 1, st, runs, c, qkv, ld, out, ldo, sl2, max_ctx, 1);
    return launch_clusters(paged_chunk8_k<HD, 2>, dim3((unsigned)c.H * S, n), Chunk<HD, 2>::THREADS, Chunk<HD, 2>::SMEM, S, st, runs, c, qkv, ld, out, ldo, sl2, max_ctx, S);
  };
  // the pieces that see the most keys first (as far as the lengths tell)
  for (int at = (most - 1) / rows * rows; at >= 0; at -= rows)
    for (int i = 0; i < n_runs; i++) {
      if (len[i] <= at || (split_short && len[i] <= P8_ROWS)) continue;
      runs.row0[nt] = row0[i] + at;
      runs.n[nt] = (uint16_t)(len[i] - at < rows ? len[i] - at : rows);
      if (++nt == CH_MAX && flush()) return -1;
    }
  return flush();
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
  max_ctx = max_ctx < max_lb * bs ? max_ctx : max_lb * bs;
  const float sl2 = scale * 1.4426950408889634f;
#define LAUNCH(HD) return launch_runs<HD>(c, (const bf16*)qkv, ld, (bf16*)out, ldo, sl2, max_ctx, (const int*)row0, (const int*)len, n_runs, (cudaStream_t)stream);
  if (hd == 128) { LAUNCH(128) }
  if (hd == 64) { LAUNCH(64) }
  LAUNCH(32)
#undef LAUNCH
}
