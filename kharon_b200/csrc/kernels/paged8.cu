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
