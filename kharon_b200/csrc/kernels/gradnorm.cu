// The 2-norm over many tensors, the factor that bounds it, and the tensors times that factor.
//
// A list of tensors is a table of {address, elements, pieces before it, type}; a CTA takes an equal share of all pieces in one run, sums squares in 64 bits (whose range
// holds every square of an fp32 number, and whose additions lose nothing that fp32 could show), and the last CTA adds the CTAs' sums in order.  Bound by memory: each
// element is read once.  The tensors are multiplied in the same shares, from their ends back to their beginnings, so that what the norm read last comes from L2.
// 5.25 GB of fp32 in 292 tensors: 740 us, 7.1 TB/s, as reads alone go; 55 MB in 76 tensors of both types multiplied into other buffers: 36 us, half of it either kernel's start, end and trips; 204 MB: 110 us,
// 0.85 of the copy rate for three passes.  In place, behind a flushed L2: 40 and 113 us, into other buffers 42 and 116.
#include <algorithm>

#include "common.cuh"

#define KH_LAUNCH_CHECK(name)                                                     \
  do {                                                                            \
    cudaError_t e_ = cudaGetLastError();                                          \
    if (e_ != cudaSuccess) { kh_set_error(name ": %s", cudaGetErrorString(e_)); return -1; } \
  } while (0)

namespace {

struct Entry {                               // one tensor
  unsigned long long at;                     // address
  long n;                                    // elements
  long before;                               // pieces of the tensors before it
  long bf;                                   // 1: bf16, 0: fp32
};
// A piece has 32 KB where the list then has no more pieces than CTAs: no CTA goes from tensor to tensor (13 MB in 52 tensors: 6.5 us, with 4 KB 8.0).  Else it has 4 KB, so that
// the shares are equal (5.25 GB: 740 us, with 32 KB 786).
constexpr int SHARE = 32768, FINE = 4096;
constexpr int BLOCK = 8192;                  // elements that are multiplied at a time
constexpr int PARTS = 2048, T = 256;         // CTAs at most, their threads
constexpr int TABLE = 1024;                  // tensors whose places are looked up in shared memory

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// norm and factor from the sum of squares; a step that is to be left out is counted
__device__ __forceinline__ void put_norm(double sum, float max_norm, float* out, int* left_out) {
  const double norm = sqrt(sum);
  if (left_out && !isfinite(norm)) ++*left_out;
  out[0] = (float)norm;
  out[1] = !isfinite(norm) ? NAN : norm <= (double)max_norm ? 1.f : (float)((double)max_norm / norm);
}
__device__ __forceinline__ double square(double s, float x) { return fma((double)x, (double)x, s); }

// the tensor whose pieces hold piece k
__device__ __forceinline__ int entry_of(const Entry* e, int n, long k, long* s_before) {
  if (n <= TABLE) {
    for (int i = threadIdx.x; i < n; i += T) s_before[i] = e[i].before;
    __syncthreads();
  }
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if ((n <= TABLE ? s_before[mid] : e[mid].before) <= k) lo = mid;
    else hi = mid;
  }
  return lo;
}
__device__ __forceinline__ long piece_of(const Entry& e, int piece) { return e.bf ? piece / 2 : piece / 4; }           // in elements
__device__ __forceinline__ long pieces_of(const Entry& e, int piece) { return (e.n + piece_of(e, piece) - 1) / piece_of(e, piece); }
// elements before the first address on 16 bytes, at most n
__device__ __forceinline__ int head_of(unsigned long long at, int size, long n) { return (int)min(n, (long)(((16 - (at & 15)) & 15) / size)); }

__device__ __forceinline__ double add4(double s, const float4& v) { return square(square(square(square(s, v.x), v.y), v.z), v.w); }
__device__ __forceinline__ double add8(double s, const uint4& v) {
  const float2 a = unpack_bf16(v.x), b = unpack_bf16(v.y), c = unpack_bf16(v.z), d = unpack_bf16(v.w);
  return square(square(square(square(square(square(square(square(s, a.x), a.y), b.x), b.y), c.x), c.y), d.x), d.y);
}
__device__ __forceinline__ float value(const float* p) { return *p; }
__device__ __forceinline__ float value(const bf16* p) { return __bfloat162float(*p); }
// squares of n elements from p: E of them to 16 bytes
template <int E, typename V, typename F>
__device__ __forceinline__ double sum_run(const F* p, long n) {
  const int tid = threadIdx.x, head = head_of((unsigned long long)p, sizeof(F), n);
  const long nv = (n - head) / E, tail = head + nv * E;
  const V* v = reinterpret_cast<const V*>(p + head);
  double s[4] = {};
  auto add = [](double t, const V& x) { if constexpr (E == 4) return add4(t, x); else return add8(t, x); };
  long i = tid;
  for (; i + 3 * T < nv; i += 4 * T) {
    const V a = v[i], b = v[i + T], c = v[i + 2 * T], d = v[i + 3 * T];
    s[0] = add(s[0], a); s[1] = add(s[1], b); s[2] = add(s[2], c); s[3] = add(s[3], d);
  }
  for (; i < nv; i += T) s[0] = add(s[0], v[i]);
  if (tid < head) s[1] = square(s[1], value(p + tid));
  if (tail + tid < n) s[1] = square(s[1], value(p + tail + tid));
  return (s[0] + s[1]) + (s[2] + s[3]);
}
__device__ __forceinline__ void share_of(long pieces, long& k0, long& k1) {
  const long per = pieces / gridDim.x, more = pieces % gridDim.x, b = blockIdx.x;
  k0 = b * per + min(b, more);
  k1 = k0 + per + (b < more);
}
__global__ void __launch_bounds__(T, 4) norm_k(const Entry* table, int n, long pieces, int piece, float max_norm, double* work, float* out, double* sumsq, int* left_out) {
  __shared__ double s_s[8];
  __shared__ long s_before[TABLE];
  __shared__ int s_last;
  pdl_wait();
  pdl_launch_dependents();
  const int tid = threadIdx.x;
  long k0, k1;
  share_of(pieces, k0, k1);
  double s = 0.0;
  if (k0 < k1) {
    for (int t = entry_of(table, n, k0, s_before); k0 < k1; t++) {
      const Entry e = table[t];
      const long end = min(k1, e.before + pieces_of(e, piece)), i0 = (k0 - e.before) * piece_of(e, piece), m = min((end - e.before) * piece_of(e, piece), e.n) - i0;
      s += e.bf ? sum_run<8, uint4>(reinterpret_cast<const bf16*>(e.at) + i0, m) : sum_run<4, float4>(reinterpret_cast<const float*>(e.at) + i0, m);
      k0 = end;
    }
  }
  s = warp_sum(s);
  if ((tid & 31) == 0) s_s[tid >> 5] = s;
  __syncthreads();
  int* ticket = reinterpret_cast<int*>(work);
  double* part = work + 2;
  if (tid == 0) {
    s = 0.0;
    for (int k = 0; k < 8; k++) s += s_s[k];
    part[blockIdx.x] = s;
    __threadfence();
    s_last = atomicInc(reinterpret_cast<unsigned*>(ticket), gridDim.x - 1) == gridDim.x - 1;      // back at 0 with the last one
  }
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  s = 0.0;
  for (int i = tid; i < (int)gridDim.x; i += T) s += __ldcg(part + i);
  s = warp_sum(s);
  __syncthreads();
  if ((tid & 31) == 0) s_s[tid >> 5] = s;
  __syncthreads();
  if (tid == 0) {
    s = 0.0;
    for (int k = 0; k < 8; k++) s += s_s[k];
    if (sumsq) *sumsq = s;
    if (out) put_norm(s, max_norm, out, left_out);
  }
}
__global__ void clip_factor_k(const double* sumsq, float max_norm, float* out, int* left_out) {
  pdl_wait();
  pdl_launch_dependents();
  put_norm(*sumsq, max_norm, out, left_out);
}
// n elements of one type times f to another place, 16 bytes at a time where both allow it
template <int E, typename V, typename F>
__device__ __forceinline__ void scale_run(const F* p, F* d, int n, float f) {
  const int tid = threadIdx.x;
  auto mul = [f](const V& x) {
    if constexpr (E == 4) return make_float4(x.x * f, x.y * f, x.z * f, x.w * f);
    else {
      const float2 a = unpack_bf16(x.x), b = unpack_bf16(x.y), c = unpack_bf16(x.z), e = unpack_bf16(x.w);
      return make_uint4(pack_bf16(a.x * f, a.y * f), pack_bf16(b.x * f, b.y * f), pack_bf16(c.x * f, c.y * f), pack_bf16(e.x * f, e.y * f));
    }
  };
  int head = n, nv = 0;
  if ((((unsigned long long)p ^ (unsigned long long)d) & 15) == 0) {
    head = head_of((unsigned long long)p, sizeof(F), n);
    nv = (n - head) / E;
    const V* v = reinterpret_cast<const V*>(p + head);
    V* w = reinterpret_cast<V*>(d + head);
    int i = tid;
    for (; i + 3 * T < nv; i += 4 * T) {
      const V x[4] = {v[i], v[i + T], v[i + 2 * T], v[i + 3 * T]};
#pragma unroll
      for (int u = 0; u < 4; u++) w[i + u * T] = mul(x[u]);
    }
    for (; i < nv; i += T) w[i] = mul(v[i]);
  }
  auto one = [&](int i) {
    if constexpr (E == 4) d[i] = p[i] * f;
    else d[i] = __float2bfloat16(__bfloat162float(p[i]) * f);
  };
  for (int i = tid; i < head; i += T) one(i);
  for (int i = head + nv * E + tid; i < n; i += T) one(i);
}
// dst = src * factor (dst may be src); a factor that is no number leaves the tensors as they are
__global__ void __launch_bounds__(T, 4) scale_k(const Entry* src, const Entry* dst, int n, long pieces, int piece, const float* factor, int same) {
  __shared__ long s_before[TABLE];
  pdl_wait();
  pdl_launch_dependents();
  float f = *factor;
  if (same && !(f != 1.f && f == f)) return;
  if (f != f) f = 1.f;
  const int tid = threadIdx.x;
  long k0, k1;
  share_of(pieces, k0, k1);
  if (k0 >= k1) return;
  for (int t = entry_of(src, n, k1 - 1, s_before); k0 < k1; t--) {
    const Entry e = src[t], d = dst[t];
    const long from = max(k0, e.before), a = (from - e.before) * piece_of(e, piece);
    for (long b = min((k1 - e.before) * piece_of(e, piece), e.n); b > a; b -= BLOCK) {
      const long i0 = max(a, b - BLOCK);
      const int m = (int)(b - i0);
      const float* pf = reinterpret_cast<const float*>(e.at) + i0;
      const bf16* pb = reinterpret_cast<const bf16*>(e.at) + i0;
      float* df = reinterpret_cast<float*>(d.at) + i0;
      bf16* db = reinterpret_cast<bf16*>(d.at) + i0;
      if (!e.bf && !d.bf) {
        scale_run<4, float4>(pf, df, m, f);
      } else if (e.bf && d.bf) {
        scale_run<8, uint4>(pb, db, m, f);
      } else if (d.bf) {
#pragma unroll 8
        for (int i = tid; i < m; i += T) db[i] = __float2bfloat16(pf[i] * f);
      } else {
#pragma unroll 8
        for (int i = tid; i < m; i += T) df[i] = __bfloat162float(pb[i]) * f;
      }
    }
    k1 = from;
  }
}
long most_ctas() {
  int dev = 0, sms = 148;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return std::min(4l * sms, (long)PARTS);
}
int grid_for(long pieces, int piece) { return (int)std::max(1l, std::min((pieces * piece + SHARE - 1) / SHARE, most_ctas())); }
bool good(int n, long pieces, int piece) { return n >= 0 && pieces >= 0 && (piece == SHARE || piece == FINE); }

}  // namespace

// Bytes of a piece for a list of so many pieces of the larger size: the table's `before` counts pieces, at least one for each tensor that is not empty.
extern "C" int kh_grad_share() { return SHARE; }
extern "C" int kh_grad_piece(long shares) { return shares <= most_ctas() ? SHARE : FINE; }
extern "C" long kh_grad_work_bytes() { return 16 + 8L * PARTS; }
extern "C" int kh_grad_norm(const void* table, int n, long pieces, int piece, float max_norm, void* work, void* out, void* sumsq, void* left_out, void* stream) {
  if (!good(n, pieces, piece)) { kh_set_error("grad_norm: a table of %d tensors, %ld pieces of %d bytes", n, pieces, piece); return -1; }
  KH_LAUNCH(norm_k, grid_for(pieces, piece), T, 0, (cudaStream_t)stream, (const Entry*)table, n, pieces, piece, max_norm, (double*)work, (float*)out, (double*)sumsq, (int*)left_out);
  KH_LAUNCH_CHECK("grad_norm");
  return 0;
}
extern "C" int kh_clip_factor(const void* sumsq, float max_norm, void* out, void* left_out, void* stream) {
  KH_LAUNCH(clip_factor_k, 1, 1, 0, (cudaStream_t)stream, (const double*)sumsq, max_norm, (float*)out, (int*)left_out);
  KH_LAUNCH_CHECK("clip_factor");
  return 0;
}
extern "C" int kh_grad_scale(const void* src, const void* dst, int n, long pieces, int piece, const void* factor, void* stream) {
  if (!good(n, pieces, piece)) { kh_set_error("grad_scale: a table of %d tensors, %ld pieces of %d bytes", n, pieces, piece); return -1; }
  if (pieces == 0) return 0;
  KH_LAUNCH(scale_k, grid_for(pieces, piece), T, 0, (cudaStream_t)stream, (const Entry*)src, (const Entry*)dst, n, pieces, piece, (const float*)factor, (int)(src == dst));
  KH_LAUNCH_CHECK("grad_scale");
  return 0;
}
