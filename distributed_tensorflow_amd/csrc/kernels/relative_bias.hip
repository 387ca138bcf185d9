// Learned relative position bias by buckets, written out (gfx950).
//
//   forward : out[h, i, j] = table[bucket(j - (q_start + i)), h]
//   backward: dtable[u, h] = sum of g[h, i, j] over the (i, j) whose distance has bucket u
//
// Both are bound by the one pass over [heads, q_len, k_len]: 2 or 4 bytes an element against a lookup or an addition. The
// bias depends on the distance alone, so a workgroup keeps its head's values by distance in the LDS (a band of
// 2 max_distance + 1, with a constant on either side).
#include "dtf_common.h"

using namespace dtf;

namespace {

constexpr int kMaxThr = 64, kRowsPerBlock = 32;

struct BiasArgs {
  int Sq, Sk, heads, start, buckets, half, exact, max_dist, right, n_thr, thr[kMaxThr];
};

__device__ __forceinline__ int bucket_of(const BiasArgs& a, int dist) {
  const int far = a.right ? (dist < 0 ? -dist : dist) : (dist < 0 ? -dist : 0);
  int b = far;
  if (far >= a.exact) {
    b = a.exact;
    for (int t = 0; t < a.n_thr; ++t) b += far >= a.thr[t] ? 1 : 0;
  }
  return b + (a.right && dist > 0 ? a.half : 0);
}

template <typename T>
__global__ __launch_bounds__(256) void bias_fwd_kernel(BiasArgs a, const T* __restrict__ table, T* __restrict__ out) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  T* band = reinterpret_cast<T*>(smem);                  // values of the distances -max_dist .. right
  const int tid = threadIdx.x, h = blockIdx.y;
  for (int i = tid; i <= a.max_dist + a.right; i += 256) band[i] = table[(long long)bucket_of(a, i - a.max_dist) * a.heads + h];
  __syncthreads();
  for (long long i = blockIdx.x; i < a.Sq; i += gridDim.x) {
    T* row = out + ((long long)h * a.Sq + i) * a.Sk;
    const int pos = a.start + (int)i;
    for (int j = tid; j < a.Sk; j += 256) row[j] = band[min(max(j - pos, -a.max_dist), a.right) + a.max_dist];
  }
}

__device__ __forceinline__ float as_float(unsigned short v) { return bf16_to_f32(v); }
__device__ __forceinline__ float as_float(float v) { return v; }

// One workgroup: kRowsPerBlock rows of one head. A thread owns distances, not columns, and adds their elements row after
// row: every sum has a fixed order.
template <typename T>
__global__ __launch_bounds__(256) void bias_bwd_kernel(BiasArgs a, const T* __restrict__ g, float* __restrict__ parts) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  float* band = reinterpret_cast<float*>(smem);          // sums of the distances -max_dist .. right
  const int tid = threadIdx.x, h = blockIdx.y;
  const int i0 = blockIdx.x * kRowsPerBlock, i1 = min(i0 + kRowsPerBlock, a.Sq);
  float far_l = 0.f, far_r = 0.f;
  for (int d = tid; d <= a.max_dist + a.right; d += 256) {
    float v = 0.f;
    for (int i = i0; i < i1; ++i) {
      const int j = a.start + i + d - a.max_dist;
      if (j >= 0 && j < a.Sk && d > 0 && d < a.max_dist + a.right) v += as_float(g[((long long)h * a.Sq + i) * a.Sk + j]);
    }
    band[d] = v;
  }
  for (int i = i0; i < i1; ++i) {
    const T* row = g + ((long long)h * a.Sq + i) * a.Sk;
    const int pos = a.start + i;
    const int left = min(max(pos - a.max_dist + 1, 0), a.Sk), right = min(max(pos + a.right, left), a.Sk);
    for (int j = tid; j < left; j += 256) far_l += as_float(row[j]);
    for (int j = right + tid; j < a.Sk; j += 256) far_r += as_float(row[j]);
  }
  __shared__ float scratch[16];
  far_l = block_sum(far_l, scratch);
  far_r = block_sum(far_r, scratch);
  __syncthreads();
  if (tid == 0) {
    band[0] += far_l;
    band[a.max_dist + a.right] += far_r;
  }
  __syncthreads();
  for (int u = tid; u < a.buckets; u += 256) {
    float v = 0.f;
    for (int d = 0; d <= a.max_dist + a.right; ++d)
      if (bucket_of(a, d - a.max_dist) == u) v += band[d];
    parts[((long long)blockIdx.x * a.heads + h) * a.buckets + u] = v;
  }
}

template <typename T>
__global__ __launch_bounds__(256) void bias_finish_kernel(const float* __restrict__ parts, T* __restrict__ out, int n_parts,
                                                         int heads, int buckets) {
  __shared__ float red[256];
  const int h = blockIdx.x, slices = 256 / buckets, u = threadIdx.x % buckets, s = threadIdx.x / buckets;
  float v = 0.f;
  if (s < slices)
    for (int p = s; p < n_parts; p += slices) v += parts[((long long)p * heads + h) * buckets + u];
  red[threadIdx.x] = v;
  __syncthreads();
  if (s == 0) {
    for (int i = 1; i < slices; ++i) v += red[i * buckets + u];
    if (sizeof(T) == 2) ((unsigned short*)out)[(long long)u * heads + h] = f32_to_bf16(v);
    else ((float*)out)[(long long)u * heads + h] = v;
  }
}

// words: q_len, k_len, heads, q_start, buckets, max_distance, bidirectional, then the bucket borders
bool unpack(const long long* w, int n, BiasArgs& a) {
  if (n < 7) return false;
  if (w[0] < 1 || w[1] < 1 || w[0] > (1 << 28) || w[1] > (1 << 28) || w[2] < 1 || w[2] > 65535) return false;
  if (w[3] > (1 << 29) || w[3] < -(1 << 29) || w[4] < 2 || w[4] > 128 || w[5] < 1 || w[5] > 2048) return false;
  a.Sq = (int)w[0]; a.Sk = (int)w[1]; a.heads = (int)w[2]; a.start = (int)w[3];
  a.buckets = (int)w[4]; a.max_dist = (int)w[5];
  a.right = w[6] ? a.max_dist : 0;
  a.half = w[6] ? a.buckets / 2 : a.buckets;
  a.exact = a.half / 2;
  a.n_thr = a.half - a.exact - 1;
  if (a.exact < 1 || a.max_dist <= a.exact || a.n_thr >= kMaxThr || n < 7 + a.n_thr) return false;
  for (int i = 0; i < a.n_thr; ++i) a.thr[i] = (int)w[7 + i];
  return true;
}

}  // namespace

DTF_API int dtf_relative_bias_fwd(const long long* words, int n_words, const void* table, void* out, int dtype,
                                  hipStream_t stream) {
  BiasArgs a = {};
  if (!unpack(words, n_words, a)) return -1;
  const dim3 grid((unsigned)min(a.Sq, 65535), (unsigned)a.heads);
  const size_t lds = (size_t)(a.max_dist + a.right + 1) * (dtype ? 2 : 4);
  if (dtype) hipLaunchKernelGGL(bias_fwd_kernel<unsigned short>, grid, dim3(256), lds, stream, a, (const unsigned short*)table, (unsigned short*)out);
  else hipLaunchKernelGGL(bias_fwd_kernel<float>, grid, dim3(256), lds, stream, a, (const float*)table, (float*)out);
  return (int)hipGetLastError();
}

// Partial sums that the backward pass writes, in units of buckets * heads floats.
DTF_API int dtf_relative_bias_parts(int Sq, int Sk) { return (Sq + kRowsPerBlock - 1) / kRowsPerBlock; }

DTF_API int dtf_relative_bias_bwd(const long long* words, int n_words, const void* g, float* parts, void* dtable, int dtype,
                                  hipStream_t stream) {
  BiasArgs a = {};
  if (!unpack(words, n_words, a)) return -1;
  const int n_parts = dtf_relative_bias_parts(a.Sq, a.Sk);
  const dim3 grid((unsigned)n_parts, (unsigned)a.heads);
  const size_t lds = (size_t)(a.max_dist + a.right + 1) * 4;
  if (dtype) hipLaunchKernelGGL(bias_bwd_kernel<unsigned short>, grid, dim3(256), lds, stream, a, (const unsigned short*)g, parts);
  else hipLaunchKernelGGL(bias_bwd_kernel<float>, grid, dim3(256), lds, stream, a, (const float*)g, parts);
  if (dtype) hipLaunchKernelGGL(bias_finish_kernel<unsigned short>, dim3(a.heads), dim3(256), 0, stream, parts, (unsigned short*)dtable, n_parts, a.heads, a.buckets);
  else hipLaunchKernelGGL(bias_finish_kernel<float>, dim3(a.heads), dim3(256), 0, stream, parts, (float*)dtable, n_parts, a.heads, a.buckets);
  return (int)hipGetLastError();
}
