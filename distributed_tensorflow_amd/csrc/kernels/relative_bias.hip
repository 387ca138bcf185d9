// Learned relative position bias by buckets, written out (gfx950).
//
//   forward : out[h, i, j] = table[bucket(j - (q_start + i)), h]
//   backward: dtable[u, h] = sum of g[h, i, j] over the (i, j) whose distance has bucket u
//
// Both are bound by the one pass over [heads, q_len, k_len]: 2 or 4 bytes an element against a lookup or an addition. The
// bias depends on the distance alone, so a workgroup keeps its head's values by distance in the LDS (a band of
// 2 max_distance + 1, with a constant on either side).
//
// Measured in bf16: 16 heads x 4099 x 4099 written in 101 us (5.3 TB/s; a copy reaches 5.3), its gradient summed in 127
// (4.2 TB/s; 64 elements a lane on 15 diagonals in registers, one LDS addition a diagonal on the band only: with an LDS
// addition an element it took 486), 12 heads x 512 x 512 in 10 and 11 us, launches and the host's work more than that.
#include "dtf_common.h"

using namespace dtf;

namespace {

constexpr int kMaxThr = 64;

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

// the distances of bucket u, inclusive (none: lo > hi)
__device__ __forceinline__ void bucket_range(const BiasArgs& a, int u, int& lo, int& hi) {
  const bool pos = a.right && u >= a.half;
  const int t = pos ? u - a.half : u, far = 0x3fffffff;
  const int from = t <= a.exact ? t : a.thr[t - a.exact - 1];
  const int to = t == a.half - 1 ? far : (t < a.exact ? t : a.thr[t - a.exact] - 1);
  lo = pos ? (from < 1 ? 1 : from) : -to;
  hi = pos ? to : (!a.right && t == 0 ? far : -from);
}

// STREAM: stores that leave no dirty lines in the caches, for a bias larger than those (see dtf_relative_bias_fwd). They go
// out 16 bytes a lane, from the first aligned address of a row on (2 bytes a lane took 185 us for 16 x 4099 x 4099).
template <typename T, bool STREAM>
__global__ __launch_bounds__(256) void bias_fwd_kernel(BiasArgs a, const T* __restrict__ table, T* __restrict__ out) {
  constexpr int V = 16 / (int)sizeof(T);
  typedef T vec_t __attribute__((ext_vector_type(V)));
  extern __shared__ __attribute__((aligned(16))) char smem[];
  T* band = reinterpret_cast<T*>(smem);                  // values of the distances -max_dist .. right
  const int tid = threadIdx.x, h = blockIdx.y;
  for (int i = tid; i <= a.max_dist + a.right; i += 256) band[i] = table[(long long)bucket_of(a, i - a.max_dist) * a.heads + h];
  __syncthreads();
  const T left = band[0], right = band[a.max_dist + a.right];
  for (long long i = blockIdx.x; i < a.Sq; i += gridDim.x) {
    T* row = out + ((long long)h * a.Sq + i) * a.Sk;
    const int pos = a.start + (int)i;
    auto value = [&](int j) { return band[min(max(j - pos, -a.max_dist), a.right) + a.max_dist]; };
    const int head = min((int)((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / (int)sizeof(T), a.Sk), n = (a.Sk - head) / V;
    if (tid < head) row[tid] = value(tid);
    for (int c = tid; c < n; c += 256) {
      const int j = head + c * V, d = j - pos;
      vec_t v;
      if (d + V - 1 <= -a.max_dist) v = left;
      else if (d >= a.right) v = right;
      else {
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = value(j + e);
      }
      if (STREAM) __builtin_nontemporal_store(v, reinterpret_cast<vec_t*>(row + j));
      else *reinterpret_cast<vec_t*>(row + j) = v;
    }
    for (int j = head + n * V + tid; j < a.Sk; j += 256) row[j] = value(j);
  }
}

// 8 elements of a row from column j on; zero from column n on. The rows have any alignment: the load is left to the
// compiler, which reads 16 bytes at once at an address of any alignment.
__device__ __forceinline__ void load8(const unsigned short* row, int j, int n, float (&o)[8]) {
  if (j + 8 <= n) {
    u16x8 v;
    __builtin_memcpy(&v, row + j, 16);
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = bf16_to_f32(v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = j + i < n ? bf16_to_f32(row[j + i]) : 0.f;
  }
}
__device__ __forceinline__ void load8(const float* row, int j, int n, float (&o)[8]) {
  if (j + 8 <= n) {
    __builtin_memcpy(o, row + j, 32);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = j + i < n ? row[j + i] : 0.f;
  }
}

// A wave takes tiles of 8 rows x 512 columns, a lane 8 x 8 of them: 64 elements on 15 diagonals, which it adds up in
// registers. Where the 15 distances are all on one far side (most of a long row) they go into one register; on the band
// they go to the wave's own LDS sums, 15 additions with the lanes 8 distances apart (the sums are stored by distance
// modulo 8 first, so that they fall on neighbouring banks). No sum depends on another wave: the order is fixed. Additions 0
// to 7 of a tile meet no word twice, nor do 8 to 14, but a lane's second eight are its neighbour's first: between the two, and
// between tiles, wave_ordered() keeps the compiler from moving one lane's read before another's write.
template <typename T>
__global__ __launch_bounds__(256) void bias_bwd_kernel(BiasArgs a, const T* __restrict__ g, float* __restrict__ parts,
                                                       int tiles_per_wave, int col_tiles, long long n_tiles) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6, h = blockIdx.y;
  const int n = a.max_dist + a.right + 1, eighth = (n + 14) / 8 + 1, size = eighth * 8;   // distances -max_dist - 7 ..
  float* sums = reinterpret_cast<float*>(smem) + wid * size;
  for (int i = lane; i < size; i += 64) sums[i] = 0.f;
  wave_ordered();
  float far_l = 0.f, far_r = 0.f;
  const long long first = ((long long)blockIdx.x * 4 + wid) * tiles_per_wave;
  for (long long t = first; t < first + tiles_per_wave && t < n_tiles; ++t) {
    const int i0 = (int)(t / col_tiles) * 8, j0 = (int)(t % col_tiles) * 512 + lane * 8;
    float acc[15];
#pragma unroll
    for (int d = 0; d < 15; ++d) acc[d] = 0.f;
    const T* row = g + ((long long)h * a.Sq + i0) * a.Sk;
    if (j0 < a.Sk) {
#pragma unroll
      for (int r = 0; r < 8; ++r)
        if (i0 + r < a.Sq) {
          float v[8];
          load8(row + (long long)r * a.Sk, j0, a.Sk, v);
#pragma unroll
          for (int c = 0; c < 8; ++c) acc[c - r + 7] += v[c];
        }
    }
    const int low = j0 - (a.start + i0) - 7;                               // distance of acc[0]
    if (low + 14 <= -a.max_dist || low >= a.right) {
      float v = 0.f;
#pragma unroll
      for (int d = 0; d < 15; ++d) v += acc[d];
      if (low < 0) far_l += v; else far_r += v;
    } else {
#pragma unroll
      for (int d = 0; d < 15; ++d) {
        // (distances beyond the borders belong to the outermost entries' buckets like these)
        const int i = min(max(low + d, -a.max_dist), a.right) + a.max_dist;
        if (low + d <= -a.max_dist) far_l += acc[d];
        else if (low + d >= a.right) far_r += acc[d];
        else sums[(i & 7) * eighth + (i >> 3)] += acc[d];
        if (d == 7) wave_ordered();
      }
    }
    wave_ordered();
  }
  __shared__ float scratch[16];
  far_l = block_sum(far_l, scratch);
  far_r = block_sum(far_r, scratch);
  __syncthreads();
  float* all = reinterpret_cast<float*>(smem);
  for (int i = tid; i < size; i += 256) all[i] = (all[i] + all[size + i]) + (all[2 * size + i] + all[3 * size + i]);
  __syncthreads();
  // a bucket's distances that lie strictly between the borders, shared out over the lanes of a group, then the far sums
  int lanes = 64;
  while (lanes * a.buckets > 256) lanes >>= 1;
  const int u = tid / lanes, part = tid & (lanes - 1);
  if (u < a.buckets) {
    float v = 0.f;
    int lo, hi;
    bucket_range(a, u, lo, hi);
    for (int d = max(lo, 1 - a.max_dist) + part; d <= min(hi, a.right - 1); d += lanes) {
      const int i = d + a.max_dist;
      v += all[(i & 7) * eighth + (i >> 3)];
    }
    for (int o = lanes >> 1; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    if (lo <= -a.max_dist && hi >= -a.max_dist) v += far_l;
    if (hi >= a.right && lo <= a.right) v += far_r;
    if (part == 0) parts[((long long)blockIdx.x * a.heads + h) * a.buckets + u] = v;
  }
}

template <typename T>
__global__ __launch_bounds__(256) void bias_finish_kernel(const float* __restrict__ parts, T* __restrict__ out, int n_parts,
                                                         int heads, int buckets) {
  __shared__ float red[256];
  const int h = blockIdx.x, slices = 256 / buckets, u = threadIdx.x % buckets, s = threadIdx.x / buckets;
  float v = 0.f;
  if (s < slices) {
#pragma unroll 8
    for (int p = s; p < n_parts; p += slices) v += parts[((long long)p * heads + h) * buckets + u];
  }
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

int tiles_per_wave(long long tiles, int heads) {
  const long long per = tiles * heads / (256 * 32);
  return (int)(per < 1 ? 1 : per);
}

}  // namespace

DTF_API int dtf_relative_bias_fwd(const long long* words, int n_words, const void* table, void* out, int dtype,
                                  hipStream_t stream) {
  BiasArgs a = {};
  if (!unpack(words, n_words, a)) return -1;
  const dim3 grid((unsigned)min(a.Sq, 65535), (unsigned)a.heads);
  const size_t lds = (size_t)(a.max_dist + a.right + 1) * (dtype ? 2 : 4);
  // A bias well beyond the 256 MiB last-level cache is streamed past it: what reads it next, or the gradient next to it, does
  // not wait for its dirty lines (16 heads, cached / streamed, us: 374 MiB written and read 313 / 280, with a gradient of
  // this size 221 / 174; 513 MiB 410 / 384, 263 / 240; smaller ones are better kept: 128 MiB written and read 98 / 115,
  // 256 MiB 96 / 122).
  const bool big = (long long)a.heads * a.Sq * a.Sk * (dtype ? 2 : 4) > 320LL << 20;
#define BIAS(T, STREAM) hipLaunchKernelGGL((bias_fwd_kernel<T, STREAM>), grid, dim3(256), lds, stream, a, (const T*)table, (T*)out)
  if (dtype) { if (big) BIAS(unsigned short, true); else BIAS(unsigned short, false); }
  else { if (big) BIAS(float, true); else BIAS(float, false); }
#undef BIAS
  return (int)hipGetLastError();
}

// Partial sums that the backward pass writes, in units of buckets * heads floats: one for each workgroup of a head. About
// eight waves a SIMD over all heads, each with as many tiles as that takes.
DTF_API int dtf_relative_bias_parts(int Sq, int Sk, int heads) {
  const long long tiles = (long long)((Sq + 7) / 8) * ((Sk + 511) / 512);
  const int per_wave = tiles_per_wave(tiles, heads);
  return (int)((tiles + 4LL * per_wave - 1) / (4LL * per_wave));
}

DTF_API int dtf_relative_bias_bwd(const long long* words, int n_words, const void* g, float* parts, void* dtable, int dtype,
                                  hipStream_t stream) {
  BiasArgs a = {};
  if (!unpack(words, n_words, a)) return -1;
  const int n_parts = dtf_relative_bias_parts(a.Sq, a.Sk, a.heads), col_tiles = (a.Sk + 511) / 512;
  const long long n_tiles = (long long)((a.Sq + 7) / 8) * col_tiles;
  const int per = tiles_per_wave(n_tiles, a.heads);
  const dim3 grid((unsigned)n_parts, (unsigned)a.heads);
  const size_t lds = (size_t)((a.max_dist + a.right + 1 + 14) / 8 + 1) * 8 * 4 * 4;
  const void* kernel = dtype ? (const void*)bias_bwd_kernel<unsigned short> : (const void*)bias_bwd_kernel<float>;
  if (lds > 64 * 1024) {
    const int rc = (int)hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (rc) return rc;
  }
  if (dtype) hipLaunchKernelGGL(bias_bwd_kernel<unsigned short>, grid, dim3(256), lds, stream, a, (const unsigned short*)g, parts, per, col_tiles, n_tiles);
  else hipLaunchKernelGGL(bias_bwd_kernel<float>, grid, dim3(256), lds, stream, a, (const float*)g, parts, per, col_tiles, n_tiles);
  if (dtype) hipLaunchKernelGGL(bias_finish_kernel<unsigned short>, dim3(a.heads), dim3(256), 0, stream, parts, (unsigned short*)dtable, n_parts, a.heads, a.buckets);
  else hipLaunchKernelGGL(bias_finish_kernel<float>, dim3(a.heads), dim3(256), 0, stream, parts, (float*)dtable, n_parts, a.heads, a.buckets);
  return (int)hipGetLastError();
}
