// Log probabilities of given tokens, the entropy, and the top alternatives of each row of logits (gfx950).
//
//   lse = log sum_v exp x_v;  logp = x[token] - lse;  H = -sum_v p_v log p_v;  the k largest x_v (ties: lowest index first)
//   backward: dx_v = -p_v (g_logp + sum_j g_top_j + g_H (log p_v + H)) + g_logp [v = token] + sum_j g_top_j [v = id_j]
//
// Bound by the one read of the logits (and one write backward). A workgroup owns a row and walks it in chunks that stay
// in registers: 4 x 16 bytes a thread.
//   * With z = x - m and m the running maximum of the THREAD, s = sum e^z and w = sum e^z z need no other thread until
//     the row ends; H = log s - w / s then has two terms of one sign, so a row that is sure of one token (H near 0) keeps
//     its digits, which lse - sum p x would not.
//   * The top k: an element is a candidate when it is no less than a threshold that at least k elements of the row reach.
//     The first threshold is the k-th largest of 64 maxima over a sixty-fourth of the chunk each, later ones the k-th
//     best so far: about 1.4 k candidates come out of the first chunk and fewer from each later one, and only they are
//     ranked. A key of 64 bits (value in an order-preserving code, then the complement of the index) makes every
//     element's key unique, so the result does not depend on the order in which candidates arrive.
// Measured in bf16: 5120 x 30522 without alternatives 54 us (5.7 TB/s; a copy reaches 5.3), with 5 of them 73 to 91, backward
// 114; 2048 x 131072 with 20 135 (4.0 TB/s). Without alternatives the pass is bound by memory; with them by vector
// instructions: 10 an element for the sums (1197 of a wave's), 3 more for 5 alternatives, 7 for 20, counted.
#include "dtf_common.h"

using namespace dtf;

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kCap = 512;            // candidates held at a time
constexpr int kKeep = 40;            // with up to 24 alternatives they are ranked in one wave
constexpr int kMaxTop = 32;
constexpr int kMaxRows = (1 << 22) - 1;      // 1024 threads a row, below 2^32 in a launch
constexpr int kMaxCols = 1 << 30;
constexpr int kU = 4;                // 16-byte vectors a thread holds of a chunk
constexpr float kFloor = -200.f;     // e^-200 is 0 in fp32: log probabilities are held above it where they meet p

typedef unsigned long long u64;

template <typename T> struct Vec;
template <> struct Vec<float> {
  static constexpr int V = 4;
  static __device__ __forceinline__ float one(const float* p) { return *p; }
  static __device__ __forceinline__ float get(const u32x4_t& r, int i) { return __uint_as_float(r[i]); }
  static __device__ __forceinline__ float pick(const u32x4_t& r, int i) {     // i not known at compile time
    const unsigned a = i & 1 ? r[1] : r[0], b = i & 1 ? r[3] : r[2];
    return __uint_as_float(i & 2 ? b : a);
  }
  static __device__ __forceinline__ void put(float* p, float v) { *p = v; }
  static __device__ __forceinline__ void putv(float* p, const float (&o)[4]) { *reinterpret_cast<f32x4*>(p) = f32x4{o[0], o[1], o[2], o[3]}; }
};
template <> struct Vec<unsigned short> {
  static constexpr int V = 8;
  static __device__ __forceinline__ float one(const unsigned short* p) { return bf16_to_f32(*p); }
  static __device__ __forceinline__ float get(const u32x4_t& r, int i) {
    return __uint_as_float(i & 1 ? r[i >> 1] & 0xffff0000u : r[i >> 1] << 16);
  }
  static __device__ __forceinline__ float pick(const u32x4_t& r, int i) {
    const unsigned a = i & 2 ? r[1] : r[0], b = i & 2 ? r[3] : r[2], w = i & 4 ? b : a;
    return __uint_as_float(i & 1 ? w & 0xffff0000u : w << 16);
  }
  static __device__ __forceinline__ void put(unsigned short* p, float v) { *p = f32_to_bf16(v); }
  static __device__ __forceinline__ void putv(unsigned short* p, const float (&o)[8]) { store8_bf16(p, o); }
};

// ascending with the value; NaN above everything, -0 equal to +0; equal values descend with the index
__device__ __forceinline__ u64 key_of(float x, int index) {
  unsigned b = __float_as_uint(x);
  if (b == 0x80000000u) b = 0u;
  unsigned o = (b >> 31) ? ~b : b | 0x80000000u;
  if (x != x) o = 0xffffffffu;
  return ((u64)o << 32) | (unsigned)~index;
}
__device__ __forceinline__ float value_of(u64 key) {
  const unsigned o = (unsigned)(key >> 32);
  return __uint_as_float((o >> 31) ? o & 0x7fffffffu : ~o);
}
// lane src's value (src the same in every lane), without a trip through the LDS
__device__ __forceinline__ u64 lane_u64(u64 v, int src) {
  const unsigned lo = __builtin_amdgcn_readlane((int)(unsigned)v, src), hi = __builtin_amdgcn_readlane((int)(unsigned)(v >> 32), src);
  return ((u64)hi << 32) | lo;
}
__device__ __forceinline__ u64 shfl_xor_u64(u64 v, int m) {
  const unsigned lo = __shfl_xor((int)(unsigned)v, m, 64), hi = __shfl_xor((int)(unsigned)(v >> 32), m, 64);
  return ((u64)hi << 32) | lo;
}

// the largest of three, a NaN if one of them is
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("v_maximum3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

// x - m - ls, the first difference first: x and m are near each other, however far from zero. The build allows the compiler to
// reassociate, and x - (m + ls), one instruction less where m + ls is the row's, loses digits with the distance from zero
// (1e-3 at logits of 30000, all of ls in a row of lowest values).
__device__ __forceinline__ float log_prob(float x, float m, float ls) {
  float z = x - m;
  asm("" : "+v"(z));
  return z - ls;
}

struct Shared {
  u64 cand[kCap];
  u64 best[kMaxTop];                 // the k best so far, descending
  u64 sorted[kMaxTop];
  u64 group[64];
  u64 threshold;
  int count;
  float red[3][16];
};

// The k best of cand[0 .. n) and best[0 .. nb), by counting the greater ones: one wave. Its lanes read what others wrote.
__device__ __forceinline__ void rank_candidates(Shared& sh, int n, int nb, int k, int lane) {
  const int total = n + nb;
  if (total <= 64) {                                     // almost always
    const u64 mine = lane < n ? sh.cand[lane] : (lane < total ? sh.best[lane - n] : 0ull);
    int rank = 0;
    for (int j = 0; j < total; ++j) rank += lane_u64(mine, j) > mine ? 1 : 0;
    wave_ordered();
    if (lane < total && rank < k) sh.best[rank] = mine;
    wave_ordered();
    return;
  }
  for (int c = 0; c < total; c += 64) {
    const int i = c + lane;
    const u64 mine = i < n ? sh.cand[i] : (i < total ? sh.best[i - n] : 0ull);
    int rank = 0;
    for (int j = 0; j < total; ++j) rank += (j < n ? sh.cand[j] : sh.best[j - n]) > mine ? 1 : 0;
    if (i < total && rank < k) sh.sorted[rank] = mine;
  }
  wave_ordered();
  if (lane < (total < k ? total : k)) sh.best[lane] = sh.sorted[lane];
  wave_ordered();
}

template <typename T, typename L, int NT, bool TOP>
__global__ __launch_bounds__(NT, 6) void token_logp_fwd_kernel(const T* __restrict__ x, const L* __restrict__ tokens,
                                                            float* __restrict__ logp, float* __restrict__ entropy,
                                                            float* __restrict__ top_logp, long long* __restrict__ top_ids,
                                                            float* __restrict__ stat, int N, int C, long long ld, int k) {
  constexpr int V = Vec<T>::V, W = NT / 64;
  __shared__ Shared sh;
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  const long long row = blockIdx.x;
  const T* xr = x + row * ld;
  int head = (int)(((16 - (reinterpret_cast<uintptr_t>(xr) & 15)) & 15) / sizeof(T));
  head = head < C ? head : C;
  const int nvec = (C - head) / V, tail = C - head - nvec * V;
  const T* body = xr + head;
  // the elements before and after the 16-byte vectors: at most V - 1 of each, one a thread
  const int odd = tid < head ? tid : (tid >= 16 && tid - 16 < tail ? head + nvec * V + tid - 16 : -1);
  const float xo = odd >= 0 ? Vec<T>::one(xr + odd) : -INFINITY;

  float m = -INFINITY, s = 0.f, w = 0.f;
  int nb = 0, held = 0;                                  // entries of sh.best; candidates of earlier chunks not ranked yet
  u64 threshold = 0;
  if (TOP && tid == 0) sh.count = 0;
  if (TOP) __syncthreads();

  for (int base = 0; base == 0 || base < nvec; base += NT * kU) {
    u32x4_t r[kU];
    bool in[kU];
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int j = base + u * NT + tid;
      in[u] = j < nvec;
      if (in[u]) r[u] = *reinterpret_cast<const u32x4_t*>(body + (long long)j * V);
    }
    // running maximum, sum and sum of e^z z of this thread's elements; the maximum of each vector is kept for the search
    const bool own = base == 0 && odd >= 0;
    float vm[kU], cm = own ? xo : -INFINITY;
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      vm[u] = -INFINITY;
      if (in[u]) {
#pragma unroll
        for (int i = 0; i < V; i += 2) vm[u] = max3(vm[u], Vec<T>::get(r[u], i), Vec<T>::get(r[u], i + 1));
      }
    }
#pragma unroll
    for (int u = 0; u < kU; u += 2) cm = max3(cm, vm[u], vm[u + 1]);
    const float mn = max3(m, m, cm), ref = mn == -INFINITY ? 0.f : mn;
    const float shift = m == -INFINITY ? kFloor : fmaxf(m - ref, kFloor), alpha = __builtin_amdgcn_exp2f(shift * kLog2e);
    w = alpha * fmaf(s, shift, w);
    s = alpha * s;
    m = mn;
    auto add = [&](float v) {
      float z = v - ref;
      z = max3(z, z, kFloor);
      const float e = __builtin_amdgcn_exp2f(z * kLog2e);
      s += e;
      w = fmaf(e, z, w);
    };
    if (own) add(xo);
#pragma unroll
    for (int u = 0; u < kU; ++u)
      if (in[u]) {
#pragma unroll
        for (int i = 0; i < V; ++i) add(Vec<T>::get(r[u], i));
      }
    if (!TOP) continue;

    const bool some = in[0] || own;      // (chunks are filled from the front)
    if (base == 0) {
      // first threshold: k-th largest of 64 maxima. The index in a thread's key is that of its first vector element where
      // this is the maximum, otherwise C or more: no element with the maximum has a lower key. An empty group has key 0
      u64 key = 0ull;
      if (some) key = key_of(cm, in[0] && cm == Vec<T>::get(r[0], 0) ? head + tid * V : C + tid);
#pragma unroll
      for (int o = 1; o < W; o <<= 1) {
        const u64 other = shfl_xor_u64(key, o);
        key = other > key ? other : key;
      }
      if (W > 1) {
        if (lane % W == 0) sh.group[wid * (64 / W) + lane / W] = key;
        __syncthreads();
      }
      if (wid == 0) {
        if (W > 1) key = sh.group[lane];
        // the value bit by bit (a value of 16 bits has 16; below them a NaN's or a negative one's are all set). Where the
        // last of the k is one of several equal groups, those of the lowest indexes are taken
        constexpr unsigned kLow = sizeof(T) == 2 ? 0xffffu : 0u;
        const unsigned value = (unsigned)(key >> 32) | kLow;
        unsigned kth = kLow;
#pragma unroll
        for (unsigned bit = 0x80000000u; bit > kLow; bit >>= 1)
          if (__popcll(__ballot(value >= (kth | bit))) >= k) kth |= bit;
        const u64 equal = __ballot(value == kth);
        const int need = k - __popcll(__ballot(value > kth));
        const bool taken = value == kth && __popcll(equal & ((1ull << lane) - 1)) < need;
        const bool vague = __ballot(taken && (unsigned)~(unsigned)key >= (unsigned)C) != 0ull;
        // the lowest key of those taken: indexes ascend with the lane, but for the ones of C or more
        const u64 lanes = __ballot(taken);
        const u64 last = lane_u64(key, 63 - __builtin_clzll(lanes));
        if (lane == 0) sh.threshold = vague ? last & ~0xffffffffull : last;
      }
      __syncthreads();
      threshold = sh.threshold;
    }
    for (;;) {
      const float tv = value_of(threshold);
      // threshold 0: everything passes (value_of(0) is a NaN, which no element is below)
      auto offer = [&](float v, int index) {
        const u64 key = key_of(v, index);
        if (key < threshold) return;
        const int at = atomicAdd(&sh.count, 1);
        if (at < kCap) sh.cand[at] = key;
      };
      if (own && !(xo < tv)) offer(xo, odd);
#pragma unroll
      for (int u = 0; u < kU; ++u)
        if (in[u] && !(vm[u] < tv)) {
          // the elements are converted again, not kept in 32 registers from the sums above
          asm volatile("" : "+v"(r[u]));
          unsigned pass = 0;
#pragma unroll
          for (int i = 0; i < V; ++i) pass |= Vec<T>::get(r[u], i) < tv ? 0u : 1u << i;
          while (pass) {
            const int i = __builtin_ctz(pass);
            pass &= pass - 1;
            offer(Vec<T>::pick(r[u], i), head + (base + u * NT + tid) * V + i);
          }
        }
      __syncthreads();
      const int count = sh.count;
      __syncthreads();                                   // (the next chunk counts on)
      // ranked when they no longer fit a wave, and at the row's end
      if (count <= kKeep && base + NT * kU < nvec) {
        held = count;
        break;
      }
      if (count <= kCap) {
        if (wid == 0) rank_candidates(sh, count, nb, k, lane);
        nb = min(nb + count, k);
        held = 0;
        if (base + NT * kU >= nvec) break;
        __syncthreads();
        if (nb == k) threshold = sh.best[k - 1] + 1;     // later elements have to beat the k-th
        if (tid == 0) sh.count = 0;
        __syncthreads();
        break;
      }
      // too many (whole ranges of equal or ordered values): the k-th best of those held is a higher threshold that k
      // elements still reach. Take the chunk again with it; at least kCap - kKeep - k candidates fall away each time.
      // Those held from earlier chunks stay, before the ones that come again
      if (wid == 0) {
        const u64 kept = lane < nb ? sh.best[lane] : 0ull;
        wave_ordered();
        rank_candidates(sh, kCap, nb, k, lane);
        if (lane == 0) sh.threshold = sh.best[k - 1];
        wave_ordered();
        if (lane < nb) sh.best[lane] = kept;
        if (lane == 0) sh.count = held;
      }
      __syncthreads();
      threshold = sh.threshold;
    }
  }

  // merge the threads' (m, s, w)
  float gm = wave_max(m);
  if (lane == 0) sh.red[0][wid] = gm;
  __syncthreads();
  gm = sh.red[0][0];
#pragma unroll
  for (int i = 1; i < W; ++i) gm = fmaxf(gm, sh.red[0][i]);
  {
    const float ref = gm == -INFINITY ? 0.f : gm;
    const float shift = m == -INFINITY ? kFloor : fmaxf(m - ref, kFloor), alpha = __builtin_amdgcn_exp2f(shift * kLog2e);
    w = wave_sum(alpha * fmaf(s, shift, w));
    s = wave_sum(alpha * s);
  }
  if (lane == 0) { sh.red[1][wid] = s; sh.red[2][wid] = w; }
  __syncthreads();
  s = 0.f;
  w = 0.f;
#pragma unroll
  for (int i = 0; i < W; ++i) { s += sh.red[1][i]; w += sh.red[2][i]; }
  const bool empty = gm == -INFINITY && s == 0.f;        // every logit -inf: no distribution
  if (wid != 0) return;
  const float ref = empty ? 0.f : gm, ls = empty ? 0.f : (float)log((double)s);
  if (lane == 0) {
    const long long tok = (long long)tokens[row];
    float lp = 0.f;
    if (tok >= 0 && tok < C) lp = log_prob(Vec<T>::one(xr + tok), ref, ls);
    logp[row] = lp;
    entropy[row] = empty ? 0.f : ls - w / s;
    if (stat) {
      stat[row] = empty ? -INFINITY : gm;
      stat[(long long)N + row] = ls;
    }
  }
  if (TOP && tid < k) {
    const u64 key = sh.best[tid];
    const int index = (int)~(unsigned)key;
    top_ids[row * k + tid] = index;
    top_logp[row * k + tid] = log_prob(Vec<T>::one(xr + index), ref, ls);
  }
}

template <typename T, typename L, int NT>
__global__ __launch_bounds__(NT) void token_logp_bwd_kernel(const T* __restrict__ x, const L* __restrict__ tokens,
                                                            const float* __restrict__ stat, const float* __restrict__ entropy,
                                                            const long long* __restrict__ top_ids,
                                                            const float* __restrict__ g_logp, const float* __restrict__ g_ent,
                                                            const float* __restrict__ g_top, T* __restrict__ dx, int N, int C,
                                                            long long ld, int k) {
  constexpr int V = Vec<T>::V;
  __shared__ int ids[kMaxTop];
  __shared__ float gts[kMaxTop];
  const int tid = threadIdx.x;
  const long long row = blockIdx.x;
  const T* xr = x + row * ld;
  T* dr = dx + row * ld;
  const float m = stat[row], ls = stat[(long long)N + row], H = entropy[row];
  const long long tok64 = (long long)tokens[row];
  const int tok = tok64 >= 0 && tok64 < C ? (int)tok64 : -1;
  const float ga = g_logp && tok >= 0 ? g_logp[row] : 0.f, gh = g_ent ? g_ent[row] : 0.f;
  if (tid < k) {
    ids[tid] = (int)top_ids[row * k + tid];
    gts[tid] = g_top[row * k + tid];
  }
  __syncthreads();
  float all = ga;
  for (int j = 0; j < k; ++j) all += gts[j];
  // d = p (A + B log p), A = -(g_logp + sum g_top + g_H H), B = -g_H; a row without a distribution has no gradient
  const bool empty = m == -INFINITY;
  const float A = -fmaf(gh, H, all), B = -gh;
  auto grad = [&](float v) {
    float lp = log_prob(v, m, ls);
    lp = lp < kFloor ? kFloor : lp;
    return empty ? 0.f : __builtin_amdgcn_exp2f(lp * kLog2e) * fmaf(B, lp, A);
  };
  int head = (int)(((16 - (reinterpret_cast<uintptr_t>(xr) & 15)) & 15) / sizeof(T));
  head = head < C ? head : C;
  const int nvec = (C - head) / V;
  if (tid < head) Vec<T>::put(dr + tid, grad(Vec<T>::one(xr + tid)));
  for (int j = tid; j < nvec; j += NT) {
    const u32x4_t r = *reinterpret_cast<const u32x4_t*>(xr + head + (long long)j * V);
    float o[V];
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = grad(Vec<T>::get(r, i));
    Vec<T>::putv(dr + head + (long long)j * V, o);
  }
  for (int i = head + nvec * V + tid; i < C; i += NT) Vec<T>::put(dr + i, grad(Vec<T>::one(xr + i)));
  for (long long i = C + tid; i < ld; i += NT) Vec<T>::put(dr + i, 0.f);      // padding between the rows
  if (empty) return;
  drain_stores();
  __syncthreads();
  // the elements that are the token or an alternative are written again, with their own terms
  if (tid < k) {
    const int v = ids[tid];
    Vec<T>::put(dr + v, grad(Vec<T>::one(xr + v)) + gts[tid] + (v == tok ? ga : 0.f));
  } else if (tid == k && tok >= 0) {
    bool listed = false;
    for (int j = 0; j < k; ++j) listed |= ids[j] == tok;
    if (!listed) Vec<T>::put(dr + tok, grad(Vec<T>::one(xr + tok)) + ga);
  }
}

// Threads a row. One wave for short rows (nothing to wait for at a barrier; 64 / 256 threads, us, bf16, 5 alternatives:
// 40000 x 4000 101 / 150, 20000 x 8000 85 / 89 and with 32 alternatives 143 / 120, 2048 x 131072 148 / 118), 1024
// where long rows are too few to fill the CUs (256 x 131072, 256 / 1024 threads: 38 / 26)
int fwd_threads(int N, int C) { return C <= 4096 ? 64 : N < 512 ? 1024 : 256; }
// Backward (64 / 256 / 1024 threads, us: 80000 x 2000 144 / 167 / 476, 20000 x 8000 134 / 120 / 166, 12000 x 16000
// 165 / 153 / 157, 5120 x 30522 143 / 136 / 127, 2048 x 131072 279 / 221 / 206: fewer rows at a time, written in longer runs)
int bwd_threads(int N, int C) { return C <= 2048 ? 64 : C > 16384 || (C > 4096 && N < 512) ? 1024 : 256; }

}  // namespace

// x [N, C] (row stride ld >= C; 0 fp32, 1 bf16), tokens [N] (0 int32, 1 int64; outside [0, C): logp 0), 0 <= k <= 32, k <= C.
// top_logp / top_ids [N, k] (unused when k is 0), stat (optional): fp32 [2, N] for the backward pass.
DTF_API int dtf_token_logp_fwd(const void* x, const void* tokens, float* logp, float* entropy, float* top_logp,
                               long long* top_ids, float* stat, int N, int C, long long ld, int k, int x_dtype,
                               int label_dtype, hipStream_t stream) {
  if (N <= 0) return 0;
  if (C <= 0 || ld < C || k < 0 || k > kMaxTop || k > C || N > kMaxRows || C > kMaxCols) return -1;
  const int nt = fwd_threads(N, C);
#define FWD(T, L, NT, TOP)                                                                                            \
  hipLaunchKernelGGL((token_logp_fwd_kernel<T, L, NT, TOP>), dim3(N), dim3(NT), 0, stream, (const T*)x, (const L*)tokens, \
                     logp, entropy, top_logp, top_ids, stat, N, C, ld, k)
#define FWD_L(T, L) \
  if (nt == 64) { if (k) FWD(T, L, 64, true); else FWD(T, L, 64, false); }        \
  else if (nt == 256) { if (k) FWD(T, L, 256, true); else FWD(T, L, 256, false); } \
  else { if (k) FWD(T, L, 1024, true); else FWD(T, L, 1024, false); }
  if (x_dtype == 0 && label_dtype == 0) { FWD_L(float, int) }
  else if (x_dtype == 0) { FWD_L(float, long long) }
  else if (label_dtype == 0) { FWD_L(unsigned short, int) }
  else { FWD_L(unsigned short, long long) }
#undef FWD_L
#undef FWD
  return (int)hipGetLastError();
}

// dx has x's row stride and its alignment modulo 16 bytes. A gradient may be null (0); g_top is needed when k > 0.
DTF_API int dtf_token_logp_bwd(const void* x, const void* tokens, const float* stat, const float* entropy,
                               const long long* top_ids, const float* g_logp, const float* g_ent, const float* g_top, void* dx,
                               int N, int C, long long ld, int k, int x_dtype, int label_dtype, hipStream_t stream) {
  if (N <= 0) return 0;
  if (C <= 0 || ld < C || k < 0 || k > kMaxTop || k > C || N > kMaxRows || C > kMaxCols || (k && (!g_top || !top_ids)))
    return -1;
  if ((reinterpret_cast<uintptr_t>(x) & 15) != (reinterpret_cast<uintptr_t>(dx) & 15)) return -2;
  const int nt = bwd_threads(N, C);
#define BWD(T, L, NT)                                                                                                  \
  hipLaunchKernelGGL((token_logp_bwd_kernel<T, L, NT>), dim3(N), dim3(NT), 0, stream, (const T*)x, (const L*)tokens, stat, \
                     entropy, top_ids, g_logp, g_ent, g_top, (T*)dx, N, C, ld, k)
#define BWD_L(T, L) if (nt == 64) BWD(T, L, 64); else if (nt == 256) BWD(T, L, 256); else BWD(T, L, 1024);
  if (x_dtype == 0 && label_dtype == 0) { BWD_L(float, int) }
  else if (x_dtype == 0) { BWD_L(float, long long) }
  else if (label_dtype == 0) { BWD_L(unsigned short, int) }
  else { BWD_L(unsigned short, long long) }
#undef BWD_L
#undef BWD
  return (int)hipGetLastError();
}
