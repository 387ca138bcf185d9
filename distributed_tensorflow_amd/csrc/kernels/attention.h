// Attention for general shapes (gfx950): bf16 and fp32, any lengths, causal, padded batches, additive key bias, a learned
// relative position bias by buckets, grouped key / value heads, strided operands. Forward and backward.
//
//   t[i, j] = scale * q_i . k_j + key_bias[b, j] + table[bucket(j - pos_i), h],   pos_i = q_start + i
//   j takes part for i when j < key_lengths[b], key_bias[b, j] != -inf and (causal) j <= pos_i
//   P = softmax_j t,  O = P V;  a row in which nothing takes part has O = 0 and all its gradients 0
//   backward: D_i = dO_i . O_i,  dP = dO V^T,  dT = P (dP - D),  dQ = scale dT K,  dK = scale dT^T Q,  dV = P^T dO,
//             dTable[u, h] = sum of dT over the batch and every (i, j) whose distance has bucket u
//
// Register-level layout, as in flash_attn.hip: S^T = K Q^T leaves in a lane the scores of ONE query (lane & 15) for four
// consecutive keys of each 16-key block, so the softmax is in-lane work plus two lane-group swaps, and the probabilities
// are, converted, the second operand of O^T = V^T P^T as they stand. bf16 uses v_mfma_f32_16x16x32_bf16; fp32 the exact
// v_mfma_f32_16x16x4_f32, eight of which cover the same 32 contraction elements (Frag below holds 8 elements of a lane
// for either type; the order of the 32 elements is free as long as both operands agree on it).
//
// Scores are kept in units of 1 / (scale log2 e): the biases are divided by that factor where they are staged and enter
// as the INITIAL VALUE of the score accumulators, so a bias costs no vector instruction per score.
#pragma once
#include "dtf_common.h"

namespace dtf {
namespace attn {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kRows = 128;           // rows (queries, or keys in the dK / dV kernel) of a workgroup: 4 waves x 32
constexpr int kMargin = 96;          // distances beyond the far borders that a 32 x 64 tile touching a border reaches
constexpr int kMaxThr = 64;
constexpr int kMaxStart = 1 << 29;   // positions and distances stay in 32 bits

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef short s16x4_f __attribute__((ext_vector_type(4)));
typedef short s16x8_f __attribute__((ext_vector_type(8)));

struct Strided {                     // [B, S, heads, hd] with unit stride in hd; strides in elements
  void* p;
  long long sb, ss, sh;
};

struct Args {
  Strided q, k, v, out, dout, dq, dk, dv;
  const float* key_bias;             // [B, Sk] or null
  const int* lens;                   // [B] or null
  const int* q_start;                // [B] or null (then q_start0 for every batch element)
  int q_start0;
  const void* table;                 // [buckets, nh] or null
  int table_bf16, buckets, half, exact, max_dist, right;   // right: max_dist when bidirectional, else 0
  int n_thr, thr[kMaxThr];           // thr[t]: smallest |distance| of bucket exact + 1 + t
  float* stat;                       // [2][B, nh, Sq]: row maximum (in score units with biases, else base 2), log2 of the row sum
  float* delta;                      // [B, nh, Sq] rowsum(dO * O)
  float* dtab;                       // [B * query tiles][nh][buckets] partial sums of the table's gradient, or null
  float* part;                       // few queries: partial results of the key splits
  int B, Sq, Sk, nh, nkv, hd, causal, splits;
  float scale;
};

template <typename T> struct Frag;
template <> struct Frag<unsigned short> { bf16x8_t v; };
template <> struct Frag<float> { f32x4 lo, hi; };

template <typename T> constexpr int key_tile() { return sizeof(T) == 2 ? 64 : 32; }
// LDS row strides in bytes. +16: the 16 rows of a ds_read_b128 fragment start 4 banks apart (mod 64) for every D.
template <typename T, int D> constexpr int row_stride() { return D * (int)sizeof(T) + 16; }

__device__ __forceinline__ f32x4 mma(const Frag<unsigned short>& a, const Frag<unsigned short>& b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v, b.v, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma(const Frag<float>& a, const Frag<float>& b, f32x4 c) {
#pragma unroll
  for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.lo[i], b.lo[i], c, 0, 0, 0);
#pragma unroll
  for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.hi[i], b.hi[i], c, 0, 0, 0);
  return c;
}

__device__ __forceinline__ float fexp2(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float flog2(float x) { return __builtin_amdgcn_logf(x); }

__device__ __forceinline__ void pack(Frag<unsigned short>& f, const f32x4& a, const f32x4& b) {
  const u32x4_t r = {pack_bf16x2(a[0], a[1]), pack_bf16x2(a[2], a[3]), pack_bf16x2(b[0], b[1]), pack_bf16x2(b[2], b[3])};
  f.v = __builtin_bit_cast(bf16x8_t, r);
}
__device__ __forceinline__ void pack(Frag<float>& f, const f32x4& a, const f32x4& b) { f.lo = a; f.hi = b; }

// 16 rows from row0 x 32 contraction elements ks of a tile image, 8 consecutive elements per lane
template <int STRIDE>
__device__ __forceinline__ void frag_row(Frag<unsigned short>& f, const char* img, int row0, int ks, int lane) {
  f.v = *reinterpret_cast<const bf16x8_t*>(img + (row0 + (lane & 15)) * STRIDE + ks * 64 + (lane >> 4) * 16);
}
template <int STRIDE>
__device__ __forceinline__ void frag_row(Frag<float>& f, const char* img, int row0, int ks, int lane) {
  const char* p = img + (row0 + (lane & 15)) * STRIDE + ks * 128 + (lane >> 4) * 32;
  f.lo = *reinterpret_cast<const f32x4*>(p);
  f.hi = *reinterpret_cast<const f32x4*>(p + 16);
}
// the transposed product's operand: column c0 + (lane & 15) of the image, its 32 rows ks in the order of pack(): rows
// 32 ks + 4 g .. +3, then 32 ks + 16 + 4 g .. +3 for lane group g
template <int STRIDE>
__device__ __forceinline__ void frag_tr(Frag<unsigned short>& f, const char* img, int c0, int ks, int lane) {
  const int g = lane >> 4, t = lane & 15, q = t >> 2, p = t & 3;
  const char* at = img + (ks * 32 + 4 * g + q) * STRIDE + c0 * 2 + p * 8;
  typedef __attribute__((address_space(3))) s16x4_f* lp_t;
  const s16x4_f lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp_t)at);
  const s16x4_f hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp_t)(at + 16 * STRIDE));
  const s16x8_f v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  f.v = __builtin_bit_cast(bf16x8_t, v);
}
template <int STRIDE>
__device__ __forceinline__ void frag_tr(Frag<float>& f, const char* img, int c0, int ks, int lane) {
  const char* at = img + (ks * 32 + 4 * (lane >> 4)) * STRIDE + (c0 + (lane & 15)) * 4;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f.lo[i] = *reinterpret_cast<const float*>(at + i * STRIDE);
    f.hi[i] = *reinterpret_cast<const float*>(at + (16 + i) * STRIDE);
  }
}

// 8 consecutive elements of one row straight from global memory; zero beyond the head size
__device__ __forceinline__ void frag_global(Frag<unsigned short>& f, const unsigned short* row, int e, bool ok) {
  const u32x4_t z = {0u, 0u, 0u, 0u};
  f.v = __builtin_bit_cast(bf16x8_t, ok ? *reinterpret_cast<const u32x4_t*>(row + e) : z);
}
__device__ __forceinline__ void frag_global(Frag<float>& f, const float* row, int e, bool ok) {
  const f32x4 z = {0.f, 0.f, 0.f, 0.f};
  f.lo = ok ? *reinterpret_cast<const f32x4*>(row + e) : z;
  f.hi = ok ? *reinterpret_cast<const f32x4*>(row + e + 4) : z;
}
__device__ __forceinline__ float dot(const Frag<unsigned short>& a, const Frag<unsigned short>& b, float s) {
#pragma unroll
  for (int i = 0; i < 8; ++i) s = fmaf((float)a.v[i], (float)b.v[i], s);
  return s;
}
__device__ __forceinline__ float dot(const Frag<float>& a, const Frag<float>& b, float s) {
#pragma unroll
  for (int i = 0; i < 4; ++i) s = fmaf(a.lo[i], b.lo[i], s);
#pragma unroll
  for (int i = 0; i < 4; ++i) s = fmaf(a.hi[i], b.hi[i], s);
  return s;
}
__device__ __forceinline__ void store4(unsigned short* p, const f32x4& v) { store4_bf16(p, v[0], v[1], v[2], v[3]); }
__device__ __forceinline__ void store4(float* p, const f32x4& v) { *reinterpret_cast<f32x4*>(p) = v; }

// over the 4 lanes that share lane & 15
__device__ __forceinline__ float group_max(float v) {
  const unsigned u = __float_as_uint(v);
  const u32x2_t r = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_permlane16_swap(u, u, false, false));
  const unsigned a = r[0], b = r[1];
  const unsigned w = __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
  const u32x2_t s = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_permlane32_swap(w, w, false, false));
  const unsigned c = s[0], d = s[1];
  return fmaxf(__uint_as_float(c), __uint_as_float(d));
}
__device__ __forceinline__ float group_sum(float v) {
  const unsigned u = __float_as_uint(v);
  const u32x2_t r = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_permlane16_swap(u, u, false, false));
  const unsigned a = r[0], b = r[1];
  const unsigned w = __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
  const u32x2_t s = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_permlane32_swap(w, w, false, false));
  const unsigned c = s[0], d = s[1];
  return __uint_as_float(c) + __uint_as_float(d);
}

// Tile of ROWS rows x D elements between global memory and a padded LDS image, through registers. Rows from `left` on and
// elements beyond the head size arrive as zeros: their addresses fail the buffer descriptor's range check. The
// descriptor covers one tile only, so offsets stay 32-bit whatever the tensor's size.
template <typename T, int D, int ROWS>
struct Tile {
  static constexpr int kChunk = 16 / (int)sizeof(T), kPerRow = D / kChunk, N = ROWS * kPerRow / 256;
  u32x4_t v[N];
  float kb[N];

  __device__ __forceinline__ void load(const T* base, long long ss, int left, int hd, int tid) {
    left = left < 0 ? 0 : (left > ROWS ? ROWS : left);
    const unsigned ldb = (unsigned)ss * (unsigned)sizeof(T);
    const unsigned bytes = left ? (unsigned)(left - 1) * ldb + (unsigned)hd * (unsigned)sizeof(T) : 0u;
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, (int)bytes, 0x00020000);
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const int p = u * 256 + tid, row = p / kPerRow, ch = p - row * kPerRow;
      const bool ok = ch * kChunk < hd && row < left;
      const unsigned off = ok ? (unsigned)row * ldb + (unsigned)ch * 16u : 0xffffffffu;
      v[u] = __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(rs, (int)off, 0, 0));
    }
  }
  // keys whose bias is -inf take no part whatever K and V hold there: their rows are zeroed on the way to the LDS
  __device__ __forceinline__ void load_bias(const float* bias, int left, int tid) {
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const int row = (u * 256 + tid) / kPerRow;
      kb[u] = row < left ? bias[row] : 0.f;
    }
  }
  __device__ __forceinline__ void store(char* img, int tid) const {
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const int p = u * 256 + tid, row = p / kPerRow, ch = p - row * kPerRow;
      *reinterpret_cast<u32x4_t*>(img + row * row_stride<T, D>() + ch * 16) = v[u];
    }
  }
  __device__ __forceinline__ void store_masked(char* img, int tid) const {
    const u32x4_t z = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const int p = u * 256 + tid, row = p / kPerRow, ch = p - row * kPerRow;
      *reinterpret_cast<u32x4_t*>(img + row * row_stride<T, D>() + ch * 16) = kb[u] == -INFINITY ? z : v[u];
    }
  }
};

// ---- relative position bias ------------------------------------------------------------------------------------
// The bias depends on the distance alone, and from max_dist on (right of the diagonal: `right`) it is one constant, so a
// head's bias is a band of max_dist + right + 1 values and two constants. A tile away from the band adds a constant.
__device__ __forceinline__ int band_size(const Args& a) { return a.max_dist + a.right + 1 + 2 * kMargin; }

__device__ __forceinline__ int bucket_of(const Args& a, int dist) {
  int far = a.right ? (dist < 0 ? -dist : dist) : (dist < 0 ? -dist : 0);
  int b = far;
  if (far >= a.exact) {
    b = a.exact;
    for (int t = 0; t < a.n_thr; ++t) b += far >= a.thr[t] ? 1 : 0;
  }
  return b + (a.right && dist > 0 ? a.half : 0);
}
__device__ __forceinline__ float table_at(const Args& a, int bucket, int h) {
  const long long i = (long long)bucket * a.nh + h;
  return a.table_bf16 ? bf16_to_f32(((const unsigned short*)a.table)[i]) : ((const float*)a.table)[i];
}
// a finite bias stays finite in score units, and so does that times scale log2 e: it is never taken for a masked key
__device__ __forceinline__ float to_score_units(const Args& a, float bias) {
  const float lim = 3.0e38f / fmaxf(1.f, a.scale * kLog2e);
  const float v = bias / a.scale;
  if (bias == -INFINITY) return bias;
  return v < -lim ? -lim : v;        // NaN and +inf pass
}
__device__ __forceinline__ void fill_band(const Args& a, int h, float* band, int tid) {
  const int n = band_size(a);
  for (int i = tid; i < n; i += 256) band[i] = to_score_units(a, table_at(a, bucket_of(a, i - kMargin - a.max_dist), h));
}
// the distances of bucket u, inclusive, clipped to the band
__device__ __forceinline__ void bucket_range(const Args& a, int u, int& lo, int& hi) {
  const int lowest = -a.max_dist - kMargin, highest = a.right + kMargin;
  const bool pos = a.right && u >= a.half;
  const int t = pos ? u - a.half : u;
  const int from = t <= a.exact ? t : a.thr[t - a.exact - 1];
  const int to = t == a.half - 1 ? 0x3fffffff : (t < a.exact ? t : a.thr[t - a.exact] - 1);
  if (pos) {
    lo = from < 1 ? 1 : from;
    hi = to;
  } else {
    lo = -to;
    hi = -from;
    if (!a.right && t == 0) hi = highest;
  }
  lo = lo < lowest ? lowest : lo;
  hi = hi > highest ? highest : hi;
}

// ---- work distribution -----------------------------------------------------------------------------------------
// Workgroups go round-robin to the 8 XCDs; give each XCD a contiguous range, so that the query tiles of one (batch,
// key head), which read the same K and V, share an L2.
__device__ __forceinline__ int xcd_contiguous(int bid, int n) {
  const int x = bid & 7, q = n >> 3, r = n & 7;
  return x * q + (x < r ? x : r) + (bid >> 3);
}

// ================================================================================================== forward
template <typename T, int D, bool BIAS>
__global__ __launch_bounds__(256, (sizeof(T) == 2 ? 2 : 1)) void fwd_kernel(Args a) {
  constexpr int KT = key_tile<T>(), JB = KT / 16, DB = D / 16, DS = D / 32, ST = row_stride<T, D>(), IMG = KT * ST;
  extern __shared__ __attribute__((aligned(16))) char smem[];      // [2][K | V], [2][key bias of the tile], band
  float* kbl = reinterpret_cast<float*>(smem + 4 * IMG);
  float* band = kbl + 2 * KT;
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int fr = lane & 15, g = lane >> 4;
  const int nqt = (a.Sq + kRows - 1) / kRows;
  const int id = xcd_contiguous(blockIdx.x, gridDim.x);
  const int qt = a.causal ? nqt - 1 - id % nqt : id % nqt, bh = id / nqt, b = bh / a.nh, h = bh - b * a.nh;
  const int kvh = h / (a.nh / a.nkv);
  const int q0 = qt * kRows + wid * 32;
  const int klen = a.lens ? min(max(a.lens[b], 0), a.Sk) : a.Sk;
  const int start = a.q_start ? min(max(a.q_start[b], -kMaxStart), kMaxStart) : a.q_start0;
  const int pos0 = start + q0;
  const float c = a.scale * kLog2e;
  const T* qp = (const T*)a.q.p + b * a.q.sb + h * a.q.sh;
  const T* kp = (const T*)a.k.p + b * a.k.sb + kvh * a.k.sh;
  const T* vp = (const T*)a.v.p + b * a.v.sb + kvh * a.v.sh;
  const float* kbp = BIAS && a.key_bias ? a.key_bias + (long long)b * a.Sk : nullptr;

  Frag<T> qf[2][DS];
#pragma unroll
  for (int qb = 0; qb < 2; ++qb) {
    const T* row = qp + (long long)min(q0 + qb * 16 + fr, a.Sq - 1) * a.q.ss;
#pragma unroll
    for (int ks = 0; ks < DS; ++ks) frag_global(qf[qb][ks], row, ks * 32 + g * 8, ks * 32 + g * 8 < a.hd);
  }
  f32x4 o[DB][2];
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int qb = 0; qb < 2; ++qb) o[db][qb] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

  // keys that any row of the workgroup sees
  const int last = start + min(qt * kRows + kRows, a.Sq) - 1;
  const int kend = a.causal ? min(klen, last + 1) : klen;
  const int nt = kend > 0 ? (kend + KT - 1) / KT : 0;

  Tile<T, D, KT> kr, vr;
  float kbr = 0.f;
  auto fetch = [&](int t) {
    kr.load(kp + (long long)t * KT * a.k.ss, a.k.ss, klen - t * KT, a.hd, tid);
    vr.load(vp + (long long)t * KT * a.v.ss, a.v.ss, klen - t * KT, a.hd, tid);
    if (BIAS && kbp) {
      kr.load_bias(kbp + t * KT, klen - t * KT, tid);
      vr.load_bias(kbp + t * KT, klen - t * KT, tid);
      if (tid < KT) kbr = t * KT + tid < klen ? to_score_units(a, kbp[t * KT + tid]) : -INFINITY;
    }
  };
  auto put = [&](int buf) {
    char* kimg = smem + buf * 2 * IMG;
    if (BIAS && kbp) {
      kr.store_masked(kimg, tid);
      vr.store_masked(kimg + IMG, tid);
      if (tid < KT) kbl[buf * KT + tid] = kbr;
    } else {
      kr.store(kimg, tid);
      vr.store(kimg + IMG, tid);
    }
  };
  if (BIAS && a.table) fill_band(a, h, band, tid);
  if (nt > 0) {
    fetch(0);
    put(0);
  }
  __syncthreads();
  for (int t = 0; t < nt; ++t) {
    const char* kimg = smem + (t & 1) * 2 * IMG;
    const char* vimg = kimg + IMG;
    const int kt = t * KT;
    if (t + 1 < nt) fetch(t + 1);
    // a wave whose rows all end before this tile, or that has no rows, only keeps step
    if (q0 < a.Sq && (!a.causal || kt <= pos0 + 31)) {
      f32x4 s[JB][2];
      if (BIAS) {
        const float* kb = kbl + (t & 1) * KT;
#pragma unroll
        for (int jb = 0; jb < JB; ++jb) {
          const f32x4 x = kbp ? *reinterpret_cast<const f32x4*>(kb + jb * 16 + g * 4) : f32x4{0.f, 0.f, 0.f, 0.f};
          s[jb][0] = x;
          s[jb][1] = x;
        }
        if (a.table) {
          if (kt + KT - 1 - pos0 <= -a.max_dist || kt - (pos0 + 31) >= a.right) {
            const float x = kt < pos0 ? band[0] : band[a.max_dist + a.right + 2 * kMargin];
#pragma unroll
            for (int jb = 0; jb < JB; ++jb) { s[jb][0] += x; s[jb][1] += x; }
          } else {
            const float* at = band + (kt + 4 * g - pos0 - fr + a.max_dist + kMargin);
            f32x4 x[JB + 1];
#pragma unroll
            for (int j = 0; j <= JB; ++j)
#pragma unroll
              for (int r = 0; r < 4; ++r) x[j][r] = at[(j - 1) * 16 + r];
#pragma unroll
            for (int jb = 0; jb < JB; ++jb) { s[jb][0] += x[jb + 1]; s[jb][1] += x[jb]; }
          }
        }
      } else {
#pragma unroll
        for (int jb = 0; jb < JB; ++jb) { s[jb][0] = f32x4{0.f, 0.f, 0.f, 0.f}; s[jb][1] = f32x4{0.f, 0.f, 0.f, 0.f}; }
      }
#pragma unroll
      for (int ks = 0; ks < DS; ++ks)
#pragma unroll
        for (int jb = 0; jb < JB; ++jb) {
          Frag<T> kf;
          frag_row<ST>(kf, kimg, jb * 16, ks, lane);
#pragma unroll
          for (int qb = 0; qb < 2; ++qb) s[jb][qb] = mma(kf, qf[qb][ks], s[jb][qb]);
        }
      if (kt + KT > klen || (a.causal && kt + KT - 1 > pos0)) {
#pragma unroll
        for (int qb = 0; qb < 2; ++qb) {
          const int end = a.causal ? min(klen, pos0 + qb * 16 + fr + 1) : klen;
#pragma unroll
          for (int jb = 0; jb < JB; ++jb)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (kt + jb * 16 + 4 * g + r >= end) s[jb][qb][r] = -INFINITY;
        }
      }
      Frag<T> pf[2][KT / 32];
#pragma unroll
      for (int qb = 0; qb < 2; ++qb) {
        float mx = -INFINITY;
#pragma unroll
        for (int jb = 0; jb < JB; ++jb)
#pragma unroll
          for (int r = 0; r < 4; ++r) mx = fmaxf(mx, s[jb][qb][r]);
        // scale > 0: the maximum commutes with the scaling. With biases the difference is taken in score units, where it
        // is exact: the product of a lowest-value mask with c is rounded by far more than 1
        const float mn = fmaxf(m[qb], BIAS ? group_max(mx) : group_max(mx) * c);
        const float ref = mn == -INFINITY ? 0.f : mn;                // nothing seen yet: every term below is exp2(-inf)
        const float alpha = fexp2(BIAS ? (m[qb] - ref) * c : m[qb] - ref);
        m[qb] = mn;
        float sum = 0.f;
#pragma unroll
        for (int jb = 0; jb < JB; ++jb)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float p = fexp2(BIAS ? (s[jb][qb][r] - ref) * c : fmaf(s[jb][qb][r], c, -ref));
            s[jb][qb][r] = p;
            sum += p;
          }
        l[qb] = l[qb] * alpha + sum;                                 // per lane; combined over the lane group at the end
#pragma unroll
        for (int db = 0; db < DB; ++db) o[db][qb] *= alpha;
#pragma unroll
        for (int ks = 0; ks < KT / 32; ++ks) pack(pf[qb][ks], s[2 * ks][qb], s[2 * ks + 1][qb]);
      }
#pragma unroll
      for (int ks = 0; ks < KT / 32; ++ks)
#pragma unroll
        for (int db = 0; db < DB; ++db) {
          Frag<T> vf;
          frag_tr<ST>(vf, vimg, db * 16, ks, lane);
#pragma unroll
          for (int qb = 0; qb < 2; ++qb) o[db][qb] = mma(vf, pf[qb][ks], o[db][qb]);
        }
    }
    if (t + 1 < nt) put((t + 1) & 1);
    __syncthreads();
  }
#pragma unroll
  for (int qb = 0; qb < 2; ++qb) {
    const int q = q0 + qb * 16 + fr;
    const float lt = group_sum(l[qb]);
    const float inv = lt == 0.f ? 0.f : 1.f / lt;
    if (q < a.Sq) {
      T* row = (T*)a.out.p + b * a.out.sb + (long long)q * a.out.ss + h * a.out.sh;
#pragma unroll
      for (int db = 0; db < DB; ++db)
        if (db * 16 + g * 4 < a.hd) store4(row + db * 16 + g * 4, o[db][qb] * inv);
      if (g == 0 && a.stat) {
        const long long i = ((long long)b * a.nh + h) * a.Sq + q, n = (long long)a.B * a.nh * a.Sq;
        a.stat[i] = lt == 0.f ? INFINITY : m[qb];       // +inf: exp2(t - inf) = 0 for a row with nothing in it
        a.stat[n + i] = lt == 0.f ? 0.f : flog2(lt);
      }
    }
  }
}

// ================================================================================================== few queries
// New tokens over a cache: at most 32 rows (queries x query heads of one key head), however many keys. Bound by the one
// read of K and V, so the keys are split over workgroups until these fill the chip, each wave walks key tiles of its own
// (32 keys, every fourth of its workgroup's), K goes from global memory straight into the product's operand, V through an
// LDS image of the wave's own, and no barrier stands in the loop. All query heads of a key head ride in one tile of rows,
// so the cache is read once, not once a query head. The waves' (maximum, sum, O) join in the LDS, the workgroups' in a
// second kernel.
constexpr int kFewRows = 32, kFewKeys = 32;

// O and the row's statistics of row r of a key head's rows
template <typename T, bool BIAS>
__device__ __forceinline__ void few_store(const Args& a, int b, int kvh, int group, int r, int d, float mm, float lt,
                                          const f32x4& acc, float c) {
  const int i = r / group, h = kvh * group + r - i * group;
  const float inv = lt == 0.f ? 0.f : 1.f / lt;
  if (d < a.hd) store4((T*)a.out.p + b * a.out.sb + (long long)i * a.out.ss + h * a.out.sh + d, acc * inv);
  if (d == 0 && a.stat) {
    const long long at = ((long long)b * a.nh + h) * a.Sq + i, n = (long long)a.B * a.nh * a.Sq;
    a.stat[at] = lt == 0.f ? INFINITY : (BIAS ? mm : mm * c);        // the units of fwd_kernel
    a.stat[n + at] = lt == 0.f ? 0.f : flog2(lt);
  }
}

template <typename T, int D, int QB, bool BIAS>
__global__ __launch_bounds__(256, 2) void few_kernel(Args a) {
  constexpr int DB = D / 16, DS = D / 32, ST = row_stride<T, D>(), IMG = kFewKeys * ST, JOIN = QB * 16 * (D + 4) * 4;
  constexpr int kChunk = 16 / (int)sizeof(T), kPerRow = D / kChunk, NV = kFewKeys * kPerRow / 64;
  extern __shared__ __attribute__((aligned(16))) char smem[];      // [4 waves][V image, then O], [4][2][rows], table
  constexpr int REGION = IMG > JOIN ? IMG : JOIN;
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int fr = lane & 15, g = lane >> 4;
  char* vimg = smem + wid * REGION;
  float* ml = reinterpret_cast<float*>(smem + 4 * REGION);
  float* tab = ml + 4 * 2 * QB * 16;
  const int group = a.nh / a.nkv, rows = a.Sq * group;
  const int split = blockIdx.x % a.splits, bk = blockIdx.x / a.splits, b = bk / a.nkv, kvh = bk - b * a.nkv;
  const int klen = a.lens ? min(max(a.lens[b], 0), a.Sk) : a.Sk;
  const int start = a.q_start ? min(max(a.q_start[b], -kMaxStart), kMaxStart) : a.q_start0;
  const float c = a.scale * kLog2e;
  const T* kp = (const T*)a.k.p + b * a.k.sb + kvh * a.k.sh;
  const T* vp = (const T*)a.v.p + b * a.v.sb + kvh * a.v.sh;
  const float* kbp = BIAS && a.key_bias ? a.key_bias + (long long)b * a.Sk : nullptr;

  if (BIAS && a.table) {
    for (int i = tid; i < group * a.buckets; i += 256) {
      const int hg = i / a.buckets;
      tab[i] = to_score_units(a, table_at(a, i - hg * a.buckets, kvh * group + hg));
    }
    __syncthreads();
  }
  Frag<T> qf[QB][DS];
  int pos[QB];
  const float* tb[QB];
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    const int r = min(qb * 16 + fr, rows - 1), i = r / group, hg = r - i * group;
    const T* row = (const T*)a.q.p + b * a.q.sb + (long long)i * a.q.ss + (kvh * group + hg) * a.q.sh;
    pos[qb] = start + i;
    tb[qb] = tab + hg * a.buckets;
#pragma unroll
    for (int ks = 0; ks < DS; ++ks) frag_global(qf[qb][ks], row, ks * 32 + g * 8, ks * 32 + g * 8 < a.hd);
  }
  f32x4 o[DB][QB];
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) o[db][qb] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m[QB], l[QB];
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) { m[qb] = -INFINITY; l[qb] = 0.f; }

  const int kend = a.causal ? min(klen, start + a.Sq) : klen;
  const int nt = kend > 0 ? (kend + kFewKeys - 1) / kFewKeys : 0, per = (nt + a.splits - 1) / a.splits;
  const int t1 = min(nt, (split + 1) * per);

  Frag<T> kf[2][DS];
  u32x4_t vr[NV];
  float kbv[NV];
  f32x4 kb[2];
  const unsigned kld = (unsigned)a.k.ss * (unsigned)sizeof(T), vld = (unsigned)a.v.ss * (unsigned)sizeof(T);
  auto rsrc = [&](const T* base, unsigned ld, int left) {
    left = min(left, kFewKeys);
    const unsigned bytes = (unsigned)(left - 1) * ld + (unsigned)a.hd * (unsigned)sizeof(T);
    return __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, (int)bytes, 0x00020000);
  };
  auto fetch = [&](int t) {                              // (left >= 1: the tile starts before kend)
    const int k0 = t * kFewKeys, left = klen - k0;
    const __amdgpu_buffer_rsrc_t kr = rsrc(kp + (long long)k0 * a.k.ss, kld, left), vs = rsrc(vp + (long long)k0 * a.v.ss, vld, left);
#pragma unroll
    for (int jb = 0; jb < 2; ++jb) {
      const int row = jb * 16 + fr;
      const bool in = row < left && !(BIAS && kbp && kbp[k0 + row] == -INFINITY);
#pragma unroll
      for (int ks = 0; ks < DS; ++ks) {
        const int e = ks * 32 + g * 8;
        const unsigned off = in && e < a.hd ? (unsigned)row * kld + (unsigned)e * (unsigned)sizeof(T) : 0xffffffffu;
        u32x4_t w[sizeof(Frag<T>) / 16];
#pragma unroll
        for (int i = 0; i < (int)sizeof(Frag<T>) / 16; ++i)
          w[i] = __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(kr, (int)(off == 0xffffffffu ? off : off + 16u * i), 0, 0));
        __builtin_memcpy(&kf[jb][ks], w, sizeof(Frag<T>));
      }
      if (BIAS && kbp) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int k = k0 + jb * 16 + 4 * g + r;
          kb[jb][r] = k < klen ? to_score_units(a, kbp[k]) : -INFINITY;
        }
      }
    }
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      const int p = u * 64 + lane, row = p / kPerRow, ch = p - row * kPerRow;
      const bool in = row < left && ch * kChunk < a.hd && !(BIAS && kbp && kbp[k0 + row] == -INFINITY);
      vr[u] = __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(vs, (int)(in ? (unsigned)row * vld + (unsigned)ch * 16u : 0xffffffffu), 0, 0));
    }
  };

  int t = split * per + wid;
  if (t < t1) fetch(t);
  for (; t < t1; t += 4) {
    const int kt = t * kFewKeys;
    f32x4 s[2][QB];
#pragma unroll
    for (int jb = 0; jb < 2; ++jb)
#pragma unroll
      for (int qb = 0; qb < QB; ++qb) {
        s[jb][qb] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (BIAS && kbp) s[jb][qb] = kb[jb];
        if (BIAS && a.table) {
#pragma unroll
          for (int r = 0; r < 4; ++r) s[jb][qb][r] += tb[qb][bucket_of(a, kt + jb * 16 + 4 * g + r - pos[qb])];
        }
      }
#pragma unroll
    for (int ks = 0; ks < DS; ++ks)
#pragma unroll
      for (int jb = 0; jb < 2; ++jb)
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) s[jb][qb] = mma(kf[jb][ks], qf[qb][ks], s[jb][qb]);
    // V of this tile to the LDS, the next tile's loads on their way (the LDS serves a wave in order: no barrier)
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      const int p = u * 64 + lane, row = p / kPerRow, ch = p - row * kPerRow;
      *reinterpret_cast<u32x4_t*>(vimg + row * ST + ch * 16) = vr[u];
    }
    if (t + 4 < t1) fetch(t + 4);
    Frag<T> pf[QB];
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
      const int end = a.causal ? min(klen, pos[qb] + 1) : klen;
      float mx = -INFINITY;
#pragma unroll
      for (int jb = 0; jb < 2; ++jb)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          if (kt + jb * 16 + 4 * g + r >= end) s[jb][qb][r] = -INFINITY;
          mx = fmaxf(mx, s[jb][qb][r]);
        }
      const float mn = fmaxf(m[qb], group_max(mx)), ref = mn == -INFINITY ? 0.f : mn;
      const float alpha = fexp2((m[qb] - ref) * c);
      m[qb] = mn;
      float sum = 0.f;
#pragma unroll
      for (int jb = 0; jb < 2; ++jb)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          s[jb][qb][r] = fexp2((s[jb][qb][r] - ref) * c);
          sum += s[jb][qb][r];
        }
      l[qb] = l[qb] * alpha + sum;
#pragma unroll
      for (int db = 0; db < DB; ++db) o[db][qb] *= alpha;
      pack(pf[qb], s[0][qb], s[1][qb]);
    }
    asm volatile("" ::: "memory");
#pragma unroll
    for (int db = 0; db < DB; ++db) {
      Frag<T> vf;
      frag_tr<ST>(vf, vimg, db * 16, 0, lane);
#pragma unroll
      for (int qb = 0; qb < QB; ++qb) o[db][qb] = mma(vf, pf[qb], o[db][qb]);
    }
    asm volatile("" ::: "memory");
  }
  // join the waves
  float* om = reinterpret_cast<float*>(vimg);
  asm volatile("" ::: "memory");
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    l[qb] = group_sum(l[qb]);
#pragma unroll
    for (int db = 0; db < DB; ++db) *reinterpret_cast<f32x4*>(om + (qb * 16 + fr) * (D + 4) + db * 16 + g * 4) = o[db][qb];
    if (g == 0) {
      ml[(wid * 2 + 0) * QB * 16 + qb * 16 + fr] = m[qb];
      ml[(wid * 2 + 1) * QB * 16 + qb * 16 + fr] = l[qb];
    }
  }
  __syncthreads();
  const long long n_rows = (long long)a.B * a.nkv * rows;
  for (int p = tid; p < rows * (D / 4); p += 256) {
    const int r = p / (D / 4), d = (p - r * (D / 4)) * 4;
    float mm = -INFINITY, lt = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) mm = fmaxf(mm, ml[w * 2 * QB * 16 + r]);
    const float ref = mm == -INFINITY ? 0.f : mm;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = fexp2((ml[w * 2 * QB * 16 + r] - ref) * c);
      lt += f * ml[(w * 2 + 1) * QB * 16 + r];
      acc += f * *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(smem + w * REGION) + r * (D + 4) + d);
    }
    const long long row = (long long)bk * rows + r;
    if (a.splits > 1) {
      // [split][row][D] of O over the split's own sum and maximum, then [split][2][row] of these
      if (d < a.hd) *reinterpret_cast<f32x4*>(a.part + ((long long)split * n_rows + row) * D + d) = acc;
      float* st = a.part + (long long)a.splits * n_rows * D + (long long)split * 2 * n_rows;
      if (d == 0) { st[row] = mm; st[n_rows + row] = lt; }
    } else {
      few_store<T, BIAS>(a, b, kvh, group, r, d, mm, lt, acc, c);
    }
  }
}

// One workgroup a row: its threads share out the row's splits as well as its elements, so that no thread waits for more
// than a few loads one after the other (one wave a row, walking the splits: 13.5 us where few_kernel itself takes 12).
template <typename T, int D, bool BIAS>
__global__ __launch_bounds__(256) void few_join_kernel(Args a) {
  constexpr int L = D / 4, S = 256 / L;                  // lanes of a row, splits taken at a time
  __shared__ __attribute__((aligned(16))) float red[S][D + 4];
  __shared__ float fac[64], stats[2];
  const int group = a.nh / a.nkv, rows = a.Sq * group, tid = threadIdx.x;
  const long long row = blockIdx.x, n_rows = gridDim.x;
  const float c = a.scale * kLog2e;
  const float* st = a.part + (long long)a.splits * n_rows * D;
  const int sub = tid / L, d = (tid - sub * L) * 4;
  if (tid < 64) {                                        // (at most 64 splits)
    const bool in = tid < a.splits;
    const float ms = in ? st[(long long)tid * 2 * n_rows + row] : -INFINITY;
    const float ls = in ? st[(long long)tid * 2 * n_rows + n_rows + row] : 0.f;
    const float mm = wave_max(ms), f = fexp2((ms - (mm == -INFINITY ? 0.f : mm)) * c);
    const float lt = wave_sum(f * ls);
    fac[tid] = f;
    if (tid == 0) { stats[0] = mm; stats[1] = lt; }
  }
  __syncthreads();
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  if (sub < S && d < a.hd)
    for (int s = sub; s < a.splits; s += S)
      acc += fac[s] * *reinterpret_cast<const f32x4*>(a.part + ((long long)s * n_rows + row) * D + d);
  if (sub < S) *reinterpret_cast<f32x4*>(&red[sub][d]) = acc;
  __syncthreads();
  if (sub == 0) {
    for (int s = 1; s < S && s < a.splits; ++s) acc += *reinterpret_cast<const f32x4*>(&red[s][d]);
    const int bk = (int)(row / rows), b = bk / a.nkv;
    few_store<T, BIAS>(a, b, bk - b * a.nkv, group, (int)(row - (long long)bk * rows), d, stats[0], stats[1], acc, c);
  }
}

// ================================================================================================== backward: dQ
// Sums over the diagonals of a wave's dT, for the relative bias's gradient. dT comes in blocks of 16 keys x 16 queries,
// lane (fr, g) holding query fr and keys 4 g + r; blocks on one block diagonal J (16 keys = one step) are added in place
// first, so e_J(fr, g, r) belongs to distance 16 J + 4 g + r - fr. Rotating a register by r lanes within its 16 brings
// the lanes of one distance together, and a lane that wraps around carries a value of distance 16 J + 16 - ..., which is
// exactly the place of the NEXT block's rotation: selecting between e_J and e_(J-1) before the rotation makes every lane
// right. Three such rotations fold r away, then one by 4 g per lane group folds g, and two half swaps sum the lane groups
// and put four blocks side by side: 64 lanes with 64 consecutive distances, one LDS addition per tile where one per
// register with colliding lanes (ds_add_f32, 20 a tile) took three quarters of the kernel (0.54 ms instead of 0.16 at
// 64 x 512 tokens, 12 heads of 64). Every sum has a fixed order.
struct DiagonalSums {
  f32x4 carry, prev;                 // block not complete yet (its other query block comes with the next tile), block J - 1
  float tprev;                       // block J - 1 with r folded

  __device__ __forceinline__ void reset() {
    carry = prev = f32x4{0.f, 0.f, 0.f, 0.f};
    tprev = 0.f;
  }
  template <int N>
  static __device__ __forceinline__ float rot(float v) {                       // lane i takes lane (i + N) mod 16
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x120 + 16 - N, 0xf, 0xf, false));
  }
  // upper half of a against lower half of b, added: {a.lo + a.hi, b.lo + b.hi}
  static __device__ __forceinline__ float halves(float a, float b) {
    const u32x2_t r = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false));
    const unsigned x = r[0], y = r[1];
    return __uint_as_float(x) + __uint_as_float(y);
  }
  static __device__ __forceinline__ float rows(float a, float b) {             // the same for rows 0, 2 against 1, 3
    const u32x2_t r = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false));
    const unsigned x = r[0], y = r[1];
    return __uint_as_float(x) + __uint_as_float(y);
  }
  // gx[j]: block diagonal j - 1 of the tile, j = 0 .. JB. Completes blocks -1 .. JB - 2; the sum of distance
  // 16 (b - 1) - fr (relative to key 0 of the tile and query 0 of the wave) is returned in lane group b.
  template <int JB>
  __device__ __forceinline__ float add(const f32x4 (&gx)[JB + 1], int fr, int g) {
    float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int b = 0; b < JB; ++b) {
      const f32x4 e = b == 0 ? gx[0] + carry : gx[b];
      float t = e[0];
      t += rot<1>(fr < 1 ? prev[1] : e[1]);
      t += rot<2>(fr < 2 ? prev[2] : e[2]);
      t += rot<3>(fr < 3 ? prev[3] : e[3]);
      prev = e;
      int x = __float_as_int(fr < 4 * g ? tprev : t);
      tprev = t;
      x = __builtin_amdgcn_update_dpp(x, x, 0x120 + 12, 0xa, 0xf, false);      // lane groups 1 and 3: by 4
      x = __builtin_amdgcn_update_dpp(x, x, 0x120 + 8, 0xc, 0xf, false);       // 2 and 3: by 8
      v[b] = __int_as_float(x);
    }
    carry = gx[JB];
    return rows(halves(v[0], v[2]), halves(v[1], v[3]));
  }
};

// A workgroup owns 128 query rows and walks the keys. It also writes D = rowsum(dO * O) for the dK / dV kernel and sums
// the relative bias's gradient: by distance (DiagonalSums, into a band of the wave's own) where a tile touches the band,
// into one of two registers where it lies beyond.
template <typename T, int D, bool BIAS>
__global__ __launch_bounds__(256, (sizeof(T) == 2 && D <= 64 ? 2 : 1)) void bwd_dq_kernel(Args a) {
  constexpr int KT = key_tile<T>(), JB = KT / 16, DB = D / 16, DS = D / 32, ST = row_stride<T, D>(), IMG = KT * ST;
  extern __shared__ __attribute__((aligned(16))) char smem[];      // [2][K | V], [2][key bias], band, band gradients
  float* kbl = reinterpret_cast<float*>(smem + 4 * IMG);
  float* band = kbl + 2 * KT;
  const int nband = BIAS && a.table ? band_size(a) : 0;
  float* gband = band + nband;                                     // [4 waves][nband], then 8 far sums
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int fr = lane & 15, g = lane >> 4;
  const int nqt = (a.Sq + kRows - 1) / kRows;
  const int id = xcd_contiguous(blockIdx.x, gridDim.x);
  const int qt = a.causal ? nqt - 1 - id % nqt : id % nqt, bh = id / nqt, b = bh / a.nh, h = bh - b * a.nh;
  const int kvh = h / (a.nh / a.nkv);
  const int q0 = qt * kRows + wid * 32;
  const int klen = a.lens ? min(max(a.lens[b], 0), a.Sk) : a.Sk;
  const int start = a.q_start ? min(max(a.q_start[b], -kMaxStart), kMaxStart) : a.q_start0;
  const int pos0 = start + q0;
  const float c = a.scale * kLog2e;
  const T* qp = (const T*)a.q.p + b * a.q.sb + h * a.q.sh;
  const T* kp = (const T*)a.k.p + b * a.k.sb + kvh * a.k.sh;
  const T* vp = (const T*)a.v.p + b * a.v.sb + kvh * a.v.sh;
  const T* op = (const T*)a.out.p + b * a.out.sb + h * a.out.sh;
  const T* dop = (const T*)a.dout.p + b * a.dout.sb + h * a.dout.sh;
  const float* kbp = BIAS && a.key_bias ? a.key_bias + (long long)b * a.Sk : nullptr;
  const bool want_tab = BIAS && a.dtab;

  Frag<T> qf[2][DS], dof[2][DS];
  float m2[2], ll[2], dl[2];
#pragma unroll
  for (int qb = 0; qb < 2; ++qb) {
    const int q = q0 + qb * 16 + fr, qc = min(q, a.Sq - 1);
    float part = 0.f;
#pragma unroll
    for (int ks = 0; ks < DS; ++ks) {
      const int e = ks * 32 + g * 8;
      Frag<T> of;
      frag_global(qf[qb][ks], qp + (long long)qc * a.q.ss, e, e < a.hd);
      frag_global(dof[qb][ks], dop + (long long)qc * a.dout.ss, e, e < a.hd);
      frag_global(of, op + (long long)qc * a.out.ss, e, e < a.hd);
      part = dot(of, dof[qb][ks], part);
    }
    const long long i = ((long long)b * a.nh + h) * a.Sq + qc, n = (long long)a.B * a.nh * a.Sq;
    dl[qb] = group_sum(part);
    if (g == 0 && q < a.Sq) a.delta[i] = dl[qb];
    m2[qb] = q < a.Sq ? a.stat[i] : INFINITY;            // rows past the end: probabilities 0
    ll[qb] = q < a.Sq ? a.stat[n + i] : 0.f;
    if (!BIAS) m2[qb] += ll[qb];
  }
  f32x4 dq[DB][2];
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int qb = 0; qb < 2; ++qb) dq[db][qb] = f32x4{0.f, 0.f, 0.f, 0.f};
  float far_l = 0.f, far_r = 0.f;

  const int last = start + min(qt * kRows + kRows, a.Sq) - 1;
  const int kend = a.causal ? min(klen, last + 1) : klen;
  const int nt = kend > 0 ? (kend + KT - 1) / KT : 0;

  Tile<T, D, KT> kr, vr;
  float kbr = 0.f;
  auto fetch = [&](int t) {
    kr.load(kp + (long long)t * KT * a.k.ss, a.k.ss, klen - t * KT, a.hd, tid);
    vr.load(vp + (long long)t * KT * a.v.ss, a.v.ss, klen - t * KT, a.hd, tid);
    if (BIAS && kbp) {
      kr.load_bias(kbp + t * KT, klen - t * KT, tid);
      vr.load_bias(kbp + t * KT, klen - t * KT, tid);
      if (tid < KT) kbr = t * KT + tid < klen ? to_score_units(a, kbp[t * KT + tid]) : -INFINITY;
    }
  };
  auto put = [&](int buf) {
    char* kimg = smem + buf * 2 * IMG;
    if (BIAS && kbp) {
      kr.store_masked(kimg, tid);
      vr.store_masked(kimg + IMG, tid);
      if (tid < KT) kbl[buf * KT + tid] = kbr;
    } else {
      kr.store(kimg, tid);
      vr.store(kimg + IMG, tid);
    }
  };
  if (BIAS && a.table) fill_band(a, h, band, tid);
  if (want_tab)
    for (int i = tid; i < 4 * nband; i += 256) gband[i] = 0.f;
  float* gmine = gband + wid * nband;
  DiagonalSums diag;
  diag.reset();
  int diag_at = 0;                                       // band entry of the next tile's first distance; 0: no tile yet
  if (nt > 0) {
    fetch(0);
    put(0);
  }
  __syncthreads();
  for (int t = 0; t < nt; ++t) {
    const char* kimg = smem + (t & 1) * 2 * IMG;
    const char* vimg = kimg + IMG;
    const int kt = t * KT;
    if (t + 1 < nt) fetch(t + 1);
    if (q0 < a.Sq && (!a.causal || kt <= pos0 + 31)) {
      const bool far = BIAS && a.table && (kt + KT - 1 - pos0 <= -a.max_dist || kt - (pos0 + 31) >= a.right);
      const int at0 = kt + 4 * g - pos0 - fr + a.max_dist + kMargin;    // band entry of (key 4 g of block 0, query fr)
      f32x4 x[JB + 1];
      if (BIAS && a.table) {
        if (far) {
          const float v = kt < pos0 ? band[0] : band[nband - 1];
#pragma unroll
          for (int j = 0; j <= JB; ++j) x[j] = f32x4{v, v, v, v};
        } else {
#pragma unroll
          for (int j = 0; j <= JB; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) x[j][r] = band[at0 + (j - 1) * 16 + r];
        }
      } else if (BIAS) {
#pragma unroll
        for (int j = 0; j <= JB; ++j) x[j] = f32x4{0.f, 0.f, 0.f, 0.f};
      }
      f32x4 gx[JB + 1];
      if (BIAS) {
#pragma unroll
        for (int j = 0; j <= JB; ++j) gx[j] = f32x4{0.f, 0.f, 0.f, 0.f};
      }
      const bool edge = kt + KT > klen || (a.causal && kt + KT - 1 > pos0);
#pragma unroll
      for (int hf = 0; hf < KT / 32; ++hf) {
        f32x4 s[2][2], dp[2][2];
#pragma unroll
        for (int jj = 0; jj < 2; ++jj) {
          const int jb = hf * 2 + jj;
          f32x4 kb = {0.f, 0.f, 0.f, 0.f};
          if (BIAS && kbp) kb = *reinterpret_cast<const f32x4*>(kbl + (t & 1) * KT + jb * 16 + g * 4);
#pragma unroll
          for (int qb = 0; qb < 2; ++qb) {
            s[jj][qb] = BIAS ? kb + x[jb + 1 - qb] : f32x4{0.f, 0.f, 0.f, 0.f};
            dp[jj][qb] = f32x4{0.f, 0.f, 0.f, 0.f};
          }
        }
#pragma unroll
        for (int ks = 0; ks < DS; ++ks)
#pragma unroll
          for (int jj = 0; jj < 2; ++jj) {
            Frag<T> kf, vf;
            frag_row<ST>(kf, kimg, (hf * 2 + jj) * 16, ks, lane);
            frag_row<ST>(vf, vimg, (hf * 2 + jj) * 16, ks, lane);
#pragma unroll
            for (int qb = 0; qb < 2; ++qb) {
              s[jj][qb] = mma(kf, qf[qb][ks], s[jj][qb]);
              dp[jj][qb] = mma(vf, dof[qb][ks], dp[jj][qb]);
            }
          }
        if (edge) {
#pragma unroll
          for (int qb = 0; qb < 2; ++qb) {
            const int end = a.causal ? min(klen, pos0 + qb * 16 + fr + 1) : klen;
#pragma unroll
            for (int jj = 0; jj < 2; ++jj)
#pragma unroll
              for (int r = 0; r < 4; ++r)
                if (kt + (hf * 2 + jj) * 16 + 4 * g + r >= end) s[jj][qb][r] = -INFINITY;
          }
        }
        Frag<T> dsf[2];
#pragma unroll
        for (int qb = 0; qb < 2; ++qb) {
#pragma unroll
          for (int jj = 0; jj < 2; ++jj) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              // with biases the row maximum may be so large (a row of lowest-value masks) that the logarithm of the
              // sum is lost next to it: the two are taken off one after the other
              const float p = fexp2(BIAS ? fmaf(s[jj][qb][r] - m2[qb], c, -ll[qb]) : fmaf(s[jj][qb][r], c, -m2[qb]));
              s[jj][qb][r] = p * (dp[jj][qb][r] - dl[qb]);
            }
            if (BIAS) gx[hf * 2 + jj + 1 - qb] += s[jj][qb];
          }
          pack(dsf[qb], s[0][qb], s[1][qb]);
        }
#pragma unroll
        for (int db = 0; db < DB; ++db) {
          Frag<T> ktr;
          frag_tr<ST>(ktr, kimg, db * 16, hf, lane);
#pragma unroll
          for (int qb = 0; qb < 2; ++qb) dq[db][qb] = mma(ktr, dsf[qb], dq[db][qb]);
        }
      }
      if (want_tab) {
        if (far) {
          float v = 0.f;
#pragma unroll
          for (int j = 0; j <= JB; ++j) v += (gx[j][0] + gx[j][1]) + (gx[j][2] + gx[j][3]);
          if (kt < pos0) far_l += v; else far_r += v;
        } else {                                         // (the tiles on the band follow one another)
          const float v = diag.template add<JB>(gx, fr, g);
          diag_at = kt - pos0 + a.max_dist + kMargin;
          const int i = diag_at + 16 * (g - 1) - fr;
          if (g < JB && i >= 0) gmine[i] += v;
          diag_at += KT;
        }
      }
    }
    if (t + 1 < nt) put((t + 1) & 1);
    __syncthreads();
  }
#pragma unroll
  for (int qb = 0; qb < 2; ++qb) {
    const int q = q0 + qb * 16 + fr;
    if (q < a.Sq) {
      T* row = (T*)a.dq.p + b * a.dq.sb + (long long)q * a.dq.ss + h * a.dq.sh;
#pragma unroll
      for (int db = 0; db < DB; ++db)
        if (db * 16 + g * 4 < a.hd) store4(row + db * 16 + g * 4, dq[db][qb] * a.scale);
    }
  }
  if (want_tab) {
    if (diag_at) {                                       // what the last tile on the band left incomplete
      f32x4 none[JB + 1];
#pragma unroll
      for (int j = 0; j <= JB; ++j) none[j] = f32x4{0.f, 0.f, 0.f, 0.f};
      const float v = diag.template add<JB>(none, fr, g);
      const int i = diag_at + 16 * (g - 1) - fr;
      if (g < JB && i < nband) gmine[i] += v;
    }
    float* fars = gband + 4 * nband;
    far_l = wave_sum(far_l);
    far_r = wave_sum(far_r);
    if (lane == 0) { fars[wid * 2] = far_l; fars[wid * 2 + 1] = far_r; }
    __syncthreads();
    for (int i = tid; i < nband; i += 256)               // (no wave reads the band any more)
      band[i] = (gband[i] + gband[nband + i]) + (gband[2 * nband + i] + gband[3 * nband + i]);
    __syncthreads();
    if (tid < a.buckets) {
      int lo, hi;
      bucket_range(a, tid, lo, hi);
      float v = 0.f;
      for (int i = lo; i <= hi; ++i) v += band[i + a.max_dist + kMargin];
      if (lo == -a.max_dist - kMargin && lo <= hi) v += (fars[0] + fars[2]) + (fars[4] + fars[6]);
      if (hi == a.right + kMargin && lo <= hi) v += (fars[1] + fars[3]) + (fars[5] + fars[7]);
      a.dtab[(((long long)b * nqt + qt) * a.nh + h) * a.buckets + tid] = v;
    }
  }
}

// ================================================================================================== backward: dK, dV
// A workgroup owns 128 keys of one key head, a wave 32 of them, and walks the query tiles of every query head of the
// group: gradients of shared heads are summed in the accumulators. The KEY rides on the lane here.
template <typename T, int D, bool BIAS>
__global__ __launch_bounds__(256, (sizeof(T) == 2 && D <= 64 ? 2 : 1)) void bwd_dkdv_kernel(Args a) {
  constexpr int QT = key_tile<T>(), IB = QT / 16, DB = D / 16, DS = D / 32, ST = row_stride<T, D>(), IMG = QT * ST;
  extern __shared__ __attribute__((aligned(16))) char smem[];      // [2][Q | dO], [2][maximum | log sum | D], band
  float* stl = reinterpret_cast<float*>(smem + 4 * IMG);
  float* band = stl + 2 * 3 * QT;
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int fr = lane & 15, g = lane >> 4;
  const int nkt = (a.Sk + kRows - 1) / kRows, group = a.nh / a.nkv;
  const int id = xcd_contiguous(blockIdx.x, gridDim.x);
  const int bk = id / nkt, b = bk / a.nkv, kvh = bk - b * a.nkv;
  const int kb0 = (id - bk * nkt) * kRows, k0 = kb0 + wid * 32;
  const int klen = a.lens ? min(max(a.lens[b], 0), a.Sk) : a.Sk;
  const int start = a.q_start ? min(max(a.q_start[b], -kMaxStart), kMaxStart) : a.q_start0;
  const float c = a.scale * kLog2e;
  const T* kp = (const T*)a.k.p + b * a.k.sb + kvh * a.k.sh;
  const T* vp = (const T*)a.v.p + b * a.v.sb + kvh * a.v.sh;
  const float* kbp = BIAS && a.key_bias ? a.key_bias + (long long)b * a.Sk : nullptr;

  Frag<T> kf[2][DS], vf[2][DS];
  float kbias[2];
#pragma unroll
  for (int kb = 0; kb < 2; ++kb) {
    const int k = k0 + kb * 16 + fr, kc = min(k, a.Sk - 1);
    kbias[kb] = kbp ? to_score_units(a, kbp[kc]) : 0.f;
    if (k >= klen) kbias[kb] = -INFINITY;
    const bool in = kbias[kb] != -INFINITY;
#pragma unroll
    for (int ks = 0; ks < DS; ++ks) {
      const int e = ks * 32 + g * 8;
      frag_global(kf[kb][ks], kp + (long long)kc * a.k.ss, e, in && e < a.hd);
      frag_global(vf[kb][ks], vp + (long long)kc * a.v.ss, e, in && e < a.hd);
    }
  }
  f32x4 dk[DB][2], dv[DB][2];
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) { dk[db][kb] = f32x4{0.f, 0.f, 0.f, 0.f}; dv[db][kb] = f32x4{0.f, 0.f, 0.f, 0.f}; }

  const int ntq = (a.Sq + QT - 1) / QT;
  // causal: the first query that sees the workgroup's first key is kb0 - start
  int t0 = a.causal ? max(kb0 - start, 0) / QT : 0;
  if (kb0 >= klen) t0 = ntq;
  const bool edge_keys = k0 + 32 > klen;

  for (int hg = 0; hg < group; ++hg) {
    if (t0 >= ntq) break;
    const int h = kvh * group + hg;
    const T* qp = (const T*)a.q.p + b * a.q.sb + h * a.q.sh;
    const T* dop = (const T*)a.dout.p + b * a.dout.sb + h * a.dout.sh;
    const long long n = (long long)a.B * a.nh * a.Sq, i0 = ((long long)b * a.nh + h) * a.Sq;
    Tile<T, D, QT> qr, dr;
    float st[3] = {INFINITY, 0.f, 0.f};
    auto fetch = [&](int t) {
      qr.load(qp + (long long)t * QT * a.q.ss, a.q.ss, a.Sq - t * QT, a.hd, tid);
      dr.load(dop + (long long)t * QT * a.dout.ss, a.dout.ss, a.Sq - t * QT, a.hd, tid);
      if (tid < QT) {
        const int q = t * QT + tid;
        const bool in = q < a.Sq;
        st[0] = in ? a.stat[i0 + q] : INFINITY;
        st[1] = in ? a.stat[n + i0 + q] : 0.f;
        st[2] = in ? a.delta[i0 + q] : 0.f;
      }
    };
    auto put = [&](int buf) {
      char* qimg = smem + buf * 2 * IMG;
      qr.store(qimg, tid);
      dr.store(qimg + IMG, tid);
      if (tid < QT) {
        float* s = stl + buf * 3 * QT + tid;
        s[0] = BIAS ? st[0] : st[0] + st[1];
        s[QT] = st[1];
        s[2 * QT] = st[2];
      }
    };
    if (BIAS && a.table) fill_band(a, h, band, tid);     // (the previous head's last barrier has passed)
    fetch(t0);
    put(t0 & 1);
    __syncthreads();
    for (int t = t0; t < ntq; ++t) {
      const char* qimg = smem + (t & 1) * 2 * IMG;
      const char* dimg = qimg + IMG;
      const float* stc = stl + (t & 1) * 3 * QT;
      const int pos = start + t * QT;                    // position of the tile's first query
      if (t + 1 < ntq) fetch(t + 1);
      if (k0 < klen && (!a.causal || k0 <= pos + QT - 1)) {
        const bool far = BIAS && a.table && (k0 + 31 - pos <= -a.max_dist || k0 - (pos + QT - 1) >= a.right);
        const bool edge = a.causal && k0 + 31 > pos;
        float xf = 0.f;
        if (far) xf = k0 < pos ? band[0] : band[band_size(a) - 1];
        const float* at = band + (k0 + fr - pos - 4 * g + a.max_dist + kMargin);   // (query 4 g of block 0, key fr of block 0)
#pragma unroll
        for (int hf = 0; hf < QT / 32; ++hf) {
          f32x4 s[2][2], dp[2][2];
#pragma unroll
          for (int ii = 0; ii < 2; ++ii)
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
              const float b0 = BIAS ? kbias[kb] + xf : 0.f;
              s[ii][kb] = f32x4{b0, b0, b0, b0};
              dp[ii][kb] = f32x4{0.f, 0.f, 0.f, 0.f};
            }
          if (BIAS && a.table && !far) {
#pragma unroll
            for (int j = 0; j < 3; ++j) {                // key block minus query block of the half: -1, 0, 1
              f32x4 x;
#pragma unroll
              for (int r = 0; r < 4; ++r) x[r] = at[(j - 1 - hf * 2) * 16 - r];
              if (j == 0) s[1][0] += x;
              if (j == 1) { s[0][0] += x; s[1][1] += x; }
              if (j == 2) s[0][1] += x;
            }
          }
#pragma unroll
          for (int ks = 0; ks < DS; ++ks)
#pragma unroll
            for (int ii = 0; ii < 2; ++ii) {
              Frag<T> qfr, dfr;
              frag_row<ST>(qfr, qimg, (hf * 2 + ii) * 16, ks, lane);
              frag_row<ST>(dfr, dimg, (hf * 2 + ii) * 16, ks, lane);
#pragma unroll
              for (int kb = 0; kb < 2; ++kb) {
                s[ii][kb] = mma(qfr, kf[kb][ks], s[ii][kb]);
                dp[ii][kb] = mma(dfr, vf[kb][ks], dp[ii][kb]);
              }
            }
          if (edge || (!BIAS && edge_keys)) {            // with biases a key past the end has -inf already
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
              const int key = k0 + kb * 16 + fr;
#pragma unroll
              for (int ii = 0; ii < 2; ++ii)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                  if (key >= klen || (a.causal && key > pos + (hf * 2 + ii) * 16 + 4 * g + r)) s[ii][kb][r] = -INFINITY;
            }
          }
          Frag<T> pf[2], dsf[2];
#pragma unroll
          for (int ii = 0; ii < 2; ++ii) {
            const float* sr = stc + (hf * 2 + ii) * 16 + g * 4;
            const f32x4 mm = *reinterpret_cast<const f32x4*>(sr);
            const f32x4 ls = *reinterpret_cast<const f32x4*>(sr + QT);
            const f32x4 de = *reinterpret_cast<const f32x4*>(sr + 2 * QT);
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                const float p = fexp2(BIAS ? fmaf(s[ii][kb][r] - mm[r], c, -ls[r]) : fmaf(s[ii][kb][r], c, -mm[r]));
                s[ii][kb][r] = p;
                dp[ii][kb][r] = p * (dp[ii][kb][r] - de[r]);
              }
          }
#pragma unroll
          for (int kb = 0; kb < 2; ++kb) {
            pack(pf[kb], s[0][kb], s[1][kb]);
            pack(dsf[kb], dp[0][kb], dp[1][kb]);
          }
#pragma unroll
          for (int db = 0; db < DB; ++db) {
            Frag<T> dot_, qt_;
            frag_tr<ST>(dot_, dimg, db * 16, hf, lane);
            frag_tr<ST>(qt_, qimg, db * 16, hf, lane);
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
              dv[db][kb] = mma(dot_, pf[kb], dv[db][kb]);
              dk[db][kb] = mma(qt_, dsf[kb], dk[db][kb]);
            }
          }
        }
      }
      if (t + 1 < ntq) put((t + 1) & 1);
      __syncthreads();
    }
  }
#pragma unroll
  for (int kb = 0; kb < 2; ++kb) {
    const int k = k0 + kb * 16 + fr;
    if (k < a.Sk) {
      T* krow = (T*)a.dk.p + b * a.dk.sb + (long long)k * a.dk.ss + kvh * a.dk.sh;
      T* vrow = (T*)a.dv.p + b * a.dv.sb + (long long)k * a.dv.ss + kvh * a.dv.sh;
#pragma unroll
      for (int db = 0; db < DB; ++db)
        if (db * 16 + g * 4 < a.hd) {
          store4(krow + db * 16 + g * 4, dk[db][kb] * a.scale);
          store4(vrow + db * 16 + g * 4, dv[db][kb]);
        }
    }
  }
}

// ---- host -----------------------------------------------------------------------------------------------------------
inline int lds_tiles(int es, int D) {                    // bytes of the two double-buffered tile images
  const int kt = es == 2 ? 64 : 32;
  return 4 * kt * (D * es + 16);
}
template <typename K>
inline int set_lds(K kernel, int bytes) {
  if (bytes <= 64 * 1024) return 0;
  return (int)hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
}
template <typename K>
inline int launch(K kernel, long long blocks, int lds, const Args& a, hipStream_t stream) {
  const int rc = set_lds(kernel, lds);
  if (rc) return rc;
  hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(256), (size_t)lds, stream, a);
  return (int)hipGetLastError();
}

// Key splits of the few-queries path: two workgroups a CU, and at least two key tiles for each of a workgroup's waves
// (fewer and the joining costs more than the splitting gains). 1: no second kernel.
inline bool few_queries(int Sq, int nh, int nkv) { return (long long)Sq * (nh / nkv) <= kFewRows; }
inline int few_splits(int B, int Sk, int nkv) {
  const long long groups = (long long)B * nkv, most = (Sk + 8 * kFewKeys - 1) / (8 * kFewKeys);
  long long n = (512 + groups - 1) / groups;
  n = n < most ? n : most;
  return (int)(n < 1 ? 1 : n > 64 ? 64 : n);
}
template <typename T, int D, int QB, bool BIAS>
int run_few(const Args& a, hipStream_t stream) {
  constexpr int img = kFewKeys * row_stride<T, D>(), join = QB * 16 * (D + 4) * 4;
  const int lds = 4 * (img > join ? img : join) + 4 * (8 * QB * 16 + (a.table ? a.nh / a.nkv * a.buckets : 0));
  const int rc = launch(few_kernel<T, D, QB, BIAS>, (long long)a.B * a.nkv * a.splits, lds, a, stream);
  if (rc || a.splits == 1) return rc;
  hipLaunchKernelGGL((few_join_kernel<T, D, BIAS>), dim3((unsigned)(a.B * a.nh * a.Sq)), dim3(256), 0, stream, a);
  return (int)hipGetLastError();
}

template <typename T, int D>
int run_fwd(const Args& a, hipStream_t stream) {
  const bool bias = a.key_bias || a.table;
  if (few_queries(a.Sq, a.nh, a.nkv)) {
    if (a.Sq * (a.nh / a.nkv) <= 16) return bias ? run_few<T, D, 1, true>(a, stream) : run_few<T, D, 1, false>(a, stream);
    return bias ? run_few<T, D, 2, true>(a, stream) : run_few<T, D, 2, false>(a, stream);
  }
  const int nqt = (a.Sq + kRows - 1) / kRows, kt = key_tile<T>();
  const int band = a.table ? a.max_dist + a.right + 1 + 2 * kMargin : 0;
  const int lds = lds_tiles(sizeof(T), D) + 4 * (2 * kt + band);
  const long long n = (long long)a.B * a.nh * nqt;
  return bias ? launch(fwd_kernel<T, D, true>, n, lds, a, stream) : launch(fwd_kernel<T, D, false>, n, lds, a, stream);
}
template <typename T, int D>
int run_bwd(const Args& a, hipStream_t stream) {
  const bool bias = a.key_bias || a.table;
  const int nqt = (a.Sq + kRows - 1) / kRows, nkt = (a.Sk + kRows - 1) / kRows, kt = key_tile<T>();
  const int band = a.table ? a.max_dist + a.right + 1 + 2 * kMargin : 0;
  int lds = lds_tiles(sizeof(T), D) + 4 * (2 * kt + band + (a.dtab ? 4 * band + 8 : 0));
  const long long nq = (long long)a.B * a.nh * nqt, nk = (long long)a.B * a.nkv * nkt;
  int rc = bias ? launch(bwd_dq_kernel<T, D, true>, nq, lds, a, stream) : launch(bwd_dq_kernel<T, D, false>, nq, lds, a, stream);
  if (rc) return rc;
  lds = lds_tiles(sizeof(T), D) + 4 * (6 * kt + band);
  return bias ? launch(bwd_dkdv_kernel<T, D, true>, nk, lds, a, stream) : launch(bwd_dkdv_kernel<T, D, false>, nk, lds, a, stream);
}
template <typename T>
int dispatch_fwd(const Args& a, hipStream_t s) {
  return a.hd <= 32 ? run_fwd<T, 32>(a, s) : a.hd <= 64 ? run_fwd<T, 64>(a, s) : a.hd <= 96 ? run_fwd<T, 96>(a, s) : run_fwd<T, 128>(a, s);
}
template <typename T>
int dispatch_bwd(const Args& a, hipStream_t s) {
  return a.hd <= 32 ? run_bwd<T, 32>(a, s) : a.hd <= 64 ? run_bwd<T, 64>(a, s) : a.hd <= 96 ? run_bwd<T, 96>(a, s) : run_bwd<T, 128>(a, s);
}

int fwd_bf16(const Args& a, hipStream_t s);
int bwd_bf16(const Args& a, hipStream_t s);
int fwd_f32(const Args& a, hipStream_t s);
int bwd_f32(const Args& a, hipStream_t s);

}  // namespace attn
}  // namespace dtf
