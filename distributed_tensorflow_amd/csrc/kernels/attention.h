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
// Scores are kept as step * t, step = unit / scale (unit 1: q . k as it is): the biases are multiplied by step where they are
// staged and enter as the INITIAL VALUE of the score accumulators, so a bias costs no vector instruction per score
// (but in few_kernel, which finds the bucket of each score). Beside a key bias unit is the power of two below a scale under 1,
// and the operand that stays in registers carries it: step is then at most 1, so any finite bias stays finite, and equal ones
// equal (1 / scale itself would carry a bias beyond 4.3e37 past the type's range at heads of 64). A power of two rounds
// nothing.
//
// Measured (bf16, us and the rate of the products): 64 x 512 tokens x 12 heads of 64, with a table: forward 111 (P in two
// parts, see PARTS), dQ and dTable 174, dK / dV 157; without one 85, 111, 120 (605, 697, 862 TFLOP/s of what each has to do);
// 4 x 8192 x 12 of 64, not causal: 893, 1206, 1237 TFLOP/s; 4 x 2048 causal, 16 heads on 4 of 128: 94, 125, 183 and 24 for
// the join. Long rows are bound by the vector instructions beside the products (the forward pass keeps them 70 % busy:
// maximum, exponential, sum, conversion of every score); at 512 tokens and less by a workgroup's beginning and end, where
// it waits for memory.
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
  unsigned bytes;                    // sizeof(Args) where it was filled in: by_head_size refuses what another layout filled in
  Strided q, k, v, out, dout, dq, dk, dv;
  const float* key_bias;             // [B, Sk] or null
  const int* lens;                   // [B] or null
  const int* q_start;                // [B] or null (then q_start0 for every batch element)
  int q_start0;
  const void* table;                 // [buckets, nh] or null
  int table_bf16, buckets, half, exact, max_dist, right;   // right: max_dist when bidirectional, else 0
  int n_thr, thr[kMaxThr];           // thr[t]: smallest |distance| of bucket exact + 1 + t
  float* stat;                       // [2][B, nh, Sq]: row maximum (in score units with biases, else base 2), log2 of the row sum
  float* rows;                       // [B * nh][64-row tiles][4][64]: what the dK / dV kernel wants of each query, see kRowStats
  float* dtab;                       // [B * query tiles][nh][buckets] partial sums of the table's gradient, or null
  unsigned char* fine;               // bf16: [B, Sq, nh, hd] the next 8 bits of O, for D (see finer); or null
  float* part;                       // partial results of the key splits (few queries), of the head splits (dK / dV)
  int B, Sq, Sk, nh, nkv, hd, causal, splits, ksplits;
  float scale;                       // of the formula: dQ and dK are multiplied by it
  float unit, score_scale, step;     // t = score_scale * score, score = unit q . k + step * biases; step = 1 / score_scale
};

// What the dK / dV kernel wants of each query, in tiles of 64 that one direct load of 1 KiB brings to the LDS: the row
// maximum with log2 of the row sum added (with key biases: without, and that on its own) and -D; rows past the end have
// the maximum +inf, that is probabilities 0. The dQ kernel writes them, for whole workgroups of 128 rows.
constexpr int kRowStats = 256;       // floats of a tile: [maximum | log sum | -D | unused][64]
__device__ __forceinline__ long long row_tile(const Args& a, long long bh, int tile) {
  return (bh * ((a.Sq + kRows - 1) / kRows * 2) + tile) * kRowStats;
}

template <typename T> struct Frag;
template <> struct Frag<unsigned short> { bf16x8_t v; };
template <> struct Frag<float> { f32x4 lo, hi; };

template <typename T> constexpr int key_tile() { return sizeof(T) == 2 ? 64 : 32; }
// Tile images in the LDS. bf16: rows of 64, 128 or 256 bytes (head sizes over 64 take 256) without padding, as the direct
// loads need them, their 16-byte chunks permuted by an XOR with swz(row). A ds_read_b128 serves 16 lanes at a time, lanes
// 0-3, 12-15 and 20-27 (then 4-11, 16-19 and 28-31, then the same 32 up), a transposing read 32 lanes in order; with
// these swizzles both fall on 64 different banks (counted: no conflict; with rows merely told apart 16 in order, the
// fragment reads took twice their time). fp32: padded by 16 bytes, which spreads its 16- and 4-byte reads.
template <typename T, int D> constexpr int row_stride() {
  return sizeof(T) == 4 ? D * 4 + 16 : (D == 32 ? 64 : D == 64 ? 128 : 256);
}
template <int STRIDE> __device__ __forceinline__ int swz(int row) {
  return STRIDE == 64 ? (row >> 1) & 2 : STRIDE == 128 ? row & 6 : (row & 7) << 1;
}

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

// v, of which the compiler forgets where it came from
__device__ __forceinline__ int opaque(int v) {
#ifdef __HIP_DEVICE_COMPILE__
  asm volatile("" : "+v"(v));
#endif
  return v;
}
__device__ __forceinline__ float fexp2(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float flog2(float x) { return __builtin_amdgcn_logf(x); }

__device__ __forceinline__ void pack(Frag<unsigned short>& f, const f32x4& a, const f32x4& b) {
  const u32x4_t r = {pack_bf16x2(a[0], a[1]), pack_bf16x2(a[2], a[3]), pack_bf16x2(b[0], b[1]), pack_bf16x2(b[2], b[3])};
  f.v = __builtin_bit_cast(bf16x8_t, r);
}
__device__ __forceinline__ void pack(Frag<float>& f, const f32x4& a, const f32x4& b) { f.lo = a; f.hi = b; }
// times a power of two
__device__ __forceinline__ void times(Frag<unsigned short>& f, float by) {
  u32x4_t r = __builtin_bit_cast(u32x4_t, f.v);
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = pack_bf16x2(__uint_as_float(r[i] << 16) * by, __uint_as_float(r[i] & 0xffff0000u) * by);
  f.v = __builtin_bit_cast(bf16x8_t, r);
}
__device__ __forceinline__ void times(Frag<float>& f, float by) {
  f.lo *= by;
  f.hi *= by;
}
// what pack() rounded off
__device__ __forceinline__ void pack_rest(Frag<unsigned short>& f, f32x4 a, f32x4 b, const Frag<unsigned short>& packed) {
  const u32x4_t r = __builtin_bit_cast(u32x4_t, packed.v);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    a[i] -= __uint_as_float(i & 1 ? r[i >> 1] & 0xffff0000u : r[i >> 1] << 16);
    b[i] -= __uint_as_float(i & 1 ? r[2 + (i >> 1)] & 0xffff0000u : r[2 + (i >> 1)] << 16);
  }
  pack(f, a, b);
}
__device__ __forceinline__ void pack_rest(Frag<float>&, const f32x4&, const f32x4&, const Frag<float>&) {}

// byte of a row's 16-byte chunk ch
template <typename T, int D> __device__ __forceinline__ int chunk_at(int row, int ch) {
  constexpr int S = row_stride<T, D>();
  return row * S + ((sizeof(T) == 2 ? ch ^ swz<S>(row) : ch) << 4);
}

// Reads of a tile image. Row: 16 rows from row0 x 32 contraction elements ks, 8 consecutive elements a lane. Tr: the
// transposed product's operand, column c0 + (lane & 15) of the image, its 32 rows ks in the order of pack(): rows
// 32 ks + 4 g .. +3, then 32 ks + 16 + 4 g .. +3 for lane group g. The lane's part of the addresses is computed once
// (the swizzle sees only the low four bits of a row); row0 and ks of Tr are immediate offsets.
template <typename T, int D, bool KEEP = true> struct Reader;
template <int D, bool KEEP> struct Reader<unsigned short, D, KEEP> {
  static constexpr int S = row_stride<unsigned short, D>();
  static constexpr bool kKeep = KEEP;                    // false: no registers to spare, one XOR an access
  int row[kKeep ? D / 32 : 1], tr[kKeep ? D / 16 : 1];
  static __device__ __forceinline__ int flip(int at, int bits) {    // at ^ bits, which the compiler does not keep in a register
    int o = 0;
#ifdef __HIP_DEVICE_COMPILE__                            // (the host pass does not know the register class)
    asm volatile("v_xor_b32 %0, %2, %1" : "=v"(o) : "v"(at), "i"(bits));
#endif
    return o;
  }
  __device__ __forceinline__ explicit Reader(int lane) {
    const int fr = lane & 15, g = lane >> 4, q = fr >> 2, p = fr & 3, k = 4 * g + q;
    const int row0 = fr * S + ((g ^ swz<S>(fr)) << 4), tr0 = k * S + (((p >> 1) ^ swz<S>(k)) << 4) + ((p & 1) << 3);
#pragma unroll
    for (int ks = 0; ks < (kKeep ? D / 32 : 1); ++ks) row[ks] = row0 ^ (ks << 6);
#pragma unroll
    for (int db = 0; db < (kKeep ? D / 16 : 1); ++db) tr[db] = tr0 ^ (db << 5);
  }
  __device__ __forceinline__ void read_row(Frag<unsigned short>& f, const char* img, int row0, int ks) const {
    f.v = *reinterpret_cast<const bf16x8_t*>(img + (kKeep ? row[kKeep ? ks : 0] : flip(row[0], ks << 6)) + row0 * S);
  }
  __device__ __forceinline__ void read_tr(Frag<unsigned short>& f, const char* img, int db, int ks) const {
    const char* at = img + (kKeep ? tr[kKeep ? db : 0] : flip(tr[0], db << 5)) + ks * 32 * S;
    typedef __attribute__((address_space(3))) s16x4_f* lp_t;
    const s16x4_f lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp_t)at);
    const s16x4_f hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp_t)(at + 16 * S));
    const s16x8_f v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    f.v = __builtin_bit_cast(bf16x8_t, v);
  }
};
template <int D, bool KEEP> struct Reader<float, D, KEEP> {
  static constexpr int S = row_stride<float, D>();
  int row, tr;
  __device__ __forceinline__ explicit Reader(int lane) {
    row = (lane & 15) * S + (lane >> 4) * 32;
    tr = 4 * (lane >> 4) * S + (lane & 15) * 4;
  }
  __device__ __forceinline__ void read_row(Frag<float>& f, const char* img, int row0, int ks) const {
    const char* at = img + row + row0 * S + ks * 128;
    f.lo = *reinterpret_cast<const f32x4*>(at);
    f.hi = *reinterpret_cast<const f32x4*>(at + 16);
  }
  __device__ __forceinline__ void read_tr(Frag<float>& f, const char* img, int db, int ks) const {
    const char* at = img + tr + ks * 32 * S + db * 64;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f.lo[i] = *reinterpret_cast<const float*>(at + i * S);
      f.hi[i] = *reinterpret_cast<const float*>(at + (16 + i) * S);
    }
  }
};

// D = rowsum(dO * O) enters every dT of its row, so an O of 8 significant bits there would cost dQ, dK and dTable as much as
// rounding dT itself does (relative error against 64 bits 0.0026 instead of 0.0024, dTable 0.0027 instead of 0.0017). The
// forward pass therefore stores, besides the rounded O, the difference of the fp32 bit pattern's upper 24 bits from it in a
// byte; the two together are O to 16 bits.
__device__ __forceinline__ unsigned finer(float o) {
  const unsigned u = __float_as_uint(o), b = (unsigned)f32_to_bf16(o) << 8;
  const int d = (int)(((u + 0x80u) >> 8) - b);
  return (unsigned)(d > 127 ? 127 : d) & 0xffu;
}
__device__ __forceinline__ unsigned finer4(const f32x4& o) {
  return finer(o[0]) | finer(o[1]) << 8 | finer(o[2]) << 16 | finer(o[3]) << 24;
}
__device__ __forceinline__ unsigned char* fine_row(const Args& a, int b, int q, int h) {
  return a.fine + (((long long)b * a.Sq + q) * a.nh + h) * a.hd;
}
// dO . O over 8 elements, O with the bits of `fine`
__device__ __forceinline__ float dot_fine(const Frag<unsigned short>& dout, const Frag<unsigned short>& o, u32x2_t fine, float s) {
  const u32x4_t w = __builtin_bit_cast(u32x4_t, o.v);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const unsigned hi = i & 1 ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16;
    const int lo = (int)(fine[i >> 2] << (24 - 8 * (i & 3))) >> 24;
    s = fmaf((float)dout.v[i], __uint_as_float(hi + (unsigned)(lo << 8)), s);
  }
  return s;
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
__device__ __forceinline__ float dot(const Frag<float>& a, const Frag<float>& b, float s) {
#pragma unroll
  for (int i = 0; i < 4; ++i) s = fmaf(a.lo[i], b.lo[i], s);
#pragma unroll
  for (int i = 0; i < 4; ++i) s = fmaf(a.hi[i], b.hi[i], s);
  return s;
}
__device__ __forceinline__ void store4(unsigned short* p, const f32x4& v) { store4_bf16(p, v[0], v[1], v[2], v[3]); }
__device__ __forceinline__ void store4(float* p, const f32x4& v) { *reinterpret_cast<f32x4*>(p) = v; }

// Results leave the accumulators with 4 consecutive elements of block 2 p in a lane and 4 of block 2 p + 1, 16 apart. Two
// swaps between lane groups make that 8 consecutive ones, at 32 p + 8 g: a row's 64 (fp32: 128) bytes go out at once instead
// of in pieces of 8 or 16. x: lane groups' four 0, 1, 2, 3, y: 4, 5, 6, 7; after it x: 0, 2, 4, 6 and y: 1, 3, 5, 7.
__device__ __forceinline__ void gather8(unsigned& x, unsigned& y) {
  const u32x2_t h = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_permlane32_swap(x, y, false, false));
  const unsigned a = h[0], b = h[1];
  const u32x2_t r = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_permlane16_swap(a, b, false, false));
  x = r[0];
  y = r[1];
}
__device__ __forceinline__ void store_pair(unsigned short* row, int p, int g, int hd, const f32x4& v0, const f32x4& v1) {
  unsigned x0 = pack_bf16x2(v0[0], v0[1]), x1 = pack_bf16x2(v0[2], v0[3]);
  unsigned y0 = pack_bf16x2(v1[0], v1[1]), y1 = pack_bf16x2(v1[2], v1[3]);
  gather8(x0, y0);
  gather8(x1, y1);
  if (p * 32 + g * 8 < hd) *reinterpret_cast<u32x4_t*>(row + p * 32 + g * 8) = u32x4_t{x0, x1, y0, y1};
}
__device__ __forceinline__ void store_pair(float* row, int p, int g, int hd, const f32x4& v0, const f32x4& v1) {
  u32x4_t x, y;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    unsigned a = __float_as_uint(v0[i]), b = __float_as_uint(v1[i]);
    gather8(a, b);
    x[i] = a;
    y[i] = b;
  }
  if (p * 32 + g * 8 >= hd) return;
  *reinterpret_cast<u32x4_t*>(row + p * 32 + g * 8) = x;
  *reinterpret_cast<u32x4_t*>(row + p * 32 + g * 8 + 4) = y;
}

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

// A tile of ROWS rows x D elements from global memory to an LDS image, by 256 threads. Rows from `left` on and elements
// beyond the head size arrive as zeros: their addresses fail the buffer descriptor's range check. The descriptor covers
// one tile only, so offsets stay 32-bit whatever the tensor's size, and a lane's offsets are the same for every tile. A
// key whose bias is -inf takes no part whatever K and V hold there: its row is read as zeros too.
// bf16: loads that go to the LDS directly (64 lanes x 16 bytes fill 1 KiB in lane order; the swizzle is in the SOURCE
// address). fp32: through registers, put() stores them.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t tile_rsrc(const void* base, unsigned row_bytes, unsigned bytes_per_row_used, int left, int rows) {
  left = left < 0 ? 0 : (left > rows ? rows : left);
  const unsigned bytes = left ? (unsigned)(left - 1) * row_bytes + bytes_per_row_used : 0u;
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, (int)bytes, 0x00020000);
}
// 8 consecutive elements of row r of a block of rows; zero outside the block, beyond the head size and where not `ok`: no
// branch and no 64-bit address a row.
__device__ __forceinline__ void block_row(Frag<unsigned short>& f, __amdgpu_buffer_rsrc_t rs, unsigned ld, int r, int e, bool ok) {
  f.v = __builtin_bit_cast(bf16x8_t, __builtin_amdgcn_raw_buffer_load_b128(rs, (int)(ok ? (unsigned)r * ld + (unsigned)e * 2u : 0xffffffffu), 0, 0));
}
__device__ __forceinline__ void block_row(Frag<float>& f, __amdgpu_buffer_rsrc_t rs, unsigned ld, int r, int e, bool ok) {
  const unsigned off = (unsigned)r * ld + (unsigned)e * 4u;
  f.lo = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, (int)(ok ? off : 0xffffffffu), 0, 0));
  f.hi = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, (int)(ok ? off + 16u : 0xffffffffu), 0, 0));
}
template <typename T, int D, int ROWS> struct Tile;
template <int D, int ROWS>
struct Tile<unsigned short, D, ROWS> {
  static constexpr int S = row_stride<unsigned short, D>(), kSlots = S / 16, N = ROWS * S / 4096, IMG = ROWS * S;
  const unsigned short* base;
  unsigned ldb, used, off[N];
  long long step;                                        // elements from tile to tile
  int row[N];
  __device__ __forceinline__ Tile(const unsigned short* p, long long ss, int hd, int tid) : base(p), step(ss * ROWS) {
    ldb = (unsigned)ss * 2u;
    used = (unsigned)hd * 2u;
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const int i = (u * 4 + (tid >> 6)) * 64 + (tid & 63);
      row[u] = i / kSlots;
      const int ch = (i % kSlots) ^ swz<S>(row[u]);
      off[u] = ch * 8 < hd ? (unsigned)row[u] * ldb + (unsigned)ch * 16u : 0xffffffffu;
    }
  }
  typedef __attribute__((address_space(3))) void* lds_t;
  __device__ __forceinline__ void load(int t, int left, char* img, int wid) const {
    const __amdgpu_buffer_rsrc_t rs = tile_rsrc(base + t * step, ldb, used, left, ROWS);
#pragma unroll
    for (int u = 0; u < N; ++u)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_t)(img + (u * 4 + wid) * 1024), 16, (int)off[u], 0, 0, 0);
  }
  __device__ __forceinline__ void load_masked(int t, int left, char* img, int wid, const float (&kb)[N]) const {
    const __amdgpu_buffer_rsrc_t rs = tile_rsrc(base + t * step, ldb, used, left, ROWS);
#pragma unroll
    for (int u = 0; u < N; ++u)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_t)(img + (u * 4 + wid) * 1024), 16, kb[u] == -INFINITY ? -1 : (int)off[u], 0, 0, 0);
  }
  __device__ __forceinline__ void put(char*) const {}
};
template <int D, int ROWS>
struct Tile<float, D, ROWS> {
  static constexpr int S = row_stride<float, D>(), kPerRow = D / 4, N = ROWS * kPerRow / 256, IMG = ROWS * S;
  const float* base;
  unsigned ldb, used, off[N];
  long long step;
  int row[N], at[N];
  u32x4_t v[N];
  __device__ __forceinline__ Tile(const float* p, long long ss, int hd, int tid) : base(p), step(ss * ROWS) {
    ldb = (unsigned)ss * 4u;
    used = (unsigned)hd * 4u;
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const int i = u * 256 + tid, ch = i % kPerRow;
      row[u] = i / kPerRow;
      at[u] = row[u] * S + ch * 16;
      off[u] = ch * 4 < hd ? (unsigned)row[u] * ldb + (unsigned)ch * 16u : 0xffffffffu;
    }
  }
  __device__ __forceinline__ void load(int t, int left, char*, int) {
    const __amdgpu_buffer_rsrc_t rs = tile_rsrc(base + t * step, ldb, used, left, ROWS);
#pragma unroll
    for (int u = 0; u < N; ++u) v[u] = __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(rs, (int)off[u], 0, 0));
  }
  __device__ __forceinline__ void load_masked(int t, int left, char*, int, const float (&kb)[N]) {
    const __amdgpu_buffer_rsrc_t rs = tile_rsrc(base + t * step, ldb, used, left, ROWS);
#pragma unroll
    for (int u = 0; u < N; ++u)
      v[u] = __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(rs, kb[u] == -INFINITY ? -1 : (int)off[u], 0, 0));
  }
  __device__ __forceinline__ void put(char* img) const {
#pragma unroll
    for (int u = 0; u < N; ++u) *reinterpret_cast<u32x4_t*>(img + at[u]) = v[u];
  }
};
// the key biases of the rows of a tile that a thread loads
template <int N>
__device__ __forceinline__ void row_bias(float (&kb)[N], const int (&row)[N], const float* bias, int left) {
#pragma unroll
  for (int u = 0; u < N; ++u) kb[u] = row[u] < left ? bias[row[u]] : 0.f;
}
// the direct loads of this wave have arrived (the barrier after it makes that true for every wave's)
__device__ __forceinline__ void loads_done() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

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
// Biases in score units. A key bias is a mask as well: only -inf is one, and a finite one stays finite, as step <= 1 beside
// key biases. A learned value is held to +-2^24 powers of two (beyond that the scores next to it would be lost in fp32
// anyway), so that the kernels without key bias may take the maximum off by one fma.
__device__ __forceinline__ float to_score_units(const Args& a, float bias) { return bias * a.step; }
__device__ __forceinline__ float learned_bias(const Args& a, float bias) {
  if (bias == -INFINITY || bias == INFINITY) return bias;
  const float lim = 16777216.f / kLog2e, v = bias > lim ? lim : bias < -lim ? -lim : bias;
  return v * a.step;
}
__device__ __forceinline__ void fill_band(const Args& a, int h, float* band, int tid) {
  const int n = band_size(a);
  for (int i = tid; i < n; i += 256) band[i] = learned_bias(a, table_at(a, bucket_of(a, i - kMargin - a.max_dist), h));
}
// What a kernel instance knows of the biases: none, the relative one alone, or a key bias with or without it.
enum Mode { kPlain = 0, kRel = 1, kKeys = 2 };
// Whether P may enter O in two parts (see fwd_kernel): it does where there is a table and any gradient is asked for.
template <typename T, int MODE>
constexpr bool two_parts() { return sizeof(T) == 2 && MODE != kPlain; }

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

// A value that is the same in every lane, in a scalar register (a quotient is computed in vector registers, and what is
// derived from it stays there unless told)
__device__ __forceinline__ int uni(int v) { return __builtin_amdgcn_readfirstlane(v); }

// Position of a batch element's first query, and how many keys any of its queries sees: what lies behind is never read, and
// has zero gradients (the unfilled end of a cache may hold anything)
__device__ __forceinline__ int first_position(const Args& a, int b) {
  return uni(a.q_start ? min(max(a.q_start[b], -kMaxStart), kMaxStart) : a.q_start0);
}
__device__ __forceinline__ int used_keys(const Args& a, int b, int start) {
  const int n = a.lens ? min(max(a.lens[b], 0), a.Sk) : a.Sk;
  return uni(a.causal ? min(n, max(start + a.Sq, 0)) : n);
}

// Workgroup -> (sequence, tile): `pairs` sequences (a batch element's head) of n tiles each. Tiles of one sequence stay on
// one XCD. Causal tiles are of unequal work, rank 0 the longest: rank by rank then, the longest of all sequences first, so
// that what comes last is short; when all workgroups are resident at once (at most two a CU) the second half of the ranks
// goes the other way round, so that a long and a short one share a CU. That deals sequences to the XCDs by eights: other
// numbers of them are dealt in order, without regard to the work (causal 8192 tokens, heads of 64, forward / dQ / dK, dV:
// 1 head 93 / 87 / 113 us, 4 heads 101 / 97 / 126, 8 heads 110 / 140 / 178, 12 heads 186 / 206 / 263, 16 heads 190 / 200 /
// 255).
__device__ __forceinline__ void place(int pairs, int n, bool causal, int& pair, int& rank) {
  const int bid = blockIdx.x;
  if (causal && !(pairs & 7)) {
    const int r = uni(bid / pairs), p = bid - r * pairs, first = (n + 1) / 2;
    pair = (p & 7) * (pairs >> 3) + (p >> 3);
    rank = pairs * n > 512 || r < first ? r : n - 1 - (r - first);
  } else {
    const int id = uni(xcd_contiguous(bid, pairs * n));
    pair = uni(id / n);
    rank = id - pair * n;
  }
}

// ================================================================================================== forward
// PARTS 2: P enters O as two bf16 numbers, its rounding and what that left. D = rowsum(dO * O) takes over the roundings of the
// P in O, each row's one error in all of its dT, and the sums over many rows in a table's gradient show it (relative error
// against 64 bits 0.0015 to 0.0033 with one part, 0.0012 to 0.0018 with two, most of that dTable's own rounding; dQ and
// dK, rounded more coarsely by themselves, keep theirs). 64 x 512 x 12 heads of 64: 91 us with one part, 111 with two. The pass
// is told that gradients are asked for, not which: with a table that takes none it is two as well.
template <typename T, int D, int MODE, int GROUPS, int PARTS>
__global__ __launch_bounds__(256 * GROUPS, (sizeof(T) == 2 ? (D <= 64 ? 4 : 2) : (D <= 64 ? 2 : GROUPS))) void fwd_kernel(Args a) {
  constexpr int KT = key_tile<T>(), JB = KT / 16, DB = D / 16, DS = D / 32, IMG = Tile<T, D, KT>::IMG;
  extern __shared__ __attribute__((aligned(16))) char smem[];      // [2][K | V], [2][key bias of the tile], band
  const int tid = threadIdx.x & 255, lane = tid & 63, wid = uni(tid >> 6), grp = GROUPS > 1 ? uni(threadIdx.x >> 8) : 0;
  char* mem = smem + grp * (4 * IMG + 8 * KT);                     // the group's tile images and key biases
  float* kbl = reinterpret_cast<float*>(mem + 4 * IMG);
  float* band = reinterpret_cast<float*>(smem + GROUPS * (4 * IMG + 8 * KT));
  const int fr = lane & 15, g = lane >> 4;
  const int nqt = (a.Sq + kRows - 1) / kRows;
  int bh, rank;
  place(a.B * a.nh, nqt, a.causal, bh, rank);
  const int b = uni(bh / a.nh), h = bh - b * a.nh, qt = a.causal ? nqt - 1 - rank : rank;
  const int kvh = uni(h / (a.nh / a.nkv));
  const int q0 = qt * kRows + wid * 32;
  const int start = first_position(a, b), klen = used_keys(a, b, start);
  const int pos0 = start + q0;
  const float c = a.score_scale * kLog2e;
  const T* qp = (const T*)a.q.p + b * a.q.sb + h * a.q.sh;
  const float* kbp = MODE == kKeys ? a.key_bias + (long long)b * a.Sk : nullptr;
  const bool rel = MODE == kRel || (MODE == kKeys && a.table);

  Frag<T> qf[2][DS];
#pragma unroll
  for (int qb = 0; qb < 2; ++qb) {
    const T* row = qp + (long long)min(q0 + qb * 16 + fr, a.Sq - 1) * a.q.ss;
#pragma unroll
    for (int ks = 0; ks < DS; ++ks) {
      frag_global(qf[qb][ks], row, ks * 32 + g * 8, ks * 32 + g * 8 < a.hd);
      if (MODE == kKeys) times(qf[qb][ks], a.unit);
    }
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

  const Reader<T, D> rd(lane);
  Tile<T, D, KT> kr((const T*)a.k.p + b * a.k.sb + kvh * a.k.sh, a.k.ss, a.hd, tid);
  Tile<T, D, KT> vr((const T*)a.v.p + b * a.v.sb + kvh * a.v.sh, a.v.ss, a.hd, tid);
  float kbr = 0.f, kbn[Tile<T, D, KT>::N];
  if (MODE == kKeys) row_bias(kbn, kr.row, kbp + grp * KT, klen - grp * KT);
  auto fetch = [&](int t) {
    char* img = mem + (t / GROUPS & 1) * 2 * IMG;
    const int left = klen - t * KT;
    if (MODE == kKeys) {
      kr.load_masked(t, left, img, wid, kbn);
      vr.load_masked(t, left, img + IMG, wid, kbn);
      if (tid < KT) kbr = tid < left ? kbp[t * KT + tid] : -INFINITY;
      row_bias(kbn, kr.row, kbp + (t + GROUPS) * KT, left - GROUPS * KT);          // (the next tile's loads must not wait for these)
    } else {
      kr.load(t, left, img, wid);
      vr.load(t, left, img + IMG, wid);
    }
  };
  auto put = [&](int t) {
    char* img = mem + (t / GROUPS & 1) * 2 * IMG;
    kr.put(img);
    vr.put(img + IMG);
    if (MODE == kKeys && tid < KT) kbl[(t / GROUPS & 1) * KT + tid] = to_score_units(a, kbr);
    loads_done();
  };
  if (grp < nt) fetch(grp);
  if (rel && grp == 0) fill_band(a, h, band, tid);
  if (grp < nt) put(grp);
  __syncthreads();
  for (int t = grp; t - grp < nt; t += GROUPS) {        // (the groups take turns; all of them keep step)
    const char* kimg = mem + (t / GROUPS & 1) * 2 * IMG;
    const char* vimg = kimg + IMG;
    const int kt = t * KT;
    if (t + GROUPS < nt) fetch(t + GROUPS);
    // a wave whose rows all end before this tile, or that has no rows, only keeps step
    if (t < nt && q0 < a.Sq && (!a.causal || kt <= pos0 + 31)) {
      f32x4 s[JB][2];
#pragma unroll
      for (int jb = 0; jb < JB; ++jb) {
        f32x4 x = {0.f, 0.f, 0.f, 0.f};
        if (MODE == kKeys) x = *reinterpret_cast<const f32x4*>(kbl + (t / GROUPS & 1) * KT + jb * 16 + g * 4);
        s[jb][0] = x;
        s[jb][1] = x;
      }
      if (rel) {
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
#pragma unroll
      for (int ks = 0; ks < DS; ++ks)
#pragma unroll
        for (int jb = 0; jb < JB; ++jb) {
          Frag<T> kf;
          rd.read_row(kf, kimg, jb * 16, ks);
#pragma unroll
          for (int qb = 0; qb < 2; ++qb) s[jb][qb] = mma(kf, qf[qb][ks], s[jb][qb]);
        }
      if (kt + KT > klen || (a.causal && kt + KT - 1 > pos0)) {
#pragma unroll
        for (int qb = 0; qb < 2; ++qb) {
          const int end = (a.causal ? min(klen, pos0 + qb * 16 + fr + 1) : klen) - kt - 4 * g;
#pragma unroll
          for (int jb = 0; jb < JB; ++jb)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (jb * 16 + r >= end) s[jb][qb][r] = -INFINITY;
        }
      }
      // The maximum that is taken off need not be the row's exact one, only near enough for the exponentials: it moves,
      // and O and the sums with it, when a row outgrows it by a factor of 2^8, which after the first tiles hardly happens.
      // scale > 0: the maximum commutes with the scaling. With key biases the difference is taken in score units, where
      // it is exact: the product of a lowest-value mask with c is rounded by far more than 1.
      float mx[2];
#pragma unroll
      for (int qb = 0; qb < 2; ++qb) {
        mx[qb] = -INFINITY;
#pragma unroll
        for (int jb = 0; jb < JB; ++jb)
#pragma unroll
          for (int r = 0; r < 4; ++r) mx[qb] = fmaxf(mx[qb], s[jb][qb][r]);
        mx[qb] = group_max(mx[qb]);
        if (MODE != kKeys) mx[qb] *= c;
      }
      const float lim = MODE == kKeys ? 8.f / c : 8.f;
      const bool grow0 = mx[0] > m[0] + lim, grow1 = mx[1] > m[1] + lim;
      if (__any(grow0 || grow1)) {
#pragma unroll
        for (int qb = 0; qb < 2; ++qb) {
          const float mn = (qb ? grow1 : grow0) ? mx[qb] : m[qb];
          const float alpha = mn == m[qb] ? 1.f : fexp2(MODE == kKeys ? (m[qb] - mn) * c : m[qb] - mn);
          m[qb] = mn;
          l[qb] *= alpha;
#pragma unroll
          for (int db = 0; db < DB; ++db) o[db][qb] *= alpha;
        }
      }
#pragma unroll
      for (int qb = 0; qb < 2; ++qb) {
        const float ref = m[qb] == -INFINITY ? 0.f : m[qb];          // nothing seen yet: every term is exp2(-inf)
        float sum = 0.f;
#pragma unroll
        for (int jb = 0; jb < JB; ++jb)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float p = fexp2(MODE == kKeys ? (s[jb][qb][r] - ref) * c : fmaf(s[jb][qb][r], c, -ref));
            s[jb][qb][r] = p;
            sum += p;
          }
        l[qb] += sum;                                                // per lane; combined over the lane group at the end
      }
#pragma unroll
      for (int ks = 0; ks < KT / 32; ++ks) {
        Frag<T> pf[2], pr[2];
#pragma unroll
        for (int qb = 0; qb < 2; ++qb) {
          pack(pf[qb], s[2 * ks][qb], s[2 * ks + 1][qb]);
          if (PARTS == 2) pack_rest(pr[qb], s[2 * ks][qb], s[2 * ks + 1][qb], pf[qb]);
        }
#pragma unroll
        for (int db = 0; db < DB; ++db) {
          Frag<T> vf;
          rd.read_tr(vf, vimg, db, ks);
#pragma unroll
          for (int qb = 0; qb < 2; ++qb) o[db][qb] = mma(vf, pf[qb], o[db][qb]);
          if (PARTS == 2) {
#pragma unroll
            for (int qb = 0; qb < 2; ++qb) o[db][qb] = mma(vf, pr[qb], o[db][qb]);
          }
        }
      }
    }
    if (t + GROUPS < nt) put(t + GROUPS);
    __syncthreads();
  }
#pragma unroll
  for (int qb = 0; qb < 2; ++qb) l[qb] = group_sum(l[qb]);
  if (GROUPS > 1) {                                     // join: the second group's sums through its images' memory
    float* oj = reinterpret_cast<float*>(smem + 4 * IMG + 8 * KT) + wid * 32 * D, *mj = band + (wid * 2) * 64;
    if (grp == 1) {
#pragma unroll
      for (int qb = 0; qb < 2; ++qb) {
#pragma unroll
        for (int db = 0; db < DB; ++db) *reinterpret_cast<f32x4*>(oj + ((qb * DB + db) * 64 + lane) * 4) = o[db][qb];
        mj[qb * 64 + lane] = m[qb];
        mj[4 * 2 * 64 + qb * 64 + lane] = l[qb];
      }
    }
    __syncthreads();
    if (grp == 1) return;
#pragma unroll
    for (int qb = 0; qb < 2; ++qb) {
      const float m1 = mj[qb * 64 + lane], l1 = mj[4 * 2 * 64 + qb * 64 + lane], mm = fmaxf(m[qb], m1), ref = mm == -INFINITY ? 0.f : mm;
      const float f0 = fexp2(MODE == kKeys ? (m[qb] - ref) * c : m[qb] - ref), f1 = fexp2(MODE == kKeys ? (m1 - ref) * c : m1 - ref);
      m[qb] = mm;
      l[qb] = l[qb] * f0 + l1 * f1;
#pragma unroll
      for (int db = 0; db < DB; ++db) o[db][qb] = o[db][qb] * f0 + *reinterpret_cast<const f32x4*>(oj + ((qb * DB + db) * 64 + lane) * 4) * f1;
    }
  }
#pragma unroll
  for (int qb = 0; qb < 2; ++qb) {
    const int q = q0 + qb * 16 + fr;
    const float lt = l[qb];
    const float inv = lt == 0.f ? 0.f : 1.f / lt;
    T* row = (T*)a.out.p + b * a.out.sb + (long long)q * a.out.ss + h * a.out.sh;
    const int hd = q < a.Sq ? a.hd : 0;                 // (every lane takes part in the swaps)
#pragma unroll
    for (int p = 0; p < DB / 2; ++p) {
      const f32x4 v0 = o[2 * p][qb] * inv, v1 = o[2 * p + 1][qb] * inv;
      store_pair(row, p, g, hd, v0, v1);
      if (sizeof(T) == 2 && a.fine) {
        unsigned x = finer4(v0), y = finer4(v1);
        gather8(x, y);
        if (p * 32 + g * 8 < hd) *reinterpret_cast<u32x2_t*>(fine_row(a, b, q, h) + p * 32 + g * 8) = u32x2_t{x, y};
      }
    }
    if (q < a.Sq) {
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
// 8 x 1 on 4001 keys, 16 heads on 4 of 128, the two kernels, us: bf16 13 + 4 (floor 9: two tiles a wave, so that the start, the
// join and the second launch dominate), fp32 28 + 5; with key biases 20 and 45. The bucket of each score is found border by
// border: with a one-sided table of 32 buckets 23 and 38, of 128 49 and 64.
constexpr int kFewRows = 32, kFewKeys = 32;

// O and the row's statistics of row r of a key head's rows
template <typename T, int MODE>
__device__ __forceinline__ void few_store(const Args& a, int b, int kvh, int group, int r, int d, float mm, float lt,
                                          const f32x4& acc, float c) {
  const int i = r / group, h = kvh * group + r - i * group;
  const float inv = lt == 0.f ? 0.f : 1.f / lt;
  if (d < a.hd) {
    store4((T*)a.out.p + b * a.out.sb + (long long)i * a.out.ss + h * a.out.sh + d, acc * inv);
    if (sizeof(T) == 2 && a.fine) *reinterpret_cast<unsigned*>(fine_row(a, b, i, h) + d) = finer4(acc * inv);
  }
  if (d == 0 && a.stat) {
    const long long at = ((long long)b * a.nh + h) * a.Sq + i, n = (long long)a.B * a.nh * a.Sq;
    a.stat[at] = lt == 0.f ? INFINITY : (MODE == kKeys ? mm : mm * c);        // the units of fwd_kernel
    a.stat[n + at] = lt == 0.f ? 0.f : flog2(lt);
  }
}

template <typename T, int D, int QB, int MODE>
__global__ __launch_bounds__(256, 2) void few_kernel(Args a) {
  constexpr int DB = D / 16, DS = D / 32, IMG = kFewKeys * row_stride<T, D>(), JOIN = QB * 16 * (D + 4) * 4;
  constexpr int kChunk = 16 / (int)sizeof(T), kPerRow = D / kChunk, NV = kFewKeys * kPerRow / 64;
  extern __shared__ __attribute__((aligned(16))) char smem[];      // [4 waves][V image, then O], [4][2][rows], table
  constexpr int REGION = IMG > JOIN ? IMG : JOIN;
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int fr = lane & 15, g = lane >> 4;
  char* vimg = smem + wid * REGION;
  float* ml = reinterpret_cast<float*>(smem + 4 * REGION);
  float* tab = ml + 4 * 2 * QB * 16;
  const int group = uni(a.nh / a.nkv), rows = a.Sq * group;
  const int bk = uni(blockIdx.x / a.splits), split = blockIdx.x - bk * a.splits, b = uni(bk / a.nkv), kvh = bk - b * a.nkv;
  const int start = first_position(a, b), klen = used_keys(a, b, start);
  const float c = a.score_scale * kLog2e;
  const T* kp = (const T*)a.k.p + b * a.k.sb + kvh * a.k.sh;
  const T* vp = (const T*)a.v.p + b * a.v.sb + kvh * a.v.sh;
  const float* kbp = MODE == kKeys ? a.key_bias + (long long)b * a.Sk : nullptr;
  const bool rel = MODE == kRel || (MODE == kKeys && a.table);
  const bool two = two_parts<T, MODE>() && a.table && a.fine;      // see fwd_kernel's PARTS

  if (rel) {
    for (int i = tid; i < group * a.buckets; i += 256) {
      const int hg = i / a.buckets;
      tab[i] = learned_bias(a, table_at(a, i - hg * a.buckets, kvh * group + hg));
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
    for (int ks = 0; ks < DS; ++ks) {
      frag_global(qf[qb][ks], row, ks * 32 + g * 8, ks * 32 + g * 8 < a.hd);
      if (MODE == kKeys) times(qf[qb][ks], a.unit);
    }
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

  const Reader<T, D> rd(lane);
  Frag<T> kf[2][DS];
  u32x4_t vr[NV];
  f32x4 kb[2];
  const unsigned kld = (unsigned)a.k.ss * (unsigned)sizeof(T), vld = (unsigned)a.v.ss * (unsigned)sizeof(T);
  auto fetch = [&](int t) {                              // (left >= 1: the tile starts before kend)
    const int k0 = t * kFewKeys, left = klen - k0;
    const unsigned used = (unsigned)a.hd * (unsigned)sizeof(T);
    const __amdgpu_buffer_rsrc_t kr = tile_rsrc(kp + (long long)k0 * a.k.ss, kld, used, left, kFewKeys);
    const __amdgpu_buffer_rsrc_t vs = tile_rsrc(vp + (long long)k0 * a.v.ss, vld, used, left, kFewKeys);
#pragma unroll
    for (int jb = 0; jb < 2; ++jb) {
      const int row = jb * 16 + fr;
      const bool in = row < left && !(MODE == kKeys && kbp[k0 + row] == -INFINITY);
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
      if (MODE == kKeys) {
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
      const bool in = row < left && ch * kChunk < a.hd && !(MODE == kKeys && kbp[k0 + row] == -INFINITY);
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
        if (MODE == kKeys) s[jb][qb] = kb[jb];
        if (rel) {
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
      *reinterpret_cast<u32x4_t*>(vimg + chunk_at<T, D>(row, ch)) = vr[u];
    }
    if (t + 4 < t1) fetch(t + 4);
    Frag<T> pf[QB], pr[QB];
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
      if (two) pack_rest(pr[qb], s[0][qb], s[1][qb], pf[qb]);
    }
    asm volatile("" ::: "memory");
#pragma unroll
    for (int db = 0; db < DB; ++db) {
      Frag<T> vf;
      rd.read_tr(vf, vimg, db, 0);
#pragma unroll
      for (int qb = 0; qb < QB; ++qb) {
        o[db][qb] = mma(vf, pf[qb], o[db][qb]);
        if (two) o[db][qb] = mma(vf, pr[qb], o[db][qb]);
      }
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
      few_store<T, MODE>(a, b, kvh, group, r, d, mm, lt, acc, c);
    }
  }
}

// One workgroup a row: its threads share out the row's splits as well as its elements, so that no thread waits for more
// than a few loads one after the other (one wave a row, walking the splits: 13.5 us where few_kernel itself takes 12).
template <typename T, int D, int MODE>
__global__ __launch_bounds__(256) void few_join_kernel(Args a) {
  constexpr int L = D / 4, S = 256 / L;                  // lanes of a row, splits taken at a time
  __shared__ __attribute__((aligned(16))) float red[S][D + 4];
  __shared__ float fac[64], stats[2];
  const int group = a.nh / a.nkv, rows = a.Sq * group, tid = threadIdx.x;
  const long long row = blockIdx.x, n_rows = gridDim.x;
  const float c = a.score_scale * kLog2e;
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
    few_store<T, MODE>(a, b, bk - b * a.nkv, group, (int)(row - (long long)bk * rows), d, stats[0], stats[1], acc, c);
  }
}

// ================================================================================================== backward: dQ
// Sums over the diagonals of a wave's dT, for the relative bias's gradient. dT comes in blocks of 16 keys x 16 queries,
// lane (fr, g) holding query fr and keys 4 g + r; blocks on one block diagonal J (16 keys = one step) are added in place
// first, so e_J(fr, g, r) belongs to distance 16 J + 4 g + r - fr. Rotating a register by r lanes within its 16 brings
// the lanes of one distance together, and a lane that wraps around carries a value of distance 16 J + 16 - ..., which is
// exactly the place of the NEXT block's rotation: selecting between e_J and e_(J-1) before the rotation makes every lane
// right. Three such rotations fold r away, then one by 4 g per lane group folds g, and two half swaps sum the lane groups
// and put two blocks side by side: 32 lanes with 32 consecutive distances, one LDS addition per 32 x 32 scores where one
// per register with colliding lanes (ds_add_f32, 12 of them) took three quarters of the kernel (0.54 ms instead of 0.17 at
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
  // gx[j]: block diagonal j - 1 of 32 keys x 32 queries, j = 0, 1, 2. Completes blocks -1 and 0: the sum of distance
  // 16 (b - 1) - fr (relative to the first key and query) is returned in lane group b = 0, 1.
  __device__ __forceinline__ float add(const f32x4 (&gx)[3], int fr, int g) {
    float v[2];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
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
    carry = gx[2];
    const float r = rows(v[0], v[1]);                    // lane groups 0, 2: block 0 of groups (0, 1), (2, 3); 1, 3: block 1
    return halves(r, r);
  }
};

// A workgroup owns 128 query rows and walks the keys. It also writes D = rowsum(dO * O) for the dK / dV kernel and sums
// the relative bias's gradient: by distance (DiagonalSums, into a band of the wave's own, where no two lanes of an
// addition meet) where a tile touches the band,
// into one of two registers where it lies beyond.
template <typename T, int D, int MODE, int GROUPS>
__global__ __launch_bounds__(256 * GROUPS, (sizeof(T) == 2 ? (D <= 32 ? 4 : D <= 64 && MODE == kPlain && GROUPS == 1 ? 3 : 2) : GROUPS)) void bwd_dq_kernel(Args a) {
  constexpr int KT = key_tile<T>(), DB = D / 16, DS = D / 32, IMG = Tile<T, D, KT>::IMG;
  extern __shared__ __attribute__((aligned(16))) char smem[];      // [2][K | V], [2][key bias], band, band gradients
  const int tid = threadIdx.x & 255, lane = tid & 63, wid = uni(tid >> 6), grp = GROUPS > 1 ? uni(threadIdx.x >> 8) : 0;
  char* mem = smem + grp * (4 * IMG + 8 * KT);                     // the group's tile images and key biases
  float* kbl = reinterpret_cast<float*>(mem + 4 * IMG);
  float* band = reinterpret_cast<float*>(smem + GROUPS * (4 * IMG + 8 * KT));
  const bool rel = MODE == kRel || (MODE == kKeys && a.table);
  const int nband = rel ? band_size(a) : 0;
  float* gband = band + nband;                                     // [waves][nband], then two far sums a wave
  const int fr = lane & 15, g = lane >> 4;
  const int nqt = (a.Sq + kRows - 1) / kRows;
  int bh, rank;
  place(a.B * a.nh, nqt, a.causal, bh, rank);
  const int b = uni(bh / a.nh), h = bh - b * a.nh, qt = a.causal ? nqt - 1 - rank : rank;
  const int kvh = uni(h / (a.nh / a.nkv));
  const int q0 = qt * kRows + wid * 32;
  const int start = first_position(a, b), klen = used_keys(a, b, start);
  const int pos0 = start + q0;
  const float c = a.score_scale * kLog2e;
  const T* qp = (const T*)a.q.p + b * a.q.sb + h * a.q.sh;
  const T* op = (const T*)a.out.p + b * a.out.sb + h * a.out.sh;
  const T* dop = (const T*)a.dout.p + b * a.dout.sb + h * a.dout.sh;
  const float* kbp = MODE == kKeys ? a.key_bias + (long long)b * a.Sk : nullptr;
  const bool want_tab = rel && a.dtab;

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
      if constexpr (sizeof(T) == 2) {
        u32x2_t fine = {0u, 0u};
        if (e < a.hd) fine = *reinterpret_cast<const u32x2_t*>(fine_row(a, b, qc, h) + e);
        part = dot_fine(dof[qb][ks], of, fine, part);
      } else {
        part = dot(of, dof[qb][ks], part);
      }
      if (MODE == kKeys) times(qf[qb][ks], a.unit);
    }
    const long long i = ((long long)b * a.nh + h) * a.Sq + qc, n = (long long)a.B * a.nh * a.Sq;
    dl[qb] = group_sum(part);
    m2[qb] = q < a.Sq ? a.stat[i] : INFINITY;            // rows past the end: probabilities 0
    ll[qb] = q < a.Sq ? a.stat[n + i] : 0.f;
    if (MODE != kKeys) m2[qb] += ll[qb];
    if (g == 0 && grp == 0) {
      float* w = a.rows + row_tile(a, bh, q >> 6) + (q & 63);
      w[0] = m2[qb];
      w[64] = ll[qb];
      w[128] = -dl[qb];
    }
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

  const Reader<T, D> rd(lane);
  Tile<T, D, KT> kr((const T*)a.k.p + b * a.k.sb + kvh * a.k.sh, a.k.ss, a.hd, tid);
  Tile<T, D, KT> vr((const T*)a.v.p + b * a.v.sb + kvh * a.v.sh, a.v.ss, a.hd, tid);
  float kbr = 0.f, kbn[Tile<T, D, KT>::N];
  if (MODE == kKeys) row_bias(kbn, kr.row, kbp + grp * KT, klen - grp * KT);
  auto fetch = [&](int t) {
    char* img = mem + (t / GROUPS & 1) * 2 * IMG;
    const int left = klen - t * KT;
    if (MODE == kKeys) {
      kr.load_masked(t, left, img, wid, kbn);
      vr.load_masked(t, left, img + IMG, wid, kbn);
      if (tid < KT) kbr = tid < left ? kbp[t * KT + tid] : -INFINITY;
      row_bias(kbn, kr.row, kbp + (t + GROUPS) * KT, left - GROUPS * KT);          // (the next tile's loads must not wait for these)
    } else {
      kr.load(t, left, img, wid);
      vr.load(t, left, img + IMG, wid);
    }
  };
  auto put = [&](int t) {
    char* img = mem + (t / GROUPS & 1) * 2 * IMG;
    kr.put(img);
    vr.put(img + IMG);
    if (MODE == kKeys && tid < KT) kbl[(t / GROUPS & 1) * KT + tid] = to_score_units(a, kbr);
    loads_done();
  };
  if (grp < nt) fetch(grp);
  if (rel && grp == 0) fill_band(a, h, band, tid);
  if (want_tab)
    for (int i = threadIdx.x; i < 4 * GROUPS * nband; i += 256 * GROUPS) gband[i] = 0.f;
  float* gmine = gband + (grp * 4 + wid) * nband;
  DiagonalSums diag;
  diag.reset();
  int diag_at = 0;                                       // band entry of the next tile's first distance; 0: no tile yet
  auto finish_diagonals = [&]() {                        // what the last block on the band left incomplete
    const f32x4 none[3] = {};
    const float v = diag.add(none, fr, g);
    if (g < 2) atomicAdd(gmine + diag_at + 16 * (g - 1) - fr, v);
    diag.reset();
    diag_at = 0;
  };
  if (grp < nt) put(grp);
  __syncthreads();
  for (int t = grp; t - grp < nt; t += GROUPS) {        // (the groups take turns; all of them keep step)
    const char* kimg = mem + (t / GROUPS & 1) * 2 * IMG;
    const char* vimg = kimg + IMG;
    const int kt = t * KT;
    if (t + GROUPS < nt) fetch(t + GROUPS);
    if (t < nt && q0 < a.Sq && (!a.causal || kt <= pos0 + 31)) {
      const bool far = rel && (kt + KT - 1 - pos0 <= -a.max_dist || kt - (pos0 + 31) >= a.right);
      const int at0 = kt + 4 * g - pos0 - fr + a.max_dist + kMargin;    // band entry of (key 4 g of block 0, query fr)
      const float xf = rel && far ? (kt < pos0 ? band[0] : band[nband - 1]) : 0.f;
      const bool edge = kt + KT > klen || (a.causal && kt + KT - 1 > pos0);
#pragma unroll
      for (int hf = 0; hf < KT / 32; ++hf) {
        f32x4 s[2][2], dp[2][2], x[3];                   // x: key block minus query block of the half -1, 0, 1
#pragma unroll
        for (int j = 0; j < 3; ++j) x[j] = f32x4{xf, xf, xf, xf};
        if (rel && !far) {
#pragma unroll
          for (int j = 0; j < 3; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) x[j][r] = band[at0 + (hf * 2 + j - 1) * 16 + r];
        }
#pragma unroll
        for (int jj = 0; jj < 2; ++jj) {
          f32x4 kb = {0.f, 0.f, 0.f, 0.f};
          if (MODE == kKeys) kb = *reinterpret_cast<const f32x4*>(kbl + (t / GROUPS & 1) * KT + (hf * 2 + jj) * 16 + g * 4);
#pragma unroll
          for (int qb = 0; qb < 2; ++qb) {
            s[jj][qb] = MODE == kKeys ? kb + x[jj + 1 - qb] : MODE == kRel ? x[jj + 1 - qb] : f32x4{0.f, 0.f, 0.f, 0.f};
            dp[jj][qb] = f32x4{-dl[qb], -dl[qb], -dl[qb], -dl[qb]};   // dP - D comes out of the product
          }
        }
#pragma unroll
        for (int ks = 0; ks < DS; ++ks)
#pragma unroll
          for (int jj = 0; jj < 2; ++jj) {
            Frag<T> kf, vf;
            rd.read_row(kf, kimg, (hf * 2 + jj) * 16, ks);
            rd.read_row(vf, vimg, (hf * 2 + jj) * 16, ks);
#pragma unroll
            for (int qb = 0; qb < 2; ++qb) {
              s[jj][qb] = mma(kf, qf[qb][ks], s[jj][qb]);
              dp[jj][qb] = mma(vf, dof[qb][ks], dp[jj][qb]);
            }
          }
        if (edge) {
#pragma unroll
          for (int qb = 0; qb < 2; ++qb) {
            const int end = (a.causal ? min(klen, pos0 + qb * 16 + fr + 1) : klen) - kt - 4 * g;
#pragma unroll
            for (int jj = 0; jj < 2; ++jj)
#pragma unroll
              for (int r = 0; r < 4; ++r)
                if ((hf * 2 + jj) * 16 + r >= end) s[jj][qb][r] = -INFINITY;
          }
        }
        Frag<T> dsf[2];
        f32x4 gx[3];
#pragma unroll
        for (int j = 0; j < 3; ++j) gx[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int qb = 0; qb < 2; ++qb) {
#pragma unroll
          for (int jj = 0; jj < 2; ++jj) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              // with key biases the row maximum may be so large (a row of lowest-value masks) that the logarithm of the
              // sum is lost next to it: the two are taken off one after the other
              const float p = fexp2(MODE == kKeys ? fmaf(s[jj][qb][r] - m2[qb], c, -ll[qb]) : fmaf(s[jj][qb][r], c, -m2[qb]));
              s[jj][qb][r] = p * dp[jj][qb][r];
            }
            if (MODE != kPlain) gx[jj + 1 - qb] += s[jj][qb];
          }
          pack(dsf[qb], s[0][qb], s[1][qb]);
        }
        if (want_tab) {
          if (far) {
            const f32x4 v = gx[0] + gx[1] + gx[2];
            if (kt < pos0) far_l += (v[0] + v[1]) + (v[2] + v[3]);
            else far_r += (v[0] + v[1]) + (v[2] + v[3]);
          } else {
            // blocks of 32 keys that follow one another hand on what is incomplete; the groups' tiles do not
            const float v = diag.add(gx, fr, g);
            diag_at = kt - pos0 + hf * 32 + a.max_dist + kMargin;
            if (g < 2) atomicAdd(gmine + diag_at + 16 * (g - 1) - fr, v);
            diag_at += 32;
            if (GROUPS > 1 && hf == KT / 32 - 1) finish_diagonals();
          }
        }
#pragma unroll
        for (int db = 0; db < DB; ++db) {
          Frag<T> ktr;
          rd.read_tr(ktr, kimg, db, hf);
#pragma unroll
          for (int qb = 0; qb < 2; ++qb) dq[db][qb] = mma(ktr, dsf[qb], dq[db][qb]);
        }
        if (D > 64) __builtin_amdgcn_sched_barrier(0);   // the halves interleaved would not fit the registers
      }
    }
    if (t + GROUPS < nt) put(t + GROUPS);
    __syncthreads();
  }
  if (GROUPS > 1) {                                     // join: the second group's sums through its images' memory
    float* oj = reinterpret_cast<float*>(smem + 4 * IMG + 8 * KT) + wid * 32 * D;
    if (grp == 1) {
#pragma unroll
      for (int qb = 0; qb < 2; ++qb)
#pragma unroll
        for (int db = 0; db < DB; ++db) *reinterpret_cast<f32x4*>(oj + ((qb * DB + db) * 64 + lane) * 4) = dq[db][qb];
    }
    __syncthreads();
    if (grp == 0) {
#pragma unroll
      for (int qb = 0; qb < 2; ++qb)
#pragma unroll
        for (int db = 0; db < DB; ++db) dq[db][qb] += *reinterpret_cast<const f32x4*>(oj + ((qb * DB + db) * 64 + lane) * 4);
    }
  }
#pragma unroll
  for (int qb = 0; qb < 2; ++qb) {
    const int q = opaque(q0 + qb * 16 + fr);             // (the rows' addresses are not for the loop to keep)
    T* row = (T*)a.dq.p + b * a.dq.sb + (long long)q * a.dq.ss + h * a.dq.sh;
    if (grp == 0) {
#pragma unroll
      for (int p = 0; p < DB / 2; ++p) store_pair(row, p, g, q < a.Sq ? a.hd : 0, dq[2 * p][qb] * a.scale, dq[2 * p + 1][qb] * a.scale);
    }
  }
  if (want_tab) {
    if (diag_at) finish_diagonals();
    float* fars = gband + 4 * GROUPS * nband;
    far_l = wave_sum(far_l);
    far_r = wave_sum(far_r);
    if (lane == 0) { fars[(grp * 4 + wid) * 2] = far_l; fars[(grp * 4 + wid) * 2 + 1] = far_r; }
    __syncthreads();
    for (int i = threadIdx.x; i < nband; i += 256 * GROUPS) {        // (no wave reads the band any more)
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < 4 * GROUPS; ++w) v += gband[w * nband + i];
      band[i] = v;
    }
    __syncthreads();
    // a bucket's distances are shared out over the lanes of a group (at least two: 128 buckets, 256 threads)
    int lanes = 64;
    while (lanes * a.buckets > 256) lanes >>= 1;
    const int u = threadIdx.x / lanes, first = threadIdx.x & (lanes - 1);
    if (u < a.buckets) {
      int lo, hi;
      bucket_range(a, u, lo, hi);
      float v = 0.f;
      for (int i = lo + first; i <= hi; i += lanes) v += band[i + a.max_dist + kMargin];
      if (first == 0 && lo == -a.max_dist - kMargin && lo <= hi)
        for (int w = 0; w < 4 * GROUPS; ++w) v += fars[w * 2];
      if (first == 0 && hi == a.right + kMargin && lo <= hi)
        for (int w = 0; w < 4 * GROUPS; ++w) v += fars[w * 2 + 1];
      for (int o = lanes >> 1; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
      if (first == 0) a.dtab[(((long long)b * nqt + qt) * a.nh + h) * a.buckets + u] = v;
    }
  }
}

// ================================================================================================== backward: dK, dV
// A workgroup owns 128 keys of one key head, a wave 32 of them, and walks the query tiles of every query head of the
// group: gradients of shared heads are summed in the accumulators. The KEY rides on the lane here.
template <typename T, int D, int MODE, int GROUPS>
__global__ __launch_bounds__(256 * GROUPS, (sizeof(T) == 2 ? (D <= 32 ? 4 : D <= 64 && MODE == kPlain && GROUPS == 1 ? 3 : 2) : GROUPS)) void bwd_dkdv_kernel(Args a) {
  constexpr int QT = key_tile<T>(), DB = D / 16, DS = D / 32, IMG = Tile<T, D, QT>::IMG;
  extern __shared__ __attribute__((aligned(16))) char smem[];      // [2][Q | dO], [2][row statistics], band
  const int tid = threadIdx.x & 255, lane = tid & 63, wid = uni(tid >> 6), grp = GROUPS > 1 ? uni(threadIdx.x >> 8) : 0;
  char* mem = smem + grp * (4 * IMG + 8 * kRowStats);              // the group's tile images and row statistics
  float* stl = reinterpret_cast<float*>(mem + 4 * IMG);
  float* band = reinterpret_cast<float*>(smem + GROUPS * (4 * IMG + 8 * kRowStats));
  const int fr = lane & 15, g = lane >> 4;
  const int nkt = (a.Sk + kRows - 1) / kRows, group = uni(a.nh / a.nkv);
  int pair, rank;
  place(a.B * a.nkv * a.ksplits, nkt, a.causal, pair, rank);
  const int bk = uni(pair / a.ksplits), b = uni(bk / a.nkv), kvh = bk - b * a.nkv, split = pair - bk * a.ksplits;
  const int heads = uni(group / a.ksplits), kb0 = rank * kRows, k0 = kb0 + wid * 32;
  const int start = first_position(a, b), klen = used_keys(a, b, start);
  const float c = a.score_scale * kLog2e;
  const T* kp = (const T*)a.k.p + b * a.k.sb + kvh * a.k.sh;
  const T* vp = (const T*)a.v.p + b * a.v.sb + kvh * a.v.sh;
  const float* kbp = MODE == kKeys ? a.key_bias + (long long)b * a.Sk : nullptr;
  const bool rel = MODE == kRel || (MODE == kKeys && a.table);
  const Reader<T, D, (D <= 64)> rd(lane);

  Frag<T> kf[2][DS], vf[2][DS];
  float kbias[2];
  const unsigned kld = (unsigned)a.k.ss * (unsigned)sizeof(T), vld = (unsigned)a.v.ss * (unsigned)sizeof(T), used = (unsigned)a.hd * (unsigned)sizeof(T);
  const __amdgpu_buffer_rsrc_t krs = tile_rsrc(kp + (long long)k0 * a.k.ss, kld, used, klen - k0, 32);
  const __amdgpu_buffer_rsrc_t vrs = tile_rsrc(vp + (long long)k0 * a.v.ss, vld, used, klen - k0, 32);
#pragma unroll
  for (int kb = 0; kb < 2; ++kb) {
    const int k = k0 + kb * 16 + fr, kc = min(k, a.Sk - 1);
    kbias[kb] = MODE == kKeys ? to_score_units(a, kbp[kc]) : 0.f;
    if (k >= klen) kbias[kb] = -INFINITY;
    const bool in = kbias[kb] != -INFINITY;
#pragma unroll
    for (int ks = 0; ks < DS; ++ks) {
      const int e = ks * 32 + g * 8;
      if (D <= 64) {
        // (with a load under a condition each, the row addresses do not fit the registers next to the fragments, and every
        // load waits for the one before, the scratch memory being in between: 96 x 197 x 12 of 64 57 us, like this 48. The
        // instances for 128 come out with slower loops like this: 4 x 2048 causal 182 and 210)
        block_row(kf[kb][ks], krs, kld, kb * 16 + fr, e, in && e < a.hd);
        block_row(vf[kb][ks], vrs, vld, kb * 16 + fr, e, in && e < a.hd);
      } else {
        frag_global(kf[kb][ks], kp + (long long)kc * a.k.ss, e, in && e < a.hd);
        frag_global(vf[kb][ks], vp + (long long)kc * a.v.ss, e, in && e < a.hd);
      }
      if (MODE == kKeys) times(kf[kb][ks], a.unit);
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

  for (int hg = split * heads; hg < (split + 1) * heads; ++hg) {
    if (t0 >= ntq) break;
    const int h = kvh * group + hg;
    const float* rows = a.rows + row_tile(a, (long long)b * a.nh + h, 0);
    Tile<T, D, QT> qr((const T*)a.q.p + b * a.q.sb + h * a.q.sh, a.q.ss, a.hd, tid);
    Tile<T, D, QT> dr((const T*)a.dout.p + b * a.dout.sb + h * a.dout.sh, a.dout.ss, a.hd, tid);
    auto fetch = [&](int t) {
      char* img = mem + (t / GROUPS & 1) * 2 * IMG;
      qr.load(t, a.Sq - t * QT, img, wid);
      dr.load(t, a.Sq - t * QT, img + IMG, wid);
      if (wid == 0) {
        const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(rows) + (t * QT / 64) * (long long)kRowStats, 0, kRowStats * 4, 0x00020000);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)(stl + (t / GROUPS & 1) * kRowStats), 16, lane * 16, 0, 0, 0);
      }
    };
    auto put = [&](int t) {
      char* img = mem + (t / GROUPS & 1) * 2 * IMG;
      qr.put(img);
      dr.put(img + IMG);
      loads_done();
    };
    const int tg = t0 + grp;
    if (tg < ntq) fetch(tg);
    if (rel && grp == 0) fill_band(a, h, band, tid);     // (the previous head's last barrier has passed)
    if (tg < ntq) put(tg);
    __syncthreads();
    for (int t = tg; t - grp < ntq; t += GROUPS) {       // (the groups take turns; all of them keep step)
      const char* qimg = mem + (t / GROUPS & 1) * 2 * IMG;
      const char* dimg = qimg + IMG;
      const float* stc = stl + (t / GROUPS & 1) * kRowStats + (t * QT & 63);
      const int pos = start + t * QT;                    // position of the tile's first query
      if (t + GROUPS < ntq) fetch(t + GROUPS);
      if (t < ntq && k0 < klen && (!a.causal || k0 <= pos + QT - 1)) {
        const bool far = rel && (k0 + 31 - pos <= -a.max_dist || k0 - (pos + QT - 1) >= a.right);
        const bool edge = a.causal && k0 + 31 > pos;
        float xf = 0.f;
        if (far) xf = k0 < pos ? band[0] : band[band_size(a) - 1];
        const float* at = band + (k0 + fr - pos - 4 * g + a.max_dist + kMargin);   // (query 4 g of block 0, key fr of block 0)
#pragma unroll
        for (int hf = 0; hf < QT / 32; ++hf) {
          f32x4 p[2][2], ds[2][2];
#pragma unroll
          for (int ii = 0; ii < 2; ++ii) {
            const float* sr = stc + (hf * 2 + ii) * 16 + g * 4;
            const f32x4 nd = *reinterpret_cast<const f32x4*>(sr + 128);
            f32x4 s[2], dp[2];
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
              const float b0 = MODE == kKeys ? kbias[kb] + xf : MODE == kRel ? xf : 0.f;
              s[kb] = f32x4{b0, b0, b0, b0};
              dp[kb] = nd;                               // dP - D comes out of the product
            }
            if (rel && !far) {
#pragma unroll
              for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int r = 0; r < 4; ++r) s[kb][r] += at[(kb - ii - hf * 2) * 16 - r];
            }
#pragma unroll
            for (int ks = 0; ks < DS; ++ks) {
              Frag<T> qfr, dfr;
              rd.read_row(qfr, qimg, (hf * 2 + ii) * 16, ks);
              rd.read_row(dfr, dimg, (hf * 2 + ii) * 16, ks);
#pragma unroll
              for (int kb = 0; kb < 2; ++kb) {
                s[kb] = mma(qfr, kf[kb][ks], s[kb]);
                dp[kb] = mma(dfr, vf[kb][ks], dp[kb]);
              }
            }
            if (edge || (MODE != kKeys && edge_keys)) {  // with key biases a key past the end has -inf already
#pragma unroll
              for (int kb = 0; kb < 2; ++kb) {
                // rows of the tile before this one do not see the key
                const int key = k0 + kb * 16 + fr, first = key >= klen ? QT : a.causal ? key - pos - 4 * g : -QT;
#pragma unroll
                for (int r = 0; r < 4; ++r)
                  if ((hf * 2 + ii) * 16 + r < first) s[kb][r] = -INFINITY;
              }
            }
            const f32x4 mm = *reinterpret_cast<const f32x4*>(sr);
            f32x4 ls;
            if (MODE == kKeys) ls = *reinterpret_cast<const f32x4*>(sr + 64);
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                p[ii][kb][r] = fexp2(MODE == kKeys ? fmaf(s[kb][r] - mm[r], c, -ls[r]) : fmaf(s[kb][r], c, -mm[r]));
                ds[ii][kb][r] = p[ii][kb][r] * dp[kb][r];
              }
          }
          Frag<T> pf[2], dsf[2];
#pragma unroll
          for (int kb = 0; kb < 2; ++kb) {
            pack(pf[kb], p[0][kb], p[1][kb]);
            pack(dsf[kb], ds[0][kb], ds[1][kb]);
          }
#pragma unroll
          for (int db = 0; db < DB; ++db) {
            Frag<T> dot_, qt_;
            rd.read_tr(dot_, dimg, db, hf);
            rd.read_tr(qt_, qimg, db, hf);
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
              dv[db][kb] = mma(dot_, pf[kb], dv[db][kb]);
              dk[db][kb] = mma(qt_, dsf[kb], dk[db][kb]);
            }
          }
          if (D > 64) __builtin_amdgcn_sched_barrier(0);
        }
      }
      if (t + GROUPS < ntq) put(t + GROUPS);
      __syncthreads();
    }
  }
  if (GROUPS > 1) {                                     // join: the second group's sums through the images' memory, dK then dV
    float* oj = reinterpret_cast<float*>(smem) + wid * 32 * D;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      __syncthreads();
      if (grp == 1) {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int db = 0; db < DB; ++db) *reinterpret_cast<f32x4*>(oj + ((kb * DB + db) * 64 + lane) * 4) = w ? dv[db][kb] : dk[db][kb];
      }
      __syncthreads();
      if (grp == 0) {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int db = 0; db < DB; ++db) {
            const f32x4 x = *reinterpret_cast<const f32x4*>(oj + ((kb * DB + db) * 64 + lane) * 4);
            if (w) dv[db][kb] += x; else dk[db][kb] += x;
          }
      }
    }
    if (grp == 1) return;
  }
#pragma unroll
  for (int kb = 0; kb < 2; ++kb) {
    const int k = opaque(k0 + kb * 16 + fr);             // (the rows' addresses are not for the loop to keep)
    if (a.ksplits > 1) {                                 // [split][2][row][D], joined by dkdv_join_kernel
      if (k >= a.Sk) continue;
      const long long rows = (long long)a.B * a.nkv * a.Sk, row = (long long)bk * a.Sk + k;
      float* kpart = a.part + ((long long)split * 2 * rows + row) * D;
#pragma unroll
      for (int db = 0; db < DB; ++db) {
        *reinterpret_cast<f32x4*>(kpart + db * 16 + g * 4) = dk[db][kb];
        *reinterpret_cast<f32x4*>(kpart + rows * D + db * 16 + g * 4) = dv[db][kb];
      }
    } else {
      T* krow = (T*)a.dk.p + b * a.dk.sb + (long long)k * a.dk.ss + kvh * a.dk.sh;
      T* vrow = (T*)a.dv.p + b * a.dv.sb + (long long)k * a.dv.ss + kvh * a.dv.sh;
      const int hd = k < a.Sk ? a.hd : 0;
#pragma unroll
      for (int p = 0; p < DB / 2; ++p) {
        store_pair(krow, p, g, hd, dk[2 * p][kb] * a.scale, dk[2 * p + 1][kb] * a.scale);
        store_pair(vrow, p, g, hd, dv[2 * p][kb], dv[2 * p + 1][kb]);
      }
    }
  }
}

// dk, dv of one key of one key head: the sums over the splits of its query heads. D / 4 lanes a row.
template <typename T, int D>
__global__ __launch_bounds__(256) void dkdv_join_kernel(Args a) {
  constexpr int L = D / 4;
  const long long rows = (long long)a.B * a.nkv * a.Sk, i = (long long)blockIdx.x * 256 + threadIdx.x, row = i / L;
  const int d = (int)(i - row * L) * 4;
  if (row >= rows || d >= a.hd) return;
  const long long bk = row / a.Sk;
  const int b = (int)(bk / a.nkv), kvh = (int)(bk - (long long)b * a.nkv), k = (int)(row - bk * a.Sk);
  f32x4 dk = {0.f, 0.f, 0.f, 0.f}, dv = dk;
  for (int s = 0; s < a.ksplits; ++s) {
    const float* p = a.part + ((long long)s * 2 * rows + row) * D + d;
    dk += *reinterpret_cast<const f32x4*>(p);
    dv += *reinterpret_cast<const f32x4*>(p + rows * D);
  }
  store4((T*)a.dk.p + b * a.dk.sb + (long long)k * a.dk.ss + kvh * a.dk.sh + d, dk * a.scale);
  store4((T*)a.dv.p + b * a.dv.sb + (long long)k * a.dv.ss + kvh * a.dv.sh + d, dv);
}

// ---- host -----------------------------------------------------------------------------------------------------------
// bytes of two double-buffered tile images, and of a band
template <typename T, int D> constexpr int lds_tiles() { return 4 * key_tile<T>() * row_stride<T, D>(); }
inline int band_floats(const Args& a) { return a.table ? a.max_dist + a.right + 1 + 2 * kMargin : 0; }
template <typename K>
inline int set_lds(K kernel, int bytes) {
  if (bytes <= 64 * 1024) return 0;
  return (int)hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
}
template <typename K>
inline int launch(K kernel, long long blocks, int threads, int lds, const Args& a, hipStream_t stream) {
  const int rc = set_lds(kernel, lds);
  if (rc) return rc;
  hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3((unsigned)threads), (size_t)lds, stream, a);
  return (int)hipGetLastError();
}

// Key splits of the few-queries path: two workgroups a CU, and at least two key tiles for each of a workgroup's waves
// (fewer and the joining costs more than the splitting gains; 8 sequences x 4001 keys, 16 heads on 4 of 128: 12 + 4 us
// against 100 unsplit). 1: no second kernel.
// Which calls: up to 32 rows (queries x heads of a group), as many as few_kernel's tile holds. The other kernels do not split
// the keys, so over a long cache they leave most CUs without work; both sides of the border, us, heads of 128, 16 on 4, causal:
// 1 x 8 on 20000 (32 rows) 13 + 6, 1 x 9 279, 1 x 128 287; 8 x 8 on 4001 18 + 4, 8 x 9 62, 8 x 128 69.
inline bool few_queries(int Sq, int nh, int nkv) { return (long long)Sq * (nh / nkv) <= kFewRows; }
inline int few_splits(int B, int Sk, int nkv) {
  const long long groups = (long long)B * nkv, most = (Sk + 8 * kFewKeys - 1) / (8 * kFewKeys);
  long long n = (512 + groups - 1) / groups;
  n = n < most ? n : most;
  return (int)(n < 1 ? 1 : n > 64 ? 64 : n);
}
template <typename T, int D, int QB, int MODE>
int run_few(const Args& a, hipStream_t stream) {
  constexpr int img = kFewKeys * row_stride<T, D>(), join = QB * 16 * (D + 4) * 4;
  const int lds = 4 * (img > join ? img : join) + 4 * (8 * QB * 16 + (a.table ? a.nh / a.nkv * a.buckets : 0));
  const int rc = launch(few_kernel<T, D, QB, MODE>, (long long)a.B * a.nkv * a.splits, 256, lds, a, stream);
  if (rc || a.splits == 1) return rc;
  hipLaunchKernelGGL((few_join_kernel<T, D, MODE>), dim3((unsigned)(a.B * a.nh * a.Sq)), dim3(256), 0, stream, a);
  return (int)hipGetLastError();
}
// Splits of the dK / dV kernel over the query heads of a key head, so that about three workgroups come to a CU (4 x 2048
// causal, 16 heads on 4 of 128, with the joining: 4 splits 180 + 24 us, 2 splits 225 + 14).
inline int dkdv_splits(int B, int Sk, int nh, int nkv) {
  const long long n = (long long)B * nkv * ((Sk + kRows - 1) / kRows), group = nh / nkv;
  for (long long s = 1; s < group; ++s)
    if (group % s == 0 && n * s >= 768) return (int)s;
  return (int)group;
}

// Workgroups of eight waves instead of four, whose two halves walk every other tile: for grids that leave the CUs with too
// few waves to hide a tile's chain of products and exponentials. Otherwise the smaller ones fill the CUs better. Kernel
// times in us in bf16, one / two halves, forward, dQ, dK / dV, heads of 64 if not said:
//   at most a workgroup a CU: 4 x 512 x 12 heads 13.6 / 13.1, 15.7 / 15.4, 17.4 / 14.4; 2048 x 16 of 128 52 / 44, 67 / 56,
//     111 / 100; more of them: 10 x 512 x 12 18 / 19, 21 / 28, 25 / 27, 16 x 512 x 12 26 / 28, 31 / 43, 35 / 44, 8 x 1000 keys
//     x 10 of 80 (640 workgroups) dK / dV 39 / 47, 4 x 2048 causal x 16 of 128 94 / 103, 126 / 144, 184 / 248
//   long rows, heads up to 64: 4096 x 16 95 / 86, 101 / 106, 133 / 134, causal 8192 x 8 148 / 113, 151 / 148, 199 / 187,
//     x 12 209 / 181, 213 / 201, 279 / 255, 2 x 8192 x 8 215 / 198, 218 / 249, 281 / 317
inline bool two_groups(long long blocks, int tiles, int D, bool backward, bool causal) {
  if (tiles < 4 || blocks <= 256) return tiles >= 4;
  return D <= 64 && tiles >= 32 && (backward ? causal && blocks <= 768 : blocks <= 1024);
}

template <typename T, int D, int MODE, int GROUPS, int PARTS>
int run_fwd_as(const Args& a, long long n, hipStream_t stream) {
  const int lds = GROUPS * (lds_tiles<T, D>() + 8 * key_tile<T>()) + 4 * (GROUPS > 1 && band_floats(a) < 1024 ? 1024 : band_floats(a));
  return launch(fwd_kernel<T, D, MODE, GROUPS, PARTS>, n, 256 * GROUPS, lds, a, stream);
}
template <typename T, int D, int MODE>
int run_fwd(const Args& a, hipStream_t stream) {
  if (few_queries(a.Sq, a.nh, a.nkv))
    return a.Sq * (a.nh / a.nkv) <= 16 ? run_few<T, D, 1, MODE>(a, stream) : run_few<T, D, 2, MODE>(a, stream);
  const long long n = (long long)a.B * a.nh * ((a.Sq + kRows - 1) / kRows);
  const bool two = two_groups(n, a.Sk / key_tile<T>(), D, false, a.causal);
  if constexpr (two_parts<T, MODE>())
    if (a.table && a.fine) return two ? run_fwd_as<T, D, MODE, 2, 2>(a, n, stream) : run_fwd_as<T, D, MODE, 1, 2>(a, n, stream);
  return two ? run_fwd_as<T, D, MODE, 2, 1>(a, n, stream) : run_fwd_as<T, D, MODE, 1, 1>(a, n, stream);
}
template <typename T, int D, int MODE, int GROUPS>
int run_dq(const Args& a, long long n, hipStream_t stream) {
  const int band = band_floats(a);
  const int lds = GROUPS * (lds_tiles<T, D>() + 8 * key_tile<T>()) + 4 * (band + (a.dtab ? 4 * GROUPS * (band + 2) : 0));
  return launch(bwd_dq_kernel<T, D, MODE, GROUPS>, n, 256 * GROUPS, lds, a, stream);
}
template <typename T, int D, int MODE, int GROUPS>
int run_dkdv(const Args& a, long long n, hipStream_t stream) {
  const int lds = GROUPS * (lds_tiles<T, D>() + 8 * kRowStats) + 4 * band_floats(a);
  return launch(bwd_dkdv_kernel<T, D, MODE, GROUPS>, n, 256 * GROUPS, lds, a, stream);
}
constexpr int kMaxLds = 160 * 1024;
template <typename T, int D, int MODE>
int run_bwd(const Args& a, hipStream_t stream) {
  const int nqt = (a.Sq + kRows - 1) / kRows, nkt = (a.Sk + kRows - 1) / kRows, kt = key_tile<T>();
  const long long nq = (long long)a.B * a.nh * nqt, nk = (long long)a.B * a.nkv * nkt * a.ksplits;
  // (a long band of sums for each of eight waves may not fit)
  const bool fits = 2 * (lds_tiles<T, D>() + 8 * kt) + 4 * (9 * band_floats(a) + 16) <= kMaxLds;
  int rc = two_groups(nq, a.Sk / kt, D, true, a.causal) && fits ? run_dq<T, D, MODE, 2>(a, nq, stream) : run_dq<T, D, MODE, 1>(a, nq, stream);
  if (rc) return rc;
  rc = two_groups(nk, a.Sq / kt, D, true, a.causal) ? run_dkdv<T, D, MODE, 2>(a, nk, stream) : run_dkdv<T, D, MODE, 1>(a, nk, stream);
  if (rc || a.ksplits == 1) return rc;
  const long long n = (long long)a.B * a.nkv * a.Sk * (D / 4);
  hipLaunchKernelGGL((dkdv_join_kernel<T, D>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, stream, a);
  return (int)hipGetLastError();
}
template <typename T, int MODE>
int by_head_size(const Args& a, bool backward, hipStream_t s) {
  if (a.bytes != sizeof(Args)) return -6;                // an object file of another state of this header
  if (a.hd <= 32) return backward ? run_bwd<T, 32, MODE>(a, s) : run_fwd<T, 32, MODE>(a, s);
  if (a.hd <= 64) return backward ? run_bwd<T, 64, MODE>(a, s) : run_fwd<T, 64, MODE>(a, s);
  if (a.hd <= 96) return backward ? run_bwd<T, 96, MODE>(a, s) : run_fwd<T, 96, MODE>(a, s);
  return backward ? run_bwd<T, 128, MODE>(a, s) : run_fwd<T, 128, MODE>(a, s);
}

// one instance of the kernels a source file: (type, mode)
typedef int (*Run)(const Args& a, bool backward, hipStream_t s);
int run_bf16_plain(const Args& a, bool backward, hipStream_t s);
int run_bf16_rel(const Args& a, bool backward, hipStream_t s);
int run_bf16_keys(const Args& a, bool backward, hipStream_t s);
int run_f32_plain(const Args& a, bool backward, hipStream_t s);
int run_f32_rel(const Args& a, bool backward, hipStream_t s);
int run_f32_keys(const Args& a, bool backward, hipStream_t s);

}  // namespace attn
}  // namespace dtf

// The kernels of one (type, mode), named one by one: left to the launches in by_head_size, the host pass drops some.
#define DTF_ATTN_KERNELS(T, D, M)                            \
  template __global__ void fwd_kernel<T, D, M, 1, 1>(Args);   \
  template __global__ void fwd_kernel<T, D, M, 2, 1>(Args);   \
  template __global__ void bwd_dq_kernel<T, D, M, 1>(Args);   \
  template __global__ void bwd_dq_kernel<T, D, M, 2>(Args);   \
  template __global__ void bwd_dkdv_kernel<T, D, M, 1>(Args); \
  template __global__ void bwd_dkdv_kernel<T, D, M, 2>(Args);
#define DTF_ATTN_KERNELS_2(D, M)                                         \
  template __global__ void fwd_kernel<unsigned short, D, M, 1, 2>(Args); \
  template __global__ void fwd_kernel<unsigned short, D, M, 2, 2>(Args);
#define DTF_ATTN_TWO_PARTS(M)  \
  namespace dtf {              \
  namespace attn {             \
  DTF_ATTN_KERNELS_2(32, M)    \
  DTF_ATTN_KERNELS_2(64, M)    \
  DTF_ATTN_KERNELS_2(96, M)    \
  DTF_ATTN_KERNELS_2(128, M)   \
  }                            \
  }
#define DTF_ATTN_INSTANCE(NAME, T, M)                                                   \
  namespace dtf {                                                                       \
  namespace attn {                                                                      \
  DTF_ATTN_KERNELS(T, 32, M)                                                            \
  DTF_ATTN_KERNELS(T, 64, M)                                                            \
  DTF_ATTN_KERNELS(T, 96, M)                                                            \
  DTF_ATTN_KERNELS(T, 128, M)                                                           \
  int NAME(const Args& a, bool backward, hipStream_t s) { return by_head_size<T, M>(a, backward, s); } \
  }                                                                                     \
  }
