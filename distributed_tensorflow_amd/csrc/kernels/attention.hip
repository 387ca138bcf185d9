// C entry points of the general attention kernels (attention.h), and the last step of the relative bias's gradient.
//
// A call is described by an array of 64-bit words (pointers, element strides, sizes): see the enum. Every entry checks
// what the kernels assume and returns a negative code without launching anything when it does not hold.
#include "attention.h"

#include <cmath>

using namespace dtf;

namespace {

enum Word {
  kTensors = 0,          // q k v out dout dq dk dv: pointer and (batch, token, head) strides in elements, four words each
  kKeyBias = 32, kLens, kQStart, kQStart0, kTable, kTableBf16, kBuckets, kMaxDist, kBidirectional,
  kStat, kRowTiles, kDtabParts, kDtabOut, kB, kSq, kSk, kNh, kNkv, kHd, kCausal, kBf16, kPart, kFine, kThr   // then the bucket borders
};

bool unpack(const long long* w, int n_words, float scale, attn::Args& a) {
  if (n_words < kThr) return false;
  a.bytes = sizeof(attn::Args);
  attn::Strided* t[8] = {&a.q, &a.k, &a.v, &a.out, &a.dout, &a.dq, &a.dk, &a.dv};
  for (int i = 0; i < 8; ++i) {
    t[i]->p = (void*)w[kTensors + 4 * i];
    t[i]->sb = w[kTensors + 4 * i + 1];
    t[i]->ss = w[kTensors + 4 * i + 2];
    t[i]->sh = w[kTensors + 4 * i + 3];
  }
  a.key_bias = (const float*)w[kKeyBias];
  a.lens = (const int*)w[kLens];
  a.q_start = (const int*)w[kQStart];
  a.q_start0 = (int)w[kQStart0];
  a.table = (const void*)w[kTable];
  a.table_bf16 = (int)w[kTableBf16];
  a.buckets = (int)w[kBuckets];
  a.max_dist = (int)w[kMaxDist];
  a.right = w[kBidirectional] ? a.max_dist : 0;
  a.half = w[kBidirectional] ? a.buckets / 2 : a.buckets;
  a.exact = a.half / 2;
  a.stat = (float*)w[kStat];
  a.rows = (float*)w[kRowTiles];
  a.dtab = (float*)w[kDtabParts];
  const long long lim = 1LL << 30;
  for (int i = kB; i <= kHd; ++i)
    if (w[i] <= 0 || w[i] > lim) return false;
  if (w[kQStart0] > lim || w[kQStart0] < -lim) return false;
  a.B = (int)w[kB]; a.Sq = (int)w[kSq]; a.Sk = (int)w[kSk]; a.nh = (int)w[kNh]; a.nkv = (int)w[kNkv]; a.hd = (int)w[kHd];
  a.causal = (int)w[kCausal];
  a.part = (float*)w[kPart];
  a.fine = (unsigned char*)w[kFine];
  a.scale = a.score_scale = scale;
  a.unit = 1.f;
  if (a.key_bias && scale < 1.f) {                       // score_scale in [1, 2)
    int e = 0;
    a.score_scale = 2.f * std::frexp(scale, &e);
    a.unit = std::ldexp(1.f, e - 1);
  }
  a.step = 1.f / a.score_scale;
  if (!(scale > 0.f) || scale > 1e30f || a.hd % 8 || a.hd > 128 || a.nh % a.nkv) return false;
  if (a.table) {
    a.n_thr = a.half - a.exact - 1;
    if (a.exact < 1 || a.buckets > 128 || a.max_dist <= a.exact || a.max_dist > 2048 || a.n_thr >= attn::kMaxThr || a.n_thr < 0)
      return false;
  }
  // no word missing and none too many: a caller with another order of words is refused, whatever it takes a word for
  if (n_words != kThr + a.n_thr) return false;
  for (int i = 0; i < a.n_thr; ++i) a.thr[i] = (int)w[kThr + i];
  return true;
}

// What the kernels read or write through: 16-byte alignment, token strides that hold a row and keep a tile's offsets in
// 31 bits.
bool operands_ok(const attn::Args& a, int size, bool backward) {
  const attn::Strided* t[8] = {&a.q, &a.k, &a.v, &a.out, &a.dout, &a.dq, &a.dk, &a.dv};
  const int per16 = 16 / size;
  for (int i = 0; i < (backward ? 8 : 4); ++i) {
    if (!t[i]->p || (reinterpret_cast<uintptr_t>(t[i]->p) & 15)) return false;
    if (t[i]->sb % per16 || t[i]->ss % per16 || t[i]->sh % per16) return false;
    if (t[i]->sb < 0 || t[i]->sh < 0 || t[i]->ss < a.hd || t[i]->ss > (1 << 22)) return false;
  }
  if (reinterpret_cast<uintptr_t>(a.fine) & 7 || (backward && size == 2 && !a.fine)) return false;
  return !backward || (a.stat && a.rows && !(reinterpret_cast<uintptr_t>(a.rows) & 15));
}

attn::Run instance(const attn::Args& a, bool bf16) {
  if (a.key_bias) return bf16 ? attn::run_bf16_keys : attn::run_f32_keys;
  if (a.table) return bf16 ? attn::run_bf16_rel : attn::run_f32_rel;
  return bf16 ? attn::run_bf16_plain : attn::run_f32_plain;
}

// Grids of the kernels that the call launches: fewer than 2^32 threads, at most 512 a workgroup. (Where keys or heads are
// split, there are fewer than 768 workgroups without the splits: those grids and the joins' stay far below.)
bool grid_ok(const attn::Args& a, bool backward) {
  const long long most = 1LL << 23;
  if (backward && (long long)a.B * a.nkv * ((a.Sk + attn::kRows - 1) / attn::kRows) >= most) return false;
  if (!backward && attn::few_queries(a.Sq, a.nh, a.nkv)) return (long long)a.B * a.nkv < most;
  return (long long)a.B * a.nh * ((a.Sq + attn::kRows - 1) / attn::kRows) < most;
}

// dtable[u, h] = sum over the parts, in a fixed order: one workgroup a head, its threads split the parts.
__global__ __launch_bounds__(256) void dtab_finish_kernel(const float* __restrict__ parts, void* __restrict__ out,
                                                         int n_parts, int nh, int buckets, int bf16) {
  __shared__ float red[256];
  const int h = blockIdx.x, slices = 256 / buckets, u = threadIdx.x % buckets, s = threadIdx.x / buckets;
  float v = 0.f;
  if (s < slices) {
#pragma unroll 8
    for (int p = s; p < n_parts; p += slices) v += parts[((long long)p * nh + h) * buckets + u];
  }
  red[threadIdx.x] = v;
  __syncthreads();
  if (s == 0) {
    for (int i = 1; i < slices; ++i) v += red[i * buckets + u];
    const long long at = (long long)u * nh + h;
    if (bf16) ((unsigned short*)out)[at] = f32_to_bf16(v);
    else ((float*)out)[at] = v;
  }
}

}  // namespace

// Splits of the backward pass over the query heads of a key head. More than one: it needs a scratch of splits * 2 * B *
// nkv * Sk * (hd rounded up to 32) floats.
DTF_API int dtf_attention_bwd_splits(int B, int Sk, int nh, int nkv) { return nkv > 0 ? attn::dkdv_splits(B, Sk, nh, nkv) : 1; }

// Key splits of the forward pass. More than one: it needs a scratch of splits * B * nh * Sq * (hd rounded up to 32, + 2)
// floats.
DTF_API int dtf_attention_splits(int B, int Sq, int Sk, int nh, int nkv) {
  return B > 0 && nkv > 0 && attn::few_queries(Sq, nh, nkv) ? attn::few_splits(B, Sk, nkv) : 1;
}

DTF_API int dtf_attention_fwd(const long long* words, int n_words, float scale, hipStream_t stream) {
  attn::Args a = {};
  if (!unpack(words, n_words, scale, a)) return -1;
  const bool bf16 = words[kBf16];
  if (!operands_ok(a, bf16 ? 2 : 4, false)) return -2;
  if (!grid_ok(a, false)) return -3;
  a.splits = dtf_attention_splits(a.B, a.Sq, a.Sk, a.nh, a.nkv);
  if (a.splits > 1 && !a.part) return -5;
  return instance(a, bf16)(a, false, stream);
}

// row tiles: fp32 scratch of B * nh * ceil(Sq / 128) * 512. dtab parts: fp32 [B * ceil(Sq / 128)][nh][buckets] scratch; dtab out: [buckets, nh] in the table's type. Both or neither.
DTF_API int dtf_attention_bwd(const long long* words, int n_words, float scale, hipStream_t stream) {
  attn::Args a = {};
  if (!unpack(words, n_words, scale, a)) return -1;
  const bool bf16 = words[kBf16];
  if (!operands_ok(a, bf16 ? 2 : 4, true)) return -2;
  if (!grid_ok(a, true)) return -3;
  void* out = (void*)words[kDtabOut];
  if ((a.dtab != nullptr) != (out != nullptr) || (out && !a.table)) return -4;
  a.ksplits = dtf_attention_bwd_splits(a.B, a.Sk, a.nh, a.nkv);
  if (a.ksplits > 1 && !a.part) return -5;
  const int rc = instance(a, bf16)(a, true, stream);
  if (rc || !a.dtab) return rc;
  hipLaunchKernelGGL(dtab_finish_kernel, dim3(a.nh), dim3(256), 0, stream, a.dtab, out,
                     a.B * ((a.Sq + attn::kRows - 1) / attn::kRows), a.nh, a.buckets, a.table_bf16);
  return (int)hipGetLastError();
}
