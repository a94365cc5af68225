// Shared declarations of the context attention kernels: attention of query tokens to states of another length
// (an encoder's text / audio / image states, a cached clip), with per-sample lengths, packed samples, key masks and
// grouped heads. context_attn_tc.cu has the tensor-memory kernel for full query tiles, context_attn_rows.cu the kernel
// for a few query rows and the join of partial results, context_attn_short.cu the one for very short states;
// context_attn_host.cu picks between them.
#pragma once
#include "tfb_api.h"
#include "tfb_common.cuh"
#include "tfb_host.h"

namespace tfb {

struct CtxParams {
  const void *q, *k, *v, *kp, *vp;
  long q_bs, q_ss, q_hs, k_bs, k_ss, k_hs, v_bs, v_ss, v_hs;  // element strides of batch, token, head
  long kp_ss, kp_hs, vp_ss, vp_hs;                             // the shared prefix has one batch entry
  void* out;        // [B, Sq, H, D] contiguous
  float* lse;       // [B, H, Sq] or null
  float* part_o;    // non-null: results go to slots [slot][B * Sq][H][D] (each slot normalised by its own sum) ...
  float* part_lse;  // ... with base-2 log-sum-exps [slot][B * Sq][H]; a slot that saw no key holds -inf and zeros
  const int* kv_lens;
  const int* cu_kv;
  const uint8_t* key_mask;
  long mask_bs;
  int B, Sq, H, Hkv, D, Skv, P;  // Skv: rows of k / v per sample (all rows when packed); P: rows of the prefix
  int ns, slot0;                 // key range split over ns slots, the first of them slot0
  float scale_log2;
  int* status;
};

// Rows [first, first + len) of the sample's own keys. Lengths and offsets come from device memory, so they are clamped
// here: no value of theirs can lead outside the tensors.
__device__ __forceinline__ void ctx_sample_range(const CtxParams& p, int b, int& first, int& len) {
  if (p.cu_kv) {
    const int a = __ldg(p.cu_kv + b), e = __ldg(p.cu_kv + b + 1);
    first = min(max(a, 0), p.Skv);
    len = max(min(e, p.Skv) - first, 0);
  } else {
    first = 0;
    len = p.kv_lens ? min(max(__ldg(p.kv_lens + b), 0), p.Skv) : p.Skv;
  }
}

// What exp2 takes off the scores of a row with the largest score m: m itself, but nothing where m is infinite. Without a key
// (m = -inf) every weight is then 0; with a score of +inf that one weighs +inf, and so does the sum, while a sum with a NaN
// score in it is NaN (the maximum passes NaN over). So the sum says all there is to know: 0 where nothing was seen, +inf or
// NaN where the log-sum-exp is the same and the row NaN, as in a plain evaluation.
__device__ __forceinline__ float ctx_exp_base(float m) { return fabsf(m) == INFINITY ? 0.f : m; }
// Factor on what was summed under the maximum m once it is m_new; 1 for an infinity that stays.
__device__ __forceinline__ float ctx_rescale(float m, float m_new) { return m == m_new ? 1.f : fast_exp2(m - m_new); }
// 1 / sum, 0 for a row that saw nothing. NaN and +inf (whose row is made of infinities and NaN) lead to NaN.
__device__ __forceinline__ float ctx_inverse(float sum) { return sum == 0.f ? 0.f : 1.f / sum; }
__device__ __forceinline__ float ctx_lse2(float m, float sum) { return sum == 0.f ? -INFINITY : m + log2f(sum); }

template <bool FP16>
__device__ __forceinline__ uint32_t ctx_pack2(float lo, float hi) {
  return FP16 ? pack_f16x2(lo, hi) : pack_bf16x2(lo, hi);
}

// [batch][token][head][channel] tensor map; a dimension of one entry may have any stride (TMA wants multiples of 16).
inline int ctx_tmap(CUtensorMap* m, const void* base, int fp16, int D, int heads, long hs, long rows, long ss, int B, long bs,
                    uint32_t box_c, uint32_t box_h, uint32_t box_s, int swizzle) {
  uint64_t dims[4] = {static_cast<uint64_t>(D), static_cast<uint64_t>(heads), static_cast<uint64_t>(rows),
                      static_cast<uint64_t>(B)};
  uint64_t str[3] = {static_cast<uint64_t>(heads > 1 ? hs : 8) * 2, static_cast<uint64_t>(rows > 1 ? ss : 8) * 2,
                     static_cast<uint64_t>(B > 1 ? bs : 8) * 2};
  uint32_t box[4] = {box_c, box_h, box_s, 1};
  return make_tmap(m, base, fp16 ? TM_F16 : TM_BF16, 4, dims, str, box, swizzle);
}

// Few query rows (Sq * H / Hkv <= CTX_FEW_ROWS) of every sample against the prefix and its own keys.
constexpr int CTX_FEW_ROWS = 32;
int launch_ctx_rows(const CtxParams& p, int fp16, cudaStream_t st);
// Many query rows against at most CTX_SHORT_KEYS rows of k / v (p.Skv, packed samples together); writes final results only.
constexpr int CTX_SHORT_KEYS = 64;
int launch_ctx_short(const CtxParams& p, int fp16, cudaStream_t st);
// Joins p.ns slots of part_o / part_lse (slot0 = 0) into out and lse.
int launch_ctx_join(const CtxParams& p, int fp16, cudaStream_t st);
// Full query tiles against the prefix and the sample's own keys.
int launch_ctx_tc(const CtxParams& p, int fp16, cudaStream_t st);
// Work items of launch_ctx_tc with p.ns = 1.
long ctx_tc_items(int B, int Sq, int H, int Hkv);

}  // namespace tfb
