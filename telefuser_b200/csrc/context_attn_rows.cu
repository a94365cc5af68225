// Context attention for a few query rows (single tokens, a handful of summary tokens): memory bound, every key and
// value row is read once per (sample, key head).
//
// One CTA of four warps owns the <= 32 query rows of one (sample, key head) - tokens x grouped heads - and one slice of the
// keys. Its warps work for themselves, 16 keys at a time: a warp has a ring of TMA boxes in shared memory (K and V of 16 keys
// each), its own running maximum, sum and fp32 accumulator, and refills a slot as soon as it has read it; the four results
// are joined once at the end. So bytes in flight cost no registers: two CTAs per SM hold 192 KB of the stream, and no
// warp waits for another. (Three with two thirds of the ring each: 187 for 154 us on 64 streams x 8 key heads x 4096 keys, whose 512
// CTAs then leave a second wave of 68.) The products run on mma.sync m16n8k16, fed by ldmatrix: with so few rows the tensor work is a
// fraction of what the loads take.
// Keys that the length or the mask hides: their scores are replaced by -inf and their V fragments by zeros, so infinities
// and NaN there never meet a product.
//
// Bound by HBM where the batch fills the device: 64 x 8 key heads x 4096 keys 154 us, 7.0 TB/s, above what a copy reaches (there
// are hardly any writes); 5 tokens x 32 / 8 heads against 131072 keys 94 us, 5.7 TB/s. By launch and load latency below that:
// 8 x 16 heads against up to 512 keys 7.7 us.
#include <string.h>

#include "context_attn.cuh"

namespace tfb {

constexpr int CR_WARPS = 4;

struct CtxRowsParams {
  CtxParams c;
  int bmul;      // 0: packed samples, the tensors have one batch entry
  int n_prefix;  // 16-key chunks of the shared prefix, in front of the sample's own
};

template <bool FP16>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (FP16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
// Byte offset of the 16-byte piece `piece` of row `row` in boxes of [16 rows][64 channels], 128B swizzle, 2 KB each.
__device__ __forceinline__ uint32_t box_at(int row, int piece) {
  return (piece >> 3) * 2048 + row * 128 + (((piece & 7) ^ (row & 7)) << 4);
}

template <int DK, int MT>
struct CtxRowsCfg {
  static constexpr int CHUNK = 2 * 16 * DK * 2;             // K and V of 16 keys
  static constexpr int CTAS = 2;                            // per SM
  static constexpr int STAGES = 24576 / CHUNK;              // per warp
  static constexpr int RING = CR_WARPS * STAGES * CHUNK;    // the join at the end lies over it
  static constexpr int Q_OFF = RING;                        // MT x 16 rows as boxes
  static constexpr int ML_OFF = Q_OFF + MT * 16 * DK * 2;   // [warps][MT * 16] of (maximum, sum)
  static constexpr int BAR_OFF = ML_OFF + CR_WARPS * MT * 16 * 8;
  static constexpr int SMEM = BAR_OFF + CR_WARPS * STAGES * 8 + 16 + 1024;
  static_assert(CR_WARPS * MT * 16 * DK * 4 <= RING, "the join fits over the ring");
  static_assert(CTAS * (SMEM + 1024) <= 228 * 1024, "CTAs per SM");
};

template <bool FP16, int DK, int MT>
__global__ void __launch_bounds__(CR_WARPS * 32, CtxRowsCfg<DK, MT>::CTAS)
    ctx_rows_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                    const __grid_constant__ CUtensorMap tmKp, const __grid_constant__ CUtensorMap tmVp,
                    const __grid_constant__ CtxRowsParams rp) {
  using Cfg = CtxRowsCfg<DK, MT>;
  constexpr int NBOX = DK / 64, ROWS = MT * 16;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const CtxParams& p = rp.c;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Cfg::BAR_OFF);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bars + CR_WARPS * Cfg::STAGES);
  const AbortCtx ctx{abort_flag, p.status};
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int c = lane & 3;
  const int G = p.H / p.Hkv, R = p.Sq * G;
  const int split = blockIdx.x % p.ns;
  const int hk = (blockIdx.x / p.ns) % p.Hkv;
  const int b = blockIdx.x / p.ns / p.Hkv;
  int first, len;
  ctx_sample_range(p, b, first, len);
  const long n16 = rp.n_prefix + ((len + 15) >> 4);
  const int i0 = static_cast<int>(n16 * split / p.ns), i1 = static_cast<int>(n16 * (split + 1) / p.ns);

  uint64_t* full = bars + warp * Cfg::STAGES;
  uint8_t* ring = smem + warp * Cfg::STAGES * Cfg::CHUNK;
  // one lane: K and V of the 16 keys of chunk `it`
  auto fetch = [&](int it, int slot) {
    uint8_t* dst = ring + slot * Cfg::CHUNK;
    mbar_expect_tx(&full[slot], Cfg::CHUNK);
    const bool pre = it < rp.n_prefix;
    const int row = pre ? it * 16 : first + (it - rp.n_prefix) * 16, bb = pre ? 0 : b * rp.bmul;
#pragma unroll
    for (int x = 0; x < NBOX; ++x) {
      tma_load_4d(dst + x * 2048, pre ? &tmKp : &tmK, &full[slot], x * 64, hk, row, bb);
      tma_load_4d(dst + (NBOX + x) * 2048, pre ? &tmVp : &tmV, &full[slot], x * 64, hk, row, bb);
    }
  };
  if (lane == 0) {
    for (int s = 0; s < Cfg::STAGES; ++s) mbar_init(&full[s], 1);
    mbar_fence_init();
    for (int s = 0; s < Cfg::STAGES; ++s) {
      const int it = i0 + warp + s * CR_WARPS;
      if (it < i1) fetch(it, s);
    }
    if (warp == 0) *abort_flag = 0;
  }
  // Q rows (token, head) as boxes, zeros behind the last
  for (int x = threadIdx.x; x < ROWS * DK / 8; x += CR_WARPS * 32) {
    const int row = x / (DK / 8), piece = x % (DK / 8);
    uint4 v = make_uint4(0, 0, 0, 0);
    if (row < R && piece * 8 < p.D)
      v = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.q) + static_cast<long>(b) * p.q_bs +
                                               (row / G) * p.q_ss + static_cast<long>(hk * G + row % G) * p.q_hs + piece * 8));
    *reinterpret_cast<uint4*>(smem + Cfg::Q_OFF + (row >> 4) * (16 * DK * 2) + box_at(row & 15, piece)) = v;
  }
  __syncthreads();

  float o[MT][DK / 8][4];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int t = 0; t < DK / 8; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[mt][t][e] = 0.f;
  float m[MT][2], l[MT][2];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) m[mt][0] = m[mt][1] = -INFINITY, l[mt][0] = l[mt][1] = 0.f;

  const uint8_t* mb = p.key_mask ? p.key_mask + static_cast<long>(b) * p.mask_bs : nullptr;
  const uint32_t q_at = smem_u32(smem + Cfg::Q_OFF);
  // ldmatrix rows of this lane: A fragments and V take rows 0..15 by halves of a k-step, K takes the two key octets
  const int a_row = lane & 15, a_half = lane >> 4;
  const int k_row = (lane & 7) + ((lane >> 4) << 3), k_half = (lane >> 3) & 1;
  int slot = 0;
  uint32_t phase = 0;
  for (int it = i0 + warp; it < i1; it += CR_WARPS) {
    // keys of this lane's score columns: 2c, 2c + 1, 2c + 8, 2c + 9 of the chunk
    const bool pre = it < rp.n_prefix;
    const int keys = pre ? p.P : len;
    bool vis[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int j = (pre ? it : it - rp.n_prefix) * 16 + 2 * c + (e & 1) + (e >> 1) * 8;
      vis[e] = j < keys && (!mb || mb[j]);
    }
    // after an expired wait (recorded in the status word) the warp goes on with what is there, to the common end
    mbar_wait_warp(&full[slot], phase, ctx, 80);
    const uint32_t k_at = smem_u32(ring + slot * Cfg::CHUNK), v_at = k_at + NBOX * 2048;
    float s[MT][2][4];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[mt][t][e] = 0.f;
#pragma unroll
    for (int kk = 0; kk < DK / 16; ++kk) {
      uint32_t kf[4];
      ldsm4(k_at + box_at(k_row, kk * 2 + k_half), kf);
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        uint32_t a[4];
        ldsm4(q_at + mt * (16 * DK * 2) + box_at(a_row, kk * 2 + a_half), a);
        mma16816<FP16>(s[mt][0], a, kf[0], kf[1]);
        mma16816<FP16>(s[mt][1], a, kf[2], kf[3]);
      }
    }
    uint32_t pf[MT][4];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float mx = -INFINITY;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float& v = s[mt][t][r * 2 + e];
            v = vis[t * 2 + e] ? v * p.scale_log2 : -INFINITY;
            mx = fmaxf(mx, v);
          }
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float m_new = fmaxf(m[mt][r], mx);
        if (__any_sync(0xffffffffu, m_new > m[mt][r])) {
          const float alpha = ctx_rescale(m[mt][r], m_new);
          l[mt][r] *= alpha;
#pragma unroll
          for (int t = 0; t < DK / 8; ++t) o[mt][t][r * 2] *= alpha, o[mt][t][r * 2 + 1] *= alpha;
          m[mt][r] = m_new;
        }
        const float base = ctx_exp_base(m[mt][r]);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const float p0 = fast_exp2(s[mt][t][r * 2] - base), p1 = fast_exp2(s[mt][t][r * 2 + 1] - base);
          l[mt][r] += p0 + p1;
          pf[mt][t * 2 + r] = ctx_pack2<FP16>(p0, p1);  // in [0, 1], rounded to the inputs' type for the product
        }
      }
    }
    const bool all = __all_sync(0xffffffffu, vis[0] && vis[1] && vis[2] && vis[3]);
    const uint32_t keep0 = (vis[0] ? 0xffffu : 0u) | (vis[1] ? 0xffff0000u : 0u);
    const uint32_t keep1 = (vis[2] ? 0xffffu : 0u) | (vis[3] ? 0xffff0000u : 0u);
#pragma unroll
    for (int t = 0; t < DK / 16; ++t) {
      uint32_t vf[4];  // keys 0..7 / 8..15 of channels 16 t .. + 7, then of the next 8
      ldsm4_t(v_at + box_at(a_row, t * 2 + a_half), vf);
      if (!all) vf[0] &= keep0, vf[1] &= keep1, vf[2] &= keep0, vf[3] &= keep1;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        mma16816<FP16>(o[mt][2 * t], pf[mt], vf[0], vf[1]);
        mma16816<FP16>(o[mt][2 * t + 1], pf[mt], vf[2], vf[3]);
      }
    }
    __syncwarp();
    if (lane == 0 && it + Cfg::STAGES * CR_WARPS < i1) fetch(it + Cfg::STAGES * CR_WARPS, slot);
    if (++slot == Cfg::STAGES) slot = 0, phase ^= 1;
  }

  // ---- join of the four warps, over the rings (every copy that was issued has been waited for) ----
  __syncthreads();
  float* s_o = reinterpret_cast<float*>(smem) + warp * ROWS * DK;
  float2* s_ml = reinterpret_cast<float2*>(smem + Cfg::ML_OFF);
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      float sum = l[mt][r];
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      const int row = mt * 16 + (lane >> 2) + r * 8;
      if (c == 0) s_ml[warp * ROWS + row] = make_float2(m[mt][r], sum);
      if (row < R)
#pragma unroll
        for (int t = 0; t < DK / 8; ++t)
          *reinterpret_cast<float2*>(s_o + row * DK + t * 8 + 2 * c) = make_float2(o[mt][t][r * 2], o[mt][t][r * 2 + 1]);
    }
  __syncthreads();
  s_o = reinterpret_cast<float*>(smem);
  const int per_row = p.D >> 2;  // float4 groups of a row
  for (int x = threadIdx.x; x < R * per_row; x += CR_WARPS * 32) {
    const int row = x / per_row, d = (x - row * per_row) * 4;
    float mm = s_ml[row].x;
#pragma unroll
    for (int w = 1; w < CR_WARPS; ++w) mm = fmaxf(mm, s_ml[w * ROWS + row].x);
    float sum = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < CR_WARPS; ++w) {
      const float2 ml = s_ml[w * ROWS + row];
      const float f = ctx_rescale(ml.x, mm);
      sum += f * ml.y;
      const float4 t = *reinterpret_cast<const float4*>(s_o + (w * ROWS + row) * DK + d);
      acc.x += f * t.x, acc.y += f * t.y, acc.z += f * t.z, acc.w += f * t.w;
    }
    const float inv = ctx_inverse(sum);
    const long token = static_cast<long>(b) * p.Sq + row / G;
    const int head = hk * G + row % G;
    const float lse2 = ctx_lse2(mm, sum);
    if (p.part_o) {
      const long at = (static_cast<long>(p.slot0 + split) * p.B * p.Sq + token) * p.H + head;
      if (d == 0) p.part_lse[at] = lse2;
      *reinterpret_cast<float4*>(p.part_o + at * p.D + d) = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
    } else {
      uint16_t* op = static_cast<uint16_t*>(p.out) + (token * p.H + head) * p.D + d;
      *reinterpret_cast<uint2*>(op) = make_uint2(ctx_pack2<FP16>(acc.x * inv, acc.y * inv), ctx_pack2<FP16>(acc.z * inv, acc.w * inv));
      if (p.lse && d == 0)
        p.lse[(static_cast<long>(b) * p.H + head) * p.Sq + row / G] = lse2 * 0.6931471805599453f;
    }
  }
}

// out = sum_s w_s o_s / sum_s w_s, w_s = 2^(lse_s - max). One CTA of four warps per (token, head): a warp adds every fourth
// slot, in an order that depends on nothing but the number of slots.
template <bool FP16>
__global__ void __launch_bounds__(128) ctx_join_kernel(const CtxParams p) {
  __shared__ float4 s_acc[4][32];
  __shared__ float s_sum[4];
  const long rows = static_cast<long>(p.B) * p.Sq * p.H;
  const long row = blockIdx.x;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float mm = -INFINITY;
  for (int s = lane; s < p.ns; s += 32) mm = fmaxf(mm, p.part_lse[s * rows + row]);
  mm = warp_max(mm);
  const float base = ctx_exp_base(mm);
  float sum = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  const int d = lane * 4;
#pragma unroll 4
  for (int s = warp; s < p.ns; s += 4) {
    const float f = fast_exp2(p.part_lse[s * rows + row] - base);  // 0 for a slot that saw no key, NaN or +inf for what came so
    float4 t = make_float4(0.f, 0.f, 0.f, 0.f);
    if (d < p.D) t = *reinterpret_cast<const float4*>(p.part_o + (s * rows + row) * p.D + d);
    sum += f;
    acc.x += f * t.x, acc.y += f * t.y, acc.z += f * t.z, acc.w += f * t.w;
  }
  s_acc[warp][lane] = acc;
  if (lane == 0) s_sum[warp] = sum;
  __syncthreads();
  if (warp) return;
#pragma unroll
  for (int w = 1; w < 4; ++w) {
    const float4 t = s_acc[w][lane];
    acc.x += t.x, acc.y += t.y, acc.z += t.z, acc.w += t.w;
    sum += s_sum[w];
  }
  const float inv = ctx_inverse(sum);
  if (d < p.D)
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + row * p.D + d) =
        make_uint2(ctx_pack2<FP16>(acc.x * inv, acc.y * inv), ctx_pack2<FP16>(acc.z * inv, acc.w * inv));
  if (p.lse && lane == 0) {
    const long token = row / p.H;
    const int h = static_cast<int>(row % p.H);
    p.lse[(token / p.Sq * p.H + h) * p.Sq + token % p.Sq] =
        ctx_lse2(mm, sum) * 0.6931471805599453f;
  }
}

template <bool FP16, int DK, int MT>
static int launch_ctx_rows_impl(const CtxParams& p, cudaStream_t st) {
  using Cfg = CtxRowsCfg<DK, MT>;
  static bool attr_set[TFB_MAX_DEVICES] = {false};
  auto kern = &ctx_rows_kernel<FP16, DK, MT>;
  if (int rc = ensure_dynamic_smem(reinterpret_cast<const void*>(kern), Cfg::SMEM, attr_set)) return rc;
  const long ctas = static_cast<long>(p.B) * p.Hkv * p.ns;
  if (ctas > 0x7fffffffL) return TFB_ERR_TOO_LARGE;
  CtxRowsParams rp;
  rp.c = p;
  rp.bmul = p.cu_kv ? 0 : 1;
  rp.n_prefix = (p.P + 15) / 16;
  CUtensorMap tk, tv, tkp, tvp;
  memset(&tk, 0, sizeof(tk));  // a map without rows is not used
  tv = tkp = tvp = tk;
  int e;
  if (p.Skv > 0) {
    const int kb = p.cu_kv ? 1 : p.B;
    if ((e = ctx_tmap(&tk, p.k, FP16, p.D, p.Hkv, p.k_hs, p.Skv, p.k_ss, kb, p.k_bs, 64, 1, 16, TM_SW_128))) return e;
    if ((e = ctx_tmap(&tv, p.v, FP16, p.D, p.Hkv, p.v_hs, p.Skv, p.v_ss, kb, p.v_bs, 64, 1, 16, TM_SW_128))) return e;
  }
  if (p.P > 0) {
    if ((e = ctx_tmap(&tkp, p.kp, FP16, p.D, p.Hkv, p.kp_hs, p.P, p.kp_ss, 1, 0, 64, 1, 16, TM_SW_128))) return e;
    if ((e = ctx_tmap(&tvp, p.vp, FP16, p.D, p.Hkv, p.vp_hs, p.P, p.vp_ss, 1, 0, 64, 1, 16, TM_SW_128))) return e;
  }
  kern<<<static_cast<int>(ctas), CR_WARPS * 32, Cfg::SMEM, st>>>(tk, tv, tkp, tvp, rp);
  return cudaGetLastError() == cudaSuccess ? TFB_OK : TFB_ERR_LAUNCH;
}

template <bool FP16>
static int launch_ctx_rows_type(const CtxParams& p, cudaStream_t st) {
  const bool one = p.Sq * (p.H / p.Hkv) <= 16;
  if (p.D <= 64) return one ? launch_ctx_rows_impl<FP16, 64, 1>(p, st) : launch_ctx_rows_impl<FP16, 64, 2>(p, st);
  return one ? launch_ctx_rows_impl<FP16, 128, 1>(p, st) : launch_ctx_rows_impl<FP16, 128, 2>(p, st);
}

int launch_ctx_rows(const CtxParams& p, int fp16, cudaStream_t st) {
  if (static_cast<long>(p.Sq) * (p.H / p.Hkv) > CTX_FEW_ROWS) return TFB_ERR_TOO_LARGE;
  return fp16 ? launch_ctx_rows_type<true>(p, st) : launch_ctx_rows_type<false>(p, st);
}

int launch_ctx_join(const CtxParams& p, int fp16, cudaStream_t st) {
  const long rows = static_cast<long>(p.B) * p.Sq * p.H;
  if (rows > 0x7fffffffL) return TFB_ERR_TOO_LARGE;
  if (fp16) ctx_join_kernel<true><<<static_cast<int>(rows), 128, 0, st>>>(p);
  else ctx_join_kernel<false><<<static_cast<int>(rows), 128, 0, st>>>(p);
  return cudaGetLastError() == cudaSuccess ? TFB_OK : TFB_ERR_LAUNCH;
}

}  // namespace tfb
