// Context attention for a few query rows (single tokens, a handful of summary tokens): memory bound, every key and
// value row is read once per (sample, key head).
//
// One CTA of four warps owns the <= 16 query rows of one (sample, key head) - tokens x grouped heads - and one slice of
// the keys; its warps take 16 keys at a time and keep their own running maximum, sum and 16 x D fp32 accumulator, joined
// once at the end through shared memory. The products run on mma.sync m16n8k16: with at most 16 rows the tensor work is
// 1/8 of what the loads take, and operands go from global memory to registers without a stop in shared memory. For
// that the fragment layouts are met by permuting the summation index instead of the data:
//   Q.K^T  lane (n = lane / 4, c = lane % 4) loads 16 bytes of key n, channels 32 i + 8 c .. + 7: two k16 steps whose
//          channel order is permuted the same way in Q and K.
//   P.V    lane loads 16 bytes (channels 64 i + 8 n .. + 7) of the keys 2c, 2c + 1, 2c + 8, 2c + 9, the keys its P fragment
//          holds; byte permutes pair two keys per register. Column n of MMA t is channel 64 i + 8 n + t.
// Rows that the lengths or the mask hide are not loaded at all: zeros take their place, so infinities and NaN there
// never meet a product, and their scores are replaced by -inf.
//
// Bound by HBM where the batch fills the device, by launch and load latency below that.
#include "context_attn.cuh"

namespace tfb {

constexpr int CR_WARPS = 4;

template <bool FP16>
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  if (FP16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint4 ctx_ld16(const uint16_t* p, bool ok) {
  uint4 r = make_uint4(0, 0, 0, 0);
  if (ok) r = __ldg(reinterpret_cast<const uint4*>(p));
  return r;
}

template <bool FP16, int DK>
__global__ void __launch_bounds__(CR_WARPS * 32) ctx_rows_kernel(const CtxParams p) {
  constexpr int NCH = DK / 32, NBLK = DK / 64;
  __shared__ float s_o[CR_WARPS][16][DK];
  __shared__ float s_m[CR_WARPS][16], s_l[CR_WARPS][16];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n = lane >> 2, c = lane & 3;
  const int G = p.H / p.Hkv, R = p.Sq * G;
  const int split = blockIdx.x % p.ns;
  const int hk = (blockIdx.x / p.ns) % p.Hkv;
  const int b = blockIdx.x / p.ns / p.Hkv;
  int first, len;
  ctx_sample_range(p, b, first, len);
  const long n16 = (len + 15) >> 4;
  const int i0 = static_cast<int>(n16 * split / p.ns), i1 = static_cast<int>(n16 * (split + 1) / p.ns);

  const uint16_t* qb = static_cast<const uint16_t*>(p.q) + static_cast<long>(b) * p.q_bs;
  const uint16_t* kb = static_cast<const uint16_t*>(p.k) + (p.cu_kv ? 0 : static_cast<long>(b) * p.k_bs) +
                       static_cast<long>(first) * p.k_ss + static_cast<long>(hk) * p.k_hs;
  const uint16_t* vb = static_cast<const uint16_t*>(p.v) + (p.cu_kv ? 0 : static_cast<long>(b) * p.v_bs) +
                       static_cast<long>(first) * p.v_ss + static_cast<long>(hk) * p.v_hs;
  const uint8_t* mb = p.key_mask ? p.key_mask + static_cast<long>(b) * p.mask_bs : nullptr;
  auto visible = [&](int j) { return j < len && (!mb || mb[j]); };

  uint4 q0[NCH], q1[NCH];
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    const int d = i * 32 + c * 8;
    const int ra = n, rb = n + 8;
    q0[i] = ctx_ld16(qb + (ra / G) * p.q_ss + static_cast<long>(hk * G + ra % G) * p.q_hs + d, ra < R && d < p.D);
    q1[i] = ctx_ld16(qb + (rb / G) * p.q_ss + static_cast<long>(hk * G + rb % G) * p.q_hs + d, rb < R && d < p.D);
  }
  float o[NBLK][8][4];
#pragma unroll
  for (int i = 0; i < NBLK; ++i)
#pragma unroll
    for (int t = 0; t < 8; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][t][e] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

  uint4 kf[2][NCH];
  auto load_k = [&](int it) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int j = it * 16 + t * 8 + n;
      const bool ok = it < i1 && visible(j);
#pragma unroll
      for (int i = 0; i < NCH; ++i) {
        const int d = i * 32 + c * 8;
        kf[t][i] = ctx_ld16(kb + static_cast<long>(j) * p.k_ss + d, ok && d < p.D);
      }
    }
  };
  load_k(i0 + warp);
  for (int it = i0 + warp; it < i1; it += CR_WARPS) {
    const int j0 = it * 16;
    bool vis[4];
    uint4 vf[4][NBLK];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int j = j0 + 2 * c + (e & 1) + (e >> 1) * 8;
      vis[e] = visible(j);
#pragma unroll
      for (int i = 0; i < NBLK; ++i) {
        const int d = i * 64 + n * 8;
        vf[e][i] = ctx_ld16(vb + static_cast<long>(j) * p.v_ss + d, vis[e] && d < p.D);
      }
    }
    float s[2][4];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int e = 0; e < 4; ++e) s[t][e] = 0.f;
#pragma unroll
      for (int i = 0; i < NCH; ++i) {
        mma16816<FP16>(s[t], q0[i].x, q1[i].x, q0[i].y, q1[i].y, kf[t][i].x, kf[t][i].y);
        mma16816<FP16>(s[t], q0[i].z, q1[i].z, q0[i].w, q1[i].w, kf[t][i].z, kf[t][i].w);
      }
    }
    load_k(it + CR_WARPS);
    // s[t][0..1]: row n, keys 8 t + 2 c + {0, 1}; s[t][2..3]: row n + 8
    float pr[2][4];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      float mx = -INFINITY;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          s[t][r * 2 + e] = vis[t * 2 + e] ? s[t][r * 2 + e] * p.scale_log2 : -INFINITY;
          mx = fmaxf(mx, s[t][r * 2 + e]);
        }
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const float m_new = fmaxf(m[r], mx);
      if (__any_sync(0xffffffffu, m_new > m[r])) {
        const float alpha = m_new == -INFINITY ? 1.f : fast_exp2(m[r] - m_new);
        l[r] *= alpha;
#pragma unroll
        for (int i = 0; i < NBLK; ++i)
#pragma unroll
          for (int t = 0; t < 8; ++t) o[i][t][r * 2] *= alpha, o[i][t][r * 2 + 1] *= alpha;
        m[r] = m_new;
      }
      const float base = m[r] == -INFINITY ? 0.f : m[r];
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          pr[t][r * 2 + e] = fast_exp2(s[t][r * 2 + e] - base);
          l[r] += pr[t][r * 2 + e];
        }
    }
    // P enters the product in the inputs' type (values in [0, 1]); its sum stays in fp32
    const uint32_t a0 = ctx_pack2<FP16>(pr[0][0], pr[0][1]), a1 = ctx_pack2<FP16>(pr[0][2], pr[0][3]);
    const uint32_t a2 = ctx_pack2<FP16>(pr[1][0], pr[1][1]), a3 = ctx_pack2<FP16>(pr[1][2], pr[1][3]);
#pragma unroll
    for (int i = 0; i < NBLK; ++i) {
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const uint32_t k0 = (&vf[0][i].x)[w], k1 = (&vf[1][i].x)[w], k8 = (&vf[2][i].x)[w], k9 = (&vf[3][i].x)[w];
        mma16816<FP16>(o[i][2 * w], a0, a1, a2, a3, __byte_perm(k0, k1, 0x5410), __byte_perm(k8, k9, 0x5410));
        mma16816<FP16>(o[i][2 * w + 1], a0, a1, a2, a3, __byte_perm(k0, k1, 0x7632), __byte_perm(k8, k9, 0x7632));
      }
    }
  }
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
    const int row = n + r * 8;
    if (c == 0) s_m[warp][row] = m[r], s_l[warp][row] = l[r];
    // column 2c of MMA t is channel 64 i + 16 c + t, column 2c + 1 the channel 8 further
    if (row < R) {
#pragma unroll
      for (int i = 0; i < NBLK; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int t = 0; t < 8; t += 4)
            *reinterpret_cast<float4*>(&s_o[warp][row][i * 64 + c * 16 + e * 8 + t]) =
                make_float4(o[i][t][r * 2 + e], o[i][t + 1][r * 2 + e], o[i][t + 2][r * 2 + e], o[i][t + 3][r * 2 + e]);
    }
  }
  __syncthreads();
  const int per_row = p.D >> 2;  // float4 groups of a row
  for (int x = threadIdx.x; x < R * per_row; x += CR_WARPS * 32) {
    const int row = x / per_row, d = (x - row * per_row) * 4;
    float mm = s_m[0][row];
#pragma unroll
    for (int w = 1; w < CR_WARPS; ++w) mm = fmaxf(mm, s_m[w][row]);
    const float base = mm == -INFINITY ? 0.f : mm;
    float sum = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < CR_WARPS; ++w) {
      const float f = fast_exp2(s_m[w][row] - base);
      sum += f * s_l[w][row];
      const float4 t = *reinterpret_cast<const float4*>(&s_o[w][row][d]);
      acc.x += f * t.x, acc.y += f * t.y, acc.z += f * t.z, acc.w += f * t.w;
    }
    const float inv = sum > 0.f ? 1.f / sum : 0.f;
    const long token = static_cast<long>(b) * p.Sq + row / G;
    const int head = hk * G + row % G;
    const float lse2 = mm == -INFINITY ? -INFINITY : mm + log2f(sum);
    if (p.part_o) {
      const long at = (static_cast<long>(p.slot0 + split) * p.B * p.Sq + token) * p.H + head;
      if (d == 0) p.part_lse[at] = lse2;
      if (mm != -INFINITY)
        *reinterpret_cast<float4*>(p.part_o + at * p.D + d) = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
    } else {
      uint16_t* op = static_cast<uint16_t*>(p.out) + (token * p.H + head) * p.D + d;
      *reinterpret_cast<uint2*>(op) = make_uint2(ctx_pack2<FP16>(acc.x * inv, acc.y * inv), ctx_pack2<FP16>(acc.z * inv, acc.w * inv));
      if (p.lse && d == 0)
        p.lse[(static_cast<long>(b) * p.H + head) * p.Sq + row / G] = lse2 * 0.6931471805599453f;
    }
  }
}

// out = sum_s w_s o_s / sum_s w_s, w_s = 2^(lse_s - max): one warp per (token, head), slots added in their order.
template <bool FP16>
__global__ void __launch_bounds__(256) ctx_join_kernel(const CtxParams p) {
  const long rows = static_cast<long>(p.B) * p.Sq * p.H;
  const long row = blockIdx.x * 8L + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row >= rows) return;
  float mm = -INFINITY;
  for (int s = lane; s < p.ns; s += 32) mm = fmaxf(mm, p.part_lse[s * rows + row]);
  mm = warp_max(mm);
  float sum = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  const int d = lane * 4;
#pragma unroll 4
  for (int s = 0; s < p.ns; ++s) {
    const float ls = p.part_lse[s * rows + row];
    if (ls == -INFINITY) continue;
    const float f = fast_exp2(ls - mm);
    sum += f;
    if (d < p.D) {
      const float4 t = *reinterpret_cast<const float4*>(p.part_o + (s * rows + row) * p.D + d);
      acc.x += f * t.x, acc.y += f * t.y, acc.z += f * t.z, acc.w += f * t.w;
    }
  }
  const float inv = sum > 0.f ? 1.f / sum : 0.f;
  if (d < p.D)
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + row * p.D + d) =
        make_uint2(ctx_pack2<FP16>(acc.x * inv, acc.y * inv), ctx_pack2<FP16>(acc.z * inv, acc.w * inv));
  if (p.lse && lane == 0) {
    const long token = row / p.H;
    const int h = static_cast<int>(row % p.H);
    p.lse[(token / p.Sq * p.H + h) * p.Sq + token % p.Sq] =
        sum > 0.f ? (mm + log2f(sum)) * 0.6931471805599453f : -INFINITY;
  }
}

int launch_ctx_rows(const CtxParams& p, int fp16, cudaStream_t st) {
  const long ctas = static_cast<long>(p.B) * p.Hkv * p.ns;
  if (p.Sq * (p.H / p.Hkv) > 16 || ctas > 0x7fffffffL) return TFB_ERR_TOO_LARGE;
  const int g = static_cast<int>(ctas);
  if (p.D <= 64) {
    if (fp16) ctx_rows_kernel<true, 64><<<g, CR_WARPS * 32, 0, st>>>(p);
    else ctx_rows_kernel<false, 64><<<g, CR_WARPS * 32, 0, st>>>(p);
  } else {
    if (fp16) ctx_rows_kernel<true, 128><<<g, CR_WARPS * 32, 0, st>>>(p);
    else ctx_rows_kernel<false, 128><<<g, CR_WARPS * 32, 0, st>>>(p);
  }
  return cudaGetLastError() == cudaSuccess ? TFB_OK : TFB_ERR_LAUNCH;
}

int launch_ctx_join(const CtxParams& p, int fp16, cudaStream_t st) {
  const long blocks = (static_cast<long>(p.B) * p.Sq * p.H + 7) / 8;
  if (blocks > 0x7fffffffL) return TFB_ERR_TOO_LARGE;
  if (fp16) ctx_join_kernel<true><<<static_cast<int>(blocks), 256, 0, st>>>(p);
  else ctx_join_kernel<false><<<static_cast<int>(blocks), 256, 0, st>>>(p);
  return cudaGetLastError() == cudaSuccess ? TFB_OK : TFB_ERR_LAUNCH;
}

}  // namespace tfb
