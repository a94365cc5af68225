// Context attention of many query rows to at most 64 keys (audio windows, image tokens, short prompts): HBM bound on the
// queries and the output, 1 KB per row and head dim 128 against a few thousand tensor operations.
//
// So nothing stands between memory and registers but warps: a CTA of four keeps the keys and values of one (sample, key
// head) in shared memory, and every warp takes tiles of 16 query rows - (token, grouped head) pairs, any group size - straight
// from global memory into mma.sync fragments, softmax in registers, results straight to global memory, the next tile's
// queries already on their way. 16 to 20 warps per SM hold 64 KB and more of loads in flight. (The tensor-memory kernel hands every
// tile through five warps and their barriers, about 10,000 clk per 256 rows whatever the keys: 258 us against 138 here for 21
// frames of 1560 tokens x 40 heads against 32 keys, 4.9 TB/s, three quarters of what a copy reaches. At its upper end the two meet: 20000 tokens
// x 32 heads take 108 us with 64 keys here, 111 with 65 there.) What bounds it then is L1: every query and output byte
// passes it in 16-byte pieces of eight rows at a time (79 % busy), half of all issue slots are taken.
// Coalescing comes from permuting indexes: a lane loads and stores whole 16-byte pieces of a row, and the copies of K and V
// in shared memory have their channels reordered to match what the fragments then hold:
//   Q.K^T  lane (n, c) = (lane / 4, lane % 4) holds channels 32 i + 8 c .. + 7 of row n; it feeds pair w (channels 2 w, 2 w + 1
//          of them) into half w % 2 of k-step w / 2
//   P.V    columns 2 c, 2 c + 1 of MMA 4 i + w are the same two channels, so a lane ends up with 16 bytes of its row and the
//          four lanes of a row with 64 bytes next to each other
// Both want channel 32 i + 8 c + 2 w + e at position 32 i + 8 w + 2 c + e.
// Hidden keys are zeros in both copies and their scores become -inf, so what lies there does not matter.
#include "context_attn.cuh"

namespace tfb {

constexpr int CS_WARPS = 4;
static_assert(CTX_SHORT_KEYS == 64, "four steps of 16 keys");

struct CtxShortParams {
  CtxParams c;
  int tiles;    // tiles of 16 rows per (sample, key head)
  int per_cta;  // ... that one CTA takes
  int chunks;   // CTAs per (sample, key head)
};

template <bool FP16>
__device__ __forceinline__ void cs_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
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

// STEPS: 16-key steps that the registers are laid out for (2 or 4).
template <bool FP16, int DK, int STEPS>
__global__ void __launch_bounds__(CS_WARPS * 32, STEPS == 2 ? 5 : 4) ctx_short_kernel(const __grid_constant__ CtxShortParams sp) {
  constexpr int NCH = DK / 32, NBLK = DK / 64, LD = DK + 8;  // row stride: 16 bytes over a multiple of 128
  __shared__ __align__(16) uint16_t s_k[STEPS * 16 * LD];
  __shared__ __align__(16) uint16_t s_v[STEPS * 16 * LD];
  const CtxParams& p = sp.c;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n = lane >> 2, c = lane & 3;
  const int G = p.H / p.Hkv;
  const unsigned uG = G, R = static_cast<unsigned>(p.Sq) * uG;  // below 2^31
  // Heads first: CTAs that run at the same time then read and write the heads of the same tokens, whole DRAM pages together.
  const int hk = blockIdx.x % p.Hkv;
  const int chunk = (blockIdx.x / p.Hkv) % sp.chunks;
  const int b = blockIdx.x / p.Hkv / sp.chunks;
  const int t0 = chunk * sp.per_cta, t1 = min(t0 + sp.per_cta, sp.tiles);

  const uint16_t* qb = static_cast<const uint16_t*>(p.q) + static_cast<long>(b) * p.q_bs + static_cast<long>(hk) * G * p.q_hs;
  uint4 q[2][NCH];  // rows n and n + 8 of the tile
  auto load_q = [&](int tile) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const unsigned row = tile * 16u + n + r * 8, token = row / uG;
      const uint16_t* at = qb + static_cast<long>(token) * p.q_ss + static_cast<long>(row - token * uG) * p.q_hs;
#pragma unroll
      for (int i = 0; i < NCH; ++i) {
        const int d = i * 32 + c * 8;
        q[r][i] = make_uint4(0, 0, 0, 0);
        if (tile < t1 && row < R && d < p.D) q[r][i] = __ldcs(reinterpret_cast<const uint4*>(at + d));
      }
    }
  };
  load_q(t0 + warp);

  int first, len;
  ctx_sample_range(p, b, first, len);
  len = min(len, STEPS * 16);  // packed samples: the rule on sizes has looked at all their rows
  const uint8_t* mb = p.key_mask ? p.key_mask + static_cast<long>(b) * p.mask_bs : nullptr;
  const int steps = (len + 15) >> 4;  // 16 keys each
  const long kv_b = p.cu_kv ? 0 : b;
  const uint16_t* kb = static_cast<const uint16_t*>(p.k) + kv_b * p.k_bs + static_cast<long>(first) * p.k_ss + static_cast<long>(hk) * p.k_hs;
  const uint16_t* vb = static_cast<const uint16_t*>(p.v) + kv_b * p.v_bs + static_cast<long>(first) * p.v_ss + static_cast<long>(hk) * p.v_hs;
  for (int x = threadIdx.x; x < steps * 16 * (DK / 8); x += CS_WARPS * 32) {
    const int key = x / (DK / 8), ch = x % (DK / 8) * 8;
    const bool ok = key < len && ch < p.D && (!mb || mb[key]);
    uint4 kw = make_uint4(0, 0, 0, 0), vw = kw;
    if (ok) {
      kw = __ldg(reinterpret_cast<const uint4*>(kb + static_cast<long>(key) * p.k_ss + ch));
      vw = __ldg(reinterpret_cast<const uint4*>(vb + static_cast<long>(key) * p.v_ss + ch));
    }
    const int at = key * LD + (ch & ~31) + (ch >> 3 & 3) * 2;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      *reinterpret_cast<uint32_t*>(s_k + at + w * 8) = (&kw.x)[w];
      *reinterpret_cast<uint32_t*>(s_v + at + w * 8) = (&vw.x)[w];
    }
  }
  // hidden keys among this lane's score columns 16 step + 8 t + 2 c + e, as bits 4 step + 2 t + e
  uint32_t hidden = 0;
#pragma unroll
  for (int x = 0; x < STEPS * 4; ++x) {
    const int key = (x >> 2) * 16 + (x >> 1 & 1) * 8 + 2 * c + (x & 1);
    if (key >= len || (mb && !mb[key])) hidden |= 1u << x;
  }
  const bool some_hidden = __any_sync(0xffffffffu, hidden != 0);
  __syncthreads();

  // ldmatrix rows of this lane (see context_attn_rows.cu): K by key octets, V by key rows of a 16-key step
  const uint32_t k_at = smem_u32(s_k) + (((lane & 7) + ((lane >> 4) << 3)) * LD + ((lane >> 3) & 1) * 8) * 2;
  const uint32_t v_at = smem_u32(s_v) + ((lane & 15) * LD + (lane >> 4) * 8) * 2;
  uint16_t* ob = static_cast<uint16_t*>(p.out) + (static_cast<long>(b) * p.Sq * p.H + static_cast<long>(hk) * G) * p.D;

  for (int tile = t0 + warp; tile < t1; tile += CS_WARPS) {
    float s[STEPS][2][4];
#pragma unroll
    for (int st = 0; st < STEPS; ++st) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[st][t][e] = 0.f;
      if (st < steps) {
#pragma unroll
        for (int i = 0; i < NCH; ++i)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            uint32_t kf[4];
            asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                         : "=r"(kf[0]), "=r"(kf[1]), "=r"(kf[2]), "=r"(kf[3])
                         : "r"(k_at + (st * 16 * LD + i * 32 + u * 16) * 2));
            const uint32_t a0 = u ? q[0][i].z : q[0][i].x, a1 = u ? q[1][i].z : q[1][i].x;
            const uint32_t a2 = u ? q[0][i].w : q[0][i].y, a3 = u ? q[1][i].w : q[1][i].y;
            cs_mma<FP16>(s[st][0], a0, a1, a2, a3, kf[0], kf[1]);
            cs_mma<FP16>(s[st][1], a0, a1, a2, a3, kf[2], kf[3]);
          }
      }
    }
    load_q(tile + CS_WARPS);
    float inv[2], lse2[2];
    uint32_t pf[STEPS][4];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      if (some_hidden) {
#pragma unroll
        for (int x = 0; x < STEPS * 4; ++x)
          if (hidden >> x & 1) s[x >> 2][x >> 1 & 1][r * 2 + (x & 1)] = -INFINITY;
      }
      float mx = -INFINITY;
#pragma unroll
      for (int st = 0; st < STEPS; ++st)
#pragma unroll
        for (int t = 0; t < 2; ++t) mx = fmax3(mx, s[st][t][r * 2], s[st][t][r * 2 + 1]);
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const float top = mx * p.scale_log2, base = ctx_exp_base(top);
      float l = 0.f;
#pragma unroll
      for (int st = 0; st < STEPS; ++st)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const float p0 = fast_exp2(s[st][t][r * 2] * p.scale_log2 - base), p1 = fast_exp2(s[st][t][r * 2 + 1] * p.scale_log2 - base);
          l += p0 + p1;
          pf[st][t * 2 + r] = ctx_pack2<FP16>(p0, p1);  // in [0, 1], rounded to the inputs' type for the product
        }
      l += __shfl_xor_sync(0xffffffffu, l, 1);
      l += __shfl_xor_sync(0xffffffffu, l, 2);
      inv[r] = ctx_inverse(l);
      lse2[r] = ctx_lse2(top, l);
    }
    long row_at[2];
    bool row_ok[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const unsigned row = tile * 16u + n + r * 8, token = row / uG;
      const int g = static_cast<int>(row - token * uG);
      row_ok[r] = row < R;
      row_at[r] = (static_cast<long>(token) * p.H + g) * p.D;
      if (p.lse && row_ok[r] && c == 0)
        p.lse[(static_cast<long>(b) * p.H + hk * G + g) * p.Sq + token] = lse2[r] * 0.6931471805599453f;
    }
#pragma unroll
    for (int blk = 0; blk < NBLK; ++blk) {
      float o[8][4];
#pragma unroll
      for (int t = 0; t < 8; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[t][e] = 0.f;
#pragma unroll
      for (int st = 0; st < STEPS; ++st) {
        if (st < steps) {
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            uint32_t vf[4];
            asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                         : "=r"(vf[0]), "=r"(vf[1]), "=r"(vf[2]), "=r"(vf[3])
                         : "r"(v_at + (st * 16 * LD + blk * 64 + t * 16) * 2));
            cs_mma<FP16>(o[2 * t], pf[st][0], pf[st][1], pf[st][2], pf[st][3], vf[0], vf[1]);
            cs_mma<FP16>(o[2 * t + 1], pf[st][0], pf[st][1], pf[st][2], pf[st][3], vf[2], vf[3]);
          }
        }
      }
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int d = blk * 64 + 32 * h + 8 * c;
          uint4 v;
#pragma unroll
          for (int w = 0; w < 4; ++w) (&v.x)[w] = ctx_pack2<FP16>(o[h * 4 + w][r * 2] * inv[r], o[h * 4 + w][r * 2 + 1] * inv[r]);
          if (row_ok[r] && d < p.D) *reinterpret_cast<uint4*>(ob + row_at[r] + d) = v;
        }
    }
  }
}

template <bool FP16, int DK, int STEPS>
static int launch_ctx_short_impl(const CtxParams& p, cudaStream_t st) {
  CtxShortParams sp;
  sp.c = p;
  const long rows = static_cast<long>(p.Sq) * (p.H / p.Hkv), heads = static_cast<long>(p.B) * p.Hkv;
  const long tiles = (rows + 15) / 16;
  if (rows > 0x7fffff00L) return TFB_ERR_TOO_LARGE;
  // About eight CTAs per resident one, so that the last wave is short, but no fewer than four tiles per warp: refilling
  // shared memory with K and V should stay small against them.
  const long want = (8L * 4 * sm_count() + heads - 1) / heads;
  long per = (tiles + want - 1) / want;
  if (per < 4 * CS_WARPS) per = 4 * CS_WARPS;
  if (heads * ((tiles + per - 1) / per) < 4 * sm_count()) per = CS_WARPS;
  sp.tiles = static_cast<int>(tiles);
  sp.per_cta = static_cast<int>((per + CS_WARPS - 1) / CS_WARPS * CS_WARPS);
  sp.chunks = static_cast<int>((tiles + sp.per_cta - 1) / sp.per_cta);
  const long ctas = heads * sp.chunks;
  if (ctas > 0x7fffffffL) return TFB_ERR_TOO_LARGE;
  ctx_short_kernel<FP16, DK, STEPS><<<static_cast<int>(ctas), CS_WARPS * 32, 0, st>>>(sp);
  return cudaGetLastError() == cudaSuccess ? TFB_OK : TFB_ERR_LAUNCH;
}

template <bool FP16>
static int launch_ctx_short_type(const CtxParams& p, cudaStream_t st) {
  const bool two = p.Skv <= 32;
  if (p.D <= 64) return two ? launch_ctx_short_impl<FP16, 64, 2>(p, st) : launch_ctx_short_impl<FP16, 64, 4>(p, st);
  return two ? launch_ctx_short_impl<FP16, 128, 2>(p, st) : launch_ctx_short_impl<FP16, 128, 4>(p, st);
}

int launch_ctx_short(const CtxParams& p, int fp16, cudaStream_t st) {
  if (p.Skv > CTX_SHORT_KEYS || p.part_o) return TFB_ERR_TOO_LARGE;
  return fp16 ? launch_ctx_short_type<true>(p, st) : launch_ctx_short_type<false>(p, st);
}

}  // namespace tfb
