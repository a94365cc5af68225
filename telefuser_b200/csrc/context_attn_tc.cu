// Context attention for full query tiles on tcgen05: o = softmax(scale q k^T) v over the keys a sample may see - a shared
// prefix, then the sample's own keys up to its length, minus masked ones. bf16 or fp16, head_dim <= 64 / <= 128.
//
// Persistent: one CTA per SM walks over work items (sample, head group, pair of 128-row query tiles, key slice). A tile's
// rows are (token, head) pairs of one key head where the head group is a power of two, so grouped heads share every K / V
// tile; otherwise a tile is 128 tokens of one head. 384 threads:
//   warps 0..3  softmax group 0 (query tile 0; TMEM lane == row)       warp 8   TMA loader
//   warps 4..7  softmax group 1 (query tile 1)                         warp 9   tcgen05.mma issuer, TMEM owner
//   warp 10     tail / mask warp: clears the V rows that nobody may see before the P.V product reads them (a product
//               with infinities or NaN there would spread through P = 0) and turns the key mask into bit words
//   warp 11     only donates registers
// TMEM (512 columns): S0 | S1 | O0 | O1. P overwrites the first 64 columns of its S tile and enters P.V from TMEM.
// Encoder states are short (a prompt is 1 .. 4 blocks of 128 keys), so the ends of an item count: the issuer starts the
// next item's Q.K^T of a tile right behind the last P.V of that tile, the loader is a whole item ahead, and a softmax
// group writes its output (through shared memory and TMA stores that clip at the tensor's edge) while the other group
// and the tensor core work on. The last block of a sample is as narrow as its keys need: 32-column steps in Q.K^T, the
// exponentials and P.V.
//
// The row maximum that exp2 uses is only raised when it grew by more than 2^8. P is rounded to the inputs' type for the
// product (at most 2^8, sum in fp32).
#include <math.h>

#include "context_attn.cuh"

namespace tfb {

constexpr int CT_TILE = 128 * 128 * 2;  // 32 KB: two boxes of [128 rows][64 channels]
constexpr int CT_BOX = 128 * 64 * 2;
constexpr int CT_Q_OFF = 0;
constexpr int CT_KV_OFF = 2 * CT_TILE;               // K ring of 2, then V ring of 2
constexpr int CT_OUT_OFF = CT_KV_OFF + 4 * CT_TILE;  // 8 warps x 2 buffers x [32 rows][32 channels]
constexpr int CT_BAR_OFF = CT_OUT_OFF + 8 * 4096;
constexpr int CT_SMEM_BYTES = CT_BAR_OFF + 256 + 1024;
static_assert(CT_SMEM_BYTES <= 227 * 1024, "shared memory of one CTA");
constexpr float CT_RESCALE_THRESHOLD = 8.0f;

struct CtxTcParams {
  CtxParams c;
  int pack;       // heads of a key head that share a tile (power of two, 1 = one head per tile)
  int n_hg;       // head groups: H / pack
  int n_qp;       // pairs of query tiles
  int tok;        // tokens per tile: 128 / pack
  int n_prefix;   // prefix blocks
  int bmul;       // 0: all samples' own keys lie in the tensors' only batch entry (packed samples)
  int n_items;
};

struct CtxItem {
  int b, hg, qp, split;
  int first, len;  // the sample's own keys
  int j0, j1;      // key blocks [j0, j1) of prefix blocks followed by own blocks
  bool two;        // the second query tile has rows
};

__device__ __forceinline__ CtxItem ctx_item(const CtxTcParams& p, int i) {
  CtxItem t;
  t.qp = i % p.n_qp;
  i /= p.n_qp;
  t.split = i % p.c.ns;
  i /= p.c.ns;
  t.hg = i % p.n_hg;
  t.b = i / p.n_hg;
  ctx_sample_range(p.c, t.b, t.first, t.len);
  const long nb = p.n_prefix + ((t.len + 127) >> 7);
  t.j0 = static_cast<int>(nb * t.split / p.c.ns);
  t.j1 = static_cast<int>(nb * (t.split + 1) / p.c.ns);
  t.two = (t.qp * 2 + 1) * p.tok < p.c.Sq;
  return t;
}
// Visible keys of block j at most 128 (before the mask).
__device__ __forceinline__ int ctx_block_keys(const CtxTcParams& p, const CtxItem& t, int j) {
  return min(128, j < p.n_prefix ? p.c.P - j * 128 : t.len - (j - p.n_prefix) * 128);
}
// The next item of this CTA that has keys.
__device__ __forceinline__ bool ctx_next(const CtxTcParams& p, int& i, CtxItem& t) {
  while (i < p.n_items) {
    t = ctx_item(p, i);
    i += gridDim.x;
    if (t.j1 > t.j0) return true;
  }
  return false;
}

template <bool FP16, int DK, bool MASK>
__global__ void __launch_bounds__(384, 1)
    ctx_tc_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                  const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmKp,
                  const __grid_constant__ CUtensorMap tmVp, const __grid_constant__ CUtensorMap tmO,
                  const __grid_constant__ CtxTcParams p) {
  constexpr int NBOX = DK / 64;
  constexpr uint32_t LOAD_BYTES = NBOX * CT_BOX;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + CT_BAR_OFF);
  uint64_t* q_full = bars + 0;    // [2] per query tile
  uint64_t* q_empty = bars + 2;   // [2]
  uint64_t* k_full = bars + 4;    // [2] per ring slot
  uint64_t* k_empty = bars + 6;   // [2]
  uint64_t* v_full = bars + 8;    // [2]
  uint64_t* v_empty = bars + 10;  // [2]
  uint64_t* v_ready = bars + 12;  // [2] hidden rows cleared, mask words written
  uint64_t* s_full = bars + 14;   // [2] per query tile
  uint64_t* p_ready = bars + 16;  // [2]
  uint64_t* o_final = bars + 18;  // [2]
  uint32_t* words = reinterpret_cast<uint32_t*>(bars + 20);  // [2 slots][4]
  uint32_t* tmem_slot = words + 8;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  AbortCtx ctx{abort_flag, p.c.status};

  if (threadIdx.x == 0) {
    for (int s = 0; s < 2; ++s) {
      mbar_init(&q_full[s], 1);
      mbar_init(&q_empty[s], 1);
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 1);
      mbar_init(&v_full[s], 1);
      mbar_init(&v_empty[s], 1);
      mbar_init(&v_ready[s], 32);
      mbar_init(&s_full[s], 1);
      mbar_init(&p_ready[s], 128);
      mbar_init(&o_final[s], 1);
    }
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 9) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  // Registers move only inside the launch allocation: 256 x 216 + 128 x 72 = 384 x 168.
  static_assert(256 * 216 + 128 * 72 <= 384 * 168, "setmaxnreg split");
  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    if (warp == 8) {
      // ------------------------------ TMA loader ------------------------------
      if (lane == 0) {
        tma_prefetch_desc(&tmQ);
        tma_prefetch_desc(&tmK);
        tma_prefetch_desc(&tmV);
        CtxItem t;
        int i = blockIdx.x, g = 0;
        int nq[2] = {0, 0};
        bool ok = true;
        while (ok && ctx_next(p, i, t)) {
          const int hk = t.hg * p.pack / (p.c.H / p.c.Hkv);
          for (int j = t.j0; j < t.j1 && ok; ++j, ++g) {
            const int slot = g & 1;
            const uint32_t ph = (g >> 1) & 1;
            const bool pre = j < p.n_prefix;
            const int row = pre ? j * 128 : t.first + (j - p.n_prefix) * 128;
            if (!(ok = mbar_wait(&k_empty[slot], ph ^ 1, ctx, 40))) break;
            uint8_t* dst = smem + CT_KV_OFF + slot * CT_TILE;
            const CUtensorMap* tm = pre ? &tmKp : &tmK;
            mbar_expect_tx(&k_full[slot], LOAD_BYTES);
            for (int x = 0; x < NBOX; ++x)
              tma_load_4d(dst + x * CT_BOX, tm, &k_full[slot], x * 64, hk, row, pre ? 0 : t.b * p.bmul);
            if (j == t.j0) {
              for (int st = 0; st < (t.two ? 2 : 1); ++st) {
                if (!(ok = mbar_wait(&q_empty[st], (nq[st] & 1) ^ 1, ctx, 41))) break;
                ++nq[st];
                mbar_expect_tx(&q_full[st], LOAD_BYTES);
                for (int x = 0; x < NBOX; ++x)
                  tma_load_4d(smem + CT_Q_OFF + st * CT_TILE + x * CT_BOX, &tmQ, &q_full[st], x * 64, t.hg * p.pack,
                              (t.qp * 2 + st) * p.tok, t.b);
              }
              if (!ok) break;
            }
            if (!(ok = mbar_wait(&v_empty[slot], ph ^ 1, ctx, 42))) break;
            dst = smem + CT_KV_OFF + (2 + slot) * CT_TILE;
            tm = pre ? &tmVp : &tmV;
            mbar_expect_tx(&v_full[slot], LOAD_BYTES);
            for (int x = 0; x < NBOX; ++x)
              tma_load_4d(dst + x * CT_BOX, tm, &v_full[slot], x * 64, hk, row, pre ? 0 : t.b * p.bmul);
          }
        }
      }
      __syncwarp();
    } else if (warp == 9) {
      // ------------------------------ MMA issuer ------------------------------
      constexpr uint32_t FMT = FP16 ? 0 : 1;
      constexpr uint32_t idesc_pv = make_idesc(128, DK, FMT, FMT, 0, 1);  // B (= V) is MN-major
      CtxItem t, nt;
      int i = blockIdx.x, g = 0;
      int nq[2] = {0, 0}, np[2] = {0, 0};
      bool ok = true;
      // Q.K^T of key block j into S of query tile st; `last`: no further block of this item reads the Q tile
      auto issue_qk = [&](int st, const CtxItem& it, int j, int gg, bool last) {
        const uint32_t idesc = make_idesc(128, (ctx_block_keys(p, it, j) + 31) & ~31, FMT, FMT, 0, 0);
        const uint32_t q_addr = smem_u32(smem + CT_Q_OFF + st * CT_TILE);
        const uint32_t k_addr = smem_u32(smem + CT_KV_OFF + (gg & 1) * CT_TILE);
#pragma unroll
        for (int kk = 0; kk < DK / 16; ++kk) {
          const uint32_t off = (kk >> 2) * CT_BOX + (kk & 3) * 32;
          umma_f16_ss(tmem_base + st * 128, make_desc_k_sw128(q_addr + off), make_desc_k_sw128(k_addr + off), idesc,
                      kk ? 1u : 0u);
        }
        umma_commit(&s_full[st]);
        if (last) umma_commit(&q_empty[st]);
      };
      auto prime = [&](int st, const CtxItem& it, int gg) {
        if (!mbar_wait_warp(&q_full[st], nq[st] & 1, ctx, 43)) return false;
        ++nq[st];
        if (!mbar_wait_warp(&k_full[gg & 1], (gg >> 1) & 1, ctx, 44)) return false;
        tc_fence_after();
        if (lane == 0) issue_qk(st, it, it.j0, gg, it.j1 - it.j0 == 1);
        __syncwarp();
        return true;
      };
      bool have = ctx_next(p, i, t);
      if (have) {
        ok = prime(0, t, 0) && (!t.two || prime(1, t, 0));
        if (ok && lane == 0) umma_commit(&k_empty[0]);
        __syncwarp();
      }
      while (have && ok) {
        const int nb = t.j1 - t.j0, gn = g + nb;
        const bool have_next = ctx_next(p, i, nt);
        for (int n = 0; n < nb && ok; ++n) {
          const int gv = g + n;
          const bool more = n + 1 < nb;
          const int steps = ((ctx_block_keys(p, t, t.j0 + n) + 31) >> 5) * 2;
          ok = mbar_wait_warp(&v_full[gv & 1], (gv >> 1) & 1, ctx, 52) &&
               mbar_wait_warp(&v_ready[gv & 1], (gv >> 1) & 1, ctx, 45) &&
               (!more || mbar_wait_warp(&k_full[(gv + 1) & 1], ((gv + 1) >> 1) & 1, ctx, 46));
          for (int st = 0; st < (t.two ? 2 : 1) && ok; ++st) {
            if (!(ok = mbar_wait_warp(&p_ready[st], np[st] & 1, ctx, 47))) break;
            ++np[st];
            tc_fence_after();
            if (lane == 0) {
              const uint32_t v_addr = smem_u32(smem + CT_KV_OFF + (2 + (gv & 1)) * CT_TILE);
              const uint32_t o_tmem = tmem_base + 256 + st * 128, p_tmem = tmem_base + st * 128;
              for (int kk = 0; kk < steps; ++kk)
                umma_f16_ts(o_tmem, p_tmem + kk * 8, make_desc_mn_sw128(v_addr + kk * 2048, CT_BOX), idesc_pv,
                            (n | kk) ? 1u : 0u);
              if (more)
                issue_qk(st, t, t.j0 + n + 1, gv + 1, n + 2 == nb);
              else
                umma_commit(&o_final[st]);
            }
            __syncwarp();
            if (!more && have_next && (st == 0 || nt.two)) ok = prime(st, nt, gn);
          }
          if (ok && lane == 0) {
            umma_commit(&v_empty[gv & 1]);
            if (more) umma_commit(&k_empty[(gv + 1) & 1]);
          }
          __syncwarp();
        }
        if (ok && have_next) {
          if (nt.two && !t.two) ok = prime(1, nt, gn);
          if (ok && lane == 0) umma_commit(&k_empty[gn & 1]);
          __syncwarp();
        }
        have = have_next;
        t = nt;
        g = gn;
      }
    } else if (warp == 10) {
      // ------------------------------ tail / mask warp ------------------------------
      CtxItem t;
      int i = blockIdx.x, g = 0;
      bool ok = true;
      while (ok && ctx_next(p, i, t)) {
        for (int j = t.j0; j < t.j1; ++j, ++g) {
          const int slot = g & 1;
          const int keys = ctx_block_keys(p, t, j), cols = (keys + 31) & ~31;
          uint32_t w[4];
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int key = x * 32 + lane;
            bool vis = key < keys;
            if (MASK && vis)
              vis = __ldg(p.c.key_mask + static_cast<long>(t.b) * p.c.mask_bs + (j - p.n_prefix) * 128 + key) != 0;
            w[x] = __ballot_sync(0xffffffffu, vis);
          }
          if (!(ok = mbar_wait_warp(&v_full[slot], (g >> 1) & 1, ctx, 48))) break;
          bool wrote = false;
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            if (x * 32 < cols && w[x] != 0xffffffffu) {
              wrote = true;
              if (!((w[x] >> lane) & 1)) {
                uint4* row = reinterpret_cast<uint4*>(smem + CT_KV_OFF + (2 + slot) * CT_TILE + (x * 32 + lane) * 128);
#pragma unroll
                for (int y = 0; y < NBOX; ++y)
#pragma unroll
                  for (int e = 0; e < 8; ++e) row[y * (CT_BOX / 16) + e] = make_uint4(0, 0, 0, 0);
              }
            }
            if (MASK && lane == x) words[slot * 4 + x] = w[x];
          }
          if (wrote) fence_proxy_async_smem();
          mbar_arrive(&v_ready[slot]);
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    // ------------------------------ softmax groups ------------------------------
    const int st = warp >> 2;
    const int row = (warp & 3) * 32 + lane;
    const uint32_t lane_addr = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t tmem_s = tmem_base + lane_addr + st * 128;
    const uint32_t tmem_o = tmem_base + lane_addr + 256 + st * 128;
    uint8_t* stage = smem + CT_OUT_OFF + warp * 4096;
    const int row_tok = row / p.pack, row_head = row % p.pack;
    int ns = 0, no = 0, g = 0, nout = 0;  // score tiles, items, key blocks and output steps so far
    bool ok = true;
    for (int i = blockIdx.x; i < p.n_items && ok; i += gridDim.x) {
      const CtxItem t = ctx_item(p, i);
      const int nb = t.j1 - t.j0;
      if (st && !t.two) {
        g += nb;
        continue;
      }
      float m_used = -INFINITY, l = 0.f;
      for (int n = 0; n < nb; ++n, ++g) {
        uint32_t w[4] = {0xffffffffu, 0xffffffffu, 0xffffffffu, 0xffffffffu};
        const int keys = ctx_block_keys(p, t, t.j0 + n);
        const int chunks = (keys + 31) >> 5;
        if (!(ok = mbar_wait_warp(&s_full[st], ns & 1, ctx, 50))) break;
        ++ns;
        tc_fence_after();
        if (MASK) {
          // behind s_full: the scores of block g exist only once v_ready of block g - 1 has completed, so the parity of
          // block g cannot be mistaken for that of block g - 4 by a group that skipped items
          if (!(ok = mbar_wait_warp(&v_ready[g & 1], (g >> 1) & 1, ctx, 49))) break;
#pragma unroll
          for (int x = 0; x < 4; ++x) w[x] = *reinterpret_cast<volatile uint32_t*>(&words[(g & 1) * 4 + x]);
        }
        uint32_t s[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c)
          if (c < chunks) tmem_ld_32x32(tmem_s + c * 32, s[c]);
        tmem_ld_wait();
        if (keys < 128 || (MASK && (w[0] & w[1] & w[2] & w[3]) != 0xffffffffu)) {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int left = keys - c * 32;
            const uint32_t vis = left >= 32 ? w[c] : left <= 0 ? 0u : w[c] & ((1u << left) - 1u);
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (!((vis >> e) & 1)) s[c][e] = 0xff800000u;  // -inf
          }
        }
        // Row maximum: 8 independent chains of 3-input max.
        float mx8[8];
#pragma unroll
        for (int a = 0; a < 8; ++a) mx8[a] = __uint_as_float(s[a >> 1][a & 1]);
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int e = 2; e < 32; e += 4) {
            mx8[c * 2] = fmax3(mx8[c * 2], __uint_as_float(s[c][e]), __uint_as_float(s[c][e + 1]));
            if (e + 3 < 32)
              mx8[c * 2 + 1] = fmax3(mx8[c * 2 + 1], __uint_as_float(s[c][e + 2]), __uint_as_float(s[c][e + 3]));
          }
        const float mx = fmax3(fmax3(mx8[0], mx8[1], mx8[2]), fmax3(mx8[3], mx8[4], mx8[5]), fmaxf(mx8[6], mx8[7]));
        const float m_new = fmaxf(m_used, mx * p.c.scale_log2);
        if (n == 0) {
          m_used = m_new;
        } else if (__any_sync(0xffffffffu, (m_new - m_used) > CT_RESCALE_THRESHOLD)) {
          // All MMAs issued before S of this block have completed, so O is stable here.
          const float alpha = m_new == -INFINITY ? 1.f : fast_exp2(m_used - m_new);
          m_used = m_new;
          l *= alpha;
#pragma unroll
          for (int c = 0; c < DK / 32; ++c) {
            uint32_t o[32];
            tmem_ld_32x32(tmem_o + c * 32, o);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
            tmem_st_32x32(tmem_o + c * 32, o);
          }
        }
        // p = 2^(s scale - m): packed fp32x2 FMAs and row sums
        const uint64_t scale2 = f2_pack(p.c.scale_log2, p.c.scale_log2);
        const float neg = m_used == -INFINITY ? 0.f : -m_used;
        const uint64_t negm2 = f2_pack(neg, neg);
        uint64_t ps[4] = {0ull, 0ull, 0ull, 0ull};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          if (c < chunks) {
            uint32_t pk[16];
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              const uint64_t x2 =
                  f2_fma(f2_pack(__uint_as_float(s[c][2 * k]), __uint_as_float(s[c][2 * k + 1])), scale2, negm2);
              float x0, x1;
              f2_unpack(x2, x0, x1);
              const float p0 = fast_exp2(x0), p1 = fast_exp2(x1);
              ps[k & 3] = f2_add(ps[k & 3], f2_pack(p0, p1));
              pk[k] = ctx_pack2<FP16>(p0, p1);
            }
            tmem_st_32x16(tmem_s + c * 16, pk);
          }
        }
        {
          float a0, a1, b0, b1;
          f2_unpack(f2_add(ps[0], ps[1]), a0, a1);
          f2_unpack(f2_add(ps[2], ps[3]), b0, b1);
          l += (a0 + a1) + (b0 + b1);
        }
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(&p_ready[st]);
      }
      if (!ok) break;

      // ------------------------------ output of one tile ------------------------------
      const int tile_tok = (t.qp * 2 + st) * p.tok;
      const int tok = tile_tok + row_tok, head = t.hg * p.pack + row_head;
      const bool row_ok = tok < p.c.Sq;
      if (nb > 0) {
        if (!(ok = mbar_wait_warp(&o_final[st], no & 1, ctx, 51))) break;
        ++no;
        tc_fence_after();
      }
      const float inv = l > 0.f ? 1.f / l : 0.f;
      const long token = static_cast<long>(t.b) * p.c.Sq + tok;
      const float lse2 = l > 0.f ? m_used + log2f(l) : -INFINITY;
      if (p.c.part_o) {
        const long at = (static_cast<long>(p.c.slot0 + t.split) * p.c.B * p.c.Sq + token) * p.c.H + head;
        if (row_ok) p.c.part_lse[at] = lse2;
        if (nb > 0) {
#pragma unroll
          for (int c = 0; c < DK / 32; ++c) {
            uint32_t o[32];
            tmem_ld_32x32(tmem_o + c * 32, o);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 32; e += 4)
              if (row_ok && c * 32 + e < p.c.D)
                *reinterpret_cast<float4*>(p.c.part_o + at * p.c.D + c * 32 + e) =
                    make_float4(__uint_as_float(o[e]) * inv, __uint_as_float(o[e + 1]) * inv,
                                __uint_as_float(o[e + 2]) * inv, __uint_as_float(o[e + 3]) * inv);
          }
        }
      } else {
        if (p.c.lse && row_ok) p.c.lse[(static_cast<long>(t.b) * p.c.H + head) * p.c.Sq + tok] = lse2 * 0.6931471805599453f;
        // 32 rows x 32 channels per step through this warp's own two buffers (64-byte rows, 64B swizzle)
#pragma unroll
        for (int c = 0; c < DK / 32; ++c) {
          if (c * 32 < p.c.D) {
            uint32_t o[32];
            if (nb > 0) {
              tmem_ld_32x32(tmem_o + c * 32, o);
              tmem_ld_wait();
            } else {
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = 0;
            }
            if (lane == 0) tma_store_wait_read1();
            __syncwarp();
            uint8_t* buf = stage + (nout++ & 1) * 2048;
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              uint4 v;
              v.x = ctx_pack2<FP16>(__uint_as_float(o[x * 8 + 0]) * inv, __uint_as_float(o[x * 8 + 1]) * inv);
              v.y = ctx_pack2<FP16>(__uint_as_float(o[x * 8 + 2]) * inv, __uint_as_float(o[x * 8 + 3]) * inv);
              v.z = ctx_pack2<FP16>(__uint_as_float(o[x * 8 + 4]) * inv, __uint_as_float(o[x * 8 + 5]) * inv);
              v.w = ctx_pack2<FP16>(__uint_as_float(o[x * 8 + 6]) * inv, __uint_as_float(o[x * 8 + 7]) * inv);
              *reinterpret_cast<uint4*>(buf + lane * 64 + ((x ^ ((lane >> 1) & 3)) << 4)) = v;
            }
            fence_proxy_async_smem();
            __syncwarp();
            const int first_tok = tile_tok + (warp & 3) * 32 / p.pack;
            if (lane == 0 && first_tok < p.c.Sq) {
              tma_store_4d(&tmO, buf, c * 32, t.hg * p.pack, first_tok, t.b);
              tma_store_commit();
            }
          }
        }
      }
    }
    if (lane == 0) tma_store_wait_all();
    __syncwarp();
  }

  if (*abort_flag) __nanosleep(200000);
  tc_fence_before();
  __syncthreads();
  if (warp == 9) tmem_dealloc(tmem_base, 512);
}

static int ctx_pack(int G) { return (G & (G - 1)) == 0 && G <= 32 ? G : 1; }

long ctx_tc_items(int B, int Sq, int H, int Hkv) {
  const int pack = ctx_pack(H / Hkv), tok = 128 / pack;
  return static_cast<long>(B) * (H / pack) * ((Sq + 2 * tok - 1) / (2 * tok));
}

// [batch][token][head][channel] tensor map; a dimension of one entry may have any stride (TMA wants multiples of 16).
static int ctx_tmap(CUtensorMap* m, const void* base, int fp16, int D, int heads, long hs, long rows, long ss, int B, long bs,
                    uint32_t box_c, uint32_t box_h, uint32_t box_s, int swizzle) {
  uint64_t dims[4] = {static_cast<uint64_t>(D), static_cast<uint64_t>(heads), static_cast<uint64_t>(rows),
                      static_cast<uint64_t>(B)};
  uint64_t str[3] = {static_cast<uint64_t>(heads > 1 ? hs : 8) * 2, static_cast<uint64_t>(rows > 1 ? ss : 8) * 2,
                     static_cast<uint64_t>(B > 1 ? bs : 8) * 2};
  uint32_t box[4] = {box_c, box_h, box_s, 1};
  return make_tmap(m, base, fp16 ? TM_F16 : TM_BF16, 4, dims, str, box, swizzle);
}

template <bool FP16, int DK, bool MASK>
static int launch_ctx_tc_impl(const CUtensorMap (&tm)[6], const CtxTcParams& p, cudaStream_t st) {
  static bool attr_set[TFB_MAX_DEVICES] = {false};
  auto kern = &ctx_tc_kernel<FP16, DK, MASK>;
  if (int rc = ensure_dynamic_smem(reinterpret_cast<const void*>(kern), CT_SMEM_BYTES, attr_set)) return rc;
  const int grid = p.n_items < sm_count() ? p.n_items : sm_count();
  kern<<<grid, 384, CT_SMEM_BYTES, st>>>(tm[0], tm[1], tm[2], tm[3], tm[4], tm[5], p);
  return cudaGetLastError() == cudaSuccess ? TFB_OK : TFB_ERR_LAUNCH;
}

int launch_ctx_tc(const CtxParams& c, const void* kp, long kp_ss, long kp_hs, const void* vp, long vp_ss, long vp_hs,
                  int fp16, cudaStream_t st) {
  CtxTcParams p;
  p.c = c;
  p.pack = ctx_pack(c.H / c.Hkv);
  p.n_hg = c.H / p.pack;
  p.tok = 128 / p.pack;
  p.n_qp = (c.Sq + 2 * p.tok - 1) / (2 * p.tok);
  p.n_prefix = (c.P + 127) / 128;
  const bool packed = c.cu_kv != nullptr;
  p.bmul = packed ? 0 : 1;
  const long items = ctx_tc_items(c.B, c.Sq, c.H, c.Hkv) * c.ns;
  if (items > 0x3fffffffL) return TFB_ERR_TOO_LARGE;
  p.n_items = static_cast<int>(items);
  CUtensorMap tm[6];
  const int kb = packed ? 1 : c.B;
  int e;
  if ((e = ctx_tmap(&tm[0], c.q, fp16, c.D, c.H, c.q_hs, c.Sq, c.q_ss, c.B, c.q_bs, 64, p.pack, p.tok, TM_SW_128))) return e;
  if (c.Skv > 0) {
    if ((e = ctx_tmap(&tm[1], c.k, fp16, c.D, c.Hkv, c.k_hs, c.Skv, c.k_ss, kb, c.k_bs, 64, 1, 128, TM_SW_128))) return e;
    if ((e = ctx_tmap(&tm[2], c.v, fp16, c.D, c.Hkv, c.v_hs, c.Skv, c.v_ss, kb, c.v_bs, 64, 1, 128, TM_SW_128))) return e;
  }
  if (c.P > 0) {
    if ((e = ctx_tmap(&tm[3], kp, fp16, c.D, c.Hkv, kp_hs, c.P, kp_ss, 1, 0, 64, 1, 128, TM_SW_128))) return e;
    if ((e = ctx_tmap(&tm[4], vp, fp16, c.D, c.Hkv, vp_hs, c.P, vp_ss, 1, 0, 64, 1, 128, TM_SW_128))) return e;
  } else {
    tm[3] = c.Skv > 0 ? tm[1] : tm[0], tm[4] = c.Skv > 0 ? tm[2] : tm[0];
  }
  if (c.Skv <= 0) tm[1] = tm[3], tm[2] = tm[4];
  if (c.part_o) {
    tm[5] = tm[0];
  } else if ((e = ctx_tmap(&tm[5], c.out, fp16, c.D, c.H, c.D, c.Sq, static_cast<long>(c.H) * c.D, c.B,
                           static_cast<long>(c.Sq) * c.H * c.D, 32, p.pack, 32 / p.pack, TM_SW_64))) {
    return e;
  }
  const bool mask = c.key_mask != nullptr;
#define TFB_CTX(F_, D_, M_) return launch_ctx_tc_impl<F_, D_, M_>(tm, p, st)
  if (c.D <= 64) {
    if (fp16) { if (mask) TFB_CTX(true, 64, true); TFB_CTX(true, 64, false); }
    if (mask) TFB_CTX(false, 64, true);
    TFB_CTX(false, 64, false);
  }
  if (fp16) { if (mask) TFB_CTX(true, 128, true); TFB_CTX(true, 128, false); }
  if (mask) TFB_CTX(false, 128, true);
  TFB_CTX(false, 128, false);
#undef TFB_CTX
}

}  // namespace tfb
