// Context attention for full query tiles on tcgen05: o = softmax(scale q k^T) v over the keys a sample may see - a shared
// prefix, then the sample's own keys up to its length, minus masked ones. bf16 or fp16, head_dim <= 64 / <= 128.
//
// Persistent: one CTA per SM walks over work items (sample, head group, pair of 128-row query tiles, key slice). A tile's
// rows are (token, head) pairs of one key head where the head group is a power of two, so grouped heads share every K / V
// tile; otherwise a tile is 128 tokens of one head. 512 threads:
//   warp 0   TMA loader                                   warps 4..7    softmax group 0 (query tile 0; TMEM lane == row)
//   warp 1   tcgen05.mma issuer, TMEM owner               warps 8..11   softmax group 1 (query tile 1)
//   warp 3   decodes the work items into a ring, writes   warps 12..15  output of finished tiles
//            the rows of items without keys
//   warp 2   tail / mask warp: clears the V rows that nobody may see before the P.V product reads them (a product with
//            infinities or NaN there would spread through P = 0) and turns the key mask into bit words
// TMEM (512 columns): S0 | S1 | O0 | O1. P overwrites the first 64 columns of its S tile and enters P.V from TMEM.
// Encoder states are short (a prompt is 1 .. 4 blocks of 128 keys), so the ends of an item count: the issuer starts the
// next item's Q.K^T of a tile right behind the last P.V of that tile, the loader is a whole item ahead, and normalising
// and writing a tile is the output warps' business (shared memory, then TMA stores that clip at the tensor's edge) while the
// softmax groups go on with the next item. The last block of a sample is as narrow as its keys need: 32-column steps in
// Q.K^T, the exponentials and P.V.
// The issuer is the warp that everything waits for: a P.V + Q.K^T pair takes the tensor core 1024 clk, and everything else
// that warp does comes on top, on a scheduler it shares with two softmax warps. So its one wait per tile and block covers
// P, V, the next K and the accumulator (the tail warp's arrival stands for the loads), its values are warp-uniform, and
// its view of an item is four integers. (An issuer per tile was slower, 594 for 558 us on two prompts of 512 and 183 tokens:
// the tensor core takes turns between two warps, and both tiles' chains get longer.)
//
// Measured, replayed from a graph: 2 x 3120 tokens x 32 heads of 128 against a prefix of 9360 and 3120 own keys 1130 us, 1130
// TFLOP/s, where the MMAs and their hand-overs alone take about 1000; two prompts of 512 and 183 keys under 37440 tokens x 32 heads
// 525 us, 810 TFLOP/s, where the ends of the short items (first Q.K^T, last P.V, hand-over to the output warps) leave tensor pipe and
// exponentials at 40 % each. (On a board that reached its power cap sooner 1313 and 606 us.)
// Head groups that are no power of two, or larger than 32, fill a tile with one head's tokens and read K and V once per head: 8 samples
// x 12 tokens x 3 heads per key head against 4096 keys take 121 us, with 4 heads per key head 46; 100 tokens 122 and 72. From a
// few hundred tokens on it makes no difference (1000 tokens, 3 and 4 heads: 385 and 482).
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
constexpr int CT_OUT_OFF = CT_KV_OFF + 4 * CT_TILE;  // 4 output warps x 2 boxes of [32 rows][64 channels]
constexpr int CT_ML_OFF = CT_OUT_OFF + 4 * 8192;     // [2 tiles][128 rows] of (maximum, sum)
constexpr int CT_ITEMS = 4;                          // ring of decoded items
constexpr int CT_ITEM_OFF = CT_ML_OFF + 2 * 128 * 8;
constexpr int CT_BAR_OFF = CT_ITEM_OFF + CT_ITEMS * 48;
constexpr int CT_N_BARS = 20 + 2 * CT_ITEMS;
constexpr int CT_ALIGN_SLACK = 512;  // dynamic shared memory starts on 1 KB here; the kernel checks that the tiles fit
constexpr int CT_SMEM_BYTES = CT_BAR_OFF + CT_N_BARS * 8 + 64 + CT_ALIGN_SLACK;
static_assert(CT_SMEM_BYTES <= 227 * 1024, "shared memory of one CTA");
constexpr int CT_ITEM_READERS = 3 + 8 + 4;  // loader, issuer and tail warp, softmax warps, output warps
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
  int b;           // -1: no more items
  int hg, qp, split;
  int first, len;  // the sample's own keys
  int j0, nb;      // key blocks [j0, j0 + nb) of prefix blocks followed by own blocks
  __device__ __forceinline__ bool two(const CtxTcParams& p) const { return (qp * 2 + 1) * p.tok < p.c.Sq; }
};

// First visible key of mask[0, n) and one past the last (n, 0 if there is none). Whole warp; reads from both ends inwards,
// so what lies between the ends is not read.
__device__ __forceinline__ void ctx_mask_ends(const uint8_t* mask, int n, int& lo, int& hi) {
  constexpr int STEP = 16;  // loads in flight per lane
  lo = n;
  hi = 0;
  for (int at = 0; at < n && lo == n; at += 32 * STEP) {
    int found = n;
#pragma unroll
    for (int x = 0; x < STEP; ++x) {
      const int j = at + x * 32 + static_cast<int>(lane_id());
      if (j < n && __ldg(mask + j)) found = min(found, j);
    }
    lo = __reduce_min_sync(0xffffffffu, found);
  }
  for (int at = n; at > lo && hi == 0; at -= 32 * STEP) {
    int found = 0;
#pragma unroll
    for (int x = 0; x < STEP; ++x) {
      const int j = at - 1 - (x * 32 + static_cast<int>(lane_id()));
      if (j >= lo && __ldg(mask + j)) found = max(found, j + 1);
    }
    hi = __reduce_max_sync(0xffffffffu, found);
  }
}

// Work item i; `ends` holds what the mask leaves of sample ends_b. Whole warp.
template <bool MASK>
__device__ __forceinline__ CtxItem ctx_item(const CtxTcParams& p, int i, int& ends_b, int2& ends) {
  CtxItem t;
  t.qp = i % p.n_qp;
  i /= p.n_qp;
  t.split = i % p.c.ns;
  i /= p.c.ns;
  t.hg = i % p.n_hg;
  t.b = i / p.n_hg;
  ctx_sample_range(p.c, t.b, t.first, t.len);
  int skip = 0;  // blocks in front of the first visible key
  if (MASK) {
    if (t.b != ends_b) ctx_mask_ends(p.c.key_mask + static_cast<long>(t.b) * p.c.mask_bs, t.len, ends.x, ends.y);
    ends_b = t.b;
    t.len = ends.y;
    skip = t.len > 0 ? ends.x >> 7 : 0;
  }
  const int nb = p.n_prefix + ((t.len + 127) >> 7) - skip;
  if (p.c.ns == 1) {
    t.j0 = skip, t.nb = nb;
  } else {
    t.j0 = skip + static_cast<int>(static_cast<long>(nb) * t.split / p.c.ns);
    t.nb = skip + static_cast<int>(static_cast<long>(nb) * (t.split + 1) / p.c.ns) - t.j0;
  }
  return t;
}
// Visible keys of block j, at most 128 (before the mask).
__device__ __forceinline__ int ctx_block_keys(const CtxTcParams& p, int j, int len) {
  return min(128, j < p.n_prefix ? p.c.P - j * 128 : len - (j - p.n_prefix) * 128);
}

// The ring of decoded items as one reader warp sees it. All of them have keys: the ring moves on with its slowest reader, and
// a reader that waits for the last V of an item, which is loaded beside the first K of the next, would hold up the decoder
// behind a run of items without any.
struct CtxItems {
  const int4* ring;
  uint64_t *full, *empty;
  int n;
  // Whole warp; every field comes out warp-uniform. False at the end of the work or on an abort.
  __device__ __forceinline__ bool next(CtxItem& t, const AbortCtx& ctx, int site) {
    const int slot = n % CT_ITEMS;
    if (!mbar_wait_warp(&full[slot], (n / CT_ITEMS) & 1, ctx, site)) return false;
    ++n;
    const int4 a = ring[slot * 3], b = ring[slot * 3 + 1];
    __syncwarp();
    if (lane_id() == 0) mbar_arrive(&empty[slot]);
    t.b = __shfl_sync(0xffffffffu, a.x, 0), t.hg = __shfl_sync(0xffffffffu, a.y, 0);
    t.qp = __shfl_sync(0xffffffffu, a.z, 0), t.split = __shfl_sync(0xffffffffu, a.w, 0);
    t.first = __shfl_sync(0xffffffffu, b.x, 0), t.len = __shfl_sync(0xffffffffu, b.y, 0);
    t.j0 = __shfl_sync(0xffffffffu, b.z, 0), t.nb = __shfl_sync(0xffffffffu, b.w, 0);
    return t.b >= 0;
  }
  // What the issuer needs of the next item: blocks, query tiles, the place of the prefix's last block among them
  // (or -1), and the columns of that block (low half) and of the item's last. False as above.
  __device__ __forceinline__ bool next_issue(int4& r, const AbortCtx& ctx, int site) {
    const int slot = n % CT_ITEMS;
    if (!mbar_wait_warp(&full[slot], (n / CT_ITEMS) & 1, ctx, site)) return false;
    ++n;
    if (lane_id() == 0) {
      r = ring[slot * 3 + 2];
      mbar_arrive(&empty[slot]);
    }
    r.x = __shfl_sync(0xffffffffu, r.x, 0), r.y = __shfl_sync(0xffffffffu, r.y, 0);
    r.z = __shfl_sync(0xffffffffu, r.z, 0), r.w = __shfl_sync(0xffffffffu, r.w, 0);
    return r.x > 0;
  }
};

// The part that both score tile forms share: raises the row maximum when it grew by more than 2^8 (or at the first tile),
// taking the accumulator and the sum along. All MMAs issued before this tile's scores have completed, so O is stable.
template <int DK>
__device__ __forceinline__ void ctx_new_max(uint32_t tmem_o, float m_new, bool first, float& m_used, float& l) {
  if (first) {
    m_used = m_new;
  } else if (__any_sync(0xffffffffu, (m_new - m_used) > CT_RESCALE_THRESHOLD)) {
    const float alpha = ctx_rescale(m_used, m_new);
    m_used = m_new;
    l *= alpha;
#pragma unroll 1
    for (int c = 0; c < DK / 32; ++c) {
      uint32_t o[32];
      tmem_ld_32x32(tmem_o + c * 32, o);
      tmem_ld_wait();
#pragma unroll
      for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
      tmem_st_32x32(tmem_o + c * 32, o);
    }
  }
}

// p = 2^(s scale - m) of 32 columns, added up in ps and packed into TMEM: packed fp32x2 FMAs and row sums.
template <bool FP16>
__device__ __forceinline__ void ctx_exp32(const uint32_t (&s)[32], uint32_t tmem_p, uint64_t scale2, uint64_t negm2,
                                          uint64_t (&ps)[4]) {
  uint32_t pk[16];
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    const uint64_t x2 = f2_fma(f2_pack(__uint_as_float(s[2 * k]), __uint_as_float(s[2 * k + 1])), scale2, negm2);
    float x0, x1;
    f2_unpack(x2, x0, x1);
    const float p0 = fast_exp2(x0), p1 = fast_exp2(x1);
    ps[k & 3] = f2_add(ps[k & 3], f2_pack(p0, p1));
    pk[k] = ctx_pack2<FP16>(p0, p1);
  }
  tmem_st_32x16(tmem_p, pk);
}
__device__ __forceinline__ float ctx_sum(const uint64_t (&ps)[4]) {
  float a0, a1, b0, b1;
  f2_unpack(f2_add(ps[0], ps[1]), a0, a1);
  f2_unpack(f2_add(ps[2], ps[3]), b0, b1);
  return (a0 + a1) + (b0 + b1);
}

// A full 128 x 128 score tile: scores from TMEM to registers, maximum, exponentials, P back over the scores.
template <bool FP16, int DK>
__device__ __forceinline__ void ctx_softmax_full(uint32_t tmem_s, uint32_t tmem_o, float scale_log2, bool first, float& m_used,
                                                 float& l) {
  uint32_t s[4][32];
#pragma unroll
  for (int c = 0; c < 4; ++c) tmem_ld_32x32(tmem_s + c * 32, s[c]);
  tmem_ld_wait();
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
  ctx_new_max<DK>(tmem_o, fmaxf(m_used, mx * scale_log2), first, m_used, l);
  const float neg = -ctx_exp_base(m_used);
  uint64_t ps[4] = {0ull, 0ull, 0ull, 0ull};
#pragma unroll
  for (int c = 0; c < 4; ++c)
    ctx_exp32<FP16>(s[c], tmem_s + c * 16, f2_pack(scale_log2, scale_log2), f2_pack(neg, neg), ps);
  l += ctx_sum(ps);
}

// A narrow tile (32-column steps) or one with hidden keys (their bits in `words` are clear): 32 columns at a time, the
// scores read from TMEM once for the maximum and once for the exponentials, which keeps the registers of the full form
// to itself. P of step c overwrites columns that steps <= c have read.
template <bool FP16, int DK, bool MASK>
__device__ __forceinline__ void ctx_softmax_part(uint32_t tmem_s, uint32_t tmem_o, float scale_log2, int keys,
                                                 volatile const uint32_t* words, bool first, float& m_used, float& l) {
  const int chunks = (keys + 31) >> 5;
  uint32_t s[32];
  auto load = [&](int c) {
    tmem_ld_32x32(tmem_s + c * 32, s);
    const int left = keys - c * 32;
    const uint32_t vis = (MASK ? words[c] : 0xffffffffu) & (left >= 32 ? 0xffffffffu : (1u << left) - 1u);
    tmem_ld_wait();
    if (vis != 0xffffffffu) {
#pragma unroll
      for (int e = 0; e < 32; ++e)
        if (!((vis >> e) & 1)) s[e] = 0xff800000u;  // -inf
    }
  };
  float mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll 1
  for (int c = 0; c < chunks; ++c) {
    load(c);
#pragma unroll
    for (int e = 0; e < 32; e += 4) {
      mx0 = fmax3(mx0, __uint_as_float(s[e]), __uint_as_float(s[e + 1]));
      mx1 = fmax3(mx1, __uint_as_float(s[e + 2]), __uint_as_float(s[e + 3]));
    }
  }
  ctx_new_max<DK>(tmem_o, fmaxf(m_used, fmaxf(mx0, mx1) * scale_log2), first, m_used, l);
  const float neg = -ctx_exp_base(m_used);
  uint64_t ps[4] = {0ull, 0ull, 0ull, 0ull};
#pragma unroll 1
  for (int c = 0; c < chunks; ++c) {
    load(c);
    ctx_exp32<FP16>(s, tmem_s + c * 16, f2_pack(scale_log2, scale_log2), f2_pack(neg, neg), ps);
  }
  l += ctx_sum(ps);
}

// An item without keys: zero rows and -inf, in its slot where the key range is split. Whole warp.
__device__ __noinline__ void ctx_no_keys(const CtxTcParams& p, const CtxItem& t) {
  const int pieces = p.c.D >> 3;  // 16 bytes each
  for (int x = lane_id(); x < 256 * pieces; x += 32) {
    const int row = x / pieces, piece = x - row * pieces;
    const int tok = t.qp * 2 * p.tok + row / p.pack, head = t.hg * p.pack + row % p.pack;
    if (tok >= p.c.Sq) break;
    const long token = static_cast<long>(t.b) * p.c.Sq + tok;
    if (p.c.part_o) {
      const long at = (static_cast<long>(p.c.slot0 + t.split) * p.c.B * p.c.Sq + token) * p.c.H + head;
      if (piece == 0) p.c.part_lse[at] = -INFINITY;
      float4* o = reinterpret_cast<float4*>(p.c.part_o + at * p.c.D) + piece * 2;
      o[0] = o[1] = make_float4(0.f, 0.f, 0.f, 0.f);
      continue;
    }
    reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.c.out) + (token * p.c.H + head) * p.c.D)[piece] = make_uint4(0, 0, 0, 0);
    if (p.c.lse && piece == 0) p.c.lse[(static_cast<long>(t.b) * p.c.H + head) * p.c.Sq + tok] = -INFINITY;
  }
}

template <bool FP16, int DK, bool MASK>
__global__ void __launch_bounds__(512, 1)
    ctx_tc_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                  const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmKp,
                  const __grid_constant__ CUtensorMap tmVp, const __grid_constant__ CUtensorMap tmO,
                  const __grid_constant__ CtxTcParams p) {
  constexpr int NBOX = DK / 64;
  constexpr uint32_t LOAD_BYTES = NBOX * CT_BOX;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  if (smem - smem_raw > CT_ALIGN_SLACK) {  // same verdict in every thread
    if (threadIdx.x == 0 && p.c.status) atomicCAS(p.c.status, 0, TFB_ERR_TOO_LARGE | (62 << 8));
    return;
  }
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + CT_BAR_OFF);
  uint64_t* q_full = bars + 0;     // [2] per query tile
  uint64_t* q_empty = bars + 2;    // [2]
  uint64_t* kv_full = bars + 4;    // [2] stage s, in slot s & 1: K of key block s and V of block s - 1
  uint64_t* kv_ready = bars + 6;   // [2] MASK: the mask words of block s - 1 are written
  uint64_t* kv_empty = bars + 8;   // [2]
  uint64_t* s_full = bars + 10;    // [2] per query tile
  uint64_t* p_ready = bars + 12;   // [2] P is written (softmax group), V and the next K are there (tail warp)
  uint64_t* o_final = bars + 14;   // [2] the tile's last P.V is done
  uint64_t* l_full = bars + 16;    // [2] the tile's maxima and sums are in shared memory
  uint64_t* o_empty = bars + 18;   // [2] accumulator, maxima and sums have been read
  uint64_t* i_full = bars + 20;    // [CT_ITEMS]
  uint64_t* i_empty = i_full + CT_ITEMS;
  uint32_t* words = reinterpret_cast<uint32_t*>(bars + CT_N_BARS);  // [2 slots][4]
  uint32_t* tmem_slot = words + 8;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float2* ml = reinterpret_cast<float2*>(smem + CT_ML_OFF);

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
  const int lane = threadIdx.x & 31;
  AbortCtx ctx{abort_flag, p.c.status};

  if (threadIdx.x == 0) {
    for (int s = 0; s < 2; ++s) {
      mbar_init(&q_full[s], 1);
      mbar_init(&q_empty[s], 1);
      mbar_init(&kv_full[s], 1);
      mbar_init(&kv_ready[s], 1);
      mbar_init(&kv_empty[s], 1);
      mbar_init(&s_full[s], 1);
      mbar_init(&p_ready[s], 129);
      mbar_init(&o_final[s], 1);
      mbar_init(&l_full[s], 128);
      mbar_init(&o_empty[s], 4);
    }
    for (int s = 0; s < CT_ITEMS; ++s) {
      mbar_init(&i_full[s], 1);
      mbar_init(&i_empty[s], CT_ITEM_READERS);
    }
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  CtxItems items{reinterpret_cast<const int4*>(smem + CT_ITEM_OFF), i_full, i_empty, 0};
  CtxItem t;

  // Registers move only inside the launch allocation of 512 x 128; these shares spill least (16 bytes).
  static_assert(256 * 176 + 128 * 88 + 128 * 72 <= 512 * 128, "setmaxnreg split");
  if (warp >= 12) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    // ------------------------------ output warps ------------------------------
    const int wq = warp & 3;
    const int row = wq * 32 + lane;
    const uint32_t lane_addr = static_cast<uint32_t>(wq * 32) << 16;
    uint8_t* stage = smem + CT_OUT_OFF + wq * 8192;
    const int row_tok = row / p.pack, row_head = row % p.pack;
    uint32_t o_phase = 0;  // bit per query tile
    int n_box = 0;
    bool ok = true;
    while (ok && items.next(t, ctx, 55)) {
      for (int st = 0; st < (t.two(p) ? 2 : 1); ++st) {
        const int tile_tok = (t.qp * 2 + st) * p.tok;
        const int tok = tile_tok + row_tok, head = t.hg * p.pack + row_head;
        const bool row_ok = tok < p.c.Sq;
        if (!(ok = mbar_wait_warp(&l_full[st], (o_phase >> st) & 1, ctx, 56))) break;
        const float2 m_l = ml[st * 128 + row];
        const float inv = ctx_inverse(m_l.y);
        if (row_ok && (p.c.part_o || p.c.lse)) {
          const float lse2 = ctx_lse2(m_l.x, m_l.y);
          if (p.c.part_o)
            p.c.part_lse[((static_cast<long>(p.c.slot0 + t.split) * p.c.B + t.b) * p.c.Sq + tok) * p.c.H + head] = lse2;
          else
            p.c.lse[(static_cast<long>(t.b) * p.c.H + head) * p.c.Sq + tok] = lse2 * 0.6931471805599453f;
        }
        if (!(ok = mbar_wait_warp(&o_final[st], (o_phase >> st) & 1, ctx, 57))) break;
        o_phase ^= 1u << st;
        tc_fence_after();
        const uint32_t tmem_o = tmem_base + lane_addr + 256 + st * 128;
        if (p.c.part_o) {
          const long at = ((static_cast<long>(p.c.slot0 + t.split) * p.c.B + t.b) * p.c.Sq + tok) * p.c.H + head;
          for (int c = 0; c < DK / 16; ++c) {
            uint32_t o[16];
            tmem_ld_32x16(tmem_o + c * 16, o);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 16; e += 4)
              if (row_ok && c * 16 + e < p.c.D)
                *reinterpret_cast<float4*>(p.c.part_o + at * p.c.D + c * 16 + e) =
                    make_float4(__uint_as_float(o[e]) * inv, __uint_as_float(o[e + 1]) * inv,
                                __uint_as_float(o[e + 2]) * inv, __uint_as_float(o[e + 3]) * inv);
          }
        } else {
          const int first_tok = tile_tok + wq * 32 / p.pack;
          const uint64_t inv2 = f2_pack(inv, inv);
#pragma unroll
          for (int x = 0; x < NBOX; ++x) {
            if (x * 64 < p.c.D) {
              if (lane == 0) tma_store_wait_read1();  // the box before the last has left this buffer
              __syncwarp();
              uint8_t* buf = stage + (n_box++ & 1) * 4096;
#pragma unroll
              for (int c = 0; c < 2; ++c) {
                uint32_t o[32];
                tmem_ld_32x32(tmem_o + x * 64 + c * 32, o);
                tmem_ld_wait();
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                  uint4 v;
#pragma unroll
                  for (int e = 0; e < 4; ++e) {
                    float a, b;
                    f2_unpack(f2_mul(f2_pack(__uint_as_float(o[y * 8 + e * 2]), __uint_as_float(o[y * 8 + e * 2 + 1])), inv2), a, b);
                    (&v.x)[e] = ctx_pack2<FP16>(a, b);
                  }
                  *reinterpret_cast<uint4*>(buf + lane * 128 + (((c * 4 + y) ^ (lane & 7)) << 4)) = v;  // 128B swizzle
                }
              }
              fence_proxy_async_smem();
              __syncwarp();
              if (lane == 0) {
                if (first_tok < p.c.Sq) tma_store_4d(&tmO, buf, x * 64, t.hg * p.pack, first_tok, t.b);
                tma_store_commit();
              }
            }
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&o_empty[st]);
      }
    }
    if (lane == 0) tma_store_wait_all();
    __syncwarp();
  } else if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (warp == 0) {
      // ------------------------------ TMA loader ------------------------------
      const bool leader = lane == 0;
      if (leader) {
        tma_prefetch_desc(&tmQ);
        tma_prefetch_desc(&tmK);
        tma_prefetch_desc(&tmV);
      }
      int g = 0;             // key blocks so far
      uint32_t q_phase = 3;  // bit per query tile; a barrier that was never used lets its first waiter through
      int v_row = 0, v_b = 0, v_hk = 0;
      bool v_pre = false, ok = true;
      auto load = [&](const CUtensorMap* tm, int off, uint64_t* bar, int hk, int row, int b) {
        for (int x = 0; x < NBOX; ++x) tma_load_4d(smem + off + x * CT_BOX, tm, bar, x * 64, hk, row, b);
      };
      while (ok && items.next(t, ctx, 40)) {
        const int hk = t.hg * p.pack / (p.c.H / p.c.Hkv);
        for (int n = 0; n < t.nb; ++n, ++g) {
          const int j = t.j0 + n;
          const bool pre = j < p.n_prefix;
          const int row = pre ? j * 128 : t.first + (j - p.n_prefix) * 128;
          const int bb = pre ? 0 : t.b * p.bmul;
          const int slot = g & 1;  // stage g
          if (!(ok = mbar_wait_warp(&kv_empty[slot], ((g >> 1) & 1) ^ 1, ctx, 41))) break;
          if (leader) {
            mbar_expect_tx(&kv_full[slot], (g > 0 ? 2 : 1) * LOAD_BYTES);
            if (g > 0) load(v_pre ? &tmVp : &tmV, CT_KV_OFF + (2 + slot) * CT_TILE, &kv_full[slot], v_hk, v_row, v_b);
            load(pre ? &tmKp : &tmK, CT_KV_OFF + slot * CT_TILE, &kv_full[slot], hk, row, bb);
          }
          v_pre = pre, v_hk = hk, v_row = row, v_b = bb;
          if (n == 0) {
            for (int st = 0; st < (t.two(p) ? 2 : 1); ++st) {
              if (!(ok = mbar_wait_warp(&q_empty[st], (q_phase >> st) & 1, ctx, 42))) break;
              q_phase ^= 1u << st;
              if (leader) {
                mbar_expect_tx(&q_full[st], LOAD_BYTES);
                load(&tmQ, CT_Q_OFF + st * CT_TILE, &q_full[st], t.hg * p.pack, (t.qp * 2 + st) * p.tok, t.b);
              }
            }
            if (!ok) break;
          }
          __syncwarp();
        }
      }
      if (ok && g > 0) {  // the last block's V has no K beside it
        const int slot = g & 1;
        if (mbar_wait_warp(&kv_empty[slot], ((g >> 1) & 1) ^ 1, ctx, 43) && leader) {
          mbar_expect_tx(&kv_full[slot], LOAD_BYTES);
          load(v_pre ? &tmVp : &tmV, CT_KV_OFF + (2 + slot) * CT_TILE, &kv_full[slot], v_hk, v_row, v_b);
        }
        __syncwarp();
      }
    } else if (warp == 1) {
      // ------------------------------ MMA issuer ------------------------------
      constexpr uint32_t FMT = FP16 ? 0 : 1;
      constexpr uint32_t idesc_pv = make_idesc(128, DK, FMT, FMT, 0, 1);  // B (= V) is MN-major
      // A descriptor holds its address in units of 16 bytes in the low bits, so tiles and k-steps are reached by addition.
      // The high words (row-group stride, swizzle) of all of them are the same constant.
      const uint32_t q_desc = static_cast<uint32_t>(make_desc_k_sw128(smem_u32(smem + CT_Q_OFF)));
      const uint32_t k_desc = static_cast<uint32_t>(make_desc_k_sw128(smem_u32(smem + CT_KV_OFF)));
      const uint32_t v_desc = static_cast<uint32_t>(make_desc_mn_sw128(smem_u32(smem + CT_KV_OFF + 2 * CT_TILE), CT_BOX));
      auto desc = [](uint32_t low) { return (make_desc_k_sw128(0) & 0xffffffff00000000ull) | low; };
      int g = 0;
      uint32_t q_phase = 0, p_phase = 0;  // bit per query tile
      bool ok = true;
      // one lane: Q.K^T of `cols` columns of ring block gg into S of query tile st; `last`: the item's last block
      auto issue_qk = [&](int st, int gg, int cols, bool last) {
        const uint32_t idesc = make_idesc(128, 0, FMT, FMT, 0, 0) | (static_cast<uint32_t>(cols >> 3) << 17);
        const uint32_t qd = q_desc + st * (CT_TILE >> 4), kd = k_desc + (gg & 1) * (CT_TILE >> 4);
        const uint32_t d = tmem_base + st * 128;
#pragma unroll
        for (int kk = 0; kk < DK / 16; ++kk) {
          const uint32_t off = ((kk >> 2) * CT_BOX + (kk & 3) * 32) >> 4;
          umma_f16_ss(d, desc(qd + off), desc(kd + off), idesc, kk ? 1u : 0u);
        }
        umma_commit(&s_full[st]);
        if (last) umma_commit(&q_empty[st]);
      };
      auto cols_of = [](const int4& r, int n) { return n == r.z ? r.w & 0xffff : n + 1 == r.x ? r.w >> 16 : 128; };
      // First scores of an item; its K is already there.
      auto prime = [&](int st, const int4& r, int gg) {
        if (!mbar_wait_warp(&q_full[st], (q_phase >> st) & 1, ctx, 45)) return false;
        q_phase ^= 1u << st;
        tc_fence_after();
        if (elect_one()) issue_qk(st, gg, cols_of(r, 0), r.x == 1);
        return true;
      };
      int4 t = make_int4(0, 0, 0, 0), nt = t;
      bool have = items.next_issue(t, ctx, 44);
      if (have) {
        ok = mbar_wait_warp(&kv_full[0], 0, ctx, 46) && prime(0, t, 0) && (t.y == 1 || prime(1, t, 0));
        if (ok && elect_one()) umma_commit(&kv_empty[0]);
      }
      while (have && ok) {
        const int gn = g + t.x, tiles = t.y;
        bool have_next = false;
        int cols = cols_of(t, 0);
        for (int n = 0; n < t.x; ++n, ++g) {
          const bool more = n + 1 < t.x;
          const int steps = cols >> 4;
          if (more) cols = cols_of(t, n + 1);
          const int slot = (g + 1) & 1;  // stage g + 1: V of this block and K of the next
          const uint32_t vd = v_desc + slot * (CT_TILE >> 4);
          for (int st = 0; st < tiles; ++st) {
            // P of this block is written, its V and the next K are there, the tile's previous accumulator has been read
            if (!(ok = mbar_wait_warp(&p_ready[st], (p_phase >> st) & 1, ctx, 49))) break;
            p_phase ^= 1u << st;
            tc_fence_after();
            if (elect_one()) {
              const uint32_t o_tmem = tmem_base + 256 + st * 128, p_tmem = tmem_base + st * 128;
              if (steps == 8) {
#pragma unroll
                for (int kk = 0; kk < 8; ++kk)
                  umma_f16_ts(o_tmem, p_tmem + kk * 8, desc(vd + kk * (2048 >> 4)), idesc_pv, kk ? 1u : n ? 1u : 0u);
              } else {
                for (int kk = 0; kk < steps; ++kk)
                  umma_f16_ts(o_tmem, p_tmem + kk * 8, desc(vd + kk * (2048 >> 4)), idesc_pv, (kk | n) ? 1u : 0u);
              }
              if (more)
                issue_qk(st, g + 1, cols, n + 2 == t.x);
              else
                umma_commit(&o_final[st]);
            }
            __syncwarp();
            // The next item is looked up behind an item's first products, while the tensor core works on them.
            if (st == 0 && n == 0) have_next = items.next_issue(nt, ctx, 44);
            if (!more && have_next && st < nt.y && !(ok = prime(st, nt, gn))) break;
          }
          if (ok && !more && have_next && tiles < nt.y) ok = prime(1, nt, gn);
          if (!ok) break;
          if (elect_one()) umma_commit(&kv_empty[slot]);
          __syncwarp();
        }
        have = have_next;
        t = nt;
      }
    } else if (warp == 2) {
      // ------------------------------ tail / mask warp ------------------------------
      int g = 0;
      uint32_t p_phase = 3;  // bit per query tile
      bool ok = true;
      while (ok && items.next(t, ctx, 52)) {
        // mask bytes of the item's block n, this lane's four keys; loaded one block ahead of their use
        auto load_mask = [&](int n, uint8_t (&m)[4]) {
          const int j = t.j0 + n, keys = ctx_block_keys(p, j, t.len);
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            m[x] = 0;
            if (x * 32 + lane < keys)
              m[x] = __ldg(p.c.key_mask + static_cast<long>(t.b) * p.c.mask_bs + j * 128L + x * 32 + lane);
          }
        };
        uint8_t m[4];
        if (MASK) load_mask(0, m);
        for (int n = 0; n < t.nb; ++n) {
          // Stage 0 has no V and no words, but its load is waited for all the same: nothing orders it before that of stage 1, and
          // until it is complete the parity that stage 2 waits for in this slot is that of a barrier that was never used.
          if (g == 0 && !(ok = mbar_wait_warp(&kv_full[0], 0, ctx, 51))) break;
          if (MASK && g == 0 && lane == 0) mbar_arrive(&kv_ready[0]);
          ++g;  // the stage with this block's V
          const int slot = g & 1;
          const int keys = ctx_block_keys(p, t.j0 + n, t.len);
          uint32_t w[4];
          if (MASK) {
#pragma unroll
            for (int x = 0; x < 4; ++x) w[x] = __ballot_sync(0xffffffffu, m[x] != 0);
            if (n + 1 < t.nb) load_mask(n + 1, m);
          }
          if (!(ok = mbar_wait_warp(&kv_full[slot], (g >> 1) & 1, ctx, 53))) break;
          bool wrote = false;
          if (MASK || keys < 128) {
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const int left = keys - x * 32;
              const uint32_t vis = MASK ? w[x] : left >= 32 ? 0xffffffffu : left <= 0 ? 0u : (1u << left) - 1u;
              if (left > 0 && vis != 0xffffffffu) {  // steps without a key are not read
                wrote = true;
                if (!((vis >> lane) & 1)) {
                  uint4* row = reinterpret_cast<uint4*>(smem + CT_KV_OFF + (2 + slot) * CT_TILE + (x * 32 + lane) * 128);
#pragma unroll
                  for (int y = 0; y < NBOX; ++y)
#pragma unroll
                    for (int e = 0; e < 8; ++e) row[y * (CT_BOX / 16) + e] = make_uint4(0, 0, 0, 0);
                }
              }
              if (MASK && lane == x) words[slot * 4 + x] = vis;
            }
          }
          if (wrote) fence_proxy_async_smem();
          __syncwarp();
          if (MASK && lane == 0) mbar_arrive(&kv_ready[slot]);
          // one arrival per tile and block: the phase of the block before has to be over
          for (int st = 0; st < (t.two(p) ? 2 : 1); ++st) {
            if (!(ok = mbar_wait_warp(&p_ready[st], (p_phase >> st) & 1, ctx, 62))) break;
            p_phase ^= 1u << st;
            if (lane == 0) mbar_arrive(&p_ready[st]);
          }
          if (!ok) break;
        }
      }
    } else if (warp == 3) {
      // ------------------------------ item decoder ------------------------------
      int4* ring = reinterpret_cast<int4*>(smem + CT_ITEM_OFF);
      int n = 0, ends_b = -1;
      int2 ends = make_int2(0, 0);
      for (int i = blockIdx.x;; i += gridDim.x) {
        const bool end = i >= p.n_items;
        if (!end) {
          t = ctx_item<MASK>(p, i, ends_b, ends);
          if (t.nb == 0) {
            ctx_no_keys(p, t);
            continue;
          }
        } else {
          t.b = -1, t.hg = t.qp = t.split = t.first = t.len = t.j0 = t.nb = 0;
        }
        const int slot = n % CT_ITEMS;
        if (!mbar_wait_warp(&i_empty[slot], ((n / CT_ITEMS) & 1) ^ 1, ctx, 54)) break;
        if (lane == 0) {
          ring[slot * 3] = make_int4(t.b, t.hg, t.qp, t.split);
          ring[slot * 3 + 1] = make_int4(t.first, t.len, t.j0, t.nb);
          const int cut = p.n_prefix - 1 - t.j0;  // the prefix's last block, if it is among the item's
          const int cut_cols = (ctx_block_keys(p, p.n_prefix - 1, t.len) + 31) & ~31;
          const int last_cols = (ctx_block_keys(p, t.j0 + t.nb - 1, t.len) + 31) & ~31;
          ring[slot * 3 + 2] = make_int4(end ? -1 : t.nb, t.two(p) ? 2 : 1, p.n_prefix > 0 && cut >= 0 && cut < t.nb ? cut : -1,
                                         (cut_cols & 0xffff) | last_cols << 16);
          mbar_arrive(&i_full[slot]);
        }
        ++n;
        if (end) break;
        __syncwarp();
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 176;");
    // ------------------------------ softmax groups ------------------------------
    const int st = (warp >> 2) - 1;
    const int row = (warp & 3) * 32 + lane;
    const uint32_t lane_addr = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t tmem_s = tmem_base + lane_addr + st * 128;
    const uint32_t tmem_o = tmem_base + lane_addr + 256 + st * 128;
    int ns = 0, no = 0, g = 0;  // score tiles, items with keys and key blocks seen so far
    bool ok = true;
    while (ok && items.next(t, ctx, 58)) {
      if (st && !t.two(p)) {
        g += t.nb;
        continue;
      }
      float m_used = -INFINITY, l = 0.f;
      for (int n = 0; n < t.nb; ++n, ++g) {
        const int keys = ctx_block_keys(p, t.j0 + n, t.len);
        if (!(ok = mbar_wait_warp(&s_full[st], ns & 1, ctx, 59))) break;
        ++ns;
        tc_fence_after();
        bool part = keys < 128;
        volatile const uint32_t* w = words + ((g + 1) & 1) * 4;
        if (MASK) {
          // Behind s_full: the scores of block g follow its K, which came with the V of block g - 1 behind the words of block
          // g - 2, so the parity of stage g + 1 cannot be mistaken for that of stage g - 3 by a group that skipped items.
          if (!(ok = mbar_wait_warp(&kv_ready[(g + 1) & 1], ((g + 1) >> 1) & 1, ctx, 60))) break;
          part = part || (w[0] & w[1] & w[2] & w[3]) != 0xffffffffu;
        }
        if (part)
          ctx_softmax_part<FP16, DK, MASK>(tmem_s, tmem_o, p.c.scale_log2, keys, w, n == 0, m_used, l);
        else
          ctx_softmax_full<FP16, DK>(tmem_s, tmem_o, p.c.scale_log2, n == 0, m_used, l);
        tmem_st_wait();
        tc_fence_before();
        if (n == 0) {  // accumulator, maxima and sums of the previous item have been read
          if (!(ok = mbar_wait_warp(&o_empty[st], (no & 1) ^ 1, ctx, 61))) break;
          ++no;
        }
        mbar_arrive(&p_ready[st]);
      }
      if (!ok) break;
      ml[st * 128 + row] = make_float2(m_used, l);
      mbar_arrive(&l_full[st]);
    }
  }

  if (*abort_flag) __nanosleep(200000);
  tc_fence_before();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem_base, 512);
}

static int ctx_pack(int G) { return (G & (G - 1)) == 0 && G <= 32 ? G : 1; }

long ctx_tc_items(int B, int Sq, int H, int Hkv) {
  const int pack = ctx_pack(H / Hkv), tok = 128 / pack;
  return static_cast<long>(B) * (H / pack) * ((Sq + 2 * tok - 1) / (2 * tok));
}

template <bool FP16, int DK, bool MASK>
static int launch_ctx_tc_impl(const CUtensorMap (&tm)[6], const CtxTcParams& p, cudaStream_t st) {
  static bool attr_set[TFB_MAX_DEVICES] = {false};
  auto kern = &ctx_tc_kernel<FP16, DK, MASK>;
  if (int rc = ensure_dynamic_smem(reinterpret_cast<const void*>(kern), CT_SMEM_BYTES, attr_set)) return rc;
  const int grid = p.n_items < sm_count() ? p.n_items : sm_count();
  kern<<<grid, 512, CT_SMEM_BYTES, st>>>(tm[0], tm[1], tm[2], tm[3], tm[4], tm[5], p);
  return cudaGetLastError() == cudaSuccess ? TFB_OK : TFB_ERR_LAUNCH;
}

int launch_ctx_tc(const CtxParams& c, int fp16, cudaStream_t st) {
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
  // An item takes about 2 us per 128 keys, and the output warps wait for all of it: well inside their bounded wait (0.8 s).
  if ((static_cast<long>(c.Skv) + c.P) / c.ns > (1L << 24)) return TFB_ERR_TOO_LARGE;
  // Nor may the decoder keep the other warps waiting: it passes over the masks of samples that see nothing at about 512 bytes a
  // microsecond, and one CTA may meet those of all samples in a row.
  if (c.key_mask && static_cast<long>(c.B) * c.Skv > (1L << 27)) return TFB_ERR_TOO_LARGE;
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
    if ((e = ctx_tmap(&tm[3], c.kp, fp16, c.D, c.Hkv, c.kp_hs, c.P, c.kp_ss, 1, 0, 64, 1, 128, TM_SW_128))) return e;
    if ((e = ctx_tmap(&tm[4], c.vp, fp16, c.D, c.Hkv, c.vp_hs, c.P, c.vp_ss, 1, 0, 64, 1, 128, TM_SW_128))) return e;
  } else {
    tm[3] = c.Skv > 0 ? tm[1] : tm[0], tm[4] = c.Skv > 0 ? tm[2] : tm[0];
  }
  if (c.Skv <= 0) tm[1] = tm[3], tm[2] = tm[4];
  if (c.part_o) {
    tm[5] = tm[0];
  } else if ((e = ctx_tmap(&tm[5], c.out, fp16, c.D, c.H, c.D, c.Sq, static_cast<long>(c.H) * c.D, c.B,
                           static_cast<long>(c.Sq) * c.H * c.D, 64, p.pack, 32 / p.pack, TM_SW_128))) {
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

