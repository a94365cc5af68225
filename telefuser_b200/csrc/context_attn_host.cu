// C entry points of context attention: argument checks, the choice of kernels and key splits.
//
// Rows kernel (context_attn_rows.cu) when a sample has at most 32 query rows per key head; otherwise the short-state kernel
// (context_attn_short.cu) up to 64 key rows in all and the tensor-memory kernel (context_attn_tc.cu) beyond. Both sides of the
// limit, 8 key heads, bf16, us in the rows kernel and in the one that would run without it:
//            head dim 64                                          head dim 128
//   keys     B  1: 1 row     17 rows    32 rows                   1 row       17 rows    32 rows
//   128      4.2 / 7.6       6.0 / 7.6    6.6 / 7.4                4.8 / 8.3     7.9 / 8.3    9.3 / 8.4
//   2048     9.8 / 12.1     13.4 / 12.5  14.0 / 12.4              11.5 / 13.0   16.9 / 13.2  18.7 / 13.1
//   32768   16.9 / 31.9     24.4 / 32.5  25.5 / 32.6              29.8 / 45.3   37.1 / 45.5  38.3 / 44.1
//            B 64
//   128      8.3 / 16.9     13.0 / 16.9  14.6 / 16.8              10.2 / 19.8   18.6 / 19.8  22.8 / 19.9
//   2048    52.2 / 103      77.1 / 104   79.9 / 104               80.9 / 126     101 / 126    107 / 126
//   8192     177 / 378       258 / 378    262 / 378                301 / 463     348 / 474    368 / 504
// The limit is right where the call takes long; below 15 us it costs up to 30 % with more than 16 rows, and up to 64 keys the
// short-state kernel would be faster for 16 rows and more (32 keys, 16 and 32 rows of B 64 at head dim 64: 8.1 / 4.5 and
// 12.1 / 4.7; 1 row of B 1 at head dim 128: 3.9 / 4.6).
// A shared prefix is visited as the first keys of every sample while re-reading it costs little: always when a sample fills a
// query tile, and below that while the batch's re-reads stay small enough for L2. Otherwise it is computed once for all
// samples - their tokens form one batch entry - as slots of its own, the samples' own keys as further slots, and the join
// adds them up: two more launches, which 16 MB of re-reads cost about as much as (a prefix of 77 keys under 3 samples: 5 us
// together, 14 apart; 64 samples of 4 rows each under 16384 keys, 4 GB of re-reads: 82 us apart).
#include "context_attn.cuh"

using namespace tfb;

namespace {

constexpr int CTX_MAX_SPLITS = 64;
constexpr long CTX_REREAD_BYTES = 16 << 20;

struct CtxPlan {
  bool apart;          // prefix in slots of its own
  int ns_prefix, ns;   // key splits of the prefix pass and of the (only or own-keys) pass
  bool rows_prefix, rows_own;
  bool short_own;      // at most 64 key rows in all and no prefix: context_attn_short.cu
  int slots() const { return (apart ? ns_prefix : 0) + ns; }
};

bool few_rows(long tokens, int H, int Hkv) { return tokens * (H / Hkv) <= CTX_FEW_ROWS; }

// Splits of the key range so that few items still fill the device: two CTAs per SM for the rows kernel (two are
// resident), one per SM for the tensor-memory kernel. A slice has no fewer than 512 and 256 keys: below that the join and
// its launch cost more than the slice saves (one token of 8 streams against 512 keys: 8.0 us in two slices and a join).
int pick_splits(bool rows, int B, long Sq, int H, int Hkv, long keys) {
  const long sms = sm_count();
  const long items = rows ? static_cast<long>(B) * Hkv : ctx_tc_items(B, static_cast<int>(Sq), H, Hkv);
  long ns = (rows ? 2 * sms : sms) / (items > 0 ? items : 1);
  const long most = keys / (rows ? 512 : 256);
  if (ns > most) ns = most;
  if (ns > CTX_MAX_SPLITS) ns = CTX_MAX_SPLITS;
  return ns < 1 ? 1 : static_cast<int>(ns);
}

int check(const tfb_context_attn_args* a) {
  if (!a || a->B < 0 || a->Sq < 0 || a->H < 1 || a->Hkv < 1 || a->H % a->Hkv || a->D < 8 || a->D > 128 || a->D % 8 ||
      a->Skv < 0 || a->P < 0 || !(a->scale > 0.f))
    return TFB_ERR_BAD_SHAPE;
  if ((a->cu_kv && (a->kv_lens || a->key_mask)) || (a->P && (a->cu_kv || a->key_mask))) return TFB_ERR_BAD_SHAPE;
  if (a->Sq > (1 << 30) || a->Skv > (1 << 30) || a->P > (1 << 30)) return TFB_ERR_TOO_LARGE;
  return TFB_OK;
}

CtxPlan make_plan(const tfb_context_attn_args* a) {
  CtxPlan pl;
  const int G = a->H / a->Hkv;
  const long reread = 4L * a->P * a->Hkv * a->D * (a->B - 1);  // bytes of K and V
  pl.apart = a->P > 0 && a->B > 1 && static_cast<long>(a->Sq) * G < 128 && reread > CTX_REREAD_BYTES;
  pl.rows_own = few_rows(a->Sq, a->H, a->Hkv);
  const long tokens = static_cast<long>(a->B) * a->Sq;
  pl.rows_prefix = few_rows(tokens, a->H, a->Hkv);
  pl.short_own = !pl.rows_own && a->P == 0 && a->Skv <= CTX_SHORT_KEYS;
  // Packed samples: the longest may hold every row.
  const long keys = a->Skv + (pl.apart ? 0 : a->P);
  pl.ns = pl.short_own ? 1 : pick_splits(pl.rows_own, a->B, a->Sq, a->H, a->Hkv, keys);
  pl.ns_prefix = pl.apart ? pick_splits(pl.rows_prefix, 1, tokens, a->H, a->Hkv, a->P) : 0;
  return pl;
}

}  // namespace

extern "C" long tfb_context_attn_work(const tfb_context_attn_args* a) {
  if (int e = check(a)) return -e;
  if (a->B == 0 || a->Sq == 0) return 0;
  const CtxPlan pl = make_plan(a);
  if (pl.slots() == 1) return 0;
  return static_cast<long>(pl.slots()) * a->B * a->Sq * a->H * (a->D + 1) * static_cast<long>(sizeof(float));
}

extern "C" int tfb_context_attn(const tfb_context_attn_args* a, void* stream) {
  if (int e = check(a)) return e;
  if (a->B == 0 || a->Sq == 0) return TFB_OK;
  if ((a->q_bs | a->q_ss | a->q_hs | a->k_bs | a->k_ss | a->k_hs | a->v_bs | a->v_ss | a->v_hs | a->kp_ss | a->kp_hs |
       a->vp_ss | a->vp_hs) % 8)
    return TFB_ERR_BAD_SHAPE;
  if ((reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->k) | reinterpret_cast<uintptr_t>(a->v) |
       reinterpret_cast<uintptr_t>(a->kp) | reinterpret_cast<uintptr_t>(a->vp) | reinterpret_cast<uintptr_t>(a->out) |
       reinterpret_cast<uintptr_t>(a->work)) & 15)
    return TFB_ERR_BAD_SHAPE;
  if (!a->q || !a->out || (a->Skv && (!a->k || !a->v)) || (a->P && (!a->kp || !a->vp))) return TFB_ERR_BAD_SHAPE;
  const CtxPlan pl = make_plan(a);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  CtxParams p;
  p.q = a->q, p.k = a->k, p.v = a->v;
  p.q_bs = a->q_bs, p.q_ss = a->q_ss, p.q_hs = a->q_hs;
  p.k_bs = a->k_bs, p.k_ss = a->k_ss, p.k_hs = a->k_hs;
  p.v_bs = a->v_bs, p.v_ss = a->v_ss, p.v_hs = a->v_hs;
  p.kp = a->kp, p.vp = a->vp;
  p.kp_ss = a->kp_ss, p.kp_hs = a->kp_hs, p.vp_ss = a->vp_ss, p.vp_hs = a->vp_hs;
  p.out = a->out;
  p.lse = a->lse;
  p.kv_lens = a->kv_lens;
  p.cu_kv = a->cu_kv;
  p.key_mask = static_cast<const uint8_t*>(a->key_mask);
  p.mask_bs = a->mask_bs;
  p.B = a->B, p.Sq = a->Sq, p.H = a->H, p.Hkv = a->Hkv, p.D = a->D, p.Skv = a->Skv;
  p.P = pl.apart ? 0 : a->P;
  p.ns = pl.ns;
  p.slot0 = pl.apart ? pl.ns_prefix : 0;
  p.scale_log2 = a->scale * 1.4426950408889634f;
  p.status = status_word();
  p.part_o = p.part_lse = nullptr;
  if (pl.slots() > 1) {
    if (!a->work) return TFB_ERR_BAD_SHAPE;
    p.part_o = a->work;
    p.part_lse = a->work + static_cast<long>(pl.slots()) * a->B * a->Sq * a->H * a->D;
  }
  if (pl.apart) {
    // All samples' tokens as one batch entry: needs one stride from token to token.
    const long ss = a->Sq == 1 ? a->q_bs : a->q_ss;
    if (a->B > 1 && a->Sq > 1 && a->q_bs != a->Sq * a->q_ss) return TFB_ERR_BAD_SHAPE;
    const long tokens = static_cast<long>(a->B) * a->Sq;
    if (tokens > (1 << 30)) return TFB_ERR_TOO_LARGE;
    CtxParams f = p;
    f.q_ss = a->B > 1 ? ss : a->q_ss;
    f.q_bs = 0;
    f.k = a->kp, f.v = a->vp;
    f.k_bs = f.v_bs = 0;
    f.k_ss = a->kp_ss, f.k_hs = a->kp_hs, f.v_ss = a->vp_ss, f.v_hs = a->vp_hs;
    f.kv_lens = nullptr;
    f.B = 1, f.Sq = static_cast<int>(tokens), f.Skv = a->P;
    f.ns = pl.ns_prefix;
    f.slot0 = 0;
    if (int e = pl.rows_prefix ? launch_ctx_rows(f, a->fp16, st) : launch_ctx_tc(f, a->fp16, st)) return e;
  }
  if (int e = pl.rows_own ? launch_ctx_rows(p, a->fp16, st)
              : pl.short_own ? launch_ctx_short(p, a->fp16, st)
                             : launch_ctx_tc(p, a->fp16, st))
    return e;
  if (pl.slots() > 1) {
    p.ns = pl.slots();
    return launch_ctx_join(p, a->fp16, st);
  }
  return TFB_OK;
}
