// The row kernel between two sub-layers of a sandwich-norm block: RMSNorm behind the sub-layer, gate, residual, RMSNorm in
// front of the next one and its modulation, in one pass:
//   x = res + g * (w * y / rms(y)),   h = (w2 * x / rms(x)) * (1 + scale) + shift
// res and y are read once, x and h written once: 8 bytes per element in 16-bit types where the two-kernel chain
// (rmsnorm_gate_residual, rmsnorm_modulate) moves 10. The second norm reads x as it is stored, so both agree.
//
// HBM bound. A thread owns 8 NV fixed columns of every row its CTA walks over, so that what per-sample tables and weights
// say about those columns (gate * w, w2 * (1 + scale), shift) stays in registers from row to row; reading the fp32 tables
// again for every row would cost L1 twice the bytes of the row itself. Rows (and per-token tables) arrive through a ring of
// bulk copies in shared memory, several rows ahead of the two block sums, whose latency would otherwise bound the kernel.
// Sums, norms and gates are fp32; x and h are rounded once to the activations' type.
#include <math.h>

#include "tfb_api.h"
#include "tfb_common.cuh"
#include "tfb_host.h"

namespace tfb {

struct SnormParams {
  const void *res, *y;
  void *x, *h;
  long ldr, ldy;
  long rows;
  int C, w_f32, post, tanh_gate;
  float eps;
  const void *w, *w2;
  const float *gate, *shift, *scale;
  long ldg, rpg, lds, rps, ldc, rpc;
  long rp;       // rows between changes of the register tables
  long per_cta;  // consecutive rows of one CTA
  int token;     // tables with a row per token, kept in the ring: bit 0 gate, 1 shift, 2 scale
  int stages, stage_bytes;
  int* status;
};

constexpr int SN_MAX_STAGES = 8;

// tanh to fp32 accuracy: its series below 1/4, else through the exponential (where 1 - 2 / (e + 1) loses nothing).
__device__ __forceinline__ float snorm_tanh(float v) {
  const float a = fabsf(v), q = v * v;
  if (a < 0.25f)
    return v * (1.f + q * (-1.f / 3.f + q * (2.f / 15.f + q * (-17.f / 315.f + q * (62.f / 2835.f)))));
  const float e = __expf(-2.f * a);
  return copysignf(__fdividef(1.f - e, 1.f + e), v);
}

template <typename T>
struct Vec8;
template <>
struct Vec8<__nv_bfloat16> {
  uint4 u;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { u = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void get(float (&f)[8]) const {
    f[0] = bf16_lo(u.x), f[1] = bf16_hi(u.x), f[2] = bf16_lo(u.y), f[3] = bf16_hi(u.y);
    f[4] = bf16_lo(u.z), f[5] = bf16_hi(u.z), f[6] = bf16_lo(u.w), f[7] = bf16_hi(u.w);
  }
  __device__ __forceinline__ void put(const float (&f)[8]) {
    u = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
  }
  __device__ __forceinline__ void store(__nv_bfloat16* p) const { *reinterpret_cast<uint4*>(p) = u; }
};
template <>
struct Vec8<__half> {
  uint4 u;
  __device__ __forceinline__ void load(const __half* p) { u = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void get(float (&f)[8]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t v = (&u.x)[i];
      const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&v));
      f[2 * i] = t.x, f[2 * i + 1] = t.y;
    }
  }
  __device__ __forceinline__ void put(const float (&f)[8]) {
    u = make_uint4(pack_f16x2(f[0], f[1]), pack_f16x2(f[2], f[3]), pack_f16x2(f[4], f[5]), pack_f16x2(f[6], f[7]));
  }
  __device__ __forceinline__ void store(__half* p) const { *reinterpret_cast<uint4*>(p) = u; }
};
template <>
struct Vec8<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p) {
    a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  }
  __device__ __forceinline__ void get(float (&f)[8]) const {
    f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
  }
  __device__ __forceinline__ void put(const float (&f)[8]) {
    a = make_float4(f[0], f[1], f[2], f[3]), b = make_float4(f[4], f[5], f[6], f[7]);
  }
  __device__ __forceinline__ void store(float* p) const {
    reinterpret_cast<float4*>(p)[0] = a, reinterpret_cast<float4*>(p)[1] = b;
  }
};

template <typename T>
__device__ __forceinline__ void snorm_weight(const void* w, int w_f32, int col, float (&f)[8]) {
  if (!w) {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = 1.f;
  } else if (w_f32) {
    Vec8<float> v;
    v.load(static_cast<const float*>(w) + col);
    v.get(f);
  } else {
    Vec8<T> v;
    v.load(static_cast<const T*>(w) + col);
    v.get(f);
  }
}
__device__ __forceinline__ void snorm_table(const float* t, long at, float (&f)[8]) {
  if (!t) {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = 0.f;
  } else {
    Vec8<float> v;
    v.load(t + at);
    v.get(f);
  }
}

// Sum over the CTA with one barrier; sums that follow each other take turns between the rows of `red`.
__device__ __forceinline__ float snorm_sum(float v, float* red) {
  v = warp_sum(v);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = blockDim.x >> 5;
  if (lane == 0) red[warp] = v;
  __syncthreads();
  return warp_sum(lane < nw ? red[lane] : 0.f);
}

template <typename T, int NV>
__global__ void __launch_bounds__(512, NV == 1 ? 2 : 1) sandwich_norm_kernel(const SnormParams p) {
  extern __shared__ __align__(16) uint8_t ring[];
  __shared__ float red[4][32];
  __shared__ uint64_t full[SN_MAX_STAGES];
  __shared__ int abort_flag;
  const int nvec = p.C >> 3;
  const long r0 = blockIdx.x * p.per_cta, r1 = min(r0 + p.per_cta, p.rows);
  const float inv_c = 1.f / p.C;
  const uint32_t row_bytes = p.C * sizeof(T), tab_bytes = p.C * 4;
  const AbortCtx ctx{&abort_flag, p.status};
  // one thread: the bulk copies of row r
  auto fetch = [&](long r) {
    const int slot = static_cast<int>((r - r0) % p.stages);
    uint8_t* dst = ring + slot * p.stage_bytes;
    mbar_expect_tx(&full[slot], p.stage_bytes);
    bulk_load(dst, static_cast<const T*>(p.y) + r * p.ldy, row_bytes, &full[slot]);
    bulk_load(dst + row_bytes, static_cast<const T*>(p.res) + r * p.ldr, row_bytes, &full[slot]);
    dst += 2 * row_bytes;
    if (p.token & 1) bulk_load(dst, p.gate + r * p.ldg, tab_bytes, &full[slot]), dst += tab_bytes;
    if (p.token & 2) bulk_load(dst, p.shift + r * p.lds, tab_bytes, &full[slot]), dst += tab_bytes;
    if (p.token & 4) bulk_load(dst, p.scale + r * p.ldc, tab_bytes, &full[slot]);
  };
  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) mbar_init(&full[s], 1);
    abort_flag = 0;
    mbar_fence_init();
    for (long r = r0; r < r1 && r < r0 + p.stages; ++r) fetch(r);
  }
  __syncthreads();

  float gw[NV][8], ws[NV][8], sh[NV][8];  // gate * w, w2 * (1 + scale), shift; w and w2 alone for per-token tables
  long next_tables = r0;
  int slot = 0, turn = 0;
  uint32_t phase = 0;
  for (long r = r0; r < r1; ++r) {
    if (r == next_tables) {
      next_tables = (r / p.rp + 1) * p.rp;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int col = (threadIdx.x + i * blockDim.x) * 8;
        if (col < p.C) {
          float t[8];
          snorm_weight<T>(p.post ? p.w : nullptr, p.w_f32, col, gw[i]);
          if (p.gate && !(p.token & 1)) {
            snorm_table(p.gate, r / p.rpg * p.ldg + col, t);
#pragma unroll
            for (int e = 0; e < 8; ++e) gw[i][e] *= p.tanh_gate ? snorm_tanh(t[e]) : t[e];
          }
          snorm_weight<T>(p.w2, p.w_f32, col, ws[i]);
          if (p.scale && !(p.token & 4)) {
            snorm_table(p.scale, r / p.rpc * p.ldc + col, t);
#pragma unroll
            for (int e = 0; e < 8; ++e) ws[i][e] *= 1.f + t[e];
          }
          snorm_table(p.token & 2 ? nullptr : p.shift, p.shift ? r / p.rps * p.lds + col : 0, sh[i]);
        }
      }
    }
    // A wait that runs out leaves its status behind; the barriers below keep every thread of the CTA together all the same.
    mbar_wait(&full[slot], phase, ctx, 70);
    const uint8_t* stage = ring + slot * p.stage_bytes;
    const float* tables = reinterpret_cast<const float*>(stage + 2 * row_bytes);
    float x[NV][8];
    Vec8<T> res[NV];
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int col = (threadIdx.x + i * blockDim.x) * 8;
      if (col < p.C) {
        Vec8<T> y;
        y.load(reinterpret_cast<const T*>(stage) + col);
        res[i].load(reinterpret_cast<const T*>(stage + row_bytes) + col);
        y.get(x[i]);
#pragma unroll
        for (int e = 0; e < 8; ++e) ss += x[i][e] * x[i][e];
      }
    }
    const float rstd = p.post ? rsqrtf(snorm_sum(ss, red[turn]) * inv_c + p.eps) : 1.f;
    ss = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int col = (threadIdx.x + i * blockDim.x) * 8;
      if (col < p.C) {
        float f[8];
        res[i].get(f);
        if (p.token & 1) {
          float t[8];
          snorm_table(tables, col, t);
#pragma unroll
          for (int e = 0; e < 8; ++e) x[i][e] *= p.tanh_gate ? snorm_tanh(t[e]) : t[e];
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] += x[i][e] * rstd * gw[i][e];
        res[i].put(f);
        res[i].get(x[i]);  // as stored
        res[i].store(static_cast<T*>(p.x) + r * p.C + col);
#pragma unroll
        for (int e = 0; e < 8; ++e) ss += x[i][e] * x[i][e];
      }
    }
    const float rstd2 = rsqrtf(snorm_sum(ss, red[2 + turn]) * inv_c + p.eps);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int col = (threadIdx.x + i * blockDim.x) * 8;
      if (col < p.C) {
        const float* tab = tables + (p.token & 1 ? p.C : 0);
        float f[8], t[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = x[i][e] * rstd2 * ws[i][e];
        if (p.token & 4) {
          snorm_table(tab + (p.token & 2 ? p.C : 0), col, t);
#pragma unroll
          for (int e = 0; e < 8; ++e) f[e] *= 1.f + t[e];
        }
        if (p.token & 2) {
          snorm_table(tab, col, t);
#pragma unroll
          for (int e = 0; e < 8; ++e) f[e] += t[e];
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] += sh[i][e];
        res[i].put(f);
        res[i].store(static_cast<T*>(p.h) + r * p.C + col);
      }
    }
    // The slot is free once nobody reads it any more: behind this row's last barrier, and with per-token tables, which
    // are read after it, behind one more.
    if (p.token) __syncthreads();
    if (threadIdx.x == 0 && r + p.stages < r1) fetch(r + p.stages);
    turn ^= 1;
    if (++slot == p.stages) slot = 0, phase ^= 1;
  }
}

template <typename T, int NV>
static int launch_snorm_nv(SnormParams& p, int threads, cudaStream_t st) {
  static bool attr_set[TFB_MAX_DEVICES] = {false};
  constexpr int SMEM_SM = 200 * 1024;
  if (int rc = ensure_dynamic_smem(reinterpret_cast<const void*>(&sandwich_norm_kernel<T, NV>), SMEM_SM, attr_set)) return rc;
  // CTAs that fit an SM by registers (64 a thread, 128 with two column groups), then as many stages as shared memory
  // gives each of them: 50 to 100 KB in flight per SM.
  int ctas = 65536 / ((NV == 1 ? 64 : 128) * threads);
  if (ctas > 8) ctas = 8;
  const int tables = (p.token & 1) + (p.token >> 1 & 1) + (p.token >> 2 & 1);
  p.stage_bytes = p.C * (2 * static_cast<int>(sizeof(T)) + 4 * tables);
  while (ctas > 1 && ctas * 2 * p.stage_bytes > SMEM_SM) --ctas;
  p.stages = SMEM_SM / ctas / p.stage_bytes;
  if (p.stages > SN_MAX_STAGES) p.stages = SN_MAX_STAGES;
  if (p.stages < 1) return TFB_ERR_TOO_LARGE;
  const long slots = static_cast<long>(sm_count()) * ctas;
  p.per_cta = (p.rows + slots - 1) / slots;
  if (p.stages > p.per_cta) p.stages = static_cast<int>(p.per_cta);
  const int grid = static_cast<int>((p.rows + p.per_cta - 1) / p.per_cta);
  sandwich_norm_kernel<T, NV><<<grid, threads, p.stages * p.stage_bytes, st>>>(p);
  return cudaGetLastError() == cudaSuccess ? TFB_OK : TFB_ERR_LAUNCH;
}

template <typename T>
static int launch_snorm(SnormParams& p, cudaStream_t st) {
  const int nvec = p.C / 8;
  const int nv = nvec > 512 ? 2 : 1;
  const int threads = ((nvec + nv - 1) / nv + 31) / 32 * 32;
  return nv == 1 ? launch_snorm_nv<T, 1>(p, threads, st) : launch_snorm_nv<T, 2>(p, threads, st);
}

}  // namespace tfb

using namespace tfb;

extern "C" int tfb_sandwich_norm(const void* res, long ldr, const void* y, long ldy, void* x, void* h, long rows, int C,
                                 float eps, int dtype, int w_f32, const void* w, const void* w2, const float* gate, long ldg,
                                 long rpg, const float* shift, long lds, long rps, const float* scale, long ldc, long rpc,
                                 int post, int tanh_gate, void* stream) {
  if (rows <= 0) return TFB_OK;
  const long align = dtype == 2 ? 4 : 8;
  if (C < 8 || C % 8 || C > 8192 || ldr % align || ldy % align || dtype < 0 || dtype > 2) return TFB_ERR_BAD_SHAPE;
  if ((gate && (ldg % 4 || rpg < 1)) || (shift && (lds % 4 || rps < 1)) || (scale && (ldc % 4 || rpc < 1))) return TFB_ERR_BAD_SHAPE;
  uintptr_t any = 0;
  for (const void* q : {res, y, static_cast<const void*>(x), static_cast<const void*>(h), w, w2,
                        static_cast<const void*>(gate), static_cast<const void*>(shift), static_cast<const void*>(scale)})
    any |= reinterpret_cast<uintptr_t>(q);
  if (any & 15) return TFB_ERR_BAD_SHAPE;
  SnormParams p;
  p.res = res, p.y = y, p.x = x, p.h = h, p.ldr = ldr, p.ldy = ldy, p.rows = rows, p.C = C, p.w_f32 = w_f32, p.post = post;
  p.tanh_gate = tanh_gate, p.eps = eps, p.w = w, p.w2 = w2, p.gate = gate, p.shift = shift, p.scale = scale;
  p.ldg = ldg, p.rpg = rpg, p.lds = lds, p.rps = rps, p.ldc = ldc, p.rpc = rpc;
  // Tables that change from row to row go through the ring; the others change together where they change at all (one row
  // per sample or one in all).
  p.token = (gate && rpg == 1 && ldg ? 1 : 0) | (shift && rps == 1 && lds ? 2 : 0) | (scale && rpc == 1 && ldc ? 4 : 0);
  p.rp = rows;
  if (gate && !(p.token & 1) && rpg < p.rp) p.rp = rpg;
  if (shift && !(p.token & 2) && rps < p.rp) p.rp = rps;
  if (scale && !(p.token & 4) && rpc < p.rp) p.rp = rpc;
  p.status = status_word();
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == 0) return launch_snorm<__nv_bfloat16>(p, st);
  if (dtype == 1) return launch_snorm<__half>(p, st);
  return launch_snorm<float>(p, st);
}
