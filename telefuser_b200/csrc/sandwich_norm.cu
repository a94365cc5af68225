// The row kernel between two sub-layers of a sandwich-norm block: RMSNorm behind the sub-layer, gate, residual, RMSNorm in
// front of the next one and its modulation, in one pass:
//   x = res + g * (w * y / rms(y)),   h = (w2 * x / rms(x)) * (1 + scale) + shift
// res and y are read once, x and h written once: 8 bytes per element in 16-bit types where the two-kernel chain
// (rmsnorm_gate_residual, rmsnorm_modulate) moves 10. The second norm reads x as it is stored, so both agree.
//
// HBM bound. Rows (and per-token tables) arrive by bulk copies in shared memory; sums, norms and gates are fp32; x and h are
// rounded once to the activations' type. Two kernels:
//   warp per row   many rows of a 16-bit type with per-sample tables. The row stays packed in a warp's registers, its two sums
//                  are shuffles, and no barrier ties warps together. What tables and weights say about a column (gate * w,
//                  w2 * (1 + scale), shift) lies in shared memory, computed once per CTA: re-reading the fp32 tables
//                  from global memory for every row would cost L1 twice the bytes of the row itself.
//   CTA per row    everything else. A thread owns 8 NV fixed columns and keeps what the tables say about them in registers;
//                  rows come through a ring several rows ahead of the two block sums. Half the latency for a few rows,
//                  but its barriers and redundant sums take about 3000 instructions per row where the other form takes 1600.
// 2 x 4224 x 3840 bf16: CTA per row 55 us (four rows behind the same barriers: 76), warp per row 51; 37441 x 2048: 116 and 110 us,
// 5.6 TB/s; three rows: 4.7 us with a CTA per row. Per-token tables, 2 x 3001 x 4096 fp16: 78 us, 6.3 TB/s.
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

// tanh to about 2^-21 of its value: its series below 1/4 (the first term left out is 1382 / 155925 v^11, 2^-26 of v there), else
// (1 - e) / (1 + e) with e = exp(-2 |v|). 1 - e loses most at 1/4, where e = 0.61 and two units in its last place are 2^-21.6 of
// the difference.
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
  // CTAs that fit an SM by registers (64 a thread, 128 with two column groups), then as many stages as an equal share of 200 KB
  // of shared memory gives each of them, at most eight and no more than it has rows: 180 to 192 KB in flight per SM with 16-bit
  // rows of 2048 to 4096 columns, less where a CTA has few rows.
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

// ---- warp per row ----
struct SnormWarpParams {
  SnormParams s;
  int per_sample;  // rows of a sample: one row of every table
  int chunks, per_chunk;
  int stages;      // rows in flight per warp
};

// Two 16-bit values as packed fp32 and back.
template <typename T>
__device__ __forceinline__ uint64_t snorm_unpack2(uint32_t v);
template <>
__device__ __forceinline__ uint64_t snorm_unpack2<__nv_bfloat16>(uint32_t v) {
  return f2_pack(bf16_lo(v), bf16_hi(v));
}
template <>
__device__ __forceinline__ uint64_t snorm_unpack2<__half>(uint32_t v) {
  const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&v));
  return f2_pack(t.x, t.y);
}
template <typename T>
__device__ __forceinline__ uint32_t snorm_pack2(uint64_t v);
template <>
__device__ __forceinline__ uint32_t snorm_pack2<__nv_bfloat16>(uint64_t v) {
  float a, b;
  f2_unpack(v, a, b);
  return pack_bf16x2(a, b);
}
template <>
__device__ __forceinline__ uint32_t snorm_pack2<__half>(uint64_t v) {
  float a, b;
  f2_unpack(v, a, b);
  return pack_f16x2(a, b);
}
__device__ __forceinline__ float snorm_total(const uint64_t (&s)[4]) {
  float a, b;
  f2_unpack(f2_add(f2_add(s[0], s[1]), f2_add(s[2], s[3])), a, b);
  return warp_sum(a + b);
}

template <typename T, int NVL>
__global__ void __launch_bounds__(384, 1) sandwich_norm_warp_kernel(const SnormWarpParams wp) {
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ uint64_t bars[24], tables_full;
  __shared__ int abort_flag;
  const SnormParams& p = wp.s;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = blockDim.x >> 5;
  const int nvec = p.C >> 3;
  const long b = blockIdx.x / wp.chunks;
  const long r0 = b * wp.per_sample + static_cast<long>(blockIdx.x % wp.chunks) * wp.per_chunk;
  const long r1 = min(r0 + wp.per_chunk, (b + 1) * wp.per_sample);
  const uint32_t row_bytes = p.C * 2, w_bytes = p.C * (p.w_f32 ? 4 : 2);
  // gate, scale, shift as they come, then in their place gate * w, w2 * (1 + scale), shift: fp32, 32 bytes per 8 columns, the
  // two halves of every second group of four swapped, so that lanes reading one half each meet no bank twice
  float* gw = reinterpret_cast<float*>(smem);
  float *ws = gw + p.C, *sh = ws + p.C;
  uint8_t* raw_w = smem + 12 * p.C;
  uint8_t* raw_w2 = raw_w + w_bytes;
  uint8_t* ring = raw_w2 + w_bytes + static_cast<long>(warp) * wp.stages * 2 * row_bytes;
  uint64_t* full = bars + warp * wp.stages;
  const AbortCtx ctx{&abort_flag, p.status};
  // one lane: y and res of row r
  auto fetch = [&](long r, int slot) {
    uint8_t* dst = ring + slot * 2 * row_bytes;
    mbar_expect_tx(&full[slot], 2 * row_bytes);
    bulk_load(dst, static_cast<const T*>(p.y) + r * p.ldy, row_bytes, &full[slot]);
    bulk_load(dst + row_bytes, static_cast<const T*>(p.res) + r * p.ldr, row_bytes, &full[slot]);
  };
  // Tables and weights first: behind the first rows of every CTA, 25 MB, they came 8 us later.
  if (threadIdx.x == 0) {
    mbar_init(&tables_full, 1);
    abort_flag = 0;
    mbar_fence_init();
    const bool post_w = p.post && p.w;
    mbar_expect_tx(&tables_full, p.C * 4 * ((p.gate != nullptr) + (p.scale != nullptr) + (p.shift != nullptr)) +
                                     w_bytes * (post_w + (p.w2 != nullptr)));
    if (p.gate) bulk_load(gw, p.gate + r0 / p.rpg * p.ldg, p.C * 4, &tables_full);
    if (p.scale) bulk_load(ws, p.scale + r0 / p.rpc * p.ldc, p.C * 4, &tables_full);
    if (p.shift) bulk_load(sh, p.shift + r0 / p.rps * p.lds, p.C * 4, &tables_full);
    if (post_w) bulk_load(raw_w, p.w, w_bytes, &tables_full);
    if (p.w2) bulk_load(raw_w2, p.w2, w_bytes, &tables_full);
  }
  if (lane == 0) {
    for (int s = 0; s < wp.stages; ++s) mbar_init(&full[s], 1);
    mbar_fence_init();
  }
  __syncthreads();
  if (lane == 0)
    for (int s = 0; s < wp.stages; ++s)
      if (r0 + warp + static_cast<long>(s) * nw < r1) fetch(r0 + warp + static_cast<long>(s) * nw, s);
  mbar_wait(&tables_full, 0, ctx, 72);
  // Four columns a step, each thread its own 8 in place. Kept small on purpose: unrolled, with a tanh per column, this was
  // mostly the fetching of instructions.
#pragma unroll 1
  for (int vi = threadIdx.x; vi < nvec; vi += blockDim.x) {
    float4 g[2], c[2], h[2];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int col = vi * 8 + q * 4;
      auto weight = [&](const uint8_t* w) {
        if (p.w_f32) return *reinterpret_cast<const float4*>(w + col * 4);
        const uint2 u = *reinterpret_cast<const uint2*>(w + col * 2);
        float4 f;
        f2_unpack(snorm_unpack2<T>(u.x), f.x, f.y);
        f2_unpack(snorm_unpack2<T>(u.y), f.z, f.w);
        return f;
      };
      const float4 one = make_float4(1.f, 1.f, 1.f, 1.f), zero = make_float4(0.f, 0.f, 0.f, 0.f);
      const float4 w = p.post && p.w ? weight(raw_w) : one, w2 = p.w2 ? weight(raw_w2) : one;
      g[q] = p.gate ? *reinterpret_cast<const float4*>(gw + col) : one;
      c[q] = p.scale ? *reinterpret_cast<const float4*>(ws + col) : zero;
      h[q] = p.shift ? *reinterpret_cast<const float4*>(sh + col) : zero;
      if (p.gate && p.tanh_gate) {
#pragma unroll 1
        for (int e = 0; e < 4; ++e) g[q] = make_float4(g[q].y, g[q].z, g[q].w, snorm_tanh(g[q].x));
      }
      g[q] = make_float4(w.x * g[q].x, w.y * g[q].y, w.z * g[q].z, w.w * g[q].w);
      c[q] = make_float4(w2.x * (1.f + c[q].x), w2.y * (1.f + c[q].y), w2.z * (1.f + c[q].z), w2.w * (1.f + c[q].w));
    }
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int at = vi * 2 + (q ^ (vi >> 2 & 1));
      reinterpret_cast<float4*>(gw)[at] = g[q];
      reinterpret_cast<float4*>(ws)[at] = c[q];
      reinterpret_cast<float4*>(sh)[at] = h[q];
    }
  }
  __syncthreads();

  const float inv_c = 1.f / p.C;
  int slot = 0;
  uint32_t phase = 0;
  for (long r = r0 + warp; r < r1; r += nw) {
    // after an expired wait (recorded in the status word) the warp goes on with what is there
    mbar_wait_warp(&full[slot], phase, ctx, 71);
    const uint4* sy = reinterpret_cast<const uint4*>(ring + slot * 2 * row_bytes);
    const uint4* sr = reinterpret_cast<const uint4*>(ring + slot * 2 * row_bytes + row_bytes);
    uint4 row[NVL];  // y, then x as stored
    uint64_t ss[4] = {0ull, 0ull, 0ull, 0ull};  // packed fp32, four chains
#pragma unroll
    for (int i = 0; i < NVL; ++i) {
      const int vi = lane + i * 32;
      if (vi < nvec) {
        row[i] = sy[vi];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint64_t y = snorm_unpack2<T>((&row[i].x)[e]);
          ss[e] = f2_fma(y, y, ss[e]);
        }
      }
    }
    const float rstd = p.post ? rsqrtf(snorm_total(ss) * inv_c + p.eps) : 1.f;
    const uint64_t rstd_2 = f2_pack(rstd, rstd);
    ss[0] = ss[1] = ss[2] = ss[3] = 0ull;
    uint4* xo = reinterpret_cast<uint4*>(static_cast<T*>(p.x) + r * p.C);
#pragma unroll
    for (int i = 0; i < NVL; ++i) {
      const int vi = lane + i * 32;
      if (vi < nvec) {
        const uint4 rv = sr[vi];
        const int at = vi * 2 + (vi >> 2 & 1);  // of the first half; the second is next to it
        const ulonglong2 g0 = reinterpret_cast<const ulonglong2*>(gw)[at], g1 = reinterpret_cast<const ulonglong2*>(gw)[at ^ 1];
        const uint64_t g[4] = {g0.x, g0.y, g1.x, g1.y};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          uint32_t& v = (&row[i].x)[e];
          v = snorm_pack2<T>(f2_fma(snorm_unpack2<T>(v), f2_mul(g[e], rstd_2), snorm_unpack2<T>((&rv.x)[e])));
          const uint64_t x = snorm_unpack2<T>(v);
          ss[e] = f2_fma(x, x, ss[e]);
        }
        xo[vi] = row[i];
      }
    }
    __syncwarp();
    if (lane == 0 && r + static_cast<long>(wp.stages) * nw < r1) fetch(r + static_cast<long>(wp.stages) * nw, slot);
    if (++slot == wp.stages) slot = 0, phase ^= 1;
    const float rstd2 = rsqrtf(snorm_total(ss) * inv_c + p.eps);
    const uint64_t rstd2_2 = f2_pack(rstd2, rstd2);
    uint4* ho = reinterpret_cast<uint4*>(static_cast<T*>(p.h) + r * p.C);
#pragma unroll
    for (int i = 0; i < NVL; ++i) {
      const int vi = lane + i * 32;
      if (vi < nvec) {
        const int at = vi * 2 + (vi >> 2 & 1);
        const ulonglong2 w0 = reinterpret_cast<const ulonglong2*>(ws)[at], w1 = reinterpret_cast<const ulonglong2*>(ws)[at ^ 1];
        const ulonglong2 s0 = reinterpret_cast<const ulonglong2*>(sh)[at], s1 = reinterpret_cast<const ulonglong2*>(sh)[at ^ 1];
        const uint64_t w[4] = {w0.x, w0.y, w1.x, w1.y}, s[4] = {s0.x, s0.y, s1.x, s1.y};
        uint4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          (&v.x)[e] = snorm_pack2<T>(f2_fma(f2_mul(snorm_unpack2<T>((&row[i].x)[e]), rstd2_2), w[e], s[e]));
        ho[vi] = v;
      }
    }
  }
}

template <typename T, int NVL>
static int launch_snorm_warp(const SnormParams& p, long per_sample, cudaStream_t st) {
  static bool attr_set[TFB_MAX_DEVICES] = {false};
  constexpr int SMEM = 220 * 1024;
  auto kern = &sandwich_norm_warp_kernel<T, NVL>;
  if (int rc = ensure_dynamic_smem(reinterpret_cast<const void*>(kern), SMEM, attr_set)) return rc;
  SnormWarpParams wp;
  wp.s = p;
  wp.per_sample = static_cast<int>(per_sample);
  const int tables = 3 * 4 * p.C + 2 * p.C * (p.w_f32 ? 4 : 2), stage = 4 * p.C;
  // twelve warps, two rows each if they fit, else one
  int fit = (SMEM - tables) / stage;
  wp.stages = fit >= 24 ? 2 : 1;
  const int warps = fit / wp.stages < 12 ? fit / wp.stages : 12;
  const long samples = p.rows / per_sample;
  long chunks = sm_count() / samples;  // one CTA per SM
  if (chunks < 1) chunks = 1;
  if (chunks > (per_sample + warps - 1) / warps) chunks = (per_sample + warps - 1) / warps;
  wp.per_chunk = static_cast<int>((per_sample + chunks - 1) / chunks);
  wp.chunks = static_cast<int>((per_sample + wp.per_chunk - 1) / wp.per_chunk);
  kern<<<static_cast<int>(samples * wp.chunks), warps * 32, tables + warps * wp.stages * stage, st>>>(wp);
  return cudaGetLastError() == cudaSuccess ? TFB_OK : TFB_ERR_LAUNCH;
}

// Warp per row: per-sample tables, 16-bit rows of up to 5120 columns (so that six rows and the tables fit), rows enough for
// eight warps on every SM, and eight rows or more under one table row: a CTA there folds the tables of one sample only. bf16, CTA
// per row against warp per row: 1000 x 2 rows of 2048 14.0 and 31.0 us, 4000 x 7 114 and 144, 1000 x 8 39 and 41, 148 x 8 8.1 and
// 6.2, 500 x 16 35.8 and 35.4, 500 x 60 98 and 87. Above 4096 columns, where a CTA per row needs two column groups per thread, warps
// are no slower with any number: 1000 x 2 rows of 5120 66 and 66, 500 x 4 47 and 39, 4000 x 7 446 and 286. 75 .. 147 samples get a
// CTA each and leave the other SMs idle, which is still as fast as a CTA per row (75 x 400 rows: 1024 columns 54.4 and 53.9,
// 2048 96 and 101, 3840 172 and 187, 5120 300 and 303; 75 x 32 of 2048 15.2 and 12.0).
template <typename T>
static bool snorm_by_warps(const SnormParams& p) {
  return sizeof(T) == 2 && !p.token && p.C <= 5120 && p.rows >= 8L * sm_count() && p.rows <= 0x7fffffffL &&
         (p.rp >= 8 || p.C > 4096);
}

template <typename T>
static int launch_snorm(SnormParams& p, cudaStream_t st) {
  if constexpr (sizeof(T) == 2) {
    if (snorm_by_warps<T>(p)) {
      if (p.C <= 1024) return launch_snorm_warp<T, 4>(p, p.rp, st);
      if (p.C <= 2048) return launch_snorm_warp<T, 8>(p, p.rp, st);
      if (p.C <= 4096) return launch_snorm_warp<T, 16>(p, p.rp, st);
      return launch_snorm_warp<T, 20>(p, p.rp, st);
    }
  }
  const int nvec = p.C / 8;
  const int nv = nvec > 512 ? 2 : 1;
  const int threads = ((nvec + nv - 1) / nv + 31) / 32 * 32;
  return nv == 1 ? launch_snorm_nv<T, 1>(p, threads, st) : launch_snorm_nv<T, 2>(p, threads, st);
}

}  // namespace tfb

using namespace tfb;

extern "C" int tfb_sandwich_norm(const tfb_sandwich_norm_args* a, void* stream) {
  if (!a) return TFB_ERR_BAD_SHAPE;
  if (a->rows <= 0) return TFB_OK;
  const long align = a->dtype == 2 ? 4 : 8;
  if (a->C < 8 || a->C % 8 || a->C > 8192 || a->ldr % align || a->ldy % align || a->dtype < 0 || a->dtype > 2) return TFB_ERR_BAD_SHAPE;
  if (!a->res || !a->y || !a->x || !a->h) return TFB_ERR_BAD_SHAPE;
  if ((a->gate && (a->ldg % 4 || a->rpg < 1)) || (a->shift && (a->lds % 4 || a->rps < 1)) || (a->scale && (a->ldc % 4 || a->rpc < 1)))
    return TFB_ERR_BAD_SHAPE;
  uintptr_t any = 0;
  for (const void* q : {a->res, a->y, static_cast<const void*>(a->x), static_cast<const void*>(a->h), a->w, a->w2,
                        static_cast<const void*>(a->gate), static_cast<const void*>(a->shift), static_cast<const void*>(a->scale)})
    any |= reinterpret_cast<uintptr_t>(q);
  if (any & 15) return TFB_ERR_BAD_SHAPE;
  SnormParams p;
  p.res = a->res, p.y = a->y, p.x = a->x, p.h = a->h, p.ldr = a->ldr, p.ldy = a->ldy, p.rows = a->rows, p.C = a->C;
  p.w_f32 = a->w_f32, p.post = a->post, p.tanh_gate = a->tanh_gate, p.eps = a->eps, p.w = a->w, p.w2 = a->w2;
  p.gate = a->gate, p.shift = a->shift, p.scale = a->scale;
  p.ldg = a->ldg, p.rpg = a->rpg, p.lds = a->lds, p.rps = a->rps, p.ldc = a->ldc, p.rpc = a->rpc;
  // Tables that change from row to row go through the ring; the others change together where they change at all (one row
  // per sample or one in all).
  p.token = (p.gate && p.rpg == 1 && p.ldg ? 1 : 0) | (p.shift && p.rps == 1 && p.lds ? 2 : 0) | (p.scale && p.rpc == 1 && p.ldc ? 4 : 0);
  p.rp = p.rows;
  if (p.gate && !(p.token & 1) && p.rpg < p.rp) p.rp = p.rpg;
  if (p.shift && !(p.token & 2) && p.rps < p.rp) p.rp = p.rps;
  if (p.scale && !(p.token & 4) && p.rpc < p.rp) p.rp = p.rpc;
  p.status = status_word();
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (a->dtype == 0) return launch_snorm<__nv_bfloat16>(p, st);
  if (a->dtype == 1) return launch_snorm<__half>(p, st);
  return launch_snorm<float>(p, st);
}
