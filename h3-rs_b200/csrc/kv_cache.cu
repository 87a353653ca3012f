// kv_cache.cu -- writing the 8-bit paged key / value cache and reading it back (kv_common.cuh has its layout).
//
// write: for a page of a head, with x its new rows and lo its older tokens,
//     s = max(s_old if lo > 0, amax * (1 / top), 1e-30),  code = round(x * (1 / s))    top = 127 (int8) or 448 (e4m3)
//     and, where s > s_old, the lo older rows become round(code * (s_old / s)).
// Only finite elements enter amax: an infinity is stored as +-top and a NaN as 0, so that neither costs the page's
// other tokens their precision.  Every step is one IEEE operation in f32 (1 / top, 1 / s and the products), so
// the codes are the same whichever kernel writes them.
// read: dense rows code * scale, rounded once to the output's type.
//
// Both are bound by HBM: a write moves 3 bytes an element from 16 bits (2 in, 1 out), a read back to 16 bits the same.
#include <cstdint>
#include <cuda_runtime.h>
#include "kv_common.cuh"
#include "h3q_internal.h"

namespace h3q {

namespace {

struct KvRows {  // rows [tokens, heads, dim] with unit stride inside a head
  const void* p;
  int64_t token_stride, head_stride;
};

// 8 elements of kind KIND as f32; `vec`: 16-byte loads are aligned
template <int KIND>
__device__ __forceinline__ void load8(const void* base, int64_t off, bool vec, float (&f)[8]) {
  if (KIND == 0) {
    const float* p = reinterpret_cast<const float*>(base) + off;
    if (vec) {
      const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
      f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
      f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = __ldg(p + i);
    }
  } else {
    const uint16_t* p = reinterpret_cast<const uint16_t*>(base) + off;
    uint32_t w[4];
    if (vec) {
      const uint4 a = __ldg(reinterpret_cast<const uint4*>(p));
      w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = (uint32_t)__ldg(p + 2 * i) | ((uint32_t)__ldg(p + 2 * i + 1) << 16);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = KIND == 1 ? h2f((uint16_t)w[i]) : __uint_as_float(w[i] << 16);
      f[2 * i + 1] = KIND == 1 ? h2f((uint16_t)(w[i] >> 16)) : __uint_as_float(w[i] & 0xffff0000u);
    }
  }
}

__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a <= 3.402823466e38f ? a : 0.f;  // NaN and infinity compare false
}

template <int CODES>
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
  if (CODES == kKvInt8) {
    const int q0 = min(127, max(-127, __float2int_rn(a))), q1 = min(127, max(-127, __float2int_rn(b)));
    const int q2 = min(127, max(-127, __float2int_rn(c))), q3 = min(127, max(-127, __float2int_rn(d)));
    return prmt(prmt(q0, q1, 0x0040), prmt(q2, q3, 0x0040), 0x5410);
  }
  uint16_t lo, hi;
  a = a == a ? a : 0.f;
  b = b == b ? b : 0.f;
  c = c == c ? c : 0.f;
  d = d == d ? d : 0.f;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
  return (uint32_t)lo | ((uint32_t)hi << 16);
}

// four codes as f32, exactly
template <int CODES>
__device__ __forceinline__ void decode4f(uint32_t w, float (&f)[4]) {
  uint32_t lo, hi;
  kv_decode4<CODES>(w, lo, hi);
  f[0] = h2f((uint16_t)lo);
  f[1] = h2f((uint16_t)(lo >> 16));
  f[2] = h2f((uint16_t)hi);
  f[3] = h2f((uint16_t)(hi >> 16));
}

// The page that slot `slot` of a write stands for: rows [lo, hi) of it are new; token0: the packed row of its row 0.
struct WritePage {
  int64_t page;
  int64_t token0;
  int lo, hi;
};
__device__ __forceinline__ bool write_page(const KvCache& c, const KvSeqs& s, const int32_t* past, int64_t slot, int b,
                                           WritePage& w) {
  const int s0 = kv_start(s, b), n = kv_start(s, b + 1) - s0;
  const int64_t had = __ldg(past + b);
  if (n <= 0 || had < 0) return false;
  const int64_t i = (had >> c.page_log2) + (slot - kv_slot_base(s, b, 1, c.page, 2));
  const int64_t p0 = i << c.page_log2;
  if (p0 >= had + n) return false;
  w.page = kv_page(c, s, b, i);
  if (w.page < 0) return false;
  w.lo = had > p0 ? (int)(had - p0) : 0;
  w.hi = had + n - p0 < c.page ? (int)(had + n - p0) : c.page;
  w.token0 = s0 + p0 - had;
  return true;
}

__host__ __device__ constexpr float top_of(int codes) { return codes == kKvInt8 ? 127.f : 448.f; }

template <int CODES>
__device__ __forceinline__ uint2 requant8(uint2 w, float ratio) {
  float f[4], g[4];
  decode4f<CODES>(w.x, f);
  decode4f<CODES>(w.y, g);
  return make_uint2(encode4<CODES>(__fmul_rn(f[0], ratio), __fmul_rn(f[1], ratio), __fmul_rn(f[2], ratio),
                                   __fmul_rn(f[3], ratio)),
                    encode4<CODES>(__fmul_rn(g[0], ratio), __fmul_rn(g[1], ratio), __fmul_rn(g[2], ratio),
                                   __fmul_rn(g[3], ratio)));
}

// One CTA for a page of a head of K or V: the page's new rows stay in registers between the maximum and the codes, so
// the input is read once.  VPT vectors of 8 elements a thread: THREADS * VPT * 8 = page * dim.
template <int KIND, int CODES, int THREADS, int VPT>
__global__ void __launch_bounds__(THREADS)
    kv_write_kernel(KvCache c, KvSeqs s, const int32_t* __restrict__ past, KvRows kr, KvRows vr, int vec) {
  const int64_t slot = blockIdx.x;
  const int h = blockIdx.y;
  const int b = kv_slot_seq_warp(s, slot, 1, c.page, 2);
  WritePage w;
  if (!write_page(c, s, past, slot, b, w)) return;
  const KvRows r = blockIdx.z ? vr : kr;
  const int64_t ph = w.page * c.kv_heads + h;
  float* scale = (blockIdx.z ? c.v_scale : c.k_scale) + ph;
  uint2* codes = reinterpret_cast<uint2*>((blockIdx.z ? c.v : c.k) + ph * c.page * c.dim);
  const float old = w.lo > 0 ? *scale : 0.f;
  const int per_row = c.dim >> 3;
  float x[VPT][8];
  float m = 0.f;
#pragma unroll
  for (int j = 0; j < VPT; ++j) {
    const int i = threadIdx.x + j * THREADS, row = i / per_row, col = (i % per_row) * 8;
    if (row >= w.lo && row < w.hi) {
      load8<KIND>(r.p, (w.token0 + row) * r.token_stride + h * r.head_stride + col, vec, x[j]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[j][e] = 0.f;
    }
  }
#pragma unroll
  for (int j = 0; j < VPT; ++j)
#pragma unroll
    for (int e = 0; e < 8; ++e) m = fmaxf(m, finite_abs(x[j][e]));
  __shared__ float part[THREADS / 32];
#pragma unroll
  for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < THREADS / 32; ++i) m = fmaxf(m, part[i]);
  const float now = fmaxf(old, fmaxf(__fmul_rn(m, 1.f / top_of(CODES)), kKvScaleFloor));
  const float inv = __fdiv_rn(1.f, now);
#pragma unroll
  for (int j = 0; j < VPT; ++j) {
    const int i = threadIdx.x + j * THREADS, row = i / per_row;
    if (row >= w.lo && row < w.hi) {
      uint2 o;
      o.x = encode4<CODES>(__fmul_rn(x[j][0], inv), __fmul_rn(x[j][1], inv), __fmul_rn(x[j][2], inv),
                           __fmul_rn(x[j][3], inv));
      o.y = encode4<CODES>(__fmul_rn(x[j][4], inv), __fmul_rn(x[j][5], inv), __fmul_rn(x[j][6], inv),
                           __fmul_rn(x[j][7], inv));
      codes[i] = o;
    } else if (row < w.lo && now > old) {
      codes[i] = requant8<CODES>(codes[i], __fdiv_rn(old, now));
    }
  }
  // every thread has read the old scale before the barrier above
  if (threadIdx.x == 0) *scale = now;
}

// One warp for a page of a head of K or V, for calls of a few tokens a sequence, where a CTA a page would idle: two
// passes over the few new rows (the second hits L1), 8 elements a lane.
template <int KIND, int CODES>
__global__ void __launch_bounds__(128)
    kv_write_few_kernel(KvCache c, KvSeqs s, const int32_t* __restrict__ past, KvRows kr, KvRows vr, int vec,
                        int64_t slots) {
  const int lane = threadIdx.x & 31;
  const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int64_t slot = unit / (2 * c.kv_heads);
  if (slot >= slots) return;
  const int rest = (int)(unit % (2 * c.kv_heads)), h = rest >> 1, isv = rest & 1;
  const int b = kv_slot_seq_warp(s, slot, 1, c.page, 2);
  WritePage w;
  if (!write_page(c, s, past, slot, b, w)) return;
  const KvRows r = isv ? vr : kr;
  const int64_t ph = w.page * c.kv_heads + h;
  float* scale = (isv ? c.v_scale : c.k_scale) + ph;
  uint2* codes = reinterpret_cast<uint2*>((isv ? c.v : c.k) + ph * c.page * c.dim);
  const float old = w.lo > 0 ? *scale : 0.f;
  const int per_row = c.dim >> 3;
  const int first = w.lo * per_row, last = w.hi * per_row;
  float m = 0.f;
  for (int i = first + lane; i < last; i += 32) {
    float x[8];
    load8<KIND>(r.p, (w.token0 + i / per_row) * r.token_stride + h * r.head_stride + (i % per_row) * 8, vec, x);
#pragma unroll
    for (int e = 0; e < 8; ++e) m = fmaxf(m, finite_abs(x[e]));
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  const float now = fmaxf(old, fmaxf(__fmul_rn(m, 1.f / top_of(CODES)), kKvScaleFloor));
  const float inv = __fdiv_rn(1.f, now);
  for (int i = first + lane; i < last; i += 32) {
    float x[8];
    load8<KIND>(r.p, (w.token0 + i / per_row) * r.token_stride + h * r.head_stride + (i % per_row) * 8, vec, x);
    uint2 o;
    o.x = encode4<CODES>(__fmul_rn(x[0], inv), __fmul_rn(x[1], inv), __fmul_rn(x[2], inv), __fmul_rn(x[3], inv));
    o.y = encode4<CODES>(__fmul_rn(x[4], inv), __fmul_rn(x[5], inv), __fmul_rn(x[6], inv), __fmul_rn(x[7], inv));
    codes[i] = o;
  }
  if (now > old) {
    const float ratio = __fdiv_rn(old, now);
    for (int i = lane; i < first; i += 32) codes[i] = requant8<CODES>(codes[i], ratio);
  }
  __syncwarp();  // every lane has read the old scale
  if (lane == 0) *scale = now;
}

// Rows of one page, all heads of a group: 16 codes (one 16-byte load) a thread and step.  OUT 0 f32, 1 f16, 2 bf16.
template <int OUT, int CODES>
__global__ void __launch_bounds__(256)
    kv_read_kernel(KvCache c, KvSeqs s, const int32_t* __restrict__ first, void* __restrict__ k_out,
                   void* __restrict__ v_out, int heads_each) {
  const int64_t slot = blockIdx.x;
  const int b = kv_slot_seq_warp(s, slot, 1, c.page, 2);
  const int s0 = kv_start(s, b), n = kv_start(s, b + 1) - s0;
  const int64_t from = first ? __ldg(first + b) : 0;
  if (n <= 0 || from < 0) return;
  const int64_t pi = (from >> c.page_log2) + (slot - kv_slot_base(s, b, 1, c.page, 2));
  const int64_t p0 = pi << c.page_log2;
  if (p0 >= from + n) return;
  const int lo = from > p0 ? (int)(from - p0) : 0;
  const int hi = from + n - p0 < c.page ? (int)(from + n - p0) : c.page;
  const int64_t token0 = s0 + p0 - from;
  const int64_t page = kv_page(c, s, b, pi);
  const int h0 = blockIdx.y * heads_each, h1 = min(c.kv_heads, h0 + heads_each);
  const uint8_t* codes = blockIdx.z ? c.v : c.k;
  const float* scale = blockIdx.z ? c.v_scale : c.k_scale;
  void* out = blockIdx.z ? v_out : k_out;
  const int per_row = c.dim >> 4, per_head = (hi - lo) * per_row;
  const int total = per_head * (h1 - h0);
  for (int i0 = threadIdx.x; i0 < total; i0 += 256 * 4) {
    uint4 w[4];
    float sc[4];
    int64_t dst[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = i0 + u * 256;
      const int h = h0 + i / per_head, j = i % per_head, row = lo + j / per_row, col = (j % per_row) * 16;
      w[u] = make_uint4(0, 0, 0, 0);
      sc[u] = 0.f;
      dst[u] = -1;
      if (i < total) {
        dst[u] = ((token0 + row) * c.kv_heads + h) * c.dim + col;
        if (page >= 0) {  // a token without a page reads as zeros
          w[u] = __ldg(reinterpret_cast<const uint4*>(codes + ((page * c.kv_heads + h) * c.page + row) * c.dim + col));
          sc[u] = __ldg(scale + page * c.kv_heads + h);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (dst[u] < 0) continue;
      const uint32_t word[4] = {w[u].x, w[u].y, w[u].z, w[u].w};
      float f[16];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        float t[4];
        decode4f<CODES>(word[q], t);
#pragma unroll
        for (int e = 0; e < 4; ++e) f[4 * q + e] = __fmul_rn(t[e], sc[u]);
      }
      if (OUT == 0) {
        float4* d = reinterpret_cast<float4*>(reinterpret_cast<float*>(out) + dst[u]);
#pragma unroll
        for (int q = 0; q < 4; ++q) d[q] = make_float4(f[4 * q], f[4 * q + 1], f[4 * q + 2], f[4 * q + 3]);
      } else {
        uint4* d = reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(out) + dst[u]);
#pragma unroll
        for (int q = 0; q < 2; ++q)
          d[q] = make_uint4(kv_pack(f[8 * q], f[8 * q + 1], OUT), kv_pack(f[8 * q + 2], f[8 * q + 3], OUT),
                            kv_pack(f[8 * q + 4], f[8 * q + 5], OUT), kv_pack(f[8 * q + 6], f[8 * q + 7], OUT));
      }
    }
  }
}

template <int KIND, int CODES>
cudaError_t write_variant(const KvCache& c, const KvSeqs& s, const int32_t* past, const KvRows& k, const KvRows& v,
                          int vec, cudaStream_t st) {
  const int64_t slots = (int64_t)s.tokens / c.page + 2 * (int64_t)s.batch;
  if ((int64_t)s.tokens <= 4 * (int64_t)s.batch) {
    const int64_t warps = slots * c.kv_heads * 2;
    kv_write_few_kernel<KIND, CODES><<<(unsigned)((warps + 3) / 4), 128, 0, st>>>(c, s, past, k, v, vec, slots);
    return cudaGetLastError();
  }
  const dim3 grid((unsigned)slots, (unsigned)c.kv_heads, 2);
  switch (c.page * c.dim) {
    case 1024: kv_write_kernel<KIND, CODES, 128, 1><<<grid, 128, 0, st>>>(c, s, past, k, v, vec); break;
    case 2048: kv_write_kernel<KIND, CODES, 128, 2><<<grid, 128, 0, st>>>(c, s, past, k, v, vec); break;
    case 4096: kv_write_kernel<KIND, CODES, 128, 4><<<grid, 128, 0, st>>>(c, s, past, k, v, vec); break;
    case 8192: kv_write_kernel<KIND, CODES, 256, 4><<<grid, 256, 0, st>>>(c, s, past, k, v, vec); break;
    case 16384: kv_write_kernel<KIND, CODES, 512, 4><<<grid, 512, 0, st>>>(c, s, past, k, v, vec); break;
    default: return cudaErrorInvalidValue;
  }
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_kv_write(const KvCache& c, const KvSeqs& s, const int32_t* past, const void* k, int64_t k_ts,
                            int64_t k_hs, const void* v, int64_t v_ts, int64_t v_hs, int kind, bool vec,
                            cudaStream_t st) {
  const KvRows kr{k, k_ts, k_hs}, vr{v, v_ts, v_hs};
#define H3Q_KV_W(K, C) \
  if (kind == K && c.codes == C) return write_variant<K, C>(c, s, past, kr, vr, vec, st);
  H3Q_KV_W(0, 0) H3Q_KV_W(1, 0) H3Q_KV_W(2, 0) H3Q_KV_W(0, 1) H3Q_KV_W(1, 1) H3Q_KV_W(2, 1)
#undef H3Q_KV_W
  return cudaErrorInvalidValue;
}

cudaError_t launch_kv_read(const KvCache& c, const KvSeqs& s, const int32_t* first, void* k_out, void* v_out, int kind,
                           cudaStream_t st) {
  const int64_t slots = (int64_t)s.tokens / c.page + 2 * (int64_t)s.batch;
  // a CTA takes the heads of a page in groups: all of them where the pages alone fill the GPU, fewer where they do not
  int groups = 1;
  while (groups < c.kv_heads && slots * 2 * groups < (int64_t)sm_count(0) * 8) ++groups;
  const int each = (c.kv_heads + groups - 1) / groups;
  const dim3 grid((unsigned)slots, (unsigned)((c.kv_heads + each - 1) / each), 2);
#define H3Q_KV_R(K, C)                                                                 \
  if (kind == K && c.codes == C) {                                                     \
    kv_read_kernel<K, C><<<grid, 256, 0, st>>>(c, s, first, k_out, v_out, each);       \
    return cudaGetLastError();                                                         \
  }
  H3Q_KV_R(0, 0) H3Q_KV_R(1, 0) H3Q_KV_R(2, 0) H3Q_KV_R(0, 1) H3Q_KV_R(1, 1) H3Q_KV_R(2, 1)
#undef H3Q_KV_R
  return cudaErrorInvalidValue;
}

}  // namespace h3q
