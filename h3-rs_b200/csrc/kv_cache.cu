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
// Measured (B200): four prompts of up to 8192 tokens, 8 heads of 128, bf16 to e4m3 in pages of 64: 26.9 us, and 23.8 us to
// read their pages back; 1019 tokens of 3 sequences, 40 heads, f32 to int8 in pages of 16 (106 MB): 30.2 us, 33 us back to
// f32; 16 sequences of up to 8192 read back to bf16 (490 MB): 87 us, 5.6 TB/s.  Copying the rows through shared memory four heads
// ahead of their maximum instead of one head ahead in registers: no gain (bf16), 41 against 30 us (f32).
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

// 8 elements of kind KIND as they lie in memory, and as f32
template <int KIND>
struct Raw8 {
  uint32_t w[KIND == 0 ? 8 : 4];
};
template <int KIND>
__device__ __forceinline__ void load8(const void* base, int64_t off, bool vec, Raw8<KIND>& r) {
  if (KIND == 0) {
    const uint32_t* p = reinterpret_cast<const uint32_t*>(base) + off;
    if (vec) {  // 16-byte loads are aligned
      const uint4 a = __ldg(reinterpret_cast<const uint4*>(p)), b = __ldg(reinterpret_cast<const uint4*>(p) + 1);
      r.w[0] = a.x; r.w[1] = a.y; r.w[2] = a.z; r.w[3] = a.w;
      r.w[KIND == 0 ? 4 : 0] = b.x; r.w[KIND == 0 ? 5 : 0] = b.y; r.w[KIND == 0 ? 6 : 0] = b.z; r.w[KIND == 0 ? 7 : 0] = b.w;
    } else {
#pragma unroll
      for (int i = 0; i < (KIND == 0 ? 8 : 4); ++i) r.w[i] = __ldg(p + i);
    }
  } else {
    const uint16_t* p = reinterpret_cast<const uint16_t*>(base) + off;
    if (vec) {
      const uint4 a = __ldg(reinterpret_cast<const uint4*>(p));
      r.w[0] = a.x; r.w[1] = a.y; r.w[2] = a.z; r.w[3] = a.w;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) r.w[i] = (uint32_t)__ldg(p + 2 * i) | ((uint32_t)__ldg(p + 2 * i + 1) << 16);
    }
  }
}
template <int KIND>
__device__ __forceinline__ void as_float8(const Raw8<KIND>& r, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (KIND == 0) {
      f[2 * i] = __uint_as_float(r.w[KIND == 0 ? 2 * i : 0]);
      f[2 * i + 1] = __uint_as_float(r.w[KIND == 0 ? 2 * i + 1 : 0]);
    } else {
      f[2 * i] = KIND == 1 ? h2f((uint16_t)r.w[i]) : __uint_as_float(r.w[i] << 16);
      f[2 * i + 1] = KIND == 1 ? h2f((uint16_t)(r.w[i] >> 16)) : __uint_as_float(r.w[i] & 0xffff0000u);
    }
  }
}
__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a <= 3.402823466e38f ? a : 0.f;  // NaN and infinity compare false
}

// Magnitudes as bits, which order as the numbers do: NaN above infinity above the finite ones.  16-bit kinds keep two
// running maxima in the halves of a word.
template <int KIND>
__device__ __forceinline__ void max_bits8(const Raw8<KIND>& r, uint32_t& m) {
#pragma unroll
  for (int i = 0; i < (KIND == 0 ? 8 : 4); ++i)
    m = KIND == 0 ? max(m, r.w[i] & 0x7fffffffu) : __vmaxu2(m, r.w[i] & 0x7fff7fffu);
}
template <int KIND>
__device__ __forceinline__ uint32_t whole_bits(uint32_t m) {  // the larger half, or the word
  return KIND == 0 ? m : max(m & 0xffffu, m >> 16);
}
template <int KIND>
__device__ __forceinline__ float bits_value(uint32_t m) {
  return KIND == 0 ? __uint_as_float(m) : KIND == 1 ? h2f((uint16_t)m) : __uint_as_float(m << 16);
}

// the largest finite magnitude
template <int KIND>
__device__ __forceinline__ float amax8(const Raw8<KIND>& r) {
  float f[8], m = 0.f;
  as_float8<KIND>(r, f);
#pragma unroll
  for (int e = 0; e < 8; ++e) m = fmaxf(m, finite_abs(f[e]));
  return m;
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
  const int64_t nth = slot - kv_slot_base(s, b, 1, c.page, 2);
  if (n <= 0 || nth < 0) return false;  // (below 0: a slot before a first sequence that does not begin at row 0)
  const int64_t i = (had >> c.page_log2) + nth;
  const int64_t p0 = i << c.page_log2;
  if (p0 >= had + n) return false;  // (a place before 0 has no page, like one behind the table's end)
  w.page = kv_page(c, s, b, i);  // -1: the page is not there; its tokens are dropped
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

// Codes of rows without NaN or infinity whose scale is at least their largest magnitude / top: no product is beyond
// +-top by more than its rounding, so nothing saturates and int8 rounds by adding 1.5 * 2^23 (nearest even, as the
// conversion does), which leaves the code in the low byte.
template <int KIND, int CODES>
__device__ __forceinline__ uint2 encode8_finite(const Raw8<KIND>& r, float inv) {
  float f[8];
  as_float8<KIND>(r, f);
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (CODES == kKvInt8) {
      uint32_t q[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) q[e] = __float_as_uint(__fadd_rn(__fmul_rn(f[4 * i + e], inv), 12582912.f));
      w[i] = prmt(prmt(q[0], q[1], 0x0040), prmt(q[2], q[3], 0x0040), 0x5410);
    } else {
      uint16_t lo, hi;
      asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;"
          : "=h"(lo)
          : "f"(__fmul_rn(f[4 * i + 1], inv)), "f"(__fmul_rn(f[4 * i], inv)));
      asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;"
          : "=h"(hi)
          : "f"(__fmul_rn(f[4 * i + 3], inv)), "f"(__fmul_rn(f[4 * i + 2], inv)));
      w[i] = (uint32_t)lo | ((uint32_t)hi << 16);
    }
  }
  return make_uint2(w[0], w[1]);
}

template <int KIND, int CODES>
__device__ __forceinline__ uint2 encode8(const Raw8<KIND>& r, float inv) {
  float f[8];
  as_float8<KIND>(r, f);
  return make_uint2(encode4<CODES>(__fmul_rn(f[0], inv), __fmul_rn(f[1], inv), __fmul_rn(f[2], inv), __fmul_rn(f[3], inv)),
                    encode4<CODES>(__fmul_rn(f[4], inv), __fmul_rn(f[5], inv), __fmul_rn(f[6], inv), __fmul_rn(f[7], inv)));
}

// One CTA for a page of K or V and a group of heads, one head after the other: a head's new rows stay in registers
// between the maximum and the codes, so the input is read once, and the next head's rows are on their way meanwhile.
// VPT vectors of 8 elements a thread: THREADS * VPT * 8 = page * dim.  Maxima are taken on the bits, two of 16 an instruction.
template <int KIND, int CODES, int THREADS, int VPT>
__global__ void __launch_bounds__(THREADS, KIND == 0 ? 768 / THREADS : 1024 / THREADS)
    kv_write_kernel(KvCache c, KvSeqs s, const int32_t* __restrict__ past, KvRows kr, KvRows vr, int vec, int heads_each) {
  const int64_t slot = blockIdx.x;
  const int b = kv_slot_seq_warp(s, slot, 1, c.page, 2);
  WritePage w;
  if (!write_page(c, s, past, slot, b, w)) return;
  const KvRows r = blockIdx.z ? vr : kr;
  const int h0 = blockIdx.y * heads_each, h1 = min(c.kv_heads, h0 + heads_each);
  const int row_log2 = c.dim == 64 ? 3 : 4;  // vectors of a row
  const bool held = w.lo > 0;
  // vector j of the thread: row (threadIdx.x + j * THREADS) >> row_log2 of the page
  const int row0 = threadIdx.x >> row_log2, row_step = THREADS >> row_log2;
  const int64_t first = (w.token0 + row0) * r.token_stride + (threadIdx.x & ((1 << row_log2) - 1)) * 8;
  Raw8<KIND> x[VPT], y[VPT];
  auto is_new = [&](int j) { return row0 + j * row_step >= w.lo && row0 + j * row_step < w.hi; };
  auto load = [&](int h, Raw8<KIND>(&d)[VPT]) {
    const int64_t at = first + h * r.head_stride;
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      if (is_new(j)) {
        load8<KIND>(r.p, at + j * row_step * r.token_stride, vec, d[j]);
      } else {
#pragma unroll
        for (int e = 0; e < (KIND == 0 ? 8 : 4); ++e) d[j].w[e] = 0;
      }
    }
  };
  load(h0, x);
  if (w.page < 0) return;
  float* scale = (blockIdx.z ? c.v_scale : c.k_scale) + w.page * c.kv_heads;
  uint2* codes = reinterpret_cast<uint2*>((blockIdx.z ? c.v : c.k) + w.page * c.kv_heads * c.page * c.dim);
  __shared__ uint32_t part[2][THREADS / 32], again[THREADS / 32];
  float old = held ? scale[h0] : 0.f;
  for (int h = h0; h < h1; ++h) {
    const bool more = h + 1 < h1;
    float old_next = 0.f;
    if (more) {
      load(h + 1, y);
      old_next = held ? scale[h + 1] : 0.f;
    }
    uint32_t mb = 0;
#pragma unroll
    for (int j = 0; j < VPT; ++j) max_bits8<KIND>(x[j], mb);
    mb = __reduce_max_sync(0xffffffffu, whole_bits<KIND>(mb));
    if ((threadIdx.x & 31) == 0) part[h & 1][threadIdx.x >> 5] = mb;
    __syncthreads();  // one a head: the other half of `part` is not written before every thread has passed the next one
#pragma unroll
    for (int i = 0; i < THREADS / 32; ++i) mb = max(mb, part[h & 1][i]);
    float m = bits_value<KIND>(mb);
    const bool finite = m <= 3.402823466e38f;
    if (!finite) {  // rare: the maximum again, without what is not finite
      m = 0.f;
#pragma unroll
      for (int j = 0; j < VPT; ++j) m = fmaxf(m, amax8<KIND>(x[j]));
      mb = __reduce_max_sync(0xffffffffu, __float_as_uint(m));
      if ((threadIdx.x & 31) == 0) again[threadIdx.x >> 5] = mb;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < THREADS / 32; ++i) mb = max(mb, again[i]);
      m = __uint_as_float(mb);
      __syncthreads();  // read before another head may come here
    }
    const float now = fmaxf(old, fmaxf(__fmul_rn(m, 1.f / top_of(CODES)), kKvScaleFloor));
    const float inv = __fdiv_rn(1.f, now);
    uint2* dst = codes + (int64_t)h * (THREADS * VPT);
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const int i = threadIdx.x + j * THREADS;
      if (is_new(j)) dst[i] = finite ? encode8_finite<KIND, CODES>(x[j], inv) : encode8<KIND, CODES>(x[j], inv);
      else if (row0 + j * row_step < w.lo && now > old) dst[i] = requant8<CODES>(dst[i], __fdiv_rn(old, now));
    }
    if (threadIdx.x == 0) scale[h] = now;  // every thread has read the old scale of head h a head ago
#pragma unroll
    for (int j = 0; j < VPT; ++j) x[j] = y[j];
    old = old_next;
  }
}

// One warp for a page of a head of K or V, for calls of up to four tokens a sequence on average, where a CTA a page would
// idle: two passes over the few new rows (the second hits L1), 8 elements a lane.  Bound by the latency of its chain of loads
// (lengths, page table, rows, scale).  Against a CTA a page (bf16 to int8, head dim 128): 64 sequences, 8 heads, page 64: one
// token 3.4 and 8.0 us, four 4.0 and 8.3, sixteen 6.9 and 9.2; 40 heads, page 16: four tokens 9.1 and 10.6, sixteen 20.7 and
// 18.0; one sequence: one token 2.3 and 2.6, four 2.7 and 2.6, sixteen 4.8 and 2.7.
template <int KIND, int CODES>
__global__ void __launch_bounds__(128)
    kv_write_few_kernel(KvCache c, KvSeqs s, const int32_t* __restrict__ past, KvRows kr, KvRows vr, int vec,
                        uint32_t slots) {
  const int lane = threadIdx.x & 31;
  const uint32_t unit = blockIdx.x * 4 + (threadIdx.x >> 5);
  const uint32_t slot = unit / (2 * c.kv_heads);
  if (slot >= slots) return;
  const int rest = (int)(unit % (2 * c.kv_heads)), h = rest >> 1, isv = rest & 1;
  const int b = kv_slot_seq_warp(s, slot, 1, c.page, 2);
  WritePage w;
  if (!write_page(c, s, past, slot, b, w)) return;
  const KvRows r = isv ? vr : kr;
  const int row_log2 = c.dim == 64 ? 3 : 4;  // vectors of a row
  const int first = w.lo << row_log2, last = w.hi << row_log2;
  auto load = [&](int i, Raw8<KIND>& x) {
    load8<KIND>(r.p, (w.token0 + (i >> row_log2)) * r.token_stride + h * r.head_stride + (i & ((1 << row_log2) - 1)) * 8, vec, x);
  };
  Raw8<KIND> x;  // the lane's first vector, which is the only one for one or two tokens
  const bool any = first + lane < last;
  if (any) load(first + lane, x);
  if (w.page < 0) return;
  const int64_t ph = w.page * c.kv_heads + h;
  float* scale = (isv ? c.v_scale : c.k_scale) + ph;
  uint2* codes = reinterpret_cast<uint2*>((isv ? c.v : c.k) + ph * c.page * c.dim);
  const float old = w.lo > 0 ? *scale : 0.f;
  float m = any ? amax8<KIND>(x) : 0.f;
  for (int i = first + lane + 32; i < last; i += 32) {
    Raw8<KIND> y;
    load(i, y);
    m = fmaxf(m, amax8<KIND>(y));
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  const float now = fmaxf(old, fmaxf(__fmul_rn(m, 1.f / top_of(CODES)), kKvScaleFloor));
  const float inv = __fdiv_rn(1.f, now);
  if (any) codes[first + lane] = encode8<KIND, CODES>(x, inv);
  for (int i = first + lane + 32; i < last; i += 32) {
    load(i, x);
    codes[i] = encode8<KIND, CODES>(x, inv);
  }
  if (now > old) {
    const float ratio = __fdiv_rn(old, now);
    for (int i = lane; i < first; i += 32) codes[i] = requant8<CODES>(codes[i], ratio);
  }
  __syncwarp();  // every lane has read the old scale
  if (lane == 0) *scale = now;
}

// Rows of one page, all heads of a group: 16 codes (one 16-byte load) a thread and step.  OUT 0 f32, 1 f16, 2 bf16.  Rows of
// no sequence are dealt to the blocks of a group of heads, and are zeros.
template <int OUT, int CODES>
__global__ void __launch_bounds__(256)
    kv_read_kernel(KvCache c, KvSeqs s, const int32_t* __restrict__ first, void* __restrict__ k_out,
                   void* __restrict__ v_out, int heads_each) {
  const int64_t slot = blockIdx.x;
  const int h0 = blockIdx.y * heads_each, h1 = min(c.kv_heads, h0 + heads_each);
  void* out = blockIdx.z ? v_out : k_out;
  const KvRest rest = kv_rest(s);
  const int b = kv_slot_seq_warp(s, slot, 1, c.page, 2);
  for (int i = blockIdx.x; i < rest.n; i += gridDim.x) {
    constexpr int size = OUT == 0 ? 4 : 2;
    uint4* d = reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(out) +
                                        ((int64_t)rest.row(i) * c.kv_heads + h0) * c.dim * size);
    for (int k = threadIdx.x; k < (h1 - h0) * c.dim * size / 16; k += 256) d[k] = make_uint4(0, 0, 0, 0);
  }
  const int s0 = kv_start(s, b), n = kv_start(s, b + 1) - s0;
  const int64_t from = first ? __ldg(first + b) : 0;
  const int64_t nth = slot - kv_slot_base(s, b, 1, c.page, 2);
  if (n <= 0 || nth < 0) return;
  const int64_t pi = (from >> c.page_log2) + nth;
  const int64_t p0 = pi << c.page_log2;
  if (p0 >= from + n) return;
  const int lo = from > p0 ? (int)(from - p0) : 0;
  const int hi = from + n - p0 < c.page ? (int)(from + n - p0) : c.page;
  const int64_t token0 = s0 + p0 - from;
  const int64_t page = kv_page(c, s, b, pi);
  const uint8_t* codes = blockIdx.z ? c.v : c.k;
  const float* scale = blockIdx.z ? c.v_scale : c.k_scale;
  // The codes of the heads of a page follow one another, `page` rows each: vector v of the group is 16 codes of head
  // h0 + v / vectors_of_a_head, and every division is a shift.
  const int row_log2 = c.dim == 64 ? 2 : 3, head_log2 = c.page_log2 + row_log2;
  const uint4* src = reinterpret_cast<const uint4*>(codes + ((page < 0 ? 0 : page) * c.kv_heads + h0) * c.page * c.dim);
  const float* sc0 = scale + (page < 0 ? 0 : page) * c.kv_heads + h0;
  const int total = (h1 - h0) << head_log2;
  for (int i0 = threadIdx.x; i0 < total; i0 += 256 * 4) {
    uint4 w[4];
    float sc[4];
    int64_t dst[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = i0 + u * 256, h = i >> head_log2, row = (i >> row_log2) & (c.page - 1);
      w[u] = make_uint4(0, 0, 0, 0);
      sc[u] = 0.f;
      dst[u] = -1;
      if (i < total && row >= lo && row < hi) {
        dst[u] = ((token0 + row) * c.kv_heads + h0 + h) * c.dim + (i & ((1 << row_log2) - 1)) * 16;
        if (page >= 0) {  // a token without a page reads as zeros
          w[u] = __ldg(src + i);
          sc[u] = __ldg(sc0 + h);
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

// Heads a CTA takes: all of them where the pages alone fill the GPU (2048 threads a multiprocessor), fewer where they do
// not.  Many share the walk to the page and overlap its loads (16 sequences of up to 8192 read back: 87 us, 173 us with one head a
// CTA), few fill the GPU (777 tokens read back: 3.6 us, 9.2 us with all eight).
int heads_each(const KvCache& c, int64_t slots, int threads) {
  int groups = 1;
  while (groups < c.kv_heads && slots * 2 * groups * threads < (int64_t)sm_count(0) * 2048) ++groups;
  return (c.kv_heads + groups - 1) / groups;
}

template <int KIND, int CODES>
cudaError_t write_variant(const KvCache& c, const KvSeqs& s, const int32_t* past, const KvRows& k, const KvRows& v,
                          int vec, cudaStream_t st) {
  const int64_t slots = (int64_t)s.tokens / c.page + 2 * (int64_t)s.batch;
  if ((int64_t)s.tokens <= 4 * (int64_t)s.batch) {
    const int64_t warps = slots * c.kv_heads * 2;
    if (warps >= (int64_t)1 << 32) return cudaErrorInvalidValue;
    kv_write_few_kernel<KIND, CODES><<<(unsigned)((warps + 3) / 4), 128, 0, st>>>(c, s, past, k, v, vec, (uint32_t)slots);
    return cudaGetLastError();
  }
  const int each = heads_each(c, slots, c.page * c.dim <= 4096 ? 128 : c.page * c.dim / 32);
  const dim3 grid((unsigned)slots, (unsigned)((c.kv_heads + each - 1) / each), 2);
  switch (c.page * c.dim) {
    case 1024: kv_write_kernel<KIND, CODES, 128, 1><<<grid, 128, 0, st>>>(c, s, past, k, v, vec, each); break;
    case 2048: kv_write_kernel<KIND, CODES, 128, 2><<<grid, 128, 0, st>>>(c, s, past, k, v, vec, each); break;
    case 4096: kv_write_kernel<KIND, CODES, 128, 4><<<grid, 128, 0, st>>>(c, s, past, k, v, vec, each); break;
    case 8192: kv_write_kernel<KIND, CODES, 256, 4><<<grid, 256, 0, st>>>(c, s, past, k, v, vec, each); break;
    case 16384: kv_write_kernel<KIND, CODES, 512, 4><<<grid, 512, 0, st>>>(c, s, past, k, v, vec, each); break;
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
  const int each = heads_each(c, slots, 256);
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
