// kv_common.cuh -- shared by the kernels of the 8-bit paged key / value cache: the cache's layout, the walk over
// ragged sequences, and the decode of codes into 16-bit floats.
//
// A cache is a pool of pages.  Page p of kv head h holds `page` tokens of D codes (int8 or e4m3) contiguously:
// codes [P, Hk, page, D], scales f32 [P, Hk] for K and for V, value = code * scale.  Sequence b's tokens
// i * page .. are in page table[b, i]; an entry outside [0, P) names no page and its tokens are not there.
#pragma once
#include <cstdint>
#include <cuda_runtime.h>
#include "ptx.cuh"

namespace h3q {

constexpr int kKvInt8 = 0, kKvE4m3 = 1;
constexpr float kKvScaleFloor = 1e-30f;  // the smallest scale a write leaves, as the row quantizer's

struct KvCache {
  uint8_t* k;
  uint8_t* v;
  float* k_scale;
  float* v_scale;
  int64_t pages;
  int kv_heads, page, page_log2, dim, codes;
};

// The sequences of one call: rows starts[b] .. starts[b + 1] of the packed token axis belong to sequence b
// (starts null: tokens / batch each).
struct KvSeqs {
  const int32_t* table;   // [batch, width]
  const int32_t* starts;  // [batch + 1] or null
  int64_t width;
  int batch;
  int tokens;
  int each;               // tokens / batch where starts is null
};

__device__ __forceinline__ int kv_start(const KvSeqs& s, int b) {
  if (!s.starts) return b * s.each;
  const int v = __ldg(s.starts + b);
  return v < 0 ? 0 : (v > s.tokens ? s.tokens : v);
}

// The rows that belong to no sequence, before the first and behind the last: their number, and the i-th of them.
struct KvRest {
  int before, end, n;
  __device__ __forceinline__ int row(int i) const { return i < before ? i : end + i - before; }
};
__device__ __forceinline__ KvRest kv_rest(const KvSeqs& s) {
  KvRest r;
  r.before = kv_start(s, 0);
  r.end = kv_start(s, s.batch);
  if (r.end < r.before) r.end = r.before;
  r.n = r.before + s.tokens - r.end;
  return r;
}

// page table[b, i], or -1 where the sequence has no such page
__device__ __forceinline__ int64_t kv_page(const KvCache& c, const KvSeqs& s, int b, int64_t i) {
  if (i < 0 || i >= s.width) return -1;
  const int64_t p = __ldg(s.table + (int64_t)b * s.width + i);
  return p >= 0 && p < c.pages ? p : -1;
}

// A call's work is cut into slots without a look at the lengths on the host: with `per` items to a slot, sequence b
// of n items owns slots floor(start * mul / per) + extra * b onwards.  floor(a + n) - floor(a) >= floor(n), so
// `extra` more than floor(n) slots are always there: one covers any n cut at its own start, two any n cut at
// an arbitrary offset.
__device__ __forceinline__ int64_t kv_slot_base(const KvSeqs& s, int b, int64_t mul, int64_t per, int extra) {
  return (int64_t)kv_start(s, b) * mul / per + (int64_t)extra * b;
}

// The sequence that owns `slot`: the last b with base(b) <= slot.  A whole warp searches, 32 candidates a step.
__device__ __forceinline__ int kv_slot_seq_warp(const KvSeqs& s, int64_t slot, int64_t mul, int64_t per, int extra) {
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = s.batch;  // answer in [lo, hi)
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32;
    const int b = lo + lane * step;
    const bool le = b < hi && kv_slot_base(s, b, mul, per, extra) <= slot;
    const unsigned m = __ballot_sync(0xffffffffu, le);
    const int last = m ? 31 - __clz(m) : 0;  // base is monotone, so the set lanes are a prefix
    lo += last * step;
    hi = lo + step < hi ? lo + step : hi;
  }
  return lo;
}

// The same by one thread.
__device__ __forceinline__ int kv_slot_seq(const KvSeqs& s, int64_t slot, int64_t mul, int64_t per, int extra) {
  int lo = 0, hi = s.batch;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (kv_slot_base(s, mid, mul, per, extra) <= slot) lo = mid;
    else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) {
  uint32_t r;
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(sel));
  return r;
}

// Four codes of a word as two f16 pairs, exactly.  int8: the byte with its sign bit flipped is u = q + 128; under
// the high byte 0x64 it is the f16 1024 + u, and 1024 + u - 1152 = q.  e4m3: every value is an f16.
template <int CODES>
__device__ __forceinline__ void kv_decode4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if (CODES == kKvInt8) {
    const uint32_t x = w ^ 0x80808080u;
    const uint32_t a = prmt(x, 0x64646464u, 0x4140), b = prmt(x, 0x64646464u, 0x4342);
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(lo) : "r"(a), "r"(0x64806480u));
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(hi) : "r"(b), "r"(0x64806480u));
  } else {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
  }
}

__device__ __forceinline__ float kv_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float kv_lg2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// low half: the first argument
__device__ __forceinline__ uint32_t kv_pack_f16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t kv_pack(float lo, float hi, int kind) {
  if (kind == 1) return kv_pack_f16(lo, hi);
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

}  // namespace h3q
