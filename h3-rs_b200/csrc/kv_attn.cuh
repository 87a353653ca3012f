// kv_attn.cuh -- shared by the attention kernels over the 8-bit paged cache (kv_common.cuh): their arguments, the rows
// and keys of a slot, and the workspace that joins a slot's parts.
//
// With c = scale * log2(e) and keys j of page p, both scales leave the matrix products:
//     t_j = c ks_p (q . kcode_j),   w_j = 2^(t_j + log2 vs_p - m),   the largest w of a row between 2^7 and 2^15
//     O = sum_j w_j vcode_j,   l = sum_p 2^(m - u - log2 vs_p) sum_{j in p} w_j = sum_j 2^(t_j - u)
//     out = O 2^(m - u) / l,   lse = ln 2 (u + log2 l)
// so K and V enter the tensor cores as their codes, which 16-bit floats hold exactly, and one scale a page is applied
// in f32.  What is rounded is w (f16) and the output; m, u, l, the scores and O are f32.  m starts 7 below the largest t_j +
// log2 vs_p and moves when a w would pass 2^15: f16 has 11 bits of a weight down to 2^-21 of the largest and drops those below
// 2^-32 of it, so that what a key of nearly all the weight leaves to tens of thousands of others still adds up (with the
// largest at 1, 12800 equal keys with a hundredth of the weight between them lost 2 % of it).
//
// u is at most the row's largest t_j.  l has a reference of its own because scales of V may lie 2^220 apart (1e-30 of a page
// of zeros, 2^121 of the largest values): below 2^-126 w is 0, and a key counts in l whatever its values are.  While a
// page's factor 2^(m - u - log2 vs_p) is at most 2^kKvFar, w is 0 only for keys below 2^(kKvFar - 126) of the row's largest
// 2^t, which l has no bits for; beyond it a kernel sums 2^(t_j - u) itself, and raises u to the largest t_j that it sees there.
//
// q enters as f16: an f16 input as it is; a bf16 row times a power of two that brings its largest element near 1, which
// is exact but for elements below 2^-14 of the row's largest (their error is under 2^-25 of it).
#pragma once
#include "kv_common.cuh"

namespace h3q {

struct KvAttnArgs {
  KvCache c;
  KvSeqs s;
  const uint16_t* q;
  int64_t q_ts, q_hs;      // element strides of a token and a head
  int kind;                // 1 f16, 2 bf16 (q and out)
  int heads, per;          // query heads, and query heads to a kv head
  const int32_t* lengths;  // [batch] tokens in the cache, the new ones included
  int64_t window;          // 0: none
  int causal;
  float scale_log2;
  uint16_t* out;           // [tokens, heads, dim]
  float* lse;              // [tokens, heads] or null
  int row_lo, row_hi;      // this launch takes the sequences whose rows (new tokens * per) are in (row_lo, row_hi]
  int last;                // no launch takes sequences of more than row_hi rows
  int one;                 // every sequence of this launch has one slot, its own index
  int64_t slots;
  // Items (a slot and kv head) are cut between workers (CTAs); worker w's parts are 2 w (its first segment) and 2 w + 1.
  // A part is O of its rows, [rows][dim] (tiles of 16 and 32) or [dim / 4][rows][4] (tiles of 256), then (m, u, l, 0) a row.
  float* part;
  int4* meta;              // [workers]: slot, kv head, first part and parts of the item that w began and did not finish
  int workers;
};
constexpr float kKvTop = 15.f;           // log2 of the largest weight: f16 ends at 2^16, room for the rounding of t up to 2^23
constexpr float kKvLift = 7.f;           // log2 of the largest weight where m is set
constexpr float kKvFar = 80.f;           // log2 of a page's largest factor in l
constexpr float kKvNoRef = -3.402823466e38f;  // u of a row without keys: finite, so that differences are numbers or -inf
constexpr int kMaxWorkers = 256;         // of the chunk kernel: one a multiprocessor
constexpr int kMaxRowWorkers = 512;      // of the row kernel: up to three

// What a slot stands for: `rows` query rows of sequence b, (token, head of the group) in that order, the first of the
// sequence's new tokens at place `first`, the tokens `len` that the table has room for, and the keys [lo, hi) that any of
// the rows sees, lo a multiple of 16.
struct KvSlot {
  int b, s0, r0, rows;
  int64_t first, len, lo, hi;
};

__device__ __forceinline__ bool kv_slot(const KvAttnArgs& a, int64_t slot, int b, int tile, KvSlot& t) {
  const int s0 = kv_start(a.s, b), n = kv_start(a.s, b + 1) - s0;
  const int64_t all = (int64_t)n * a.per;  // beyond row_hi, which fits an int, only where a sequence breaks max_new
  t.rows = 0;
  t.lo = t.hi = 0;
  if (n <= 0 || all <= a.row_lo || all > a.row_hi) return false;
  const int64_t r0 = (slot - (a.one ? b : kv_slot_base(a.s, b, a.per, tile, 1))) * tile;
  if (r0 < 0 || r0 >= all) return false;  // (below 0: a slot before a first sequence that does not begin at row 0)
  t.b = b;
  t.s0 = s0;
  t.r0 = (int)r0;
  t.rows = (int)(all - r0 < tile ? all - r0 : tile);
  int64_t len = __ldg(a.lengths + b);
  len = len < 0 ? 0 : len;
  t.first = len - n;
  const int64_t most = a.s.width << a.c.page_log2;
  len = len > most ? most : len;  // what lies behind the table is not there; the queries keep their places
  t.len = len;
  const int64_t first = t.first + t.r0 / a.per, last = t.first + (t.r0 + t.rows - 1) / a.per;
  int64_t hi = a.causal ? (last + 1 < len ? last + 1 : len) : len;
  int64_t lo = a.window > 0 && first + 1 > a.window ? first + 1 - a.window : 0;
  hi = hi < 0 ? 0 : hi;
  t.lo = lo & ~(int64_t)15;
  t.hi = hi > t.lo ? hi : t.lo;
  return true;
}

// the keys [lo, hi) that row r of the slot sees
__device__ __forceinline__ void kv_row_keys(const KvAttnArgs& a, const KvSlot& t, int r, int64_t& lo, int64_t& hi) {
  const int64_t pos = t.first + (t.r0 + r) / a.per;
  hi = a.causal && pos + 1 < t.len ? pos + 1 : t.len;
  lo = a.window > 0 && pos + 1 > a.window ? pos + 1 - a.window : 0;
}

// packed row and query head of row r of the slot, as an index into [tokens, heads]
__device__ __forceinline__ int64_t kv_row_out(const KvAttnArgs& a, const KvSlot& t, int kvh, int r) {
  const int rr = t.r0 + r;
  return (int64_t)(t.s0 + rr / a.per) * a.heads + kvh * a.per + rr % a.per;
}

// For a bf16 row of largest magnitude mx: f, the power of two that brings it into [1, 4) ([1, 2) but for the last
// binade, whose inverse is no normal number; a row below the normal range comes out smaller), and c times its inverse.
__device__ __forceinline__ void kv_row_scale(float mx, float& f, float& c) {
  f = 1.f;
  if (mx > 0.f && mx < INFINITY) {
    int e = (int)(__float_as_uint(mx) >> 23) - 127;
    e = e < -126 ? -126 : (e > 126 ? 126 : e);
    f = __uint_as_float((uint32_t)(127 - e) << 23);
    c *= __uint_as_float((uint32_t)(127 + e) << 23);
  }
}

// A row's statistics, and what its sums O become its output by: O * inv * half * half (2^(m - u) in two factors, as it may be
// beyond a float where the product is not).  A row without keys: zeros; a NaN in l goes through.
struct KvStat {
  float m, u, l;
  __device__ __forceinline__ float inv() const { return l > 0.f ? __fdiv_rn(1.f, l) : (l == 0.f ? 0.f : l); }
  __device__ __forceinline__ float half() const { return kv_ex2(0.5f * (m - u)); }
  __device__ __forceinline__ float lse() const { return l == 0.f ? -INFINITY : 0.6931471805599453f * (u + log2f(l)); }
};

// four columns (chunk ch) of output row ro, from the unnormalised sums and the row's statistics
__device__ __forceinline__ void kv_put_row(const KvAttnArgs& a, int64_t ro, int ch, int dim, float4 o, const KvStat& e) {
  const float inv = e.inv(), f = e.half();
  uint2 w;
  w.x = kv_pack(o.x * inv * f * f, o.y * inv * f * f, a.kind);
  w.y = kv_pack(o.z * inv * f * f, o.w * inv * f * f, a.kind);
  *reinterpret_cast<uint2*>(a.out + ro * dim + ch * 4) = w;
  if (a.lse && ch == 0) a.lse[ro] = e.lse();
}

// joins the parts of items that were cut between CTAs, and writes the rows of slots without keys
cudaError_t launch_kv_attn_join(const KvAttnArgs& a, int tile, cudaStream_t st);

}  // namespace h3q
