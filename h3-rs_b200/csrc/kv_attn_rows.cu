// kv_attn_rows.cu -- attention over the 8-bit paged cache for few query rows to a kv head (one generated token, a few
// drafted ones): bound by reading the cache once.
//
// The rows of a (sequence, kv head) -- its new tokens times the query heads that share the kv head -- are the 16 (or
// 2 x 16) rows of mma.sync.m16n8k16 tiles, so the codes of a kv head are read once for all of them.  A warp takes 16
// keys a step: 2 KB of K and of V codes arrive by cp.async in a ring of its own, are widened to f16 in registers and
// go straight into the fragments.  The order of the head dim in Q.K and of the columns of O is free, so it is chosen to make
// every lane's codes contiguous: lane (g, t) of the B fragment of K holds d = 32 t .. 32 t + 31 of key g, and of V
// d = 16 g .. 16 g + 15 of keys 2t, 2t + 1, 2t + 8, 2t + 9.  The ring is swizzled so that both reads are free of
// bank conflicts.
//
// Work is cut by keys, not by sequences: the units (64 keys of a sequence and kv head) of the whole call, in order,
// are dealt to the CTAs in equal contiguous ranges.  A CTA's four warps take the 16-key steps of a range in turn and
// join their running (m, l, O) at its end; a (sequence, kv head) cut between CTAs goes through f32 parts in the
// workspace, joined in order by a second kernel, so results do not depend on timing.  The chain of loads at the begin
// of a range's next sequence (lengths, page table, codes) takes about 3 us; three CTAs a multiprocessor (two of 32 rows) hide it
// behind each other's work, which one CTA of twelve warps could not, not even by starting it ahead of the join (64
// sequences of 1024 tokens, 8 kv heads: 52.4 us with one CTA, 53.7 with the early start, 40.2 with three; two warps and
// six CTAs: 39.4, but 5 us more to join and 47.9 against 40.8 us for 25 rows).
//
// Measured (B200; head dim 128, 8 kv heads): one token of 64 sequences of up to 16384, int8, 5 query heads to a kv head,
// 1.2 GB: 224 us, 5.4 TB/s; one of a sequence of 131000, 268 MB: 58 us, 4.6 TB/s; five of 16 sequences of up to 4099
// (25 rows), e4m3: 42 us.  The copies alone reach 6.1 TB/s in the first: what keeps the rest is the widening of codes (five
// instructions for four; the ALU pipe is busy 45 % of the time) and its latencies, with 12 warps a multiprocessor for their
// registers.  Tried and slower: scores in two accumulator chains (spills), two steps at a time (spills), 14 warps.
#include <cstdint>
#include <cuda_runtime.h>
#include "kv_attn.cuh"
#include "h3q_internal.h"

namespace h3q {

namespace {

template <int D, int MT>
struct RowsCfg {
  static constexpr int kWarps = 4, kThreads = kWarps * 32;
  static constexpr int kCtas = MT == 1 ? 3 : 2;    // of a multiprocessor
  static constexpr int kUnit = kWarps * 16;  // keys of a unit
  static constexpr int kStages = MT == 1 ? 3 : 4;
  static constexpr int kStageBytes = 2 * 16 * D;           // K and V codes of 16 keys
  static constexpr int kRing = kStages * kStageBytes;      // a warp's ring; its O of 16 MT rows fits there too
  static constexpr int kQBytes = MT * 16 * D * 2;
  static constexpr int kSmem = kWarps * kRing + kQBytes;
  static_assert(kRing >= MT * 16 * D * 4, "the ring holds a warp's partial output");
};

__device__ __forceinline__ void cp16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 r;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(a) : "memory");
  return r;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
  uint2 r;
  asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(r.x), "=r"(r.y) : "r"(a) : "memory");
  return r;
}
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// byte offset of 16-byte chunk `ch` of key row `row` in a 16-key tile of D bytes a row
template <int D>
__device__ __forceinline__ uint32_t tile_off(int row, int ch) {
  if (D == 128) return (uint32_t)(row * 128 + ((ch ^ (row & 7)) << 4));
  return (uint32_t)((row >> 1) * 128 + (((((row & 1) << 2) | ch) ^ (2 * ((row >> 1) & 3))) << 4));
}

// The units of the call in order, and this CTA's place in them: the units of kThreads slots at a time in shared
// memory with their running sum.
template <int W>
struct Sched {
  static constexpr int kWarps = W, kThreads = W * 32;
  int units[kThreads], pre[kThreads], seq[kThreads];
  int warp_sum[kWarps];
  int found;
};

template <int TILE, int UNIT>
__device__ __forceinline__ int slot_units(const KvAttnArgs& a, int64_t slot, int& b) {
  b = 0;
  if (slot >= a.slots) return 0;
  b = a.one ? (int)slot : kv_slot_seq(a.s, slot, a.per, TILE, 1);
  KvSlot t;
  if (!kv_slot(a, slot, b, TILE, t)) return 0;
  return (int)((t.hi - t.lo + UNIT - 1) / UNIT);
}

// Fills `sc` with the slots from `base` on; returns the sum of their units.  All threads of the CTA.
template <int TILE, int W>
__device__ __forceinline__ int sched_load(const KvAttnArgs& a, Sched<W>& sc, int64_t base) {
  constexpr int kWarps = W;
  __syncthreads();
  int b;
  const int u = slot_units<TILE, W * 16>(a, base + threadIdx.x, b);
  int x = u;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) sc.warp_sum[warp] = x;
  __syncthreads();
  int before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before += sc.warp_sum[w];
    total += sc.warp_sum[w];
  }
  sc.units[threadIdx.x] = u;
  sc.pre[threadIdx.x] = before + x - u;
  sc.seq[threadIdx.x] = b;
  __syncthreads();
  return total;
}

template <int D, int CODES, int MT>
__global__ void __launch_bounds__(RowsCfg<D, MT>::kThreads, RowsCfg<D, MT>::kCtas) kv_attn_rows_kernel(const KvAttnArgs a) {
  using C = RowsCfg<D, MT>;
  constexpr int TILE = MT * 16, NT = D / 8, kWarps = C::kWarps, kThreads = C::kThreads, kUnit = C::kUnit;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ Sched<kWarps> sc;
  __shared__ float row_c[TILE];                   // c of the row: scale * log2 e and the power of two taken out of q
  __shared__ KvStat ml[kWarps][TILE], ml_all[TILE];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
  uint8_t* ring = smem + warp * C::kRing;
  const uint32_t ring_u = smem_u32(ring);
  const uint32_t q_u = smem_u32(smem + kWarps * C::kRing);

  // the sum of all units, and this CTA's range of them
  int64_t all = 0;
  int here = 0;
  for (int64_t base = 0; base < a.slots; base += kThreads) {
    here = sched_load<TILE, kWarps>(a, sc, base);
    all += here;
  }
  all *= a.c.kv_heads;
  // no more workers than units: every worker's range then holds a unit, and an item's parts are consecutive workers'
  const int64_t workers = all < gridDim.x ? all : gridDim.x, w = blockIdx.x;
  if (w >= workers) {
    if (threadIdx.x == 0) a.meta[w] = make_int4(0, 0, 0, 0);
    return;
  }
  int64_t x = all * w / workers;
  const int64_t x_end = all * (w + 1) / workers;
  // find x: the slots' units before `base`, then inside the chunk
  int64_t base = 0, before = 0;
  if (a.slots > kThreads) here = sched_load<TILE, kWarps>(a, sc, 0);
  while (x >= (before + here) * a.c.kv_heads) {
    before += here;
    base += kThreads;
    here = sched_load<TILE, kWarps>(a, sc, base);
  }
  {
    const int64_t p0 = (before + sc.pre[threadIdx.x]) * a.c.kv_heads;
    if (x >= p0 && x < p0 + (int64_t)sc.units[threadIdx.x] * a.c.kv_heads) sc.found = threadIdx.x;
  }
  __syncthreads();
  int li = sc.found;
  bool first_segment = true, cut = false;
  const int group_log2 = a.c.page_log2 - 4, group_mask = (1 << group_log2) - 1;  // 16-key groups of a page
  const uint32_t pool = (uint32_t)a.c.pages;
  const int64_t page_bytes = (int64_t)a.c.kv_heads * a.c.page * D;
  // Places in a 16-key tile.  Copies: lane's 16-byte piece of rows lane / (D / 16) + 32 i / (D / 16).
  const uint32_t cp_off[2] = {tile_off<D>(lane / (D / 16), lane % (D / 16)),
                              tile_off<D>((lane + 32) / (D / 16), (lane + 32) % (D / 16))};
  // K: codes 32 t .. of key g (D = 128; the second 16 bytes are the place with bit 4 flipped) or 16 t .. (D = 64).
  const uint32_t k_off = tile_off<D>(g, t4 * (D / 64));
  // V: codes (D / 8) g .. of key 2 t; key 2 t + 1 is beside it, keys 2 t + 8 and + 9 eight rows on.
  const uint32_t v_off0 = tile_off<D>(2 * t4, g * (D / 8) / 16) + (g * (D / 8)) % 16;
  const uint32_t v_off1 = tile_off<D>(2 * t4 + 1, g * (D / 8) / 16) + (g * (D / 8)) % 16;

  while (true) {
    // ---------------------------------------------------------------- the segment: units [u0, u1) of (slot, kvh)
    const int units = sc.units[li];
    const int64_t item0 = (before + sc.pre[li]) * a.c.kv_heads;  // units before the slot
    const int kvh = (int)((x - item0) / units);
    const int u0 = (int)((x - item0) % units);
    const int u1 = (int)(x_end - x < units - u0 ? u0 + (x_end - x) : units);
    const bool whole = u0 == 0 && u1 == units;
    KvSlot sl;
    kv_slot(a, base + li, sc.seq[li], TILE, sl);
    const int64_t key0 = sl.lo + (int64_t)u0 * kUnit;
    const int64_t key1 = sl.lo + (int64_t)u1 * kUnit < sl.hi ? sl.lo + (int64_t)u1 * kUnit : sl.hi;
    const int steps_all = (int)((key1 - key0 + 15) / 16);
    const int steps = steps_all > warp ? (steps_all - warp + kWarps - 1) / kWarps : 0;
    const int group0 = (int)(key0 / 16) + warp;
    const int32_t* table = a.s.table + (int64_t)sl.b * a.s.width;
    const float* k_scale = a.c.k_scale + kvh;
    const float* v_scale = a.c.v_scale + kvh;

    // table entry of step st or of the last one (keys below sl.hi lie within the table's width; a warp without a step
    // looks at the item's first page).  It is looked at only where it is used, steps later: the load is not waited for here.
    auto entry_of = [&](int st) -> int {
      const int grp = steps > 0 ? group0 + min(st, steps - 1) * kWarps : group0 - warp;
      return __ldg(table + (grp >> group_log2));
    };
    auto issue = [&](int st, int page, uint32_t dst) {
      if ((uint32_t)page < pool && st < steps) {
        const int64_t off = page * page_bytes + lane * 16 +
                            (int64_t)(((kvh << group_log2) + ((group0 + st * kWarps) & group_mask)) * (16 * D));
        const uint8_t* ks = a.c.k + off;
        const uint8_t* vs = a.c.v + off;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
          const uint32_t o = dst + cp_off[i & 1] + (i >> 1) * 1024;
          cp16(o, ks + i * 512);
          cp16(o + 16 * D, vs + i * 512);
        }
      }
      cp_commit();
    };

    int pages[C::kStages + 1];  // pages of the steps from the one consumed next on
#pragma unroll
    for (int i = 0; i <= C::kStages; ++i) pages[i] = entry_of(i);
    uint32_t cur = ring_u, put = ring_u;
    auto next = [&](uint32_t& x) {
      x += C::kStageBytes;
      if (x == ring_u + C::kRing) x = ring_u;
    };
#pragma unroll
    for (int i = 0; i < C::kStages - 1; ++i) {
      issue(i, pages[i], put);
      next(put);
    }
    auto scale_of = [&](const float* s, int page) {
      return __ldg(s + (int64_t)((uint32_t)page < pool ? page : 0) * a.c.kv_heads);
    };
    float ks_next = scale_of(k_scale, pages[0]), vs_next = scale_of(v_scale, pages[0]);

    // ---------------------------------------------------------------- q: f16 in the order of the A fragments
    for (int r = warp; r < TILE; r += kWarps) {
      float f[D / 32];
      float mx = 0.f;
      const bool in = r < sl.rows;
      const int rr = sl.r0 + r;
      const uint16_t* src =
          a.q + (int64_t)(sl.s0 + rr / a.per) * a.q_ts + (int64_t)(kvh * a.per + rr % a.per) * a.q_hs;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        const uint16_t v = in ? __ldg(src + lane + 32 * i) : (uint16_t)0;
        f[i] = a.kind == 1 ? h2f(v) : bf2f(v);
        mx = fmaxf(mx, fabsf(f[i]));
      }
      float c = a.scale_log2;
      if (a.kind == 2) {
#pragma unroll
        for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        float p2;
        kv_row_scale(mx, p2, c);
#pragma unroll
        for (int i = 0; i < D / 32; ++i) f[i] *= p2;
      }
      if (lane == 0) row_c[r] = c;
      // element d of the row: lane t = d / (D / 4) of the quad, its element e = d % (D / 4), k-step e / 4; the four
      // registers of a fragment are (row g, first pair), (row g + 8, first), (row g, second), (row g + 8, second)
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        const int d = lane + 32 * i, tt = d / (D / 4), e = d % (D / 4);
        const int mt = r >> 4, half = (r >> 3) & 1, gg = r & 7;
        const uint32_t o = (uint32_t)(((mt * (D / 16) + e / 4) * 32 + gg * 4 + tt) * 16 + ((e & 2) + half) * 4 + (e & 1) * 2);
        asm volatile("st.shared.b16 [%0], %1;" ::"r"(q_u + o), "h"(f2h(f[i])) : "memory");
      }
    }
    __syncthreads();

    float o_acc[MT][NT][4];
    float m_run[MT][2], u_run[MT][2], l_run[MT][2], cr[MT][2];
    int rlo[MT][2], rhi[MT][2];  // the row's keys, relative to key0
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o_acc[mt][j][e] = 0.f;
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        const int r = mt * 16 + hf * 8 + g;
        m_run[mt][hf] = -INFINITY;
        u_run[mt][hf] = kKvNoRef;
        l_run[mt][hf] = 0.f;
        cr[mt][hf] = row_c[r];
        int64_t lo = 0, hi = 0;
        if (r < sl.rows) kv_row_keys(a, sl, r, lo, hi);
        lo -= key0;
        hi -= key0;
        rlo[mt][hf] = (int)(lo < 0 ? 0 : (lo > 0x3fffffff ? 0x3fffffff : lo));
        rhi[mt][hf] = (int)(hi < 0 ? 0 : (hi > 0x3fffffff ? 0x3fffffff : hi));
      }
    }
    // keys of this segment that every row sees need no mask
    const int64_t pos0 = sl.first + sl.r0 / a.per, pos1 = sl.first + (sl.r0 + sl.rows - 1) / a.per;
    const int64_t all_hi64 = (a.causal && pos0 + 1 < sl.len ? pos0 + 1 : sl.len) - key0;
    const int64_t all_lo64 = (a.window > 0 && pos1 + 1 > a.window ? pos1 + 1 - a.window : 0) - key0;
    const int all_hi = (int)(all_hi64 < 0 ? 0 : (all_hi64 > 0x3fffffff ? 0x3fffffff : all_hi64));
    const int all_lo = (int)(all_lo64 < 0 ? 0 : (all_lo64 > 0x3fffffff ? 0x3fffffff : all_lo64));
    const int left_all = sl.len - key0 > 0x3fffffff ? 0x3fffffff : (int)(sl.len - key0);

    int rel = warp * 16;  // first key of the step, relative to key0
    for (int st = 0; st < steps; ++st, rel += kUnit) {
      cp_wait<C::kStages - 2>();
      __syncwarp();
      issue(st + C::kStages - 1, pages[C::kStages - 1], put);
      next(put);
      const int page = pages[0];
      const float ks = fmaxf(ks_next, kKvScaleFloor), vs = fmaxf(vs_next, kKvScaleFloor);  // (the floor for a NaN)
#pragma unroll
      for (int i = 0; i < C::kStages; ++i) pages[i] = pages[i + 1];
      pages[C::kStages] = entry_of(st + C::kStages + 1);
      ks_next = scale_of(k_scale, pages[0]);
      vs_next = scale_of(v_scale, pages[0]);
      const uint32_t kt = cur, vt = cur + 16 * D;
      next(cur);
      if ((uint32_t)page >= pool) continue;

      // ------------------------------------------------------------ S = Q K^T: two 8-key tiles
      float s[MT][2][4];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int nt = 0; nt < 2; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[mt][nt][e] = 0.f;
#pragma unroll
      for (int hb = 0; hb < D / 64; ++hb) {  // 16 codes a lane and key: four k-steps
        uint32_t kw[2][4];
#pragma unroll
        for (int nt = 0; nt < 2; ++nt) {
          const uint4 r = lds128((kt + nt * 8 * D + k_off) ^ (hb << 4));
          kw[nt][0] = r.x;
          kw[nt][1] = r.y;
          kw[nt][2] = r.z;
          kw[nt][3] = r.w;
        }
#pragma unroll
        for (int sp = 0; sp < 2; ++sp) {
          uint32_t b[2][4];
#pragma unroll
          for (int nt = 0; nt < 2; ++nt) {
            kv_decode4<CODES>(kw[nt][2 * sp], b[nt][0], b[nt][1]);
            kv_decode4<CODES>(kw[nt][2 * sp + 1], b[nt][2], b[nt][3]);
          }
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            const uint32_t qo = q_u + (uint32_t)(((mt * (D / 16) + 4 * hb + 2 * sp) * 32 + lane) * 16);
            const uint4 qa = lds128(qo), qb = lds128(qo + 512);
#pragma unroll
            for (int nt = 0; nt < 2; ++nt) {
              mma16816(s[mt][nt], qa.x, qa.y, qa.z, qa.w, b[nt][0], b[nt][1]);
              mma16816(s[mt][nt], qb.x, qb.y, qb.z, qb.w, b[nt][2], b[nt][3]);
            }
          }
        }
      }

      // ------------------------------------------------------------ weights
      const float lv = kv_lg2(vs);
      const bool edge = rel < all_lo || rel + 16 > all_hi;
      uint32_t pa[MT][4];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        float ck[2], tv[2][4];  // [row half][key]: t + log2 vs - m; before the first maximum (m = -inf) it is +inf
        float to_l[2];          // log2 of the factor of the weights in l
        bool up = false;
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          ck[hf] = cr[mt][hf] * ks;
          const float off = lv - m_run[mt][hf];
#pragma unroll
          for (int k4 = 0; k4 < 4; ++k4) tv[hf][k4] = __fmaf_rn(s[mt][k4 >> 1][hf * 2 + (k4 & 1)], ck[hf], off);
          if (edge) {
#pragma unroll
            for (int k4 = 0; k4 < 4; ++k4) {
              const int key = rel + (k4 >> 1) * 8 + 2 * t4 + (k4 & 1);
              if (key < rlo[mt][hf] || key >= rhi[mt][hf]) tv[hf][k4] = -INFINITY;
            }
          }
          to_l[hf] = (m_run[mt][hf] - u_run[mt][hf]) - lv;
          up |= max3f(max3f(tv[hf][0], tv[hf][1], tv[hf][2]), tv[hf][3], to_l[hf] - (kKvFar - kKvTop)) > kKvTop;
        }
        if (__any_sync(0xffffffffu, up)) {  // rare after the first steps: move the references of the rows that need it
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {
            float t[4], mx = -INFINITY;
#pragma unroll
            for (int k4 = 0; k4 < 4; ++k4) {
              t[k4] = tv[hf][k4] == -INFINITY ? -INFINITY : __fmaf_rn(s[mt][k4 >> 1][hf * 2 + (k4 & 1)], ck[hf], lv);
              mx = fmaxf(mx, t[k4]);
            }
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            auto raise = [&](float u) {
              if (u > u_run[mt][hf]) {
                l_run[mt][hf] *= kv_ex2(u_run[mt][hf] - u);
                u_run[mt][hf] = u;
              }
            };
            if (mx > m_run[mt][hf] + kKvTop) {
              const float m = mx - kKvLift, f = kv_ex2(m_run[mt][hf] - m);  // 0 from -inf
              m_run[mt][hf] = m;
              raise(mx - lv);
              to_l[hf] = (m_run[mt][hf] - u_run[mt][hf]) - lv;
#pragma unroll
              for (int j = 0; j < NT; ++j) {
                o_acc[mt][j][2 * hf] *= f;
                o_acc[mt][j][2 * hf + 1] *= f;
              }
#pragma unroll
              for (int k4 = 0; k4 < 4; ++k4) tv[hf][k4] = t[k4] - m;
            }
            if (to_l[hf] > kKvFar) {  // this page's values are far below the row's largest: its keys' 2^t by themselves
              raise(mx - lv);
#pragma unroll
              for (int k4 = 0; k4 < 4; ++k4)
                if (t[k4] != -INFINITY)
                  l_run[mt][hf] += kv_ex2(__fmaf_rn(s[mt][k4 >> 1][hf * 2 + (k4 & 1)], ck[hf], -u_run[mt][hf]));
              to_l[hf] = -INFINITY;
            }
          }
        }
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          float p[4];
#pragma unroll
          for (int k4 = 0; k4 < 4; ++k4) p[k4] = kv_ex2(tv[hf][k4]);
          l_run[mt][hf] = __fmaf_rn((p[0] + p[1]) + (p[2] + p[3]), kv_ex2(to_l[hf]), l_run[mt][hf]);
          pa[mt][hf] = kv_pack_f16(p[0], p[1]);
          pa[mt][2 + hf] = kv_pack_f16(p[2], p[3]);
        }
      }

      // ------------------------------------------------------------ O += W V
      uint32_t vr[4][D / 32];
#pragma unroll
      for (int k4 = 0; k4 < 4; ++k4) {
        const uint32_t at = vt + (k4 & 1 ? v_off1 : v_off0) + (k4 >> 1) * 8 * D;
        if (D == 128) {
          const uint4 r = lds128(at);
          vr[k4][0] = r.x;
          vr[k4][1] = r.y;
          vr[k4][D / 32 - 2] = r.z;
          vr[k4][D / 32 - 1] = r.w;
        } else {
          const uint2 r = lds64(at);
          vr[k4][0] = r.x;
          vr[k4][1] = r.y;
        }
      }
      if (CODES == kKvE4m3 && left_all - rel < 16) {  // what lies behind the last token may be any bits, NaN among them
#pragma unroll
        for (int k4 = 0; k4 < 4; ++k4)
          if ((k4 >> 1) * 8 + 2 * t4 + (k4 & 1) >= left_all - rel)
#pragma unroll
            for (int i = 0; i < D / 32; ++i) vr[k4][i] = 0;
      }
#pragma unroll
      for (int jq = 0; jq < NT / 4; ++jq) {  // 4 column tiles: one word of each of the lane's four keys
        const uint32_t vw[4] = {vr[0][jq], vr[1][jq], vr[2][jq], vr[3][jq]};
        uint32_t b0[4], b1[4];
        kv_decode4<CODES>(prmt(vw[0], vw[1], 0x5140), b0[0], b0[1]);
        kv_decode4<CODES>(prmt(vw[0], vw[1], 0x7362), b0[2], b0[3]);
        kv_decode4<CODES>(prmt(vw[2], vw[3], 0x5140), b1[0], b1[1]);
        kv_decode4<CODES>(prmt(vw[2], vw[3], 0x7362), b1[2], b1[3]);
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
            mma16816(o_acc[mt][jq * 4 + j], pa[mt][0], pa[mt][1], pa[mt][2], pa[mt][3], b0[j], b1[j]);
      }
    }
    cp_wait<0>();
    __syncwarp();

    // ---------------------------------------------------------------- join the warps
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        float l = l_run[mt][hf];
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        if (t4 == 0) ml[warp][mt * 16 + hf * 8 + g] = KvStat{m_run[mt][hf], u_run[mt][hf], l};
      }
    __syncthreads();
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        const int r = mt * 16 + hf * 8 + g;
        float m = -INFINITY;
#pragma unroll
        for (int i = 0; i < kWarps; ++i) m = fmaxf(m, ml[i][r].m);
        const float f = m_run[mt][hf] == -INFINITY ? 0.f : kv_ex2(m_run[mt][hf] - m);
        // lane t holds d = t (D / 4) .. of the row: columns 2t and 2t + 1 of the tiles
#pragma unroll
        for (int hc = 0; hc < 2; ++hc)
#pragma unroll
          for (int jq = 0; jq < NT / 4; ++jq) {
            const int ch = t4 * (D / 16) + hc * (D / 32) + jq;  // 16-byte chunk of the row
            const uint32_t o = (uint32_t)(r * D * 4 + ((ch ^ ((t4 * 2 + (r & 1)) & 7)) << 4));
            float v[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = o_acc[mt][jq * 4 + j][2 * hf + hc] * f;
            asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(ring_u + o), "f"(v[0]), "f"(v[1]), "f"(v[2]),
                         "f"(v[3])
                         : "memory");
          }
      }
    if (threadIdx.x < TILE) {
      KvStat e{-INFINITY, kKvNoRef, 0.f};
#pragma unroll
      for (int k = 0; k < kWarps; ++k) {
        e.m = fmaxf(e.m, ml[k][threadIdx.x].m);
        e.u = fmaxf(e.u, ml[k][threadIdx.x].u);
      }
#pragma unroll
      for (int k = 0; k < kWarps; ++k) {
        const KvStat x = ml[k][threadIdx.x];
        e.l += x.l * kv_ex2(x.u - e.u);  // (a warp without keys: 0; one whose every score is NaN: NaN)
      }
      ml_all[threadIdx.x] = e;
    }
    __syncthreads();
    const int part_slot = (int)(w * 2 + (first_segment ? 0 : 1));
    float* part = a.part + (int64_t)part_slot * TILE * (D + 4);
    for (int i = threadIdx.x; i < sl.rows * (D / 4); i += kThreads) {
      const int r = i / (D / 4), ch = i % (D / 4), tt = ch / (D / 16);
      const uint32_t o = (uint32_t)(r * D * 4 + ((ch ^ ((tt * 2 + (r & 1)) & 7)) << 4));
      const KvStat e = ml_all[r];
      float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int k = 0; k < kWarps; ++k) {
        const float4 v = *reinterpret_cast<const float4*>(smem + k * C::kRing + o);
        sum.x += v.x;
        sum.y += v.y;
        sum.z += v.z;
        sum.w += v.w;
      }
      if (whole) {
        kv_put_row(a, kv_row_out(a, sl, kvh, r), ch, D, sum, e);
      } else {
        *reinterpret_cast<float4*>(part + (int64_t)r * D + ch * 4) = sum;
        if (ch == 0) *reinterpret_cast<float4*>(part + (int64_t)TILE * D + 4 * r) = make_float4(e.m, e.u, e.l, 0.f);
      }
    }
    if (u0 == 0 && !whole && threadIdx.x == 0) {
      // who holds the rest: the worker of unit y is the last one whose range begins at or before y
      const int64_t y = item0 + (int64_t)kvh * units + units - 1;
      const int64_t w1 = ((y + 1) * workers - 1) / all;
      a.meta[w] = make_int4((int)(base + li), kvh, part_slot, (int)(w1 - w) + 1);
      cut = true;
    }
    first_segment = false;
    x += u1 - u0;
    if (x >= x_end) {
      if (threadIdx.x == 0 && !cut) a.meta[w] = make_int4(0, 0, 0, 0);
      break;
    }
    __syncthreads();  // the rings, q and the statistics are read: the next segment may fill them
    if (x >= item0 + (int64_t)units * a.c.kv_heads) {  // the next slot that has units
      ++li;
      while (true) {
        while (li < kThreads && sc.units[li] == 0) ++li;
        if (li < kThreads) break;
        before += here;
        base += kThreads;
        here = sched_load<TILE, kWarps>(a, sc, base);
        li = 0;
      }
    }
  }
}

}  // namespace

// Block (w, y) of the first a.workers: rows of the item that worker w began and others went on with (at most one).  A
// thread takes four columns of a row and adds the parts in their order, each with its factor 2^(m_i - m).  The blocks
// after them look through the slots for those without any key, whose rows are zeros, and for sequences that no kernel of
// the call takes, whose rows are NaN.  The blocks after those, up to kRestBlocks of the launch for few rows of a call with starts
// (which always has that launch), deal out the rows of no sequence, which are zeros too.  (Dealt to all blocks they cost a call
// without any such row 0.9 us: two more loads ahead of every block's own.)
// Latency: 4 to 6 us for most calls of few rows, 10 us for a sequence of 131000 in 55 parts a kv head (14.5 us with four
// loads in flight); 15 us for the 148 items of 256 rows of head dim 128 that a large chunk call cuts (23 us with a block for eight
// rows instead of 32).
constexpr int kRestBlocks = 64;
template <int D, int TILE>
__global__ void __launch_bounds__(256, 4) kv_attn_join_kernel(const KvAttnArgs a) {
  // 16-byte chunks of a row; rows of a block, those of a thread BY apart; loads of a thread in flight: a large tile has many
  // rows of few parts, a small one few rows of, at times, hundreds
  constexpr int CH = D / 4, BY = 256 / CH, R = TILE == 256 ? 4 : 1, ROWS = BY * R, AT_ONCE = 8 / R;
  constexpr int LANES = TILE == 256 ? 8 : 32;  // that look at the statistics of a row's parts
  __shared__ KvStat ml[ROWS];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if ((int)blockIdx.x >= a.workers) {
    const int first = a.workers + (int)((a.slots + 255) / 256);
    if (TILE != 256 && (int)blockIdx.x >= first) {
      const KvRest rest = kv_rest(a.s);
      for (int i = (blockIdx.x - first) * gridDim.y + blockIdx.y; i < rest.n; i += (gridDim.x - first) * gridDim.y) {
        const int64_t row = (int64_t)rest.row(i) * a.heads;
        for (int k = threadIdx.x; k < a.heads * CH; k += 256)
          kv_put_row(a, row + k / CH, k % CH, D, make_float4(0.f, 0.f, 0.f, 0.f), KvStat{0.f, 0.f, 0.f});
      }
      return;
    }
    if (blockIdx.y > 0) return;
    const int64_t slot0 = ((int64_t)(blockIdx.x - a.workers) * 8 + warp) * 32;
    KvSlot t;
    bool none = false, over = false;
    if (slot0 + lane < a.slots) {
      const int b = a.one ? (int)(slot0 + lane) : kv_slot_seq(a.s, slot0 + lane, a.per, TILE, 1);
      none = kv_slot(a, slot0 + lane, b, TILE, t) && t.hi <= t.lo;
      if (a.last) {  // a sequence of more new tokens than the caller allowed for
        t.s0 = kv_start(a.s, b);
        const int64_t all = (int64_t)(kv_start(a.s, b + 1) - t.s0) * a.per;
        over = all > a.row_hi;
        if (over) {
          t.r0 = 0;
          t.rows = (int)all;
        }
      }
    }
    unsigned todo = __ballot_sync(0xffffffffu, none || over);
    const unsigned bad = __ballot_sync(0xffffffffu, over);
    while (todo) {
      const int src = __ffs(todo) - 1;
      todo &= todo - 1;
      KvSlot e;
      e.s0 = __shfl_sync(0xffffffffu, t.s0, src);
      e.r0 = __shfl_sync(0xffffffffu, t.r0, src);
      const int rows = __shfl_sync(0xffffffffu, t.rows, src);
      const float l = bad >> src & 1 ? __int_as_float(0x7fffffff) : 0.f;
      for (int64_t i = lane; i < (int64_t)rows * a.c.kv_heads * CH; i += 32) {
        const int64_t row = i / CH;
        kv_put_row(a, kv_row_out(a, e, (int)(row / rows), (int)(row % rows)), (int)(i % CH), D, make_float4(0.f, 0.f, 0.f, 0.f),
                   KvStat{0.f, 0.f, l});
      }
    }
    return;
  }
  const int4 meta = a.meta[blockIdx.x];
  // no cut item; or the worker gave up (a time-out, latched in the error word) before it wrote its entry
  if (meta.w <= 1 || meta.w > a.workers - (int)blockIdx.x || meta.x < 0 || meta.x >= a.slots || meta.y < 0 ||
      meta.y >= a.c.kv_heads || (meta.z >> 1) != (int)blockIdx.x)
    return;
  const int64_t slot = meta.x;
  const int kvh = meta.y, n = meta.w;
  const int b = a.one ? (int)slot : kv_slot_seq_warp(a.s, slot, a.per, TILE, 1);
  KvSlot sl;
  if (!kv_slot(a, slot, b, TILE, sl)) return;
  // the first part is in the slot that its worker says, the others are their worker's first segment
  auto part_of = [&](int i) { return a.part + (int64_t)(i == 0 ? meta.z : 2 * ((int)blockIdx.x + i)) * TILE * (D + 4); };
  auto ml_of = [&](int i, int row) { return reinterpret_cast<const float4*>(part_of(i) + (int64_t)TILE * D) + row; };
  // neighbours in a warp are rows where the parts are [chunk][row] (tiles of 256), chunks where they are [row][chunk]
  const int tr = TILE == 256 ? threadIdx.x % BY : threadIdx.x / CH, ch = TILE == 256 ? threadIdx.x / BY : threadIdx.x % CH;
  for (int row0 = blockIdx.y * ROWS; row0 < sl.rows; row0 += gridDim.y * ROWS) {
    for (int r = threadIdx.x / LANES; r < ROWS; r += 256 / LANES) {
      KvStat x{-INFINITY, kKvNoRef, 0.f};
      if (row0 + r < sl.rows)
        for (int i = lane % LANES; i < n; i += LANES) {
          const float4 e = __ldg(ml_of(i, row0 + r));
          const float to = fmaxf(x.u, e.y);
          x.l = __fmaf_rn(kv_ex2(e.y - to), e.z, x.l * kv_ex2(x.u - to));
          x.u = to;
          x.m = fmaxf(x.m, e.x);
        }
#pragma unroll
      for (int o = LANES / 2; o; o >>= 1) {
        const float u2 = __shfl_xor_sync(0xffffffffu, x.u, o), l2 = __shfl_xor_sync(0xffffffffu, x.l, o), to = fmaxf(x.u, u2);
        x.l = __fadd_rn(__fmul_rn(x.l, kv_ex2(x.u - to)), __fmul_rn(l2, kv_ex2(u2 - to)));  // the same in both lanes
        x.u = to;
        x.m = fmaxf(x.m, __shfl_xor_sync(0xffffffffu, x.m, o));
      }
      if (lane % LANES == 0) ml[r] = x;
    }
    __syncthreads();
    float4 o[R];
#pragma unroll
    for (int k = 0; k < R; ++k) o[k] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i0 = 0; i0 < n; i0 += AT_ONCE) {
      float4 v[AT_ONCE][R];
      float f[AT_ONCE][R];
#pragma unroll
      for (int u = 0; u < AT_ONCE; ++u)
#pragma unroll
        for (int k = 0; k < R; ++k) {
          const int row = row0 + tr + k * BY;
          f[u][k] = -INFINITY;
          if (i0 + u < n && row < sl.rows) {
            const int64_t at = TILE == 256 ? ((int64_t)ch * TILE + row) * 4 : (int64_t)row * D + ch * 4;
            v[u][k] = *reinterpret_cast<const float4*>(part_of(i0 + u) + at);
            f[u][k] = __ldg(&ml_of(i0 + u, row)->x);
          }
        }
#pragma unroll
      for (int u = 0; u < AT_ONCE; ++u)
#pragma unroll
        for (int k = 0; k < R; ++k) {
          const float w = f[u][k] == -INFINITY ? 0.f : kv_ex2(f[u][k] - ml[tr + k * BY].m);
          if (w != 0.f) {  // a part that saw no key of the row may hold anything
            o[k].x = __fmaf_rn(v[u][k].x, w, o[k].x);
            o[k].y = __fmaf_rn(v[u][k].y, w, o[k].y);
            o[k].z = __fmaf_rn(v[u][k].z, w, o[k].z);
            o[k].w = __fmaf_rn(v[u][k].w, w, o[k].w);
          }
        }
    }
#pragma unroll
    for (int k = 0; k < R; ++k) {
      const int row = row0 + tr + k * BY;
      if (row < sl.rows) kv_put_row(a, kv_row_out(a, sl, kvh, row), ch, D, o[k], ml[tr + k * BY]);
    }
    __syncthreads();  // the statistics are read
  }
}

cudaError_t launch_kv_attn_join(const KvAttnArgs& a, int tile, cudaStream_t st) {
  if (a.workers > (tile == 256 ? kMaxWorkers : kMaxRowWorkers)) return cudaErrorInvalidValue;
  const int blocks = tile / (1024 / a.c.dim);  // of 256 threads with a 16-byte chunk each, for a tile's rows
  const int rest = tile == 256 || !a.s.starts ? 0 : a.s.tokens < kRestBlocks ? a.s.tokens : kRestBlocks;
  const dim3 grid((unsigned)(a.workers + (a.slots + 255) / 256 + rest),
                  (unsigned)(tile == 256 ? blocks / 4 : blocks > 1 ? blocks : 1));
#define H3Q_KV_J(DD, TT)                                     \
  if (a.c.dim == DD && tile == TT) {                         \
    kv_attn_join_kernel<DD, TT><<<grid, 256, 0, st>>>(a);    \
    return cudaGetLastError();                               \
  }
  H3Q_KV_J(64, 16) H3Q_KV_J(64, 32) H3Q_KV_J(64, 256) H3Q_KV_J(128, 16) H3Q_KV_J(128, 32) H3Q_KV_J(128, 256)
#undef H3Q_KV_J
  return cudaErrorInvalidValue;
}

namespace {

template <int D, int CODES, int MT>
cudaError_t launch_rows(KvAttnArgs a, cudaStream_t st) {
  using C = RowsCfg<D, MT>;
  auto kern = kv_attn_rows_kernel<D, CODES, MT>;
  static bool ready[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  if (!ready[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
    if (e != cudaSuccess) return e;
    ready[dev] = true;
  }
  a.workers = sm_count(dev) * C::kCtas < kMaxRowWorkers ? sm_count(dev) * C::kCtas : kMaxRowWorkers;
  kern<<<(unsigned)a.workers, C::kThreads, C::kSmem, st>>>(a);
  if (const cudaError_t e = cudaGetLastError()) return e;
  return launch_kv_attn_join(a, MT * 16, st);
}

}  // namespace

size_t kv_attn_rows_part_bytes(int dim, int tile) { return (size_t)kMaxRowWorkers * 2 * tile * (dim + 4) * 4; }

// tile: 16 or 32 rows
cudaError_t launch_kv_attn_rows(const KvAttnArgs& a, int tile, cudaStream_t st) {
#define H3Q_KV_A(DD, CC, MM) \
  if (a.c.dim == DD && a.c.codes == CC && tile == MM * 16) return launch_rows<DD, CC, MM>(a, st);
  H3Q_KV_A(64, 0, 1) H3Q_KV_A(64, 1, 1) H3Q_KV_A(128, 0, 1) H3Q_KV_A(128, 1, 1)
  H3Q_KV_A(64, 0, 2) H3Q_KV_A(64, 1, 2) H3Q_KV_A(128, 0, 2) H3Q_KV_A(128, 1, 2)
#undef H3Q_KV_A
  return cudaErrorInvalidValue;
}

}  // namespace h3q
