// kv_attn_chunk.cu -- attention over the 8-bit paged cache for many query rows to a kv head (prompts, chunks of one,
// blocks of a stream): bound by the 16-bit tensor cores and the exponentials.
//
// A slot is 256 rows of a (sequence, kv head) -- (token, query head of the group) in that order, so a kv head's keys
// serve all its query heads -- as two 128-row tiles.  512 threads:
//   warp 0       one lane issues the MMAs (tcgen05 kind::f16): per tile pair O_t += W_t V_j and then S_t = Q_t K_(j+1)^T,
//                t = 0, 1, so that one softmax works while the other's products run; it also holds the TMEM allocation;
//   warps 4-11   softmax of tile 0 and 1: thread = row = TMEM lane; scales, maximum, W = 2^(t - m) as f16 back into TMEM
//                over the scores it came from (the A operand of the second product is read from there: with W in
//                shared memory the products alone would take the SM's whole shared-memory bandwidth), row sums; the
//                reference moves only when a weight would pass 2^15;
//   warp 1       walks the work ahead of them: which rows and keys come next and, from the page table, the scales of each
//                16 keys go into rings in shared memory, and the codes of two tiles ahead are copied there (cp.async.bulk),
//                so that the others never wait for a length, a table entry or memory;
//   warps 12-15  widen the codes to f16 into a ring of three 128-key tiles, K and V in turn: K rows go out as they are,
//                V is transposed on the way (byte permutes between eight keys of a thread), both in the K-major
//                128-byte-swizzle layout.  V's codes lie in groups of eight keys 16 bytes further apart than they are long,
//                so that a warp reads eight groups at once without a bank conflict.
// A page's scales never touch the codes (kv_attn.cuh).  Work is cut in 128-key tiles: a first kernel lists the slots
// that have keys with their running sum, and the CTAs take equal contiguous ranges of the tiles of all (slot, kv head)
// in order, so no wave is left part full; an item cut between CTAs is joined from f32 parts in order.
//
// Measured (B200): 2048 new tokens of 2 sequences over 10240, 32 heads (8 kv heads) of 128, causal, e4m3: 645 us for 0.62
// TFLOP, 0.96 PFLOP/s; 1000 over 32760, 40 heads, int8: 757 us for 0.67 TFLOP; up to 1500 of 6 sequences, 16 heads of 64, a
// window of 1024: 86 us (617, 716 and 81 us before l had a reference of its own: the kernel is sensitive to a few more
// instructions and registers in its loop).  A stretch costs 2.3 (head dim 64) to 2.9 us a tile and 12 to 14 us for its start and end: q in (by
// cp.async; loads through the few KB that are left of L1 took three times as long, and 20 us more of the first case), the first
// scores, O out.  What bounds it is a row tile's chain (scores out of TMEM, maximum, 128 exponentials a thread, weights
// into TMEM, two products), about 4000 cycles of which the products are 1024 and the exponentials 1024 at their rates, with two
// row tiles to overlap.  In a small case (1024 new tokens of one sequence over 6144, 127 us) the tensor cores work 36 % of the
// time, the exponential units 37 %, the issue slots 34 %; by its flops the first case keeps the tensor cores busy for 42 % of
// it at 1.9 GHz.  A third row tile has no room in TMEM at head dim 128 (2 x (128 + 128) columns are all of it); two threads a
// row, and at head dim 64 the room that is left for a next stretch's q and outputs, are not tried.  156 bytes (168 there) of a
// thread's registers are spilled.
// Tried before that, no faster: weights in shared memory, passes of 16 or 32 columns, the maximum in the weights' pass with a redo, the second
// product on halves of the weights, a late start of the second softmax, other register splits, codes widened from registers.
// Every wait is bounded: on time-out the CTA latches an error code, waits for its MMAs, frees TMEM and returns.
#include <cstdint>
#include <cuda_runtime.h>
#include "kv_attn.cuh"
#include "h3q_internal.h"

namespace h3q {

namespace {

constexpr int BM = 128, BN = 128, NQ = 2, ROWS = NQ * BM;
constexpr int THREADS = 512;
constexpr int RING = 3, RAW = 2, WR = 8;
// setmaxnreg split of the 128 registers a thread at launch (512 x 128 = the whole file): MMA and walker 48, softmax
// 2 x 192, decode 80: 48 + 2 * 192 + 80 = 512 = 4 * 128.
constexpr int REGS_MMA = 48, REGS_SOFT = 192, REGS_DEC = 80;
static_assert(REGS_MMA + 2 * REGS_SOFT + REGS_DEC <= 4 * 128, "setmaxnreg split exceeds the launch");
constexpr uint32_t TMEM_COLS = 512;

template <int D>
struct Cfg {
  static constexpr int Q_SLAB = BM * 128;            // 64 columns of a 128-row tile
  static constexpr int Q_TILE = (D / 64) * Q_SLAB;
  static constexpr int KV_TILE = BN * D * 2;         // K: D / 64 slabs of 128 keys; V^T: 2 slabs of 64 keys x D
  static constexpr int V_SLAB = D * 128;
  static constexpr int OFF_KV = NQ * Q_TILE;
  static constexpr int RAW_K = BN * D;               // codes of a tile
  static constexpr int V_OCTET = 8 * D + 16;
  static constexpr int RAW_V = 16 * V_OCTET;
  static constexpr int OFF_RK = OFF_KV + RING * KV_TILE;
  static constexpr int OFF_RV = OFF_RK + RAW * RAW_K;
  static constexpr int OFF_SC = OFF_RV + RAW * RAW_V;
  static constexpr int OFF_SEG = OFF_SC + WR * 8 * 16;
  static constexpr int OFF_BAR = OFF_SEG + 2 * 48;
  static constexpr int NBAR = 2 * RING + 4 * RAW + 2 * WR + 4 * NQ + 1 + 4;
  static constexpr size_t SMEM = 1024 + OFF_BAR + NBAR * 8 + 16;
  static_assert(SMEM + 16 <= 232448, "shared memory exceeds the sm_100 per-CTA limit");
};

// 16 bytes from global memory, or zeros
__device__ __forceinline__ void cp16_zfill(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}

// the K-major 128-byte-swizzle descriptor of shared memory at 16 * `lo` bytes
__device__ __forceinline__ uint64_t desc_of(uint32_t lo) {
  constexpr uint32_t hi = (1024 >> 4) | (1u << 14) | (2u << 29);  // 8-row stride, version, swizzle
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(lo | (1u << 16)), "n"(hi));
  return d;
}

// the n lowest bits (none for n <= 0, all from 32 on)
__device__ __forceinline__ uint32_t below(int n) { return n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1; }
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 r;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(a) : "memory");
  return r;
}
__device__ __forceinline__ void sts128(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

}  // namespace

// x, as a value that the compiler cannot compute ahead of a loop and keep: what is derived from it costs an add where it
// is used, not a register (or a spill) for the whole kernel
__device__ __forceinline__ uint32_t fresh(uint32_t x) {
  asm volatile("" : "+r"(x));
  return x;
}

template <int V>
struct Int {
  static constexpr int value = V;
};

// A slot that has keys, and the 128-key tiles of all kv heads before it.
struct KvListed {
  int64_t before;
  int slot, b, tiles, pad;
};
struct KvChunkWork {
  KvListed* list;
  int64_t* head;  // [0] listed slots, [1] tiles of all
};

// One CTA: lists the slots with keys in order, 1024 at a time with a running sum.  Latency: 4 to 5 us.
__global__ void __launch_bounds__(1024) kv_attn_list_kernel(const KvAttnArgs a, const KvChunkWork wk) {
  __shared__ int sum_n[32], sum_t[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t tiles_before = 0;
  int64_t count = 0;
  for (int64_t base = 0; base < a.slots; base += 1024) {
    const int64_t slot = base + threadIdx.x;
    int b = 0, tiles = 0;
    if (slot < a.slots) {
      b = a.one ? (int)slot : kv_slot_seq(a.s, slot, a.per, ROWS, 1);
      KvSlot t;
      if (kv_slot(a, slot, b, ROWS, t)) tiles = (int)((t.hi - t.lo + BN - 1) / BN);
    }
    int n = tiles > 0, x = tiles;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int n2 = __shfl_up_sync(0xffffffffu, n, o), x2 = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) {
        n += n2;
        x += x2;
      }
    }
    if (lane == 31) {
      sum_n[warp] = n;
      sum_t[warp] = x;
    }
    __syncthreads();
    int bn = 0, an = 0;
    int64_t bt = 0, at = 0;
    for (int w = 0; w < 32; ++w) {
      if (w < warp) {
        bn += sum_n[w];
        bt += sum_t[w];
      }
      an += sum_n[w];
      at += sum_t[w];
    }
    if (tiles > 0) {
      KvListed e;
      e.before = (tiles_before + bt + x - tiles) * a.c.kv_heads;
      e.slot = (int)slot;
      e.b = b;
      e.tiles = tiles;
      e.pad = 0;
      wk.list[count + bn + n - 1] = e;
    }
    count += an;
    tiles_before += at;
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    wk.head[0] = count;
    wk.head[1] = tiles_before * a.c.kv_heads;
  }
}

namespace {

// A stretch of tiles of one item, as the walker hands it to the other roles.
struct Stretch {
  int rows, n;          // rows of the slot, tiles (0: the end)
  int s0, r0;           // of the slot's sequence: first packed row, first row of the slot
  int kvh, whole;
  int64_t first, len, key_base;  // place of its first new token, tokens that the table has room for, first key
};
static_assert(sizeof(Stretch) == 48, "two of them in shared memory");

// The walker's place in its CTA's range of tiles.
struct Walk {
  int64_t x, end;
  int i;  // index into the list
};
struct Segment {
  KvSlot sl;
  KvListed e;
  int kvh, t0, t1;  // tiles [t0, t1) of the item
};
__device__ __forceinline__ bool next_segment(const KvAttnArgs& a, const KvChunkWork& wk, Walk& w, Segment& s) {
  if (w.x >= w.end) return false;
  s.e = wk.list[w.i];
  if (w.x >= s.e.before + (int64_t)s.e.tiles * a.c.kv_heads) s.e = wk.list[++w.i];
  const int64_t rel = w.x - s.e.before;
  s.kvh = (int)(rel / s.e.tiles);
  s.t0 = (int)(rel - (int64_t)s.kvh * s.e.tiles);
  s.t1 = (int)(w.end - w.x < s.e.tiles - s.t0 ? s.t0 + (w.end - w.x) : s.e.tiles);
  kv_slot(a, s.e.slot, s.e.b, ROWS, s.sl);
  w.x += s.t1 - s.t0;
  return true;
}

}  // namespace

// A tile with a page whose values are far below others of the stretch: its keys may count in l and have no w, so the row's
// 2^t of the whole tile are summed here, by themselves.  Scores at tS, keys a0 .. a1 - 1 of the tile seen; u and l in and out.
// A call, so that the loop over tiles, whose instructions barely fit the cache, is not longer for what is rare (2048-token
// chunk: 651 us, 672 in line).
__device__ __noinline__ float2 far_sums(uint32_t tS, const float4* cs, int a0, int a1, float c, float u, float l) {
#pragma unroll 1
  for (int q = 0; q < 8; ++q) {
    const float4 e = cs[q];
    if (e.y == -INFINITY) continue;
    uint32_t y[16];
    tmem_ld_32x32b_x16(tS + 16 * q, y);
    tmem_wait_ld();
    const uint32_t bits = below(a1 - 16 * q) & ~below(a0 - 16 * q);
    const float ce = fmaxf(c * e.x, 1e-37f);
    float to = u;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      y[i] = bits >> i & 1 ? y[i] : 0xff800000u;
      to = fmaxf(to, __uint_as_float(y[i]) * ce);
    }
    l *= kv_ex2(u - to);
    u = to;
#pragma unroll
    for (int i = 0; i < 16; ++i) l += kv_ex2(__fmaf_rn(__uint_as_float(y[i]), ce, -u));
  }
  return make_float2(u, l);
}

template <int D, int CODES>
__global__ void __launch_bounds__(THREADS, 1)
    kv_attn_chunk_kernel(const KvAttnArgs a, const KvChunkWork wk, int q_vec, int* err) {
  using C = Cfg<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  // [WR][8]: k scale, log2 of the v scale (-inf where there is no page), the tile's largest v scale over it (0), and in .w
  // the logarithm of that largest one (entries 1 ..; inf without a page, which makes the weights' factor in l 0) and how far
  // the least is below the largest of the stretch until then (entry 0)
  float4* consts = reinterpret_cast<float4*>(smem + C::OFF_SC);
  uint64_t* kv_full = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
  uint64_t* kv_empty = kv_full + RING;
  uint64_t* rk_full = kv_empty + RING;
  uint64_t* rk_free = rk_full + RAW;
  uint64_t* rv_full = rk_free + RAW;
  uint64_t* rv_free = rv_full + RAW;
  uint64_t* wr_full = rv_free + RAW;
  uint64_t* wr_free = wr_full + WR;
  uint64_t* q_full = wr_free + WR;
  uint64_t* s_full = q_full + NQ;
  uint64_t* p_full = s_full + NQ;
  uint64_t* o_full = p_full + NQ;
  uint64_t* sg_full = o_full + NQ;
  uint64_t* sg_free = sg_full + 2;
  uint64_t* mma_done = sg_free + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(mma_done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const Stretch* stretches = reinterpret_cast<const Stretch*>(smem + C::OFF_SEG);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t all = wk.head[1], workers = all < gridDim.x ? all : gridDim.x;
  if (blockIdx.x >= workers) {
    if (threadIdx.x == 0) a.meta[blockIdx.x] = make_int4(0, 0, 0, 0);
    return;
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < RING; ++i) { mbar_init(&kv_full[i], 4); mbar_init(&kv_empty[i], 1); }
    for (int i = 0; i < RAW; ++i) {
      mbar_init(&rk_full[i], 1);
      mbar_init(&rk_free[i], 4);
      mbar_init(&rv_full[i], 1);
      mbar_init(&rv_free[i], 4);
    }
    for (int i = 0; i < WR; ++i) { mbar_init(&wr_full[i], 1); mbar_init(&wr_free[i], 4); }
    for (int t = 0; t < NQ; ++t) {
      mbar_init(&q_full[t], 4);
      mbar_init(&s_full[t], 1);
      mbar_init(&p_full[t], 4);
      mbar_init(&o_full[t], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sg_full[i], 1);
      mbar_init(&sg_free[i], 1 + 4 + 8);  // the MMA thread, the decode and the softmax warps
    }
    mbar_init(mma_done, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 0) {
    tmem_alloc(tmem_slot, TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  // the i-th stretch by one thread, and by a warp: waits for it, copies it and tells the walker so
  auto copy = [&](uint32_t i, Stretch& s) {
    if (!mbar_wait_prompt(&sg_full[i & 1], (i >> 1) & 1, abort_flag, err, kDevTimeoutScale)) return false;
    s = stretches[i & 1];
    return s.n > 0;
  };
  auto take = [&](uint32_t i, Stretch& s) {
    if (!copy(i, s)) return false;
    mbar_arrive(&sg_free[i & 1]);
    return true;
  };
  auto take_warp = [&](uint32_t i, Stretch& s) {
    if (!__all_sync(0xffffffffu, copy(i, s))) return false;  // every lane has its copy
    if (lane == 0) mbar_arrive(&sg_free[i & 1]);
    return true;
  };

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_MMA));
    if (warp == 0 && elect_one()) {
      // ------------------------------------------------------------------ MMA issuer
      constexpr uint32_t idq = idesc_f16(BM, BN, false);
      constexpr uint32_t idp = idesc_f16(BM, D, false);
      // shared-memory addresses in units of 16 bytes: a step in K of 16 columns is 2, of 64 a slab
      const uint32_t q0 = smem_u32(smem) >> 4, kv0 = smem_u32(smem + C::OFF_KV) >> 4;
      uint32_t slot = 0, phase = 0;  // place in the ring
      uint32_t segs0 = 0, segs1 = 0, done0 = 0, done1 = 0;  // segments and tiles of each row tile
      bool ok = true;
      auto advance = [&]() {
        if (++slot == RING) {
          slot = 0;
          phase ^= 1;
        }
      };
      auto wait_kv = [&]() {
        if (!mbar_wait_prompt(&kv_full[slot], phase, abort_flag, err, kDevTimeoutFull)) return false;
        tc_fence_after();
        return true;
      };
      // S_t = Q_t K^T
      auto issue_qk = [&](auto tc) {
        constexpr int t = decltype(tc)::value;
        const uint32_t qb = fresh(q0 + t * (C::Q_TILE >> 4)), kb = fresh(kv0 + slot * (C::KV_TILE >> 4));
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint32_t o = (k >> 2) * (C::Q_SLAB >> 4) + 2 * (k & 3);
          mma_f16(tmem_base + t * BN, desc_of(qb + o), desc_of(kb + o), idq, k != 0);
        }
        mma_commit(&s_full[t]);  // completes with every MMA before it, so O_t is also up to date then
      };
      // O_t += W_t V, W_t over the first 64 columns of S_t
      auto issue_pv = [&](auto tc, uint32_t vslot, uint32_t tiles, bool add) {
        constexpr int t = decltype(tc)::value;
        if (!mbar_wait_prompt(&p_full[t], tiles & 1, abort_flag, err, kDevTimeoutProbs)) return false;
        tc_fence_after();
        const uint32_t vb = fresh(kv0 + vslot * (C::KV_TILE >> 4));
#pragma unroll
        for (int k = 0; k < BN / 16; ++k)
          mma_f16_ts(tmem_base + NQ * BN + t * D, tmem_base + t * BN + 8 * k,
                     desc_of(vb + (k >> 2) * (C::V_SLAB >> 4) + 2 * (k & 3)), idp, add || k != 0);
        return true;
      };
      constexpr Int<0> t0{};
      constexpr Int<1> t1{};
      Stretch s;
      for (uint32_t si = 0; ok && take(si, s); ++si) {
        const bool two = s.rows > BM;
        const int n = s.n;
        if (!(ok = wait_kv() && mbar_wait_prompt(&q_full[0], segs0++ & 1, abort_flag, err, kDevTimeoutFull))) break;
        tc_fence_after();
        issue_qk(t0);
        if (two) {
          if (!(ok = mbar_wait_prompt(&q_full[1], segs1++ & 1, abort_flag, err, kDevTimeoutFull))) break;
          tc_fence_after();
          issue_qk(t1);
        }
        mma_commit(&kv_empty[slot]);
        advance();
        for (int j = 0; j < n; ++j) {
          const bool more = j + 1 < n;
          const uint32_t vslot = slot;
          if (!(ok = wait_kv())) break;
          advance();
          if (!(ok = issue_pv(t0, vslot, done0, j > 0) && (!more || wait_kv()))) break;
          if (more) issue_qk(t0);
          else mma_commit(&o_full[0]);
          ++done0;
          if (two) {
            if (!(ok = issue_pv(t1, vslot, done1, j > 0))) break;
            if (more) issue_qk(t1);
            else mma_commit(&o_full[1]);
            ++done1;
          }
          mma_commit(&kv_empty[vslot]);
          if (more) {
            mma_commit(&kv_empty[slot]);
            advance();
          }
        }
      }
      mma_commit(mma_done);  // every MMA issued here completes before TMEM is released
      mbar_drain(mma_done, 0, err, kDevTimeoutDrain);
    }
    if (warp == 1) {
      // ------------------------------------------------------------------ walker: for tiles, eight lanes of 16 keys each
      Walk walk{all * blockIdx.x / workers, all * (blockIdx.x + 1) / workers, 0};
      for (int hi = (int)wk.head[0]; hi - walk.i > 1;) {  // the last listed slot whose tiles begin at or before x
        const int mid = (walk.i + hi) >> 1;
        if (wk.list[mid].before <= walk.x) walk.i = mid;
        else hi = mid;
      }
      uint32_t tile = 0, si = 0, asked_k = 0, asked_v = 0;
      bool ok = true;
      Segment s{};
      auto hand = [&](int n) {  // stretch si to the others
        if (si >= 2 && !__all_sync(0xffffffffu, mbar_wait_prompt(&sg_free[si & 1], ((si >> 1) - 1) & 1, abort_flag, err,
                                                                 kDevTimeoutEmpty)))
          return false;
        if (lane == 0) {
          Stretch& d = reinterpret_cast<Stretch*>(smem + C::OFF_SEG)[si & 1];
          d.rows = s.sl.rows;
          d.n = n;
          d.s0 = s.sl.s0;
          d.r0 = s.sl.r0;
          d.first = s.sl.first;
          d.kvh = s.kvh;
          d.whole = s.t0 == 0 && s.t1 == s.e.tiles;
          d.len = s.sl.len;
          d.key_base = s.sl.lo + (int64_t)s.t0 * BN;
          mbar_arrive(&sg_full[si & 1]);
        }
        ++si;
        return true;
      };
      bool cut = false;
      while (ok && next_segment(a, wk, walk, s)) {
        if (lane == 0 && s.t0 == 0 && s.t1 < s.e.tiles) {  // begun here, and others go on with it
          const int64_t y = s.e.before + (int64_t)(s.kvh + 1) * s.e.tiles - 1;
          const int64_t w1 = ((y + 1) * workers - 1) / all;
          a.meta[blockIdx.x] =
              make_int4(s.e.slot, s.kvh, (int)blockIdx.x * 2 + (si > 0), (int)(w1 - blockIdx.x) + 1);
          cut = true;
        }
        if (!(ok = hand(s.t1 - s.t0))) break;
        int64_t key = s.sl.lo + (int64_t)s.t0 * BN + (lane & 7) * 16;  // lane l + 8 does as lane l does
        auto page_at = [&](int64_t k) { return k < s.sl.hi ? kv_page(a.c, a.s, s.sl.b, k >> a.c.page_log2) : (int64_t)-1; };
        int64_t page_next = page_at(key);
        float loudest = -INFINITY;
        for (int j = s.t0; j < s.t1; ++j, ++tile, key += BN) {
          const int64_t page = page_next, ph = page * a.c.kv_heads + s.kvh;
          float4 c = make_float4(0.f, -INFINITY, 0.f, 0.f);
          if (page >= 0) {
            c.x = fmaxf(__ldg(a.c.k_scale + ph), kKvScaleFloor);  // (the floor for a NaN)
            c.y = kv_lg2(fmaxf(__ldg(a.c.v_scale + ph), kKvScaleFloor));
          }
          float least = page >= 0 ? c.y : INFINITY, most = c.y;
#pragma unroll
          for (int o = 1; o < 8; o <<= 1) {
            least = fminf(least, __shfl_xor_sync(0xffffffffu, least, o));
            most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
          }
          loudest = fmaxf(loudest, most);
          if (page >= 0) c.z = kv_ex2(fminf(most - c.y, kKvFar));
          c.w = lane == 0 ? loudest - least : most > -INFINITY ? most : INFINITY;
          if (j + 1 < s.t1) page_next = page_at(key + BN);
          const int64_t off = (ph * a.c.page + (key & (a.c.page - 1))) * D;  // of the lane's 16 keys' codes
          // entry tile - 8 is read once the decode warps may fill K of tile - 4: its ring slot held V of tile - 6, whose
          // product is done (a barrier a ring entry: the decode warps may be several tiles past f)
          const uint32_t f = tile - 4;
          const int r = tile % RAW;
          const uint32_t freed = ((tile / RAW) & 1) ^ 1;
          if ((tile >= 4 && !__all_sync(0xffffffffu, mbar_wait_prompt(&wr_free[f % WR], (f / WR) & 1, abort_flag, err,
                                                                      kDevTimeoutEmpty))) ||
              !__all_sync(0xffffffffu, mbar_wait_prompt(&rk_free[r], freed, abort_flag, err, kDevTimeoutEmpty))) {
            ok = false;
            break;
          }
          if (lane < 8) consts[(tile % WR) * 8 + lane] = c;
          // codes of 16 keys that are not there are zeros (their weights are, and 0 times what lay there may not be)
          uint8_t* const rk = smem + C::OFF_RK + r * C::RAW_K;
          uint8_t* const rv = smem + C::OFF_RV + r * C::RAW_V;
          const uint32_t there = __ballot_sync(0xffffffffu, page >= 0) & 0xffu;
          auto zero = [&](uint8_t* at, int bytes) {
            for (int i = lane * 16; i < bytes; i += 512) sts128(smem_u32(at + i), 0, 0, 0, 0);
          };
          for (uint32_t gone = ~there & 0xffu; gone; gone &= gone - 1) zero(rk + (__ffs(gone) - 1) * 16 * D, 16 * D);
          fence_proxy_async_smem();  // zeros of an earlier tile come before the copies over them
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(&wr_full[tile % WR]);
            mbar_arrive_expect_tx(&rk_full[r], __popc(there) * 16 * D);
          }
          __syncwarp();
          if (lane < 8 && page >= 0) bulk_load_1d(rk + lane * 16 * D, a.c.k + off, 16 * D, &rk_full[r]);
          ++asked_k;
          if (!__all_sync(0xffffffffu, mbar_wait_prompt(&rv_free[r], freed, abort_flag, err, kDevTimeoutEmpty))) {
            ok = false;
            break;
          }
          for (uint32_t gone = ~there & 0xffu; gone; gone &= gone - 1) {
            zero(rv + (__ffs(gone) - 1) * 2 * C::V_OCTET, 8 * D);
            zero(rv + (__ffs(gone) - 1) * 2 * C::V_OCTET + C::V_OCTET, 8 * D);
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive_expect_tx(&rv_full[r], __popc(there) * 16 * D);
          __syncwarp();
          if (lane < 16 && page >= 0)  // lanes l and l + 8: the two octets of 16 keys
            bulk_load_1d(rv + ((lane & 7) * 2 + (lane >> 3)) * C::V_OCTET, a.c.v + off + (lane >> 3) * 8 * D, 8 * D, &rv_full[r]);
          ++asked_v;
        }
      }
      // every copy asked for lands before the CTA ends
      if (lane == 0) {
        for (uint32_t t = asked_k < RAW ? 0 : asked_k - RAW; t < asked_k; ++t)
          mbar_drain(&rk_full[t % RAW], (t / RAW) & 1, err, kDevTimeoutDrain);
        for (uint32_t t = asked_v < RAW ? 0 : asked_v - RAW; t < asked_v; ++t)
          mbar_drain(&rv_full[t % RAW], (t / RAW) & 1, err, kDevTimeoutDrain);
      }
      __syncwarp();
      if (lane == 0 && !cut) a.meta[blockIdx.x] = make_int4(0, 0, 0, 0);
      if (ok) hand(0);
    }
  } else if (warp >= 12) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_DEC));
    // -------------------------------------------------------------------- decode warps
    const int dw = warp - 12;
    constexpr int LPR = D / 16;                 // lanes to a K row
    constexpr int RPP = 128 / LPR;              // K rows of a pass of the four warps: 16 (D = 128) or 32
    constexpr int KP = BN / RPP;                // passes
    const int krow = (dw * 32 + lane) / LPR, kch = lane % LPR;
    // V: eight keys (octet vo of the tile) and D / 8 columns (chunk vc) a thread
    const int vo = (lane & 7) + 8 * (dw >> 1), vc = (lane >> 3) + 4 * (dw & 1);
    constexpr int VW = D / 32;                  // words of a chunk
    uint32_t seq = 0, tile = 0;
    bool ok = true;
    Stretch s;
    // a free place in the ring, and the codes that go there
    auto wait_both = [&](uint64_t* full) {
      return __all_sync(0xffffffffu,
                        mbar_wait_prompt(&kv_empty[seq % RING], ((seq / RING) & 1) ^ 1, abort_flag, err, kDevTimeoutEmpty) &&
                            mbar_wait_prompt(full, (tile / RAW) & 1, abort_flag, err, kDevTimeoutFull));
    };
    auto publish = [&](uint64_t* free) {
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(free);
        mbar_arrive(&kv_full[seq % RING]);
      }
      ++seq;
    };
    for (uint32_t si = 0; ok && take_warp(si, s); ++si) {
      for (int j = 0; j < s.n; ++j, ++tile) {
        const int r = tile % RAW;
        if (!(ok = wait_both(&rk_full[r]))) break;
        if (lane == 0) mbar_arrive(&wr_free[tile % WR]);
        {
          const uint32_t dst = smem_u32(smem + C::OFF_KV + (seq % RING) * C::KV_TILE);
          const uint32_t src = smem_u32(smem + C::OFF_RK + r * C::RAW_K) + krow * D + kch * 16;
          const bool odd = kch >= 4;  // the second slab's lanes store their pieces in the other order: no two meet in a bank
#pragma unroll
          for (int p = 0; p < KP; ++p) {
            const uint4 v = lds128(src + p * RPP * D);
            uint32_t h[8];
            kv_decode4<CODES>(odd ? v.z : v.x, h[0], h[1]);
            kv_decode4<CODES>(odd ? v.w : v.y, h[2], h[3]);
            kv_decode4<CODES>(odd ? v.x : v.z, h[4], h[5]);
            kv_decode4<CODES>(odd ? v.y : v.w, h[6], h[7]);
            const int row = p * RPP + krow, ch = (kch & 3) * 2 + odd;  // 16 columns: two 16-byte chunks of slab kch / 4
            const uint32_t rb = dst + (kch >> 2) * C::Q_SLAB + row * 128;
            sts128(rb + ((ch ^ (row & 7)) << 4), h[0], h[1], h[2], h[3]);
            sts128(rb + (((ch ^ 1) ^ (row & 7)) << 4), h[4], h[5], h[6], h[7]);
          }
        }
        publish(&rk_free[r]);
        if (!(ok = wait_both(&rv_full[r]))) break;
        {
          const uint32_t dst = smem_u32(smem + C::OFF_KV + (seq % RING) * C::KV_TILE) + (vo >> 3) * C::V_SLAB;
          const uint32_t src = smem_u32(smem + C::OFF_RV + r * C::RAW_V) + vo * C::V_OCTET + vc * (D / 8);
          uint32_t v[8][VW];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            if (VW == 4) {
              const uint4 q = lds128(src + e * D);
              v[e][0] = q.x;
              v[e][1] = q.y;
              v[e][VW - 2] = q.z;
              v[e][VW - 1] = q.w;
            } else {
              asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v[e][0]), "=r"(v[e][1]) : "r"(src + e * D) : "memory");
            }
          }
          const int64_t left = s.len - (s.key_base + (int64_t)j * BN + vo * 8);
          if (left < 8) {  // what lies behind the last token may be any bits
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (e >= left)
#pragma unroll
                for (int q = 0; q < VW; ++q) v[e][q] = 0;
          }
#pragma unroll
          for (int q = 0; q < VW; ++q) {
            uint32_t h[4][4];  // [column][key pair]
#pragma unroll
            for (int kp = 0; kp < 4; ++kp) {
              kv_decode4<CODES>(prmt(v[2 * kp][q], v[2 * kp + 1][q], 0x5140), h[0][kp], h[1][kp]);
              kv_decode4<CODES>(prmt(v[2 * kp][q], v[2 * kp + 1][q], 0x7362), h[2][kp], h[3][kp]);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int d = vc * (D / 8) + q * 4 + e;
              sts128(dst + d * 128 + (((vo & 7) ^ (d & 7)) << 4), h[e][0], h[e][1], h[e][2], h[e][3]);
            }
          }
        }
        publish(&rv_free[r]);
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS_SOFT));
    // -------------------------------------------------------------------- softmax warps
    const int g = (warp - 4) >> 2;
    const int quarter = warp & 3;
    const int rloc = quarter * 32 + lane;
    const uint32_t lane_off = (uint32_t)(quarter * 32) << 16;
    const uint32_t tS = tmem_base + lane_off + g * BN;
    const uint32_t tO = tmem_base + lane_off + NQ * BN + g * D;
    const uint32_t qrow = smem_u32(smem + g * C::Q_TILE) + rloc * 128;
    const uint32_t swz = rloc & 7;
    uint32_t done = 0, segs = 0, tile0 = 0;
    bool ok = true;
    Stretch s;
    for (uint32_t si = 0; ok && take_warp(si, s); ++si) {
      const int n = s.n;
      const int part_slot = (int)blockIdx.x * 2 + (si > 0);
      if (g * BM >= s.rows) {  // a slot of one tile
        tile0 += n;
        continue;
      }
      const int r = g * BM + rloc;
      const bool in = r < s.rows;
      const int token = (s.r0 + (in ? r : 0)) / a.per;  // of the sequence's new ones
      const int64_t ro = (int64_t)(s.s0 + token) * a.heads + s.kvh * a.per + (s.r0 + (in ? r : 0)) % a.per;
      // ------------------------------------------------------------ q as f16, the sign of the scale in it
      // The last stretch's scores of this tile are read, so its products are done with Q.  A warp's 32 rows come in whole
      // rows, LPQ lanes each, to their places; then every thread scales its own row there.
      float c = fabsf(a.scale_log2);
      {
        constexpr int LPQ = D / 8;  // 16-byte pieces of a row
        const uint32_t qtile = smem_u32(smem + g * C::Q_TILE) + quarter * 32 * 128;
        const int64_t src =
            in ? (int64_t)(s.s0 + token) * a.q_ts + (int64_t)(s.kvh * a.per + (s.r0 + r) % a.per) * a.q_hs : -1;
        const int ch = lane % LPQ, row0 = lane / LPQ;
        auto place = [&](int row) { return qtile + row * 128 + (ch >> 3) * C::Q_SLAB + (((ch & 7) ^ (row & 7)) << 4); };
        if (q_vec) {  // past L1, of which this much shared memory leaves little
#pragma unroll 4
          for (int i = 0; i < LPQ; ++i) {
            const int row = i * (32 / LPQ) + row0;
            const int64_t at = __shfl_sync(0xffffffffu, src, row);
            cp16_zfill(place(row), a.q + (at < 0 ? 0 : at + ch * 8), at >= 0);
          }
          asm volatile("cp.async.wait_all;" ::: "memory");
        } else {
#pragma unroll 1
          for (int i = 0; i < LPQ; ++i) {
            const int64_t at = __shfl_sync(0xffffffffu, src, i * (32 / LPQ) + row0);
            uint32_t e[4] = {0, 0, 0, 0};
            if (at >= 0)
#pragma unroll
              for (int k = 0; k < 4; ++k)
                e[k] = (uint32_t)__ldg(a.q + at + ch * 8 + 2 * k) | ((uint32_t)__ldg(a.q + at + ch * 8 + 2 * k + 1) << 16);
            sts128(place(i * (32 / LPQ) + row0), e[0], e[1], e[2], e[3]);
          }
        }
        __syncwarp();
        // (small loops here too: what runs once a stretch is fetched anew each time)
        const uint32_t sign = a.scale_log2 < 0.f ? 0x80008000u : 0u;
        auto piece = [&](int i) { return qrow + (i >> 3) * C::Q_SLAB + (((i & 7) ^ swz) << 4); };
        if (a.kind == 2) {
          float mx = 0.f, f;
#pragma unroll 4
          for (int i = 0; i < LPQ; ++i) {
            const uint4 v = lds128(piece(i));
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int k = 0; k < 4; ++k)
              mx = max3f(mx, fabsf(__uint_as_float(w[k] << 16)), fabsf(__uint_as_float(w[k] & 0xffff0000u)));
          }
          kv_row_scale(mx, f, c);
#pragma unroll 4
          for (int i = 0; i < LPQ; ++i) {
            const uint4 v = lds128(piece(i));
            uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int k = 0; k < 4; ++k)
              w[k] = kv_pack_f16(__uint_as_float(w[k] << 16) * f, __uint_as_float(w[k] & 0xffff0000u) * f) ^ sign;
            sts128(piece(i), w[0], w[1], w[2], w[3]);
          }
        } else if (sign) {
#pragma unroll 4
          for (int i = 0; i < LPQ; ++i) {
            const uint4 v = lds128(piece(i));
            sts128(piece(i), v.x ^ sign, v.y ^ sign, v.z ^ sign, v.w ^ sign);
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&q_full[g]);
      }
      // the keys of the row; a row that is not there sees all: its warp is spared the mask
      const int64_t pos = s.first + token;
      const int64_t key_base = s.key_base;
      const int64_t hi = in && a.causal && pos + 1 < s.len ? pos + 1 : s.len;
      const int64_t lo = in && a.window > 0 && pos + 1 > a.window ? pos + 1 - a.window : 0;
      const int64_t span = (int64_t)n * BN;
      const int klo = (int)(lo < key_base ? 0 : (lo - key_base < span ? lo - key_base : span));
      const int khi = (int)(hi < key_base ? 0 : (hi - key_base < span ? hi - key_base : span));
      // the tiles that every row of the warp sees whole
      const int full_lo = __reduce_max_sync(0xffffffffu, klo), full_hi = __reduce_min_sync(0xffffffffu, khi);
      float m_used = -INFINITY, u_used = kKvNoRef, l = 0.f;
      for (int j = 0; j < n; ++j) {
        const uint32_t T = tile0 + j;
        // (the ring only after the scores: a group that sat out slots may not look at it before it has come to them)
        if (!__all_sync(0xffffffffu, mbar_wait_prompt(&s_full[g], done & 1, abort_flag, err, kDevTimeoutScores)) ||
            !__all_sync(0xffffffffu,
                        mbar_wait_prompt(&wr_full[T % WR], (T / WR) & 1, abort_flag, err, kDevTimeoutScale))) {
          ok = false;
          break;
        }
        tc_fence_after();
        // The row's scores pass through registers 32 at a time, twice: for the maximum and for the weights.  Small
        // loops: two softmax warps and a decode warp share an instruction cache, and straight-line code for 128
        // scores is fetched more slowly than it runs.
        const float4* cs = consts + (T % WR) * 8;
        const int k0 = j * BN;
        const bool edge = k0 < full_lo || k0 + BN > full_hi;  // some row does not see the whole tile
        const int a0 = klo - k0, a1 = khi - k0;
        const bool far = cs[0].w > kKvFar;  // (m - u is at most the stretch's largest log2 vs)
        if (__builtin_expect(far, 0)) {
          const float2 e = far_sums(tS, cs, a0, a1, c, u_used, l);
          u_used = e.x;
          l = e.y;
        }
        uint32_t x[4][32];
#pragma unroll
        for (int k = 0; k < 4; ++k) tmem_ld_32x32b_x32(tS + 32 * k, x[k]);
        float4 cq[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) cq[q] = cs[q];
        tmem_wait_ld();
        if (edge) {
#pragma unroll
          for (int k = 0; k < BN / 32; ++k) {  // a bit a score: predicates come from the bits several at a time
            const uint32_t bits = below(a1 - 32 * k) & ~below(a0 - 32 * k);
#pragma unroll
            for (int i = 0; i < 32; ++i) x[k][i] = bits >> i & 1 ? x[k][i] : 0xff800000u;
          }
        }
        float mx = -INFINITY;
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          const uint32_t* v = &x[q >> 1][(q & 1) * 16];
          auto f = [&](int i) { return __uint_as_float(v[i]); };
          const float u0 = max3f(f(0), f(1), f(2)), u1 = max3f(f(3), f(4), f(5)), u2 = max3f(f(6), f(7), f(8)),
                      u3 = max3f(f(9), f(10), f(11)), u4 = max3f(f(12), f(13), f(14));
          // the factor is not 0, so that a masked -inf stays -inf for a scale of 0
          cq[q].x = fmaxf(c * cq[q].x, 1e-37f);
          mx = fmaxf(mx, __fmaf_rn(fmaxf(max3f(u0, u1, u2), max3f(u3, u4, f(15))), cq[q].x, cq[q].y));
        }
        const bool move = mx > m_used + kKvTop;
        float alpha = 1.f;
        if (move) {
          alpha = kv_ex2(m_used - (mx - kKvLift));
          m_used = mx - kKvLift;
          const float u = mx - cq[1].w;  // at most the t of the key that mx is of
          const float to = fmaxf(u_used, u);
          l *= kv_ex2(u_used - to);
          u_used = to;
        }
        const float m = m_used == -INFINITY ? 0.f : m_used;
        const float l_f = far ? 0.f : kv_ex2(m_used - u_used - cq[1].w);  // of the loudest page's weights in l
        float sum = 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          uint32_t w[16];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int q = 2 * k + h;
            const float off = cq[q].y - m;
            const f2 c2 = pk(cq[q].x, cq[q].x), o2 = pk(off, off);
            f2 la = pk(0.f, 0.f);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              float t0, t1;
              upk(fma2(pk(__uint_as_float(x[k][h * 16 + 2 * i]), __uint_as_float(x[k][h * 16 + 2 * i + 1])), c2, o2), t0, t1);
              const float p0 = kv_ex2(t0), p1 = kv_ex2(t1);
              la = add2(la, pk(p0, p1));
              w[h * 8 + i] = kv_pack_f16(p0, p1);
            }
            float s0, s1;
            upk(la, s0, s1);
            sum = __fmaf_rn(s0 + s1, cs[q].z, sum);
          }
          tmem_st_32x32b_x16(tS + 16 * k, w);
        }
        l = __fmaf_rn(sum, l_f, l);
        // O_g holds every product before these scores
        if (j > 0 && __any_sync(0xffffffffu, move)) {
#pragma unroll 1
          for (int k = 0; k < D / 16; ++k) {
            uint32_t o[16];
            tmem_ld_32x32b_x16(tO + 16 * k, o);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
            tmem_st_32x32b_x16(tO + 16 * k, o);
          }
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[g]);
        ++done;
      }
      if (!ok) break;
      tile0 += n;
      if (!__all_sync(0xffffffffu, mbar_wait_prompt(&o_full[g], segs++ & 1, abort_flag, err, kDevTimeoutPV))) {
        ok = false;
        break;
      }
      tc_fence_after();
      float* part = a.part + (int64_t)part_slot * ROWS * (D + 4);
      const KvStat stat{m_used, u_used, l};
      const float inv = stat.inv(), f = stat.half();
#pragma unroll 1
      for (int k = 0; k < D / 32; ++k) {
        uint32_t o[32];
        tmem_ld_32x32b_x32(tO + 32 * k, o);
        tmem_wait_ld();
        if (s.whole) {  // 16-bit rows, through the tile's Q (its products are done), so that whole rows go out
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
              w[e] = kv_pack(__uint_as_float(o[8 * i + 2 * e]) * inv * f * f, __uint_as_float(o[8 * i + 2 * e + 1]) * inv * f * f,
                             a.kind);
            const int ch = 4 * k + i;
            sts128(qrow + (ch >> 3) * C::Q_SLAB + (((ch & 7) ^ swz) << 4), w[0], w[1], w[2], w[3]);
          }
        } else if (in) {
          uint4* d4 = reinterpret_cast<uint4*>(part) + (int64_t)(8 * k) * ROWS + r;  // a warp's rows are neighbours
#pragma unroll
          for (int i = 0; i < 8; ++i) d4[i * ROWS] = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
        }
      }
      if (s.whole) {
        __syncwarp();
        constexpr int LPQ = D / 8;
        const uint32_t qtile = smem_u32(smem + g * C::Q_TILE) + quarter * 32 * 128;
        const int ch = lane % LPQ;
#pragma unroll 4
        for (int i = 0; i < LPQ; ++i) {
          const int row = i * (32 / LPQ) + lane / LPQ;
          const uint4 v = lds128(qtile + row * 128 + (ch >> 3) * C::Q_SLAB + (((ch & 7) ^ (row & 7)) << 4));
          const int64_t to = __shfl_sync(0xffffffffu, ro, row);
          if (__shfl_sync(0xffffffffu, (int)in, row)) *reinterpret_cast<uint4*>(a.out + to * D + ch * 8) = v;
        }
        __syncwarp();  // read before the next stretch's rows go there
      }
      if (in) {
        if (!s.whole) *reinterpret_cast<float4*>(part + (int64_t)ROWS * D + 4 * r) = make_float4(m_used, u_used, l, 0.f);
        else if (a.lse) a.lse[ro] = stat.lse();
      }
      tc_fence_before();  // the reads of O are ordered before the next segment's first product, through p_full
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

namespace {

template <int D, int CODES>
cudaError_t launch_chunk(KvAttnArgs a, const KvChunkWork& wk, int q_vec, int* err, cudaStream_t st) {
  auto kern = kv_attn_chunk_kernel<D, CODES>;
  static bool ready[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  if (!ready[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Cfg<D>::SMEM);
    if (e != cudaSuccess) return e;
    ready[dev] = true;
  }
  kv_attn_list_kernel<<<1, 1024, 0, st>>>(a, wk);
  if (const cudaError_t e = cudaGetLastError()) return e;
  a.workers = sm_count(dev) < kMaxWorkers ? sm_count(dev) : kMaxWorkers;
  kern<<<(unsigned)a.workers, THREADS, Cfg<D>::SMEM, st>>>(a, wk, q_vec, err);
  if (const cudaError_t e = cudaGetLastError()) return e;
  return launch_kv_attn_join(a, ROWS, st);
}

}  // namespace

size_t kv_attn_chunk_part_bytes(int dim) { return (size_t)kMaxWorkers * 2 * ROWS * (dim + 4) * 4; }
size_t kv_attn_chunk_list_bytes(int64_t slots) { return 256 + (size_t)slots * sizeof(KvListed); }

cudaError_t launch_kv_attn_chunk(const KvAttnArgs& a, void* list, int* err, cudaStream_t st) {
  KvChunkWork wk;
  wk.head = static_cast<int64_t*>(list);
  wk.list = reinterpret_cast<KvListed*>(static_cast<uint8_t*>(list) + 256);
  const int q_vec = (reinterpret_cast<uintptr_t>(a.q) & 15u) == 0 && a.q_ts % 8 == 0 && a.q_hs % 8 == 0;
#define H3Q_KV_C(DD, CC) \
  if (a.c.dim == DD && a.c.codes == CC) return launch_chunk<DD, CC>(a, wk, q_vec, err, st);
  H3Q_KV_C(64, 0) H3Q_KV_C(64, 1) H3Q_KV_C(128, 0) H3Q_KV_C(128, 1)
#undef H3Q_KV_C
  return cudaErrorInvalidValue;
}

}  // namespace h3q
