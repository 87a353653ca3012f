// kv_capi.cu -- C ABI of the 8-bit paged key / value cache (include/h3q.h): argument checks, workspace carving and the
// choice of the attention kernel.
#include <cmath>
#include <cstdarg>
#include <cstdint>
#include <cstdio>
#include <cuda_runtime.h>
#include "../../include/h3q.h"
#include "h3q_internal.h"
#include "kv_attn.cuh"

namespace h3q {
void set_last_error(const char* msg);
cudaError_t launch_kv_write(const KvCache& c, const KvSeqs& s, const int32_t* past, const void* k, int64_t k_ts,
                            int64_t k_hs, const void* v, int64_t v_ts, int64_t v_hs, int kind, bool vec,
                            cudaStream_t st);
cudaError_t launch_kv_read(const KvCache& c, const KvSeqs& s, const int32_t* first, void* k_out, void* v_out, int kind,
                           cudaStream_t st);
size_t kv_attn_rows_part_bytes(int dim, int tile);
cudaError_t launch_kv_attn_rows(const KvAttnArgs& a, int tile, cudaStream_t st);
size_t kv_attn_chunk_part_bytes(int dim);
size_t kv_attn_chunk_list_bytes(int64_t slots);
cudaError_t launch_kv_attn_chunk(const KvAttnArgs& a, void* list, int* err, cudaStream_t st);
}  // namespace h3q

using namespace h3q;

namespace {

h3q_status fail(h3q_status s, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof buf, fmt, ap);
  va_end(ap);
  set_last_error(buf);
  return s;
}

h3q_status cuda_status(cudaError_t e, const char* what) {
  if (e == cudaSuccess) return H3Q_OK;
  return fail(H3Q_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

bool aligned(const void* p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
size_t a256(size_t v) { return (v + 255) / 256 * 256; }

h3q_status check_cache(const h3q_kv_cache* c, const char* what) {
  if (!c) return fail(H3Q_ERR_ARG, "%s: null cache", what);
  if (c->pages < 0 || c->kv_heads < 1) return fail(H3Q_ERR_ARG, "%s: negative pages or no heads", what);
  if (c->codes != H3Q_KV_INT8 && c->codes != H3Q_KV_E4M3)
    return fail(H3Q_ERR_ARG, "%s: unknown code type %d (0 int8, 1 e4m3)", what, c->codes);
  if (c->head_dim != 64 && c->head_dim != 128)
    return fail(H3Q_ERR_UNSUPPORTED, "%s: this build handles head_dim 64 and 128 (got %d)", what, c->head_dim);
  if (c->page != 16 && c->page != 32 && c->page != 64 && c->page != 128)
    return fail(H3Q_ERR_UNSUPPORTED, "%s: this build handles pages of 16, 32, 64 or 128 tokens (got %d)", what, c->page);
  if (c->kv_heads > 4096 || c->pages >= (int64_t)1 << 31)
    return fail(H3Q_ERR_UNSUPPORTED, "%s: this build handles up to 4096 kv heads and less than 2^31 pages", what);
  if (c->pages > 0) {
    if (!c->k || !c->v || !c->k_scale || !c->v_scale) return fail(H3Q_ERR_ARG, "%s: null cache pointer", what);
    if (!aligned(c->k, 16) || !aligned(c->v, 16) || !aligned(c->k_scale, 4) || !aligned(c->v_scale, 4))
      return fail(H3Q_ERR_ARG, "%s: codes must be 16-byte aligned and scales 4-byte aligned", what);
  }
  return H3Q_OK;
}

h3q_status check_seqs(const int32_t* table, int64_t width, const int32_t* starts, int64_t batch, int64_t tokens,
                      const char* what) {
  if (tokens < 0 || batch < 0 || width < 0) return fail(H3Q_ERR_ARG, "%s: negative shape", what);
  if (tokens == 0 || batch == 0) {
    if (tokens > 0) return fail(H3Q_ERR_ARG, "%s: tokens without a sequence", what);
    return H3Q_OK;
  }
  if (tokens > (int64_t)1 << 24 || batch > (int64_t)1 << 20 || width > (int64_t)1 << 26)
    return fail(H3Q_ERR_UNSUPPORTED, "%s: this build handles 2^24 tokens, 2^20 sequences and 2^26 pages a sequence", what);
  if (!starts && tokens % batch != 0)
    return fail(H3Q_ERR_ARG, "%s: without starts, tokens (%lld) must divide evenly over the batch (%lld)", what,
                (long long)tokens, (long long)batch);
  if (width > 0 && !table) return fail(H3Q_ERR_ARG, "%s: null page table", what);
  return H3Q_OK;
}

KvCache cache_of(const h3q_kv_cache* c) {
  KvCache r{};
  r.k = static_cast<uint8_t*>(c->k);
  r.v = static_cast<uint8_t*>(c->v);
  r.k_scale = c->k_scale;
  r.v_scale = c->v_scale;
  r.pages = c->pages;
  r.kv_heads = (int)c->kv_heads;
  r.page = c->page;
  r.page_log2 = c->page == 16 ? 4 : c->page == 32 ? 5 : c->page == 64 ? 6 : 7;
  r.dim = c->head_dim;
  r.codes = c->codes;
  return r;
}

KvSeqs seqs_of(const int32_t* table, int64_t width, const int32_t* starts, int64_t batch, int64_t tokens) {
  KvSeqs s{};
  s.table = table;
  s.starts = starts;
  s.width = width;
  s.batch = (int)batch;
  s.tokens = (int)tokens;
  s.each = starts ? 0 : (int)(tokens / batch);
  return s;
}

// How a call's attention is cut: the row kernel takes the sequences of up to 32 query rows (new tokens times the query
// heads of a kv head), the chunk kernel the others.  Each has its own part of the workspace.  Measured with their joins (int8, 8
// kv heads of 128; 16 sequences of 4096 tokens / 64 of 1024): 16 rows 44 / 54 us as a tile of 16, 59 / 69 us as one of 32, 104 /
// 140 us in the chunk kernel; 32 rows 65 / 80 us as a tile of 32, 105 / 142 us in the chunk kernel.  Beyond 32 rows a row tile's
// accumulators no longer fit a warp's registers.  The host knows no more than max_new: a call of ragged sequences without it is
// planned for the worst, with tiles of 32 and the chunk kernel's launches (one token of 64 sequences of up to 16384, 40 heads:
// 351 us in four kernels for 228 in two).
struct AttnPlan {
  int tile;        // rows of a slot of the row kernel, 0: none of the sequences can be its
  int chunk;       // the chunk kernel runs
  int64_t slots, chunk_slots;
  size_t part, meta, chunk_part, chunk_meta, chunk_list, bytes;
};

constexpr int kRowsMax = 32;

AttnPlan plan(int64_t tokens, int64_t batch, int64_t heads, int64_t kv_heads, int64_t max_new, bool even, int dim) {
  AttnPlan p{};
  const int64_t per = heads / kv_heads, most = max_new * per;
  p.chunk = most > kRowsMax;
  p.tile = p.chunk && even ? 0 : (most <= 16 ? 16 : kRowsMax);
  if (p.tile) {
    p.slots = batch;
    p.part = a256(kv_attn_rows_part_bytes(dim, p.tile));
    p.meta = a256(kMaxRowWorkers * sizeof(int4));
  }
  if (p.chunk) {
    p.chunk_slots = tokens * per / 256 + batch;
    p.chunk_part = a256(kv_attn_chunk_part_bytes(dim));
    p.chunk_meta = a256(kMaxWorkers * sizeof(int4));
    p.chunk_list = a256(kv_attn_chunk_list_bytes(p.chunk_slots));
  }
  p.bytes = p.part + p.meta + p.chunk_part + p.chunk_meta + p.chunk_list;
  return p;
}

int64_t max_new_of(int64_t max_new, const int32_t* starts, int64_t batch, int64_t tokens) {
  if (!starts) return tokens / batch;
  return max_new <= 0 || max_new > tokens ? tokens : max_new;
}

h3q_status check_heads(int64_t heads, int64_t kv_heads, const char* what) {
  if (heads < 1 || kv_heads < 1 || heads % kv_heads != 0)
    return fail(H3Q_ERR_ARG, "%s: %lld query heads do not share %lld kv heads evenly", what, (long long)heads,
                (long long)kv_heads);
  if (heads > 65536) return fail(H3Q_ERR_UNSUPPORTED, "%s: this build handles up to 65536 query heads", what);
  return H3Q_OK;
}

}  // namespace

extern "C" {

h3q_status h3q_kv_write(const h3q_kv_cache* cache, const void* k, int64_t k_token_stride, int64_t k_head_stride,
                        const void* v, int64_t v_token_stride, int64_t v_head_stride, int kind, int64_t tokens,
                        const int32_t* page_table, int64_t table_width, const int32_t* past, const int32_t* starts,
                        int64_t batch, void* stream) {
  const char* what = "kv_write";
  if (h3q_status s = check_cache(cache, what)) return s;
  if (kind < 0 || kind > 2) return fail(H3Q_ERR_ARG, "%s: unsupported kind %d (0 f32, 1 f16, 2 bf16)", what, kind);
  if (h3q_status s = check_seqs(page_table, table_width, starts, batch, tokens, what)) return s;
  if (tokens == 0 || table_width == 0 || cache->pages == 0) return H3Q_OK;
  if (!k || !v || !past) return fail(H3Q_ERR_ARG, "%s: null pointer", what);
  if (k_token_stride < 0 || k_head_stride < 0 || v_token_stride < 0 || v_head_stride < 0)
    return fail(H3Q_ERR_ARG, "%s: negative stride", what);
  const unsigned size = kind == 0 ? 4 : 2;
  if (!aligned(k, size) || !aligned(v, size)) return fail(H3Q_ERR_ARG, "%s: k and v must be aligned to their type", what);
  const int64_t step = 16 / size;
  const bool vec = aligned(k, 16) && aligned(v, 16) && k_token_stride % step == 0 && k_head_stride % step == 0 &&
                   v_token_stride % step == 0 && v_head_stride % step == 0;
  return cuda_status(launch_kv_write(cache_of(cache), seqs_of(page_table, table_width, starts, batch, tokens), past, k,
                                     k_token_stride, k_head_stride, v, v_token_stride, v_head_stride, kind, vec,
                                     static_cast<cudaStream_t>(stream)),
                     what);
}

h3q_status h3q_kv_read(const h3q_kv_cache* cache, const int32_t* page_table, int64_t table_width, const int32_t* first,
                       const int32_t* starts, int64_t batch, int64_t tokens, void* k_out, void* v_out, int kind,
                       void* stream) {
  const char* what = "kv_read";
  if (h3q_status s = check_cache(cache, what)) return s;
  if (kind < 0 || kind > 2) return fail(H3Q_ERR_ARG, "%s: unsupported kind %d (0 f32, 1 f16, 2 bf16)", what, kind);
  if (h3q_status s = check_seqs(page_table, table_width, starts, batch, tokens, what)) return s;
  if (tokens == 0) return H3Q_OK;
  if (!k_out || !v_out) return fail(H3Q_ERR_ARG, "%s: null pointer", what);
  if (!aligned(k_out, 16) || !aligned(v_out, 16)) return fail(H3Q_ERR_ARG, "%s: outputs must be 16-byte aligned", what);
  return cuda_status(launch_kv_read(cache_of(cache), seqs_of(page_table, table_width, starts, batch, tokens), first,
                                    k_out, v_out, kind, static_cast<cudaStream_t>(stream)),
                     what);
}

size_t h3q_kv_attention_workspace_size(int64_t tokens, int64_t batch, int64_t heads, int64_t kv_heads, int head_dim,
                                       int64_t max_new) {
  if (tokens <= 0 || batch <= 0 || heads <= 0 || kv_heads <= 0 || max_new < 0) return 0;
  const int64_t most = max_new == 0 || max_new > tokens ? tokens : max_new;
  return plan(tokens, batch, heads, kv_heads, most, false, head_dim).bytes;
}

h3q_status h3q_kv_attention(const h3q_kv_cache* cache, const void* q, int kind, int64_t q_token_stride,
                            int64_t q_head_stride, int64_t tokens, int64_t heads, const int32_t* page_table,
                            int64_t table_width, const int32_t* lengths, const int32_t* starts, int64_t batch,
                            int64_t max_new, float scale, int causal, int64_t window, void* out, float* lse,
                            void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "kv_attention";
  if (h3q_status s = check_cache(cache, what)) return s;
  if (kind != H3Q_KIND_F16 && kind != H3Q_KIND_BF16)
    return fail(H3Q_ERR_ARG, "%s: unsupported kind %d (1 f16, 2 bf16)", what, kind);
  if (h3q_status s = check_heads(heads, cache->kv_heads, what)) return s;
  if (h3q_status s = check_seqs(page_table, table_width, starts, batch, tokens, what)) return s;
  if (max_new < 0 || window < 0) return fail(H3Q_ERR_ARG, "%s: negative max_new or window", what);
  if (window > 0 && !causal) return fail(H3Q_ERR_ARG, "%s: a window needs causal attention", what);
  if (!std::isfinite(scale)) return fail(H3Q_ERR_ARG, "%s: scale must be finite", what);
  if (tokens == 0) return H3Q_OK;
  if (!q || !out || !lengths) return fail(H3Q_ERR_ARG, "%s: null pointer", what);
  if (q_token_stride < 0 || q_head_stride < 0) return fail(H3Q_ERR_ARG, "%s: negative stride", what);
  if (!aligned(q, 2) || !aligned(out, 16)) return fail(H3Q_ERR_ARG, "%s: out must be 16-byte aligned", what);
  const int64_t most = max_new_of(max_new, starts, batch, tokens);
  if (most * (heads / cache->kv_heads) > (int64_t)1 << 30)
    return fail(H3Q_ERR_UNSUPPORTED, "%s: this build handles 2^30 query rows to a sequence and kv head", what);
  const AttnPlan p = plan(tokens, batch, heads, cache->kv_heads, most, !starts, cache->head_dim);
  const size_t need = h3q_kv_attention_workspace_size(tokens, batch, heads, cache->kv_heads, cache->head_dim,
                                                      starts ? max_new : most);
  if (!workspace || workspace_bytes < need)
    return fail(H3Q_ERR_WORKSPACE, "%s: workspace of %zu bytes, need %zu", what, workspace_bytes, need);
  if (!aligned(workspace, 16)) return fail(H3Q_ERR_ARG, "%s: workspace must be 16-byte aligned", what);
  KvAttnArgs a{};
  a.c = cache_of(cache);
  a.s = seqs_of(page_table, cache->pages > 0 ? table_width : 0, starts, batch, tokens);  // no pages: no keys
  a.q = static_cast<const uint16_t*>(q);
  a.q_ts = q_token_stride;
  a.q_hs = q_head_stride;
  a.kind = kind;
  a.heads = (int)heads;
  a.per = (int)(heads / cache->kv_heads);
  a.lengths = lengths;
  a.window = window;
  a.causal = causal != 0;
  a.scale_log2 = scale * 1.44269504088896340736f;
  a.out = static_cast<uint16_t*>(out);
  a.lse = lse;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  if (p.chunk) {
    int* err = error_word_current();
    if (!err) return fail(H3Q_ERR_CUDA, "%s: could not set up the device error word", what);
    KvAttnArgs b = a;
    b.row_lo = p.tile;
    b.row_hi = 0x7fffffff;
    b.one = 0;
    b.slots = p.chunk_slots;
    b.part = reinterpret_cast<float*>(ws);
    b.meta = reinterpret_cast<int4*>(ws + p.chunk_part);
    if (h3q_status s = cuda_status(launch_kv_attn_chunk(b, ws + p.chunk_part + p.chunk_meta, err, st), what)) return s;
    ws += p.chunk_part + p.chunk_meta + p.chunk_list;
  }
  if (!p.tile) return H3Q_OK;
  a.row_lo = 0;
  a.row_hi = p.tile;
  a.last = !p.chunk;
  a.one = 1;
  a.slots = p.slots;
  a.part = reinterpret_cast<float*>(ws);
  a.meta = reinterpret_cast<int4*>(ws + p.part);
  return cuda_status(launch_kv_attn_rows(a, p.tile, st), what);
}

}  // extern "C"
