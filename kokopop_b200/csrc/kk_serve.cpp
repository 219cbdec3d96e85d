// C ABI of the serving operators of a token model (include/kokopop_b200.h):
// argument checks, workspaces and launches.
#include "kk_host.h"

#include <algorithm>
#include <cstdint>

using namespace kk;

namespace {

[[noreturn]] void invalid(const std::string &m) { throw KKError(KK_ERROR_INVALID_ARGUMENT, m); }

void need(bool ok, const char *m) {
    if (!ok) invalid(m);
}

bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }
bool aligned4(const int32_t *p) { return ((uintptr_t)p & 3) == 0; }
bool aligned8(const int64_t *p) { return ((uintptr_t)p & 7) == 0; }
bool dtype16(int dtype) { return dtype == KK_DTYPE_F16 || dtype == KK_DTYPE_BF16; }
bool dtype_any(int dtype) { return dtype == KK_DTYPE_F32 || dtype16(dtype); }

// whether [a, a + n) and [b, b + m) have nothing in common
bool apart(const int32_t *a, int64_t n, const int32_t *b, int64_t m) {
    return (uintptr_t)(a + n) <= (uintptr_t)b || (uintptr_t)(b + m) <= (uintptr_t)a;
}

constexpr int64_t kMaxTokens = INT32_MAX / 2;  // rows, or requests, of one call
// outputs and inputs of a product: the kernel's 32-bit indices reach a chunk
// of k and a block of outputs further
constexpr int32_t kMaxSide = INT32_MAX - 65535;

PagedCacheView cache_view(const kk_paged_cache *c) {
    need(c && c->k && c->v, "null cache");
    need(dtype16(c->dtype), "cache dtype is not F16 or BF16");
    need(c->n_kv_heads >= 1 && c->n_kv_heads <= 65535, "cache n_kv_heads out of range [1, 65535]");
    need(c->head_dim >= 8 && c->head_dim <= KK_PAGED_MAX_HEAD_DIM && c->head_dim % 8 == 0,
         "cache head_dim is not a multiple of 8 in [8, 128]");
    need(c->page_size >= 1 && c->n_pages >= 1 && c->n_pages <= INT32_MAX, "cache page_size or n_pages out of range");
    need(aligned16(c->k) && aligned16(c->v), "cache k and v must be 16-byte aligned");
    need(c->page_stride >= 0 && c->token_stride >= 0 && c->head_stride >= 0 && c->page_stride % 8 == 0 &&
             c->token_stride % 8 == 0 && c->head_stride % 8 == 0,
         "cache strides must be multiples of 8 values");
    PagedCacheView v;
    v.k = c->k;
    v.v = c->v;
    v.bf16 = c->dtype == KK_DTYPE_BF16;
    v.n_kv_heads = c->n_kv_heads;
    v.head_dim = c->head_dim;
    v.page_size = c->page_size;
    v.n_pages = c->n_pages;
    v.page_stride = c->page_stride;
    v.token_stride = c->token_stride;
    v.head_stride = c->head_stride;
    return v;
}

cudaStream_t stream_of(kk_ctx *ctx, void *stream) { return stream ? (cudaStream_t)stream : ctx->st; }

bool capturing(cudaStream_t st) {
    cudaStreamCaptureStatus s = cudaStreamCaptureStatusNone;
    if (cudaStreamIsCapturing(st, &s) != cudaSuccess) {
        cudaGetLastError();  // the legacy stream while another one captures
        return false;
    }
    return s != cudaStreamCaptureStatusNone;
}

// Pieces of the key axis for the chunk kernel: the number that gives the
// shortest time of whole rounds of 148 blocks, a block's start and end costing
// as much as kPieceEnds of its steps of 128 keys (1.6 us each) and the join
// with its traffic as much as kJoinSteps. Both are fitted to a sweep on B200:
// 8 to 448 blocks, 1000 to 30000 keys, heads of 64 and of 128, 1 to 64 pieces.
// With them the chosen number is 1 % slower than the best one on average and
// 13 % at most; with 3 and 3 6 % and 46 % (200 blocks over 2000 keys: 117 us in
// two pieces, 80 in one).
constexpr int kPieceEnds = 8, kJoinSteps = 8;
int chunk_pieces(int64_t blocks, int64_t keys) {
    const int64_t most = std::min<int64_t>((keys + 255) / 256, 64);
    int best = 1;
    int64_t best_cost = INT64_MAX;
    for (int64_t s = 1; s <= most; ++s) {
        const int64_t steps = (keys + 128 * s - 1) / (128 * s);
        const int64_t cost = (blocks * s + 147) / 148 * (steps + kPieceEnds) + (s > 1 ? kJoinSteps : 0);
        if (cost < best_cost) best = (int)s, best_cost = cost;
    }
    return best;
}

// For the row kernel: about two blocks for each of the two places on an SM,
// 256 keys or more each. Measured on B200 at 148, 296, 592, 888, 1184, 2368
// blocks, 32 heads on 8, one token each: 64 requests of 17-4099 keys 113, 113,
// 106, 106, 104, 113 us (heads of 64: 64, 64, 60, 60, 67, 64); 7 of 30011-65000
// keys 264, 229, 218, 227, 229, 230; one of 65000 51, 52, 57, 64, 67, 84.
int row_pieces(int64_t blocks, int64_t keys) {
    return (int)std::min<int64_t>(std::min((592 + blocks - 1) / blocks, (keys + 255) / 256), 256);
}

}  // namespace

extern "C" {

int kk_page_tables_device(kk_ctx *ctx, int32_t n_seqs, int32_t page_size, int32_t max_pages, const int32_t *ctx_len,
                          const int32_t *new_len, const int32_t *free_pages, int32_t n_free,
                          const int32_t *free_range, int32_t *table, int32_t *seq_len, int32_t *cu_new,
                          int64_t n_tokens, int64_t *slots, int32_t *positions, int32_t *status, void *stream) {
    return guarded([&] {
        need(ctx && ctx_len && new_len && free_range && table && seq_len && cu_new && status, "null argument");
        need(n_seqs >= 1 && page_size >= 1 && max_pages >= 1, "n_seqs, page_size or max_pages below 1");
        need(n_seqs <= kMaxTokens, "n_seqs out of range");
        need(n_free >= 0 && (free_pages || n_free == 0), "null free_pages or negative n_free");
        need(n_tokens >= 0 && n_tokens <= kMaxTokens, "n_tokens out of range");
        need(slots || n_tokens == 0, "null slots");
        need(aligned4(ctx_len) && aligned4(new_len) && aligned4(free_pages) && aligned4(free_range) &&
                 aligned4(table) && aligned4(seq_len) && aligned4(cu_new) && aligned4(positions) && aligned4(status) &&
                 aligned8(slots),
             "an argument is not aligned to its type");
        need(apart(status, 3, free_range, 2), "status overlaps free_range");
        need(apart(seq_len, n_seqs, ctx_len, n_seqs) && apart(seq_len, n_seqs, new_len, n_seqs) &&
                 apart(cu_new, n_seqs + 1ll, ctx_len, n_seqs) && apart(cu_new, n_seqs + 1ll, new_len, n_seqs),
             "seq_len or cu_new overlaps ctx_len or new_len");
        use_device(ctx);
        PageTablesArgs a;
        a.n_seqs = n_seqs;
        a.page_size = page_size;
        a.max_pages = max_pages;
        a.ctx_len = ctx_len;
        a.new_len = new_len;
        a.free_pages = free_pages;
        a.free_cap = n_free;
        a.free_range = free_range;
        a.table = table;
        a.seq_len = seq_len;
        a.cu_new = cu_new;
        a.n_tokens = n_tokens;
        a.slots = slots;
        a.positions = positions;
        a.status = status;
        check_cuda(page_tables(a, stream_of(ctx, stream)), "page tables launch");
        ++ctx->n_launches;
        return KK_OK;
    });
}

int kk_cache_append_device(kk_ctx *ctx, const kk_paged_cache *cache, int64_t n_tokens, const int64_t *slots,
                           int32_t dtype, const void *k, int64_t k_stride, const void *v, int64_t v_stride,
                           void *stream) {
    return guarded([&] {
        need(ctx != nullptr, "null argument");
        CacheAppendArgs a;
        a.cache = cache_view(cache);
        need(n_tokens >= 0 && n_tokens <= kMaxTokens, "n_tokens out of range");
        need(dtype_any(dtype), "dtype is not F32, F16 or BF16");
        if (n_tokens == 0) return KK_OK;
        need(slots && k && v, "null argument");
        need(aligned8(slots), "slots is not aligned to its type");
        const int64_t row = (int64_t)a.cache.n_kv_heads * a.cache.head_dim, step = dtype == KK_DTYPE_F32 ? 4 : 8;
        need(aligned16(k) && aligned16(v), "k and v must be 16-byte aligned");
        need(k_stride >= row && v_stride >= row && k_stride % step == 0 && v_stride % step == 0,
             "k and v strides must hold a row and be multiples of 16 bytes");
        use_device(ctx);
        a.n_tokens = n_tokens;
        a.slots = slots;
        a.dtype = dtype;
        a.k = k;
        a.v = v;
        a.k_stride = k_stride;
        a.v_stride = v_stride;
        check_cuda(cache_append(a, stream_of(ctx, stream)), "cache append launch");
        ++ctx->n_launches;
        return KK_OK;
    });
}

int kk_paged_attention_device(kk_ctx *ctx, const kk_paged_cache *cache, int32_t n_seqs, const int32_t *seq_len,
                              const int32_t *cu_new, int64_t n_tokens, int32_t max_new, int32_t max_len,
                              const int32_t *table, int32_t max_pages, const void *q, int64_t q_stride,
                              int32_t n_heads, float scale, int32_t window, void *out, int64_t out_stride,
                              void *stream) {
    return guarded([&] {
        need(ctx != nullptr, "null argument");
        PagedAttnArgs a;
        a.cache = cache_view(cache);
        need(seq_len && cu_new && table, "null argument");
        need(aligned4(seq_len) && aligned4(cu_new) && aligned4(table),
             "seq_len, cu_new or table is not aligned to its type");
        need(n_seqs >= 1 && max_pages >= 1 && max_new >= 0 && max_len >= 0,
             "n_seqs or max_pages below 1, or a negative max_new or max_len");
        need(n_seqs <= kMaxTokens, "n_seqs out of range");
        need(n_tokens >= 0 && n_tokens <= kMaxTokens, "n_tokens out of range");
        need(n_heads >= 1 && n_heads % a.cache.n_kv_heads == 0, "n_heads is not a multiple of the cache's n_kv_heads");
        need(scale == scale, "scale is not a number");
        need(window >= 0, "negative window");
        if (n_tokens == 0) return KK_OK;
        need(q && out, "null argument");
        const int64_t row = (int64_t)n_heads * a.cache.head_dim;
        need(aligned16(q) && aligned16(out), "q and out must be 16-byte aligned");
        need(q_stride >= row && out_stride >= row && q_stride % 8 == 0 && out_stride % 8 == 0,
             "q and out strides must hold a row and be multiples of 8 values");
        const int group = n_heads / a.cache.n_kv_heads;
        int64_t keys = std::max(max_len, 1);  // that a query sees, from the lengths that the caller names
        if (window > 0) keys = std::min<int64_t>(keys, window);
        const PagedAttnPlan plan = paged_attn_plan(a.cache, n_heads, n_tokens, n_seqs, max_new, keys);
        need(plan.tiles <= INT32_MAX && n_tokens * group <= INT32_MAX,
             "n_tokens x query heads per key head out of range");
        use_device(ctx);
        cudaStream_t st = stream_of(ctx, stream);
        a.n_seqs = n_seqs;
        a.n_heads = n_heads;
        a.max_pages = max_pages;
        a.seq_len = seq_len;
        a.cu_new = cu_new;
        a.table = table;
        a.n_tokens = n_tokens;
        a.q = q;
        a.out = out;
        a.q_stride = q_stride;
        a.out_stride = out_stride;
        a.scale = scale;
        a.window = window;
        a.part_o = nullptr;
        a.part_ml = nullptr;
        a.count = nullptr;
        a.part_n = nullptr;
        a.err = ctx->serving_err();
        // pieces of the key axis
        const int64_t rows = std::min<int64_t>(n_tokens, std::max(max_new, 1)) * group;
        // (all rows are in some tile, whatever max_new says)
        const int64_t least = (n_tokens * group + plan.unit - 1) / plan.unit;
        const int64_t blocks =
            std::max(least, std::min(plan.tiles - n_seqs + plan.busy,  // idle slots have no block
                                     plan.busy * ((rows + plan.unit - 1) / plan.unit))) *
            a.cache.n_kv_heads;
        if (window > 0) keys = std::min<int64_t>(std::max(max_len, 1), (int64_t)window + plan.unit / group + 16);
        a.splits = capturing(st) ? 1 : plan.chunk ? chunk_pieces(blocks, keys) : row_pieces(blocks, keys);
        const int64_t step = plan.chunk ? 128 : 64;
        a.split_keys = (int)std::min<int64_t>(((keys + a.splits - 1) / a.splits + step - 1) / step * step,
                                              INT32_MAX / 128 * 128);
        if (a.splits == 1) {
            check_cuda(paged_attn(plan, a, st), "paged attention launch");
            ++ctx->n_launches;
            return KK_OK;
        }
        CallScope call_scope(*ctx, st, false);
        const size_t parts = (size_t)n_tokens * n_heads * a.splits;
        a.part_o = ctx->buf("paged_part_o", parts * a.cache.head_dim);
        a.part_ml = (float2 *)ctx->buf("paged_part_ml", parts * 2);
        if (plan.chunk) {
            a.part_n = (int *)ctx->buf("paged_part_n", (size_t)n_tokens * n_heads);
        } else {
            DevBuf &count = ctx->ws["paged_count"];
            const size_t count_bytes = (size_t)plan.tiles * a.cache.n_kv_heads * sizeof(unsigned);
            if (count.bytes < count_bytes) {
                count.ensure(count_bytes);
                const cudaError_t e = cudaMemsetAsync(count.p, 0, count.bytes, st);
                if (e != cudaSuccess) count.release();  // not to be taken for cleared
                check_cuda(e, "clear the piece counters");
            }
            a.count = (unsigned *)count.p;
        }
        check_cuda(paged_attn(plan, a, st), "paged attention launch");
        ctx->n_launches += plan.chunk ? 2 : 1;
        return KK_OK;
    });
}

int kk_q4_matvec_device(kk_ctx *ctx, int64_t n_rows, int32_t n_out, int32_t n_in, int32_t group, const uint8_t *w,
                        const uint16_t *scales, int32_t dtype, const void *x, int64_t x_stride, const float *bias,
                        void *out, int64_t out_stride, void *stream) {
    return guarded([&] {
        need(ctx && w && scales, "null argument");
        need(n_rows >= 0 && n_rows <= 8 * 65535 && n_out >= 1 && n_out <= kMaxSide && n_in >= 1 &&
                 n_in <= kMaxSide,
             "n_rows, n_out or n_in out of range");
        need(group == 32 || group == 64 || group == 128, "group is not 32, 64 or 128");
        need(n_in % group == 0, "n_in is not a multiple of the group");
        need(dtype_any(dtype), "dtype is not F32, F16 or BF16");
        if (n_rows == 0) return KK_OK;
        need(x && out, "null argument");
        need(aligned16(w) && aligned16(x), "w and x must be 16-byte aligned");
        need(((uintptr_t)scales & 1) == 0 && ((uintptr_t)bias & 3) == 0 &&
                 ((uintptr_t)out & (dtype == KK_DTYPE_F32 ? 3 : 1)) == 0,
             "scales, bias or out is not aligned to its type");
        need(x_stride >= n_in && x_stride % (dtype == KK_DTYPE_F32 ? 4 : 8) == 0,
             "x stride must hold a row and be a multiple of 16 bytes");
        need(out_stride >= n_out, "out stride must hold a row");
        use_device(ctx);
        Q4MatvecArgs a;
        a.n_rows = n_rows;
        a.n_out = n_out;
        a.n_in = n_in;
        a.group = group;
        a.w = w;
        a.scales = (const __half *)scales;
        a.dtype = dtype;
        a.x = x;
        a.x_stride = x_stride;
        a.bias = bias;
        a.out = out;
        a.out_stride = out_stride;
        a.err = ctx->serving_err();
        check_cuda(q4_matvec(a, stream_of(ctx, stream)), "4-bit product launch");
        ++ctx->n_launches;
        return KK_OK;
    });
}

int kk_serving_status(kk_ctx *ctx, void *stream) {
    return guarded([&] {
        need(ctx != nullptr, "null argument");
        use_device(ctx);
        cudaStream_t st = stream_of(ctx, stream);
        need(!capturing(st), "the stream is being captured");
        int code = 0;
        check_cuda(cudaMemcpyAsync(&code, ctx->serving_err(), sizeof code, cudaMemcpyDeviceToHost, st),
                   "read serving status");
        check_cuda(cudaStreamSynchronize(st), "serving operators");
        if (code == 0) return KK_OK;
        check_cuda(cudaMemsetAsync(ctx->serving_err(), 0, sizeof code, st), "clear serving status");
        check_cuda(cudaStreamSynchronize(st), "clear serving status");
        const std::string c = " (code " + std::to_string(code) + ")";
        if (code == kErrPagedWait) throw KKError(KK_ERROR_INFERENCE, "paged attention timed out waiting" + c);
        if (code == kErrQ4Wait) throw KKError(KK_ERROR_INFERENCE, "4-bit product timed out waiting" + c);
        throw KKError(KK_ERROR_INFERENCE, "bounded wait ran out, self-test" + c);
    });
}

int kk_serving_wait_selftest(kk_ctx *ctx, int64_t limit_us, void *stream) {
    return guarded([&] {
        need(ctx && limit_us >= 1 && limit_us <= 2000000, "bad argument");
        use_device(ctx);
        check_cuda(wait_tight_selftest(ctx->serving_err(), (unsigned long long)limit_us * 1000ull,
                                       stream_of(ctx, stream)),
                   "wait self-test launch");
        return KK_OK;
    });
}

}  // extern "C"
