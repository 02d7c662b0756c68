// The paged KV cache's entry points of include/ktmoe.h: writing new keys and values, reading them back, and attention
// over the cache. All on device buffers, ordered on the caller's stream, nothing allocated and no workspace kept, so
// calls on several streams and captured graphs share nothing but the caller's own buffers.

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "context.cuh"
#include "kv_host.h"
#include "kv_attend_few.cuh"
#include "kv_attend_tile.cuh"
#include "kv_kernels.cuh"

namespace {

bool aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

kv::Error error_of(ktmoe_ctx* ctx) {
    return kv::Error{ctx->d_err, ktc::ERR_BAD_PAGE, ktc::ERR_BAD_LENGTH, ktc::ERR_BAD_POSITION};
}

// The cache and the batch of a call; KTMOE_OK, or the status of what is wrong with them.
int check_cache(ktmoe_ctx* ctx, const ktmoe_kv_cache* c, const ktmoe_kv_batch* b, kv::Cache* kc, kv::Batch* kb) {
    if (!c->k || !c->v || !c->k_scale || !c->v_scale) return fail(ctx, KTMOE_ERR_ARG, "a pool of the cache is null");
    if (!aligned(c->k, 16) || !aligned(c->v, 16) || !aligned(c->k_scale, 16) || !aligned(c->v_scale, 16))
        return fail(ctx, KTMOE_ERR_ARG, "the cache's pools need 16-byte alignment");
    if (c->head_dim < 16 || c->head_dim > kv::MAX_DIM || c->head_dim % 16 != 0)
        return fail(ctx, KTMOE_ERR_UNSUPPORTED, "head_dim must be a multiple of 16 from 16 to 256");
    int shift = 4;
    while (shift < 7 && (1 << shift) != c->page_tokens) ++shift;
    if ((1 << shift) != c->page_tokens) return fail(ctx, KTMOE_ERR_UNSUPPORTED, "page_tokens must be 16, 32, 64 or 128");
    if (c->n_kv_heads < 1 || c->n_kv_heads > 1024 || c->n_pages < 1 || c->n_pages > INT32_MAX)
        return fail(ctx, KTMOE_ERR_ARG, "the cache needs 1 to 1024 KV heads and 1 to 2^31 - 1 pages");
    if (b->n_seqs < 0 || b->n_seqs > 1 << 30 || b->rows < 0 || b->rows > (int64_t)1 << 30 || b->max_pages < 0 ||
        (int64_t)b->max_pages * c->page_tokens > (int64_t)1 << 24)
        return fail(ctx, KTMOE_ERR_ARG, "a batch holds at most 2^30 sequences, 2^30 rows and a page table at most 2^24 tokens a sequence, none of them negative");
    if (b->n_seqs > 0 && (!b->q_begin || !b->kv_len || (b->max_pages > 0 && !b->page_table)))
        return fail(ctx, KTMOE_ERR_ARG, "the batch's offsets, lengths or page table are null");
    *kc = kv::Cache{c->k, c->v, c->k_scale, c->v_scale, c->n_pages, shift, c->n_kv_heads, c->head_dim};
    *kb = kv::Batch{b->q_begin, b->kv_len, b->page_table, b->n_seqs, b->max_pages, b->rows};
    return KTMOE_OK;
}

int check_rope(ktmoe_ctx* ctx, const ktmoe_rope* r, int head_dim, kv::Rope* out) {
    *out = kv::Rope{nullptr, 0, 0, 0};
    if (!r) return KTMOE_OK;
    if (!r->table || !aligned(r->table, 8) || r->positions < 1)
        return fail(ctx, KTMOE_ERR_ARG, "the rotation table is null, not 8-byte aligned or empty");
    if (r->rot_dim < 2 || r->rot_dim % 2 != 0 || r->rot_dim > head_dim)
        return fail(ctx, KTMOE_ERR_ARG, "rot_dim must be even, from 2 to head_dim");
    *out = kv::Rope{(const int2*)r->table, r->positions, r->rot_dim / 2, r->interleaved ? 1 : 0};
    return KTMOE_OK;
}

int check_scale(ktmoe_ctx* ctx, const ktmoe_scale* s, int32_t stride) {
    if (!aligned(s, 16) || (stride != 0 && stride != 1))
        return fail(ctx, KTMOE_ERR_ARG, "scales need 16-byte alignment and a stride of 0 (one scale) or 1 (one a row)");
    return KTMOE_OK;
}

// The TMA map of a pool: boxes of one page of one KV head, 128 bytes of its rows. Bytes behind head_dim read as zero.
int make_pool_map(ktmoe_ctx* ctx, CUtensorMap* map, const int8_t* pool, const kv::Cache& c) {
    ktc::EncodeTiledFn enc = ktc::encode_fn();
    if (!enc) return fail(ctx, KTMOE_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable");
    const cuuint64_t ps = (cuuint64_t)1 << c.page_shift;
    cuuint64_t gdim[4] = {(cuuint64_t)c.dim, ps, (cuuint64_t)c.heads, (cuuint64_t)c.n_pages};
    cuuint64_t gstride[3] = {(cuuint64_t)c.dim, ps * c.dim, ps * c.dim * c.heads};
    cuuint32_t box[4] = {128, (cuuint32_t)ps, 1, 1};
    cuuint32_t estride[4] = {1, 1, 1, 1};
    CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<int8_t*>(pool), gdim, gstride, box, estride,
                     CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(ctx, KTMOE_ERR_CUDA, "cuTensorMapEncodeTiled failed (" + std::to_string((int)r) + ")");
    return KTMOE_OK;
}

// Blocks of ROW_WARPS warps, a warp per row and chunk of its heads (counted in 32 bits on the device).
int row_blocks(ktmoe_ctx* ctx, int64_t rows, int chunks, unsigned* blocks) {
    if (rows * chunks > INT32_MAX) return fail(ctx, KTMOE_ERR_UNSUPPORTED, "too many rows for one launch");
    *blocks = (unsigned)((rows * chunks + kv::ROW_WARPS - 1) / kv::ROW_WARPS);
    return KTMOE_OK;
}

template <int NB, int B = kv::BATCH<NB>>
int launch_append(ktmoe_ctx* ctx, cudaStream_t st, const kv::AppendArgs& a) {
    // few heads leave a batch half empty, and its instructions are what bounds the kernel: half the batch (writing and
    // reading 131072 tokens of one head of 128 took 261 us with four, 169 with one; 65536 of two heads 152 and 122)
    if constexpr (B > 1)
        if (a.c.heads <= B / 2) return launch_append<NB, B / 2>(ctx, st, a);
    const int chunks = 2 * ((a.c.heads + B - 1) / B);  // of keys and of values
    unsigned blocks;
    if (int r = row_blocks(ctx, a.b.rows, chunks, &blocks)) return r;
    KLAUNCH(st, blocks, 32 * kv::ROW_WARPS, 0, (kv::append_kernel<NB, B>), a, (unsigned)chunks);
    return KTMOE_OK;
}

template <int NB>
int launch_read(ktmoe_ctx* ctx, cudaStream_t st, const kv::ReadArgs& a) {
    constexpr int B = kv::READ_ROWS / NB;
    const int chunks = (2 * a.c.heads + B - 1) / B;
    unsigned blocks;
    if (int r = row_blocks(ctx, a.b.rows, chunks, &blocks)) return r;
    KLAUNCH(st, blocks, 32 * kv::ROW_WARPS, 0, (kv::read_kernel<NB>), a, (unsigned)chunks);
    return KTMOE_OK;
}

template <int NK>
int launch_tile(ktmoe_ctx* ctx, cudaStream_t st, const kv::AttendArgs& a) {
    static bool attr_set[64] = {};
    if (!attr_set[ctx->device & 63]) {
        CK(cudaFuncSetAttribute(kv::attend_tile_kernel<NK>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                kv::TileCfg<NK>::BYTES));
        attr_set[ctx->device & 63] = true;
    }
    const int64_t slots = a.b.rows * a.group / kv::TILE_ROWS + a.b.n_seqs;
    if (slots * a.c.heads > INT32_MAX) return fail(ctx, KTMOE_ERR_UNSUPPORTED, "too many query rows for one launch");
    CUtensorMap mk, mv;
    if (int r = make_pool_map(ctx, &mk, a.c.k, a.c)) return r;
    if (int r = make_pool_map(ctx, &mv, a.c.v, a.c)) return r;
    const int chunks = (a.c.heads * a.group + kv::BATCH<NK> - 1) / kv::BATCH<NK>;
    unsigned blocks;
    if (int r = row_blocks(ctx, a.b.rows, chunks, &blocks)) return r;
    KLAUNCH(st, blocks, 32 * kv::ROW_WARPS, 0, (kv::query_kernel<NK>), a, (unsigned)chunks);
    KLAUNCH(st, (unsigned)(slots * a.c.heads), kv::TILE_THREADS, kv::TileCfg<NK>::BYTES, (kv::attend_tile_kernel<NK>), mk,
            mv, a, (long long)slots);
    return KTMOE_OK;
}

// Tiles of keys that a row may see, as far as the host knows: the lengths are on the device.
int64_t key_tiles(const kv::AttendArgs& a) {
    const int64_t tiles = (((int64_t)a.b.max_pages << a.c.page_shift) + kv::TILE_KEYS - 1) / kv::TILE_KEYS;
    return a.window ? std::min(tiles, ((int64_t)a.window + a.sinks) / kv::TILE_KEYS + 2) : tiles;
}

// Blocks of `block` rows, if all sequences had as many rows.
int64_t even_blocks(const kv::AttendArgs& a, int64_t block) {
    const int64_t rows = (a.b.rows * a.group + a.b.n_seqs - 1) / a.b.n_seqs;
    return a.b.n_seqs * ((rows + block - 1) / block) * a.c.heads;
}

// Blocks of a cluster: twice as many while they are less than 4/3 of what the GPU holds at once. Eights are harder to
// place (a GPC's SMs do not divide by them; with one block an SM, 16 clusters of eight already take two rounds): only
// where they fill half of the GPU at most, or where the keys are long. Measured (us, from a flushed L2), clusters of 1, 2,
// 4, 8 at 4 query heads to one of 8 KV heads of 128: 1 sequence of 1000 keys 18, 16, 14, 12, of 8000 76, 43, 29, 20; 4 of
// 2000 29, 20, 18, 20; 8 of 16384 164, 84, 61, 74; 16 of 4096 45, 39, 51, 72; 64 of 1024 47, 68, 108, 209, of 4096 113, 129,
// 168, 262. Over 160 sizes drawn at random (1 to 128 sequences of one token, 100 to 65536 keys, heads of 64 to 256) the
// choice of cluster and kernel takes 7 % more than the best of each, in 41 of them more than 10 %.
int few_cluster(const ktmoe_ctx* ctx, const kv::AttendArgs& a, int per_sm) {
    const int64_t jobs = even_blocks(a, kv::FEW_ROWS), tiles = key_tiles(a), at_once = (int64_t)per_sm * ctx->num_sms;
    int c = 1;
    while (c < 4 && tiles > c && 3 * jobs * c < 2 * at_once) c *= 2;
    const bool few_eights = 2 * 8 * jobs <= at_once;
    if (c == 4 && tiles > 4 && (few_eights || (per_sm == 2 && tiles >= 64 && 3 * jobs * 4 < 2 * at_once))) c = 8;
    return c;
}

// Which kernel. Where the GPU is full, a block of 128 rows is the better one (three times for many rows), but it walks
// all keys alone, while sixteens of rows spread over more SMs and split the keys in clusters. Both times are rounds of
// blocks by tiles of keys and a start; an SM passes a tile by 16 rows in 3/7 of the time it takes by 128, and starts
// count as 8 and 6 tiles. Measured (us, from a flushed L2) at 8 KV heads of 128, one query head each, and 8192 keys: 1
// sequence of 64 rows 39 against 156, of 256 80 against 156, of 512 137 against 156, of 1024 258 against 160; 16 sequences
// of 32 rows 154 against 166, of 64 279 against 168; at 512 keys 1 sequence of 256 rows 25 against 29. Over 160 sizes drawn at
// random (2 to 1024 tokens a sequence) the choice of kernel and cluster takes 3 % more than the best of each, in 12 of them
// more than 10 %. The host knows neither lengths nor rows: a page table wider than the sequences, or one chunk among
// single tokens, counts as if every sequence were as long and had as many rows, which changes the time alone.
bool few_rows(const ktmoe_ctx* ctx, const kv::AttendArgs& a, int per_sm) {
    auto rounds = [](int64_t blocks, int64_t at_once) { return (blocks + at_once - 1) / at_once; };
    const int64_t c = few_cluster(ctx, a, per_sm), tiles = key_tiles(a);
    return 3 * per_sm * rounds(even_blocks(a, kv::FEW_ROWS) * c, (int64_t)per_sm * ctx->num_sms) * (8 * c + tiles) <=
           7 * c * rounds(even_blocks(a, kv::TILE_ROWS), ctx->num_sms) * (6 + tiles);
}

template <int NK, int PER_SM>
int launch_few(ktmoe_ctx* ctx, cudaStream_t st, const kv::AttendArgs& a) {
    using C = kv::FewCfg<NK, PER_SM>;
    const auto kernel = kv::attend_few_kernel<NK, PER_SM>;
    static bool attr_set[64] = {};
    if (!attr_set[ctx->device & 63]) {
        CK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::BYTES));
        attr_set[ctx->device & 63] = true;
    }
    // the sixteens of all rows, and one more a sequence, by the KV heads
    const int64_t jobs = (a.b.rows * a.group / kv::FEW_ROWS + a.b.n_seqs) * a.c.heads;
    const int c = few_cluster(ctx, a, PER_SM);
    if (jobs * c > INT32_MAX) return fail(ctx, KTMOE_ERR_UNSUPPORTED, "too many query rows for one launch");
    CUtensorMap mk, mv;
    if (int r = make_pool_map(ctx, &mk, a.c.k, a.c)) return r;
    if (int r = make_pool_map(ctx, &mv, a.c.v, a.c)) return r;
    KLAUNCHC(st, (unsigned)(jobs * c), C::THREADS, C::BYTES, (unsigned)c, kernel, mk, mv, a);
    return KTMOE_OK;
}

}  // namespace

extern "C" {

int ktmoe_rope_table(double theta, int32_t rot_dim, int64_t positions, int32_t* table) {
    if (!table || rot_dim < 2 || rot_dim % 2 != 0 || positions < 1 || !(theta > 0.0) || !std::isfinite(theta))
        return KTMOE_ERR_ARG;
    const int half = rot_dim / 2;
    for (int i = 0; i < half; ++i) {
        const double f = std::pow(theta, -(double)i / half);
        for (int64_t p = 0; p < positions; ++p) {
            table[2 * (p * half + i)] = (int32_t)std::nearbyint(std::cos(p * f) * 1073741824.0);
            table[2 * (p * half + i) + 1] = (int32_t)std::nearbyint(std::sin(p * f) * 1073741824.0);
        }
    }
    return KTMOE_OK;
}

int ktmoe_kv_append_dev(ktmoe_ctx* ctx, const ktmoe_kv_cache* cache, const ktmoe_kv_batch* batch, const int32_t* k,
                        int64_t ld_k, const int32_t* v, int64_t ld_v, const ktmoe_scale* k_scale,
                        const ktmoe_scale* v_scale, int32_t scale_stride, const ktmoe_rope* rope, void* stream) {
    if (!ctx || !cache || !batch) return KTMOE_ERR_ARG;
    std::lock_guard<std::mutex> lk(ctx->mu);
    return kv_append(ctx, cache, batch, k, ld_k, v, ld_v, k_scale, v_scale, scale_stride, rope, stream);
}

}  // extern "C"

int kv_append(ktmoe_ctx* ctx, const ktmoe_kv_cache* cache, const ktmoe_kv_batch* batch, const int32_t* k, int64_t ld_k,
              const int32_t* v, int64_t ld_v, const ktmoe_scale* k_scale, const ktmoe_scale* v_scale,
              int32_t scale_stride, const ktmoe_rope* rope, void* stream) {
    if (!v_scale) v_scale = k_scale;
    kv::AppendArgs a{};
    if (int r = check_cache(ctx, cache, batch, &a.c, &a.b)) return r;
    if (int r = check_rope(ctx, rope, a.c.dim, &a.rope)) return r;
    if (int r = check_scale(ctx, k_scale, scale_stride)) return r;
    if (int r = check_scale(ctx, v_scale, scale_stride)) return r;
    const int64_t width = (int64_t)a.c.heads * a.c.dim;
    if (ld_k < width || ld_v < width) return fail(ctx, KTMOE_ERR_ARG, "a row stride is below n_kv_heads * head_dim");
    if (batch->n_seqs == 0 || batch->rows == 0) return KTMOE_OK;
    if (!k || !v || !k_scale || !aligned(k, 4) || !aligned(v, 4))
        return fail(ctx, KTMOE_ERR_ARG, "keys, values or scales are null or not aligned");
    if (int r = set_device(ctx)) return r;
    a.err = error_of(ctx);
    a.k = k;
    a.v = v;
    a.ld_k = ld_k;
    a.ld_v = ld_v;
    a.scale[0] = (const longlong2*)k_scale;
    a.scale[1] = (const longlong2*)v_scale;
    a.scale_stride = scale_stride;
    a.vec = aligned(k, 16) && aligned(v, 16) && ld_k % 4 == 0 && ld_v % 4 == 0;
    cudaStream_t st = stream ? (cudaStream_t)stream : ctx->stream;
    return a.c.dim <= 128 ? launch_append<1>(ctx, st, a) : launch_append<2>(ctx, st, a);
}

extern "C" {

int ktmoe_kv_read_dev(ktmoe_ctx* ctx, const ktmoe_kv_cache* cache, const ktmoe_kv_batch* batch, float* k, int64_t ld_k,
                      float* v, int64_t ld_v, void* stream) {
    if (!ctx || !cache || !batch) return KTMOE_ERR_ARG;
    std::lock_guard<std::mutex> lk(ctx->mu);
    kv::ReadArgs a{};
    if (int r = check_cache(ctx, cache, batch, &a.c, &a.b)) return r;
    const int64_t width = (int64_t)a.c.heads * a.c.dim;
    if (ld_k < width || ld_v < width) return fail(ctx, KTMOE_ERR_ARG, "a row stride is below n_kv_heads * head_dim");
    if (batch->n_seqs == 0 || batch->rows == 0) return KTMOE_OK;
    if (!k || !v || !aligned(k, 4) || !aligned(v, 4)) return fail(ctx, KTMOE_ERR_ARG, "an output is null or not aligned");
    if (int r = set_device(ctx)) return r;
    a.err = error_of(ctx);
    a.k = k;
    a.v = v;
    a.ld_k = ld_k;
    a.ld_v = ld_v;
    a.vec = aligned(k, 16) && aligned(v, 16) && ld_k % 4 == 0 && ld_v % 4 == 0;
    cudaStream_t st = stream ? (cudaStream_t)stream : ctx->stream;
    return a.c.dim <= 128 ? launch_read<1>(ctx, st, a) : launch_read<2>(ctx, st, a);
}

int ktmoe_attention_dev(ktmoe_ctx* ctx, const ktmoe_kv_cache* cache, const ktmoe_kv_batch* batch, const int32_t* q,
                        int64_t ld_q, const ktmoe_scale* scale, int32_t scale_stride, const ktmoe_rope* rope,
                        int32_t n_heads, double softmax_scale, int32_t window, int32_t sinks, int32_t* o, int64_t ld_o,
                        ktmoe_scale* o_scale, void* stream) {
    if (!ctx || !cache || !batch) return KTMOE_ERR_ARG;
    std::lock_guard<std::mutex> lk(ctx->mu);
    return kv_attention(ctx, cache, batch, q, ld_q, scale, scale_stride, rope, n_heads, softmax_scale, window, sinks, o, ld_o,
                        o_scale, stream);
}

}  // extern "C"

int kv_attention(ktmoe_ctx* ctx, const ktmoe_kv_cache* cache, const ktmoe_kv_batch* batch, const int32_t* q, int64_t ld_q,
                 const ktmoe_scale* scale, int32_t scale_stride, const ktmoe_rope* rope, int32_t n_heads,
                 double softmax_scale, int32_t window, int32_t sinks, int32_t* o, int64_t ld_o, ktmoe_scale* o_scale,
                 void* stream) {
    kv::AttendArgs a{};
    if (int r = check_cache(ctx, cache, batch, &a.c, &a.b)) return r;
    if (int r = check_rope(ctx, rope, a.c.dim, &a.rope)) return r;
    if (int r = check_scale(ctx, scale, scale_stride)) return r;
    if (n_heads < 1 || n_heads % a.c.heads != 0)
        return fail(ctx, KTMOE_ERR_ARG, "n_heads must be a positive multiple of n_kv_heads");
    if (!(softmax_scale > 0.0) || !std::isfinite(softmax_scale) || window < 0 || sinks < 0)
        return fail(ctx, KTMOE_ERR_ARG, "softmax_scale must be positive and finite, window and sinks not negative");
    const int64_t width = (int64_t)n_heads * a.c.dim;
    if (ld_q < width || ld_o < width) return fail(ctx, KTMOE_ERR_ARG, "a row stride is below n_heads * head_dim");
    if (batch->rows * (n_heads / a.c.heads) > INT32_MAX) return fail(ctx, KTMOE_ERR_UNSUPPORTED, "too many query rows for one launch");
    if (batch->n_seqs == 0 || batch->rows == 0) return KTMOE_OK;
    if (!q || !o || !o_scale || !scale || !aligned(q, 4) || !aligned(o, 4) || !aligned(o_scale, 16))
        return fail(ctx, KTMOE_ERR_ARG, "queries, scales or outputs are null or not aligned");
    if (o == q && ld_o != ld_q && batch->rows > 1)
        return fail(ctx, KTMOE_ERR_ARG, "o may be q at the same row stride only");
    if (int r = set_device(ctx)) return r;
    a.err = error_of(ctx);
    a.q = q;
    a.ld_q = ld_q;
    a.scale = (const longlong2*)scale;
    a.scale_stride = scale_stride;
    a.vec = aligned(q, 16) && ld_q % 4 == 0;
    a.group = n_heads / a.c.heads;
    a.soft = softmax_scale * 1.4426950408889634;
    a.window = window;
    a.sinks = sinks;
    a.o = o;
    a.ld_o = ld_o;
    a.o_scale = (longlong2*)o_scale;
    a.vec_o = aligned(o, 16) && ld_o % 4 == 0;
    cudaStream_t st = stream ? (cudaStream_t)stream : ctx->stream;
    if (a.c.dim <= 128) return few_rows(ctx, a, 2) ? launch_few<1, 2>(ctx, st, a) : launch_tile<1>(ctx, st, a);
    return few_rows(ctx, a, 1) ? launch_few<2, 1>(ctx, st, a) : launch_tile<2>(ctx, st, a);
}
