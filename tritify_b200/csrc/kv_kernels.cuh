// The paged KV cache of 8-bit codes on the device: writing rows (rotation, quantisation, scatter into pages), reading
// them back, and what the attention kernels share with them (batch lookup, row quantisation, the weight of a score).
//
// A cached row is one token's key or value of one KV head: int8 codes within +-127 and a scale sigma of 8 significant
// bits, kept as the 16 bits of a bfloat16 (always positive and normal, so its bits order like its value). Pools:
// codes [n_pages][n_kv_heads][page_tokens][head_dim], scales [n_pages][n_kv_heads][page_tokens].
//
// Every rounding below is one IEEE operation written out (__dmul_rn, __ddiv_rn, __fmaf_rn, ...), so that the compiler
// contracts nothing and the CPU path of the tests gives the same integers.
#pragma once

#include <stdint.h>

#include "fixed_point.cuh"

namespace kv {

using kt::Scale;

constexpr int MAX_DIM = 256;

struct Cache {
    int8_t *k, *v;
    uint16_t *ks, *vs;
    long long n_pages;
    int page_shift;  // log2(page_tokens)
    int heads;       // KV heads
    int dim;
};

struct Batch {
    const int* begin;   // [n_seqs + 1]: first row of each sequence's new tokens
    const int* kv_len;  // [n_seqs]: tokens of the sequence, the new ones among them
    const int* pages;   // [n_seqs][max_pages]
    int n_seqs, max_pages;
    long long rows;  // rows the callers' buffers hold
};

struct Rope {
    const int2* table;  // [positions][half] (cosine, sine) times 2^30; null: no rotation
    long long positions;
    int half;
    int interleaved;  // pairs (2i, 2i + 1) instead of (i, i + half)
};

// The context's error words: `word` ends its waits, the one behind it takes what is wrong in a batch (the codes of
// context.cuh).
struct Error {
    int* word;
    int bad_page, bad_length, bad_position;
    __device__ __forceinline__ void raise(int code) const { atomicCAS(word + 1, 0, code); }
};

// Whether a sequence's length fits its row of the page table (which holds 2^24 tokens at most).
__device__ __forceinline__ bool length_fits(const Batch& b, int len, int page_shift) {
    return len >= 0 && len <= b.max_pages << page_shift;
}

// The sequence that row t belongs to, found by a whole warp: begin[] is sampled 32 ways a step, so 64 sequences take
// two rounds of independent loads instead of six dependent ones. -1: t lies before the first or behind the last.
__device__ __forceinline__ int find_seq(const Batch& b, int t) {
    const int lane = threadIdx.x & 31;
    int lo = 0, hi = b.n_seqs;  // the answer is the last i in [lo, hi] with begin[i] <= t
    if (b.begin[0] > t || b.begin[b.n_seqs] <= t) return -1;
    while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32;
        const int i = min(lo + lane * step, hi);
        const unsigned le = __ballot_sync(0xffffffffu, b.begin[i] <= t);
        const int n = max(1, 32 - __clz(le));  // lanes up to the last one that is <= t
        const int nlo = min(lo + (n - 1) * step, hi);
        hi = min(nlo + step, hi);
        lo = nlo;
    }
    return min(lo, b.n_seqs - 1);
}

// Row t's sequence and position; false (with the error word set where the description is wrong) when the row has no
// place in the cache. A position below zero (a length shorter than the new tokens) is no error: the row has no place.
struct Place {
    int seq, pos;
};
__device__ __forceinline__ bool locate(const Batch& b, const Error& err, int t, int page_shift, Place& p) {
    p.seq = find_seq(b, t);
    if (p.seq < 0) return false;
    const int begin = b.begin[p.seq], end = b.begin[p.seq + 1], len = b.kv_len[p.seq];
    // the offsets around t have to ascend and stay within the rows, the length has to fit the page table
    if (t < begin || t >= end || end > b.begin[b.n_seqs] || end > b.rows || !length_fits(b, len, page_shift)) {
        err.raise(err.bad_length);
        return false;
    }
    p.pos = len - (end - t);
    return true;
}

// The pool page of page-table entry i of a sequence; an entry outside the pool raises the error word and page 0 is
// used, so that no access leaves the pool.
__device__ __forceinline__ long long pool_page(const Batch& b, const Cache& c, const Error& err, int seq, int i) {
    const int page = b.pages[(long long)seq * b.max_pages + i];
    if ((unsigned)page >= (unsigned long long)c.n_pages) {
        err.raise(err.bad_page);
        return 0;
    }
    return page;
}

// A scale in float64, its shift held within [-900, 2000] so that the value is finite; `extra_shift` (at most 30) more
// places down. The power of two in halves: the first product is a normal number, so only the second one rounds.
__device__ __forceinline__ double scale_value(longlong2 s, int extra_shift) {
    const int shift = max(-900, min(2000, (int)s.y)) + extra_shift, half = shift >> 1;
    if (s.x <= 0) return 0.0;
    return (double)s.x * __hiloint2double((1023 - half) << 20, 0) * __hiloint2double((1023 - (shift - half)) << 20, 0);
}

// Element e of a row after the rotation. x: the row; cs: its row of the rotation table.
__device__ __forceinline__ int64_t rotated(const int32_t* x, int e, const Rope& r, const int2* cs) {
    const int64_t v = x[e];
    if (e >= 2 * r.half) return v * (1 << 30);
    int j, mate;
    bool first;
    if (r.interleaved) {
        j = e >> 1;
        first = !(e & 1);
        mate = e ^ 1;
    } else {
        first = e < r.half;
        j = first ? e : e - r.half;
        mate = first ? e + r.half : e - r.half;
    }
    const int2 t = cs[j];
    const int64_t o = x[mate];
    return first ? v * t.x - o * t.y : v * t.x + o * t.y;
}

// The rotation table's row for a position, or null without rotation. A position beyond the table raises the error
// word and the last row is used.
__device__ __forceinline__ const int2* rope_row(const Rope& r, const Error& err, int pos) {
    if (!r.table) return nullptr;
    long long p = pos;
    if (p >= r.positions) {
        err.raise(err.bad_position);
        p = r.positions - 1;
    }
    return r.table + p * r.half;
}

// sigma of a row: t held within [2^-64, 2^63] and rounded up to 8 significant bits, as bfloat16 bits. Rounding up to
// 24 bits first changes nothing, since the 8-bit grid lies on the 24-bit one.
__device__ __forceinline__ uint32_t sigma_bits(double t) {
    t = fmin(fmax(t, 0x1p-64), 0x1p63);
    return (__float_as_uint(__double2float_ru(t)) + 0xffffu) >> 16;
}

__device__ __forceinline__ float bf16_value(uint32_t bits) { return __uint_as_float(bits << 16); }

// RN64 of an integer, and the nearest whole number to a double (ties to even, |v| < 2^31): the addition leaves it in the
// low word. The conversions run at a quarter of the FP64 pipe's rate, but put nothing on the pipe of the integer
// operations, which has the most to do here: built of those and FP64 additions instead, the decode of 64 sequences of
// 4096 took 121 us against 117, a window's 8192 tokens 563 against 551.
__device__ __forceinline__ double to_double(int64_t v) { return __ll2double_rn(v); }
__device__ __forceinline__ double to_double(int32_t v) { return __int2double_rn(v); }
__device__ __forceinline__ int to_int(double v) { return __double2loint(__dadd_rn(v, 6755399441055744.0)); }

__device__ __forceinline__ uint32_t uabs(int32_t v) { return v < 0 ? 0u - (uint32_t)v : (uint32_t)v; }

// ── rows of codes: rotation, largest element, quantisation ──
// A warp takes up to B heads of one token (BATCH, fewer where there are no more), which share the rotation's entries, the scale and one division; lane l has
// the elements 4 l .. 4 l + 3 of each 128 (NB of them). Elements are turned into RN64 of their codes at once, which is
// all that what follows needs: RN64 keeps the order, so the largest element's is the largest.
template <int NB>
constexpr int BATCH = NB == 1 ? 4 : 2;
template <int NB, int B = BATCH<NB>>
struct RowBatch {
    double y[B][NB][4];
    double top;  // lane i: of head i
};

// The rotation's entries of elements e .. e + 3, the sine with the sign it takes. by_four: a four and its mates lie in
// aligned fours (else element by element).
__device__ __forceinline__ bool turns_by_four(const Rope& r) { return (r.interleaved ? 2 * r.half : r.half) % 4 == 0; }
__device__ __forceinline__ void fetch_turn(int2 (&c)[4], const Rope& r, const int2* cs, int e) {
    const int j = r.interleaved ? e / 2 : e < r.half ? e : e - r.half;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        c[k] = e < 2 * r.half ? __ldg(cs + j + (r.interleaved ? k >> 1 : k)) : make_int2(1 << 30, 0);
        if (r.interleaved ? !(k & 1) : e < r.half) c[k].y = -c[k].y;
    }
}

// The elements as they lie and those that the rotation mixes them with: asked for before anything is known of the row's
// place, so that both arrive together. x: the first head's row, `heads` of them (the others count as zeros).
template <int NB, int B = BATCH<NB>>
struct RawBatch {
    int4 v[B][NB], o[B][NB];
};
template <int NB, int B = BATCH<NB>>
__device__ __forceinline__ RawBatch<NB, B> fetch_rows(const int32_t* __restrict__ x, int heads, int dim, int vec, const Rope& r) {
    const int lane = threadIdx.x & 31;
    const bool far = r.table && turns_by_four(r) && !r.interleaved;
    RawBatch<NB, B> w;
    auto fetch = [&](auto four) {
#pragma unroll
        for (int i = 0; i < B; ++i)
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const int e = 4 * lane + 128 * b;
                w.v[i][b] = w.o[i][b] = make_int4(0, 0, 0, 0);
                if (i < heads && e < dim) w.v[i][b] = four(x + i * dim + e);
                if (far && i < heads && e < 2 * r.half) w.o[i][b] = four(x + i * dim + (e < r.half ? e + r.half : e - r.half));
            }
    };
    if (vec) fetch([](const int32_t* p) { return __ldg((const int4*)p); });
    else fetch([](const int32_t* p) { return make_int4(__ldg(p), __ldg(p + 1), __ldg(p + 2), __ldg(p + 3)); });
    return w;
}

// cs: the rotation table's row (null: none).
template <int NB, int B>
__device__ __forceinline__ void turn_rows(RowBatch<NB, B>& out, const RawBatch<NB, B>& w, const int32_t* __restrict__ x, int heads,
                                          int dim, const Rope& r, const int2* cs) {
    const int lane = threadIdx.x & 31;
    const bool by_four = cs && turns_by_four(r);
    const auto& v = w.v;
    if (by_four) {
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            int2 c[4];
            fetch_turn(c, r, cs, 4 * lane + 128 * b);
#pragma unroll
            for (int i = 0; i < B; ++i) {  // |.| <= 2^31 (2^30 + 2^30) = 2^62
                const int4 p = v[i][b], q = r.interleaved ? make_int4(p.y, p.x, p.w, p.z) : w.o[i][b];
                out.y[i][b][0] = to_double((int64_t)p.x * c[0].x + (int64_t)q.x * c[0].y);
                out.y[i][b][1] = to_double((int64_t)p.y * c[1].x + (int64_t)q.y * c[1].y);
                out.y[i][b][2] = to_double((int64_t)p.z * c[2].x + (int64_t)q.z * c[2].y);
                out.y[i][b][3] = to_double((int64_t)p.w * c[3].x + (int64_t)q.w * c[3].y);
            }
        }
    } else if (!cs) {
#pragma unroll
        for (int i = 0; i < B; ++i)
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                out.y[i][b][0] = to_double(v[i][b].x);
                out.y[i][b][1] = to_double(v[i][b].y);
                out.y[i][b][2] = to_double(v[i][b].z);
                out.y[i][b][3] = to_double(v[i][b].w);
            }
    } else {
#pragma unroll
        for (int i = 0; i < B; ++i)
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int e = 4 * lane + 128 * b + k;
                    out.y[i][b][k] = i < heads && e < dim ? to_double(rotated(x + i * dim, e, r, cs)) : 0.0;
                }
    }
    if (!cs) {  // the elements are whole 32-bit numbers
#pragma unroll
        for (int i = 0; i < B; ++i) {
            uint32_t most = 0;
#pragma unroll
            for (int b = 0; b < NB; ++b)
                most = max(max(most, max(uabs(v[i][b].x), uabs(v[i][b].y))), max(uabs(v[i][b].z), uabs(v[i][b].w)));
            most = __reduce_max_sync(0xffffffffu, most);
            if (lane == i || i == 0) out.top = (double)most;
        }
        return;
    }
    // the largest: the upper words of |y| first, then the lower words of those that have it
#pragma unroll
    for (int i = 0; i < B; ++i) {
        uint32_t hi = 0, lo = 0;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int k = 0; k < 4; ++k) hi = max(hi, (uint32_t)__double2hiint(out.y[i][b][k]) & 0x7fffffffu);
        hi = __reduce_max_sync(0xffffffffu, hi);
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (((uint32_t)__double2hiint(out.y[i][b][k]) & 0x7fffffffu) == hi)
                    lo = max(lo, (uint32_t)__double2loint(out.y[i][b][k]));
        lo = __reduce_max_sync(0xffffffffu, lo);
        if (lane == i || i == 0) out.top = __hiloint2double((int)hi, (int)lo);
    }
}

// rne(RN64(y m)) of four elements, |y m| < 2^31, as the bytes of a word.
__device__ __forceinline__ uint32_t codes4(const double (&y)[4], double m) {
    int c[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) c[k] = to_int(__dmul_rn(y[k], m));
    return __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
}

// ── writing ──
// A warp per (token, keys or values, up to four KV heads). Four bytes are read and one written per element; bound by the
// instructions all the same (issue slots 68 % busy: the exact products, conversions, the largest, two divisions
// a warp): 16384 tokens of 8 + 8 heads of 128, 168 MB, take 61 us, 703 instructions a warp. Eight blocks an SM although a few registers are
// spilled: with six, and none, writing and reading those tokens took 107 us against 99.
struct AppendArgs {
    Cache c;
    Batch b;
    Rope rope;
    Error err;
    const int32_t *k, *v;
    long long ld_k, ld_v;
    const longlong2* scale[2];  // of K, of V
    int scale_stride;
    int vec;  // rows are 16-byte aligned: 16-byte loads
};

constexpr int ROW_WARPS = 4;

template <int NB, int B>
__global__ void __launch_bounds__(32 * ROW_WARPS, 8) append_kernel(const AppendArgs a, unsigned chunks) {
    kt::pdl_enter();
    const int lane = threadIdx.x & 31, dim = a.c.dim;
    const unsigned u = blockIdx.x * ROW_WARPS + (threadIdx.x >> 5);
    const int t = (int)(u / chunks), c = (int)(u % chunks);
    if (t >= a.b.rows) return;
    const int half = (int)chunks / 2;
    const bool is_v = c >= half;
    const int h0 = (is_v ? c - half : c) * B, heads = min(B, a.c.heads - h0);
    const int32_t* x = (is_v ? a.v + (long long)t * a.ld_v : a.k + (long long)t * a.ld_k) + (long long)h0 * dim;
    Rope rope = a.rope;
    if (is_v) rope.table = nullptr;
    const RawBatch<NB, B> raw = fetch_rows<NB, B>(x, heads, dim, a.vec, rope);
    Place p;
    if (!locate(a.b, a.err, t, a.c.page_shift, p) || p.pos < 0) return;
    const longlong2 sc = a.scale[is_v][(long long)t * a.scale_stride];
    const long long page = pool_page(a.b, a.c, a.err, p.seq, p.pos >> a.c.page_shift);
    const int2* cs = rope_row(rope, a.err, p.pos);
    RowBatch<NB, B> rows;
    turn_rows(rows, raw, x, heads, dim, rope, cs);
    const double s = scale_value(sc, cs ? 30 : 0);
    const double want = __ddiv_rn(__dmul_rn(rows.top, s), 127.0);
    const uint32_t sg = sigma_bits(want);
    const double m = __ddiv_rn(s, (double)bf16_value(sg));
    // sigma >= want, so that |y m| <= 127 (1 + 2^-51) and the codes stay within +-127; but for rows whose scale would
    // be above the largest sigma, 2^63: those are held within +-127 first
    if (__any_sync(0xffffffffu, want > 0x1p63)) {
#pragma unroll
        for (int i = 0; i < B; ++i) {
            const double mi = __shfl_sync(0xffffffffu, m, i), limit = __ddiv_rn(127.0, mi);
            if (__shfl_sync(0xffffffffu, want, i) > 0x1p63)
#pragma unroll
                for (int j = 0; j < 4 * NB; ++j)
                    rows.y[i][j / 4][j % 4] = fmin(fmax(rows.y[i][j / 4][j % 4], -limit), limit);
        }
    }
    const long long row0 = ((page * a.c.heads + h0) << a.c.page_shift) + (p.pos & ((1 << a.c.page_shift) - 1));
    if (lane < heads) (is_v ? a.c.vs : a.c.ks)[row0 + ((long long)lane << a.c.page_shift)] = (uint16_t)sg;
#pragma unroll
    for (int i = 0; i < B; ++i) {
        const double mi = __shfl_sync(0xffffffffu, m, i);
        int8_t* dst = (is_v ? a.c.v : a.c.k) + (row0 + ((long long)i << a.c.page_shift)) * dim;
#pragma unroll
        for (int b = 0; b < NB; ++b)
            if (i < heads && 4 * lane + 128 * b < dim)
                *(uint32_t*)(dst + 4 * lane + 128 * b) = codes4(rows.y[i][b], mi);
    }
}

// ── reading back ──
// A warp per token and eight rows (four of more than 128 elements): all its codes and scales are asked for together.
constexpr int READ_ROWS = 8;

struct ReadArgs {
    Cache c;
    Batch b;
    Error err;
    float *k, *v;
    long long ld_k, ld_v;
    int vec;
};

template <int NB>
__global__ void __launch_bounds__(32 * ROW_WARPS) read_kernel(const ReadArgs a, unsigned chunks) {
    kt::pdl_enter();
    constexpr int B = READ_ROWS / NB;
    const int lane = threadIdx.x & 31, dim = a.c.dim;
    const unsigned u = blockIdx.x * ROW_WARPS + (threadIdx.x >> 5);
    const int t = (int)(u / chunks), r0 = (int)(u % chunks) * B, rows = min(B, 2 * a.c.heads - r0);
    if (t >= a.b.rows) return;
    Place p;
    if (!locate(a.b, a.err, t, a.c.page_shift, p) || p.pos < 0) return;
    const long long page = pool_page(a.b, a.c, a.err, p.seq, p.pos >> a.c.page_shift);
    const int in_page = p.pos & ((1 << a.c.page_shift) - 1);
    const long long row0 = ((page * a.c.heads) << a.c.page_shift) + in_page;
    uint32_t code[B][NB];
    float sigma[B];
#pragma unroll
    for (int i = 0; i < B; ++i) {
        if (i >= rows) break;
        const bool is_v = r0 + i >= a.c.heads;
        const long long row = row0 + ((long long)(r0 + i - (is_v ? a.c.heads : 0)) << a.c.page_shift);
        sigma[i] = bf16_value((is_v ? a.c.vs : a.c.ks)[row]);
#pragma unroll
        for (int b = 0; b < NB; ++b)
            if (4 * lane + 128 * b < dim) code[i][b] = *(const uint32_t*)((is_v ? a.c.v : a.c.k) + row * dim + 4 * lane + 128 * b);
    }
#pragma unroll
    for (int i = 0; i < B; ++i) {
        if (i >= rows) break;
        const bool is_v = r0 + i >= a.c.heads;
        float* dst = (is_v ? a.v + (long long)t * a.ld_v - (long long)a.c.heads * dim : a.k + (long long)t * a.ld_k) + (long long)(r0 + i) * dim;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const int e = 4 * lane + 128 * b;
            if (e >= dim) continue;
            const char4 o = *(const char4*)&code[i][b];
            const float4 f = {__fmul_rn((float)o.x, sigma[i]), __fmul_rn((float)o.y, sigma[i]), __fmul_rn((float)o.z, sigma[i]),
                              __fmul_rn((float)o.w, sigma[i])};  // 7 by 8 significant bits: exact
            if (a.vec) {
                *(float4*)(dst + e) = f;
            } else {
                dst[e] = f.x;
                dst[e + 1] = f.y;
                dst[e + 2] = f.z;
                dst[e + 3] = f.w;
            }
        }
    }
}

// ── attention ──
struct AttendArgs {
    Cache c;
    Batch b;
    Rope rope;
    Error err;
    const int32_t* q;
    long long ld_q;
    const longlong2* scale;
    int scale_stride;
    int vec;    // rows of q are 16-byte aligned
    int group;  // query heads per KV head
    double soft;  // softmax_scale * log2(e)
    int window, sinks;
    int32_t* o;
    long long ld_o;
    int vec_o;  // rows of o are 16-byte aligned
    longlong2* o_scale;  // [rows][KV heads]
};

// The weight of a score: distance d = RN24(X - x), in octaves d * theta rounded to 2^-10 and held at 32 (there the
// weight rounds to zero), split into a whole part n and a remainder r in [-1/2, 1/2], 2^r by a cubic (relative error
// at most 1.1e-4) of amplitude 32512. The fused multiply-add onto 12288 does the rounding to 2^-10 (the spacing of
// floats there), the addition that carries it to 3 * 2^22 the rounding to a whole number, and the low bits of that sum are -n: shifted
// into the exponent field they scale the cubic's value. `lift`: an exponent taken off the result (w * 2^-lift).
constexpr float W_C0 = 32512.0f, W_C1 = 127.0f * 45435.0f / 256.0f, W_C2 = 127.0f * 15874.0f / 256.0f,
                W_C3 = 127.0f * 3605.0f / 256.0f;

__device__ __forceinline__ float weight(float x, float top, float theta) {
    const float d = __fsub_rn(top, x);
    const float f = fmaxf(__fmaf_rn(d, -theta, 12288.0f), 12256.0f);
    const float f0 = __fadd_rn(f, 12570624.0f);  // 3 * 2^22 - n
    const float r = __fsub_rn(f, __fsub_rn(f0, 12570624.0f));
    float e = __fmaf_rn(W_C3, r, W_C2);
    e = __fmaf_rn(e, r, W_C1);
    e = __fmaf_rn(e, r, W_C0);
    return __uint_as_float(__float_as_uint(e) + (__float_as_uint(f0) << 23));
}

// E of a row: the least whole number with 2^E >= the largest visible sigma_v, from that sigma's bits.
__device__ __forceinline__ int scale_exp(uint32_t sigma) { return (int)(sigma >> 7) - 127 + ((sigma & 127) != 0); }
__device__ __forceinline__ float pow2f(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// theta of a row from its largest element, its scale and softmax_scale * log2(e).
__device__ __forceinline__ float row_theta(double top, double s, double soft) {
    return top > 0.0 ? __double2float_rn(fmin(__dmul_rn(__ddiv_rn(__dmul_rn(top, s), 127.0), soft), 0x1p60)) : 0.0f;
}

// Quantised queries wait for the tile kernel where its output will be: the head_dim int32 words of a row and head first
// hold the head_dim codes, then theta; whoever reads them writes the output over them. No other memory is needed. Bound
// by memory at large sizes: 4 bytes read and 1 written per element.
template <int NB>
__global__ void __launch_bounds__(32 * ROW_WARPS, 8) query_kernel(const AttendArgs a, unsigned chunks) {
    kt::pdl_enter();
    constexpr int B = BATCH<NB>;
    const int lane = threadIdx.x & 31, dim = a.c.dim;
    const unsigned u = blockIdx.x * ROW_WARPS + (threadIdx.x >> 5);
    const int t = (int)(u / chunks), h0 = (int)(u % chunks) * B, heads = min(B, a.c.heads * a.group - h0);
    if (t >= a.b.rows) return;
    const int32_t* x = a.q + (long long)t * a.ld_q + (long long)h0 * dim;
    const RawBatch<NB> raw = fetch_rows<NB>(x, heads, dim, a.vec, a.rope);
    Place p;
    if (!locate(a.b, a.err, t, a.c.page_shift, p) || p.pos < 0) return;
    const longlong2 sc = a.scale[(long long)t * a.scale_stride];
    const int2* cs = rope_row(a.rope, a.err, p.pos);
    RowBatch<NB> rows;
    turn_rows(rows, raw, x, heads, dim, a.rope, cs);
    const double m = __ddiv_rn(127.0, fmax(rows.top, 1.0));
    int32_t* out = a.o + (long long)t * a.ld_o + (long long)h0 * dim;
    const float theta = row_theta(rows.top, scale_value(sc, cs ? 30 : 0), a.soft);
    __syncwarp();  // o may be q: every lane has read its elements
    if (lane < heads) out[lane * dim + dim / 4] = __float_as_int(theta);
#pragma unroll
    for (int i = 0; i < B; ++i) {
        const double mi = __shfl_sync(0xffffffffu, m, i);
#pragma unroll
        for (int b = 0; b < NB; ++b)  // |y m| <= 127 (1 + 2^-52): the codes stay within +-127
            if (i < heads && 4 * lane + 128 * b < dim) out[i * dim + lane + 32 * b] = (int)codes4(rows.y[i][b], mi);
    }
}

__device__ __forceinline__ int32_t out_code(int64_t num, double inv) {
    return to_int(__dmul_rn(to_double(num), inv));
}

}  // namespace kv
