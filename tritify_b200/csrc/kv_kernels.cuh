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

// The error word and what to raise in it (the codes of context.cuh).
struct Error {
    int* word;
    int bad_page, bad_length, bad_position;
    __device__ __forceinline__ void raise(int code) const { atomicCAS(word, 0, code); }
};

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
    if (t < begin || t >= end || end > b.begin[b.n_seqs] || end > b.rows || len < 0 || ((len + (1 << page_shift) - 1) >> page_shift) > b.max_pages) {
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

__device__ __forceinline__ uint64_t uabs(int64_t v) { return v < 0 ? (uint64_t)(-v) : (uint64_t)v; }

__device__ __forceinline__ uint64_t warp_umax(uint64_t v) {
    const uint32_t hi = (uint32_t)(v >> 32);
    const uint32_t mh = __reduce_max_sync(0xffffffffu, hi);
    const uint32_t ml = __reduce_max_sync(0xffffffffu, hi == mh ? (uint32_t)v : 0u);
    return (uint64_t)mh << 32 | ml;
}

// A scale in float64, its shift held within [-900, 2000] so that the value is finite; `extra_shift` more places down.
__device__ __forceinline__ double scale_value(longlong2 s, int extra_shift) {
    const int shift = max(-900, min(2000, (int)s.y)) + extra_shift;
    return s.x <= 0 ? 0.0 : ldexp((double)s.x, -shift);
}

// A row's codes after the rotation, four per lane and step: element e = 4 * lane + 128 * step.
// x: the row's int32 codes (all of head_dim readable).
__device__ __forceinline__ int64_t rotated(const int32_t* x, int e, const Rope& r, const int2* cs) {
    const int64_t v = x[e];
    if (!cs) return v;
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
    return first ? v * t.x - o * t.y : v * t.x + o * t.y;  // |.| <= 2^31 (2^30 + 2^30) = 2^62
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

// rne(RN64(y m)) held within +-127.
__device__ __forceinline__ int code8(int64_t y, double m) {
    return max(-127, min(127, __double2int_rn(__dmul_rn((double)y, m))));
}

// ── writing ──
// One block per row of the batch, one warp per (key or value, KV head) row of head_dim codes in turn. Bound by memory:
// 4 bytes read and 1 written per element.
struct AppendArgs {
    Cache c;
    Batch b;
    Rope rope;
    Error err;
    const int32_t *k, *v;
    long long ld_k, ld_v;
    const longlong2* scale;
    int scale_stride;
    int vec;  // rows are 16-byte aligned: 16-byte loads
};

constexpr int APPEND_WARPS = 8;

__device__ __forceinline__ void stage_row(int32_t* dst, const int32_t* __restrict__ src, int dim, int vec) {
    const int lane = threadIdx.x & 31;
    if (vec) {
        for (int e = 4 * lane; e < dim; e += 128) *(int4*)(dst + e) = __ldg((const int4*)(src + e));
    } else {
        for (int e = lane; e < dim; e += 32) dst[e] = src[e];
    }
    __syncwarp();
}

__global__ void __launch_bounds__(32 * APPEND_WARPS) append_kernel(const AppendArgs a) {
    kt::pdl_enter();
    __shared__ __align__(16) int32_t stage[APPEND_WARPS][MAX_DIM];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int t = blockIdx.x;
    Place p;
    if (!locate(a.b, a.err, t, a.c.page_shift, p) || p.pos < 0) return;
    const long long page = pool_page(a.b, a.c, a.err, p.seq, p.pos >> a.c.page_shift);
    const int in_page = p.pos & ((1 << a.c.page_shift) - 1);
    const longlong2 sc = a.scale[(long long)t * a.scale_stride];
    const int2* cs = rope_row(a.rope, a.err, p.pos);
    const int dim = a.c.dim;
    for (int r = warp; r < 2 * a.c.heads; r += APPEND_WARPS) {
        const bool is_v = r >= a.c.heads;
        const int h = is_v ? r - a.c.heads : r;
        const int32_t* src = (is_v ? a.v + (long long)t * a.ld_v : a.k + (long long)t * a.ld_k) + (long long)h * dim;
        stage_row(stage[warp], src, dim, a.vec);
        const int2* rot = is_v ? nullptr : cs;
        int64_t y[8];
        uint64_t top = 0;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int e = 4 * lane + 128 * i;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                y[4 * i + q] = e < dim ? rotated(stage[warp], e + q, a.rope, rot) : 0;
                top = max(top, uabs(y[4 * i + q]));
            }
        }
        top = warp_umax(top);
        const double s = scale_value(sc, rot ? 30 : 0);
        const uint32_t sg = sigma_bits(__ddiv_rn(__dmul_rn((double)(int64_t)top, s), 127.0));
        const double m = __ddiv_rn(s, (double)bf16_value(sg));
        const long long row = ((page * a.c.heads + h) << a.c.page_shift) + in_page;
        int8_t* dst = (is_v ? a.c.v : a.c.k) + row * dim;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int e = 4 * lane + 128 * i;
            if (e < dim) {
                char4 o;
                o.x = (signed char)code8(y[4 * i], m);
                o.y = (signed char)code8(y[4 * i + 1], m);
                o.z = (signed char)code8(y[4 * i + 2], m);
                o.w = (signed char)code8(y[4 * i + 3], m);
                *(char4*)(dst + e) = o;
            }
        }
        if (lane == 0) (is_v ? a.c.vs : a.c.ks)[row] = (uint16_t)sg;
        __syncwarp();
    }
}

// ── reading back ──
struct ReadArgs {
    Cache c;
    Batch b;
    Error err;
    float *k, *v;
    long long ld_k, ld_v;
    int vec;
};

__global__ void __launch_bounds__(32 * APPEND_WARPS) read_kernel(const ReadArgs a) {
    kt::pdl_enter();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int t = blockIdx.x;
    Place p;
    if (!locate(a.b, a.err, t, a.c.page_shift, p) || p.pos < 0) return;
    const long long page = pool_page(a.b, a.c, a.err, p.seq, p.pos >> a.c.page_shift);
    const int in_page = p.pos & ((1 << a.c.page_shift) - 1);
    const int dim = a.c.dim;
    for (int r = warp; r < 2 * a.c.heads; r += APPEND_WARPS) {
        const bool is_v = r >= a.c.heads;
        const int h = is_v ? r - a.c.heads : r;
        const long long row = ((page * a.c.heads + h) << a.c.page_shift) + in_page;
        const int8_t* src = (is_v ? a.c.v : a.c.k) + row * dim;
        const float sg = bf16_value((is_v ? a.c.vs : a.c.ks)[row]);
        float* dst = (is_v ? a.v + (long long)t * a.ld_v : a.k + (long long)t * a.ld_k) + (long long)h * dim;
        for (int e = 4 * lane; e < dim; e += 128) {
            const char4 o = *(const char4*)(src + e);
            const float4 f = {__fmul_rn((float)o.x, sg), __fmul_rn((float)o.y, sg), __fmul_rn((float)o.z, sg),
                              __fmul_rn((float)o.w, sg)};  // 7 by 8 significant bits: exact
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

// A query row's codes and theta, by a whole warp. stage: head_dim int32 of shared memory. dst: the row's int8 codes; with
// SW128, row r of a K-major operand in 128-byte blocks of 16384 bytes with the 128-byte swizzle.
template <bool SW128>
__device__ __forceinline__ float quantise_query(int8_t* dst, int32_t* stage, const int32_t* src, int dim, int vec,
                                                const Rope& rope, const int2* cs, double s, double soft, int r = 0) {
    const int lane = threadIdx.x & 31;
    stage_row(stage, src, dim, vec);
    int64_t y[8];
    uint64_t top = 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int e = 4 * lane + 128 * i;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            y[4 * i + q] = e < dim ? rotated(stage, e + q, rope, cs) : 0;
            top = max(top, uabs(y[4 * i + q]));
        }
    }
    top = warp_umax(top);
    const double td = (double)(int64_t)top;
    const double m = __ddiv_rn(127.0, fmax(td, 1.0));
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int e = 4 * lane + 128 * i;
        if (e < dim) {
            char4 o;
            o.x = (signed char)code8(y[4 * i], m);
            o.y = (signed char)code8(y[4 * i + 1], m);
            o.z = (signed char)code8(y[4 * i + 2], m);
            o.w = (signed char)code8(y[4 * i + 3], m);
            *(char4*)(dst + (SW128 ? i * 16384 + (((lane >> 2) ^ (r & 7)) << 4) + 4 * (lane & 3) : e)) = o;
        }
    }
    __syncwarp();
    if (top == 0) return 0.0f;
    return __double2float_rn(fmin(__dmul_rn(__ddiv_rn(__dmul_rn(td, s), 127.0), soft), 0x1p60));
}

// RN64 of a 64-bit integer and the nearest whole number to a double (ties to even, |v| < 2^31) on the FP64 pipe: the
// conversion instructions run at a quarter of its rate. 2^52 + 2^31 + hi and 2^52 + lo are doubles whose low words are
// the integer's halves.
__device__ __forceinline__ double to_double(int64_t v) {
    const double hi = __dsub_rn(__hiloint2double(0x43300000, (int)(v >> 32) ^ (int)0x80000000), 4503601774854144.0);
    const double lo = __dsub_rn(__hiloint2double(0x43300000, (int)v), 4503599627370496.0);
    return __fma_rn(hi, 4294967296.0, lo);
}
__device__ __forceinline__ double to_double(int32_t v) {
    return __dsub_rn(__hiloint2double(0x43300000, v ^ (int)0x80000000), 4503601774854144.0);
}
__device__ __forceinline__ int to_int(double v) { return __double2loint(__dadd_rn(v, 6755399441055744.0)); }

// Where a query row stands: its position, its row of the caller's buffers and its query head. pos < 0: no row.
struct QueryRow {
    int pos;
    long long row;
    int head;
};

// Four elements e .. e + 3 of a query row after the rotation. x: the row; cs: its row of the rotation table.
__device__ __forceinline__ void rotated4(int64_t (&y)[4], const AttendArgs& a, const int32_t* x, const int2* cs, int e) {
    int4 v;
    if (a.vec) {
        v = __ldg((const int4*)(x + e));
    } else {
        v = make_int4(x[e], x[e + 1], x[e + 2], x[e + 3]);
    }
    const int half = a.rope.half;
    if (!a.rope.table) {
        y[0] = v.x, y[1] = v.y, y[2] = v.z, y[3] = v.w;
    } else if (e >= 2 * half) {
        y[0] = (int64_t)v.x << 30, y[1] = (int64_t)v.y << 30, y[2] = (int64_t)v.z << 30, y[3] = (int64_t)v.w << 30;
    } else if (a.rope.interleaved && e + 4 <= 2 * half) {
        const int2 c0 = __ldg(cs + e / 2), c1 = __ldg(cs + e / 2 + 1);
        y[0] = (int64_t)v.x * c0.x - (int64_t)v.y * c0.y;
        y[1] = (int64_t)v.y * c0.x + (int64_t)v.x * c0.y;
        y[2] = (int64_t)v.z * c1.x - (int64_t)v.w * c1.y;
        y[3] = (int64_t)v.w * c1.x + (int64_t)v.z * c1.y;
    } else if (!a.rope.interleaved && half % 4 == 0 && a.vec) {
        const bool first = e < half;
        const int4 o = __ldg((const int4*)(x + (first ? e + half : e - half)));
        const int2* c = cs + (first ? e : e - half);
        const int2 c0 = __ldg(c), c1 = __ldg(c + 1), c2 = __ldg(c + 2), c3 = __ldg(c + 3);
        const int sg = first ? -1 : 1;
        y[0] = (int64_t)v.x * c0.x + (int64_t)o.x * (sg * c0.y);
        y[1] = (int64_t)v.y * c1.x + (int64_t)o.y * (sg * c1.y);
        y[2] = (int64_t)v.z * c2.x + (int64_t)o.z * (sg * c2.y);
        y[3] = (int64_t)v.w * c3.x + (int64_t)o.w * (sg * c3.y);
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) y[k] = rotated(x, e + k, a.rope, cs);
    }
}

// N query rows by one warp: codes of row r, r0 <= r < r0 + N, into row r of a K-major operand in 128-byte blocks with the
// 128-byte swizzle (16384 bytes a block), theta into theta[r]. NB: blocks of a row. The rows are rotated twice, for
// their largest element and for their codes (from L1 then), so that one division serves all rows and the loads of
// many rows overlap: what this costs is latency, not work.
template <int N, int NB, class RowOf>
__device__ __forceinline__ void quantise_rows(const AttendArgs& a, RowOf row_of, int r0, int8_t* dst, float* theta) {
    const int lane = threadIdx.x & 31, dim = a.c.dim;
    uint64_t mine = 0;  // lane i: the largest element of row r0 + i
#pragma unroll 4
    for (int i = 0; i < N; ++i) {
        const QueryRow at = row_of(r0 + i);
        uint64_t top = 0;
        if (at.pos >= 0) {
            const int32_t* x = a.q + at.row * a.ld_q + (long long)at.head * dim;
            const int2* cs = rope_row(a.rope, a.err, at.pos);
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const int e = 4 * lane + 128 * b;
                if (e >= dim) continue;
                int64_t y[4];
                rotated4(y, a, x, cs, e);
                top = max(max(top, max(uabs(y[0]), uabs(y[1]))), max(uabs(y[2]), uabs(y[3])));
            }
        }
        top = warp_umax(top);
        if (lane == i) mine = top;
    }
    const double td = to_double((int64_t)mine);
    const double m = __ddiv_rn(127.0, fmax(td, 1.0));
    if (lane < N) {
        const QueryRow me = row_of(r0 + lane);
        if (me.pos >= 0) {
            const double s = scale_value(a.scale[me.row * a.scale_stride], a.rope.table ? 30 : 0);
            theta[r0 + lane] =
                mine ? __double2float_rn(fmin(__dmul_rn(__ddiv_rn(__dmul_rn(td, s), 127.0), a.soft), 0x1p60)) : 0.0f;
        }
    }
#pragma unroll 4
    for (int i = 0; i < N; ++i) {
        const QueryRow at = row_of(r0 + i);
        const double mi = __shfl_sync(0xffffffffu, m, i);
        if (at.pos < 0) continue;
        const int32_t* x = a.q + at.row * a.ld_q + (long long)at.head * dim;
        const int2* cs = rope_row(a.rope, a.err, at.pos);
        const int r = r0 + i;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const int e = 4 * lane + 128 * b;
            if (e >= dim) continue;
            int64_t y[4];
            rotated4(y, a, x, cs, e);
            // |y m| <= 127 (1 + 2^-52): the codes stay within +-127
            char4 o;
            o.x = (signed char)to_int(__dmul_rn(to_double(y[0]), mi));
            o.y = (signed char)to_int(__dmul_rn(to_double(y[1]), mi));
            o.z = (signed char)to_int(__dmul_rn(to_double(y[2]), mi));
            o.w = (signed char)to_int(__dmul_rn(to_double(y[3]), mi));
            *(char4*)(dst + b * 16384 + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + 4 * (lane & 3)) = o;
        }
    }
}

__device__ __forceinline__ int32_t out_code(int64_t num, double inv) {
    return to_int(__dmul_rn(to_double(num), inv));
}

}  // namespace kv
