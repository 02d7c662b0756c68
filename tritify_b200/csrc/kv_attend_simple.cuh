// Attention over the paged cache, the plain kernel: a block per (row, KV head, eight query heads), the scores of 128
// keys at a time by dp4a, once for the maximum and once for the weights, and the values summed in 64 bits.
#pragma once

#include "kv_kernels.cuh"

namespace kv {

constexpr int SIMPLE_HEADS = 8;

__global__ void __launch_bounds__(128) attend_simple_kernel(const AttendArgs a) {
    kt::pdl_enter();
    __shared__ __align__(16) int8_t q8[SIMPLE_HEADS][MAX_DIM];
    __shared__ float theta[SIMPLE_HEADS];
    __shared__ float top[SIMPLE_HEADS];
    __shared__ float red[4][SIMPLE_HEADS];
    __shared__ unsigned red_s[4];
    __shared__ int p8[SIMPLE_HEADS][128];
    __shared__ long long rows8[128];
    __shared__ long long total[SIMPLE_HEADS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tid = threadIdx.x;
    const int t = blockIdx.x, h = blockIdx.y, g0 = blockIdx.z * SIMPLE_HEADS;
    const int ng = min(SIMPLE_HEADS, a.group - g0), dim = a.c.dim, words = dim / 4;
    if (t < a.b.begin[0] || t >= a.b.begin[a.b.n_seqs]) return;  // behind the last sequence: left as it was
    Place p;
    bool ok = locate(a.b, a.err, t, a.c.page_shift, p);
    int32_t* out = a.o + (long long)t * a.ld_o + (long long)(h * a.group + g0) * dim;
    if (!ok || p.pos < 0) {  // nothing is visible
        for (int i = tid; i < ng * dim; i += 128) out[i] = 0;
        if (tid == 0 && g0 == 0) a.o_scale[(long long)t * a.c.heads + h] = make_longlong2(0, 0);
        return;
    }
    const int2* cs = rope_row(a.rope, a.err, p.pos);
    const double s = scale_value(a.scale[(long long)t * a.scale_stride], cs ? 30 : 0);
    for (int i = warp; i < ng; i += 4) {
        RowBatch<2> rows;
        const int32_t* x = a.q + (long long)t * a.ld_q + (long long)(h * a.group + g0 + i) * dim;
        turn_rows<2>(rows, fetch_rows<2>(x, 1, dim, a.vec, a.rope), x, 1, dim, a.rope, cs);
        const double m = __shfl_sync(0xffffffffu, __ddiv_rn(127.0, fmax(rows.top, 1.0)), 0);
        for (int b = 0; b < 2; ++b)
            if (4 * lane + 128 * b < dim) *(uint32_t*)(q8[i] + 4 * lane + 128 * b) = codes4<false>(rows.y[0][b], m);
        if (lane == 0) theta[i] = row_theta(rows.top, s, a.soft);
    }
    for (int i = tid; i < SIMPLE_HEADS; i += 128) total[i] = 0;
    __syncthreads();
    const int lo = a.window ? max(0, p.pos + 1 - a.window) : 0;  // [0, min(sinks, lo)) and [lo, pos]
    const int n_sink = min(a.sinks, lo), n = n_sink + p.pos + 1 - lo;
    float mx[SIMPLE_HEADS];
    unsigned ms = 0;
    for (int i = 0; i < SIMPLE_HEADS; ++i) mx[i] = -INFINITY;
    long long acc[SIMPLE_HEADS][2];
    for (int i = 0; i < SIMPLE_HEADS; ++i) acc[i][0] = acc[i][1] = 0;
    float lift = 1.0f;
    int e_row = 0;
    for (int pass = 0; pass < 2; ++pass) {
        for (int j0 = 0; j0 < n; j0 += 128) {
            const int jj = j0 + tid;
            const bool live = jj < n;
            float x[SIMPLE_HEADS];
            unsigned sv = 0;
            if (live) {
                const int j = jj < n_sink ? jj : lo + jj - n_sink;
                const long long page = pool_page(a.b, a.c, a.err, p.seq, j >> a.c.page_shift);
                const long long row = ((page * a.c.heads + h) << a.c.page_shift) + (j & ((1 << a.c.page_shift) - 1));
                const int* kr = (const int*)(a.c.k + row * dim);
                int d[SIMPLE_HEADS];
                for (int i = 0; i < SIMPLE_HEADS; ++i) d[i] = 0;
                for (int w = 0; w < words; ++w) {
                    const int kw = kr[w];
                    for (int i = 0; i < SIMPLE_HEADS; ++i) d[i] = __dp4a(kw, ((const int*)q8[i])[w], d[i]);
                }
                const float kf = bf16_value(a.c.ks[row]);
                for (int i = 0; i < SIMPLE_HEADS; ++i) x[i] = __fmul_rn((float)d[i], kf);
                sv = a.c.vs[row];
                rows8[tid] = row;
            }
            if (pass == 0) {
                if (live) {
                    for (int i = 0; i < SIMPLE_HEADS; ++i) mx[i] = fmaxf(mx[i], x[i]);
                    ms = max(ms, sv);
                }
                continue;
            }
            for (int i = 0; i < ng; ++i) {
                int w8 = 0, w = 0;
                if (live) {
                    const float wt = weight(x[i], top[i], theta[i]);
                    w = __float2int_rn(wt);
                    w8 = __float_as_int(__fmaf_rn(wt, __fmul_rn(bf16_value(sv), lift), 12582912.0f)) - 0x4B400000;
                }
                p8[i][tid] = w8;
                w = __reduce_add_sync(0xffffffffu, w);
                if (lane == 0) atomicAdd((unsigned long long*)&total[i], (unsigned long long)w);
            }
            __syncthreads();
            for (int c = 0; c < 2; ++c) {
                const int d = tid + 128 * c;
                if (d < dim) {
                    int sum[SIMPLE_HEADS];
                    for (int i = 0; i < SIMPLE_HEADS; ++i) sum[i] = 0;
                    const int m = min(128, n - j0);
                    for (int j = 0; j < m; ++j) {
                        const int vv = a.c.v[rows8[j] * dim + d];
                        for (int i = 0; i < SIMPLE_HEADS; ++i) sum[i] += vv * p8[i][j];
                    }
                    for (int i = 0; i < SIMPLE_HEADS; ++i) acc[i][c] += sum[i];
                }
            }
            __syncthreads();
        }
        if (pass == 0) {
            for (int i = 0; i < SIMPLE_HEADS; ++i) {
                float m = mx[i];
                for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
                if (lane == 0) red[warp][i] = m;
            }
            ms = __reduce_max_sync(0xffffffffu, ms);
            if (lane == 0) red_s[warp] = ms;
            __syncthreads();
            if (tid < SIMPLE_HEADS)
                top[tid] = fmaxf(fmaxf(red[0][tid], red[1][tid]), fmaxf(red[2][tid], red[3][tid]));
            e_row = scale_exp(max(max(red_s[0], red_s[1]), max(red_s[2], red_s[3])));
            lift = pow2f(-e_row);
            __syncthreads();
        }
    }
    for (int i = 0; i < ng; ++i) {
        const double inv = __ddiv_rn(2097152.0, (double)total[i]);
        for (int c = 0; c < 2; ++c) {
            const int d = tid + 128 * c;
            if (d < dim) out[(long long)i * dim + d] = out_code(acc[i][c], inv);
        }
    }
    if (tid == 0 && g0 == 0)
        a.o_scale[(long long)t * a.c.heads + h] = make_longlong2(1, (long long)(uint32_t)(21 - e_row));
}

}  // namespace kv
