// Attention over the paged cache for few query rows of a sequence (decode, short chunks): a cluster of blocks takes up to
// 16 rows (token, query head) of one sequence and KV head, and each block an even share of the keys they see. Bound by
// memory: every key and value byte once; everything else has to pass under that stream.
//
// Operands are swapped against the tile kernel, so that few rows still fill the tensor cores and K and V go from their
// pages to the products by TMA alone: S^T = K Q^T (128 keys by 16 rows) and O^T = V^T P^T (128 columns by 16 rows, both
// digits of the weights in one product of 32 columns). A thread has one key of a tile.
//
// The row maxima must be known before the first weight is rounded, so there are two phases; K is read once all the same,
// because the scores wait in TMEM, 4, 8, 12 or 16 columns a tile for as many rows (with 16 for any number the decode of 64
// sequences of 4096 by 4 rows took 111 us, not 96). Only tiles beyond what a block has room for are formed again. While the
// cluster exchanges its maxima, V is already on its way. Sums over the keys are integers, so the shares of a cluster
// add up to the same bits in any order: each block adds its own into the shared memory of the block that writes them out.
//
// A block's start, exchange and end are latency (10 us of a block's 26 at 12 tiles), so two blocks share an SM, one's waits
// under the other's stream, although each then has room for the scores of 12 to 48 tiles only (26 to 104 alone): four
// sequences of 65536 keys by 12 rows took 155 us, against 264 with one block an SM.
//
// Roles: softmax warps, in one or two groups of four that take the tiles in turn; then one warp each for TMA, the
// products and the keys' scales.
#pragma once

#include "kv_attend_tile.cuh"

namespace kv {

constexpr int FEW_ROWS = 16;

// NK: 128-byte blocks of a key row; PER_SM: blocks that share an SM.
template <int NK, int PER_SM>
struct FewCfg {
    static constexpr int SLOT = TILE_KEYS * 128;
    static constexpr int SLOTS = 8 / PER_SM;
    static constexpr int SOFT = 8;  // softmax warps
    static constexpr int THREADS = 32 * (SOFT + 3);
    static constexpr int COLS = 512 / PER_SM;  // of TMEM
    static constexpr int SCALES = 4;
    static constexpr int SUMS = COLS - 32 * NK;        // O^T of each 128 columns: 16 hi, 16 lo
    static constexpr int KEEP = SUMS - 32;             // columns for scores that stay: 192 (NK 1, PER_SM 2), 416 (NK 2, PER_SM 1)
    static constexpr int FRESH = KEEP;                 // two score buffers of 16 columns, written by the products
    static constexpr int RING = 0;
    static constexpr int Q = RING + SLOTS * SLOT;               // [NK][16 rows][128]
    static constexpr int P = Q + NK * 16 * 128;                 // [2][16 hi, 16 lo][128 keys]
    static constexpr int RED = P + 2 * 32 * 128;                // int64 [16 rows][NK * 128]
    static constexpr int KEY_SCALES = RED + 16 * NK * 128 * 8;  // [SCALES][sigma_k, sigma_v][128]
    static constexpr int ROWS = KEY_SCALES + SCALES * 2 * TILE_KEYS * 4;
    // per row: theta; position; max and largest sigma of each warp and of each block of the cluster; total of the cluster;
    // the row's (max, -theta, 2^-E, 2^E); 2^21 / L
    static constexpr int BARS = ROWS + FEW_ROWS * (4 + 4 + 64 + 64 + 8 + 16 + 8);
    static constexpr int BYTES = 1024 + BARS + 512;
    static_assert(PER_SM * (BYTES + 1024) <= 233472, "shared memory of an SM");
};

__device__ __forceinline__ uint32_t cluster_ctarank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_nctarank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}
// Every thread of every block of the cluster meets; what was written to shared memory before the arrival is seen after
// the wait.
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t peer_addr(const void* local, uint32_t rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(local)), "r"(rank));
    return a;
}
__device__ __forceinline__ void peer_store(uint32_t a, uint32_t v) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(a), "r"(v) : "memory");
}
// One arrival at a barrier of another block of the cluster; what this thread wrote before is seen after the wait.
__device__ __forceinline__ void peer_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// wait() for arrivals from other blocks.
__device__ __forceinline__ bool wait_cluster(uint64_t* bar, uint32_t parity, int* err, int code) {
    const uint64_t t0 = dg::globaltimer();
    for (uint32_t it = 1;; ++it) {
        uint32_t ok;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok)
            : "r"(smem_u32(bar)), "r"(parity)
            : "memory");
        if (ok) return true;
        if ((it & 255u) == 0) {
            if (*(volatile int*)err != 0) return false;
            if (dg::globaltimer() - t0 > 2000000000ull) {
                atomicCAS(err, 0, code);
                return false;
            }
        }
    }
}
__device__ __forceinline__ void peer_add(uint32_t a, uint64_t v) {
    asm volatile("red.relaxed.cluster.shared::cluster.add.u64 [%0], %1;" ::"r"(a), "l"(v) : "memory");
}
// The first 4, 8, 12 or 16 of a thread's scores to that many columns of TMEM.
__device__ __forceinline__ void tmem_put(uint32_t taddr, int width, const int32_t (&r)[16]) {
    if (width == 12)
        asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1,%2,%3,%4};" ::"r"(taddr + 8), "r"(r[8]), "r"(r[9]),
                     "r"(r[10]), "r"(r[11]));
    if (width == 4)
        asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1,%2,%3,%4};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]),
                     "r"(r[3]));
    else if (width <= 12)
        asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]),
                     "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]));
    else
        tmem_st16(taddr, r);
}
// A float as an integer of the same order, and back.
__device__ __forceinline__ int ordered(int b) { return b ^ ((b >> 31) & 0x7fffffff); }

template <int NK, int PER_SM>
__global__ void __launch_bounds__(FewCfg<NK, PER_SM>::THREADS, PER_SM)
    attend_few_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                      const AttendArgs a) {
    kt::pdl_enter();
    using C = FewCfg<NK, PER_SM>;
    constexpr int GROUPS = C::SOFT / 4;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* sm = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    float4* s_row = (float4*)(sm + C::ROWS);                  // max, -theta, 2^-E, 2^E
    unsigned long long* s_total = (unsigned long long*)(s_row + FEW_ROWS);
    double* s_inv = (double*)(s_total + FEW_ROWS);
    int* s_tops = (int*)(s_inv + FEW_ROWS);                   // [8 warps][16]
    uint32_t* s_sigs = (uint32_t*)(s_tops + 8 * FEW_ROWS);    // [8 warps][16]
    uint32_t* s_top = s_sigs + 8 * FEW_ROWS;                  // [8 ranks][16], written by the ranks
    uint32_t* s_sig = s_top + 8 * FEW_ROWS;                  // [8 ranks][16]
    float* s_theta = (float*)(s_sig + 8 * FEW_ROWS);
    int* s_pos = (int*)(s_theta + FEW_ROWS);
    uint64_t* full = (uint64_t*)(sm + C::BARS);  // [SLOTS]
    // [SLOTS] the products of a block are done: its slot is free, the scores of its tile are there (K), the digits of its
    // tile have been read (V). One arrival for all: each costs the issuing warp 130 clocks.
    uint64_t* empty = full + C::SLOTS;
    uint64_t* s_free = empty + C::SLOTS;         // [2] scores have been read
    uint64_t* p_full = s_free + 2;               // [2]
    uint64_t* k_full = p_full + 2;               // [SCALES]
    uint64_t* k_free = k_full + C::SCALES;       // [SCALES]
    uint64_t* q_full = k_free + C::SCALES;
    uint64_t* o_full = q_full + 1;
    uint64_t* o_free = o_full + 1;
    uint64_t* x_full = o_free + 1;  // every block's maxima have arrived
    uint64_t* done = x_full + 1;
    uint32_t* tmem_slot = (uint32_t*)(done + 1);
    int* s_job = (int*)(tmem_slot + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = a.group, dim = a.c.dim;
    const uint32_t rank = cluster_ctarank(), ranks = cluster_nctarank();
    const unsigned job = blockIdx.x / ranks;
    const int head = (int)(job % (unsigned)a.c.heads);
    const long long slot = job / (unsigned)a.c.heads;
    // Sequence b's groups of 16 rows stand at slots begin_b g / 16 + b and on; slots without rows leave, whole clusters.
    if (warp == 0) {
        auto first_slot = [&](int b) { return (long long)a.b.begin[b] * g / FEW_ROWS + b; };
        const int b = warp_search(a.b.n_seqs, slot, first_slot);
        const int begin = a.b.begin[b], end = a.b.begin[b + 1], len = a.b.kv_len[b];
        const long long row0 = (slot - first_slot(b)) * FEW_ROWS;
        bool live = row0 >= 0 && row0 < (long long)(end - begin) * g;
        if (begin < 0 || begin > end || end > a.b.begin[a.b.n_seqs] || end > a.b.rows ||
            !length_fits(a.b, len, a.c.page_shift)) {
            if (lane == 0) a.err.raise(a.err.bad_length);
            live = false;
        }
        if (lane == 0) {
            s_job[0] = live ? b : -1;
            s_job[1] = begin;
            s_job[2] = end - begin;
            s_job[3] = len;
            s_job[4] = (int)row0;
        }
    }
    if (threadIdx.x == 32) {
        for (int i = 0; i < C::SLOTS; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&s_free[i], 4);
            mbar_init(&p_full[i], 4);
        }
        for (int i = 0; i < C::SCALES; ++i) {
            mbar_init(&k_full[i], 1);
            mbar_init(&k_free[i], 4);
        }
        mbar_init(q_full, C::SOFT);
        mbar_init(o_full, 1);
        mbar_init(o_free, 4);
        mbar_init(x_full, FEW_ROWS * ranks);
        mbar_init(done, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    const int seq = s_job[0];
    if (seq < 0) return;
    const int begin = s_job[1], n_new = s_job[2], len = s_job[3], row0 = s_job[4];
    const int n_rows = min(FEW_ROWS, n_new * g - row0);
    const int p0 = len - n_new + row0 / g, p1 = len - n_new + (row0 + n_rows - 1) / g;
    const KeyTiles all_tiles(p0, p1, a.window, a.sinks);
    // this block's share of the tiles
    const int i_first = (int)((long long)all_tiles.n * rank / ranks), i_last = (int)((long long)all_tiles.n * (rank + 1) / ranks);
    const int n = i_last - i_first;
    // the scores of the first `keep` tiles stay, `width` columns a tile
    const int width = (n_rows + 3) & ~3, keep = C::KEEP / width;
    auto tile_at = [&](int i) { return all_tiles.at(i_first + i); };
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "n"(C::COLS));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
        asm volatile("tcgen05.fence::before_thread_sync;");
    }
    for (int i = threadIdx.x; i < FEW_ROWS * NK * 128; i += C::THREADS) ((long long*)(sm + C::RED))[i] = 0;
    if (threadIdx.x < FEW_ROWS) s_total[threadIdx.x] = 0;
    // the blocks of the cluster are there, their barriers stand and their sums are zero
    __syncwarp();
    cluster_arrive();
    cluster_wait();
    asm volatile("tcgen05.fence::after_thread_sync;");
    const uint32_t tmem = *tmem_slot;
    const int ps = 1 << a.c.page_shift;
    const int* pages = a.b.pages + (long long)seq * a.b.max_pages;
    int* err = a.err.word;
    // Blocks of K and V in the order in which they are loaded and used: all K, then V of tile i, preceded by K of tile
    // i + 1 where its scores did not stay. The number of the last block of K (first, again) and of V of tile i:
    auto k_block = [&](int i) { return (i + 1) * NK - 1; };
    auto k_again = [&](int i) { return (n + i - 1 + (i - keep) + 1) * NK - 1; };
    auto v_block = [&](int i) { return (n + i + max(0, min(i + 2, n) - keep) + 1) * NK - 1; };
    const bool soft = warp < C::SOFT;

    if (warp == C::SOFT) {
        // K of every tile; then V of tile after tile, and K of tile i + 1 ahead of V of tile i where its scores did not
        // stay. A lane holds one page of a tile; page numbers are read two tiles ahead.
        const int per_tile = TILE_KEYS >> a.c.page_shift, last_page = p1 >> a.c.page_shift;
        uint32_t q = 0;
        int s = 0;
        uint32_t phase = 1;
        bool alive = true;
        auto page_of = [&](int i) -> int {
            const int at = tile_at(min(i, n - 1)) * per_tile + lane;
            return lane < per_tile && at <= last_page ? __ldg(pages + at) : 0;
        };
        // Of K that is read again as much as fits should be in L2 by then: what is read for the last time, and by no other
        // block (one group of rows a head), leaves it first.
        const bool alone = n_new * g <= FEW_ROWS;
        const uint64_t policy = once_policy();
        auto load = [&](const CUtensorMap* map, int i, int page, bool last) {
            const int np = min(per_tile, last_page - tile_at(i) * per_tile + 1);
            if ((unsigned)page >= (unsigned long long)a.c.n_pages) {
                a.err.raise(a.err.bad_page);
                page = 0;
            }
#pragma unroll
            for (int x = 0; x < NK; ++x) {
                bool ok = alive;
                if (ok && lane == 0) {
                    ok = wait(&empty[s], phase, err, dg::ERR_TIMEOUT_EMPTY);
                    if (ok) mbar_arrive_expect_tx(&full[s], (uint32_t)(np * ps * 128));
                }
                alive = __shfl_sync(0xffffffffu, (int)ok, 0);
                if (!alive) return;
                if (lane < np) {
                    const uint32_t dst = smem_u32(sm + C::RING + s * C::SLOT + lane * ps * 128);
                    if (last && alone) tma_load_4d_once(dst, map, x * 128, 0, head, page, &full[s], policy);
                    else tma_load_4d(dst, map, x * 128, 0, head, page, &full[s]);
                }
                ++q;
                if (++s == C::SLOTS) s = 0, phase ^= 1;
            }
        };
        for (int ph = 0; alive && n > 0 && ph < 2; ++ph) {
            int pa = page_of(0), pb = page_of(1);
            for (int i = 0; alive && i < n; ++i) {
                const int pc = page_of(i + 2);
                if (ph == 0) {
                    load(&map_k, i, pa, i < keep);
                } else {
                    if (i + 1 >= keep && i + 1 < n) load(&map_k, i + 1, pb, true);
                    if (alive) load(&map_v, i, pa, true);
                }
                pa = pb;
                pb = pc;
            }
        }
        if (lane == 0)  // copies still in flight land before the block leaves
            for (uint32_t j = q > (uint32_t)C::SLOTS ? q - C::SLOTS : 0; j < q; ++j)
                dg::mbar_wait_drain(&full[j % C::SLOTS], (j / C::SLOTS) & 1u, err, dg::ERR_TIMEOUT_FULL);
        __syncwarp();
    } else if (warp == C::SOFT + 1) {
        if (n > 0) {
            const bool issue = lane == 0;
            const int ksteps = (dim + 31) / 32;
            const uint32_t id_s = idesc_i8(FEW_ROWS, 0), id_o = idesc_i8(2 * FEW_ROWS, 1u << 15);
            const uint32_t qd = desc_k(smem_u32(sm + C::Q)), kd = desc_k(smem_u32(sm + C::RING)),
                           pd = desc_k(smem_u32(sm + C::P)), vd = desc_mn(smem_u32(sm + C::RING));
            int s = 0;
            uint32_t phase = 0, number = 0, oc = 0;
            bool ok = warp_wait(q_full, 0, err, dg::ERR_TIMEOUT_FULL);
            auto next = [&]() {
                if (++s == C::SLOTS) s = 0, phase ^= 1;
            };
            auto scores = [&]() {  // number `number` over both phases: two ahead of their readers
                const uint32_t b = number & 1, d = tmem + C::FRESH + 16 * b;
                ok = ok && warp_wait(&s_free[b], ((number >> 1) & 1u) ^ 1u, err, dg::ERR_TIMEOUT_ACCUM);
                ++number;
#pragma unroll
                for (int x = 0; x < NK; ++x) {
                    ok = ok && warp_wait(&full[s], phase, err, dg::ERR_TIMEOUT_FULL);
                    if (!ok) return;
                    asm volatile("tcgen05.fence::after_thread_sync;");
                    const uint32_t kx = kd + s * (C::SLOT >> 4), qx = qd + x * (16 * 128 >> 4);
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk)
                        if (4 * x + kk < ksteps) umma(issue, d, kx + 2 * kk, qx + 2 * kk, id_s, x + kk > 0);
                    umma_arrive(issue, &empty[s]);
                    next();
                }
            };
            for (int i = 0; ok && i < n; ++i) scores();
            for (int i = 0; ok && i < n; ++i) {
                if (i + 1 >= keep && i + 1 < n) scores();
                ok = ok && warp_wait(&p_full[i & 1], (i >> 1) & 1u, err, dg::ERR_TIMEOUT_ACCUM);
#pragma unroll
                for (int x = 0; x < NK; ++x) {
                    ok = ok && warp_wait(&full[s], phase, err, dg::ERR_TIMEOUT_FULL);
                    if (!ok) break;
                    asm volatile("tcgen05.fence::after_thread_sync;");
                    const uint32_t vx = vd + s * (C::SLOT >> 4), px = pd + (i & 1) * (32 * 128 >> 4);
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk)
                        umma(issue, tmem + C::SUMS + 32 * x, vx + kk * (32 * 128 >> 4), px + 2 * kk, id_o, i % FLUSH_TILES + kk > 0);
                    umma_arrive(issue, &empty[s]);
                    next();
                }
                if (!ok) break;
                if (i + 1 == n || (i + 1) % FLUSH_TILES == 0) {
                    umma_arrive(issue, o_full);
                    if (i + 1 < n) {  // the sums are taken out and begin anew
                        ok = warp_wait(o_free, oc & 1u, err, dg::ERR_TIMEOUT_ACCUM);
                        asm volatile("tcgen05.fence::after_thread_sync;");
                    }
                    ++oc;
                }
            }
            umma_arrive(issue, done);
            if (issue) dg::mbar_wait_drain(done, 0u, err, dg::ERR_TIMEOUT_ACCUM);
        }
        __syncwarp();
    } else if (warp == C::SOFT + 2) {
        // The scales of each tile's keys, four keys a lane, for both phases: read four tiles ahead, their pages eight.
        const int total = 2 * n;
        auto key_of = [&](int u) { return tile_at(u >= n ? u - n : u) * TILE_KEYS + 4 * lane; };
        auto page_of = [&](int u) -> int {
            const int j = u < total ? key_of(u) : p1 + 1;
            return j <= p1 ? __ldg(pages + (j >> a.c.page_shift)) : 0;
        };
        auto scales_of = [&](int u, int page) -> uint4 {  // four bfloat16 of K, four of V
            uint4 r = {0, 0, 0, 0};
            const int j = u < total ? key_of(u) : p1 + 1;
            if (j <= p1) {
                if ((unsigned)page >= (unsigned long long)a.c.n_pages) {
                    a.err.raise(a.err.bad_page);
                    page = 0;
                }
                const long long row = (((long long)page * a.c.heads + head) << a.c.page_shift) + (j & (ps - 1));
                const uint2 k = __ldg((const uint2*)(a.c.ks + row)), v = __ldg((const uint2*)(a.c.vs + row));
                r = make_uint4(k.x, k.y, v.x, v.y);
            }
            return r;
        };
        if (total > 0) {
            int pg[4];
            uint4 val[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) pg[j] = page_of(j);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                val[j] = scales_of(j, pg[j]);
                pg[j] = page_of(j + 4);
            }
            bool alive = true;
            for (int u0 = 0; alive && u0 < total; u0 += 4) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {  // stage j: C::SCALES is 4
                    const int u = u0 + j;
                    if (u >= total || !alive) break;
                    alive = wait(&k_free[j], ((u >> 2) & 1u) ^ 1u, err, dg::ERR_TIMEOUT_EMPTY);
                    alive = __all_sync(0xffffffffu, alive);
                    if (!alive) break;
                    uint32_t* f = (uint32_t*)(sm + C::KEY_SCALES) + j * 2 * TILE_KEYS;
                    uint4 w = val[j];
                    w.z = held_scales(w.z);
                    w.w = held_scales(w.w);
                    const uint32_t hi16 = 0xffff0000u;
                    *(uint4*)(f + 4 * lane) = make_uint4(w.x << 16, w.x & hi16, w.y << 16, w.y & hi16);
                    *(uint4*)(f + TILE_KEYS + 4 * lane) = make_uint4(w.z << 16, w.z & hi16, w.w << 16, w.w & hi16);
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&k_full[j]);
                    val[j] = scales_of(u + 4, pg[j]);
                    pg[j] = page_of(u + 8);
                }
            }
        }
        __syncwarp();
    }

    // ── the softmax warps; the others go on to where the cluster meets ──
    const int key = 32 * (warp & 3) + lane, grp = (warp >> 2) % GROUPS;  // of a tile; a group takes every GROUPSth
    const uint32_t lane_addr = tmem + ((uint32_t)(32 * (warp & 3)) << 16);
    bool ok = true;
    int32_t s16[16];
    float kf = 0.0f;
    uint32_t vf = 0;
    // the products of block q of K and V are done
    auto block_done = [&](int q) {
        return wait(&empty[q % C::SLOTS], (uint32_t)(q / C::SLOTS) & 1u, err, dg::ERR_TIMEOUT_ACCUM);
    };
    // the scores of tile i and its keys' scales, for the u'th time
    auto next_scores = [&](int i, int u) {
        const bool fresh = u < n || i >= keep;
        const uint32_t b = (uint32_t)(u < n ? i : n + i - keep) & 1;
        if (fresh) ok = block_done(u < n ? k_block(i) : k_again(i));
        ok = ok && wait(&k_full[u & 3], (u >> 2) & 1u, err, dg::ERR_TIMEOUT_FULL);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) return;
        asm volatile("tcgen05.fence::after_thread_sync;");
        const uint32_t kept = lane_addr + width * i;
        dg::tmem_ld16(fresh ? lane_addr + C::FRESH + 16 * b : kept, s16);  // what lies behind the rows is not looked at
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
        if (u < n && i < keep) tmem_put(kept, width, s16);
        asm volatile("tcgen05.fence::before_thread_sync;");
        const uint32_t* f = (const uint32_t*)(sm + C::KEY_SCALES) + (u & 3) * 2 * TILE_KEYS;
        kf = __uint_as_float(f[key]);
        vf = f[TILE_KEYS + key];
        __syncwarp();
        if (lane == 0) {
            mbar_arrive(&k_free[u & 3]);
            if (fresh) mbar_arrive(&s_free[b]);
        }
    };
    // bit r: row r sees this thread's key of the tile
    auto seen_rows = [&](int j0) -> uint32_t {
        if (j0 + TILE_KEYS - 1 <= p0 && (!a.window || j0 > p1 - a.window || j0 + TILE_KEYS <= a.sinks)) return 0xffffu;
        const int j = j0 + key;
        uint32_t m = 0;
        for (int r = 0; r < n_rows; ++r) {
            const int pos = s_pos[r];
            m |= (uint32_t)(j <= pos && (!a.window || j > pos - a.window || j < a.sinks)) << r;
        }
        return m;
    };
    if (soft) {
        // the queries, up to B rows of one token at a time: two a warp, since the
        // block waits for them (with four, one sequence of 1000 keys took 16.4 us, not 15.4)
        if (threadIdx.x < FEW_ROWS) s_pos[threadIdx.x] = threadIdx.x < n_rows ? len - n_new + (row0 + (int)threadIdx.x) / g : -1;
        constexpr int B = 2;
#pragma unroll 1
        for (int rb = B * warp; rb < n_rows; rb += C::SOFT * B) {
            int count = 0;
#pragma unroll 1
            for (int r = rb; r < min(rb + B, n_rows); r += count) {
                const int t = (row0 + r) / g, hq = (row0 + r) % g, pos = len - n_new + t;
                count = min(min(rb + B, n_rows) - r, g - hq);
                if (pos < 0) continue;
                const int32_t* x = a.q + ((long long)begin + t) * a.ld_q + (long long)(head * g + hq) * dim;
                const RawBatch<NK, B> raw = fetch_rows<NK, B>(x, count, dim, a.vec, a.rope);
                const longlong2 sc = a.scale[((long long)begin + t) * a.scale_stride];
                const int2* cs = rope_row(a.rope, a.err, pos);
                RowBatch<NK, B> rows;
                turn_rows(rows, raw, x, count, dim, a.rope, cs);
                const double m = __ddiv_rn(127.0, fmax(rows.top, 1.0));
                if (lane < count) s_theta[r + lane] = row_theta(rows.top, scale_value(sc, cs ? 30 : 0), a.soft);
#pragma unroll
                for (int i = 0; i < B; ++i) {
                    const double mi = __shfl_sync(0xffffffffu, m, i);
                    const int ri = r + i;
#pragma unroll
                    for (int b = 0; b < NK; ++b)
                        if (i < count && 4 * lane + 128 * b < dim)
                            *(uint32_t*)(sm + C::Q + b * 2048 + ri * 128 + (((lane >> 2) ^ (ri & 7)) << 4) + 4 * (lane & 3)) =
                                codes4(rows.y[i][b], mi);
                }
            }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(q_full);
        asm volatile("bar.sync 1, %0;" ::"n"(32 * C::SOFT) : "memory");  // s_pos, s_theta
        // ── phase 0: the maxima ──
        float top[FEW_ROWS];
        uint32_t sig[FEW_ROWS];
#pragma unroll
        for (int r = 0; r < FEW_ROWS; ++r) top[r] = -INFINITY, sig[r] = 0;
        for (int i = grp; i < n; i += GROUPS) {
            next_scores(i, i);
            if (!ok) break;
            const uint32_t m = seen_rows(tile_at(i) * TILE_KEYS);
#pragma unroll
            for (int r = 0; r < FEW_ROWS; ++r) {
                if (r >= n_rows) break;
                const float x = __fmul_rn(__int2float_rn(s16[r]), kf);
                if (m >> r & 1) {
                    top[r] = fmaxf(top[r], x);
                    sig[r] = max(sig[r], vf);
                }
            }
        }
        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");  // what was kept
#pragma unroll
        for (int r = 0; r < FEW_ROWS; ++r) {
            if (r >= n_rows) break;
            const int t = __reduce_max_sync(0xffffffffu, ordered(__float_as_int(top[r])));
            const uint32_t sg = __reduce_max_sync(0xffffffffu, sig[r]);
            if (lane == 0) {
                s_tops[warp * FEW_ROWS + r] = t;
                s_sigs[warp * FEW_ROWS + r] = sg;
            }
        }
        asm volatile("bar.sync 1, %0;" ::"n"(32 * C::SOFT) : "memory");
        const int r = threadIdx.x % FEW_ROWS;
        int t = ordered(__float_as_int(-INFINITY));
        uint32_t sg = 0;
        if (r < n_rows)
            for (int w = 0; w < C::SOFT; ++w) {
                t = max(t, s_tops[w * FEW_ROWS + r]);
                sg = max(sg, s_sigs[w * FEW_ROWS + r]);
            }
        for (uint32_t c = threadIdx.x / FEW_ROWS; c < ranks; c += 2 * C::SOFT) {  // to every block of the cluster
            peer_store(peer_addr(s_top + rank * FEW_ROWS + r, c), (uint32_t)t);
            peer_store(peer_addr(s_sig + rank * FEW_ROWS + r, c), sg);
            peer_arrive(peer_addr(x_full, c));
        }
        __syncwarp();
    }
    uint32_t row_sig = 0;  // threads 0 .. 15: of their row
    if (soft) {
        bool met = wait_cluster(x_full, 0, err, dg::ERR_TIMEOUT_ACCUM);
        ok = __all_sync(0xffffffffu, met && ok);
        if (threadIdx.x < FEW_ROWS) {
            int t = (int)s_top[threadIdx.x];
            for (uint32_t c = 0; c < ranks; ++c) {
                t = max(t, (int)s_top[c * FEW_ROWS + threadIdx.x]);
                row_sig = max(row_sig, s_sig[c * FEW_ROWS + threadIdx.x]);
            }
            const int e = row_sig ? scale_exp(row_sig >> 16) : 0;
            s_row[threadIdx.x] = make_float4(__int_as_float(ordered(t)), s_pos[threadIdx.x] >= 0 ? -s_theta[threadIdx.x] : 0.0f, pow2f(-e), pow2f(e));
        }
        asm volatile("bar.sync 1, %0;" ::"n"(32 * C::SOFT) : "memory");
        // ── phase 1: the weights and the sums ──
        uint32_t total[FEW_ROWS];  // at most 131072 tiles of one key a thread: below 2^32
#pragma unroll
        for (int r = 0; r < FEW_ROWS; ++r) total[r] = 0;
        // Sums number oc are taken by the group whose tile was the last; thread `key` has column 128 x + key of O. The 32
        // columns of a warp's row go to one block of the cluster, the rows and warps round the blocks.
        auto take_sums = [&](uint32_t oc) {
            ok = ok && wait(o_full, oc & 1u, err, dg::ERR_TIMEOUT_ACCUM);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) return;
            asm volatile("tcgen05.fence::after_thread_sync;");
#pragma unroll
            for (int x = 0; x < NK; ++x) {
                int32_t h[32];
                dg::tmem_ld32(lane_addr + C::SUMS + 32 * x, h);
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                for (int r = 0; r < FEW_ROWS; ++r) {
                    if (r >= n_rows) break;
                    const uint32_t w = r * (NK * 128) + x * 128 + key;
                    peer_add(peer_addr((long long*)(sm + C::RED) + w, (w >> 5) % ranks),
                             (uint64_t)((long long)h[r] * 256 + h[16 + r]));
                }
            }
            asm volatile("tcgen05.fence::before_thread_sync;");
            __syncwarp();
            if (lane == 0) mbar_arrive(o_free);
        };
        for (int i = grp; ok && i < n; i += GROUPS) {
            next_scores(i, n + i);
            if (!ok) break;
            ok = i < 2 || block_done(v_block(i - 2));  // the digits of tile i - 2 have been read
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            const uint32_t m = seen_rows(tile_at(i) * TILE_KEYS);
            const float sv = __uint_as_float(vf);
            uint8_t* pp = sm + C::P + (i & 1) * 4096 + (key & 15);
            const int chunk = key >> 4;
#pragma unroll
            for (int r = 0; r < FEW_ROWS; ++r) {
                if (r >= n_rows) break;
                const float4 row = s_row[r];
                const float x = __fmul_rn(__int2float_rn(s16[r]), kf);
                float w = weight(x, row.x, -row.y);
                if (!(m >> r & 1)) w = 0.0f;
                total[r] += __float_as_uint(__fadd_rn(w, MAGIC)) - MAGIC_BITS;
                const uint32_t d = __float_as_uint(__fmaf_rn(w, __fmul_rn(sv, row.z), MAGIC + 128.0f));
                uint8_t* at = pp + r * 128 + ((chunk ^ (r & 7)) << 4);
                at[0] = (uint8_t)(d >> 8);
                at[16 * 128] = (uint8_t)(d ^ 0x80u);
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_full[i & 1]);
            if ((i + 1) % FLUSH_TILES == 0 || i + 1 == n) take_sums((uint32_t)i / FLUSH_TILES);
        }
#pragma unroll
        for (int r = 0; r < FEW_ROWS; ++r) {
            if (r >= n_rows) break;
            const unsigned long long lo = __reduce_add_sync(0xffffffffu, total[r] & 0xffffu),
                                     hi = __reduce_add_sync(0xffffffffu, total[r] >> 16);
            if (lane < (int)ranks) peer_add(peer_addr(s_total + r, lane), lo + (hi << 16));
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;");
    __syncwarp();
    cluster_arrive();
    cluster_wait();  // all sums are in; nobody touches another block's memory from here on
    if (soft) {
        if (threadIdx.x < FEW_ROWS) {
            const int r = threadIdx.x;
            const unsigned long long t = s_total[r];
            s_inv[r] = t ? __ddiv_rn(2097152.0, (double)t) : 0.0;
            if (rank == 0 && r < n_rows && (row0 + r) % g == 0)
                a.o_scale[((long long)begin + (row0 + r) / g) * a.c.heads + head] =
                    t ? make_longlong2(1, (long long)(uint32_t)(21 - scale_exp(row_sig >> 16))) : make_longlong2(0, 0);
        }
        asm volatile("bar.sync 1, %0;" ::"n"(32 * C::SOFT) : "memory");
        const long long* red = (const long long*)(sm + C::RED);
        for (uint32_t w = rank + ranks * (uint32_t)warp; w < (uint32_t)(n_rows * NK * 4); w += ranks * C::SOFT) {
            const int r = (int)w / (NK * 4), d = (int)(w % (NK * 4)) * 32 + lane;
            if (d < dim)
                a.o[((long long)begin + (row0 + r) / g) * a.ld_o + (long long)(head * g + (row0 + r) % g) * dim + d] =
                    out_code(red[w * 32 + lane], s_inv[r]);
        }
    }
    if (warp == 0) {
        asm volatile("tcgen05.fence::after_thread_sync;");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(C::COLS));
    }
}

}  // namespace kv
