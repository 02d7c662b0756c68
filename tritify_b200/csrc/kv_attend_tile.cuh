// Attention over the paged cache for many query rows: a block takes 128 rows (token, query head) of one sequence and KV
// head and walks the keys they see in tiles of 128.
//
// The maximum of a row has to be known before its first weight is rounded, so the keys are walked twice: pass 0 forms
// the scores for the row maxima (and the largest visible value scale), pass 1 forms them again and the weights. That
// costs the score products twice and K's bytes from L2 twice; in return every weight is final when it is formed, and the
// sums over the keys are plain integer sums that no later tile rescales.
//
// Per tile: S = Q K^T, 128 x 128 int32 in TMEM (tcgen05.mma kind::i8, K by TMA with the 128-byte swizzle); the weights
// as two balanced 8-bit digits, w = 256 hi + lo, in shared memory; O_hi += P_hi V, O_lo += P_lo V in TMEM (V as it lies
// in its pages, the MN-major operand). The int32 sums hold 132104 keys (127 * 128 each); every 131072 keys the carry of
// lo goes into hi and that of hi into a 16-bit word of shared memory, which holds 2^25 keys.
//
// Roles (640 threads): warps 0-15 softmax, in two groups that take the tiles in turn; warp 16 TMA, warp 17 the products of
// the scores, warp 18 the keys' scales, warp 19 the products of the values. Waits are bounded as in digit_gemm.cuh.
#pragma once

#include <cuda.h>

#include "digit_gemm.cuh"
#include "kv_kernels.cuh"

namespace kv {

using dg::mbar_arrive;
using dg::mbar_arrive_expect_tx;
using dg::mbar_init;
using dg::smem_u32;

constexpr int TILE_KEYS = 128;
constexpr int TILE_ROWS = 128;

// A bounded wait (2 s): false when it expires, or when another wait of the context has. The loop is out of line: the kernels wait in
// some twenty places, and with it inline a sixth of the few-row kernel's stalls were for instructions, and it took 126 us against 120.
static __device__ __noinline__ bool wait_on(uint32_t bar, uint32_t parity, int* err, int code) {
    const uint64_t t0 = dg::globaltimer();
    for (uint32_t it = 1;; ++it) {
        uint32_t ok;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok)
            : "r"(bar), "r"(parity)
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
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, int* err, int code) {
    return dg::mbar_try_wait(bar, parity) || wait_on(smem_u32(bar), parity, err, code);
}

// wait() by a whole warp.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, int* err, int code) {
    return __all_sync(0xffffffffu, wait(bar, parity, err, code));
}

// The same copy of bytes that are read once: their lines leave L2 before others.
__device__ __forceinline__ uint64_t once_policy() {
    uint64_t p;
    asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(p));
    return p;
}
__device__ __forceinline__ void tma_load_4d_once(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int w,
                                                 uint64_t* bar, uint64_t policy) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%2, %3, "
        "%4, %5}], [%6], %7;" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar)), "l"(policy)
        : "memory");
}

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int w,
                                            uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
        "[%6];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar))
        : "memory");
}

// Low words of shared-memory descriptors with the 128-byte swizzle: the address in units of 16 bytes and a stride. K-major
// operands do not use the stride; an MN-major operand one 128-byte block wide has rows that are steps of K, and neither
// does it. The high word (8-row groups 1024 bytes apart, version, swizzle) is the same for all.
constexpr uint32_t DESC_HI = (1024u >> 4) | 1u << 14 | 2u << 29;
__device__ __forceinline__ uint32_t desc_k(uint32_t addr) { return (addr >> 4) | 1u << 16; }
__device__ __forceinline__ uint32_t desc_mn(uint32_t addr) { return (addr >> 4) | (1024u >> 4) << 16; }

// D += A B (or D = A B, accumulate = 0) of 8-bit operands given by their descriptors' low words, and the arrival of a
// barrier when every product issued so far is done. A whole warp comes here and the one lane with `issue` set acts, so
// that the loop around them stays uniform. A product of K = 32 takes some 67 clocks whatever N up to 128 is, an arrival
// about 130 of the issuing warp's: a tile's four products and two arrivals, 530.
__device__ __forceinline__ void umma(bool issue, uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t.reg .b64 da, db;\n\t"
        "setp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %6, 0;\n\tmov.b64 da, {%1, %5};\n\tmov.b64 db, {%2, %5};\n\t"
        "@q tcgen05.mma.cta_group::1.kind::i8 [%0], da, db, %3, p;\n\t}" ::"r"(d),
        "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "r"(DESC_HI), "r"((int)issue)
        : "memory");
}
__device__ __forceinline__ void umma_arrive(bool issue, uint64_t* bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar)),
        "r"((int)issue)
        : "memory");
}

// kind::i8, s32 += s8 x s8, M = 128, N = n; `mn` bits 15 and 16: A, B MN-major.
__device__ __forceinline__ uint32_t idesc_i8(int n, uint32_t mn) {
    return (2u << 4) | (1u << 7) | (1u << 10) | mn | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}

// ── pairs of binary32 in one instruction ──
typedef unsigned long long f2;
__device__ __forceinline__ f2 pk(float a, float b) {
    f2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void upk(f2 v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) {
    f2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ f2 add2(f2 a, f2 b) {
    f2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

template <bool V>
struct Bool {
    static constexpr bool value = V;
};

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const int32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
            taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]));
}

constexpr float MAGIC = 12582912.0f;  // 3 * 2^22: adding it rounds to a whole number, left in the low bits
constexpr uint32_t MAGIC_BITS = 0x4B400000u;

// Dot products (|s| <= 2^22, exact in binary32) of two adjacent keys times their scales, RN24.
__device__ __forceinline__ f2 scaled2(int32_t s0, int32_t s1, f2 sigma) {
    f2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(pk(__int2float_rn(s0), __int2float_rn(s1))), "l"(sigma));
    return r;
}

// What a row's weights need: the maximum, -theta, the cubic's coefficients times 2^-E, and 2^E.
struct RowWeights {
    f2 top, ntheta, c0, c1, c2, c3, two_e;
};

__device__ __forceinline__ RowWeights row_weights(float top, float theta, int e) {
    const float l = pow2f(-e);
    RowWeights r;
    r.top = pk(top, top);
    r.ntheta = pk(-theta, -theta);
    r.c0 = pk(W_C0 * l, W_C0 * l);
    r.c1 = pk(W_C1 * l, W_C1 * l);
    r.c2 = pk(W_C2 * l, W_C2 * l);
    r.c3 = pk(W_C3 * l, W_C3 * l);
    r.two_e = pk(pow2f(e), pow2f(e));
    return r;
}

// weight() for a pair, times 2^-E. MASK: keys whose bit of `seen` is clear weigh nothing, exactly: even 2^-32 of a weight
// would show, since 2^E bounds the value scales of visible keys alone.
template <bool MASK>
__device__ __forceinline__ f2 weight2(f2 x, const RowWeights& w, uint32_t seen) {
    const f2 minus = pk(-1.0f, -1.0f);
    const f2 d = fma2(x, minus, w.top);
    float a, b;
    upk(fma2(d, w.ntheta, pk(12288.0f, 12288.0f)), a, b);
    a = fmaxf(a, 12256.0f);
    b = fmaxf(b, 12256.0f);
    const f2 f = pk(a, b);
    const f2 f0 = add2(f, pk(12570624.0f, 12570624.0f));
    const f2 r = fma2(add2(f0, pk(-12570624.0f, -12570624.0f)), minus, f);
    f2 e = fma2(w.c3, r, w.c2);
    e = fma2(e, r, w.c1);
    e = fma2(e, r, w.c0);
    float e0, e1, n0, n1;
    upk(e, e0, e1);
    upk(f0, n0, n1);
    e0 = __uint_as_float(__float_as_uint(e0) + (__float_as_uint(n0) << 23));
    e1 = __uint_as_float(__float_as_uint(e1) + (__float_as_uint(n1) << 23));
    if (MASK) {
        e0 = (seen & 1) ? e0 : 0.0f;
        e1 = (seen & 2) ? e1 : 0.0f;
    }
    return pk(e0, e1);
}

// The keys that a tile's rows at positions p0 .. p1 see, as a list of 128-key tiles: first those of the sinks, then
// those from the first row's window on.
struct KeyTiles {
    int n, n_sink, first;
    __device__ __forceinline__ KeyTiles(int p0, int p1, int window, int sinks) {
        const int lo = window && p0 >= window ? p0 + 1 - window : 0;  // p0 may lie far below zero
        first = lo / TILE_KEYS;
        n_sink = min((min(sinks, lo) + TILE_KEYS - 1) / TILE_KEYS, first);
        n = p1 < 0 ? 0 : n_sink + p1 / TILE_KEYS - first + 1;
    }
    __device__ __forceinline__ int at(int i) const { return i < n_sink ? i : i - n_sink + first; }
};

// Bit k set: key j0 + k (k < 32) is visible to a row at position pos.
__device__ __forceinline__ uint32_t seen_bits(int j0, int pos, int window, int sinks) {
    auto below = [&](int end) -> uint32_t {  // keys j < end
        const int k = end - j0;
        return k <= 0 ? 0u : k >= 32 ? ~0u : (1u << k) - 1;
    };
    if (pos < 0) return 0;
    uint32_t m = below(pos + 1);
    if (window && pos >= window) m &= ~below(pos + 1 - window) | below(sinks);
    return m;
}

// Two value scales (bfloat16) held at the largest there is, 2^63. A tile may hold places that no row sees and that were
// never written: whatever lies there, 0xffff among it, is then a number, which a hidden key's weight of zero takes away.
__device__ __forceinline__ uint32_t held_scales(uint32_t v) { return __vminu2(v, 0x5f005f00u); }

// The last i in [0, n) with f(i) <= target (f ascends), by a whole warp; 0 when there is none.
template <class F>
__device__ __forceinline__ int warp_search(int n, long long target, F f) {
    const int lane = threadIdx.x & 31;
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32;
        const int i = min(lo + lane * step, hi - 1);
        const bool in = lo + lane * step < hi;
        const unsigned le = __ballot_sync(0xffffffffu, in && f(i) <= target);
        const int k = max(1, 32 - __clz(le));
        lo = lo + (k - 1) * step;
        hi = min(lo + step, hi);
    }
    return lo;
}

// NK: 128-byte blocks of a key row (head_dim up to 128, or up to 256).
template <int NK>
struct TileCfg {
    static constexpr int SLOT = TILE_KEYS * 128;  // bytes of one block of a key or value tile
    static constexpr int K_SLOTS = 3, V_SLOTS = NK == 1 ? 3 : 2;  // rings of K and V blocks
    static constexpr int SLOTS = K_SLOTS + V_SLOTS;
    static constexpr int SCALES = 4;  // tiles of key scales in flight
    static constexpr int Q = 0;
    static constexpr int P = Q + NK * SLOT;           // [2][hi, lo]
    static constexpr int RING = P + 4 * SLOT;
    static constexpr int CARRY = RING + SLOTS * SLOT;  // int16 [128 columns][128 rows]
    // [SCALES]: sigma_k and sigma_v [128], the largest sigma_v
    static constexpr int KEY_STAGE = 2 * TILE_KEYS + 4;
    static constexpr int KEY_SCALES = CARRY + TILE_ROWS * 128 * 2;
    static constexpr int ROWS = KEY_SCALES + SCALES * KEY_STAGE * 4;  // theta, max [4], largest sigma [4], L [4]
    static constexpr int BARS = ROWS + TILE_ROWS * (4 + 16 + 16 + 32);
    static constexpr int BYTES = 1024 + BARS + 512;
    static_assert(BYTES <= 232448, "shared memory per block");
};

constexpr int SOFTMAX_WARPS = 16;
constexpr int TILE_THREADS = 32 * (SOFTMAX_WARPS + 4);
constexpr int FLUSH_TILES = 1024;  // 131072 keys: |sum| <= 131072 * 127 * 128 < 2^31

template <int NK>
__global__ void __launch_bounds__(TILE_THREADS, 1)
    attend_tile_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                       const AttendArgs a, long long slots) {
    kt::pdl_enter();
    using C = TileCfg<NK>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* sm = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    float* s_theta = (float*)(sm + C::ROWS);
    float* s_top = s_theta + TILE_ROWS;
    uint32_t* s_sig = (uint32_t*)(s_top + 4 * TILE_ROWS);
    unsigned long long* s_total = (unsigned long long*)(s_sig + 4 * TILE_ROWS);
    uint64_t* full = (uint64_t*)(sm + C::BARS);  // [SLOTS] a block of K or V has landed (K's slots, then V's)
    uint64_t* empty = full + C::SLOTS;           // [SLOTS] its products are done
    uint64_t* s_full = empty + C::SLOTS;         // [2] scores in TMEM
    uint64_t* s_free = s_full + 2;               // [2] scores read
    uint64_t* m_full = s_free + 2;               // [4] the same in pass 0, which has no sums in TMEM and uses it all
    uint64_t* m_free = m_full + 4;               // [4]
    uint64_t* p_full = m_free + 4;               // [2] digits of the weights in shared memory
    uint64_t* p_free = p_full + 2;               // [2] their products are done
    uint64_t* k_full = p_free + 2;               // [SCALES]
    uint64_t* k_free = k_full + C::SCALES;       // [SCALES]
    uint64_t* q_full = k_free + C::SCALES;
    uint64_t* o_full = q_full + 1;
    uint64_t* o_free = o_full + 1;
    uint64_t* done = o_free + 1;  // [2] every product of an issuing warp is done
    uint32_t* tmem_slot = (uint32_t*)(done + 2);
    int* s_job = (int*)(tmem_slot + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = a.group, dim = a.c.dim;
    const int head = (int)(blockIdx.x % (unsigned)a.c.heads);
    // later tiles of a sequence see more keys: they start first
    const long long slot = slots - 1 - (long long)(blockIdx.x / (unsigned)a.c.heads);
    // Sequence b's tiles stand at slots begin_b g / 128 + b and on: there is room for them before the next sequence's,
    // and the few slots that stay empty leave at once.
    if (warp == 0) {
        auto first_slot = [&](int b) { return (long long)a.b.begin[b] * g / TILE_ROWS + b; };
        const int b = warp_search(a.b.n_seqs, slot, first_slot);
        const int begin = a.b.begin[b], end = a.b.begin[b + 1], len = a.b.kv_len[b];
        const long long row0 = (slot - first_slot(b)) * TILE_ROWS;
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
            mbar_init(&s_full[i], 1);
            mbar_init(&s_free[i], SOFTMAX_WARPS / 2);
            mbar_init(&p_full[i], SOFTMAX_WARPS / 2);
            mbar_init(&p_free[i], 1);
        }
        for (int i = 0; i < 4; ++i) {
            mbar_init(&m_full[i], 1);
            mbar_init(&m_free[i], SOFTMAX_WARPS / 2);
        }
        for (int i = 0; i < C::SCALES; ++i) {
            mbar_init(&k_full[i], 1);
            mbar_init(&k_free[i], SOFTMAX_WARPS / 2);
        }
        mbar_init(q_full, SOFTMAX_WARPS);
        mbar_init(o_full, 1);
        mbar_init(o_free, SOFTMAX_WARPS);
        mbar_init(&done[0], 1);
        mbar_init(&done[1], 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    const int seq = s_job[0];
    if (seq < 0) return;
    const int begin = s_job[1], n_new = s_job[2], len = s_job[3], row0 = s_job[4];
    const int n_rows = min(TILE_ROWS, n_new * g - row0);
    const int t0 = row0 / g;
    const int p0 = len - n_new + t0, p1 = len - n_new + (row0 + n_rows - 1) / g;
    const KeyTiles kt_(p0, p1, a.window, a.sinks);
    const int n = kt_.n;
    const int n_pass = n > 0 ? 1 + NK : 0;  // the maxima, then the values of each 128-column block
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_slot)));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
        asm volatile("tcgen05.fence::before_thread_sync;");
    }
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;");
    const uint32_t tmem = *tmem_slot;
    const int ps = 1 << a.c.page_shift;

    if (warp == SOFTMAX_WARPS) {
        // Step i takes K of tile i and, after pass 0, V of tile i - 1. A lane holds one page of a tile; page numbers are
        // read three steps ahead.
        const int per_tile = TILE_KEYS >> a.c.page_shift, last_page = p1 >> a.c.page_shift;
        const int* pages = a.b.pages + (long long)seq * a.b.max_pages;
        int ks = 0, vs = C::K_SLOTS;                // the next slots
        uint32_t kph = 1, vph = 1, kq = 0, vq = 0;  // the parities of their release; blocks loaded so far
        bool alive = true;
        auto page_of = [&](int i) -> int {
            const int at = kt_.at(min(i, n - 1)) * per_tile + lane;
            return lane < per_tile && at <= last_page ? pages[at] : 0;
        };
        auto load = [&](const CUtensorMap* map, int i, int x, int page, int s, uint32_t phase) {
            // pages that hold keys up to the last row's position; the others' keys are not visible
            const int np = min(per_tile, last_page - kt_.at(i) * per_tile + 1);
            if ((unsigned)page >= (unsigned long long)a.c.n_pages) {
                a.err.raise(a.err.bad_page);
                page = 0;
            }
            bool ok = true;
            if (lane == 0) {
                ok = wait(&empty[s], phase, a.err.word, dg::ERR_TIMEOUT_EMPTY);
                if (ok) mbar_arrive_expect_tx(&full[s], (uint32_t)(np * ps * 128));
            }
            ok = __shfl_sync(0xffffffffu, (int)ok, 0);
            if (!ok) {
                alive = false;
                return;
            }
            if (lane < np)
                tma_load_4d(smem_u32(sm + C::RING + s * C::SLOT + lane * ps * 128), map, x, 0, head, page, &full[s]);
        };
        for (int pass = 0; alive && pass < n_pass; ++pass) {
            int pg[4];
#pragma unroll
            for (int j = 0; j < 3; ++j) pg[j] = page_of(j);
            for (int i0 = 0; alive && i0 <= n; i0 += 4) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int i = i0 + j;
                    if (!alive || i > n) break;
                    if (i < n) {
#pragma unroll
                        for (int x = 0; x < NK; ++x) {
                            if (alive) load(&map_k, i, x * 128, pg[j], ks, kph);
                            kq += alive;
                            if (alive && ++ks == C::K_SLOTS) ks = 0, kph ^= 1;
                        }
                    }
                    if (pass > 0 && i > 0 && alive) {
                        load(&map_v, i - 1, (pass - 1) * 128, pg[(j + 3) & 3], vs, vph);
                        vq += alive;
                        if (alive && ++vs == C::SLOTS) vs = C::K_SLOTS, vph ^= 1;
                    }
                    pg[(j + 3) & 3] = page_of(i + 3);
                }
            }
        }
        if (lane == 0) {  // copies still in flight land before the block leaves
            for (uint32_t j = kq > (uint32_t)C::K_SLOTS ? kq - C::K_SLOTS : 0; j < kq; ++j)
                dg::mbar_wait_drain(&full[j % C::K_SLOTS], (j / C::K_SLOTS) & 1u, a.err.word, dg::ERR_TIMEOUT_FULL);
            for (uint32_t j = vq > (uint32_t)C::V_SLOTS ? vq - C::V_SLOTS : 0; j < vq; ++j)
                dg::mbar_wait_drain(&full[C::K_SLOTS + j % C::V_SLOTS], (j / C::V_SLOTS) & 1u, a.err.word,
                                    dg::ERR_TIMEOUT_FULL);
        }
    } else if (warp == SOFTMAX_WARPS + 1) {
        // scores: S of tile after tile, as soon as K has landed and the buffer has been read
        {
            const bool issue = lane == 0;
            const int ksteps = (dim + 31) / 32;
            const uint32_t id_s = idesc_i8(TILE_KEYS, 0);
            const uint32_t qd = desc_k(smem_u32(sm + C::Q)), kd = desc_k(smem_u32(sm + C::RING));
            int ks = 0;
            uint32_t kph = 0;
            bool ok = n_pass == 0 || warp_wait(q_full, 0, a.err.word, dg::ERR_TIMEOUT_FULL);
            const int total = n_pass * n;
            for (int u = 0; ok && u < total; ++u) {
                // scores number u go to buffer u % 4 in pass 0 and to buffer u % 2 later, first when pass 0 has read it
                const bool maxima = u < n;
                const uint32_t b = maxima ? u & 3 : u & 1;
                const uint32_t use = (uint32_t)(maxima ? u >> 2 : (u - n) >> 1);
                if (!maxima && use == 0) {
                    const uint32_t uses = (uint32_t)(n - (int)b + 3) / 4;
                    ok = uses == 0 || warp_wait(&m_free[b], (uses - 1) & 1u, a.err.word, dg::ERR_TIMEOUT_ACCUM);
                }
                ok = ok && warp_wait(maxima ? &m_free[b] : &s_free[b], (use & 1u) ^ 1u, a.err.word, dg::ERR_TIMEOUT_ACCUM);
#pragma unroll
                for (int x = 0; x < NK; ++x) {
                    ok = ok && warp_wait(&full[ks], kph, a.err.word, dg::ERR_TIMEOUT_FULL);
                    if (!ok) break;
                    asm volatile("tcgen05.fence::after_thread_sync;");
                    // descriptors hold addresses in units of 16 bytes
                    const uint32_t qx = qd + x * (C::SLOT >> 4), kx = kd + ks * (C::SLOT >> 4);
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk)
                        if (4 * x + kk < ksteps) umma(issue, tmem + b * 128, qx + 2 * kk, kx + 2 * kk, id_s, x + kk > 0);
                    umma_arrive(issue, &empty[ks]);
                    if (++ks == C::K_SLOTS) ks = 0, kph ^= 1;
                }
                if (!ok) break;
                umma_arrive(issue, maxima ? &m_full[b] : &s_full[b]);
            }
            umma_arrive(issue, &done[0]);
            if (issue) dg::mbar_wait_drain(&done[0], 0u, a.err.word, dg::ERR_TIMEOUT_ACCUM);
        }
    } else if (warp == SOFTMAX_WARPS + 3) {
        // the values: O += P V with both digits, as soon as a tile's weights are there
        {
            const bool issue = lane == 0;
            const uint32_t pd = desc_k(smem_u32(sm + C::P)), vd = desc_mn(smem_u32(sm + C::RING));
            int vs = C::K_SLOTS;
            uint32_t vph = 0, b = (uint32_t)n & 1, pph = 0, oc = 0;  // pass 1 begins with scores number n
            bool ok = true, second = false;
            for (int pass = 1; ok && pass < n_pass; ++pass) {
                const uint32_t id_o = idesc_i8(min(128, dim - (pass - 1) * 128), 1u << 16);
                for (int i = 0; i < n; ++i) {
                    ok = warp_wait(&p_full[b], pph, a.err.word, dg::ERR_TIMEOUT_ACCUM) &&
                         warp_wait(&full[vs], vph, a.err.word, dg::ERR_TIMEOUT_FULL);
                    if (!ok) break;
                    asm volatile("tcgen05.fence::after_thread_sync;");
                    const uint32_t px = pd + b * (2 * C::SLOT >> 4), vx = vd + vs * (C::SLOT >> 4);
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk) {
                        umma(issue, tmem + 256, px + 2 * kk, vx + kk * (32 * 128 >> 4), id_o, i + kk > 0);
                        umma(issue, tmem + 384, px + (C::SLOT >> 4) + 2 * kk, vx + kk * (32 * 128 >> 4), id_o, i + kk > 0);
                    }
                    umma_arrive(issue, &empty[vs]);
                    umma_arrive(issue, &p_free[b]);
                    if (++vs == C::SLOTS) vs = C::K_SLOTS, vph ^= 1;
                    b ^= 1;
                    if (second) pph ^= 1;
                    second = !second;
                    // the sums are read at the end of the block, and carried on every FLUSH_TILES tiles
                    if (i + 1 == n || (i + 1) % FLUSH_TILES == 0) {
                        umma_arrive(issue, o_full);
                        if (i + 1 < n || pass + 1 < n_pass) {
                            ok = warp_wait(o_free, oc & 1u, a.err.word, dg::ERR_TIMEOUT_ACCUM);
                            if (!ok) break;
                            asm volatile("tcgen05.fence::after_thread_sync;");
                        }
                        ++oc;
                    }
                }
            }
            umma_arrive(issue, &done[1]);
            if (issue) dg::mbar_wait_drain(&done[1], 0u, a.err.word, dg::ERR_TIMEOUT_ACCUM);
        }
    } else if (warp == SOFTMAX_WARPS + 2) {
        // The scales of each tile's keys, four keys a lane: read four tiles ahead, their page numbers eight.
        const int* pages = a.b.pages + (long long)seq * a.b.max_pages;
        const int total = n_pass * n;
        auto key_of = [&](int u) {
            for (; u >= n; u -= n) {}  // at most two passes back
            return kt_.at(u) * TILE_KEYS + 4 * lane;
        };
        auto page_of = [&](int u) -> int {
            const int j = u < total ? key_of(u) : p1 + 1;
            return j <= p1 ? pages[j >> a.c.page_shift] : 0;
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
                    alive = wait(&k_free[j], ((u >> 2) & 1u) ^ 1u, a.err.word, dg::ERR_TIMEOUT_EMPTY);
                    alive = __all_sync(0xffffffffu, alive);
                    if (!alive) break;
                    float* f = (float*)(sm + C::KEY_SCALES) + j * C::KEY_STAGE;
                    uint4 w = val[j];
                    w.z = held_scales(w.z);
                    w.w = held_scales(w.w);
                    const uint32_t hi16 = 0xffff0000u;
                    const float4 kf = {__uint_as_float(w.x << 16), __uint_as_float(w.x & hi16),
                                       __uint_as_float(w.y << 16), __uint_as_float(w.y & hi16)};
                    const uint4 vf = {w.z << 16, w.z & hi16, w.w << 16, w.w & hi16};
                    *(float4*)(f + 4 * lane) = kf;
                    *(uint4*)(f + TILE_KEYS + 4 * lane) = vf;
                    const unsigned big = max(max(vf.x, vf.y), max(vf.z, vf.w));
                    const unsigned tile_big = __reduce_max_sync(0xffffffffu, big);
                    if (lane == 0) ((uint32_t*)f)[2 * TILE_KEYS] = tile_big;
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&k_full[j]);
                    val[j] = scales_of(u + 4, pg[j]);
                    pg[j] = page_of(u + 8);
                }
            }
        }
    } else {
        // Two groups of eight warps take the tiles in turn, each with its own buffer of scores and of digits, so that
        // one group's waits pass under the other's arithmetic. A warp has the rows of TMEM lanes 32 quad .. and the
        // keys 64 part .. of its group's tiles.
        const int quad = warp & 3, part = (warp >> 2) & 1, grp = warp >> 3;
        const uint32_t lane_addr = tmem + ((uint32_t)(quad * 32) << 16);
        const uint32_t s_addr = lane_addr + grp * 128 + part * 64;
        // the queries' codes, from where query_kernel left them, into the K-major operand
        if (n_pass > 0) {
            const int per_row = dim / 16;
            for (int i = threadIdx.x; i < n_rows * per_row; i += 32 * SOFTMAX_WARPS) {
                const int r = i / per_row, c = i - r * per_row, rr = row0 + r;
                const int32_t* x = a.o + ((long long)begin + rr / g) * a.ld_o + (long long)(head * g + rr % g) * dim;
                const int4 v = a.vec_o ? *(const int4*)(x + 4 * c) : make_int4(x[4 * c], x[4 * c + 1], x[4 * c + 2], x[4 * c + 3]);
                *(int4*)(sm + C::Q + (c >> 3) * C::SLOT + r * 128 + (((c & 7) ^ (r & 7)) << 4)) = v;
                if (c == 0) s_theta[r] = __int_as_float(x[dim / 4]);
            }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(q_full);
        const int r = quad * 32 + lane;  // row of the tile
        const bool row_live = r < n_rows;
        const int t = (row0 + min(r, n_rows - 1)) / g;
        const int pos = row_live ? len - n_new + t : -1;
        uint32_t sc = 0, oc = 0;  // sc: number of the scores at hand, over all passes
        bool ok = true;
        float top = -INFINITY;
        uint32_t sig = 0;
        // whether every live row sees all of tile j0 .. j0 + 127 (the same for all warps)
        auto whole = [&](int j0) {
            if (j0 + TILE_KEYS - 1 > p0) return false;
            return !a.window || j0 > p1 - a.window || j0 + TILE_KEYS <= a.sinks;
        };
        // the first tile of a pass that this group takes: scores number sc with sc % 2 == grp
        auto first_of = [&](int pass) { return (grp ^ (pass * n)) & 1; };
        // wait for scores number sc, the `use`th in their buffer, and their key scales
        auto next_scores = [&](uint64_t* bar, uint32_t use) {
            ok = wait(bar, use & 1u, a.err.word, dg::ERR_TIMEOUT_ACCUM) &&
                 wait(&k_full[sc % C::SCALES], (sc / C::SCALES) & 1u, a.err.word, dg::ERR_TIMEOUT_FULL);
            ok = __all_sync(0xffffffffu, ok);
            asm volatile("tcgen05.fence::after_thread_sync;");
        };
        auto key_scales = [&]() { return (const float*)(sm + C::KEY_SCALES) + (sc % C::SCALES) * C::KEY_STAGE + part * 64; };
        // the buffer of scores goes back to the products
        auto scores_read = [&]() {
            asm volatile("tcgen05.fence::before_thread_sync;");
            __syncwarp();
            if (lane == 0) mbar_arrive(&s_free[grp]);
        };
        auto scales_read = [&]() {
            __syncwarp();
            if (lane == 0) mbar_arrive(&k_free[sc % C::SCALES]);
        };
        // ── pass 0: the maxima ──
        for (int i = first_of(0); ok && n_pass && i < n; i += 2) {
            sc = i;
            next_scores(&m_full[i & 3], i >> 2);
            if (!ok) break;
            const int j0 = kt_.at(i) * TILE_KEYS;
            const bool all = whole(j0);
            const float* f = key_scales();
            if (all) sig = max(sig, ((const uint32_t*)f)[2 * TILE_KEYS - part * 64]);
            int32_t s64[2][32];
            dg::tmem_ld32(s_addr + (i & 2) * 128, s64[0]);
            dg::tmem_ld32(s_addr + (i & 2) * 128 + 32, s64[1]);
            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
            asm volatile("tcgen05.fence::before_thread_sync;");
            __syncwarp();
            if (lane == 0) mbar_arrive(&m_free[i & 3]);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                if (all) {
#pragma unroll
                    for (int k = 0; k < 32; k += 4) {
                        const ulonglong2 kf = *(const ulonglong2*)(f + c * 32 + k);
                        float x0, x1, x2, x3;
                        upk(scaled2(s64[c][k], s64[c][k + 1], kf.x), x0, x1);
                        upk(scaled2(s64[c][k + 2], s64[c][k + 3], kf.y), x2, x3);
                        top = fmaxf(fmaxf(top, x0), x1);
                        top = fmaxf(fmaxf(top, x2), x3);
                    }
                } else {
                    const uint32_t m = seen_bits(j0 + part * 64 + c * 32, pos, a.window, a.sinks);
#pragma unroll
                    for (int k = 0; k < 32; k += 2) {
                        const f2 kf = *(const f2*)(f + c * 32 + k);
                        const uint2 vf = *(const uint2*)(f + TILE_KEYS + c * 32 + k);
                        float x0, x1;
                        upk(scaled2(s64[c][k], s64[c][k + 1], kf), x0, x1);
                        if (m >> k & 1) {
                            top = fmaxf(top, x0);
                            sig = max(sig, vf.x);
                        }
                        if (m >> k & 2) {
                            top = fmaxf(top, x1);
                            sig = max(sig, vf.y);
                        }
                    }
                }
            }
            scales_read();
        }
        // the four parts of a row (two groups, two halves of a tile) meet
        const int mine = (grp * 2 + part) * TILE_ROWS + r;
        s_top[mine] = top;
        s_sig[mine] = sig;
        asm volatile("bar.sync 1, 512;" ::: "memory");
#pragma unroll
        for (int p = 0; p < 4; ++p) {
            top = fmaxf(top, s_top[p * TILE_ROWS + r]);
            sig = max(sig, s_sig[p * TILE_ROWS + r]);
        }
        const int e_row = sig ? scale_exp(sig >> 16) : 0;
        const RowWeights rw = row_weights(top, row_live && pos >= 0 ? s_theta[r] : 0.0f, e_row);
        uint64_t total = 0;
        bool met = n_pass == 0;
        int16_t* carry = (int16_t*)(sm + C::CARRY);
        const int col0 = (grp * 2 + part) * 32;  // the columns of the sums that this warp reads
        // ── the weights and the sums ──
        uint32_t used = 0;  // times this group's digit buffer has been filled
        for (int pass = 1; ok && pass < n_pass; ++pass) {
            const int cols = min(128, dim - (pass - 1) * 128);
            int flushed = 0;
            auto flush = [&]() {
                ok = wait(o_full, oc & 1u, a.err.word, dg::ERR_TIMEOUT_ACCUM);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) return;
                asm volatile("tcgen05.fence::after_thread_sync;");
                for (int c = col0; c < min(cols, col0 + 32); c += 16) {
                    int32_t h[16], l[16];
                    dg::tmem_ld16(lane_addr + 256 + c, h);
                    dg::tmem_ld16(lane_addr + 384 + c, l);
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                    for (int k = 0; k < 16; ++k) {
                        // lo = 256 q + rest: q into hi; hi = 2^24 q + rest: q into the carry
                        h[k] += l[k] >> 8;
                        l[k] &= 255;
                        int16_t* cw = carry + (c + k) * TILE_ROWS + r;
                        *cw = (int16_t)((flushed ? *cw : 0) + (h[k] >> 24));
                        h[k] &= 0xffffff;
                    }
                    tmem_st16(lane_addr + 256 + c, h);
                    tmem_st16(lane_addr + 384 + c, l);
                }
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                asm volatile("tcgen05.fence::before_thread_sync;");
                __syncwarp();
                if (lane == 0) mbar_arrive(o_free);
                ++flushed;
                ++oc;
            };
            for (int i = first_of(pass); ok && i < n; i += 2) {
                while (ok && flushed < i / FLUSH_TILES) flush();
                if (!ok) break;
                sc = pass * n + i;
                next_scores(&s_full[grp], (sc - n) >> 1);
                if (!ok) break;
                const int j0 = kt_.at(i) * TILE_KEYS;
                const bool all = whole(j0);
                ok = wait(&p_free[grp], (used & 1u) ^ 1u, a.err.word, dg::ERR_TIMEOUT_EMPTY);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                uint8_t* hi = sm + C::P + grp * 2 * C::SLOT + r * 128;
                uint8_t* lo = hi + C::SLOT;
                uint32_t sum = 0;
                const float* f = key_scales();
                auto digits = [&](auto mask_tag, const int32_t (&s)[16], int k0, uint32_t seen) {  // of keys k0 .. k0 + 15
                    constexpr bool MASK = decltype(mask_tag)::value;
                    uint32_t h4[4], l4[4];
#pragma unroll
                    for (int k4 = 0; k4 < 4; ++k4) {
                        const int k = 4 * k4;
                        const ulonglong2 kf = *(const ulonglong2*)(f + k0 + k);
                        const ulonglong2 vf = *(const ulonglong2*)(f + TILE_KEYS + k0 + k);
                        const uint32_t m = MASK ? seen >> k : 0u;
                        const f2 w0 = weight2<MASK>(scaled2(s[k], s[k + 1], kf.x), rw, m);
                        const f2 w1 = weight2<MASK>(scaled2(s[k + 2], s[k + 3], kf.y), rw, m >> 2);
                        const f2 mg = pk(MAGIC, MAGIC), mg128 = pk(MAGIC + 128.0f, MAGIC + 128.0f);
                        float a0, a1, a2, a3;
                        upk(fma2(w0, rw.two_e, mg), a0, a1);
                        upk(fma2(w1, rw.two_e, mg), a2, a3);
                        sum += __float_as_uint(a0) + __float_as_uint(a1);
                        sum += __float_as_uint(a2) + __float_as_uint(a3);
                        upk(fma2(w0, vf.x, mg128), a0, a1);
                        upk(fma2(w1, vf.y, mg128), a2, a3);
                        // w + 128 in the low 16 bits: the upper byte is hi, the lower one lo + 128
                        const uint32_t u = __byte_perm(__float_as_uint(a0), __float_as_uint(a1), 0x5140);
                        const uint32_t v = __byte_perm(__float_as_uint(a2), __float_as_uint(a3), 0x5140);
                        l4[k4] = __byte_perm(u, v, 0x5410) ^ 0x80808080u;
                        h4[k4] = __byte_perm(u, v, 0x7632);
                    }
                    const int chunk = ((part * 4 + (k0 >> 4)) ^ (r & 7)) * 16;
                    *(uint4*)(hi + chunk) = make_uint4(h4[0], h4[1], h4[2], h4[3]);
                    *(uint4*)(lo + chunk) = make_uint4(l4[0], l4[1], l4[2], l4[3]);
                };
                // 16 of this thread's 64 scores at a time: the next ones asked for under the arithmetic cost as much in
                // registers as they gained (380 us against 378 for a prompt of 4096)
                auto walk = [&](auto mask_tag) {
                    constexpr bool MASK = decltype(mask_tag)::value;
#pragma unroll 1
                    for (int k0 = 0; k0 < 64; k0 += 16) {
                        int32_t s[16];
                        dg::tmem_ld16(s_addr + k0, s);
                        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                        if (k0 == 48) scores_read();
                        digits(mask_tag, s, k0, MASK ? seen_bits(j0 + part * 64 + k0, pos, a.window, a.sinks) : 0u);
                    }
                };
                if (all) walk(Bool<false>{});
                else walk(Bool<true>{});
                if (pass == 1) total += sum - 64u * MAGIC_BITS;
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[grp]);
                ++used;
                scales_read();
            }
            while (ok && flushed < (n - 1) / FLUSH_TILES) flush();
            if (pass == 1) {  // the row's total over its parts
                s_total[mine] = total;
                asm volatile("bar.sync 1, 512;" ::: "memory");
                met = true;
                total = 0;
#pragma unroll
                for (int p = 0; p < 4; ++p) total += s_total[p * TILE_ROWS + r];
            }
            if (!ok) break;
            ok = wait(o_full, oc & 1u, a.err.word, dg::ERR_TIMEOUT_ACCUM);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            ++oc;
            asm volatile("tcgen05.fence::after_thread_sync;");
            const double inv = total ? __ddiv_rn(2097152.0, (double)total) : 0.0;
            int32_t* out = a.o + ((long long)begin + t) * a.ld_o +
                           (long long)(head * g + (row0 + min(r, n_rows - 1)) % g) * dim + (pass - 1) * 128;
            for (int c = col0; c < min(cols, col0 + 32); c += 16) {
                int32_t h[16], l[16];
                dg::tmem_ld16(lane_addr + 256 + c, h);
                dg::tmem_ld16(lane_addr + 384 + c, l);
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                if (row_live) {
#pragma unroll
                    for (int k = 0; k < 16; ++k) {
                        int64_t num = (int64_t)h[k] * 256 + l[k];
                        if (flushed) num += (int64_t)carry[(c + k) * TILE_ROWS + r] << 32;
                        h[k] = total ? out_code(num, inv) : 0;
                    }
                    if (a.vec_o) {
#pragma unroll
                        for (int k = 0; k < 16; k += 4) *(int4*)(out + c + k) = make_int4(h[k], h[k + 1], h[k + 2], h[k + 3]);
                    } else {
#pragma unroll
                        for (int k = 0; k < 16; ++k) out[c + k] = h[k];
                    }
                }
            }
            asm volatile("tcgen05.fence::before_thread_sync;");
            __syncwarp();
            if (lane == 0) mbar_arrive(o_free);
        }
        if (!met) asm volatile("bar.sync 1, 512;" ::: "memory");  // a wait failed: the other warps still meet here
        if (n_pass == 0 && row_live && grp == 0 && part == 0) {  // no row of the tile sees anything
            int32_t* out = a.o + ((long long)begin + t) * a.ld_o + (long long)(head * g + (row0 + r) % g) * dim;
            for (int k = 0; k < dim; ++k) out[k] = 0;
        }
        if (row_live && grp == 0 && part == 0 && (row0 + r) % g == 0)
            a.o_scale[((long long)begin + t) * a.c.heads + head] =
                total ? make_longlong2(1, (long long)(uint32_t)(21 - e_row)) : make_longlong2(0, 0);
    }
    asm volatile("tcgen05.fence::before_thread_sync;");
    __syncthreads();
    if (warp == 0) {
        asm volatile("tcgen05.fence::after_thread_sync;");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
    }
}

}  // namespace kv
