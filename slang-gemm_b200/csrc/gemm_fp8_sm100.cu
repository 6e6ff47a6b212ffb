// gemm_fp8_sm100.cu -- FP8 matrix products with one f32 scale per 128 elements
// along K (or per 128 x 128 block), dense and over ragged groups, for sm_100a.
//
//   C[i, j] = alpha * sum_b sA(i, b) * sB(j, b) * S_b[i, j] + beta * C[i, j],
//   S_b[i, j] = sum over the 128 K elements of block b of op(A)[i, p] * op(B)[p, j]
//
// The scales are arbitrary f32 numbers, so they cannot be folded into the
// tensor core's accumulation over K: each block's S_b is computed by four
// tcgen05.mma (kind::f8f6f4, K = 32) into a TMEM slot of its own, and the
// epilogue warps ("promoters") read the slot and add scale * S_b to f32 sums
// in registers with packed FMAs while the tensor core fills the next slot.
// Products of two FP8 values are exact in f32 and a block sums 128 of them.
//
// A tile is P rows (TMEM lanes, one per promoter thread) by Q columns. Two
// orientations:
//  - wide tiles (BN = 256): P = op(B)'s columns (tokens), Q = op(A)'s rows
//    (features). With tokens scaled per vector and weights per block a thread's
//    scale of a K block is one number, and a thread's row of C is contiguous, so
//    C leaves through 128-byte swizzled staging and TMA stores. CTA pairs
//    (cta_group::2) compute 256 x 256.
//  - narrow tiles (BN = 32, 64, 128; few tokens, bound by reading A): P = op(A)'s
//    rows, Q = op(B)'s columns, so no row of the tensor core is spent on
//    tokens that are not there; 32 lanes store 32 consecutive rows of C.
// A scale per Q column is the same for all lanes: it is read from shared memory
// as a broadcast, and costs one more packed multiply.
//
// One CTA (or CTA pair) per SM runs tiles persistently:
//  - warp 0: TMA producer, 128 x 128 bytes of P and BN / CG x 128 of Q a stage;
//    transposes live in the tensor maps and the UMMA major bits;
//  - warp 1: TMEM allocation, and tcgen05.mma from one thread (even CTA);
//  - warp 2: copies each K block's scales into a ring in shared memory with
//    cp.async, which completes on the ring's mbarriers;
//  - warps 4..: promoters, BN / (warps / 4) columns each. With 128 columns a
//    thread they need more registers than an even split gives: of the 3 x 168 a
//    lane triple is launched with, the first warpgroup hands 96 or 112 to the
//    two promoter warpgroups (72 / 216 / 216, or 56 / 224 / 224 where the
//    scale warp copies no vector of Q).
// Ragged groups: offsets are read from device memory; tile counts are scanned
// once per CTA into shared memory and each tile finds its group by bisection.
//
// Split-K (few tiles, long K): the CTAs of a cluster take K slices of one tile
// and sum their f32 results in rank order through distributed shared memory,
// so there is no workspace and the result does not depend on timing.
//
// Bounds. Wide tiles: the promoters and the two slots' handshake, 776 cycles a K
// block with a scale per row and block, 1358 with one per row and column, for 512
// of tensor core, and about 4000 cycles a tile in which the promoters store C and
// the tensor core waits; 8192^3 to bf16 takes 561 to 577 us in repeated calls (1910
// to 1960 TFLOP/s; the clock falls to 1.5 GHz), 480 to 490 in a short run. Narrow
// tiles: reading A; 64 groups of 2048 x 2048 with two rows each on average, 44 of
// them not empty, take 39 to 41 us (185 MB, 4.6 TB/s; 704 tiles on 148 SMs are 4.8
// rounds), 4096 x 16 x 4096 7.2 us, of which 2.6 would be the bytes and the rest is
// launch, first loads and the reduction.
#include <type_traits>

#include "gs_epilogue.cuh"
#include "gs_float.cuh"
#include "gs_fp8.h"
#include "gs_internal.h"
#include "gs_ptx.cuh"

namespace gs {
namespace fp8 {

constexpr int BM = 128;
constexpr int BK = 128;
constexpr int SC_STAGES = 8;
constexpr int MAX_SPLIT = 8;  // portable cluster size

template <int CG, int BN>
struct Cfg {
    static constexpr bool WIDE = BN == 256;  // P = B's columns, Q = A's rows
    static constexpr int EPI_WARPS = BN >= 128 ? 8 : 4;
    static constexpr int EPI_COLS = BN / (EPI_WARPS / 4);
    static constexpr int THREADS = 128 + 32 * EPI_WARPS;
    static constexpr int Q_ROWS = BN / CG;
    static constexpr int P_STAGE = BM * BK;
    static constexpr int Q_STAGE = Q_ROWS * BK;
    static constexpr int STAGE = P_STAGE + Q_STAGE;
    static constexpr int STAGES = WIDE ? 4 : (STAGE >= 32 * 1024 ? 6 : 8);
    static_assert(!WIDE || CG == 2, "the wide tile is a CTA-pair tile");
    static constexpr int STG_BLOCK = 32 * 128;  // a promoter warp's staging: 32 rows of 128 bytes
    static constexpr int STG_BYTES = WIDE ? 2 * EPI_WARPS * STG_BLOCK : 0;  // two to a warp
    static constexpr int SLOTS = BN == 256 ? 2 : 4;
    static constexpr int TMEM_COLS = BN * SLOTS;
    static constexpr int SC_FLOATS = BN + BM;
    static constexpr int TILE_P = BM * CG;
    static constexpr int BARS = 2 * STAGES + 2 * SLOTS + 2 * SC_STAGES + 1;
    static constexpr int SMEM = STAGES * STAGE + STG_BYTES + SC_STAGES * SC_FLOATS * 4 + BARS * 8 + 16 + 1024 /*alignment*/;
};

// One operand as the kernel sees it: `extent` rows (P) or columns (Q) besides K.
struct Side {
    int extent;
    int mn;                    // stored with the non-K axis contiguous
    int grouped;               // the tensor map's third coordinate is the group
    const float *scale;
    long long s_i, s_k, s_g;   // element strides: index (or its block of 128), K block, group
};

struct Args {
    Side p, q;
    int k;
    int p_blocks, q_blocks, k_blocks;  // tiles along each axis (of the ragged one: unused)
    int groups;                        // 0 = dense
    int ragged;                        // GS_GROUP_N / GS_GROUP_K, -1 = dense
    const int32_t *offsets;
    int split;                         // cluster CTAs sharing a tile's K blocks (1 = none)
    uint32_t total_tiles;              // dense and ragged K
    uint32_t idesc;
    void *C;
    long long ldc, stride_c;
    int out_kind;
    int tma_store;                     // C can be written through tmC
    int whole_c;                       // C's rows end on 16 bytes
    int vec_c;                         // C's rows can be read and written 16 bytes at a time
    Epilogue ep;
    uint32_t *err;
    long long spin_limit;
    int debug_skip_kb;                 // test hook (>= 0): the producer leaves this K block of its first tile out, then stops
};

// A tile of group g: rows p0.. (p_end: behind the last), columns q0.., K blocks kb0..kb0+nkb.
struct Item {
    int g, p0, p_end, q0, q_end, kb0, nkb;
    bool bad;  // ragged-K group whose offsets are not multiples of 128
};

constexpr int RASTER = 8;  // rows of tiles visited together, so that concurrent tiles share operands in L2

template <int CG, int BN>
__device__ __forceinline__ bool item_at(const Args &a, const int *tile_start, const int *off, uint32_t t, uint32_t rank,
                                        Item &it) {
    using C_ = Cfg<CG, BN>;
    int p_blocks = a.p_blocks, q_blocks = a.q_blocks, p_base = 0, q_base = 0;
    uint32_t r = t;
    it.g = 0;
    it.bad = false;
    it.kb0 = 0;
    it.nkb = a.k_blocks;
    it.p_end = a.p.extent;
    it.q_end = a.q.extent;
    if (a.ragged == GS_GROUP_N) {
        if (t >= static_cast<uint32_t>(tile_start[a.groups])) return false;
        int lo = 0, hi = a.groups;  // the last group whose first tile is <= t
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (static_cast<uint32_t>(tile_start[mid]) <= t) lo = mid;
            else hi = mid;
        }
        it.g = lo;
        r = t - static_cast<uint32_t>(tile_start[lo]);
        if (C_::WIDE) {
            p_base = off[lo];
            it.p_end = off[lo + 1];
            p_blocks = (it.p_end - p_base + C_::TILE_P - 1) / C_::TILE_P;
        } else {
            q_base = off[lo];
            it.q_end = off[lo + 1];
            q_blocks = (it.q_end - q_base + BN - 1) / BN;
        }
    } else {
        if (t >= a.total_tiles) return false;
        if (a.ragged == GS_GROUP_K) {
            const uint32_t per = static_cast<uint32_t>(p_blocks) * static_cast<uint32_t>(q_blocks), g = t / per;
            it.g = static_cast<int>(g);
            r = t - g * per;
            const int k_lo = off[it.g], k_hi = off[it.g + 1];
            it.kb0 = k_lo / BK;
            it.nkb = (k_hi - k_lo + BK - 1) / BK;
            it.bad = k_hi > k_lo && (k_lo % BK != 0 || (k_hi % BK != 0 && k_hi != a.k));
            if (it.bad) it.nkb = 0;
        }
    }
    // Tile counts fit 32 bits (checked on entry): every warp of a role works this out for every tile, and 64-bit
    // divisions here cost the promoters a microsecond a tile.
    const int height = p_blocks < RASTER ? p_blocks : RASTER;
    const uint32_t span = static_cast<uint32_t>(height) * static_cast<uint32_t>(q_blocks), gi = r / span;
    const int within = static_cast<int>(r - gi * span);
    const int first = static_cast<int>(gi) * height;
    const int rows = min(height, p_blocks - first);
    const int column = within / rows;
    it.p0 = p_base + (first + within - column * rows) * C_::TILE_P + static_cast<int>(CG == 2 ? rank : 0) * BM;
    it.q0 = q_base + column * BN;
    if (CG == 1 && a.split > 1) {  // this CTA's share of the K blocks
        const int lo = it.nkb * static_cast<int>(rank) / a.split, hi = it.nkb * static_cast<int>(rank + 1) / a.split;
        it.kb0 += lo;
        it.nkb = hi - lo;
    }
    return true;
}

__device__ __forceinline__ uint64_t pack2(float x, float y) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float &x, float &y) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

// True in one lane of a converged warp.
__device__ __forceinline__ uint32_t elect_one() {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}\n" : "=r"(r));
    return r;
}

// The MMA and its commits, executed by the whole warp and issued by the lane with `lead` set: with uniform control flow
// the descriptors stay in uniform registers, where the instruction wants them.
template <int CG>
__device__ __forceinline__ void umma_f8(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate,
                                        uint32_t lead) {
    if constexpr (CG == 2) {
        asm volatile(
            "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
            "@q tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d_tmem), "l"(adesc), "l"(bdesc),
            "r"(idesc), "r"(accumulate), "r"(lead)
            : "memory");
    } else {
        asm volatile(
            "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
            "@q tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d_tmem), "l"(adesc), "l"(bdesc),
            "r"(idesc), "r"(accumulate), "r"(lead)
            : "memory");
    }
}
template <int CG>
__device__ __forceinline__ void umma_commit_lead(uint64_t *bar, uint32_t lead) {
    if constexpr (CG == 2) {
        asm volatile(
            "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %2, 0;\n\t"
            "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n\t}\n" ::"r"(
                smem_u32(bar)),
            "h"(static_cast<uint16_t>(3)), "r"(lead)
            : "memory");
    } else {
        asm volatile(
            "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
            "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}\n" ::"r"(smem_u32(bar)),
            "r"(lead)
            : "memory");
    }
}

__device__ __forceinline__ void st_shared_f32(uint32_t addr, float v) {
    asm volatile("st.shared.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}
// Volatile, so that the compiler keeps each load next to its use: hoisted, they would cost the sums their registers.
__device__ __forceinline__ float4 ld_shared_f32x4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr));
    return v;
}
__device__ __forceinline__ float4 ld_cluster_f32x4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(addr)
                 : "memory");
    return v;
}

// Waits for two barriers, both polled once before either is waited for: a poll's latency is paid once.
__device__ __forceinline__ bool mbar_wait2(uint64_t *b1, uint32_t parity1, uint32_t site1, uint64_t *b2, uint32_t parity2,
                                           uint32_t site2, uint32_t *err, long long limit) {
    const bool r1 = mbar_try_wait(smem_u32(b1), parity1), r2 = mbar_try_wait(smem_u32(b2), parity2);
    if (r1 && r2) return true;
    return (r1 || mbar_wait(b1, parity1, err, site1, limit)) && (r2 || mbar_wait(b2, parity2, err, site2, limit));
}

// 4-byte asynchronous copy global -> shared.
__device__ __forceinline__ void cp_async_f32(uint32_t dst, const float *src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
// Arrives on the barrier when this thread's earlier cp.async have completed.
__device__ __forceinline__ void cp_async_arrive(uint64_t *bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }

__device__ __forceinline__ void st_shared_v4(uint32_t addr, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}

// One element of C, rounded once from f32 (to nearest even).
template <typename T>
__device__ __forceinline__ void store_one(const Args &a, T *c, float v) {
    if (!a.ep.beta_zero) v = __fmaf_rn(a.ep.beta_f, to_f32(*c), v);
    *c = from_f32<T>(v);
}
__device__ __forceinline__ float scaled(const Args &a, float acc) { return a.ep.identity ? acc : __fmul_rn(a.ep.alpha_f, acc); }
__device__ __forceinline__ void store_c(const Args &a, void *C, size_t i, float acc) {
    const float v = scaled(a, acc);
    if (a.out_kind == OUT_F32) store_one(a, static_cast<float *>(C) + i, v);
    else if (a.out_kind == OUT_F16) store_one(a, static_cast<__half *>(C) + i, v);
    else store_one(a, static_cast<__nv_bfloat16 *>(C) + i, v);
}
// C of group g (ragged K).
__device__ __forceinline__ void *group_c(const Args &a, int g) {
    if (a.ragged != GS_GROUP_K) return a.C;
    return static_cast<uint8_t *>(a.C) + static_cast<size_t>(g) * a.stride_c * (a.out_kind == OUT_F32 ? 4 : 2);
}

// 128 consecutive elements of one row of C from a thread's sums (alpha applied), `n` of them inside.
template <typename T>
__device__ __forceinline__ void store_row(const Args &a, T *c, int n, const uint64_t (&acc)[64]) {
#pragma unroll
    for (int j = 0; j < 128; j += 8) {
        float v[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) unpack2(acc[j / 2 + i], v[2 * i], v[2 * i + 1]);
        if (a.vec_c && j + 8 <= n) {
            Pack<T, 8> out;
            if (!a.ep.beta_zero) {
                const Pack<T, 8> old = load_pack<T, 8>(c + j);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = __fmaf_rn(a.ep.beta_f, to_f32(old.v[i]), v[i]);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) out.v[i] = from_f32<T>(v[i]);
            store_pack<T, 8>(c + j, out);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (j + i < n) store_one(a, c + j + i, v[i]);
        }
    }
}

// A narrow tile's thread: N columns of one row of C, ldc apart (32 lanes store 32 consecutive rows); n of them inside.
// Type and beta are settled outside the loop: decided per element they made this 25 instructions a column, 6.8 us a
// 128 x 128 tile.
template <typename T, int N>
__device__ __forceinline__ void store_columns(const Args &a, T *c, int n, const uint64_t (&acc)[N / 2]) {
    const float alpha = a.ep.alpha_f;
    if (a.ep.beta_zero) {
#pragma unroll
        for (int j = 0; j < N; j += 2) {
            float x, y;
            unpack2(acc[j / 2], x, y);
            if (j < n) *c = from_f32<T>(__fmul_rn(alpha, x));
            c += a.ldc;
            if (j + 1 < n) *c = from_f32<T>(__fmul_rn(alpha, y));
            c += a.ldc;
        }
    } else {
#pragma unroll
        for (int j = 0; j < N; j += 2) {
            float x, y;
            unpack2(acc[j / 2], x, y);
            if (j < n) store_one(a, c, __fmul_rn(alpha, x));
            c += a.ldc;
            if (j + 1 < n) store_one(a, c, __fmul_rn(alpha, y));
            c += a.ldc;
        }
    }
}

// MODE bit 0: P has a scale per row (else per 128 rows); bit 1: Q has a scale
// per column (else per 128 columns).
template <int CG, int BN, int MODE>
__global__ void __launch_bounds__(Cfg<CG, BN>::THREADS, 1)
    k_gemm_fp8(const __grid_constant__ CUtensorMap tmP, const __grid_constant__ CUtensorMap tmQ,
               const __grid_constant__ CUtensorMap tmC, const Args args) {
    using C_ = Cfg<CG, BN>;
    constexpr bool P_VEC = (MODE & 1) != 0, Q_VEC = (MODE & 2) != 0;
    constexpr int STAGES = C_::STAGES, SLOTS = C_::SLOTS, EPI_COLS = C_::EPI_COLS;

    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *smP = smem;
    uint8_t *smQ = smem + STAGES * C_::P_STAGE;
    uint8_t *stg = smQ + STAGES * C_::Q_STAGE;
    float *scales = reinterpret_cast<float *>(stg + C_::STG_BYTES);
    uint64_t *full = reinterpret_cast<uint64_t *>(scales + SC_STAGES * C_::SC_FLOATS);
    uint64_t *empty = full + STAGES;
    uint64_t *tfull = empty + STAGES;
    uint64_t *tempty = tfull + SLOTS;
    uint64_t *sfull = tempty + SLOTS;
    uint64_t *sempty = sfull + SC_STAGES;
    uint64_t *drain = sempty + SC_STAGES;
    uint32_t *tmem_holder = reinterpret_cast<uint32_t *>(drain + 1);
    int *off = reinterpret_cast<int *>(tmem_holder + 2);   // groups + 1 clamped offsets, then groups + 1 first tiles
    int *tile_start = off + args.groups + 1;

    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);  // uniform for the compiler too
    const int lane = threadIdx.x & 31;
    const bool clustered = CG == 2 || args.split > 1;
    const uint32_t rank = clustered ? cluster_ctarank() : 0u;
    const bool leader = CG == 1 || rank == 0;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int i = 0; i < SLOTS; ++i) {
            mbar_init(&tfull[i], 1);
            mbar_init(&tempty[i], CG * C_::EPI_WARPS);
        }
        for (int i = 0; i < SC_STAGES; ++i) {
            mbar_init(&sfull[i], 32);
            mbar_init(&sempty[i], C_::EPI_WARPS);
        }
        mbar_init(drain, 1);
        fence_barrier_init();
    }
    if (warp == 0 && lane == 0 && args.k_blocks > 0) {
        prefetch_tensormap(&tmP);
        prefetch_tensormap(&tmQ);
    }
    if (warp == 1) {
        if constexpr (CG == 2) {
            tmem_alloc_2sm(tmem_holder, C_::TMEM_COLS);
            tmem_relinquish_2sm();
        } else {
            tmem_alloc(tmem_holder, C_::TMEM_COLS);
            tmem_relinquish();
        }
    }
    grid_dep_wait();
    if (warp == 2 && args.groups > 0) {
        // Clamped, never decreasing offsets (whatever the caller's memory holds, every access stays inside the
        // operands) and, for ragged N, the running count of tiles.
        const int limit = args.ragged == GS_GROUP_K ? args.k : C_::WIDE ? args.p.extent : args.q.extent;
        const int per = (args.groups + 32) / 32;  // of groups + 1 offsets
        const int lo = min(lane * per, args.groups + 1), hi = min(lo + per, args.groups + 1);
        int top = 0;
        for (int i = lo; i < hi; ++i) {
            top = max(top, min(args.offsets[i], limit));
            off[i] = top;
        }
        int before = top;  // running maximum over lanes
        for (int d = 1; d < 32; d <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, before, d);
            if (lane >= d) before = max(before, v);
        }
        before = __shfl_up_sync(0xffffffffu, before, 1);
        if (lane == 0) before = 0;
        for (int i = lo; i < hi; ++i) off[i] = max(off[i], before);
        __syncwarp();
        if (args.ragged == GS_GROUP_N) {
            constexpr int TILE = C_::WIDE ? C_::TILE_P : BN;
            const int across = C_::WIDE ? args.q_blocks : args.p_blocks;
            int sum = 0;
            for (int i = lo; i < hi; ++i) {
                tile_start[i] = sum;
                if (i < args.groups) sum += (off[i + 1] - off[i] + TILE - 1) / TILE * across;
            }
            int incl = sum;
            for (int d = 1; d < 32; d <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, incl, d);
                if (lane >= d) incl += v;
            }
            for (int i = lo; i < hi; ++i) tile_start[i] += incl - sum;
        }
    }
    tc_fence_before();
    __syncthreads();
    if constexpr (CG == 2) cluster_sync();
    tc_fence_after();
    grid_dep_launch();  // after this CTA has its TMEM: a dependent kernel's CTA cannot take it first
    const uint32_t tmem_base = *tmem_holder;

    const uint32_t tile0 = blockIdx.x / (CG * (CG == 1 ? args.split : 1));
    const uint32_t tile_step = gridDim.x / (CG * (CG == 1 ? args.split : 1));
    Item it;

    if (warp < 4) {
    if constexpr (EPI_COLS == 128) {
        if constexpr (Q_VEC) asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        else asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    }
    if (warp == 0) {
        // ---------------- TMA producer ----------------
        if (lane == 0) {
            const uint64_t pol = l2_policy_evict_normal();
            int stage = 0;
            uint32_t phase = 0, issued = 0;
            bool ok = true;
            for (uint32_t t = tile0; ok && item_at<CG, BN>(args, tile_start, off, t, rank, it); t += tile_step) {
                const int qc = it.q0 + static_cast<int>(CG == 2 ? rank : 0) * C_::Q_ROWS;
                const int gp = args.p.grouped ? it.g : 0, gq = args.q.grouped ? it.g : 0;
                for (int kb = 0; kb < it.nkb; ++kb) {
                    if (kb == args.debug_skip_kb && t == tile0) { ok = false; break; }
                    if (!mbar_wait(&empty[stage], phase ^ 1u, args.err, 1, args.spin_limit)) { ok = false; break; }
                    uint8_t *dP = smP + stage * C_::P_STAGE;
                    uint8_t *dQ = smQ + stage * C_::Q_STAGE;
                    const int k0 = (it.kb0 + kb) * BK;
                    if constexpr (CG == 2) {
                        const uint32_t fbar = mapa_shared(smem_u32(&full[stage]), 0);
                        if (leader) mbar_arrive_expect_tx(&full[stage], 2 * C_::STAGE);
                        if (args.p.mn) tma_load_3d_2sm(dP, &tmP, fbar, it.p0, k0, gp, pol);
                        else tma_load_3d_2sm(dP, &tmP, fbar, k0, it.p0, gp, pol);
                        if (args.q.mn) tma_load_3d_2sm(dQ, &tmQ, fbar, qc, k0, gq, pol);
                        else tma_load_3d_2sm(dQ, &tmQ, fbar, k0, qc, gq, pol);
                    } else {
                        mbar_arrive_expect_tx(&full[stage], C_::STAGE);
                        if (args.p.mn) tma_load_3d_hint(dP, &tmP, &full[stage], it.p0, k0, gp, pol);
                        else tma_load_3d_hint(dP, &tmP, &full[stage], k0, it.p0, gp, pol);
                        if (args.q.mn) tma_load_3d_hint(dQ, &tmQ, &full[stage], qc, k0, gq, pol);  // only with BN = 128
                        else tma_load_3d_hint(dQ, &tmQ, &full[stage], k0, qc, gq, pol);
                    }
                    ++issued;
                    if (++stage == STAGES) { stage = 0; phase ^= 1u; }
                }
            }
            // Giving up: the copies still in flight (a pair's: both CTAs' complete on the even one's barriers) land before
            // the CTA goes.
            if (!ok && leader)
                for (uint32_t i = issued > STAGES ? issued - STAGES : 0; i < issued; ++i)
                    mbar_wait(&full[i % STAGES], (i / STAGES) & 1u, args.err, 8, args.spin_limit);
        }
    } else if (warp == 1) {
        // ---------------- MMA issuer (even CTA) ----------------
        if (leader) {
            // Descriptors of stage 0; a stage and a K step of 32 only move the address field. The issue loop is a chain of
            // dependent instructions on a scheduler that two promoters share: with descriptors built in it by one lane
            // it, and not the tensor core, set the pace (815 cycles a K block without promoters for 512 of MMA).
            uint64_t pdesc = umma_smem_desc_sw128(smem_u32(smP), args.p.mn ? 128 * BK : 16, 1024);
            uint64_t qdesc = umma_smem_desc_sw128(smem_u32(smQ), args.q.mn ? 128 * BK : 16, 1024);
            const uint32_t p_step = (args.p.mn ? 32 * 128 : 32) >> 4, q_step = (args.q.mn ? 32 * 128 : 32) >> 4;
            const uint32_t lead = elect_one();
            int stage = 0, slot = 0;
            uint32_t phase = 0, sphase = 0;
            bool ok = true;
            for (uint32_t t = tile0; ok && item_at<CG, BN>(args, tile_start, off, t, rank, it); t += tile_step) {
#pragma unroll 1
                for (int kb = 0; kb < it.nkb; ++kb) {
                    if (!__all_sync(0xffffffffu, mbar_wait2(&tempty[slot], sphase ^ 1u, 2, &full[stage], phase, 3, args.err,
                                                            args.spin_limit))) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t d_tmem = tmem_base + slot * BN;
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk)
                        umma_f8<CG>(d_tmem, pdesc + kk * p_step, qdesc + kk * q_step, args.idesc, kk != 0 ? 1u : 0u, lead);
                    umma_commit_lead<CG>(&tfull[slot], lead);
                    umma_commit_lead<CG>(&empty[stage], lead);
                    pdesc += C_::P_STAGE >> 4;
                    qdesc += C_::Q_STAGE >> 4;
                    if (++stage == STAGES) {
                        stage = 0;
                        phase ^= 1u;
                        pdesc -= STAGES * C_::P_STAGE >> 4;
                        qdesc -= STAGES * C_::Q_STAGE >> 4;
                    }
                    if (++slot == SLOTS) { slot = 0; sphase ^= 1u; }
                }
            }
            if (!ok) {  // the MMAs already issued end before the CTA frees its TMEM
                umma_commit_lead<CG>(drain, lead);
                mbar_wait(drain, 0, args.err, 5, args.spin_limit);
            }
        }
    } else if (warp == 2) {
        // ---------------- scales: [BN] of Q (per column, or one per 128), then [128] (or one) of P ----------------
        int ss = 0;
        uint32_t sp = 0;
        bool ok = true;
        for (uint32_t t = tile0; ok && item_at<CG, BN>(args, tile_start, off, t, rank, it); t += tile_step) {
            // This lane's first scale of either side (a scale per vector has its non-K index contiguous), and which of its
            // copies lie inside. What is not copied scales rows and columns that are not stored.
            constexpr int NP = P_VEC ? BM / 32 : 1, NQ = Q_VEC ? BN / 32 : 1;
            const int pi = P_VEC ? it.p0 + lane : it.p0 / 128, qi = Q_VEC ? it.q0 + lane : it.q0 / 128 + lane;
            const float *pp = args.p.scale + it.g * args.p.s_g + pi * args.p.s_i + it.kb0 * args.p.s_k;
            const float *pq = args.q.scale + it.g * args.q.s_g + qi * args.q.s_i + it.kb0 * args.q.s_k;
            const int np = P_VEC ? (it.p_end - pi + 31) / 32 : (lane == 0 && it.p0 < it.p_end ? 1 : 0);
            const int nq = Q_VEC ? (it.q_end - qi + 31) / 32 : (lane < (BN + 127) / 128 && it.q0 + lane * 128 < it.q_end ? 1 : 0);
            for (int kb = 0; kb < it.nkb; ++kb) {
                // one answer for the warp: its lanes arrive together
                if (!__all_sync(0xffffffffu, mbar_wait(&sempty[ss], sp ^ 1u, args.err, 6, args.spin_limit))) {
                    ok = false;
                    break;
                }
                const uint32_t dst = smem_u32(scales + ss * C_::SC_FLOATS) + lane * 4;
#pragma unroll
                for (int i = 0; i < NQ; ++i)
                    if (i < nq) cp_async_f32(dst + i * 128, pq + i * 32);
#pragma unroll
                for (int i = 0; i < NP; ++i)
                    if (i < np) cp_async_f32(dst + BN * 4 + i * 128, pp + i * 32);
                cp_async_arrive(&sfull[ss]);
                pp += args.p.s_k;
                pq += args.q.s_k;
                if (++ss == SC_STAGES) { ss = 0; sp ^= 1u; }
            }
        }
        cp_async_wait_all();
    }
    } else {
        // ---------------- promoters ----------------
        if constexpr (EPI_COLS == 128) {
            if constexpr (Q_VEC) asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
            else asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
        }
        const int quad = warp & 3;
        const int ew = warp - 4;
        const int c_lo = (ew / 4) * EPI_COLS;
        const int row = quad * 32 + lane;
        const uint32_t t_lane = tmem_base + (static_cast<uint32_t>(quad * 32) << 16);
        const uint32_t tempty_leader = CG == 2 ? mapa_shared(smem_u32(&tempty[0]), 0) : 0u;
        const uint64_t pol_c = l2_policy_evict_first();
        int slot = 0, ss = 0;
        uint32_t phase = 0, sp = 0;
        bool ok = true;
        for (uint32_t t = tile0; ok && item_at<CG, BN>(args, tile_start, off, t, rank, it); t += tile_step) {
            if (it.bad) {
                if (ew == 0 && lane == 0) atomicOr(args.err, GS_DEVERR_OFFSETS);
                continue;
            }
            uint64_t acc[EPI_COLS / 2];
#pragma unroll
            for (int j = 0; j < EPI_COLS / 2; ++j) acc[j] = 0;
#pragma unroll 1
            for (int kb = 0; kb < it.nkb; ++kb) {
                // every lane takes the same way out (tcgen05.ld is warp-aligned)
                if (!__all_sync(0xffffffffu, mbar_wait2(&sfull[ss], sp, 7, &tfull[slot], phase, 4, args.err, args.spin_limit))) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                // The next 32 columns are on their way while these are added (16 at a time: 849 instead of 774 cycles a K
                // block of a wide tile).
                const uint32_t t_slot = t_lane + slot * BN + c_lo;
                uint32_t r[2][32];
                tmem_ld_32x32b_x32(t_slot, r[0]);
                const float *sc = scales + ss * C_::SC_FLOATS;
                const uint32_t sc_addr = smem_u32(sc + c_lo);
                float s = sc[BN + (P_VEC ? row : 0)];
                if constexpr (!Q_VEC) s = __fmul_rn(s, sc[c_lo / 128]);
                const uint64_t s2 = pack2(s, s);
#pragma unroll
                for (int c = 0; c < EPI_COLS; c += 32) {
                    const int cur = (c / 32) & 1;
                    tmem_wait_ld();
                    if (c + 32 < EPI_COLS) {
                        tmem_ld_32x32b_x32(t_slot + c + 32, r[cur ^ 1]);
                    } else {  // the slot is read: the tensor core may fill it again
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) {
                            if constexpr (CG == 2) mbar_arrive_cluster(tempty_leader + slot * sizeof(uint64_t));
                            else mbar_arrive(&tempty[slot]);
                        }
                    }
#pragma unroll
                    for (int j = 0; j < 32; j += 4) {
                        const uint64_t p0 = pack2(__uint_as_float(r[cur][j]), __uint_as_float(r[cur][j + 1]));
                        const uint64_t p1 = pack2(__uint_as_float(r[cur][j + 2]), __uint_as_float(r[cur][j + 3]));
                        uint64_t &a0 = acc[(c + j) / 2], &a1 = acc[(c + j) / 2 + 1];
                        if constexpr (Q_VEC) {
                            const float4 s4 = ld_shared_f32x4(sc_addr + (c + j) * 4);
                            a0 = fma2(mul2(p0, s2), pack2(s4.x, s4.y), a0);
                            a1 = fma2(mul2(p1, s2), pack2(s4.z, s4.w), a1);
                        } else {
                            a0 = fma2(p0, s2, a0);
                            a1 = fma2(p1, s2, a1);
                        }
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&sempty[ss]);
                if (++slot == SLOTS) { slot = 0; phase ^= 1u; }
                if (++ss == SC_STAGES) { ss = 0; sp ^= 1u; }
            }
            if (!ok) break;
            if constexpr (C_::WIDE) {
                // Row p of C is contiguous. Whole warps go out through staging: 32 rows of 128 bytes, 16-byte chunks
                // swizzled by the row so that neither side has bank conflicts; rows past a ragged group's end
                // belong to the next group, which a TMA store would overwrite.
                const int n = it.q_end - it.q0 - c_lo;
                const int p = it.p0 + row, p_warp = it.p0 + quad * 32;
                if (!args.ep.identity) {
                    const uint64_t al = pack2(args.ep.alpha_f, args.ep.alpha_f);
#pragma unroll
                    for (int j = 0; j < 64; ++j) acc[j] = mul2(acc[j], al);
                }
                // A TMA store stops at the tensor's end only to the next 16 bytes: what lies behind a row that ends
                // between them would be overwritten, so such an end is stored directly.
                if (args.tma_store && (args.whole_c || n >= 128) && (args.ragged != GS_GROUP_N || p_warp + 32 <= it.p_end)) {
                    const int gc = args.ragged == GS_GROUP_K ? it.g : 0;
                    // `words` packs the 16 bytes of chunk x of block b
                    auto blocks = [&](auto cols_c, auto words) {
                        constexpr int COLS = decltype(cols_c)::value;  // columns of 128 bytes
#pragma unroll
                        for (int b = 0; b < 128 / COLS; ++b) {
                            if (b * COLS >= n || p_warp >= it.p_end) break;
                            // The store that last used this buffer has read it: the one before the last within a tile, any
                            // of the tile before (a part tile's stores may be odd in number, and end on either buffer).
                            if (lane == 0) {
                                if (b == 0) bulk_wait_group_read<0>();
                                else bulk_wait_group_read<1>();
                            }
                            uint8_t *buf = stg + (ew * 2 + (b & 1)) * C_::STG_BLOCK;
                            const uint32_t dst = smem_u32(buf) + lane * 128;
                            __syncwarp();
#pragma unroll
                            for (int x = 0; x < 8; ++x) {
                                uint32_t w[4];
                                words(b * COLS + x * (COLS / 8), w);
                                st_shared_v4(dst + ((x ^ (lane & 7)) << 4), w[0], w[1], w[2], w[3]);
                            }
                            fence_proxy_async();
                            __syncwarp();
                            if (lane == 0) {
                                tma_store_3d(&tmC, buf, it.q0 + c_lo + b * COLS, p_warp, gc, pol_c);
                                bulk_commit_group();
                            }
                        }
                    };
                    if (args.out_kind == OUT_F32) {
                        blocks(std::integral_constant<int, 32>{}, [&](int j, uint32_t (&w)[4]) {
#pragma unroll
                            for (int i = 0; i < 2; ++i) {
                                float x, y;
                                unpack2(acc[j / 2 + i], x, y);
                                w[2 * i] = __float_as_uint(x);
                                w[2 * i + 1] = __float_as_uint(y);
                            }
                        });
                    } else {
                        const bool half = args.out_kind == OUT_F16;
                        blocks(std::integral_constant<int, 64>{}, [&](int j, uint32_t (&w)[4]) {
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                float x, y;
                                unpack2(acc[j / 2 + i], x, y);
                                if (half) {
                                    const __half2 h = __floats2half2_rn(x, y);
                                    w[i] = *reinterpret_cast<const uint32_t *>(&h);
                                } else {
                                    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
                                    w[i] = *reinterpret_cast<const uint32_t *>(&h);
                                }
                            }
                        });
                    }
                } else if (p < it.p_end && n > 0) {
                    void *Cb = group_c(args, it.g);
                    const size_t i = static_cast<size_t>(p) * args.ldc + it.q0 + c_lo;
                    if (args.out_kind == OUT_F32) store_row(args, static_cast<float *>(Cb) + i, n, acc);
                    else if (args.out_kind == OUT_F16) store_row(args, static_cast<__half *>(Cb) + i, n, acc);
                    else store_row(args, static_cast<__nv_bfloat16 *>(Cb) + i, n, acc);
                }
            } else {
                if (args.split > 1) {
                    // This slice's sums, column by column, over the operand stages: every load has landed and every
                    // MMA that read them has committed.
                    const uint32_t base = smem_u32(smem) + (c_lo * BM + row) * 4;
#pragma unroll
                    for (int j = 0; j < EPI_COLS / 2; ++j) {
                        float x, y;
                        unpack2(acc[j], x, y);
                        st_shared_f32(base + (2 * j) * BM * 4, x);
                        st_shared_f32(base + (2 * j + 1) * BM * 4, y);
                    }
                    break;  // one tile per cluster
                }
                const int p = it.p0 + row, n = it.q_end - it.q0 - c_lo;
                if (p < it.p_end && n > 0) {
                    void *Cb = group_c(args, it.g);
                    const size_t i = static_cast<size_t>(p) + static_cast<size_t>(it.q0 + c_lo) * args.ldc;
                    if (args.out_kind == OUT_F32) store_columns<float, EPI_COLS>(args, static_cast<float *>(Cb) + i, n, acc);
                    else if (args.out_kind == OUT_F16) store_columns<__half, EPI_COLS>(args, static_cast<__half *>(Cb) + i, n, acc);
                    else store_columns<__nv_bfloat16, EPI_COLS>(args, static_cast<__nv_bfloat16 *>(Cb) + i, n, acc);
                }
            }
        }
        if (C_::WIDE && lane == 0) bulk_wait_group_all();  // C is written before the kernel ends
    }

    __syncwarp();
    if (!C_::WIDE && args.split > 1) {
        cluster_sync();  // every slice's sums are in its CTA's shared memory
        if (item_at<CG, BN>(args, tile_start, off, tile0, rank, it) && !it.bad) {
            // The tile's columns inside C are shared out over the cluster; an element's slices are all on their way before
            // the first is added.
            const int inside = min(BN, it.q_end - it.q0), cols = (inside + args.split - 1) / args.split;
            const int first = static_cast<int>(rank) * cols, last = min(first + cols, inside);
            void *Cb = group_c(args, it.g);
            uint32_t base[MAX_SPLIT];
#pragma unroll
            for (int x = 0; x < MAX_SPLIT; ++x) base[x] = mapa_shared(smem_u32(smem), static_cast<uint32_t>(min(x, args.split - 1)));
            // Four consecutive rows a thread.
            for (int e = first * (BM / 4) + static_cast<int>(threadIdx.x); e < last * (BM / 4); e += C_::THREADS) {
                const int p = it.p0 + e % (BM / 4) * 4;
                if (p >= it.p_end) continue;
                float4 v[MAX_SPLIT];
#pragma unroll
                for (int x = 0; x < MAX_SPLIT; ++x) v[x] = x < args.split ? ld_cluster_f32x4(base[x] + e * 16) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                float4 sum = v[0];
#pragma unroll
                for (int x = 1; x < MAX_SPLIT; ++x) {
                    sum.x = __fadd_rn(sum.x, v[x].x);
                    sum.y = __fadd_rn(sum.y, v[x].y);
                    sum.z = __fadd_rn(sum.z, v[x].z);
                    sum.w = __fadd_rn(sum.w, v[x].w);
                }
                const size_t i = static_cast<size_t>(p) + static_cast<size_t>(it.q0 + e / (BM / 4)) * args.ldc;
                store_c(args, Cb, i, sum.x);
                if (p + 1 < it.p_end) store_c(args, Cb, i + 1, sum.y);
                if (p + 2 < it.p_end) store_c(args, Cb, i + 2, sum.z);
                if (p + 3 < it.p_end) store_c(args, Cb, i + 3, sum.w);
            }
        }
        __syncwarp();
    }
    tc_fence_before();
    __syncthreads();
    if (clustered) cluster_sync();  // no CTA leaves while a peer may signal its barriers or read its sums
    if (warp == 1) {
        __syncwarp();
        tc_fence_after();
        if constexpr (CG == 2) tmem_dealloc_2sm(tmem_base, C_::TMEM_COLS);
        else tmem_dealloc(tmem_base, C_::TMEM_COLS);
    }
}

struct Maps {
    CUtensorMap p, q, c;
};

// CTA pairs that can be resident at once.
template <int CG, int BN, int MODE>
static int max_pairs(Context &ctx, size_t smem) {
    static int cached[64] = {};  // per instantiation and device
    if (ctx.device >= 0 && ctx.device < 64 && cached[ctx.device] > 0) return cached[ctx.device];
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(2 * (ctx.sm_count / 2)), 1, 1);
    cfg.blockDim = dim3(Cfg<CG, BN>::THREADS, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = 2;
    attr.val.clusterDim.y = 1;
    attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, k_gemm_fp8<CG, BN, MODE>, &cfg) != cudaSuccess || n <= 0) {
        cudaGetLastError();
        n = ctx.sm_count / 2;
    }
    if (ctx.device >= 0 && ctx.device < 64) cached[ctx.device] = n;
    return n;
}

template <int CG, int BN, int MODE>
static cudaError_t launch(Context &ctx, const Maps &maps, const Args &a, long long tiles) {
    using C_ = Cfg<CG, BN>;
    auto kern = k_gemm_fp8<CG, BN, MODE>;
    constexpr size_t kMost = C_::SMEM + 2 * sizeof(int) * (GS_FP8_MAX_GROUPS + 1);
    static_assert(kMost <= 227 * 1024, "shared memory of one CTA");
    static bool attr_set[64] = {};  // per instantiation and device
    cudaError_t e = cudaSuccess;
    if (ctx.device < 0 || ctx.device >= 64 || !attr_set[ctx.device]) {
        e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kMost));
        if (e != cudaSuccess) return e;
        if (ctx.device >= 0 && ctx.device < 64) attr_set[ctx.device] = true;
    }
    const size_t smem = C_::SMEM + (a.groups > 0 ? 2 * sizeof(int) * (static_cast<size_t>(a.groups) + 1) : 0);
    const int cluster = CG == 2 ? 2 : a.split;
    long long units = CG == 2 ? max_pairs<CG, BN, MODE>(ctx, kMost) : ctx.sm_count;
    if (CG == 1 && a.split > 1) units = tiles;  // one tile per cluster
    if (tiles < units) units = tiles;
    e = launch_pdl(kern, dim3(static_cast<unsigned>(units * cluster)), dim3(C_::THREADS), smem, ctx.stream, cluster, maps.p, maps.q, maps.c, a);
    ctx.launches++;
    return e;
}

template <int CG, int BN>
static cudaError_t launch_mode(Context &ctx, int mode, const Maps &maps, const Args &a, long long tiles) {
    switch (mode) {
    case 0: return launch<CG, BN, 0>(ctx, maps, a, tiles);
    case 1: return launch<CG, BN, 1>(ctx, maps, a, tiles);
    case 2: return launch<CG, BN, 2>(ctx, maps, a, tiles);
    default: return launch<CG, BN, 3>(ctx, maps, a, tiles);
    }
}

static int cdiv(long long a, long long b) { return static_cast<int>((a + b - 1) / b); }

// C's rows can be moved 16 bytes at a time.
static bool aligned_c(const GemmFp8Desc &d) {
    const size_t es = out_elem_size(d.out_kind);
    const bool many = d.groups > 1 && d.ragged == GS_GROUP_K;
    return reinterpret_cast<uintptr_t>(d.C) % 16 == 0 && d.ldc * es % 16 == 0 && (!many || d.stride_c * es % 16 == 0);
}

// Tile of a product: bn columns, cg CTAs, split K slices. Each kind of tile is given the microseconds that its K blocks
// and the rest of it took in a sweep of 13 shapes from 512^3 to 8192^3, dense and ragged, alone on the GPU (a pair's 256 x 256
// tile 0.46 a K block, 0.82 with a scale per row and per column; 128 x 128, 64 and 32 tiles of one SM 0.41, 0.30 and
// 0.25); the cheapest rounds-times-tile wins. Against a rule on the column count alone: 1024^3 12.5 -> 6.9 us, 1024 x 1024 x 4096
// with both scales per vector 32 -> 17 us, 64 groups of 32 rows 82 -> 53 us.
// Narrow tiles that leave SMs without work may share their K blocks over a cluster, as long as all clusters run at once
// (4096 x 16 x 4096, 32 tiles as 128 CTAs: 11.7 -> 8.6 us; clusters of eight do not pack a GPU that is nearly full).
Tile choose_tile(const GemmFp8Desc &d, int sm_count) {
    const bool ragged_n = d.groups > 0 && d.ragged == GS_GROUP_N, ragged_k = d.groups > 0 && d.ragged == GS_GROUP_K;
    const double kb = ragged_k ? static_cast<double>(d.k) / BK / d.groups : static_cast<double>(cdiv(d.k, BK));
    const double live = ragged_n ? (d.groups < d.n ? d.groups : d.n) : 0;  // groups that can hold a column
    const bool f32_out = d.out_kind == OUT_F32;
    struct Kind { int bn; double per_kb, rest, part; };  // part: the share of a tile a ragged group wastes
    const Kind kinds[4] = {{32, 0.25, 1.1, 0.5},
                           {64, 0.30, 1.25, 0.5},
                           {128, 0.41, 1.7, 0.5},
                           {256, d.a_vec ? (d.b_vec ? 0.82 : 0.72) : 0.46, !aligned_c(d) ? 20.0 : f32_out ? 4.0 : 2.0, 0.75}};
    Tile best{2, 256, 1};
    double least = 1e300;
    for (const Kind &kind : kinds) {
        if (d.trans_b && kind.bn < 128) continue;  // op(B) = T is read in panels of 128 columns
        const bool wide = kind.bn == 256;
        const double across = cdiv(d.m, wide ? kind.bn : BM);
        double along = ragged_n ? static_cast<double>(d.n) / kind.bn + kind.part * live : static_cast<double>(cdiv(d.n, kind.bn));
        if (ragged_n && along < live) along = live;
        const double tiles = across * along * (ragged_k ? d.groups : 1);
        const double at_once = wide ? (sm_count > 1 ? sm_count / 2 : 1) : sm_count;
        // the launch must hold every cluster: count the tiles as it does
        const double most = ragged_n ? across * (d.n / kind.bn + live) : tiles;
        for (int split = 1; split <= (wide ? 1 : MAX_SPLIT); split *= 2) {
            if (split > 1 && (kb < 2 * split || most * split > (split == 8 ? 96.0 : split == 4 ? 132.0 : 148.0) * sm_count / 148.0)) break;
            double rounds = tiles * split / at_once;
            rounds = rounds <= 1.0 ? 1.0 : static_cast<double>(static_cast<long long>(rounds + 0.999));
            const double cost = rounds * (kb / split * kind.per_kb + kind.rest) + (split > 1 ? 1.0 + 0.025 * kind.bn : 0.0);
            if (cost < least) {
                least = cost;
                best = Tile{wide ? 2 : 1, kind.bn, split};
            }
        }
    }
    return best;
}

}  // namespace fp8

cudaError_t launch_gemm_fp8(Context &ctx, const GemmFp8Desc &d) {
    using namespace fp8;
    const Tile t = choose_tile(d, ctx.sm_count);
    const bool wide = t.bn == 256;
    const bool ragged_n = d.groups > 0 && d.ragged == GS_GROUP_N, ragged_k = d.groups > 0 && d.ragged == GS_GROUP_K;
    // A scale matrix per 128 x 128 block is laid out as its operand is; a scale per vector has the non-K index first.
    Side sa{}, sb{};
    sa.extent = d.m;
    sa.mn = d.trans_a ? 0 : 1;
    sa.grouped = ragged_n && d.groups > 1 && d.stride_a > 0 ? 1 : 0;
    sa.scale = d.sa;
    sa.s_i = d.a_vec || !d.trans_a ? 1 : d.ldsa;
    sa.s_k = d.a_vec || !d.trans_a ? d.ldsa : 1;
    sa.s_g = ragged_n ? d.stride_sa : 0;
    sb.extent = d.n;
    sb.mn = d.trans_b ? 1 : 0;
    sb.scale = d.sb;
    sb.s_i = d.b_vec || d.trans_b ? 1 : d.ldsb;
    sb.s_k = d.b_vec || d.trans_b ? d.ldsb : 1;
    Args a{};
    a.p = wide ? sb : sa;
    a.q = wide ? sa : sb;
    a.k = d.k;
    a.p_blocks = cdiv(a.p.extent, static_cast<long long>(BM) * t.cg);
    a.q_blocks = cdiv(a.q.extent, t.bn);
    a.k_blocks = cdiv(d.k, BK);
    a.groups = d.groups;
    a.ragged = d.groups > 0 ? d.ragged : -1;
    a.offsets = d.offsets;
    a.split = t.split;
    // Ragged N: an upper bound (each group may end in a part tile); the kernel counts the tiles itself.
    const long long tile_n = wide ? BM * t.cg : t.bn, across = wide ? a.q_blocks : a.p_blocks;
    const long long tiles = ragged_n ? across * (d.n / tile_n + (d.groups < d.n ? d.groups : d.n))
                                     : static_cast<long long>(a.p_blocks) * a.q_blocks * (ragged_k ? d.groups : 1);
    a.total_tiles = static_cast<uint32_t>(tiles);
    const uint32_t p_e5m2 = wide ? d.b_e5m2 : d.a_e5m2, q_e5m2 = wide ? d.a_e5m2 : d.b_e5m2;
    a.idesc = (1u << 4) | (p_e5m2 << 7) | (q_e5m2 << 10) | (static_cast<uint32_t>(a.p.mn) << 15) |
              (static_cast<uint32_t>(a.q.mn) << 16) | ((static_cast<uint32_t>(t.bn) >> 3) << 17) |
              ((static_cast<uint32_t>(BM * t.cg) >> 4) << 24);
    a.C = d.C;
    a.ldc = d.ldc;
    a.stride_c = d.stride_c;
    a.out_kind = d.out_kind;
    a.ep = d.ep;
    a.err = ctx.dev_err;
    a.spin_limit = ctx.spin_limit;
    a.debug_skip_kb = ctx.debug_skip_kb;
    const size_t es = out_elem_size(d.out_kind);
    a.vec_c = aligned_c(d) ? 1 : 0;
    a.whole_c = d.m * es % 16 == 0 ? 1 : 0;

    Maps maps{};
    std::string why;
    if (d.k > 0) {
        const uint64_t a0 = d.trans_a ? d.k : d.m, a1 = d.trans_a ? d.m : d.k;
        const uint64_t batch = sa.grouped ? static_cast<uint64_t>(d.groups) : 1;
        const uint64_t a2 = sa.grouped ? static_cast<uint64_t>(d.stride_a) : a1 * static_cast<uint64_t>(d.lda);
        const uint64_t b0 = d.trans_b ? d.n : d.k, b1 = d.trans_b ? d.k : d.n;
        const uint32_t q_box = a.q.mn ? 128 : static_cast<uint32_t>(t.bn / t.cg);
        if (!encode_tmap_3d(wide ? &maps.q : &maps.p, CU_TENSOR_MAP_DATA_TYPE_UINT8, d.A, a0, a1, batch, static_cast<uint64_t>(d.lda),
                            a2, 128, wide ? q_box : 128, &why) ||
            !encode_tmap_3d(wide ? &maps.p : &maps.q, CU_TENSOR_MAP_DATA_TYPE_UINT8, d.B, b0, b1, 1, static_cast<uint64_t>(d.ldb),
                            b1 * static_cast<uint64_t>(d.ldb), 128, wide ? 128 : q_box, &why)) {
            ctx.last_error = "tensor map encode failed: " + why;
            return cudaErrorInvalidValue;
        }
    }
    if (wide && a.vec_c && a.ep.beta_zero) {
        const CUtensorMapDataType dt = d.out_kind == OUT_F32   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                       : d.out_kind == OUT_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                               : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
        const uint64_t row = static_cast<uint64_t>(d.ldc) * es;
        const bool many = ragged_k && d.groups > 1;
        a.tma_store = encode_tmap_3d(&maps.c, dt, d.C, d.m, d.n, many ? d.groups : 1, row,
                                     many ? static_cast<uint64_t>(d.stride_c) * es : row * static_cast<uint64_t>(d.n),
                                     static_cast<uint32_t>(128 / es), 32, nullptr)
                          ? 1
                          : 0;
    }
    const bool p_vec = wide ? d.b_vec : d.a_vec, q_vec = wide ? d.a_vec : d.b_vec;
    const int mode = (p_vec ? 1 : 0) | (q_vec ? 2 : 0);
    ctx.last_kernels |= GS_KERNEL_TC_F8;
    if (t.cg == 2) return launch_mode<2, 256>(ctx, mode, maps, a, tiles);
    if (t.bn == 128) return launch_mode<1, 128>(ctx, mode, maps, a, tiles);
    if (t.bn == 64) return launch_mode<1, 64>(ctx, mode, maps, a, tiles);
    return launch_mode<1, 32>(ctx, mode, maps, a, tiles);
}

}  // namespace gs
