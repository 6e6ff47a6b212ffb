// gemm_fp8_sm100.cu -- FP8 matrix products with one f32 scale per 128 elements
// along K (or per 128 x 128 block), dense and over ragged groups, for sm_100a.
//
//   C[i, j] = alpha * sum_b sA(i, b) * sB(j, b) * P_b[i, j] + beta * C[i, j],
//   P_b[i, j] = sum over the 128 K elements of block b of op(A)[i, p] * op(B)[p, j]
//
// The scales are arbitrary f32 numbers, so they cannot be folded into the
// tensor core's accumulation over K: each block's P_b is computed by four
// tcgen05.mma (kind::f8f6f4, K = 32) into a TMEM slot of its own, and the
// epilogue warps ("promoters") read the slot and add scale * P_b to f32 sums
// in registers with packed FMAs while the tensor core fills the next slot.
// Products of two FP8 values are exact in f32 and a block sums 128 of them.
//
// One CTA (or CTA pair) per SM runs tiles persistently:
//  - warp 0: TMA producer, 128 x 128 bytes of A and BN / CG x 128 of B a stage;
//    transposes live in the tensor maps and the UMMA major bits;
//  - warp 1: TMEM allocation, and tcgen05.mma from one thread (even CTA);
//  - warp 2: copies each K block's scales into a ring in shared memory;
//  - warps 4..: promoters, one accumulator row per thread, BN / (warps / 4)
//    columns each. With 128 columns a thread they need more registers than an
//    even split gives: of the 3 x 168 a lane triple is launched with, the first
//    warpgroup hands 96 to the two promoter warpgroups (72 / 216 / 216).
// Ragged groups: offsets are read from device memory; tile counts are scanned
// once per CTA into shared memory and each tile finds its group by bisection.
//
// Split-K (few tiles, long K): the CTAs of a cluster take K slices of one tile
// and sum their f32 results in rank order through distributed shared memory,
// so there is no workspace and the result does not depend on timing.
#include <type_traits>

#include "gs_epilogue.cuh"
#include "gs_fp8.h"
#include "gs_internal.h"
#include "gs_ptx.cuh"

namespace gs {
namespace fp8 {

constexpr int BM = 128;
constexpr int BK = 128;
constexpr int SC_STAGES = 8;

template <int CG, int BN>
struct Cfg {
    static constexpr int EPI_WARPS = BN >= 128 ? 8 : 4;
    static constexpr int EPI_COLS = BN / (EPI_WARPS / 4);
    static constexpr int THREADS = 128 + 32 * EPI_WARPS;
    static constexpr int B_ROWS = BN / CG;
    static constexpr int A_STAGE = BM * BK;
    static constexpr int B_STAGE = B_ROWS * BK;
    static constexpr int STAGE = A_STAGE + B_STAGE;
    static constexpr int STAGES = STAGE >= 48 * 1024 ? 4 : (STAGE >= 32 * 1024 ? 6 : 8);
    static constexpr int SLOTS = BN == 256 ? 2 : 4;
    static constexpr int TMEM_COLS = BN * SLOTS;
    static constexpr int SC_FLOATS = BN + BM;
    static constexpr int TILE_M = BM * CG;
    static constexpr int BARS = 2 * STAGES + 2 * SLOTS + 2 * SC_STAGES + 1;
    static constexpr int SMEM = STAGES * STAGE + SC_STAGES * SC_FLOATS * 4 + BARS * 8 + 16 + 1024 /*alignment*/;
};

struct Args {
    int m, n, k;
    int m_blocks, n_blocks, k_blocks;  // n_blocks: of the dense / ragged-K product
    int groups;                        // 0 = dense
    int ragged;                        // GS_GROUP_N / GS_GROUP_K when groups > 0
    const int32_t *offsets;
    int group_m;
    int split;                         // cluster CTAs sharing a tile's K blocks (1 = none)
    long long total_tiles;             // dense and ragged-K
    int a_mn, b_mn;
    int a_bcast;                       // every group multiplies by the same A
    uint32_t idesc;
    const float *sa;
    long long sa_i, sa_k, sa_g;        // element strides: row or row block, K block, group
    const float *sb;
    long long sb_i, sb_k;
    void *C;
    long long ldc, stride_c;
    int out_kind;
    Epilogue ep;
    uint32_t *err;
    long long spin_limit;
};

// A tile: rows m0.. of group g, columns n0..n_end, K blocks kb0..kb0+nkb.
struct Item {
    int g, m0, n0, n_end, kb0, nkb;
    bool bad;  // ragged-K group whose offsets are not multiples of 128
};

template <int CG, int BN>
__device__ __forceinline__ bool item_at(const Args &a, const int *tile_start, const int *off, long long t, uint32_t rank,
                                        Item &it) {
    int mb, nb, n_blocks = a.n_blocks;
    long long r = t;
    it.g = 0;
    it.bad = false;
    it.kb0 = 0;
    it.nkb = a.k_blocks;
    int n_base = 0;
    it.n_end = a.n;
    if (a.groups == 0) {
        if (t >= a.total_tiles) return false;
    } else if (a.ragged == GS_GROUP_N) {
        if (t >= tile_start[a.groups]) return false;
        int lo = 0, hi = a.groups;  // the last group whose first tile is <= t
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (tile_start[mid] <= t) lo = mid;
            else hi = mid;
        }
        it.g = lo;
        r = t - tile_start[lo];
        n_base = off[lo];
        it.n_end = off[lo + 1];
        n_blocks = (it.n_end - n_base + BN - 1) / BN;
    } else {
        if (t >= a.total_tiles) return false;
        const long long per = static_cast<long long>(a.m_blocks) * a.n_blocks;
        it.g = static_cast<int>(t / per);
        r = t - it.g * per;
        const int k_lo = off[it.g], k_hi = off[it.g + 1];
        it.kb0 = k_lo / BK;
        it.nkb = (k_hi - k_lo + BK - 1) / BK;
        it.bad = k_hi > k_lo && (k_lo % BK != 0 || (k_hi % BK != 0 && k_hi != a.k));
        if (it.bad) it.nkb = 0;
    }
    const long long span = static_cast<long long>(a.group_m) * n_blocks;
    const int gi = static_cast<int>(r / span);
    const int within = static_cast<int>(r - gi * span);
    const int first = gi * a.group_m;
    const int gm = min(a.group_m, a.m_blocks - first);
    mb = first + within % gm;
    nb = within / gm;
    it.m0 = mb * Cfg<CG, BN>::TILE_M + static_cast<int>(CG == 2 ? rank : 0) * BM;
    it.n0 = n_base + nb * BN;
    if (CG == 1 && a.split > 1) {  // this CTA's share of the K blocks
        const int lo = static_cast<int>(static_cast<long long>(it.nkb) * rank / a.split);
        const int hi = static_cast<int>(static_cast<long long>(it.nkb) * (rank + 1) / a.split);
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

template <int CG>
__device__ __forceinline__ void umma_f8(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    if constexpr (CG == 2) {
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d_tmem), "l"(adesc), "l"(bdesc),
            "r"(idesc), "r"(accumulate)
            : "memory");
    } else {
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d_tmem), "l"(adesc), "l"(bdesc),
            "r"(idesc), "r"(accumulate)
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
__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}

// One element of C, rounded once from f32 (to nearest even).
__device__ __forceinline__ void store_c(const Args &a, void *C, size_t i, float acc) {
    float v = a.ep.identity ? acc : __fmul_rn(a.ep.alpha_f, acc);
    if (a.out_kind == OUT_F32) {
        float *c = static_cast<float *>(C) + i;
        if (!a.ep.beta_zero) v = __fmaf_rn(a.ep.beta_f, *c, v);
        *c = v;
    } else if (a.out_kind == OUT_F16) {
        __half *c = static_cast<__half *>(C) + i;
        if (!a.ep.beta_zero) v = __fmaf_rn(a.ep.beta_f, __half2float(*c), v);
        *c = __float2half_rn(v);
    } else {
        __nv_bfloat16 *c = static_cast<__nv_bfloat16 *>(C) + i;
        if (!a.ep.beta_zero) v = __fmaf_rn(a.ep.beta_f, __bfloat162float(*c), v);
        *c = __float2bfloat16_rn(v);
    }
}

// MODE bit 0: A has a scale per row (else per 128 rows); bit 1: B has a scale
// per column (else per 128 columns).
template <int CG, int BN, int MODE>
__global__ void __launch_bounds__(Cfg<CG, BN>::THREADS, 1)
    k_gemm_fp8(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const Args args) {
    using C_ = Cfg<CG, BN>;
    constexpr bool A_VEC = (MODE & 1) != 0, B_VEC = (MODE & 2) != 0;
    constexpr int STAGES = C_::STAGES, SLOTS = C_::SLOTS, EPI_COLS = C_::EPI_COLS;

    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *smA = smem;
    uint8_t *smB = smem + STAGES * C_::A_STAGE;
    float *scales = reinterpret_cast<float *>(smB + STAGES * C_::B_STAGE);
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

    const int warp = threadIdx.x >> 5;
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
        prefetch_tensormap(&tmA);
        prefetch_tensormap(&tmB);
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
        const int limit = args.ragged == GS_GROUP_N ? args.n : args.k;
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
            int sum = 0;
            for (int i = lo; i < hi; ++i) {
                tile_start[i] = sum;
                if (i < args.groups) sum += (off[i + 1] - off[i] + BN - 1) / BN * args.m_blocks;
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

    const long long tile0 = blockIdx.x / (CG * (CG == 1 ? args.split : 1));
    const long long tile_step = gridDim.x / (CG * (CG == 1 ? args.split : 1));
    Item it;

    if (warp < 4) {
    if constexpr (EPI_COLS == 128) asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    if (warp == 0) {
        if (lane == 0) {
            const uint64_t pol = l2_policy_evict_normal();
            int stage = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (long long t = tile0; ok && item_at<CG, BN>(args, tile_start, off, t, rank, it); t += tile_step) {
                const int nc = it.n0 + static_cast<int>(CG == 2 ? rank : 0) * C_::B_ROWS;
                const int ga = args.a_bcast ? 0 : it.g;
                for (int kb = 0; kb < it.nkb; ++kb) {
                    if (!mbar_wait(&empty[stage], phase ^ 1u, args.err, 1, args.spin_limit)) { ok = false; break; }
                    uint8_t *dA = smA + stage * C_::A_STAGE;
                    uint8_t *dB = smB + stage * C_::B_STAGE;
                    const int k0 = (it.kb0 + kb) * BK;
                    if constexpr (CG == 2) {
                        const uint32_t fbar = mapa_shared(smem_u32(&full[stage]), 0);
                        if (leader) mbar_arrive_expect_tx(&full[stage], 2 * C_::STAGE);
                        if (args.a_mn) tma_load_3d_2sm(dA, &tmA, fbar, it.m0, k0, ga, pol);
                        else tma_load_3d_2sm(dA, &tmA, fbar, k0, it.m0, ga, pol);
                        if (args.b_mn) tma_load_3d_2sm(dB, &tmB, fbar, nc, k0, 0, pol);
                        else tma_load_3d_2sm(dB, &tmB, fbar, k0, nc, 0, pol);
                    } else {
                        mbar_arrive_expect_tx(&full[stage], C_::STAGE);
                        if (args.a_mn) tma_load_3d_hint(dA, &tmA, &full[stage], it.m0, k0, ga, pol);
                        else tma_load_3d_hint(dA, &tmA, &full[stage], k0, it.m0, ga, pol);
                        if (args.b_mn) {  // only with BN >= 128: panels of 128 columns
#pragma unroll
                            for (int c = 0; c < (BN + 127) / 128; ++c)
                                tma_load_3d_hint(dB + c * 128 * BK, &tmB, &full[stage], nc + c * 128, k0, 0, pol);
                        } else {
                            tma_load_3d_hint(dB, &tmB, &full[stage], k0, nc, 0, pol);
                        }
                    }
                    if (++stage == STAGES) { stage = 0; phase ^= 1u; }
                }
            }
        }
    } else if (warp == 1) {
        if (lane == 0 && leader) {
            int stage = 0, slot = 0;
            uint32_t phase = 0, sphase = 0;
            bool ok = true;
            for (long long t = tile0; ok && item_at<CG, BN>(args, tile_start, off, t, rank, it); t += tile_step) {
                for (int kb = 0; kb < it.nkb; ++kb) {
                    if (!mbar_wait(&tempty[slot], sphase ^ 1u, args.err, 2, args.spin_limit) ||
                        !mbar_wait(&full[stage], phase, args.err, 3, args.spin_limit)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t a_base = smem_u32(smA + stage * C_::A_STAGE);
                    const uint32_t b_base = smem_u32(smB + stage * C_::B_STAGE);
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk) {
                        const uint64_t adesc = args.a_mn ? umma_smem_desc_sw128(a_base + kk * 32 * 128, 128 * BK, 1024)
                                                         : umma_smem_desc_sw128(a_base + kk * 32, 16, 1024);
                        const uint64_t bdesc = args.b_mn ? umma_smem_desc_sw128(b_base + kk * 32 * 128, 128 * BK, 1024)
                                                         : umma_smem_desc_sw128(b_base + kk * 32, 16, 1024);
                        umma_f8<CG>(tmem_base + slot * BN, adesc, bdesc, args.idesc, kk != 0 ? 1u : 0u);
                    }
                    if constexpr (CG == 2) {
                        umma_commit_2sm(&empty[stage], 0x3);
                        umma_commit_2sm(&tfull[slot], 0x3);
                    } else {
                        umma_commit(&empty[stage]);
                        umma_commit(&tfull[slot]);
                    }
                    if (++stage == STAGES) { stage = 0; phase ^= 1u; }
                    if (++slot == SLOTS) { slot = 0; sphase ^= 1u; }
                }
            }
            if (!ok) {  // the MMAs already issued end before the CTA frees its TMEM
                if constexpr (CG == 2) umma_commit_2sm(drain, 0x3);
                else umma_commit(drain);
                mbar_wait(drain, 0, args.err, 5, args.spin_limit);
            }
        }
    } else if (warp == 2) {
        // Scales. A few K blocks are fetched at a time so that their loads overlap.
        constexpr int NB = B_VEC ? BN / 32 : 1, NA = A_VEC ? BM / 32 : 1, U = EPI_COLS == 128 ? 2 : 4;
        int ss = 0;
        uint32_t sp = 0;
        bool ok = true;
        for (long long t = tile0; ok && item_at<CG, BN>(args, tile_start, off, t, rank, it); t += tile_step) {
            const float *pa = args.sa + it.g * args.sa_g;
            for (int kb = 0; ok && kb < it.nkb; kb += U) {
                float va[U][NA], vb[U][NB];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const long long ka = it.kb0 + min(kb + u, it.nkb - 1);
#pragma unroll
                    for (int i = 0; i < NA; ++i) {
                        const int r = A_VEC ? it.m0 + i * 32 + lane : it.m0 / 128;
                        const bool in = A_VEC ? r < args.m : it.m0 < args.m;
                        va[u][i] = in ? pa[r * args.sa_i + ka * args.sa_k] : 0.0f;
                    }
#pragma unroll
                    for (int i = 0; i < NB; ++i) {
                        const int c = B_VEC ? it.n0 + i * 32 + lane : it.n0 / 128 + lane;
                        const bool in = B_VEC ? c < it.n_end : (lane < (BN + 127) / 128 && it.n0 + lane * 128 < args.n);
                        vb[u][i] = in ? args.sb[c * args.sb_i + ka * args.sb_k] : 0.0f;
                    }
                }
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    if (!ok || kb + u >= it.nkb) break;
                    // one answer for the warp: its lanes arrive together
                    if (!__all_sync(0xffffffffu, mbar_wait(&sempty[ss], sp ^ 1u, args.err, 6, args.spin_limit))) {
                        ok = false;
                        break;
                    }
                    float *dst = scales + ss * C_::SC_FLOATS;
#pragma unroll
                    for (int i = 0; i < NB; ++i) {
                        const float v = A_VEC ? vb[u][i] : __fmul_rn(va[u][0], vb[u][i]);
                        if (B_VEC || lane < (BN + 127) / 128) dst[i * 32 + lane] = v;
                    }
                    if constexpr (A_VEC) {
#pragma unroll
                        for (int i = 0; i < NA; ++i) dst[BN + i * 32 + lane] = va[u][i];
                    }
                    mbar_arrive(&sfull[ss]);
                    if (++ss == SC_STAGES) { ss = 0; sp ^= 1u; }
                }
            }
        }
    }
    } else {
        if constexpr (EPI_COLS == 128) asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
        const int quad = warp & 3;
        const int ew = warp - 4;
        const int c_lo = (ew / 4) * EPI_COLS;
        const int row = quad * 32 + lane;
        const uint32_t t_lane = tmem_base + (static_cast<uint32_t>(quad * 32) << 16);
        const uint32_t tempty_leader = CG == 2 ? mapa_shared(smem_u32(&tempty[0]), 0) : 0u;
        int slot = 0, ss = 0;
        uint32_t phase = 0, sp = 0;
        bool ok = true;
        for (long long t = tile0; ok && item_at<CG, BN>(args, tile_start, off, t, rank, it); t += tile_step) {
            if (it.bad) {
                if (ew == 0 && lane == 0) atomicOr(args.err, 2u);
                continue;
            }
            uint64_t acc[EPI_COLS / 2];
#pragma unroll
            for (int j = 0; j < EPI_COLS / 2; ++j) acc[j] = 0;
#pragma unroll 1
            for (int kb = 0; kb < it.nkb; ++kb) {
                // every lane takes the same way out (tcgen05.ld is warp-aligned)
                if (!__all_sync(0xffffffffu, mbar_wait(&sfull[ss], sp, args.err, 7, args.spin_limit) &&
                                                 mbar_wait(&tfull[slot], phase, args.err, 4, args.spin_limit))) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const float *sc = scales + ss * C_::SC_FLOATS;
                const uint32_t sc_addr = smem_u32(sc + c_lo);
                uint64_t sa2 = 0;
                if constexpr (A_VEC && B_VEC) {
                    const float sa = sc[BN + row];
                    sa2 = pack2(sa, sa);
                } else if constexpr (!B_VEC) {
                    float s = sc[c_lo / 128];
                    if constexpr (A_VEC) s = __fmul_rn(sc[BN + row], s);
                    sa2 = pack2(s, s);
                }
#pragma unroll
                for (int c = 0; c < EPI_COLS; c += 32) {
                    uint32_t r[32];
                    tmem_ld_32x32b_x32(t_lane + slot * BN + c_lo + c, r);
                    tmem_wait_ld();
                    if (c + 32 == EPI_COLS) {  // the slot is read: the tensor core may fill it again
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) {
                            if constexpr (CG == 2) mbar_arrive_cluster(tempty_leader + slot * sizeof(uint64_t));
                            else mbar_arrive(&tempty[slot]);
                        }
                    }
#pragma unroll
                    for (int j = 0; j < 32; j += 4) {
                        uint64_t p0 = pack2(__uint_as_float(r[j]), __uint_as_float(r[j + 1]));
                        uint64_t p1 = pack2(__uint_as_float(r[j + 2]), __uint_as_float(r[j + 3]));
                        if constexpr (B_VEC) {
                            const float4 s4 = ld_shared_f32x4(sc_addr + (c + j) * 4);
                            if constexpr (A_VEC) {
                                p0 = mul2(p0, sa2);
                                p1 = mul2(p1, sa2);
                            }
                            acc[(c + j) / 2] = fma2(p0, pack2(s4.x, s4.y), acc[(c + j) / 2]);
                            acc[(c + j) / 2 + 1] = fma2(p1, pack2(s4.z, s4.w), acc[(c + j) / 2 + 1]);
                        } else {
                            acc[(c + j) / 2] = fma2(p0, sa2, acc[(c + j) / 2]);
                            acc[(c + j) / 2 + 1] = fma2(p1, sa2, acc[(c + j) / 2 + 1]);
                        }
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&sempty[ss]);
                if (++slot == SLOTS) { slot = 0; phase ^= 1u; }
                if (++ss == SC_STAGES) { ss = 0; sp ^= 1u; }
            }
            if (!ok) break;
            if (CG == 1 && args.split > 1) {
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
            const int m = it.m0 + row;
            if (m < args.m) {
                void *Cb = args.C;
                if (args.ragged == GS_GROUP_K)
                    Cb = static_cast<uint8_t *>(args.C) + static_cast<size_t>(it.g) * args.stride_c * (args.out_kind == OUT_F32 ? 4 : 2);
#pragma unroll
                for (int j = 0; j < EPI_COLS / 2; ++j) {
                    float x, y;
                    unpack2(acc[j], x, y);
                    const int n = it.n0 + c_lo + 2 * j;
                    const size_t i = static_cast<size_t>(m) + static_cast<size_t>(n) * args.ldc;
                    if (n < it.n_end) store_c(args, Cb, i, x);
                    if (n + 1 < it.n_end) store_c(args, Cb, i + args.ldc, y);
                }
            }
        }
    }

    __syncwarp();
    if (CG == 1 && args.split > 1) {
        cluster_sync();  // every slice's sums are in its CTA's shared memory
        if (item_at<CG, BN>(args, tile_start, off, tile0, rank, it) && !it.bad) {
            const int cols = (BN + args.split - 1) / args.split;
            const int first = static_cast<int>(rank) * cols, last = min(first + cols, BN);
            void *Cb = args.C;
            if (args.ragged == GS_GROUP_K)
                Cb = static_cast<uint8_t *>(args.C) + static_cast<size_t>(it.g) * args.stride_c * (args.out_kind == OUT_F32 ? 4 : 2);
            for (int e = first * BM + static_cast<int>(threadIdx.x); e < last * BM; e += C_::THREADS) {
                const int col = it.n0 + e / BM, r = it.m0 + e % BM;
                if (col >= it.n_end || r >= args.m) continue;
                float sum = 0.0f;
                for (int q = 0; q < args.split; ++q)
                    sum = __fadd_rn(sum, ld_cluster_f32(mapa_shared(smem_u32(smem) + e * 4, static_cast<uint32_t>(q))));
                store_c(args, Cb, static_cast<size_t>(r) + static_cast<size_t>(col) * args.ldc, sum);
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
static cudaError_t launch(Context &ctx, const CUtensorMap &ta, const CUtensorMap &tb, const Args &a, long long tiles) {
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
    e = launch_pdl(kern, dim3(static_cast<unsigned>(units * cluster)), dim3(C_::THREADS), smem, ctx.stream, cluster, ta, tb, a);
    ctx.launches++;
    return e;
}

template <int CG, int BN>
static cudaError_t launch_mode(Context &ctx, int mode, const CUtensorMap &ta, const CUtensorMap &tb, const Args &a, long long tiles) {
    switch (mode) {
    case 0: return launch<CG, BN, 0>(ctx, ta, tb, a, tiles);
    case 1: return launch<CG, BN, 1>(ctx, ta, tb, a, tiles);
    case 2: return launch<CG, BN, 2>(ctx, ta, tb, a, tiles);
    default: return launch<CG, BN, 3>(ctx, ta, tb, a, tiles);
    }
}

static int cdiv(long long a, long long b) { return static_cast<int>((a + b - 1) / b); }

// Tile of a product: bn columns, cg CTAs, split K slices.
Tile choose_tile(const GemmFp8Desc &d, int sm_count) {
    Tile t{1, 256, 1};
    // Columns a tile can expect to fill: a ragged group's mean share, or all of them.
    const long long cols = d.groups > 0 && d.ragged == GS_GROUP_N ? cdiv(d.n, d.groups) : d.n;
    if (!d.trans_b) t.bn = cols <= 32 ? 32 : cols <= 64 ? 64 : cols <= 128 ? 128 : 256;
    else t.bn = cols <= 128 ? 128 : 256;
    if (t.bn == 256 && d.m > BM && sm_count >= 2) t.cg = 2;
    return t;
}

}  // namespace fp8

cudaError_t launch_gemm_fp8(Context &ctx, const GemmFp8Desc &d) {
    using namespace fp8;
    const Tile t = choose_tile(d, ctx.sm_count);
    Args a{};
    a.m = d.m;
    a.n = d.n;
    a.k = d.k;
    a.m_blocks = cdiv(d.m, static_cast<long long>(BM) * t.cg);
    a.n_blocks = cdiv(d.n, t.bn);
    a.k_blocks = cdiv(d.k, BK);
    a.groups = d.groups;
    a.ragged = d.groups > 0 ? d.ragged : -1;
    a.offsets = d.offsets;
    a.group_m = a.m_blocks < 8 ? a.m_blocks : 8;
    a.split = t.split;
    const bool ragged_n = a.groups > 0 && a.ragged == GS_GROUP_N;
    // Ragged N: an upper bound (each group may end in a part tile); the kernel counts the tiles itself.
    const long long tiles = ragged_n ? static_cast<long long>(a.m_blocks) * (d.n / t.bn + (d.groups < d.n ? d.groups : d.n))
                                     : static_cast<long long>(a.m_blocks) * a.n_blocks * (a.groups > 0 ? a.groups : 1);
    a.total_tiles = tiles;
    a.a_mn = d.trans_a ? 0 : 1;
    a.b_mn = d.trans_b ? 1 : 0;
    a.a_bcast = ragged_n && d.groups > 1 && d.stride_a > 0 ? 0 : 1;
    a.idesc = (1u << 4) | (static_cast<uint32_t>(d.a_e5m2) << 7) | (static_cast<uint32_t>(d.b_e5m2) << 10) |
              (static_cast<uint32_t>(a.a_mn) << 15) | (static_cast<uint32_t>(a.b_mn) << 16) |
              ((static_cast<uint32_t>(t.bn) >> 3) << 17) | ((static_cast<uint32_t>(BM * t.cg) >> 4) << 24);
    // A scale matrix per 128 x 128 block is laid out as its operand is; a scale per vector has the non-K index first.
    a.sa = d.sa;
    a.sa_i = d.a_vec ? 1 : (d.trans_a ? d.ldsa : 1);
    a.sa_k = d.a_vec ? d.ldsa : (d.trans_a ? 1 : d.ldsa);
    a.sa_g = ragged_n ? d.stride_sa : 0;
    a.sb = d.sb;
    a.sb_i = d.b_vec ? 1 : (d.trans_b ? 1 : d.ldsb);
    a.sb_k = d.b_vec ? d.ldsb : (d.trans_b ? d.ldsb : 1);
    a.C = d.C;
    a.ldc = d.ldc;
    a.stride_c = d.stride_c;
    a.out_kind = d.out_kind;
    a.ep = d.ep;
    a.err = ctx.dev_err;
    a.spin_limit = ctx.spin_limit;

    CUtensorMap ta{}, tb{};
    if (d.k > 0) {
        std::string why;
        const uint64_t a0 = d.trans_a ? d.k : d.m, a1 = d.trans_a ? d.m : d.k;
        const uint64_t batch = a.a_bcast ? 1 : static_cast<uint64_t>(d.groups);
        const uint64_t a2 = batch > 1 ? static_cast<uint64_t>(d.stride_a) : a1 * static_cast<uint64_t>(d.lda);
        const uint64_t b0 = d.trans_b ? d.n : d.k, b1 = d.trans_b ? d.k : d.n;
        const uint32_t b_rows = static_cast<uint32_t>(t.bn / t.cg);
        if (!encode_tmap_3d(&ta, CU_TENSOR_MAP_DATA_TYPE_UINT8, d.A, a0, a1, batch, static_cast<uint64_t>(d.lda), a2, 128, 128, &why) ||
            !encode_tmap_3d(&tb, CU_TENSOR_MAP_DATA_TYPE_UINT8, d.B, b0, b1, 1, static_cast<uint64_t>(d.ldb),
                            b1 * static_cast<uint64_t>(d.ldb), 128, d.trans_b ? 128 : b_rows, &why)) {
            ctx.last_error = "tensor map encode failed: " + why;
            return cudaErrorInvalidValue;
        }
    }
    const int mode = (d.a_vec ? 1 : 0) | (d.b_vec ? 2 : 0);
    ctx.last_kernels |= GS_KERNEL_TC_F8;
    if (t.cg == 2) return launch_mode<2, 256>(ctx, mode, ta, tb, a, tiles);
    if (t.bn == 256) return launch_mode<1, 256>(ctx, mode, ta, tb, a, tiles);
    if (t.bn == 128) return launch_mode<1, 128>(ctx, mode, ta, tb, a, tiles);
    if (t.bn == 64) return launch_mode<1, 64>(ctx, mode, ta, tb, a, tiles);
    return launch_mode<1, 32>(ctx, mode, ta, tb, a, tiles);
}

}  // namespace gs
