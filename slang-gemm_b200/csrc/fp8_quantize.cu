// fp8_quantize.cu -- casts f32 / f16 / bf16 matrices to FP8 with one scale per
// vector of 128 elements (along either axis) or per 128 x 128 block: the operand
// preparation of the FP8 products (gemm_fp8_sm100.cu).
//
//   amax  = largest |x| of the block's finite elements
//   scale = the smallest power of two with amax / scale <= the type's largest
//           value (448 for E4M3, 57344 for E5M2), at least 2^-126; 1 when amax = 0
//   q     = x / scale rounded to nearest even
//
// A power of two leaves x / scale exact, so q carries one rounding and does not
// depend on how a division is carried out; a float format's relative step is the
// same at every scale, so nothing is lost but part of the subnormal range.
// NaN stays NaN; an infinity becomes NaN in E4M3 (which has none) and stays in
// E5M2. Columns may be gathered: column c reads source column index[c] / div,
// and a negative (or out-of-range) index gives zeros with scale 1.
//
// Bound by memory: every element is read once with 16-byte loads and held in
// registers between the maximum and the cast. 8192 x 8192 f32 in blocks: 51 us, 6.5
// TB/s. Vectors of bf16 come near it (4096 x 16384: 36 us, 5.6 TB/s) and, gathered from
// a source that fits L2, are bound by instruction issue (31 us). Vectors along the
// rows cross threads and three barriers a tile: 72 us, 2.8 TB/s (f32: 87 us, 3.9).
#include <cuda_fp8.h>

#include <cstring>
#include <type_traits>

#include "gs_float.cuh"
#include "gs_fp8.h"

namespace gs {
namespace quant {

constexpr uint32_t kInf = 0x7f800000u;

// Scale exponent from the bits of amax.
template <bool E5M2>
__device__ __forceinline__ int scale_exp(uint32_t amax) {
    if (amax == 0) return 0;
    const int e = static_cast<int>(amax >> 23) - 127;
    const int up = (amax & 0x7fffffu) > 0x600000u ? 1 : 0;  // both types' largest value is 1.75 * 2^e
    return max(e - (E5M2 ? 15 : 8) + up, -126);
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }

template <bool E5M2>
__device__ __forceinline__ uint32_t cast2(float x, float y) {
    return __nv_cvt_float2_to_fp8x2(make_float2(x, y), __NV_SATFINITE, E5M2 ? __NV_E5M2 : __NV_E4M3);
}

__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

template <bool VEC>
__device__ __forceinline__ void store8(uint8_t *col, int r, int rows, uint2 q) {
    if (VEC && r + 8 <= rows) {
        *reinterpret_cast<uint2 *>(col + r) = q;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (r + i < rows) col[r + i] = static_cast<uint8_t>((i < 4 ? q.x >> (8 * i) : q.y >> (8 * (i - 4))) & 0xffu);
    }
}

// Source column of column c, or null for a column of zeros.
template <typename T>
__device__ __forceinline__ const T *source(const QuantDesc &d, int c) {
    long long s = c;
    if (d.index != nullptr) {
        const int i = d.index[c];
        s = i < 0 ? -1 : i / d.index_div;
        if (s >= d.src_cols) s = -1;
    }
    return s < 0 ? nullptr : static_cast<const T *>(d.src) + s * d.ld_src;
}

// Eight elements as they lie in memory.
template <typename T>
struct Raw {
    uint4 w[sizeof(T) / 2];
};

template <typename T>
__device__ __forceinline__ void widen(const Raw<T> &p, float (&x)[8]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            x[4 * i] = __uint_as_float(p.w[i].x);
            x[4 * i + 1] = __uint_as_float(p.w[i].y);
            x[4 * i + 2] = __uint_as_float(p.w[i].z);
            x[4 * i + 3] = __uint_as_float(p.w[i].w);
        }
    } else {
        const uint32_t w[4] = {p.w[0].x, p.w[0].y, p.w[0].z, p.w[0].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (std::is_same<T, __nv_bfloat16>::value) {
                x[2 * i] = __uint_as_float(w[i] << 16);
                x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
            } else {
                const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
                x[2 * i] = f.x;
                x[2 * i + 1] = f.y;
            }
        }
    }
}

// Bits of the largest |x| of eight raw elements as f32. NaN is passed over (all eight NaN: NaN), an infinity is not:
// at or above kInf, ask again with finite_top.
template <typename T>
__device__ __forceinline__ uint32_t top_bits(const Raw<T> &p) {
    if constexpr (sizeof(T) == 4) {
        float x[8];
        widen(p, x);
        float top = fabsf(x[0]);
#pragma unroll
        for (int i = 1; i < 8; ++i) top = fmaxf(top, fabsf(x[i]));
        return abs_bits(top);
    } else {
        using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
        const uint32_t w[4] = {p.w[0].x, p.w[0].y, p.w[0].z, p.w[0].w};
        T2 m = __habs2(*reinterpret_cast<const T2 *>(&w[0]));
#pragma unroll
        for (int i = 1; i < 4; ++i) m = __hmax2(m, __habs2(*reinterpret_cast<const T2 *>(&w[i])));
        const uint32_t b = *reinterpret_cast<const uint32_t *>(&m);
        if constexpr (std::is_same<T, __half>::value) {
            const float2 f = __half22float2(m);
            return abs_bits(fmaxf(f.x, f.y));
        } else {
            return max(b << 16, b & 0xffff0000u);
        }
    }
}
// Cold: blocks that hold values that are not finite.
template <typename T>
__device__ __noinline__ uint32_t finite_top(const Raw<T> p) {
    float x[8];
    widen(p, x);
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t b = abs_bits(x[i]);
        top = max(top, b < kInf ? b : 0u);
    }
    return top;
}
// The conversion saturates infinities: puts E4M3's NaN or E5M2's infinity in their places.
template <typename T, bool E5M2>
__device__ __noinline__ uint2 mend_infinities(const Raw<T> p, uint2 q) {
    float x[8];
    widen(p, x);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t b = __float_as_uint(x[i]);
        if ((b & 0x7fffffffu) == kInf) {
            const uint32_t v = ((b >> 24) & 0x80u) | (E5M2 ? 0x7cu : 0x7fu);
            const int s = 8 * (i & 3);
            uint32_t &w = i < 4 ? q.x : q.y;
            w = (w & ~(0xffu << s)) | (v << s);
        }
    }
    return q;
}

// Eight raw elements times inv[0..7] (or inv[0]) as FP8 bytes. `odd`: there may be infinities among them.
template <typename T, bool E5M2, int N>
__device__ __forceinline__ uint2 cast8(const Raw<T> &p, const float (&inv)[N], bool odd) {
    float x[8];
    widen(p, x);
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 y = __fmul2_rn(make_float2(x[2 * i], x[2 * i + 1]), make_float2(inv[(2 * i) % N], inv[(2 * i + 1) % N]));
        w[i] = cast2<E5M2>(y.x, y.y);
    }
    uint2 q = make_uint2(__byte_perm(w[0], w[1], 0x5410), __byte_perm(w[2], w[3], 0x5410));
    if (odd) q = mend_infinities<T, E5M2>(p, q);
    return q;
}

template <typename T>
__device__ __forceinline__ Raw<T> zero_raw() {
    Raw<T> p;
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) p.w[i] = make_uint4(0, 0, 0, 0);
    return p;
}
template <typename T>
__device__ __forceinline__ Raw<T> load_whole(const T *p) {
    Raw<T> q;
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) q.w[i] = reinterpret_cast<const uint4 *>(p)[i];
    return q;
}
// Element by element: the edge of the matrix, and addresses that are not multiples of 16 bytes.
template <typename T>
__device__ __noinline__ Raw<T> load_part(const T *col, int r, int rows) {
    T v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = r + i < rows ? col[r + i] : from_f32<T>(0.0f);
    Raw<T> p;
    memcpy(&p, v, sizeof(p));
    return p;
}
template <typename T, bool VEC>
__device__ __forceinline__ Raw<T> load_raw(const T *col, int r, int rows) {
    if (VEC && r + 8 <= rows) return load_whole<T>(col + r);
    return load_part<T>(col, r, rows);
}

// Vectors down the columns: 8 lanes hold one vector of 128 rows, each rows 8 s .. and 64 + 8 s .. of it (so that what the
// lanes of a vector share -- the maximum's last steps, the scale, the addresses -- is spread over 16 elements a lane).
// `lanes` (8 to 256) threads of a block take a column, DEPTH vectors of each on their way at once.
template <typename T, bool E5M2, bool VEC>
__global__ void __launch_bounds__(256, 4) k_quant_down(const QuantDesc d, int lanes) {
    constexpr int DEPTH = sizeof(T) == 4 ? 1 : 2;
    grid_dep_wait();
    grid_dep_launch();
    const int sub = threadIdx.x & 7, per = 256 / lanes;  // columns a block takes at once
    const uint32_t mates = 0xffu << (threadIdx.x & 24);
    const int first = (threadIdx.x % lanes) / 8 * 128 + sub * 8, step = lanes * 16;
    const long long sc_step = static_cast<long long>(step / 128) * d.ld_scale;
    for (long long c = static_cast<long long>(blockIdx.x) * per + threadIdx.x / lanes; c < d.cols; c += static_cast<long long>(gridDim.x) * per) {
        const T *src = source<T>(d, static_cast<int>(c));
        uint8_t *dst = static_cast<uint8_t *>(d.dst) + c * d.ld_dst;
        float *sc = d.scale + c + static_cast<long long>(first / 128) * d.ld_scale;
        for (int r0 = first; r0 - sub * 8 < d.rows; r0 += DEPTH * step) {
            Raw<T> raw[DEPTH][2];
            // Whole vectors in all steps: no branch between the loads.
            const bool whole = VEC && src != nullptr && r0 - sub * 8 + (DEPTH - 1) * step + 128 <= d.rows;
            if (whole) {
#pragma unroll
                for (int i = 0; i < DEPTH; ++i) {
                    raw[i][0] = load_whole<T>(src + r0 + i * step);
                    raw[i][1] = load_whole<T>(src + r0 + i * step + 64);
                }
            } else {
#pragma unroll
                for (int i = 0; i < DEPTH; ++i)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int r = r0 + i * step + 64 * h;
                        raw[i][h] = src != nullptr && r < d.rows ? load_raw<T, VEC>(src, r, d.rows) : zero_raw<T>();
                    }
            }
#pragma unroll
            for (int i = 0; i < DEPTH; ++i) {
                const int r = r0 + i * step;
                if (!whole && r - sub * 8 >= d.rows) break;  // the same answer in all 8 lanes
                uint32_t top = max(top_bits(raw[i][0]), top_bits(raw[i][1]));
#pragma unroll
                for (int s = 4; s > 0; s >>= 1) top = max(top, __shfl_xor_sync(mates, top, s));
                const bool odd = top >= kInf;
                if (odd) {
                    top = max(finite_top(raw[i][0]), finite_top(raw[i][1]));
#pragma unroll
                    for (int s = 4; s > 0; s >>= 1) top = max(top, __shfl_xor_sync(mates, top, s));
                }
                const int e = scale_exp<E5M2>(top);
                if (sub == 0) *sc = pow2(e);
                sc += sc_step;
                const float inv[1] = {pow2(-e)};
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint2 q = cast8<T, E5M2>(raw[i][h], inv, odd);
                    if (whole) *reinterpret_cast<uint2 *>(dst + r + 64 * h) = q;
                    else if (r + 64 * h < d.rows) store8<VEC>(dst, r + 64 * h, d.rows, q);
                }
            }
        }
    }
}

// Tiles of 128 columns: vectors along the rows (BLK false, 64 rows a tile) or
// 128 x 128 blocks. A thread holds 8 rows of COLS columns, as they were loaded.
template <typename T, bool E5M2, bool VEC, bool BLK>
__global__ void __launch_bounds__(256, sizeof(T) == 4 ? 2 : 3) k_quant_tile(const QuantDesc d) {
    constexpr int ROWS = BLK ? 128 : 64, LANES = ROWS / 8, STEP = 256 / LANES, COLS = 128 / STEP;
    __shared__ uint32_t red[8][ROWS];
    __shared__ __align__(16) uint32_t all[ROWS];
    grid_dep_wait();
    grid_dep_launch();
    const int rt_n = (d.rows + ROWS - 1) / ROWS, ct_n = (d.cols + 127) / 128;
    const long long tasks = static_cast<long long>(rt_n) * ct_n;
    const int lr = threadIdx.x % LANES, lc = threadIdx.x / LANES, warp = threadIdx.x / 32;
    for (long long task = blockIdx.x; task < tasks; task += gridDim.x) {
        const int ct = static_cast<int>(task / rt_n), rt = static_cast<int>(task - static_cast<long long>(ct) * rt_n);
        const int r = rt * ROWS + lr * 8;
        Raw<T> x[COLS];
        // Whole tiles load without a branch between the loads, so that all of them are on their way at once.
        const bool whole = VEC && d.index == nullptr && (rt + 1) * ROWS <= d.rows && (ct + 1) * 128 <= d.cols;
        if (whole) {
            const T *src = static_cast<const T *>(d.src) + (static_cast<long long>(ct) * 128 + lc) * d.ld_src + r;
#pragma unroll
            for (int i = 0; i < COLS; ++i) x[i] = load_whole<T>(src + static_cast<long long>(i * STEP) * d.ld_src);
        } else {
#pragma unroll
            for (int i = 0; i < COLS; ++i) {
                const int c = ct * 128 + lc + i * STEP;
                const T *src = c < d.cols ? source<T>(d, c) : nullptr;
                x[i] = src != nullptr ? load_raw<T, VEC>(src, r, d.rows) : zero_raw<T>();
            }
        }
        uint32_t top[BLK ? 1 : 8];
        bool odd = false;
        for (int pass = 0; pass < 2; ++pass) {  // a second time over the finite values, if there are others
            if constexpr (BLK) {
                uint32_t m = 0;
#pragma unroll
                for (int i = 0; i < COLS; ++i) m = max(m, pass == 0 ? top_bits(x[i]) : finite_top(x[i]));
                m = __reduce_max_sync(0xffffffffu, m);
                if ((threadIdx.x & 31) == 0) red[warp][0] = m;
                __syncthreads();
#pragma unroll
                for (int w = 0; w < 8; ++w) m = max(m, red[w][0]);
                top[0] = m;
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) top[j] = 0;
#pragma unroll
                for (int i = 0; i < COLS; ++i) {
                    float v[8];
                    widen(x[i], v);
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const uint32_t b = abs_bits(v[j]);
                        top[j] = max(top[j], pass == 1 && b >= kInf ? 0u : b);
                    }
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    top[j] = max(top[j], __shfl_xor_sync(0xffffffffu, top[j], 8));
                    top[j] = max(top[j], __shfl_xor_sync(0xffffffffu, top[j], 16));
                    if ((threadIdx.x & 31) < 8) red[warp][lr * 8 + j] = top[j];
                }
                __syncthreads();
                if (threadIdx.x < ROWS) {
                    uint32_t m = red[0][threadIdx.x];
#pragma unroll
                    for (int w = 1; w < 8; ++w) m = max(m, red[w][threadIdx.x]);
                    all[threadIdx.x] = m;
                }
                __syncthreads();
                const uint4 lo = *reinterpret_cast<const uint4 *>(all + lr * 8), hi = *reinterpret_cast<const uint4 *>(all + lr * 8 + 4);
                top[0] = lo.x; top[1] = lo.y; top[2] = lo.z; top[3] = lo.w;
                top[4] = hi.x; top[5] = hi.y; top[6] = hi.z; top[7] = hi.w;
            }
            bool any = false;
#pragma unroll
            for (int j = 0; j < (BLK ? 1 : 8); ++j) any |= top[j] >= kInf;
            if (!__syncthreads_or(any)) break;
            odd = true;
        }
        float inv[BLK ? 1 : 8];
#pragma unroll
        for (int j = 0; j < (BLK ? 1 : 8); ++j) {
            const int e = scale_exp<E5M2>(top[j]);
            inv[j] = pow2(-e);
            if constexpr (BLK) {
                if (threadIdx.x == 0) d.scale[rt + ct * d.ld_scale] = pow2(e);
            } else {
                if (lc == 0 && r + j < d.rows) d.scale[r + j + ct * d.ld_scale] = pow2(e);
            }
        }
        uint8_t *dst = static_cast<uint8_t *>(d.dst) + (static_cast<long long>(ct) * 128 + lc) * d.ld_dst;
#pragma unroll
        for (int i = 0; i < COLS; ++i) {
            const uint2 q = cast8<T, E5M2>(x[i], inv, odd);
            uint8_t *col = dst + static_cast<long long>(i * STEP) * d.ld_dst;
            if (whole) *reinterpret_cast<uint2 *>(col + r) = q;
            else if (ct * 128 + lc + i * STEP < d.cols) store8<VEC>(col, r, d.rows, q);
        }
    }
}

template <typename T, bool E5M2, bool VEC>
static cudaError_t launch(Context &ctx, const QuantDesc &d) {
    cudaError_t e;
    if (!d.blk && d.axis == 0) {
        const int depth = sizeof(T) == 4 ? 1 : 2;  // the kernel's DEPTH
        // A warp a column (finding the source column then costs little); more threads where columns are few, fewer where
        // they are short.
        int lanes = 8;
        while (lanes < 256 && lanes * 16 * depth < d.rows && (lanes < 32 || static_cast<long long>(d.cols) * lanes < 2048LL * ctx.sm_count))
            lanes *= 2;
        const long long blocks = (static_cast<long long>(d.cols) * lanes + 255) / 256, most = 64LL * ctx.sm_count;
        e = launch_pdl(k_quant_down<T, E5M2, VEC>, dim3(static_cast<unsigned>(blocks < most ? blocks : most)), dim3(256), 0, ctx.stream, 1, d, lanes);
    } else {
        const int rows = d.blk ? 128 : 64;
        const long long blocks = static_cast<long long>((d.rows + rows - 1) / rows) * ((d.cols + 127) / 128), most = 64LL * ctx.sm_count;
        auto kern = d.blk ? k_quant_tile<T, E5M2, VEC, true> : k_quant_tile<T, E5M2, VEC, false>;
        e = launch_pdl(kern, dim3(static_cast<unsigned>(blocks < most ? blocks : most)), dim3(256), 0, ctx.stream, 1, d);
    }
    ctx.launches++;
    return e;
}

}  // namespace quant

cudaError_t launch_quantize(Context &ctx, const QuantDesc &d) {
    ctx.last_kernels |= GS_KERNEL_QUANTIZE;
    return with_float_type(d.src_type, [&](auto z) {
        using T = decltype(z);
        const bool vec = reinterpret_cast<uintptr_t>(d.src) % 16 == 0 && (d.ld_src * sizeof(T)) % 16 == 0 &&
                         reinterpret_cast<uintptr_t>(d.dst) % 8 == 0 && d.ld_dst % 8 == 0;
        if (d.e5m2) return vec ? quant::launch<T, true, true>(ctx, d) : quant::launch<T, true, false>(ctx, d);
        return vec ? quant::launch<T, false, true>(ctx, d) : quant::launch<T, false, false>(ctx, d);
    });
}

}  // namespace gs
