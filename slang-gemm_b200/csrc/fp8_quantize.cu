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
// registers between the maximum and the cast.
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

// Eight values times 2^-e as FP8 bytes. `odd`: the block holds a value that is not finite.
template <bool E5M2>
__device__ __forceinline__ uint2 cast8(const float (&x)[8], float inv, bool odd) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = cast2<E5M2>(__fmul_rn(x[2 * i], inv), __fmul_rn(x[2 * i + 1], inv));
    if (odd) {  // the conversion saturates infinities: put E4M3's NaN or E5M2's infinity in their places
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t b = __float_as_uint(x[i]);
            if ((b & 0x7fffffffu) == kInf) {
                const uint32_t q = ((b >> 24) & 0x80u) | (E5M2 ? 0x7cu : 0x7fu);
                const int s = 8 * (i & 1);
                w[i / 2] = (w[i / 2] & ~(0xffu << s)) | (q << s);
            }
        }
    }
    return make_uint2(w[0] | (w[1] << 16), w[2] | (w[3] << 16));
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

// amax as f32 bits of eight raw elements: of all of them, or (second time, where that is not finite) of the finite ones.
__device__ __forceinline__ uint32_t top_bits(const Pack<float, 8> &p, bool finite) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t b = abs_bits(p.v[i]);
        top = max(top, finite && b >= kInf ? 0u : b);
    }
    return top;
}
template <typename T>
__device__ __forceinline__ uint32_t top_bits(const Pack<T, 8> &p, bool finite) {  // 16-bit types: two at a time, as integers
    static_assert(sizeof(T) == 2, "two elements to a word");
    constexpr uint32_t inf = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
    const uint32_t *w = reinterpret_cast<const uint32_t *>(&p);
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t b = w[i] & 0x7fff7fffu;
        if (finite) {
            if ((b & 0xffffu) >= inf) b &= 0xffff0000u;
            if ((b >> 16) >= inf) b &= 0xffffu;
        }
        top = __vmaxu2(top, b);
    }
    T v;
    const uint16_t h = static_cast<uint16_t>(max(top & 0xffffu, top >> 16));
    memcpy(&v, &h, 2);
    return __float_as_uint(to_f32(v));
}

template <typename T, bool VEC>
__device__ __forceinline__ Pack<T, 8> load_raw(const T *col, int r, int rows) {
    Pack<T, 8> p;
    if (VEC && r + 8 <= rows) {
        p = load_pack<T, 8>(col + r);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) p.v[i] = r + i < rows ? col[r + i] : from_f32<T>(0.0f);
    }
    return p;
}
template <typename T>
__device__ __forceinline__ Pack<T, 8> zero_raw() {
    Pack<T, 8> p;
#pragma unroll
    for (int i = 0; i < 8; ++i) p.v[i] = from_f32<T>(0.0f);
    return p;
}
template <typename T>
__device__ __forceinline__ void widen(const Pack<T, 8> &p, float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_f32(p.v[i]);
}

// Vectors down the columns: 16 lanes hold one vector of 128 rows. `lanes` (16 to 256) threads of a block take a
// column, DEPTH vectors of each thread's on their way at once.
template <typename T, bool E5M2, bool VEC>
__global__ void __launch_bounds__(256) k_quant_down(const QuantDesc d, int lanes) {
    constexpr int DEPTH = sizeof(T) == 4 ? 2 : 4;
    grid_dep_wait();
    grid_dep_launch();
    const int sub = threadIdx.x & 15, per = 256 / lanes;  // columns a block takes at once
    const uint32_t half = 0xffffu << (threadIdx.x & 16);
    for (long long c = static_cast<long long>(blockIdx.x) * per + threadIdx.x / lanes; c < d.cols; c += static_cast<long long>(gridDim.x) * per) {
        const T *src = source<T>(d, static_cast<int>(c));
        uint8_t *dst = static_cast<uint8_t *>(d.dst) + c * d.ld_dst;
        const int first = (threadIdx.x % lanes) * 8, step = lanes * 8;
        for (int r0 = first; r0 - sub * 8 < d.rows; r0 += DEPTH * step) {
            Pack<T, 8> raw[DEPTH];
#pragma unroll
            for (int i = 0; i < DEPTH; ++i) {
                const int r = r0 + i * step;
                raw[i] = src != nullptr && r < d.rows ? load_raw<T, VEC>(src, r, d.rows) : zero_raw<T>();
            }
#pragma unroll
            for (int i = 0; i < DEPTH; ++i) {
                const int r = r0 + i * step;
                if (r - sub * 8 >= d.rows) break;  // the same answer in all 16 lanes
                uint32_t top = top_bits(raw[i], false);
#pragma unroll
                for (int s = 8; s > 0; s >>= 1) top = max(top, __shfl_xor_sync(half, top, s));
                const bool odd = top >= kInf;
                if (odd) {
                    top = top_bits(raw[i], true);
#pragma unroll
                    for (int s = 8; s > 0; s >>= 1) top = max(top, __shfl_xor_sync(half, top, s));
                }
                const int e = scale_exp<E5M2>(top);
                if (sub == 0) d.scale[c + (r / 128) * d.ld_scale] = pow2(e);
                float x[8];
                widen(raw[i], x);
                if (r < d.rows) store8<VEC>(dst, r, d.rows, cast8<E5M2>(x, pow2(-e), odd));
            }
        }
    }
}

// Tiles of 128 columns: vectors along the rows (BLK false, 64 rows a tile) or
// 128 x 128 blocks. A thread holds 8 rows of COLS columns, as they were loaded.
template <typename T, bool E5M2, bool VEC, bool BLK>
__global__ void __launch_bounds__(256, sizeof(T) == 4 && BLK ? 2 : 3) k_quant_tile(const QuantDesc d) {
    constexpr int ROWS = BLK ? 128 : 64, LANES = ROWS / 8, STEP = 256 / LANES, COLS = 128 / STEP;
    __shared__ uint32_t red[8][ROWS];
    grid_dep_wait();
    grid_dep_launch();
    const int rt_n = (d.rows + ROWS - 1) / ROWS, ct_n = (d.cols + 127) / 128;
    const long long tasks = static_cast<long long>(rt_n) * ct_n;
    const int lr = threadIdx.x % LANES, lc = threadIdx.x / LANES, warp = threadIdx.x / 32;
    for (long long task = blockIdx.x; task < tasks; task += gridDim.x) {
        const int ct = static_cast<int>(task / rt_n), rt = static_cast<int>(task - static_cast<long long>(ct) * rt_n);
        const int r = rt * ROWS + lr * 8;
        Pack<T, 8> x[COLS];
        // Whole tiles load without a branch between the loads, so that all of them are on their way at once.
        const bool whole = VEC && d.index == nullptr && (rt + 1) * ROWS <= d.rows && (ct + 1) * 128 <= d.cols;
        if (whole) {
            const T *src = static_cast<const T *>(d.src) + (static_cast<long long>(ct) * 128 + lc) * d.ld_src + r;
#pragma unroll
            for (int i = 0; i < COLS; ++i) x[i] = load_pack<T, 8>(src + static_cast<long long>(i * STEP) * d.ld_src);
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
                for (int i = 0; i < COLS; ++i) m = max(m, top_bits(x[i], pass == 1));
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
#pragma unroll
                for (int j = 0; j < 8; ++j)
#pragma unroll
                    for (int w = 0; w < 8; ++w) top[j] = max(top[j], red[w][lr * 8 + j]);
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
#pragma unroll
        for (int i = 0; i < COLS; ++i) {
            const int c = ct * 128 + lc + i * STEP;
            if (c >= d.cols) continue;
            float y[8];
            widen(x[i], y);
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] = __fmul_rn(y[j], inv[BLK ? 0 : j]);  // keeps NaN and infinity
            store8<VEC>(static_cast<uint8_t *>(d.dst) + static_cast<long long>(c) * d.ld_dst, r, d.rows, cast8<E5M2>(y, 1.0f, odd));
        }
    }
}

template <typename T, bool E5M2, bool VEC>
static cudaError_t launch(Context &ctx, const QuantDesc &d) {
    cudaError_t e;
    if (!d.blk && d.axis == 0) {
        int lanes = 16;
        while (lanes < 256 && lanes * 8 < d.rows) lanes *= 2;
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
