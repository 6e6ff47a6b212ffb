// moe_combine.cu -- sums the experts' rows back to their tokens, and the gradient.
//
//   out[t] = sum over j of w[t, j] * y[slot_row[t, j]]          (in order of j)
//   dy[r]  = w[row_slot[r]] * dout[row_slot[r] / top_k]   (0 for a row of no slot)
//   dw[t, j] = <dout[t], y[slot_row[t, j]]>
//
// Sums are f32 with one rounding at the end and a fixed order. Bound by memory:
// 16-byte loads, up to four rows of a token in flight at once. bf16, 8192 tokens,
// top_k 8, 4096 columns: 104 us forward (5.8 TB/s); 4096 tokens, top_k 4: 67 us
// backward (5.5 TB/s), a warp a row (a block a row with its barrier: 78 us).
#include "gs_float.cuh"
#include "gs_fp8.h"

namespace gs {
namespace combine {

// Elements a thread handles at once: 16 bytes of the 16-bit types, 32 of f32.
constexpr int V = 8;

template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T *p, int h, int hidden, float (&x)[V]) {
    if (VEC && h + V <= hidden) {
        const Pack<T, V> q = load_pack<T, V>(p + h);
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = to_f32(q.v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = h + i < hidden ? to_f32(p[h + i]) : 0.0f;
    }
}
template <typename T, bool VEC>
__device__ __forceinline__ void store8(T *p, int h, int hidden, const float (&x)[V]) {
    if (VEC && h + V <= hidden) {
        Pack<T, V> q;
#pragma unroll
        for (int i = 0; i < V; ++i) q.v[i] = from_f32<T>(x[i]);
        store_pack<T, V>(p + h, q);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (h + i < hidden) p[h + i] = from_f32<T>(x[i]);
    }
}

// A thread sums V columns of one token; the token's rows and weights are read first, then up to four of its rows'
// columns are on their way at once.
template <typename T, typename TO, bool VEC>
__global__ void __launch_bounds__(256) k_combine(const CombineDesc d, int lanes) {
    grid_dep_wait();
    grid_dep_launch();
    const int per = 256 / lanes;  // tokens a block takes at once
    const int chunks = (d.hidden + V - 1) / V, splits = (chunks + lanes - 1) / lanes;
    const long long tasks = (static_cast<long long>(d.tokens) + per - 1) / per * splits;
    for (long long i = blockIdx.x; i < tasks; i += gridDim.x) {
        const long long t = i / splits * per + threadIdx.x / lanes;
        const int h = (static_cast<int>(i % splits) * lanes + threadIdx.x % lanes) * V;
        if (t >= d.tokens || h >= d.hidden) continue;
        const int32_t *rows = d.slot_row + t * d.top_k;
        const float *weights = d.weights != nullptr ? d.weights + t * d.top_k : nullptr;
        float sum[V] = {};
        for (int j = 0; j < d.top_k; j += 4) {
            int r[4];
            float w[4], x[4][V];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                r[q] = j + q < d.top_k ? rows[j + q] : -1;
                if (r[q] >= d.rows) r[q] = -1;
                w[q] = weights != nullptr && r[q] >= 0 ? weights[j + q] : 1.0f;
            }
            if (VEC && h + V <= d.hidden && min(min(r[0], r[1]), min(r[2], r[3])) >= 0) {  // the usual case, without a branch between the loads
                Pack<T, V> raw[4];
#pragma unroll
                for (int q = 0; q < 4; ++q) raw[q] = load_pack<T, V>(static_cast<const T *>(d.y) + r[q] * d.ldy + h);
#pragma unroll
                for (int q = 0; q < 4; ++q)
#pragma unroll
                    for (int v = 0; v < V; ++v) sum[v] = fmaf(w[q], to_f32(raw[q].v[v]), sum[v]);
            } else {
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    if (r[q] < 0) continue;
                    load8<T, VEC>(static_cast<const T *>(d.y) + r[q] * d.ldy, h, d.hidden, x[q]);
#pragma unroll
                    for (int v = 0; v < V; ++v) sum[v] = fmaf(w[q], x[q][v], sum[v]);
                }
            }
        }
        store8<TO, VEC>(static_cast<TO *>(d.out) + t * d.ldo, h, d.hidden, sum);
    }
}

// A warp handles one row of y: its dy, and its slot's weight gradient; four steps of 256 columns on their way at once.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) k_combine_backward(const CombineDesc d) {
    constexpr int DEPTH = sizeof(T) == 4 ? 2 : 4;
    grid_dep_wait();
    grid_dep_launch();
    const int lane = threadIdx.x & 31;
    const long long slots = static_cast<long long>(d.tokens) * d.top_k;
    for (long long i = blockIdx.x * 256LL + threadIdx.x; i < slots; i += gridDim.x * 256LL) {
        const int r = d.slot_row[i];
        if (r < 0 || r >= d.rows) d.dweights[i] = 0.0f;  // a slot without a row
    }
    for (long long r = blockIdx.x * 8LL + (threadIdx.x >> 5); r < d.rows; r += gridDim.x * 8LL) {
        const int slot = d.row_slot[r];
        T *dy = static_cast<T *>(d.dy) + r * d.lddy;
        if (slot < 0 || slot >= slots) {
            const float zero[V] = {};
            for (int h = lane * V; h < d.hidden; h += 32 * V) store8<T, VEC>(dy, h, d.hidden, zero);
            continue;
        }
        const float w = d.weights[slot];
        const T *y = static_cast<const T *>(d.y) + r * d.ldy;
        const T *g = static_cast<const T *>(d.dout) + static_cast<long long>(slot / d.top_k) * d.lddo;
        float dot = 0.0f;
        int h = lane * V;
        if (VEC) {
            for (; h - lane * V + DEPTH * 32 * V <= d.hidden; h += DEPTH * 32 * V) {
                Pack<T, V> a[DEPTH], b[DEPTH];
#pragma unroll
                for (int i = 0; i < DEPTH; ++i) {
                    a[i] = load_pack<T, V>(g + h + i * 32 * V);
                    b[i] = load_pack<T, V>(y + h + i * 32 * V);
                }
#pragma unroll
                for (int i = 0; i < DEPTH; ++i) {
                    Pack<T, V> o;
#pragma unroll
                    for (int v = 0; v < V; ++v) {
                        const float x = to_f32(a[i].v[v]);
                        dot = fmaf(x, to_f32(b[i].v[v]), dot);
                        o.v[v] = from_f32<T>(w * x);
                    }
                    store_pack<T, V>(dy + h + i * 32 * V, o);
                }
            }
        }
        for (; h < d.hidden; h += 32 * V) {
            float a[V], b[V], o[V];
            load8<T, VEC>(g, h, d.hidden, a);
            load8<T, VEC>(y, h, d.hidden, b);
#pragma unroll
            for (int v = 0; v < V; ++v) {
                dot = fmaf(a[v], b[v], dot);
                o[v] = w * a[v];
            }
            store8<T, VEC>(dy, h, d.hidden, o);
        }
#pragma unroll
        for (int s = 16; s > 0; s >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, s);
        if (lane == 0) d.dweights[slot] = dot;
    }
}

static bool aligned(const void *p, long long ld, size_t es) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && (ld * es) % 16 == 0; }

}  // namespace combine

cudaError_t launch_combine(Context &ctx, const CombineDesc &d) {
    ctx.last_kernels |= GS_KERNEL_COMBINE;
    const int chunks = (d.hidden - 1) / combine::V + 1;
    int lanes = 32;  // threads to a token
    while (lanes < 256 && lanes < chunks) lanes *= 2;
    const int per = 256 / lanes;
    const long long want = (static_cast<long long>(d.tokens) + per - 1) / per * ((chunks + lanes - 1) / lanes), most = 64LL * ctx.sm_count;
    const unsigned blocks = static_cast<unsigned>(want < most ? want : most);
    return with_float_type(d.type, [&](auto z) {
        return with_float_type(d.out_type, [&](auto zo) {
            using T = decltype(z);
            using TO = decltype(zo);
            const bool vec = combine::aligned(d.y, d.ldy, sizeof(T)) && combine::aligned(d.out, d.ldo, sizeof(TO));
            const cudaError_t e = launch_pdl(vec ? combine::k_combine<T, TO, true> : combine::k_combine<T, TO, false>, dim3(blocks),
                                             dim3(256), 0, ctx.stream, 1, d, lanes);
            ctx.launches++;
            return e;
        });
    });
}

cudaError_t launch_combine_backward(Context &ctx, const CombineDesc &d) {
    ctx.last_kernels |= GS_KERNEL_COMBINE;
    const long long want = (static_cast<long long>(d.rows) + 7) / 8, most = 32LL * ctx.sm_count;
    const unsigned blocks = static_cast<unsigned>(want < 1 ? 1 : want < most ? want : most);
    return with_float_type(d.type, [&](auto z) {
        using T = decltype(z);
        const bool vec = combine::aligned(d.y, d.ldy, sizeof(T)) && combine::aligned(d.dout, d.lddo, sizeof(T)) &&
                         combine::aligned(d.dy, d.lddy, sizeof(T));
        const cudaError_t e = launch_pdl(vec ? combine::k_combine_backward<T, true> : combine::k_combine_backward<T, false>, dim3(blocks),
                                         dim3(256), 0, ctx.stream, 1, d);
        ctx.launches++;
        return e;
    });
}

}  // namespace gs
