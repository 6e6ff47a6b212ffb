// gs_fp8.h -- descriptors of the FP8 block-scaled products, the quantiser and
// the routed-expert operators, as the kernels see them after the C-ABI layer
// (fp8_capi.cu) has validated them. Pointers are device pointers.
#pragma once
#include <cstdint>

#include "gs_internal.h"

namespace gs {

struct GemmFp8Desc {
    int trans_a, trans_b;
    int m, n, k;
    int groups;                    // 0 = dense
    int ragged;                    // GS_GROUP_N / GS_GROUP_K when groups > 0
    const int32_t *offsets;        // groups + 1
    const void *A; long long lda, stride_a; int a_e5m2;
    const float *sa; int a_vec; long long ldsa, stride_sa;
    const void *B; long long ldb; int b_e5m2;
    const float *sb; int b_vec; long long ldsb;
    void *C; long long ldc, stride_c;
    OutKind out_kind;
    Epilogue ep;
};

namespace fp8 {
// Tile of a product: bn columns, cg CTAs (cg * 128 rows), split K slices over a cluster.
struct Tile { int cg, bn, split; };
Tile choose_tile(const GemmFp8Desc &d, int sm_count);
}  // namespace fp8

struct QuantDesc {
    int blk;                       // 1 = 128 x 128 blocks, 0 = vectors of 128
    int axis;                      // vectors: 0 = down a column, 1 = along a row
    int rows, cols;
    const void *src; int src_type; long long ld_src; int src_cols;
    const int32_t *index; int index_div;
    void *dst; int e5m2; long long ld_dst;
    float *scale; long long ld_scale;
};

struct RouteDesc {
    int tokens, experts, top_k;
    const void *logits; int type; long long ld;
    const float *bias;
    int sigmoid, groups, top_groups, renorm;
    int group_size; uint32_t group_magic;  // expert e's group is e * group_magic >> 20 (e and group_size <= 1024)
    float scale;
    const int32_t *token_count;
    int align;
    int32_t *ids; float *weights;
    int32_t *offsets, *slot_row, *row_slot;  // offsets null: choice and weights only
    int rows;
    int32_t *hist;                 // workspace: route_blocks x experts counts
};
// Blocks of the two-kernel plan (0: the one-block kernel, no workspace).
int route_blocks(int tokens, int top_k);

struct RouteBwdDesc {
    int tokens, experts, top_k;
    const void *logits; int type; long long ld;
    const int32_t *ids; const float *dweights;
    int sigmoid, renorm;
    float scale;
    void *dlogits; int dtype; long long ldd;
};

struct CombineDesc {
    int tokens, top_k, hidden, rows;
    const void *y; int type; long long ldy;
    const int32_t *slot_row, *row_slot;
    const float *weights;          // null = 1
    void *out; int out_type; long long ldo;          // forward
    const void *dout; long long lddo;                // backward
    void *dy; long long lddy;
    float *dweights;
};

cudaError_t launch_gemm_fp8(Context &ctx, const GemmFp8Desc &d);
cudaError_t launch_quantize(Context &ctx, const QuantDesc &d);
cudaError_t launch_route(Context &ctx, const RouteDesc &d);
cudaError_t launch_route_backward(Context &ctx, const RouteBwdDesc &d);
cudaError_t launch_combine(Context &ctx, const CombineDesc &d);
cudaError_t launch_combine_backward(Context &ctx, const CombineDesc &d);

}  // namespace gs
