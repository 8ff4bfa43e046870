// Kernel arguments of the operators over 8-bit blocks (ptowsp_blocks.h) and of
// paged_norm_rotate (ptowsp_rotate.h), shared by the host library and the
// kernels.  Strides are in elements.
#pragma once

namespace ptowsp {

constexpr int kScaleBlock = 128;  // columns, and rows of weights, that share a scale

struct QuantizeArgs {
    const char* x;
    char* codes;
    float* scales;
    long long s_x, s_codes;  // row
    long long s_scales[2];   // row, block
    long long rows, cols;
    unsigned int blocks;     // of a row
    unsigned int many;       // blocks of columns in all
};

struct MatmulArgs {
    const char* a;
    const char* b;
    const float* a_scale;
    const float* b_scale;
    char* out;
    long long s_a, s_b, s_out;         // row
    long long s_as[2], s_bs[2];        // row (of b: block of rows), block
    long long M, N, K;
    int stages;                        // blocks of K
    int tiles_m, tiles_n;
    int splits;                        // workgroups that share a tile's stages
    float* parts;                      // their sums, [split, M, N], if they are several
};

struct RotateArgs {
    const char* x[2];  // queries, keys
    char* out[2];
    const char* weight[2];
    const float* cos;
    const float* sin;
    const int* lengths;
    const int* starts;
    const int* offsets;  // null: none
    long long s_x[2][2], s_out[2][2];  // row, head
    long long s_cos, s_sin, s_lengths, s_starts, s_offsets;
    long long batch, rows, positions;
    int heads[2];
    float eps;
    int* err;  // 8: starts or a position out of range
};

}  // namespace ptowsp
