// The product behind scenerf_hip_linear_*: C[i][j] = sum_k A(i, k) B(j, k), with the layer's epilogue.
#pragma once
#include "rowops.h"

struct LinArgs {
    const void* A; const void* B;        // A(i, k) = A[i * a_i + k * a_k], B(j, k) = B[j * b_j + k * b_k]; one of each pair is 1
    long a_i, a_k, b_j, b_k;
    int M, N, K;
    int a_ext, b_ext;                    // staged kernel, operand read across: i (j) may be read up to here, a whole number of 16-byte pieces
    // epilogue: v = acc * row_scale[i] * col_scale[j] + bias[j]; z = v; out = act(v) + residual
    const float* row_scale; const float* col_scale;
    const void* bias; const void* residual; long ld_residual;
    void* out; void* z;                  // dense [M][N]
    float* part;                         // not NULL: the raw sums of split s go to part[s][M][N] instead
    int act, tiles_i, tiles_j, splits, k_split;     // k_split: contraction elements per split
    const void* A2;                      // not NULL (16 bits, backward): laid out like A, its products are added to A's
    const float* unscale;                // not NULL (fp16, backward): A and A2 hold their values times 1 / *unscale, a power of two
};

template <typename O, int W> __device__ static inline void act_any(int act, float (&v)[W]) {
    constexpr bool FINE = O::code == SCENERF_T_F32;
    if (act == SCENERF_ACT_RELU) act_fwd<SCENERF_ACT_RELU, W, FINE>(v);
    else if (act == SCENERF_ACT_GELU) act_fwd<SCENERF_ACT_GELU, W, FINE>(v);
    else if (act == SCENERF_ACT_SILU) act_fwd<SCENERF_ACT_SILU, W, FINE>(v);
}
// z as it is kept for the backward pass, in O.  A positive z that rounds to zero (fp16) is kept as the smallest positive value: relu's
// slope there is 1, and the other slopes do not notice.  (A finite z past O's range is kept as an infinity: act_slope.)
template <typename O> __device__ static inline float keep_z(float v) {
    if constexpr (O::code == SCENERF_T_F16) return v > 0.f && v < 5.9604645e-8f ? 5.9604645e-8f : v;
    return v;
}
template <typename O> __device__ static inline void epilogue_one(const LinArgs& p, long i, int j, float v) {
    typedef typename O::raw raw;
    if (p.row_scale) v = v * p.row_scale[i] * p.col_scale[j];
    if (p.unscale) v *= *p.unscale;
    if (p.bias) v += O::to_f32(((const raw*)p.bias)[j]);
    if (p.z) ((raw*)p.z)[i * p.N + j] = O::from_f32(keep_z<O>(v));
    float one[1] = {v};
    act_any<O, 1>(p.act, one);
    v = one[0];
    if (p.residual) v += O::to_f32(((const raw*)p.residual)[i * p.ld_residual + j]);
    ((raw*)p.out)[i * p.N + j] = O::from_f32(v);
}
// W = 16 / sizeof(O::raw) neighbouring elements, of which n are inside the row: what depends on the columns alone, then one row's (its
// residual in hand)
template <typename O, int W, bool WHOLE> struct EpilogueCols {
    float bias[W], scale[W];
    __device__ inline void load(const LinArgs& p, int j, int n) {
#pragma unroll
        for (int e = 0; e < W; ++e) bias[e] = 0.f;
        if (p.bias) load_some<O, W, WHOLE>((const typename O::raw*)p.bias + j, n, p.N % W, bias);
        if (p.row_scale) load_some<TypeF32, W, WHOLE>(p.col_scale + j, n, p.N % W, scale);
    }
};
template <typename O, int W, bool WHOLE> __device__ static inline uint4 residual_piece(const LinArgs& p, long i, int j, int n) {
    typedef typename O::raw raw;
    const raw* at = (const raw*)p.residual + i * p.ld_residual + j;
    if (WHOLE || n >= W) return load16(at);
    float v[W];
    load_some<O, W>(at, n, p.N % W, v);
    if constexpr (sizeof(raw) == 4) return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
    else return make_uint4(pack2<O>(v[0], v[1]), pack2<O>(v[2], v[3]), pack2<O>(v[4], v[5]), pack2<O>(v[6], v[7]));     // (exact)
}
template <typename O, int W, bool WHOLE>
__device__ static inline void epilogue_vec(const LinArgs& p, const EpilogueCols<O, W, WHOLE>& ec, long i, int j, int n, uint4 res, float (&v)[W]) {
    typedef typename O::raw raw;
    if (p.row_scale) {
        const float s = p.row_scale[i];
#pragma unroll
        for (int e = 0; e < W; ++e) v[e] = v[e] * s * ec.scale[e];
    }
    if (p.unscale) {
        const float s = *p.unscale;
#pragma unroll
        for (int e = 0; e < W; ++e) v[e] *= s;
    }
#pragma unroll
    for (int e = 0; e < W; ++e) v[e] += ec.bias[e];
    if (p.z) {
        float t[W];
#pragma unroll
        for (int e = 0; e < W; ++e) t[e] = keep_z<O>(v[e]);
        store_some<O, W, WHOLE>((raw*)p.z + i * p.N + j, n, p.N % W, t);
    }
    act_any<O, W>(p.act, v);
    if (p.residual) {
        float t[W];
        unpack16<O>(res, t);
#pragma unroll
        for (int e = 0; e < W; ++e) v[e] += t[e];
    }
    store_some<O, W, WHOLE>((raw*)p.out + i * p.N + j, n, p.N % W, v);
}

// Tile shapes of the staged kernel (linear_tile.h): rows x columns of the result per workgroup
enum LinTile { LIN_256x256, LIN_128x128, LIN_64x64, LIN_128x32, LIN_TILES };
static const int kLinTileRows[LIN_TILES] = {256, 128, 64, 128}, kLinTileCols[LIN_TILES] = {256, 128, 64, 32};
#define LIN_CHUNK_BYTES 128             // of the contraction per step: 32 fp32, 64 16-bit, 128 8-bit elements

// a_k == 1 / b_k == 1: read along the contraction, else across
int linear_tile_f32(const LinArgs& a, LinTile tile, hipStream_t s);
int linear_tile_bf16(const LinArgs& a, LinTile tile, hipStream_t s);
int linear_tile_f16(const LinArgs& a, LinTile tile, hipStream_t s);
// a layer's two gradients on tiles of one shape
int linear_pair_f32(const LinArgs& dx, const LinArgs& dw, LinTile tile, hipStream_t s);
int linear_pair_bf16(const LinArgs& dx, const LinArgs& dw, LinTile tile, hipStream_t s);
int linear_pair_f16(const LinArgs& dx, const LinArgs& dw, LinTile tile, hipStream_t s);
int linear_tile_e4m3(const LinArgs& a, LinTile tile, int out_type, hipStream_t s);
