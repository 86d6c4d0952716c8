// Linear layer with its epilogue, forward and backward, fp32 / bf16 / fp16, and its 8-bit form (gfx950).
//
//   y = act(x w^T + bias) + residual      dz = dy act'(z)   dx = dz w   dw = dz^T x   db = column sums of dz
//
// Three matrix products of one shape family, C[i][j] = sum_k A(i, k) B(j, k): the forward contracts the features (both operands are
// read along k), dx contracts the outputs (w is read across), dw contracts the rows (both are read across).
#include "linear.h"

typedef __attribute__((ext_vector_type(8))) __bf16 lin_bf16x8;
typedef __attribute__((ext_vector_type(8))) _Float16 lin_f16x8;
typedef __attribute__((ext_vector_type(16))) float lin_f32x16;

int launch_sum_parts(int type, const float* part, int count, int width, void* out, hipStream_t s);

// ---- any strides, any alignment: 64 x 64 tiles, 32 of the contraction a step, element loads into LDS -------------------------------
// e4m3 operands are widened to bf16 (exact) on their way into LDS: the 8-bit matrix instructions add 8 neighbouring products to 2^-13 of the
// largest of them only (measured with powers of two: beside 1024 a neighbour of 2^-4 vanishes, one 8 places on stays down to 2^-13)
template <typename T> struct Staged { typedef T type; };
template <> struct Staged<TypeE4M3> { typedef TypeBF16 type; };
template <typename T> struct Mma;
template <> struct Mma<TypeBF16> {
    __device__ static inline lin_f32x16 run(uint4 a, uint4 b, lin_f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(lin_bf16x8, a), __builtin_bit_cast(lin_bf16x8, b), c, 0, 0, 0);
    }
};
template <> struct Mma<TypeF16> {
    __device__ static inline lin_f32x16 run(uint4 a, uint4 b, lin_f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(lin_f16x8, a), __builtin_bit_cast(lin_f16x8, b), c, 0, 0, 0);
    }
};
#define ANY_TILE 64
#define ANY_K 32
template <typename T, typename O>
__global__ __launch_bounds__(256) void linear_any_kernel(LinArgs p) {
    typedef typename T::raw raw;
    typedef typename Staged<T>::type S;
    typedef typename S::raw staged;
    constexpr int PITCH = ANY_K * sizeof(staged) + 16;
    auto stage = [](raw v) -> staged {
        if constexpr (sizeof(raw) == 1) return S::from_f32(T::to_f32(v));
        else return v;
    };
    __shared__ __attribute__((aligned(16))) char lds[2 * ANY_TILE * PITCH];
    char* la = lds;
    char* lb = lds + ANY_TILE * PITCH;
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const long i0 = (long)(blockIdx.x / p.tiles_j) * ANY_TILE;
    const int j0 = (blockIdx.x % p.tiles_j) * ANY_TILE;
    const int kb = blockIdx.y * p.k_split, ke = min(p.K, kb + p.k_split);
    lin_f32x16 acc;
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[e] = 0.f;
    for (int k0 = kb; k0 < ke; k0 += ANY_K) {
        __syncthreads();
        // consecutive threads along the operand's unit stride
        for (int t = tid; t < ANY_TILE * ANY_K; t += 256) {
            const int r = p.a_k == 1 ? t / ANY_K : t % ANY_TILE, k = p.a_k == 1 ? t % ANY_K : t / ANY_TILE;
            const bool ok = i0 + r < p.M && k0 + k < ke;
            ((staged*)(la + r * PITCH))[k] = ok ? stage(((const raw*)p.A)[(i0 + r) * p.a_i + (k0 + k) * p.a_k]) : (staged)0;
        }
        for (int t = tid; t < ANY_TILE * ANY_K; t += 256) {
            const int r = p.b_k == 1 ? t / ANY_K : t % ANY_TILE, k = p.b_k == 1 ? t % ANY_K : t / ANY_TILE;
            const bool ok = j0 + r < p.N && k0 + k < ke;
            ((staged*)(lb + r * PITCH))[k] = ok ? stage(((const raw*)p.B)[(long)(j0 + r) * p.b_j + (k0 + k) * p.b_k]) : (staged)0;
        }
        __syncthreads();
        const char* ra = la + ((wv >> 1) * 32 + (lane & 31)) * PITCH;
        const char* rb = lb + ((wv & 1) * 32 + (lane & 31)) * PITCH;
#pragma unroll
        for (int kk = 0; kk < ANY_K; kk += 16) {
            const int k = kk + (lane >> 5) * 8;
            // operands swapped: the accumulator's 16 registers run along j
            if constexpr (sizeof(staged) == 4) {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    acc = __builtin_amdgcn_mfma_f32_32x32x2f32(((const float*)rb)[k + e], ((const float*)ra)[k + e], acc, 0, 0, 0);
            } else {
                acc = Mma<S>::run(*(const uint4*)(rb + k * 2), *(const uint4*)(ra + k * 2), acc);
            }
        }
    }
    const long i = i0 + (wv >> 1) * 32 + (lane & 31);
    if (i >= p.M) return;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        const int j = j0 + (wv & 1) * 32 + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3);
        if (j >= p.N) continue;
        if (p.part) p.part[((size_t)blockIdx.y * p.M + i) * p.N + j] = acc[e];
        else epilogue_one<O>(p, i, j, acc[e]);
    }
}
// the splits' sums, added in order, then the epilogue
template <typename O> __global__ __launch_bounds__(256) void linear_join_kernel(LinArgs p, int splits) {
    const size_t total = (size_t)p.M * p.N;
    for (size_t t = (size_t)blockIdx.x * 256 + threadIdx.x; t < total; t += (size_t)gridDim.x * 256) {
        float v = 0.f;
        for (int s = 0; s < splits; ++s) v += p.part[s * total + t];
        epilogue_one<O>(p, (long)(t / p.N), (int)(t % p.N), v);
    }
}

// ---- dz = dy act'(z), and the column sums of dz by strips of rows ------------------------------------------------------------------
// thread: 8 neighbouring columns, every 8th row of the strip
template <typename O, bool VEC>
__global__ __launch_bounds__(256) void linear_dz_kernel(const void* dy_, long ld_dy, const void* z_, void* dz_, float* part, int M, int N, int act,
                                                        int strip) {
    typedef typename O::raw raw;
    __shared__ float red[8][32][9];
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const int j0 = blockIdx.y * 256 + tx * 8;
    const long r0 = (long)blockIdx.x * strip, r1 = min((long)M, r0 + strip);
    float sum[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) sum[e] = 0.f;
    if (j0 < N) {
        for (long r = r0 + ty; r < r1; r += 8) {
            float g[8], z[8];
            const raw* dy = (const raw*)dy_ + r * ld_dy + j0;
            if constexpr (VEC) {
                load_vec<O, 8>(dy, g);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) g[e] = j0 + e < N ? O::to_f32(dy[e]) : 0.f;
            }
            if (act != SCENERF_ACT_NONE) {
                const raw* zp = (const raw*)z_ + r * N + j0;
                if constexpr (VEC) {
                    load_vec<O, 8>(zp, z);
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) z[e] = j0 + e < N ? O::to_f32(zp[e]) : 0.f;
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) g[e] *= slope_any(act, z[e]);
                if (dz_) {
                    raw* out = (raw*)dz_ + r * N + j0;
                    if constexpr (VEC) {
                        store_vec<O, 8>(out, g);
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            if (j0 + e < N) out[e] = O::from_f32(g[e]);
                    }
                }
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) sum[e] += g[e];
        }
    }
    if (!part) return;
#pragma unroll
    for (int e = 0; e < 8; ++e) red[ty][tx][e] = sum[e];
    __syncthreads();
    const int c = threadIdx.x >> 3, e = threadIdx.x & 7, j = blockIdx.y * 256 + threadIdx.x;
    if (j < N) {
        float s = 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k) s += red[k][c][e];
        part[(size_t)blockIdx.x * N + j] = s;
    }
}

// ---------------------------------------------------------------------------------------------------------------- host side
static int lin_es(int type) { return type == SCENERF_T_F32 ? 4 : type == SCENERF_T_E4M3 ? 1 : 2; }
static bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
static int64_t align256(int64_t v) { return (v + 255) & ~255LL; }

// the contraction is split where the tiles alone leave CUs idle; a split keeps at least 256 elements
static int lin_splits(long M, int N, long K) {
    if (M < 1) return 1;
    const long tiles = ((M + ANY_TILE - 1) / ANY_TILE) * ((N + ANY_TILE - 1) / ANY_TILE);
    long s = 1024 / tiles;
    if (s > K / 256) s = K / 256;
    return s < 1 ? 1 : s > 256 ? 256 : (int)s;
}
static int64_t lin_part_bytes(long M, int N, long K) {
    const int s = lin_splits(M, N, K);
    return s > 1 ? align256((int64_t)s * M * N * 4) : 0;
}
template <typename T, typename O> static int lin_launch(LinArgs a, void* ws, hipStream_t s) {
    const int splits = lin_splits(a.M, a.N, a.K);
    a.tiles_j = cdiv(a.N, ANY_TILE);
    a.part = splits > 1 ? (float*)ws : nullptr;
    a.k_split = cdiv(cdiv(a.K, splits), ANY_K) * ANY_K;
    const long blocks = (long)((a.M + ANY_TILE - 1L) / ANY_TILE) * a.tiles_j;
    SRF_CHECK(blocks <= ROWOPS_GRID_MAX, "linear: %ld tiles are more than one launch holds", blocks);
    linear_any_kernel<T, O><<<dim3((unsigned)blocks, splits), 256, 0, s>>>(a);
    SRF_LAUNCH_CHECK("linear_any_kernel");
    if (splits > 1) {
        const long total = (long)a.M * a.N;
        linear_join_kernel<O><<<(unsigned)((total + 255) / 256 < 8192 ? (total + 255) / 256 : 8192), 256, 0, s>>>(a, splits);
        SRF_LAUNCH_CHECK("linear_join_kernel");
    }
    return 0;
}
template <typename T> static int lin_launch_out(int out_type, const LinArgs& a, void* ws, hipStream_t s) {
    if constexpr (T::code != SCENERF_T_E4M3) return lin_launch<T, T>(a, ws, s);
    else if (out_type == SCENERF_T_F32) return lin_launch<T, TypeF32>(a, ws, s);
    else if (out_type == SCENERF_T_BF16) return lin_launch<T, TypeBF16>(a, ws, s);
    else return lin_launch<T, TypeF16>(a, ws, s);
}
static int lin_product(int in_type, int out_type, const LinArgs& a, void* ws, hipStream_t s) {
    switch (in_type) {
        case SCENERF_T_F32: return lin_launch_out<TypeF32>(out_type, a, ws, s);
        case SCENERF_T_BF16: return lin_launch_out<TypeBF16>(out_type, a, ws, s);
        case SCENERF_T_F16: return lin_launch_out<TypeF16>(out_type, a, ws, s);
        default: return lin_launch_out<TypeE4M3>(out_type, a, ws, s);
    }
}

#define DZ_STRIPS 512
static int dz_strip(int64_t rows) {
    const int64_t per = (rows + DZ_STRIPS - 1) / DZ_STRIPS;
    return per < 8 ? 8 : (int)((per + 7) / 8 * 8);
}
struct BackwardPlan {
    bool need_dz;                   // dz is not dy itself
    int strip, strips;
    int64_t part, dz, sums;         // offsets of the column sums' parts, of dz and of the split sums
    int64_t bytes;
};
static BackwardPlan lin_backward_plan(const scenerf_linear* p) {
    BackwardPlan b = {};
    b.need_dz = p->activation != SCENERF_ACT_NONE;
    b.strip = dz_strip(p->rows);
    b.strips = (int)((p->rows + b.strip - 1) / b.strip);
    int64_t at = 0;
    if (p->db) { b.part = at; at += align256((int64_t)b.strips * p->n * 4); }
    if (b.need_dz && (p->dx || p->dw)) { b.dz = at; at += align256(p->rows * p->n * lin_es(p->out_type)); }
    b.sums = at;
    const int64_t sx = p->dx ? lin_part_bytes(p->rows, p->k, p->n) : 0, sw = p->dw ? lin_part_bytes(p->n, p->k, p->rows) : 0;
    b.bytes = at + (sx > sw ? sx : sw);
    return b;
}
static int lin_check(const scenerf_linear* p, const char* what, bool backward) {
    SRF_CHECK(p, "%s: NULL argument", what);
    SRF_CHECK(p->in_type >= SCENERF_T_F32 && p->in_type <= SCENERF_T_E4M3 && p->out_type >= SCENERF_T_F32 && p->out_type <= SCENERF_T_F16,
              "%s: types must be F32, BF16, F16 or (x and w) E4M3", what);
    SRF_CHECK(p->in_type == SCENERF_T_E4M3 || p->in_type == p->out_type, "%s: in_type and out_type differ", what);
    SRF_CHECK(p->activation >= SCENERF_ACT_NONE && p->activation <= SCENERF_ACT_SILU, "%s: unknown activation %d", what, p->activation);
    SRF_CHECK(p->n >= 1 && p->k >= 1 && p->n < ROWOPS_GRID_MAX - 1024 && p->k < ROWOPS_GRID_MAX - 1024, "%s: n and k must be in [1, 2^31 - 1024)", what);
    SRF_CHECK(p->rows >= 0 && p->rows < ROWOPS_GRID_MAX - 1024, "%s: rows must be in [0, 2^31 - 1024)", what);
    SRF_CHECK(p->ldx >= 0 && p->ldw >= 0 && p->ld_residual >= 0 && p->ld_dy >= 0, "%s: negative leading dimension", what);
    if (backward) {
        SRF_CHECK(p->in_type != SCENERF_T_E4M3, "%s: the 8-bit form has no gradients", what);
        SRF_CHECK(p->dx || p->dw || p->db, "%s: nothing to compute", what);
        if (p->rows == 0) return 0;
        SRF_CHECK(p->dy && (p->w || !p->dx) && (p->x || !p->dw), "%s: NULL dy, w or x", what);
        SRF_CHECK(p->activation == SCENERF_ACT_NONE || p->z, "%s: z is NULL", what);
    } else if (p->rows > 0) {
        SRF_CHECK(p->x && p->w && p->y, "%s: NULL x, w or y", what);
        SRF_CHECK(p->in_type != SCENERF_T_E4M3 || (p->x_scale && p->w_scale), "%s: NULL x_scale or w_scale", what);
    }
    return 0;
}
template <typename O> static int lin_dz(const scenerf_linear* p, const BackwardPlan& b, void* dz, float* part, hipStream_t s) {
    const bool vec = p->n % 8 == 0 && p->ld_dy % 8 == 0 && aligned16(p->dy) && (!b.need_dz || aligned16(p->z));
    const dim3 grid(b.strips, cdiv(p->n, 256));
    SRF_CHECK(grid.y <= 65535, "linear_backward: n is too large");
    if (vec) linear_dz_kernel<O, true><<<grid, 256, 0, s>>>(p->dy, p->ld_dy, p->z, dz, part, (int)p->rows, p->n, p->activation, b.strip);
    else linear_dz_kernel<O, false><<<grid, 256, 0, s>>>(p->dy, p->ld_dy, p->z, dz, part, (int)p->rows, p->n, p->activation, b.strip);
    SRF_LAUNCH_CHECK("linear_dz_kernel");
    return 0;
}

extern "C" {

int64_t scenerf_hip_linear_workspace(const scenerf_linear* p, int backward) {
    if (lin_check(p, "linear_workspace", backward != 0)) return -1;
    return backward ? lin_backward_plan(p).bytes : lin_part_bytes(p->rows, p->n, p->k);
}

int scenerf_hip_linear_forward(const scenerf_linear* p, scenerf_stream_t stream) {
    if (int e = lin_check(p, "linear_forward", false)) return e;
    if (p->rows == 0) return 0;
    const int64_t need = lin_part_bytes(p->rows, p->n, p->k);
    SRF_CHECK(need == 0 || (p->workspace && aligned16(p->workspace) && p->workspace_bytes >= need), "linear_forward: workspace of %lld bytes needed",
              (long long)need);
    const double m = (double)p->rows, es = lin_es(p->in_type), eo = lin_es(p->out_type);
    SrfLaunchScope ps(as_stream(stream), "linear_forward", 2 * m * p->n * p->k, es * (m * p->k + (double)p->n * p->k) + eo * m * p->n);
    LinArgs a = {};
    a.A = p->x; a.a_i = p->ldx; a.a_k = 1;
    a.B = p->w; a.b_j = p->ldw; a.b_k = 1;
    a.M = (int)p->rows; a.N = p->n; a.K = p->k;
    if (p->in_type == SCENERF_T_E4M3) { a.row_scale = p->x_scale; a.col_scale = p->w_scale; }
    a.bias = p->bias; a.residual = p->residual; a.ld_residual = p->ld_residual;
    a.out = p->y; a.z = p->z; a.act = p->activation;
    return lin_product(p->in_type, p->out_type, a, p->workspace, as_stream(stream));
}

int scenerf_hip_linear_backward(const scenerf_linear* p, scenerf_stream_t stream) {
    if (int e = lin_check(p, "linear_backward", true)) return e;
    hipStream_t s = as_stream(stream);
    const BackwardPlan b = lin_backward_plan(p);
    SRF_CHECK(b.bytes == 0 || (p->workspace && aligned16(p->workspace) && p->workspace_bytes >= b.bytes),
              "linear_backward: workspace of %lld bytes needed", (long long)b.bytes);
    const double m = (double)p->rows, es = lin_es(p->in_type);
    SrfLaunchScope ps(s, "linear_backward", 2 * m * p->n * p->k * (!!p->dx + !!p->dw), es * m * (p->n + 2. * p->k));
    char* ws = (char*)p->workspace;
    float* part = (float*)(ws + b.part);
    const void* dz = b.need_dz ? ws + b.dz : p->dy;
    const long ld_dz = b.need_dz ? p->n : p->ld_dy;
    if (p->rows > 0 && (b.need_dz || p->db)) {
        float* sums = p->db ? part : nullptr;
        void* to = b.need_dz && (p->dx || p->dw) ? (void*)dz : nullptr;
        int e = p->out_type == SCENERF_T_F32 ? lin_dz<TypeF32>(p, b, to, sums, s)
                : p->out_type == SCENERF_T_BF16 ? lin_dz<TypeBF16>(p, b, to, sums, s) : lin_dz<TypeF16>(p, b, to, sums, s);
        if (e) return e;
    }
    if (p->db) {
        if (int e = launch_sum_parts(p->out_type, part, b.strips, p->n, p->db, s)) return e;
    }
    if (p->dx && p->rows > 0) {
        LinArgs a = {};
        a.A = dz; a.a_i = ld_dz; a.a_k = 1;
        a.B = p->w; a.b_j = 1; a.b_k = p->ldw;
        a.M = (int)p->rows; a.N = p->k; a.K = p->n;
        a.out = p->dx;
        if (int e = lin_product(p->in_type, p->out_type, a, ws + b.sums, s)) return e;
    }
    if (p->dw) {     // rows == 0: an empty sum, zeros
        LinArgs a = {};
        a.A = dz; a.a_i = 1; a.a_k = ld_dz;
        a.B = p->x; a.b_j = 1; a.b_k = p->ldx;
        a.M = p->n; a.N = p->k; a.K = (int)p->rows;
        a.out = p->dw;
        if (int e = lin_product(p->in_type, p->out_type, a, ws + b.sums, s)) return e;
    }
    return 0;
}

}  // extern "C"
