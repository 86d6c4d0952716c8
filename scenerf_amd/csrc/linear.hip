// Linear layer with its epilogue, forward and backward, fp32 / bf16 / fp16, and its 8-bit form (gfx950).
//
//   y = act(x w^T + bias) + residual      dz = dy act'(z)   dx = dz w   dw = dz^T x   db = column sums of dz
//
// Three matrix products of one shape family, C[i][j] = sum_k A(i, k) B(j, k): the forward contracts the features (both operands are
// read along k), dx contracts the outputs (w is read across), dw contracts the rows (both are read across).
//
// Products of many rows run on staged tiles (linear_tile.h): bound by the chip's power where the contraction is long (153,600 x 2,480
// x 1,536 bf16 1,000 to 1,060 us from card to card, 1.10 to 1.17 PFLOP/s; the library's product of that shape without an epilogue takes the same;
// 8 bits 615 to 646; 4,096 x 8,192 x 4,096 takes 256 us, and 162 if all of it is zeros), by the operands' and results' bytes where it is short
// (153,600 x 512 x 512 bf16 with gelu, residual and kept sums 169 to 188 us for 629 MB).
#include "linear.h"

typedef __attribute__((ext_vector_type(8))) __bf16 lin_bf16x8;
typedef __attribute__((ext_vector_type(8))) _Float16 lin_f16x8;
typedef __attribute__((ext_vector_type(16))) float lin_f32x16;

int launch_sum_parts(int type, const float* part, int count, int width, void* out, hipStream_t s);

// ---- any strides, any alignment: 64 x 64 tiles, 32 of the contraction a step, element loads into LDS -------------------------------
// For C callers whose rows are not in 16-byte pieces and not copied into them (scenerf_hip_linear_pad), and for rows shorter than 16 bytes.
// Bound by the element loads and their wait, nothing in flight meanwhile: 153,600 x 2,480 x 1,536 bf16 15.3 ms.
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
    const void* A = p.A;
    const long kb = (long)blockIdx.y * p.k_split, ke = min((long)p.K, kb + p.k_split);
    lin_f32x16 acc;
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[e] = 0.f;
    for (long k0 = kb; k0 < ke; k0 += ANY_K) {
        __syncthreads();
        // consecutive threads along the operand's unit stride
        for (int t = tid; t < ANY_TILE * ANY_K; t += 256) {
            const int r = p.a_k == 1 ? t / ANY_K : t % ANY_TILE, k = p.a_k == 1 ? t % ANY_K : t / ANY_TILE;
            const bool ok = i0 + r < p.M && k0 + k < ke;
            ((staged*)(la + r * PITCH))[k] = ok ? stage(((const raw*)A)[(i0 + r) * p.a_i + (k0 + k) * p.a_k]) : (staged)0;
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
        if (k0 + ANY_K >= ke && p.A2 && A == p.A) {        // once more, with A2
            A = p.A2;
            k0 = kb - ANY_K;
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
// the splits' sums, added in a fixed order, then the epilogue: a workgroup owns 32 pieces of W results, 8 threads each, thread y of them
// adds splits y, y + 8, ..  Bound by the sums' bytes: 64 splits of 512 x 512 (67 MB) 16.7 us, 4.0 TB/s
// db's column sums ride along in front of dw's join, a launch less: each of `sums.blocks` workgroups adds 16 columns in 16 chains
struct ColumnSums { const float* part; void* out; int count, width, blocks; };
template <typename O> __global__ __launch_bounds__(256) void linear_join_kernel(LinArgs p, ColumnSums sums) {
    constexpr int W = 16 / (int)sizeof(typename O::raw);
    __shared__ float red[8][32][W + 1];
    if ((int)blockIdx.x < sums.blocks) {
        float (*chain)[17] = (float (*)[17])red;
        const int cx = threadIdx.x & 15, cy = threadIdx.x >> 4, col = blockIdx.x * 16 + cx;
        float s = 0.f;
        if (col < sums.width) {
#pragma unroll 8
            for (int i = cy; i < sums.count; i += 16) s += sums.part[(size_t)i * sums.width + col];
        }
        chain[cy][cx] = s;
        __syncthreads();
        s = chain[cx][cy];            // column cy, chain cx
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) s += __shfl_xor(s, o, WAVE);
        if (cx == 0 && (int)blockIdx.x * 16 + cy < sums.width) ((typename O::raw*)sums.out)[blockIdx.x * 16 + cy] = O::from_f32(s);
        return;
    }
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5, per = (p.N + W - 1) / W;
    const long pieces = (long)p.M * per;
    for (long t0 = (long)(blockIdx.x - sums.blocks) * 32; t0 < pieces; t0 += (long)(gridDim.x - sums.blocks) * 32) {
        const long i = (t0 + tx) / per;
        const int j = (int)((t0 + tx) - i * per) * W;
        const bool ok = t0 + tx < pieces;
        float v[W];
#pragma unroll
        for (int e = 0; e < W; ++e) v[e] = 0.f;
        if (ok) {
#pragma unroll 4
            for (int s = ty; s < p.splits; s += 8) {
                float u[W];
                load_some<TypeF32, W>(p.part + ((size_t)s * p.M + i) * p.N + j, p.N - j, p.N % W, u);
#pragma unroll
                for (int e = 0; e < W; ++e) v[e] += u[e];
            }
        }
        __syncthreads();
#pragma unroll
        for (int e = 0; e < W; ++e) red[ty][tx][e] = v[e];
        __syncthreads();
        if (ty == 0 && ok) {
#pragma unroll
            for (int e = 0; e < W; ++e) {
                v[e] = 0.f;
#pragma unroll
                for (int y = 0; y < 8; ++y) v[e] += red[y][tx][e];
            }
            EpilogueCols<O, W, false> ec;
            ec.load(p, j, p.N - j);
            uint4 res = make_uint4(0, 0, 0, 0);
            if (p.residual) res = residual_piece<O, W, false>(p, i, j, p.N - j);
            epilogue_vec<O, W, false>(p, ec, i, j, p.N - j, res, v);
        }
    }
}

// ---- a few rows: every weight read once, straight into registers ------------------------------------------------------------------
// A workgroup owns COLS columns (per wave where KW == 1: its four waves take four groups of them; KW == 4: the four waves split the
// contraction of one group), a lane every 64th (256th) 16 bytes of their rows of w and of up to MR rows of x; products and sums in fp32 on the vector
// units, which idle otherwise: the call is bound by the latency of one round of loads and by w's bytes.  One row x 2,480 x 1,536 bf16: 3.0 us
// replayed from a graph, 7.6 MB of w, of which an empty launch is about 2.
#define FEW_COLS 4
template <typename T, typename O, int MR, int KW>
__global__ __launch_bounds__(256) void linear_few_kernel(LinArgs p) {
    typedef typename T::raw raw;
    constexpr int W = 16 / (int)sizeof(raw);
    __shared__ float red[KW][FEW_COLS * MR];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    const int j0 = (KW == 1 ? blockIdx.x * 4 + wv : blockIdx.x) * FEW_COLS;
    const int pieces = (p.K + W - 1) / W;
    float acc[FEW_COLS][MR];
#pragma unroll
    for (int c = 0; c < FEW_COLS; ++c)
#pragma unroll
        for (int m = 0; m < MR; ++m) acc[c][m] = 0.f;
    const raw* wrow[FEW_COLS];
#pragma unroll
    for (int c = 0; c < FEW_COLS; ++c) wrow[c] = (const raw*)p.B + (long)min(j0 + c, p.N - 1) * p.b_j;
    for (int t = KW == 1 ? lane : (int)threadIdx.x; t < pieces; t += 64 * KW) {
        // a last piece that the row does not fill: the row's last 16 bytes (K >= W), those that another piece has set to zero in both operands
        const int at = min(t * W, p.K - W), seen = (t * W - at) * (int)sizeof(raw);
        uint32_t fresh[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) fresh[i] = seen >= 4 * i + 4 ? 0u : seen <= 4 * i ? ~0u : ~0u << (8 * (seen - 4 * i));
        auto piece = [&](const raw* row) -> uint4 {
            const uint4 v = load16(row + at);
            return make_uint4(v.x & fresh[0], v.y & fresh[1], v.z & fresh[2], v.w & fresh[3]);
        };
        uint4 w[FEW_COLS], x[MR];
#pragma unroll
        for (int c = 0; c < FEW_COLS; ++c) w[c] = piece(wrow[c]);
#pragma unroll
        for (int m = 0; m < MR; ++m) x[m] = piece((const raw*)p.A + (long)min(m, p.M - 1) * p.a_i);
#pragma unroll
        for (int m = 0; m < MR; ++m) {
            float xv[W];
            unpack16<T>(x[m], xv);
#pragma unroll
            for (int c = 0; c < FEW_COLS; ++c) {
                float wf[W];
                unpack16<T>(w[c], wf);
#pragma unroll
                for (int e = 0; e < W; ++e) acc[c][m] = fmaf(xv[e], wf[e], acc[c][m]);
            }
        }
    }
    // The lanes' sums added: with every exchange a lane gives away half of its sums and keeps the other, so that SUMS of them take
    // SUMS - 1 exchanges instead of 6 each (8 rows x 512 x 512 bf16: 9.1 us with 6 each, 3.7 so); in the end SPAN neighbouring lanes hold sum o
    constexpr int SUMS = FEW_COLS * MR, SPAN = 64 / SUMS;
    float v[SUMS];
#pragma unroll
    for (int t = 0; t < SUMS; ++t) v[t] = acc[t / MR][t % MR];
#pragma unroll
    for (int step = 0; step < 6; ++step) {
        const int half = SUMS >> (step + 1), far = 32 >> step;
        const bool up = lane & far;
        if (half == 0) v[0] += __shfl_xor(v[0], far, WAVE);
#pragma unroll
        for (int t = 0; t < SUMS / 2; ++t)
            if (t < half) {
                const float low = v[t], high = v[t + half];        // (v[up ? .. : ..] becomes a search through the registers)
                const float give = __shfl_xor(up ? low : high, far, WAVE);
                v[t] = (up ? high : low) + give;
            }
    }
    int o = lane / SPAN;
    bool mine = lane % SPAN == 0;
    if constexpr (KW == 4) {
        if (mine) red[wv][o] = v[0];
        __syncthreads();
        o = (int)threadIdx.x;
        mine = o < SUMS;
        if (mine) v[0] = (red[0][o] + red[1][o]) + (red[2][o] + red[3][o]);
    }
    const int m = o % MR, j = j0 + o / MR;
    if (mine && m < p.M && j < p.N) epilogue_one<O>(p, m, j, v[0]);
}

// ---- rows laid out anew: pitch a whole number of 16-byte pieces, zeros behind the row's end -----------------------------------------
// (4,801 + 515 rows of 42 fp16: 5 us, most of it the launch)
struct PadSide { const void* src; void* dst; long ld, rows; };
template <typename R>
__global__ __launch_bounds__(256) void linear_pad_kernel(PadSide x, PadSide w, int cols, int pitch) {
    constexpr int W = 16 / sizeof(R);
    const int per = pitch / W;
    const long first = x.rows * per, pieces = first + w.rows * per;
    for (long t = (long)blockIdx.x * 256 + threadIdx.x; t < pieces; t += (long)gridDim.x * 256) {
        const PadSide& s = t < first ? x : w;
        const long u = t < first ? t : t - first, r = u / per;
        const int c = (int)(u - r * per) * W;
        union { R e[W]; uint4 v; } o;
        const R* at = (const R*)s.src + r * s.ld + c;
        if (c + W <= cols) {
            o.v = load16(at);
        } else {
#pragma unroll
            for (int e = 0; e < W; ++e) o.e[e] = c + e < cols ? at[e] : (R)0;
        }
        *(uint4*)((R*)s.dst + r * pitch + c) = o.v;
    }
}

// ---- dz = dy act'(z), and the column sums of dz by strips of rows ------------------------------------------------------------------
template <int ACT, typename O> __device__ static inline void slopes(float (&g)[8], float (&z)[8], int valid) {
    act_slope<ACT, 8, O::code == SCENERF_T_F32>(z);
#pragma unroll
    for (int e = 0; e < 8; ++e) g[e] = e < valid ? g[e] * z[e] : 0.f;
}
// fp16's dz with a slope that is no whole number: dy times up to 1.13 may pass 65,504, and a dy of few bits (2^-20, say) times a slope would keep
// fewer still.  So dz is held times the power of two that brings the largest finite |dy| into [2^14, 2^15), and the products' results are
// divided by it, exactly: what is left below the largest dy's 2^-39 is all that fp16 does not hold.  This is that maximum, by strips of rows (157
// MB of dy once more at 153,600 x 512: 541 -> 595 us there and back); a dy of bf16 or fp32 has its dz's range, and relu's slopes, 0 and 1, leave dy as it is.
template <bool WHOLE>
__global__ __launch_bounds__(256) void linear_dy_max_kernel(const void* dy_, long ld_dy, float* most, int M, int N, int strip) {
    __shared__ float red[4];
    const int per = (N + 7) / 8;
    const long r0 = (long)blockIdx.x * strip, pieces = (min((long)M, r0 + strip) - r0) * per;
    float m = 0.f;
#pragma unroll 4
    for (long t = threadIdx.x; t < pieces; t += 256) {
        const long r = t / per;
        const int j = (int)(t - r * per) * 8;
        float v[8];
        load_some<TypeF16, 8, WHOLE>((const uint16_t*)dy_ + (r0 + r) * ld_dy + j, N - j, N % 8, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) m = fabsf(v[e]) < __builtin_inff() ? fmaxf(m, fabsf(v[e])) : m;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, WAVE));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
    __syncthreads();
    if (threadIdx.x == 0) most[blockIdx.x] = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
}
// the power of two from the strips' maxima, by every workgroup for itself; `red` is used before and may be used behind it
__device__ static inline float dz_scale(const float* most, int count, float* red) {
    float m = 0.f;
    for (int t = threadIdx.x; t < count; t += 256) m = fmaxf(m, most[t]);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, WAVE));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
    __syncthreads();
    m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    __syncthreads();
    return m > 0.f ? __uint_as_float((127u + 14u + 127u - (__float_as_uint(m) >> 23)) << 23) : 1.f;
}
// A workgroup's 256 threads stand as 2^lx columns of 8 by 256 / 2^lx rows (2^lx: 64, a wave a row, or what a narrower matrix needs: at 128
// columns a fixed 32 left half the threads idle, 150 us for 262,144 x 128 fp32 instead of 78; 32 at 512 columns took 111 us for 153,600 rows
// of bf16, 64 100); two rows a thread are in flight.  Bound by HBM: 4.7 and 5.2 TB/s.
// `most`, not NULL (fp16): the strips' largest |dy|; dz is held scaled, and `unscale` says by what to multiply its products
template <typename O, bool WHOLE>
__global__ __launch_bounds__(256) void linear_dz_kernel(const void* dy_, long ld_dy, const void* z_, void* dz_, void* rest_, int pitch, float* part,
                                                        const float* most, float* unscale, int M, int N, int act, int strip, int lx) {
    typedef typename O::raw raw;
    __shared__ float red[256 * 9];
    float scale = 1.f;
    if constexpr (O::code == SCENERF_T_F16) {
        if (most) {
            scale = dz_scale(most, gridDim.x, red);
            if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) *unscale = 1.f / scale;
        }
    }
    const int tx = threadIdx.x & ((1 << lx) - 1), ty = threadIdx.x >> lx, rows = 256 >> lx;
    const int j0 = ((blockIdx.y << lx) + tx) * 8;           // (a pitch above N: zeros in the columns between)
    const long r0 = (long)blockIdx.x * strip, r1 = min((long)M, r0 + strip);
    float sum[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) sum[e] = 0.f;
    auto get = [&](const raw* p, float (&v)[8]) { load_some<O, 8, WHOLE>(p, N - j0, N % 8, v); };
    if (j0 < N) {
        for (long r = r0 + ty; r < r1; r += 2 * rows) {
            const bool two = r + rows < r1;
            float g[2][8], z[2][8];
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const long at = q == 0 || two ? r + q * rows : r;
                get((const raw*)dy_ + at * ld_dy + j0, g[q]);
                if (act != SCENERF_ACT_NONE) get((const raw*)z_ + at * N + j0, z[q]);
            }
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                if (q == 1 && !two) continue;
                if (act == SCENERF_ACT_GELU) slopes<SCENERF_ACT_GELU, O>(g[q], z[q], N - j0);
                else if (act == SCENERF_ACT_SILU) slopes<SCENERF_ACT_SILU, O>(g[q], z[q], N - j0);
                else if (act == SCENERF_ACT_RELU) slopes<SCENERF_ACT_RELU, O>(g[q], z[q], N - j0);
#pragma unroll
                for (int e = 0; e < 8; ++e) sum[e] += g[q][e];
                if constexpr (O::code == SCENERF_T_F16) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) g[q][e] *= scale;
                }
                if (dz_) store_vec<O, 8>((raw*)dz_ + (r + q * rows) * pitch + j0, g[q]);
                if (rest_) {            // what dz's rounding left out
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float left = g[q][e] - O::to_f32(O::from_f32(g[q][e]));
                        g[q][e] = fabsf(left) < 3.0e38f ? left : 0.f;            // (dz infinite or NaN: says it itself)
                    }
                    store_vec<O, 8>((raw*)rest_ + (r + q * rows) * pitch + j0, g[q]);
                }
            }
        }
    }
    if (!part) return;
#pragma unroll
    for (int e = 0; e < 8; ++e) red[threadIdx.x * 9 + e] = sum[e];
    __syncthreads();
    for (int t = threadIdx.x; t < 8 << lx; t += 256) {
        const int j = (blockIdx.y << lx) * 8 + t;
        if (j >= N) continue;
        float s = 0.f;
        for (int k = 0; k < rows; ++k) s += red[((k << lx) + (t >> 3)) * 9 + (t & 7)];
        part[(size_t)blockIdx.x * N + j] = s;
    }
}

// ---------------------------------------------------------------------------------------------------------------- host side
static int lin_es(int type) { return type == SCENERF_T_F32 ? 4 : type == SCENERF_T_E4M3 ? 1 : 2; }
static bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
static int64_t align256(int64_t v) { return (v + 255) & ~255LL; }
static int round_up(int v, int to) { return (v + to - 1) / to * to; }

// How a product runs.  kind 0: element loads (any strides), 1: a few rows, 2: staged tiles
struct LinPlan {
    int kind, splits, k_split;
    LinTile tile;
};
// What a tile costs, in us: a workgroup's start and end, and a chunk of 128 bytes of the contraction with 1, 2, 3 workgroups on a CU (as many as
// their LDS lets in).  Fitted to products of 1,024 to 153,600 rows by 48 to 2,480 features, forward and both gradients: on 364 of 366 of them
// (bf16 and fp32) what the plan chooses took no more than 7 percent or 2 us above the fastest of all tiles and splits.  fp16, whose
// instructions have bf16's rates, and e4m3, which has half its chunks (where it is widened, each of twice the matrix time), take bf16's
// costs, and were not gone through like that.  Where the tiles differ most (on one box): 153,600 x 2,480 x 1,536 bf16 256^2 1,034 us and 128^2 1,521; 262,144 x 128 x 128 50 and 32; 1,024 x 512 x 512 20, 9.8 and 64^2
// 6.1; dw of 12,288 rows x 512 x 2,480 54, 52 (6 splits) and 64^2 unsplit 108.
struct LinTileCost { LinTile tile; int per_cu; double ends, chunk[3]; };
static const LinTileCost kLinCost16[] = {{LIN_256x256, 1, 9.0, {1.7}}, {LIN_128x128, 2, 4.7, {0.61, 1.1}}, {LIN_64x64, 3, 1.8, {0.35, 0.55, 0.78}}};
static const LinTileCost kLinCost32[] = {{LIN_128x128, 2, 4.7, {1.8, 3.6}}, {LIN_64x64, 3, 1.8, {0.5, 0.95, 1.55}}};
#define LIN_BYTES_US 5.0e6          // of HBM
#define LIN_PART_BYTES_US 7.0e6     // of splits' sums, written and read again from the last cache
#define LIN_MIN_CHUNKS 8            // a split keeps at least so many: its ends cost as much

// `staged`: both operands are in 16-byte pieces
// `like`: a tile whose product could share another one's launch, worth a tenth; `large`: 256 x 256 tiles are among them
static LinPlan lin_plan(int type, bool ax, bool bx, bool staged, long M, int N, long K, LinTile like = LIN_TILES, bool large = true) {
    LinPlan r = {0, 1, 0, LIN_128x128};
    // (bf16, this kernel against staged tiles: 1 row x 512 x 512 2.2 against 4.9 us, 8 rows 3.7 against 4.9, 8 x 2,480 x 1,536 5.5 against 9.7;
    // 16 rows 5.3 against 5.0.  It reads whole 16 bytes inside the row: a shorter row takes the element loads; a launch holds 2^32 threads)
    if (!ax && !bx && M <= 8 && K >= 16 / lin_es(type) && N < 1 << 26) {
        r.kind = 1;
        return r;
    }
    const int bk = staged ? LIN_CHUNK_BYTES / lin_es(type) : ANY_K;
    const long chunks = (K + bk - 1) / bk;
    auto tiles_of = [&](long rows, long cols) { return ((M + rows - 1) / rows) * ((N + cols - 1) / cols); };
    long splits = 1;
    if (!staged) {
        const long tiles = tiles_of(ANY_TILE, ANY_TILE);
        splits = min(tiles > 0 ? 512 / tiles : 1, chunks / LIN_MIN_CHUNKS);
    } else if (N <= 32) {
        r.kind = 2;
        r.tile = LIN_128x32;
        const long tiles = tiles_of(128, 32);
        splits = min(tiles > 0 ? (chunks < 256 ? 256 : 768) / tiles : 1, chunks / LIN_MIN_CHUNKS);
    } else {
        r.kind = 2;
        const LinTileCost* cost = type == SCENERF_T_F32 ? kLinCost32 : kLinCost16;
        const int kinds = type == SCENERF_T_F32 ? 2 : 3;
        const double bytes = ((double)M * K + (double)N * K + (double)M * N) * lin_es(type) / LIN_BYTES_US;
        double best = 1e300;
        for (int c = 0; c < kinds; ++c) {
            const LinTileCost& t = cost[c];
            if (!large && t.tile == LIN_256x256) continue;
            const long tiles = tiles_of(kLinTileRows[t.tile], kLinTileCols[t.tile]), slots = 256L * t.per_cu;
            const long most = max(1L, min(slots / max(1L, tiles), chunks / LIN_MIN_CHUNKS));
            // 1, 2 or 3 workgroups a CU, or none of it split
            for (int per_cu = 0; per_cu <= t.per_cu; ++per_cu) {
                const long s = per_cu == 0 ? 1 : min(most, 256L * per_cu / max(1L, tiles));
                if (s < 1) continue;
                const long work = tiles * s, each = (chunks + s - 1) / s, full = work / slots, rest = work % slots;
                double us = full * (each * t.chunk[t.per_cu - 1] + t.ends);
                if (rest > 0) {         // (a CU gets along faster where others have nothing to do)
                    const int on_cu = (int)((rest + 255) / 256);
                    us += each * t.chunk[on_cu - 1] * (0.75 + 0.25 * rest / (256.0 * on_cu)) + t.ends;
                }
                us = max(us, bytes + 2.0);
                if (s > 1) us += 5.0 + 8.0 * s * M * N / LIN_PART_BYTES_US;
                if (t.tile == like) us *= 0.9;
                if (us < best) { best = us; r.tile = t.tile; splits = s; }
            }
        }
    }
    r.splits = (int)max(1L, min(splits, 256L));
    r.k_split = (int)(((K + r.splits - 1) / r.splits + bk - 1) / bk * bk);
    return r;
}
// `sums`: a result in fp32 of 16-bit operands (dw as it is summed), which the join alone writes
static int64_t lin_part_bytes(const LinPlan& p, long M, int N, bool sums = false) { return p.splits > 1 || sums ? align256((int64_t)p.splits * M * N * 4) : 0; }

template <typename T, typename O, int MR> static void lin_few(const LinArgs& a, hipStream_t s) {
    // one piece a lane and row of w: one wave a group of columns; longer rows: four (bf16, 8 rows, 512 outputs, one wave against four: 512
    // features 3.64 and 3.55 us, 1,024 4.47 and 3.66, 2,480 6.96 and 4.61; one row of 512: 2.22 and 2.44)
    if (a.K <= 64 * (16 / (int)sizeof(typename T::raw))) linear_few_kernel<T, O, MR, 1><<<cdiv(a.N, 4 * FEW_COLS), 256, 0, s>>>(a);
    else linear_few_kernel<T, O, MR, 4><<<cdiv(a.N, FEW_COLS), 256, 0, s>>>(a);
}
static void lin_fill(LinArgs& a, const LinPlan& plan, void* ws, bool sums = false) {
    a.splits = plan.splits;
    a.k_split = plan.k_split;
    a.part = a.splits > 1 || sums ? (float*)ws : nullptr;
    if (plan.kind == 2) {
        a.tiles_i = (int)((a.M + (long)kLinTileRows[plan.tile] - 1) / kLinTileRows[plan.tile]);
        a.tiles_j = (int)((a.N + (long)kLinTileCols[plan.tile] - 1) / kLinTileCols[plan.tile]);
    }
}
template <typename O> static int lin_join(const LinArgs& a, const ColumnSums& sums, hipStream_t s) {
    if (!a.part) return 0;
    constexpr int W = 16 / (int)sizeof(typename O::raw);
    const long work = ((long)a.M * ((a.N + W - 1) / W) + 31) / 32;
    linear_join_kernel<O><<<(unsigned)(work < 16384 ? work : 16384) + sums.blocks, 256, 0, s>>>(a, sums);
    SRF_LAUNCH_CHECK("linear_join_kernel");
    return 0;
}
// `sums`: column sums that ride along where the product is joined; `in_sums`: lin_part_bytes
template <typename T, typename O> static int lin_run(LinArgs a, const LinPlan& plan, void* ws, bool in_sums, const ColumnSums& sums, hipStream_t s) {
    lin_fill(a, plan, ws, in_sums);
    if (plan.kind == 1) {
        if (a.M == 1) lin_few<T, O, 1>(a, s);
        else if (a.M == 2) lin_few<T, O, 2>(a, s);
        else if (a.M <= 4) lin_few<T, O, 4>(a, s);
        else lin_few<T, O, 8>(a, s);
        SRF_LAUNCH_CHECK("linear_few_kernel");
        return 0;
    }
    if (plan.kind == 2) {
        int e;
        if constexpr (T::code == SCENERF_T_F32) e = linear_tile_f32(a, plan.tile, s);
        else if constexpr (T::code == SCENERF_T_BF16) e = linear_tile_bf16(a, plan.tile, s);
        else if constexpr (T::code == SCENERF_T_F16) e = linear_tile_f16(a, plan.tile, s);
        else e = linear_tile_e4m3(a, plan.tile, O::code, s);
        if (e) return e;
    } else {
        a.tiles_j = cdiv(a.N, ANY_TILE);
        const long blocks = (long)((a.M + ANY_TILE - 1L) / ANY_TILE) * a.tiles_j;
        SRF_CHECK(blocks < (1L << 32) / 256, "linear: %ld tiles are more than one launch holds", blocks);
        linear_any_kernel<T, O><<<dim3((unsigned)blocks, a.splits), 256, 0, s>>>(a);
        SRF_LAUNCH_CHECK("linear_any_kernel");
    }
    return in_sums ? lin_join<TypeF32>(a, sums, s) : lin_join<O>(a, sums, s);
}
static int lin_product(int in_type, int out_type, const LinArgs& a, const LinPlan& plan, void* ws, const ColumnSums& sums, hipStream_t s) {
    const bool in_sums = in_type != SCENERF_T_E4M3 && out_type != in_type;
    switch (in_type) {
        case SCENERF_T_F32: return lin_run<TypeF32, TypeF32>(a, plan, ws, false, sums, s);
        case SCENERF_T_BF16: return lin_run<TypeBF16, TypeBF16>(a, plan, ws, in_sums, sums, s);
        case SCENERF_T_F16: return lin_run<TypeF16, TypeF16>(a, plan, ws, in_sums, sums, s);
        default:
            if (out_type == SCENERF_T_F32) return lin_run<TypeE4M3, TypeF32>(a, plan, ws, false, sums, s);
            if (out_type == SCENERF_T_BF16) return lin_run<TypeE4M3, TypeBF16>(a, plan, ws, false, sums, s);
            return lin_run<TypeE4M3, TypeF16>(a, plan, ws, false, sums, s);
    }
}
// dx and dw in one launch, then dw's join
static int lin_pair(int type, int dw_type, LinArgs dx, const LinPlan& plan_x, LinArgs dw, const LinPlan& plan_w, void* ws, const ColumnSums& sums, hipStream_t s) {
    lin_fill(dx, plan_x, nullptr);
    lin_fill(dw, plan_w, ws, dw_type != type);
    if (int e = type == SCENERF_T_F32 ? linear_pair_f32(dx, dw, plan_x.tile, s) : type == SCENERF_T_BF16 ? linear_pair_bf16(dx, dw, plan_x.tile, s) : linear_pair_f16(dx, dw, plan_x.tile, s)) return e;
    return dw_type == SCENERF_T_F32 ? lin_join<TypeF32>(dw, sums, s) : dw_type == SCENERF_T_BF16 ? lin_join<TypeBF16>(dw, sums, s) : lin_join<TypeF16>(dw, sums, s);
}

// A matrix whose rows the staged kernel can read in 16-byte pieces: aligned base and pitch, a length of whole pieces (or zeros up to one),
// and a pitch whose 256 rows stay inside a 32-bit offset
#define LIN_MAX_PITCH_BYTES (1 << 22)
static int lin_pitch(int cols, int es) { return round_up(cols, 16 / es); }
static bool lin_pieces(const void* p, int64_t ld, int cols, int es, bool padded) {
    return aligned16(p) && (ld * es) % 16 == 0 && ld * es <= LIN_MAX_PITCH_BYTES && (padded ? ld >= lin_pitch(cols, es) : (cols * (int64_t)es) % 16 == 0);
}
// Large tiles read w once per row of tiles: rows of w that start inside a line make every 128-byte chunk touch two (1,536 x 2,480 bf16
// against 153,600 rows: 1,073 us, 1,043 with w's rows on lines, 8 bit 686 and 646), so w is copied to a pitch of whole lines where it is
// small beside x.
static int lin_line_pitch(int k, int es) { return round_up(k, 128 / es); }
static bool lin_onto_lines(const scenerf_linear* p, const LinPlan& plan) {
    const int es = lin_es(p->in_type);
    return plan.kind == 2 && plan.tile == LIN_256x256 && ((p->ldw * es) % 128 || (uintptr_t)p->w % 128) && p->rows >= 16LL * p->n &&
           (int64_t)lin_line_pitch(p->k, es) * es <= LIN_MAX_PITCH_BYTES;
}
static int64_t lin_onto_lines_bytes(const scenerf_linear* p, const LinPlan& plan) {
    return lin_onto_lines(p, plan) ? align256((int64_t)p->n * lin_line_pitch(p->k, lin_es(p->in_type)) * lin_es(p->in_type)) : 0;
}
static LinPlan lin_forward_plan(const scenerf_linear* p) {
    const int es = lin_es(p->in_type);
    const bool staged = lin_pieces(p->x, p->ldx, p->k, es, p->padded) && lin_pieces(p->w, p->ldw, p->k, es, p->padded);
    return lin_plan(p->in_type, false, false, staged, p->rows, p->n, p->k);
}

static int lin_copy_rows(int es, int cols, int pitch, PadSide x, PadSide w, hipStream_t s) {
    const long pieces = (x.rows + w.rows) * (pitch / (16 / es));
    if (pieces == 0) return 0;
    const unsigned blocks = (unsigned)(pieces < 8192L * 256 ? (pieces + 255) / 256 : 8192);
    if (es == 4) linear_pad_kernel<uint32_t><<<blocks, 256, 0, s>>>(x, w, cols, pitch);
    else if (es == 2) linear_pad_kernel<uint16_t><<<blocks, 256, 0, s>>>(x, w, cols, pitch);
    else linear_pad_kernel<uint8_t><<<blocks, 256, 0, s>>>(x, w, cols, pitch);
    SRF_LAUNCH_CHECK("linear_pad_kernel");
    return 0;
}

#define DZ_STRIPS 1024               // strips of rows: four workgroups a CU at 32 columns of 8
static int dz_strip(int64_t rows) {
    const int64_t per = (rows + DZ_STRIPS - 1) / DZ_STRIPS;
    return per < 8 ? 8 : (int)((per + 7) / 8 * 8);
}
struct BackwardPlan {
    bool make_dz;                   // dz is not dy itself
    // dz of 16 bits is rounded in front of its products (z, in its slopes, as it was kept): dx and dw are 1.45 times as far from exact, in the
    // 2-norm, as their own rounding makes them, whatever the inputs and sizes.  Where dz, or dx or dw, has few values the rounding is undone: its
    // rest is a second operand of the product, 1.05 times.  The counts are not a caller's accuracy, they are where that is worth its cost: of
    // few values the worst is now and then twice as far, which a mean over many hides, and going over a short contraction again costs
    // little (a layer above them is less exact than one below, at 1.45).
    bool rest_x, rest_w;
    int strip, strips, dz_pitch;
    bool scaled;                    // dz is held times a power of two (linear_dy_max_kernel)
    int64_t part, dz, rest, most, sums;     // offsets of the column sums' parts, of dz, of its rest, of the strips' largest |dy| and of the split sums
    int64_t bytes;
    LinPlan dx, dw;
    // One launch for both where they are on tiles of one shape, two workgroups or more a CU: dw's start first, dx's fill the CUs behind them.
    // With dz and all: 64 x 512 x 512 bf16 14.3 -> 11.2 us, 4,800 x 512 x 512 36 -> 30 and fp32 80 -> 71, 262,144 x 128 x 128 fp32 263 -> 248; with dx in
    // front 20,000 x 256 x 256 fp32 took 90 us, not 74 (apart 83).  Tiles of 256, one a CU, gain nothing (153,600 x 512 x 512: 325 and 326).
    bool pair;
};
static BackwardPlan lin_backward_plan(const scenerf_linear* p) {
    BackwardPlan b = {};
    const int es = lin_es(p->in_type);
    const bool products = (p->dx || p->dw) && p->rows > 0;
    b.dz_pitch = round_up(p->n, 8);
    const bool dz_fits = (int64_t)b.dz_pitch * es <= LIN_MAX_PITCH_BYTES;
    // (a dy that cannot be read in pieces becomes a dz that can, with zeros behind its rows)
    b.make_dz = products && (p->activation != SCENERF_ACT_NONE || (dz_fits && !lin_pieces(p->dy, p->ld_dy, p->n, es, false)));
    b.strip = dz_strip(p->rows);
    b.strips = (int)((p->rows + b.strip - 1) / b.strip);
    const bool few = (int64_t)p->rows * p->n < 32768, rounds = products && es == 2 && p->activation != SCENERF_ACT_NONE;
    b.rest_x = rounds && p->dx && (few || (int64_t)p->rows * p->k < 16384);
    b.rest_w = rounds && p->dw && (few || (int64_t)p->n * p->k < 16384);
    b.dx = lin_plan(p->in_type, false, true, dz_fits && lin_pieces(p->w, p->ldw, p->k, es, p->padded), p->rows, p->k, p->n, LIN_TILES, !b.rest_x);
    b.dw = lin_plan(p->in_type, true, true, dz_fits && lin_pieces(p->x, p->ldx, p->k, es, p->padded), p->n, p->k, p->rows,
                    p->dx && b.dx.kind == 2 && b.dx.splits == 1 && b.dx.tile != LIN_256x256 ? b.dx.tile : LIN_TILES, !b.rest_w);
    b.pair = p->dx && p->dw && p->rows > 0 && b.dx.kind == 2 && b.dw.kind == 2 && b.dx.tile == b.dw.tile && b.dx.tile != LIN_256x256 && b.dx.splits == 1;
    b.scaled = b.make_dz && p->in_type == SCENERF_T_F16 && (p->activation == SCENERF_ACT_GELU || p->activation == SCENERF_ACT_SILU);
    int64_t at = 0;
    if (p->db) { b.part = at; at += align256((int64_t)b.strips * p->n * 4); }
    if (b.make_dz) { b.dz = at; at += align256(p->rows * b.dz_pitch * es); }
    if (b.rest_x || b.rest_w) { b.rest = at; at += align256(p->rows * b.dz_pitch * es); }
    if (b.scaled) { b.most = at; at += align256((b.strips + 1) * 4LL); }        // (the last one: the products' factor)
    b.sums = at;
    const int64_t sx = p->dx ? lin_part_bytes(b.dx, p->rows, p->k) : 0, sw = p->dw ? lin_part_bytes(b.dw, p->n, p->k, p->out_type != p->in_type) : 0;
    b.bytes = at + (sx > sw ? sx : sw);
    return b;
}
static int lin_check(const scenerf_linear* p, const char* what, bool backward) {
    SRF_CHECK(p, "%s: NULL argument", what);
    SRF_CHECK(p->in_type >= SCENERF_T_F32 && p->in_type <= SCENERF_T_E4M3 && p->out_type >= SCENERF_T_F32 && p->out_type <= SCENERF_T_F16,
              "%s: types must be F32, BF16, F16 or (x and w) E4M3", what);
    SRF_CHECK(p->in_type == SCENERF_T_E4M3 || p->in_type == p->out_type || (backward && p->out_type == SCENERF_T_F32), "%s: in_type and out_type differ", what);
    SRF_CHECK(p->activation >= SCENERF_ACT_NONE && p->activation <= SCENERF_ACT_SILU, "%s: unknown activation %d", what, p->activation);
    SRF_CHECK(p->n >= 1 && p->k >= 1 && p->n < ROWOPS_GRID_MAX - 1024 && p->k < ROWOPS_GRID_MAX - 1024, "%s: n and k must be in [1, 2^31 - 1024)", what);
    SRF_CHECK(p->rows >= 0 && p->rows < ROWOPS_GRID_MAX - 1024, "%s: rows must be in [0, 2^31 - 1024)", what);
    SRF_CHECK(p->ldx >= 0 && p->ldw >= 0 && p->ld_residual >= 0 && p->ld_dy >= 0, "%s: negative leading dimension", what);
    if (backward) {
        SRF_CHECK(p->in_type != SCENERF_T_E4M3, "%s: the 8-bit form has no gradients", what);
        if (p->rows == 0) return 0;         // (an empty dx has no address)
        SRF_CHECK(p->dx || p->dw || p->db, "%s: nothing to compute", what);
        SRF_CHECK(p->dy && (p->w || !p->dx) && (p->x || !p->dw), "%s: NULL dy, w or x", what);
        SRF_CHECK(p->activation == SCENERF_ACT_NONE || p->z, "%s: z is NULL", what);
    } else if (p->rows > 0) {
        SRF_CHECK(p->x && p->w && p->y, "%s: NULL x, w or y", what);
        SRF_CHECK(p->in_type != SCENERF_T_E4M3 || (p->x_scale && p->w_scale), "%s: NULL x_scale or w_scale", what);
    }
    return 0;
}
template <typename O> static int lin_dz(const scenerf_linear* p, const BackwardPlan& b, void* dz, void* rest, float* part, float* most, hipStream_t s) {
    float* unscale = most ? most + b.strips : nullptr;
    if (most) {
        if (p->n % 8 == 0) linear_dy_max_kernel<true><<<b.strips, 256, 0, s>>>(p->dy, p->ld_dy, most, (int)p->rows, p->n, b.strip);
        else linear_dy_max_kernel<false><<<b.strips, 256, 0, s>>>(p->dy, p->ld_dy, most, (int)p->rows, p->n, b.strip);
        SRF_LAUNCH_CHECK("linear_dy_max_kernel");
    }
    int lx = 2;
    while (lx < 6 && (8 << lx) < p->n) ++lx;
    const dim3 grid(b.strips, cdiv(p->n, 8 << lx));
    SRF_CHECK(grid.y <= 65535, "linear_backward: n is too large");
    if (p->n % 8 == 0) linear_dz_kernel<O, true><<<grid, 256, 0, s>>>(p->dy, p->ld_dy, p->z, dz, rest, b.dz_pitch, part, most, unscale, (int)p->rows, p->n, p->activation,
                                                                         b.strip, lx);
    else linear_dz_kernel<O, false><<<grid, 256, 0, s>>>(p->dy, p->ld_dy, p->z, dz, rest, b.dz_pitch, part, most, unscale, (int)p->rows, p->n, p->activation,
                                                                         b.strip, lx);
    SRF_LAUNCH_CHECK("linear_dz_kernel");
    return 0;
}

extern "C" {

int scenerf_hip_linear_pad(int type, int k, const void* x, int64_t ldx, int64_t rows, void* x_out, const void* w, int64_t ldw, int n, void* w_out,
                           scenerf_stream_t stream) {
    SRF_CHECK(type >= SCENERF_T_F32 && type <= SCENERF_T_E4M3, "linear_pad: unknown type %d", type);
    SRF_CHECK(k >= 1 && k < ROWOPS_GRID_MAX - 1024 && rows >= 0 && rows < ROWOPS_GRID_MAX - 1024 && n >= 0 && ldx >= 0 && ldw >= 0, "linear_pad: bad sizes");
    SRF_CHECK(!x == !x_out && !w == !w_out, "linear_pad: a matrix and its copy go together");
    SRF_CHECK(aligned16(x_out) && aligned16(w_out), "linear_pad: the copies must be aligned to 16 bytes");
    const int es = lin_es(type);
    SrfLaunchScope ps(as_stream(stream), "linear_pad", 0, 2. * (rows + n) * k * es);
    return lin_copy_rows(es, k, lin_pitch(k, es), PadSide{x, x_out, ldx, x ? rows : 0}, PadSide{w, w_out, ldw, w ? n : 0}, as_stream(stream));
}

int64_t scenerf_hip_linear_workspace(const scenerf_linear* p, int backward) {
    if (lin_check(p, "linear_workspace", backward != 0)) return -1;
    if (backward) return lin_backward_plan(p).bytes;
    const LinPlan plan = lin_forward_plan(p);
    return lin_onto_lines_bytes(p, plan) + lin_part_bytes(plan, p->rows, p->n);
}

int scenerf_hip_linear_forward(const scenerf_linear* p, scenerf_stream_t stream) {
    if (int e = lin_check(p, "linear_forward", false)) return e;
    if (p->rows == 0) return 0;
    const LinPlan plan = lin_forward_plan(p);
    const int64_t lines = lin_onto_lines_bytes(p, plan), need = lines + lin_part_bytes(plan, p->rows, p->n);
    if (need > 0 && !(p->workspace && aligned16(p->workspace) && p->workspace_bytes >= need)) {
        srf_set_error("linear_forward: workspace of %lld bytes needed", (long long)need);
        return SCENERF_NEEDS_WORKSPACE;
    }
    const double m = (double)p->rows, es = lin_es(p->in_type), eo = lin_es(p->out_type);
    hipStream_t s = as_stream(stream);
    SrfLaunchScope ps(s, "linear_forward", 2 * m * p->n * p->k, es * (m * p->k + (double)p->n * p->k) + eo * m * p->n);
    LinArgs a = {};
    a.A = p->x; a.a_i = p->ldx; a.a_k = 1;
    a.B = p->w; a.b_j = p->ldw; a.b_k = 1;
    a.M = (int)p->rows; a.N = p->n; a.K = plan.kind == 2 && p->padded ? lin_pitch(p->k, (int)es) : p->k;
    if (p->in_type == SCENERF_T_E4M3) { a.row_scale = p->x_scale; a.col_scale = p->w_scale; }
    a.bias = p->bias; a.residual = p->residual; a.ld_residual = p->ld_residual;
    a.out = p->y; a.z = p->z; a.act = p->activation;
    if (lines) {
        const int pitch = lin_line_pitch(p->k, (int)es), cols = p->padded ? lin_pitch(p->k, (int)es) : p->k;
        if (int e = lin_copy_rows((int)es, cols, pitch, PadSide{nullptr, nullptr, 0, 0}, PadSide{p->w, p->workspace, p->ldw, p->n}, s)) return e;
        a.B = p->workspace;
        a.b_j = pitch;
    }
    return lin_product(p->in_type, p->out_type, a, plan, (char*)p->workspace + lines, ColumnSums{}, s);
}

int scenerf_hip_linear_backward(const scenerf_linear* p, scenerf_stream_t stream) {
    if (int e = lin_check(p, "linear_backward", true)) return e;
    hipStream_t s = as_stream(stream);
    const BackwardPlan b = lin_backward_plan(p);
    if (b.bytes > 0 && !(p->workspace && aligned16(p->workspace) && p->workspace_bytes >= b.bytes)) {
        srf_set_error("linear_backward: workspace of %lld bytes needed", (long long)b.bytes);
        return SCENERF_NEEDS_WORKSPACE;
    }
    const double m = (double)p->rows, es = lin_es(p->in_type);
    SrfLaunchScope ps(s, "linear_backward", 2 * m * p->n * p->k * (!!p->dx + !!p->dw), es * m * (p->n + 2. * p->k));
    char* ws = (char*)p->workspace;
    float* part = (float*)(ws + b.part);
    const void* dz = b.make_dz ? ws + b.dz : p->dy;
    const long ld_dz = b.make_dz ? b.dz_pitch : p->ld_dy;
    void* rest = b.rest_x || b.rest_w ? ws + b.rest : nullptr;
    const float* unscale = b.scaled ? (const float*)(ws + b.most) + b.strips : nullptr;
    if (p->rows > 0 && (b.make_dz || p->db)) {
        float* sums = p->db ? part : nullptr;
        void* to = b.make_dz ? (void*)dz : nullptr;
        int e = p->in_type == SCENERF_T_F32 ? lin_dz<TypeF32>(p, b, to, nullptr, sums, nullptr, s)
                : p->in_type == SCENERF_T_BF16 ? lin_dz<TypeBF16>(p, b, to, rest, sums, nullptr, s)
                : lin_dz<TypeF16>(p, b, to, rest, sums, b.scaled ? (float*)(ws + b.most) : nullptr, s);
        if (e) return e;
    }
    ColumnSums sums = {};
    if (p->db && p->dw && b.dw.splits > 1) sums = {part, p->db, b.strips, p->n, cdiv(p->n, 16)};
    else if (p->db) {
        if (int e = launch_sum_parts(p->out_type, part, b.strips, p->n, p->db, s)) return e;
    }
    const int pitch = lin_pitch(p->k, (int)es);
    LinArgs ax = {}, aw = {};
    if (p->dx && p->rows > 0) {
        ax.A = dz; ax.a_i = ld_dz; ax.a_k = 1;
        ax.B = p->w; ax.b_j = 1; ax.b_k = p->ldw;
        ax.M = (int)p->rows; ax.N = p->k; ax.K = p->n;
        ax.b_ext = pitch;
        ax.out = p->dx;
        ax.A2 = b.rest_x ? rest : nullptr;
        ax.unscale = unscale;
    }
    if (p->dw) {     // rows == 0: an empty sum, zeros
        aw.A = dz; aw.a_i = 1; aw.a_k = ld_dz;
        aw.B = p->x; aw.b_j = 1; aw.b_k = p->ldx;
        aw.M = p->n; aw.N = p->k; aw.K = (int)p->rows;
        aw.a_ext = b.make_dz ? b.dz_pitch : p->n; aw.b_ext = pitch;
        aw.out = p->dw;
        aw.A2 = b.rest_w ? rest : nullptr;
        aw.unscale = unscale;
    }
    if (b.pair) return lin_pair(p->in_type, p->out_type, ax, b.dx, aw, b.dw, ws + b.sums, sums, s);
    if (ax.out)
        if (int e = lin_product(p->in_type, p->in_type, ax, b.dx, ws + b.sums, ColumnSums{}, s)) return e;
    if (aw.out)
        if (int e = lin_product(p->in_type, p->out_type, aw, b.dw, ws + b.sums, sums, s)) return e;
    return 0;
}

}  // extern "C"
