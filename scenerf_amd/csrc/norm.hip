// RMS norm of rows with the residual's addition, rows in 8 bits with scales, and the norm's gradients (gfx950).
//
//   h = x + r;  rstd = (mean h^2 + eps)^-1/2;  v = h rstd w;  y = v;  scale = max(max|v| / 448, 2^-126), q = e4m3(v / scale)
//   dx = rstd (dy w - xhat mean(dy w xhat)) + dh,  xhat = h rstd;  dw = sum over rows of dy xhat
//
// All of it is bound by HBM: each input is read once and each output written once, everything in between lives in registers.  One
// wave owns a row (the two row sums are one 6-step exchange, no barrier), holds it in registers up to ROW_REGS elements a lane, and
// walks the rows in a grid stride, so that the weight is loaded once per wave.  Wider rows, and few
// wide ones, go through a workgroup that reads the row twice (the second time from L2).  The weight's gradient is summed per lane over the wave's rows, then over the workgroup's waves in
// LDS, then over the workgroups by a second kernel in a fixed order: no atomics, the same bits every time.  Rows of any length and
// alignment move 16 bytes at a time, but for a last piece that the row does not fill.
// 153,600 x 512 bf16: forward with residual 107 us for 629 MB (5.9 TB/s; a large copy reaches 5.2), gradients with residual 159 + 5 for 786 MB (5.0), 8
// bits 101 to 108 us for 551 MB; 40,001 x 2,480 fp16 to 8 bits 62 to 66 us for 298 MB; 4,801 x 515 fp32 out of wider rows 8.6 us.  20,000 x 8,192
// bf16, wider than a wave holds: forward 251 us for 1,311 MB, dx 331 for 1,638 MB at dh with it, dweight 525 (x, residual and dy once more,
// two bytes a lane: 1.9 TB/s, the slowest pass here by its bytes).
#include "rowops.h"

#define ROW_WAVES 4
#define ROW_REGS 64                 // elements of a row a lane holds at most: 4096 columns
#define WIDE_THREADS 1024

// the largest |v| as bits: NaN is above infinity, so a row's NaN survives the maximum
__device__ static inline uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }
__device__ static inline uint32_t wave_max_u32(uint32_t v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const uint32_t t = (uint32_t)__shfl_xor((int)v, o, WAVE);
        v = t > v ? t : v;
    }
    return v;
}
__device__ static inline float row_scale(uint32_t max_bits) {
    const float m = __uint_as_float(max_bits) / 448.f;
    return m < 1.1754943508222875e-38f ? 1.1754943508222875e-38f : m;   // NaN stays
}
// v / s of a row's values.  Values of 16 bits lie on e4m3's ties often, so the quotient has to be a rounded one: a product with 1 / s put one of
// 80 bf16 values a whole step off.  v (1 / s) is off by 1.5 units at most, its remainder against s brings it to the quotient but for 2^-23 of a
// unit, rounded once (Markstein's correction).  The remainder of a row under 2^-80 would underflow: such a row is `small`, and its
// values come times 2^64, as s does here.  The compiler's full division took 70 us for 40,001 x 2,480 fp16 rows, this 62, the product
// alone 60.  s not finite: 0 or NaN.
struct RowQuotient {
    float inv, s;
    bool small;
    __device__ inline RowQuotient(float scale) {
        small = scale < 0x1p-88f;
        s = small ? scale * 0x1p64f : scale;
        inv = 1.f / s;
        if (!(s < __builtin_inff())) s = 0.f;
    }
    __device__ inline float operator()(float v) const {
        const float q = v * inv;
        return fmaf(-fmaf(q, s, -v), inv, q);       // (in this order -0 stays -0)
    }
};

struct RmsArgs {
    const void* x; const void* residual; const void* weight;
    void* h; void* y; uint8_t* q; float* scale; float* rstd;
    const void* dy; const void* dh; void* dx;
    float* partial;
    long ldx, ld_residual, ld_dy, ld_dh;
    int rows, width;
    float eps, inv_width;
};

// C chunks of 64 * VW columns: lane l holds columns c * 64 * VW + l * VW ..+ VW
template <typename E, int VW, int C, bool WHOLE>
__global__ __launch_bounds__(64 * ROW_WAVES) void rms_rows_kernel(RmsArgs p) {
    typedef typename E::raw raw;
    const int lane = threadIdx.x & 63;
    const int D = p.width;
    float w[C][VW];
    int in[C];          // elements of the lane's pieces that are inside the row
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int col = (c * 64 + lane) * VW;
        in[c] = D - col;
#pragma unroll
        for (int e = 0; e < VW; ++e) w[c][e] = 0.f;
        if (in[c] > 0 && p.weight) load_some<E, VW, WHOLE>((const raw*)p.weight + col, in[c], D % VW, w[c]);
    }
    const int waves = gridDim.x * ROW_WAVES;
    for (long row = (long)blockIdx.x * ROW_WAVES + (threadIdx.x >> 6); row < p.rows; row += waves) {
        float h[C][VW];
        float ss = 0.f;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int col = (c * 64 + lane) * VW;
#pragma unroll
            for (int e = 0; e < VW; ++e) h[c][e] = 0.f;
            if (in[c] > 0) load_some<E, VW, WHOLE>((const raw*)p.x + row * p.ldx + col, in[c], D % VW, h[c]);
        }
        if (p.residual) {
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const int col = (c * 64 + lane) * VW;
                if (in[c] > 0) {
                    float r[VW];
                    load_some<E, VW, WHOLE>((const raw*)p.residual + row * p.ld_residual + col, in[c], D % VW, r);
#pragma unroll
                    for (int e = 0; e < VW; ++e) h[c][e] += r[e];
                    if (p.h) store_some<E, VW, WHOLE>((raw*)p.h + row * D + col, in[c], D % VW, h[c]);
                }
            }
        }
        if (p.weight) {
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int e = 0; e < VW; ++e) ss = fmaf(h[c][e], h[c][e], ss);
            ss = wave_sum(ss);
            const float rstd = 1.f / sqrtf(fmaf(ss, p.inv_width, p.eps));
            if (p.rstd && lane == 0) p.rstd[row] = rstd;
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int e = 0; e < VW; ++e) h[c][e] = h[c][e] * rstd * w[c][e];
        }
        if (p.y) {
#pragma unroll
            for (int c = 0; c < C; ++c)
                if (in[c] > 0) store_some<E, VW, WHOLE>((raw*)p.y + row * D + (c * 64 + lane) * VW, in[c], D % VW, h[c]);
        }
        if (p.q) {
            uint32_t m = 0;
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int e = 0; e < VW; ++e) {
                    const uint32_t b = (WHOLE ? in[c] > 0 : e < in[c]) ? abs_bits(h[c][e]) : 0u;
                    m = b > m ? b : m;
                }
            const float s = row_scale(wave_max_u32(m));
            if (lane == 0) p.scale[row] = s;
            const RowQuotient over(s);
            if (over.small)
#pragma unroll
                for (int c = 0; c < C; ++c)
#pragma unroll
                    for (int e = 0; e < VW; ++e) h[c][e] *= 0x1p64f;
#pragma unroll
            for (int c = 0; c < C; ++c)
                if (in[c] > 0) {
                    float v[VW];
#pragma unroll
                    for (int e = 0; e < VW; ++e) v[e] = over(h[c][e]);
                    store_some<TypeE4M3, VW, WHOLE>(p.q + row * D + (c * 64 + lane) * VW, in[c], D % VW, v);
                }
        }
    }
}

// rows wider than a wave's registers: one workgroup a row, two reads
__device__ static inline float block_sum(float v, float* red) {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.f;
    for (int i = 0; i < WIDE_THREADS / 64; ++i) v += red[i];
    return v;
}
__device__ static inline uint32_t block_max_u32(uint32_t v, uint32_t* red) {
    v = wave_max_u32(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0;
    for (int i = 0; i < WIDE_THREADS / 64; ++i) v = red[i] > v ? red[i] : v;
    return v;
}
template <typename E, int VW, bool WHOLE>
__global__ __launch_bounds__(WIDE_THREADS) void rms_rows_wide_kernel(RmsArgs p) {
    typedef typename E::raw raw;
    __shared__ float red[WIDE_THREADS / 64];
    const long D = p.width;
    for (long row = blockIdx.x; row < p.rows; row += gridDim.x) {
        float ss = 0.f;
        uint32_t m = 0;
        for (long col = (long)threadIdx.x * VW; col < D; col += WIDE_THREADS * VW) {
            float h[VW];
            load_some<E, VW, WHOLE>((const raw*)p.x + row * p.ldx + col, (int)min(D - col, (long)VW), (int)(D % VW), h);
            if (p.residual) {
                float r[VW];
                load_some<E, VW, WHOLE>((const raw*)p.residual + row * p.ld_residual + col, (int)min(D - col, (long)VW), (int)(D % VW), r);
#pragma unroll
                for (int e = 0; e < VW; ++e) h[e] += r[e];
                if (p.h) store_some<E, VW, WHOLE>((raw*)p.h + row * D + col, (int)min(D - col, (long)VW), (int)(D % VW), h);
            }
            float w[VW];
#pragma unroll
            for (int e = 0; e < VW; ++e) w[e] = 1.f;
            if (p.weight) load_some<E, VW, WHOLE>((const raw*)p.weight + col, (int)min(D - col, (long)VW), (int)(D % VW), w);
#pragma unroll
            for (int e = 0; e < VW; ++e) {
                ss = fmaf(h[e], h[e], ss);
                const uint32_t b = abs_bits(h[e] * w[e]);
                m = b > m ? b : m;
            }
        }
        float rstd = 1.f;
        if (p.weight) {
            rstd = 1.f / sqrtf(fmaf(block_sum(ss, red), p.inv_width, p.eps));
            if (p.rstd && threadIdx.x == 0) p.rstd[row] = rstd;
        }
        float s = 1.f;
        if (p.q) {
            // max |h rstd w| = rstd max |h w|: the last bit may differ from the largest value's own, the scale's rounding
            m = block_max_u32(m, (uint32_t*)red);
            float top = __uint_as_float(m) * rstd;
            // h w alone overflows, or is too small to hold its bits (and its scale is not at its floor): once more, in the order that y has
            if (p.weight && (m == 0x7f800000u || (m < 0x00800000u && rstd > 448.f))) {
                m = 0;
                for (long col = threadIdx.x; col < D; col += WIDE_THREADS) {
                    float h = E::to_f32(((const raw*)p.x)[row * p.ldx + col]);
                    if (p.residual) h += E::to_f32(((const raw*)p.residual)[row * p.ld_residual + col]);
                    const uint32_t b = abs_bits(h * rstd * E::to_f32(((const raw*)p.weight)[col]));
                    m = b > m ? b : m;
                }
                top = __uint_as_float(block_max_u32(m, (uint32_t*)red));
            }
            s = row_scale(abs_bits(top));
            if (threadIdx.x == 0) p.scale[row] = s;
        }
        const RowQuotient over(s);
        for (long col = (long)threadIdx.x * VW; col < D; col += WIDE_THREADS * VW) {
            float h[VW];
            load_some<E, VW, WHOLE>((const raw*)p.x + row * p.ldx + col, (int)min(D - col, (long)VW), (int)(D % VW), h);
            if (p.residual) {
                float r[VW];
                load_some<E, VW, WHOLE>((const raw*)p.residual + row * p.ld_residual + col, (int)min(D - col, (long)VW), (int)(D % VW), r);
#pragma unroll
                for (int e = 0; e < VW; ++e) h[e] += r[e];
            }
            if (p.weight) {
                float w[VW];
                load_some<E, VW, WHOLE>((const raw*)p.weight + col, (int)min(D - col, (long)VW), (int)(D % VW), w);
#pragma unroll
                for (int e = 0; e < VW; ++e) h[e] = h[e] * rstd * w[e];
            }
            if (p.y) store_some<E, VW, WHOLE>((raw*)p.y + row * D + col, (int)min(D - col, (long)VW), (int)(D % VW), h);
            if (p.q) {
#pragma unroll
                for (int e = 0; e < VW; ++e) h[e] = over(over.small ? h[e] * 0x1p64f : h[e]);
                store_some<TypeE4M3, VW, WHOLE>(p.q + row * D + col, (int)min(D - col, (long)VW), (int)(D % VW), h);
            }
        }
    }
}

// gradients: dx, and this workgroup's part of dweight in partial[blockIdx.x][width]
template <typename E, int VW, int C, bool WHOLE>
__global__ __launch_bounds__(64 * ROW_WAVES) void rms_grad_kernel(RmsArgs p) {
    typedef typename E::raw raw;
    __shared__ float red[ROW_WAVES][64 * VW];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    const int D = p.width;
    float w[C][VW], dw[C][VW];
    int in[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int col = (c * 64 + lane) * VW;
        in[c] = D - col;
#pragma unroll
        for (int e = 0; e < VW; ++e) w[c][e] = dw[c][e] = 0.f;
        if (in[c] > 0) load_some<E, VW, WHOLE>((const raw*)p.weight + col, in[c], D % VW, w[c]);
    }
    const int waves = gridDim.x * ROW_WAVES;
    // the next row's three loads are under way while this one is worked on (narrow rows: with one row at a time the 8 waves a CU had too
    // few bytes in flight, 180 us for 153,600 x 512 bf16)
    constexpr bool AHEAD = C * VW <= 16;
    float nh[C][VW], ng[C][VW], nd[C][VW], nr = 0.f;
    auto get = [&](long row, float (&h)[C][VW], float (&g)[C][VW], float (&d)[C][VW], float& rstd) {
        rstd = p.rstd[row];
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int col = (c * 64 + lane) * VW;
#pragma unroll
            for (int e = 0; e < VW; ++e) h[c][e] = g[c][e] = d[c][e] = 0.f;
            if (in[c] > 0) {
                load_some<E, VW, WHOLE>((const raw*)p.x + row * p.ldx + col, in[c], D % VW, h[c]);
                load_some<E, VW, WHOLE>((const raw*)p.dy + row * p.ld_dy + col, in[c], D % VW, g[c]);
                if (p.residual) {
                    float r[VW];
                    load_some<E, VW, WHOLE>((const raw*)p.residual + row * p.ld_residual + col, in[c], D % VW, r);
#pragma unroll
                    for (int e = 0; e < VW; ++e) h[c][e] += r[e];
                }
                if (AHEAD && p.dh) load_some<E, VW, WHOLE>((const raw*)p.dh + row * p.ld_dh + col, in[c], D % VW, d[c]);
            }
        }
    };
    const long first = (long)blockIdx.x * ROW_WAVES + wv;
    if (AHEAD && first < p.rows) get(first, nh, ng, nd, nr);
    for (long row = first; row < p.rows; row += waves) {
        float h[C][VW], g[C][VW], d[C][VW], rstd;
        if constexpr (AHEAD) {
            rstd = nr;
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int e = 0; e < VW; ++e) {
                    h[c][e] = nh[c][e];
                    g[c][e] = ng[c][e];
                    d[c][e] = nd[c][e];
                }
            if (row + waves < p.rows) get(row + waves, nh, ng, nd, nr);
        } else {
            get(row, h, g, d, rstd);
        }
        float dot = 0.f;
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int e = 0; e < VW; ++e) {
                h[c][e] *= rstd;
                dw[c][e] = fmaf(g[c][e], h[c][e], dw[c][e]);
                g[c][e] *= w[c][e];
                dot = fmaf(g[c][e], h[c][e], dot);
            }
        if (!p.dx) continue;
        dot = wave_sum(dot) * p.inv_width;
#pragma unroll
        for (int c = 0; c < C; ++c)
            if (in[c] > 0) {
                const int col = (c * 64 + lane) * VW;
                if (!AHEAD && p.dh) load_some<E, VW, WHOLE>((const raw*)p.dh + row * p.ld_dh + col, in[c], D % VW, d[c]);
#pragma unroll
                for (int e = 0; e < VW; ++e) d[c][e] = fmaf(rstd, fmaf(-dot, h[c][e], g[c][e]), d[c][e]);
                store_some<E, VW, WHOLE>((raw*)p.dx + row * D + col, in[c], D % VW, d[c]);
            }
    }
    if (!p.partial) return;
#pragma unroll
    for (int c = 0; c < C; ++c) {
        __syncthreads();
#pragma unroll
        for (int e = 0; e < VW; ++e) red[wv][lane * VW + e] = dw[c][e];
        __syncthreads();
        for (int i = threadIdx.x; i < 64 * VW; i += 64 * ROW_WAVES) {
            const int col = c * 64 * VW + i;
            if (col < D) {
                float s = 0.f;
#pragma unroll
                for (int k = 0; k < ROW_WAVES; ++k) s += red[k][i];
                p.partial[(size_t)blockIdx.x * D + col] = s;
            }
        }
    }
}
template <typename E, int VW, bool WHOLE>
__global__ __launch_bounds__(WIDE_THREADS) void rms_grad_wide_kernel(RmsArgs p) {
    typedef typename E::raw raw;
    __shared__ float red[WIDE_THREADS / 64];
    const long D = p.width;
    auto row_values = [&](long row, long col, float (&h)[VW]) {
        load_some<E, VW, WHOLE>((const raw*)p.x + row * p.ldx + col, (int)min(D - col, (long)VW), (int)(D % VW), h);
        if (p.residual) {
            float r[VW];
            load_some<E, VW, WHOLE>((const raw*)p.residual + row * p.ld_residual + col, (int)min(D - col, (long)VW), (int)(D % VW), r);
#pragma unroll
            for (int e = 0; e < VW; ++e) h[e] += r[e];
        }
    };
    for (long row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const float rstd = p.rstd[row];
        float dot = 0.f;
        for (long col = (long)threadIdx.x * VW; col < D; col += WIDE_THREADS * VW) {
            float h[VW], g[VW], w[VW];
            row_values(row, col, h);
            load_some<E, VW, WHOLE>((const raw*)p.dy + row * p.ld_dy + col, (int)min(D - col, (long)VW), (int)(D % VW), g);
            load_some<E, VW, WHOLE>((const raw*)p.weight + col, (int)min(D - col, (long)VW), (int)(D % VW), w);
#pragma unroll
            for (int e = 0; e < VW; ++e) dot = fmaf(g[e] * w[e], h[e] * rstd, dot);
        }
        dot = block_sum(dot, red) * p.inv_width;
        for (long col = (long)threadIdx.x * VW; col < D; col += WIDE_THREADS * VW) {
            float h[VW], g[VW], w[VW], d[VW];
            row_values(row, col, h);
            load_some<E, VW, WHOLE>((const raw*)p.dy + row * p.ld_dy + col, (int)min(D - col, (long)VW), (int)(D % VW), g);
            load_some<E, VW, WHOLE>((const raw*)p.weight + col, (int)min(D - col, (long)VW), (int)(D % VW), w);
#pragma unroll
            for (int e = 0; e < VW; ++e) d[e] = 0.f;
            if (p.dh) load_some<E, VW, WHOLE>((const raw*)p.dh + row * p.ld_dh + col, (int)min(D - col, (long)VW), (int)(D % VW), d);
#pragma unroll
            for (int e = 0; e < VW; ++e) d[e] = fmaf(rstd, fmaf(-dot, h[e] * rstd, g[e] * w[e]), d[e]);
            store_some<E, VW, WHOLE>((raw*)p.dx + row * D + col, (int)min(D - col, (long)VW), (int)(D % VW), d);
        }
    }
}
// the weight's gradient of wide rows, by columns: workgroup (x: 64 columns, y: a strip of rows)
template <typename E>
__global__ __launch_bounds__(256) void rms_dweight_cols_kernel(RmsArgs p, int strip) {
    typedef typename E::raw raw;
    __shared__ float red[4][64];
    const int col = blockIdx.x * 64 + (threadIdx.x & 63), ty = threadIdx.x >> 6;
    const long r0 = (long)blockIdx.y * strip, r1 = min((long)p.rows, r0 + strip);
    float s = 0.f;
    if (col < p.width)
        for (long r = r0 + ty; r < r1; r += 4) {
            float h = E::to_f32(((const raw*)p.x)[r * p.ldx + col]);
            if (p.residual) h += E::to_f32(((const raw*)p.residual)[r * p.ld_residual + col]);
            s = fmaf(E::to_f32(((const raw*)p.dy)[r * p.ld_dy + col]), h * p.rstd[r], s);
        }
    red[ty][threadIdx.x & 63] = s;
    __syncthreads();
    if (ty == 0 && col < p.width)
        p.partial[(size_t)blockIdx.y * p.width + col] = red[0][threadIdx.x] + red[1][threadIdx.x] + red[2][threadIdx.x] + red[3][threadIdx.x];
}

// out[col] = the sum of part[0..count)[col], in a fixed order: 32 interleaved chains per column, then their sum.  A workgroup owns 32 columns,
// so that each of its loads is a line; bound by the latency of count / 32 loads in a row, which the unrolling overlaps (1,011 x 512: 6.7 us)
template <typename E>
__global__ __launch_bounds__(1024) void sum_parts_kernel(const float* __restrict__ part, int count, int width, typename E::raw* __restrict__ out) {
    __shared__ float red[32][33];
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5, col = blockIdx.x * 32 + tx;
    float s = 0.f;
    if (col < width) {
#pragma unroll 8
        for (int i = ty; i < count; i += 32) s += part[(size_t)i * width + col];
    }
    red[ty][tx] = s;
    __syncthreads();
    s = red[tx][ty];              // column ty of the 32, chain tx: the halves of a wave add one column each
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor(s, o, WAVE);
    if (tx == 0 && blockIdx.x * 32 + ty < width) out[blockIdx.x * 32 + ty] = E::from_f32(s);
}
int launch_sum_parts(int type, const float* part, int count, int width, void* out, hipStream_t s) {
    const int blocks = cdiv(width, 32);
    if (type == SCENERF_T_F32) sum_parts_kernel<TypeF32><<<blocks, 1024, 0, s>>>(part, count, width, (float*)out);
    else if (type == SCENERF_T_BF16) sum_parts_kernel<TypeBF16><<<blocks, 1024, 0, s>>>(part, count, width, (uint16_t*)out);
    else sum_parts_kernel<TypeF16><<<blocks, 1024, 0, s>>>(part, count, width, (uint16_t*)out);
    SRF_LAUNCH_CHECK("sum_parts_kernel");
    return 0;
}

// ---------------------------------------------------------------------------------------------------------------- host side
static int rms_es(int type) { return type == SCENERF_T_F32 ? 4 : 2; }
static bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
static bool rms_in_registers(const scenerf_rms* p) { return p->width <= 64 * ROW_REGS; }
#define RMS_GRAD_BLOCKS 1024        // workgroups (and parts of dweight) of the gradient kernel: four per CU
static int rms_strip(int64_t rows) {                            // of rows in the wide dweight: 512, or what keeps the grid's second axis
    const int64_t per = (rows + 65534) / 65535;
    return per < 512 ? 512 : (int)per;
}
static int rms_grad_parts(const scenerf_rms* p) {
    if (!rms_in_registers(p)) return (int)((p->rows + rms_strip(p->rows) - 1) / rms_strip(p->rows));
    const long want = (p->rows + ROW_WAVES - 1) / ROW_WAVES;
    return (int)(want < RMS_GRAD_BLOCKS ? want : RMS_GRAD_BLOCKS);
}
static int rms_check(const scenerf_rms* p, const char* what, bool backward) {
    SRF_CHECK(p, "%s: NULL argument", what);
    SRF_CHECK(p->type >= SCENERF_T_F32 && p->type <= SCENERF_T_F16, "%s: type must be F32, BF16 or F16", what);
    SRF_CHECK(p->width >= 1 && p->rows >= 0 && p->rows < ROWOPS_GRID_MAX - 1024, "%s: width >= 1 and 0 <= rows < 2^31 - 1024", what);
    SRF_CHECK(p->eps >= 0.f, "%s: eps must not be negative", what);
    SRF_CHECK(p->dweight_f32 == 0 || p->dweight_f32 == 1, "%s: dweight_f32 is 0 or 1", what);
    SRF_CHECK(p->ldx >= 0 && p->ld_residual >= 0 && p->ld_dy >= 0 && p->ld_dh >= 0, "%s: negative leading dimension", what);
    if (p->rows == 0 && !(backward && p->dweight)) return 0;
    if (backward) {
        SRF_CHECK(p->rows == 0 || (p->x && p->weight && p->rstd && p->dy), "%s: NULL x, weight, rstd or dy", what);
        SRF_CHECK(p->dx || p->dweight, "%s: nothing to compute", what);
    } else {
        SRF_CHECK(p->x, "%s: x is NULL", what);
        SRF_CHECK(p->y || p->q || p->h, "%s: nothing to compute", what);
        SRF_CHECK(!p->h || p->residual, "%s: h is written only where a residual is added", what);
        SRF_CHECK(!p->q == !p->scale, "%s: q and scale go together", what);
        SRF_CHECK(p->weight || !p->rstd, "%s: rstd without weight", what);
    }
    return 0;
}
static RmsArgs rms_args(const scenerf_rms* p) {
    RmsArgs a = {};
    a.x = p->x; a.residual = p->residual; a.weight = p->weight; a.h = p->h; a.y = p->y; a.q = p->q; a.scale = p->scale; a.rstd = p->rstd;
    a.dy = p->dy; a.dh = p->dh; a.dx = p->dx;
    a.ldx = p->ldx; a.ld_residual = p->ld_residual; a.ld_dy = p->ld_dy; a.ld_dh = p->ld_dh;
    a.rows = (int)p->rows; a.width = p->width; a.eps = p->eps; a.inv_width = 1.f / (float)p->width;
    return a;
}

template <typename E, int VW, int C, bool WHOLE> static void rms_launch(const RmsArgs& a, bool backward, int blocks, hipStream_t s) {
    if (backward) rms_grad_kernel<E, VW, C, WHOLE><<<blocks, 64 * ROW_WAVES, 0, s>>>(a);
    else rms_rows_kernel<E, VW, C, WHOLE><<<blocks, 64 * ROW_WAVES, 0, s>>>(a);
}
// the smallest number of chunks that holds the row
template <typename E, int VW, bool WHOLE> static void rms_launch_chunks(const RmsArgs& a, bool backward, int blocks, hipStream_t s) {
    const int chunks = cdiv(a.width, 64 * VW);
    if (chunks <= 1) return rms_launch<E, VW, 1, WHOLE>(a, backward, blocks, s);
    if (chunks <= 2) return rms_launch<E, VW, 2, WHOLE>(a, backward, blocks, s);
    if (chunks <= 3) return rms_launch<E, VW, 3, WHOLE>(a, backward, blocks, s);
    if (chunks <= 4) return rms_launch<E, VW, 4, WHOLE>(a, backward, blocks, s);
    if (chunks <= 5) return rms_launch<E, VW, 5, WHOLE>(a, backward, blocks, s);
    if (chunks <= 6) return rms_launch<E, VW, 6, WHOLE>(a, backward, blocks, s);
    if (chunks <= 8) return rms_launch<E, VW, 8, WHOLE>(a, backward, blocks, s);
    if constexpr (VW == 4) {
        if (chunks <= 10) return rms_launch<E, VW, 10, WHOLE>(a, backward, blocks, s);
        if (chunks <= 12) return rms_launch<E, VW, 12, WHOLE>(a, backward, blocks, s);
        rms_launch<E, VW, 16, WHOLE>(a, backward, blocks, s);
    }
}
template <typename E, bool WHOLE> static int rms_dispatch(const scenerf_rms* p, bool backward, hipStream_t s) {
    constexpr int VW = 16 / sizeof(typename E::raw);
    RmsArgs a = rms_args(p);
    if (backward) {
        const int parts = rms_grad_parts(p);
        a.partial = p->dweight ? (float*)p->workspace : nullptr;
        if (p->rows > 0 && rms_in_registers(p)) {
            rms_launch_chunks<E, VW, WHOLE>(a, true, parts, s);
            SRF_LAUNCH_CHECK("rms_grad_kernel");
        } else if (p->rows > 0) {
            if (p->dx) {
                const int blocks = p->rows < 4096 ? (int)p->rows : 4096;
                rms_grad_wide_kernel<E, VW, WHOLE><<<blocks, WIDE_THREADS, 0, s>>>(a);
                SRF_LAUNCH_CHECK("rms_grad_wide_kernel");
            }
            if (p->dweight) {
                rms_dweight_cols_kernel<E><<<dim3(cdiv(p->width, 64), parts), 256, 0, s>>>(a, rms_strip(p->rows));
                SRF_LAUNCH_CHECK("rms_dweight_cols_kernel");
            }
        }
        if (p->dweight) return launch_sum_parts(p->dweight_f32 ? SCENERF_T_F32 : E::code, a.partial, parts, p->width, p->dweight, s);
        return 0;
    }
    // (few and wide rows: a workgroup a row is done sooner than a wave -- 64 x 4,096 bf16 4.1 against 7.5 us, 256 x 2,048 4.1 against 5.0, but
    // 256 x 1,024 4.0 against 3.8, 1,024 x 2,048 7.9 against 5.9 and 20,000 x 4,096 176 against 150)
    if (rms_in_registers(p) && !(p->rows <= 256 && p->width > 1024)) {
        const long want = (p->rows + ROW_WAVES - 1) / ROW_WAVES;
        const int blocks = (int)(want < 8192 ? want : 8192);
        rms_launch_chunks<E, VW, WHOLE>(a, false, blocks, s);
        SRF_LAUNCH_CHECK("rms_rows_kernel");
    } else {
        const int blocks = p->rows < 4096 ? (int)p->rows : 4096;
        rms_rows_wide_kernel<E, VW, WHOLE><<<blocks, WIDE_THREADS, 0, s>>>(a);
        SRF_LAUNCH_CHECK("rms_rows_wide_kernel");
    }
    return 0;
}
template <typename E> static int rms_run_type(const scenerf_rms* p, bool backward, hipStream_t s) {
    return p->width % (16 / (int)sizeof(typename E::raw)) == 0 ? rms_dispatch<E, true>(p, backward, s) : rms_dispatch<E, false>(p, backward, s);
}
static int rms_run(const scenerf_rms* p, bool backward, hipStream_t s) {
    if (p->type == SCENERF_T_F32) return rms_run_type<TypeF32>(p, backward, s);
    if (p->type == SCENERF_T_BF16) return rms_run_type<TypeBF16>(p, backward, s);
    return rms_run_type<TypeF16>(p, backward, s);
}

extern "C" {

int64_t scenerf_hip_rms_workspace(const scenerf_rms* p, int backward) {
    if (rms_check(p, "rms_workspace", backward != 0)) return -1;
    return backward && p->dweight ? (int64_t)rms_grad_parts(p) * p->width * 4 : 0;
}

int scenerf_hip_rms_forward(const scenerf_rms* p, scenerf_stream_t stream) {
    if (int e = rms_check(p, "rms_forward", false)) return e;
    if (p->rows == 0) return 0;
    const double es = rms_es(p->type), e = (double)p->rows * p->width;
    SrfLaunchScope ps(as_stream(stream), "rms_forward", 5 * e, e * (es * (1 + !!p->residual + !!p->h + !!p->y) + !!p->q));
    return rms_run(p, false, as_stream(stream));
}

int scenerf_hip_rms_backward(const scenerf_rms* p, scenerf_stream_t stream) {
    if (int e = rms_check(p, "rms_backward", true)) return e;
    if (p->rows == 0 && !p->dweight) return 0;
    const int64_t need = scenerf_hip_rms_workspace(p, 1);
    if (need > 0 && !(p->workspace && aligned16(p->workspace) && p->workspace_bytes >= need)) {
        srf_set_error("rms_backward: workspace of %lld bytes needed", (long long)need);
        return SCENERF_NEEDS_WORKSPACE;
    }
    const double es = rms_es(p->type), e = (double)p->rows * p->width;
    SrfLaunchScope ps(as_stream(stream), "rms_backward", 10 * e, e * es * (2 + !!p->dh + !!p->dx));
    return rms_run(p, true, as_stream(stream));
}

}  // extern "C"
