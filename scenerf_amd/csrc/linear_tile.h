// The staged matrix product of linear.hip: operands from HBM straight into LDS, matrix instructions fed from there, the layer's epilogue
// behind the sums.  Included by one translation unit per operand type.
//
// A workgroup owns BM x BN results and walks the contraction in chunks of 64 bytes per row.  Chunks live in a ring of NST stages, filled
// by asynchronous global -> LDS loads (16 bytes a lane, 1 KiB a wave and instruction) that run NST - 1 chunks ahead: one barrier a chunk,
// in front of which each wave waits for its own loads of that chunk by count.
//
// LDS image of an operand read ALONG the contraction: row r is 64 bytes, its 16-byte slots XORed with (r >> 1) & 3, so that the 8 lanes
// of a ds_read_b128 phase cover all banks.  The swizzle is applied on the source side of the load (LDS-bound loads place lanes in
// sequence).  An operand read ACROSS (contraction along the rows in memory) keeps its rows: [k][tile columns]; 16-bit fragments come
// out of it by the transposing read ds_read_b64_tr_b16 (within 16 lanes, lane 4r + c gives the address of 4 columns of row r, lane i
// receives rows 0..3 of column i), its 64-byte pieces XORed with k & 3; fp32 fragments are single elements anyway.
// Any order of k inside a chunk is valid as long as both operands use the same.
//
// The matrix instruction gets the operands swapped (B's rows first), so that a lane's four consecutive accumulators are four
// consecutive columns of one result row; the tile passes through LDS once more, 32 rows of a wave at a time, and leaves as full lines.
#pragma once
#include "linear.h"

typedef __attribute__((ext_vector_type(8))) __bf16 lin_bf16x8;
typedef __attribute__((ext_vector_type(8))) _Float16 lin_f16x8;
typedef __attribute__((ext_vector_type(16))) float lin_f32x16;
typedef __attribute__((ext_vector_type(8))) int lin_i32x8;
typedef __attribute__((ext_vector_type(4))) short lin_s16x4;

__device__ __attribute__((aligned(16))) const unsigned lin_zeros[4] = {0, 0, 0, 0};

// 64 lanes x 16 bytes, global -> LDS at lds_base + lane * 16 (m0 is the base; saved around, the compiler owns it)
__device__ static inline void lin_copy(const void* sbase, unsigned voff, unsigned lds_base) {
    unsigned keep;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep) : "v"(voff), "s"(sbase), "s"(lds_base) : "memory");
}
__device__ static inline void lin_copy_v(const void* vaddr, unsigned lds_base) {
    unsigned keep;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep) : "v"(vaddr), "s"(lds_base) : "memory");
}

// contiguous ranges of work per XCD (blocks go round-robin over the 8 XCDs, each with its own L2); any count
__device__ static inline int lin_xcd_order(int id, int total) {
    const int q = total >> 3, r = total & 7, xcd = id & 7, slot = id >> 3;
    return (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + slot;
}

// one operand's side of a stage: TILE rows (or columns) x 64 bytes of the contraction
template <typename T, bool ACROSS, int TILE> struct LinSide {
    static constexpr int ES = sizeof(typename T::raw);
    static constexpr int BK = LIN_CHUNK_BYTES / ES;
    static constexpr int BYTES = TILE * LIN_CHUNK_BYTES;
    static constexpr int PIECES = BYTES / 1024;
    static constexpr int LINE = TILE * ES;                          // ACROSS: bytes of one k
    static constexpr int SWZ = (LINE / 64 >= 4 ? 4 : LINE / 64) - 1; // ACROSS, 16-bit: which pieces a row's XOR reaches

    // what lane's 16 bytes of piece q are: element offset of the operand relative to (first row, first k), and its k inside the chunk
    __device__ static inline void place(int q, int lane, int& across_idx, int& k) {
        if constexpr (ACROSS) {
            const int byte = q * 1024 + lane * 16;
            k = byte / LINE;
            int col = byte % LINE;
            if constexpr (ES == 2) col = (((col >> 6) ^ (k & SWZ)) << 6) | (col & 63);
            across_idx = col / ES;
        } else {
            const int r = q * 16 + (lane >> 2);
            across_idx = r;
            k = ((lane & 3) ^ ((r >> 1) & 3)) * (16 / ES);
        }
    }
};

template <typename T, typename O, bool AX, bool BX, int BM, int BN, int WM, int WN, int NST>
__global__ __launch_bounds__(64 * WM * WN) void linear_tile_kernel(LinArgs p) {
    typedef typename T::raw raw;
    typedef LinSide<T, AX, BM> SA;
    typedef LinSide<T, BX, BN> SB;
    constexpr int ES = SA::ES, BK = SA::BK, WAVES = WM * WN;
    constexpr int STAGE = SA::BYTES + SB::BYTES;
    constexpr int PIECES = SA::PIECES + SB::PIECES, LOADS = (PIECES + WAVES - 1) / WAVES;
    constexpr int I = BM / WM / 32, J = BN / WN / 32;
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const unsigned lds0 = (unsigned)(uintptr_t)lds;

    const int tiles = p.tiles_i * p.tiles_j;
    const int id = lin_xcd_order(blockIdx.x, gridDim.x);
    const int split = id / tiles, tile = id - split * tiles;
    const long i0 = (long)(tile / p.tiles_j) * BM;
    const int j0 = (tile % p.tiles_j) * BN;
    const int kb = (int)min((long)p.K, (long)split * p.k_split), ke = (int)min((long)p.K, (long)kb + p.k_split);
    const int chunks = ke > kb ? (ke - kb + BK - 1) / BK : 0;

    // ---- loads: wave w moves pieces w, w + WAVES, ... (past the last one: the last one again, the same bytes to the same place)
    const char* baseA = (const char*)p.A + i0 * p.a_i * ES;
    const char* baseB = (const char*)p.B + (long)j0 * p.b_j * ES;
    unsigned off[LOADS];
    int kin[LOADS];
#pragma unroll
    for (int u = 0; u < LOADS; ++u) {
        const int q = min(wv + u * WAVES, PIECES - 1);
        int r, k;
        if (q < SA::PIECES) {
            SA::place(q, lane, r, k);
            // rows past the last: the last again (their results are dropped); ACROSS: the last whole 16 bytes
            r = (int)min((long)r, (AX ? (long)p.a_ext - 16 / ES : (long)p.M - 1) - i0);
            off[u] = (unsigned)((long)r * p.a_i + (long)k * p.a_k) * ES;
        } else {
            SB::place(q - SA::PIECES, lane, r, k);
            r = min(r, (BX ? p.b_ext - 16 / ES : p.N - 1) - j0);
            off[u] = (unsigned)((long)r * p.b_j + (long)k * p.b_k) * ES;
        }
        kin[u] = k;
    }
    auto issue = [&](int c) {
        const long k0 = kb + (long)c * BK;
        const char* a = baseA + k0 * p.a_k * ES;
        const char* b = baseB + k0 * p.b_k * ES;
        const unsigned stage = lds0 + (c % NST) * STAGE;
        if (k0 + BK <= p.K) {
#pragma unroll
            for (int u = 0; u < LOADS; ++u) {
                const int q = min(wv + u * WAVES, PIECES - 1);
                lin_copy(q < SA::PIECES ? a : b, off[u], stage + q * 1024);
            }
        } else {      // the last chunk: what lies past the contraction's end comes from a zero
#pragma unroll
            for (int u = 0; u < LOADS; ++u) {
                const int q = min(wv + u * WAVES, PIECES - 1);
                const char* src = (q < SA::PIECES ? a : b) + off[u];
                lin_copy_v(k0 + kin[u] < p.K ? src : (const char*)lin_zeros, stage + q * 1024);
            }
        }
    };

    // ---- fragments
    const int wi = (wv / WN) * (BM / WM), wj = (wv % WN) * (BN / WN);   // this wave's corner of the tile
    const int h = lane >> 5, l31 = lane & 31;
    lin_f32x16 acc[I][J];
#pragma unroll
    for (int i = 0; i < I; ++i)
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;

    // 16 bytes of the lane's row for slot `slot` of a side read along k
    auto along = [&](const char* side, int row, int slot) -> uint4 {
        return *(const uint4*)(side + row * LIN_CHUNK_BYTES + ((slot ^ ((row >> 1) & 3)) << 4));
    };
    const int tg = lane >> 4, tr = (lane >> 2) & 3, tc = lane & 3;
    // 8 consecutive k of column `first + lane % 32` (16-bit, a side read across), k-step s
    auto across16 = [&](const char* side, int line, int swz, int first, int s) -> uint4 {
        const int k = 16 * s + 8 * (tg >> 1) + tr;
        const char* at = side + k * line + ((((first >> 5) ^ (k & swz)) << 6)) + (16 * (tg & 1) + 4 * tc) * 2;
        const lin_s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) lin_s16x4*)(at));
        const lin_s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) lin_s16x4*)(at + 4 * line));
        const uint2 a = __builtin_bit_cast(uint2, lo), b = __builtin_bit_cast(uint2, hi);
        return make_uint4(a.x, a.y, b.x, b.y);
    };

    auto widen2 = [&](unsigned w, bool high) -> unsigned {      // two e4m3 as two bf16, exact
        return __builtin_bit_cast(unsigned, high ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, true)
                                                 : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, false));
    };
    auto multiply = [&](int c) {
        const char* sa = lds + (c % NST) * STAGE;
        const char* sb = sa + SA::BYTES;
        if constexpr (ES == 2) {
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                uint4 a[I], b[J];
#pragma unroll
                for (int i = 0; i < I; ++i) {
                    if constexpr (AX) a[i] = across16(sa, SA::LINE, SA::SWZ, wi + i * 32, s);
                    else a[i] = along(sa, wi + i * 32 + l31, 2 * s + h);
                }
#pragma unroll
                for (int j = 0; j < J; ++j) {
                    if constexpr (BX) b[j] = across16(sb, SB::LINE, SB::SWZ, wj + j * 32, s);
                    else b[j] = along(sb, wj + j * 32 + l31, 2 * s + h);
                }
#pragma unroll
                for (int i = 0; i < I; ++i)
#pragma unroll
                    for (int j = 0; j < J; ++j) {
                        if constexpr (T::code == SCENERF_T_BF16)
                            acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(lin_bf16x8, b[j]), __builtin_bit_cast(lin_bf16x8, a[i]),
                                                                                acc[i][j], 0, 0, 0);
                        else
                            acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(lin_f16x8, b[j]), __builtin_bit_cast(lin_f16x8, a[i]),
                                                                               acc[i][j], 0, 0, 0);
                    }
            }
        } else if constexpr (ES == 1 && O::code == SCENERF_T_F32) {
            // the 8-bit matrix instruction adds 8 neighbouring products to 2^-13 of the largest of them (measured: linear.hip): not enough
            // for a result in 32 bits.  e4m3 is exact in bf16: widened here, at half the rate
            uint4 a[I][4], b[J][4];
            auto widen = [&](const char* side, int row, uint4 (&f)[4]) {
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    const uint4 v = along(side, row, h + 2 * t);
                    f[2 * t] = make_uint4(widen2(v.x, false), widen2(v.x, true), widen2(v.y, false), widen2(v.y, true));
                    f[2 * t + 1] = make_uint4(widen2(v.z, false), widen2(v.z, true), widen2(v.w, false), widen2(v.w, true));
                }
            };
#pragma unroll
            for (int i = 0; i < I; ++i) widen(sa, wi + i * 32 + l31, a[i]);
#pragma unroll
            for (int j = 0; j < J; ++j) widen(sb, wj + j * 32 + l31, b[j]);
#pragma unroll
            for (int s = 0; s < 4; ++s)
#pragma unroll
                for (int i = 0; i < I; ++i)
#pragma unroll
                    for (int j = 0; j < J; ++j)
                        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(lin_bf16x8, b[j][s]), __builtin_bit_cast(lin_bf16x8, a[i][s]),
                                                                            acc[i][j], 0, 0, 0);
        } else if constexpr (ES == 1) {
            // 64 k in one instruction: the lane's half takes slots h and h + 2; every scale is 1 (127 as an exponent)
            lin_i32x8 a[I], b[J];
            auto two = [&](const char* side, int row) -> lin_i32x8 {
                const uint4 x = along(side, row, h), y = along(side, row, h + 2);
                return lin_i32x8{(int)x.x, (int)x.y, (int)x.z, (int)x.w, (int)y.x, (int)y.y, (int)y.z, (int)y.w};
            };
#pragma unroll
            for (int i = 0; i < I; ++i) a[i] = two(sa, wi + i * 32 + l31);
#pragma unroll
            for (int j = 0; j < J; ++j) b[j] = two(sb, wj + j * 32 + l31);
#pragma unroll
            for (int i = 0; i < I; ++i)
#pragma unroll
                for (int j = 0; j < J; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(b[j], a[i], acc[i][j], 0, 0, 0, 0x7f7f7f7f, 0, 0x7f7f7f7f);
        } else {
#pragma unroll
            for (int s = 0; s < 2; ++s) {           // the lane's half holds k = 8 s + 4 h + e
                float a[I][4], b[J][4];
#pragma unroll
                for (int i = 0; i < I; ++i) {
                    if constexpr (AX) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) a[i][e] = *(const float*)(sa + (8 * s + 4 * h + e) * SA::LINE + (wi + i * 32 + l31) * 4);
                    } else {
                        const uint4 v = along(sa, wi + i * 32 + l31, 2 * s + h);
                        a[i][0] = __uint_as_float(v.x); a[i][1] = __uint_as_float(v.y); a[i][2] = __uint_as_float(v.z); a[i][3] = __uint_as_float(v.w);
                    }
                }
#pragma unroll
                for (int j = 0; j < J; ++j) {
                    if constexpr (BX) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) b[j][e] = *(const float*)(sb + (8 * s + 4 * h + e) * SB::LINE + (wj + j * 32 + l31) * 4);
                    } else {
                        const uint4 v = along(sb, wj + j * 32 + l31, 2 * s + h);
                        b[j][0] = __uint_as_float(v.x); b[j][1] = __uint_as_float(v.y); b[j][2] = __uint_as_float(v.z); b[j][3] = __uint_as_float(v.w);
                    }
                }
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int i = 0; i < I; ++i)
#pragma unroll
                        for (int j = 0; j < J; ++j)
                            acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x2f32(b[j][e], a[i][e], acc[i][j], 0, 0, 0);
            }
        }
    };

#pragma unroll 1
    for (int c = 0; c < NST - 1 && c < chunks; ++c) issue(c);
#pragma unroll 1
    for (int c = 0; c < chunks; ++c) {
        // this wave's loads of chunk c have landed (at most those of the NST - 2 chunks behind it are outstanding), its reads of
        // chunk c - 1 are done: behind the barrier that holds for every wave, and the stage of chunk c - 1 may be overwritten
        if (c + NST - 2 < chunks) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((NST - 2) * LOADS) : "memory");
        else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (c + NST - 1 < chunks) issue(c + NST - 1);
        multiply(c);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();       // the ring is free: it becomes the waves' store slabs
    asm volatile("" ::: "memory");

    // ---- results: 32 rows of the wave at a time through a slab of [32][BN / WN] floats (rows 16 bytes apart in the banks)
    constexpr int WCOLS = BN / WN, PITCH = WCOLS + 4, W = 16 / (int)sizeof(typename O::raw), LANES_ROW = WCOLS / W, ROWS_PASS = 64 / LANES_ROW;
    static_assert(WAVES * 32 * PITCH * 4 <= NST * STAGE, "the slabs fit the ring");
    float* slab = (float*)lds + wv * 32 * PITCH;
#pragma unroll
    for (int i = 0; i < I; ++i) {
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                *(float4*)(slab + l31 * PITCH + j * 32 + 8 * e + 4 * h) =
                    make_float4(acc[i][j][4 * e], acc[i][j][4 * e + 1], acc[i][j][4 * e + 2], acc[i][j][4 * e + 3]);
        wave_sync();
        const long row0 = i0 + wi + i * 32;
        if (p.part) {
            float* part = p.part + (size_t)split * p.M * p.N;
            for (int r = 0; r < 32; ++r)
                for (int c = lane; c < WCOLS; c += 64)
                    if (row0 + r < p.M && j0 + wj + c < p.N) part[(size_t)(row0 + r) * p.N + j0 + wj + c] = slab[r * PITCH + c];
        } else if (p.vec) {
            const int c = (lane % LANES_ROW) * W, col = j0 + wj + c;
#pragma unroll
            for (int r = lane / LANES_ROW; r < 32; r += ROWS_PASS) {
                float v[W];
#pragma unroll
                for (int e = 0; e < W; e += 4) {
                    const float4 t = *(const float4*)(slab + r * PITCH + c + e);
                    v[e] = t.x; v[e + 1] = t.y; v[e + 2] = t.z; v[e + 3] = t.w;
                }
                if (row0 + r < p.M && col < p.N) epilogue_vec<O, W>(p, row0 + r, col, v);
            }
        } else {
            for (int r = 0; r < 32; ++r)
                for (int c = lane; c < WCOLS; c += 64)
                    if (row0 + r < p.M && j0 + wj + c < p.N) epilogue_one<O>(p, row0 + r, j0 + wj + c, slab[r * PITCH + c]);
        }
        wave_sync();
    }
}

template <typename T, typename O, bool AX, bool BX, int BM, int BN, int WM, int WN, int NST> static int lin_tile_launch(const LinArgs& a, hipStream_t s) {
    constexpr int LDS = NST * (BM + BN) * LIN_CHUNK_BYTES;
    auto kernel = linear_tile_kernel<T, O, AX, BX, BM, BN, WM, WN, NST>;
    SRF_ONCE_PER_DEVICE(SRF_HIP(hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, LDS)));
    const long blocks = (long)a.tiles_i * a.tiles_j * a.splits;
    SRF_CHECK(blocks <= ROWOPS_GRID_MAX, "linear: %ld tiles are more than one launch holds", blocks);
    kernel<<<(unsigned)blocks, 64 * WM * WN, LDS, s>>>(a);
    SRF_LAUNCH_CHECK("linear_tile_kernel");
    return 0;
}
template <typename T, typename O, bool AX, bool BX> static int lin_tile_pick(const LinArgs& a, LinTile tile, hipStream_t s) {
    switch (tile) {
        case LIN_256x256:
            if constexpr (T::code != SCENERF_T_F32) return lin_tile_launch<T, O, AX, BX, 256, 256, 2, 4, 4>(a, s);
            break;
        case LIN_256x128:
            if constexpr (T::code != SCENERF_T_F32) return lin_tile_launch<T, O, AX, BX, 256, 128, 4, 2, 4>(a, s);
            break;
        case LIN_128x128: return lin_tile_launch<T, O, AX, BX, 128, 128, 2, 2, 3>(a, s);
        case LIN_128x32: return lin_tile_launch<T, O, AX, BX, 128, 32, 4, 1, 4>(a, s);
        case LIN_32x128: return lin_tile_launch<T, O, AX, BX, 32, 128, 1, 4, 4>(a, s);
        default: break;
    }
    srf_set_error("linear: no such tile for this type");
    return 1;
}
template <typename T> static int lin_tile_layout(const LinArgs& a, LinTile tile, hipStream_t s) {
    const bool ax = a.a_k != 1, bx = a.b_k != 1;
    if (!ax && !bx) return lin_tile_pick<T, T, false, false>(a, tile, s);
    if (!ax && bx) return lin_tile_pick<T, T, false, true>(a, tile, s);
    if (ax && bx) return lin_tile_pick<T, T, true, true>(a, tile, s);
    srf_set_error("linear: no such operand layout");
    return 1;
}
