// The staged matrix product of linear.hip: operands from HBM straight into LDS, matrix instructions fed from there, the layer's epilogue
// behind the sums.  Included by one translation unit per operand type.
//
// A workgroup owns BM x BN results and walks the contraction in chunks of 128 bytes per row (a line: with 64-byte chunks every line was
// asked for twice, 1.35 against 1.27 ms for 153,600 x 2,480 x 1,536 bf16).  Chunks live in two rings, NSA stages of A's and NSB of B's, filled by
// asynchronous global -> LDS loads (16 bytes a lane, 1 KiB a wave and instruction) that run a ring's length ahead: one barrier a chunk, in
// front of which each wave waits for its own loads of the next chunk by count.
//
// LDS image of an operand read ALONG the contraction: row r is 128 bytes, its 16-byte slots XORed with (r >> 1) & 7, so that the 16 lanes
// of a ds_read_b128 phase cover all 64 banks.  The swizzle is applied on the source side of the load (LDS-bound loads place lanes in
// sequence).  An operand read ACROSS (contraction along the rows in memory) keeps its rows: [k][tile columns]; 16-bit fragments come
// out of it by the transposing read ds_read_b64_tr_b16 (within 16 lanes, lane 4r + c gives the address of 4 columns of row r, lane i
// receives rows 0..3 of column i), its 64-byte pieces XORed with k & 3; fp32 fragments are single elements anyway.
// Any order of k inside a chunk is valid as long as both operands use the same.
//
// A chunk is multiplied in 4 (8 bits: 2) parts; while the matrix instructions of one run from registers, the next is read from LDS.
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

template <bool V> struct Bool { static constexpr bool value = V; };

// 64 lanes x 16 bytes, global -> LDS at lds_base + lane * 16.  (m0 is the base.  Nothing else in these kernels reads it; saving and
// restoring it around every load cost 5 to 10 percent of a call.)
__device__ static inline void lin_copy(const void* src, unsigned lds_base) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src), "s"(lds_base) : "memory", "m0");
}

// the same from a base all lanes share and an offset of each: no vector instruction but the load itself
__device__ static inline void lin_copy_from(const void* base, unsigned offset, unsigned lds_base) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(offset), "s"(base), "s"(lds_base) : "memory", "m0");
}

// contiguous ranges of work per XCD (blocks go round-robin over the 8 XCDs, each with its own L2); any count
__device__ static inline int lin_xcd_order(int id, int total) {
    const int q = total >> 3, r = total & 7, xcd = id & 7, slot = id >> 3;
    return (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + slot;
}

// one operand's side of a stage: TILE rows (or columns) x one chunk of the contraction
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
            const int r = q * 8 + (lane >> 3);
            across_idx = r;
            k = ((lane & 7) ^ ((r >> 1) & 7)) * (16 / ES);
        }
    }
};

// workgroup `block` of `blocks` of one product
template <typename T, typename O, bool AX, bool BX, int BM, int BN, int WM, int WN, int NSA, int NSB, bool WHOLE>
__device__ static inline void linear_tile(const LinArgs& p, int block, int blocks) {
    typedef LinSide<T, AX, BM> SA;
    typedef LinSide<T, BX, BN> SB;
    constexpr int ES = SA::ES, BK = SA::BK, WAVES = WM * WN;
    constexpr int LA = SA::PIECES / WAVES, LB = SB::PIECES / WAVES;     // loads per wave and chunk
    static_assert(NSA >= 2 && (NSB == NSA || NSB == NSA - 1) && NSB >= 2, "the order of the loads and their counts");
    constexpr int I = BM / WM / 32, J = BN / WN / 32;
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const unsigned lds0 = (unsigned)(uintptr_t)lds;

    const int tiles = p.tiles_i * p.tiles_j;
    const int id = lin_xcd_order(block, blocks);
    const int split = id / tiles, tile = id - split * tiles;
    const long i0 = (long)(tile / p.tiles_j) * BM;
    const int j0 = (tile % p.tiles_j) * BN;
    const int kb = (int)min((long)p.K, (long)split * p.k_split), ke = (int)min((long)p.K, (long)kb + p.k_split);
    const int chunks = ke > kb ? (ke - kb + BK - 1) / BK : 0;

    // ---- loads: of each side wave w moves pieces w, w + WAVES, ...  A's ring has NSA stages, B's behind it NSB.
    const char* baseA = (const char*)p.A + i0 * p.a_i * ES;
    const char* baseB = (const char*)p.B + (long)j0 * p.b_j * ES;
    const unsigned ringB = lds0 + NSA * SA::BYTES;
    // (the k of a wave's loads inside a chunk: the same for all of a side read along, equal steps apart for one read across)
    constexpr int KA = AX ? WAVES * 1024 / SA::LINE : 0, KB = BX ? WAVES * 1024 / SB::LINE : 0;
    static_assert((AX || WAVES % 2 == 0) && (BX || WAVES % 2 == 0) && (!AX || WAVES * 1024 % SA::LINE == 0) && (!BX || WAVES * 1024 % SB::LINE == 0) &&
                  (AX ? KA % 4 == 0 : true) && (BX ? KB % 4 == 0 : true) && SA::PIECES % WAVES == 0 && SB::PIECES % WAVES == 0, "the steps of the loads");
    unsigned offA[AX ? 1 : LA], offB[BX ? 1 : LB];
    int kinA, kinB;
#pragma unroll
    for (int u = 0; u < (AX ? 1 : LA); ++u) {
        int r;
        SA::place(wv + u * WAVES, lane, r, kinA);
        // rows past the last: the last again (their results are dropped); ACROSS: the last whole 16 bytes
        r = (int)min((long)r, (AX ? (long)p.a_ext - 16 / ES : (long)p.M - 1) - i0);
        offA[u] = (unsigned)((long)r * p.a_i + (long)kinA * p.a_k) * ES;
    }
#pragma unroll
    for (int u = 0; u < (BX ? 1 : LB); ++u) {
        int r;
        SB::place(wv + u * WAVES, lane, r, kinB);
        r = min(r, (BX ? p.b_ext - 16 / ES : p.N - 1) - j0);
        offB[u] = (unsigned)((long)r * p.b_j + (long)kinB * p.b_k) * ES;
    }
    // load u of chunk c of a side.  What lies past the end of the split comes from a zero, and so do chunks past the last (nobody reads
    // them): every turn of the loop issues the same loads, without a branch.
    // (inside: the chunk is known to end before the split does)
    auto loadA = [&](int c, int u, auto inside) {
        const long k0 = kb + (long)c * BK;
        if constexpr (decltype(inside)::value) {
            lin_copy_from(baseA + (k0 + u * KA) * p.a_k * ES, offA[AX ? 0 : u], lds0 + (c % NSA) * SA::BYTES + (wv + u * WAVES) * 1024);
        } else {
            const char* src = baseA + (k0 + u * KA) * p.a_k * ES + offA[AX ? 0 : u];
            lin_copy(kinA < ke - k0 - u * KA ? src : (const char*)lin_zeros, lds0 + (c % NSA) * SA::BYTES + (wv + u * WAVES) * 1024);
        }
    };
    auto loadB = [&](int c, int u, auto inside) {
        const long k0 = kb + (long)c * BK;
        if constexpr (decltype(inside)::value) {
            lin_copy_from(baseB + (k0 + u * KB) * p.b_k * ES, offB[BX ? 0 : u], ringB + (c % NSB) * SB::BYTES + (wv + u * WAVES) * 1024);
        } else {
            const char* src = baseB + (k0 + u * KB) * p.b_k * ES + offB[BX ? 0 : u];
            lin_copy(kinB < ke - k0 - u * KB ? src : (const char*)lin_zeros, ringB + (c % NSB) * SB::BYTES + (wv + u * WAVES) * 1024);
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
        return *(const uint4*)(side + row * LIN_CHUNK_BYTES + ((slot ^ ((row >> 1) & 7)) << 4));
    };
    const int tg = lane >> 4, tr = (lane >> 2) & 3, tc = lane & 3;
    // 8 consecutive k of column `first + lane % 32` (16-bit, a side read across), from 16 s on
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
    // a chunk's contraction in PARTS, each one fragment of FR registers a lane per 32 rows: 16 (16-bit), 64 (8-bit), 8 (fp32) of it
    constexpr bool WIDEN = ES == 1 && O::code != SCENERF_T_BF16;
    constexpr int PARTS = ES == 1 ? 2 : 4, FR = ES == 1 ? 8 : 4;
    struct Frag { unsigned a[I][FR], b[J][FR]; };
    // item t of the READS that fetch a part: 16 bytes of the lane's for 32 rows of one side
    constexpr int READS = FR / 4 * (I + J);
    auto fetch = [&](int c, int part, Frag& f, int t) {
        const int s = t % (FR / 4), n = t / (FR / 4);
        auto side = [&](auto across, const char* base, int first, int line, int swz, unsigned (&o)[FR]) {
            if constexpr (decltype(across)::value && ES == 4) {
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] = *(const unsigned*)(base + (8 * part + 4 * h + e) * line + (first + l31) * 4);
            } else {
                uint4 v;
                if constexpr (decltype(across)::value) v = across16(base, line, swz, first, part);
                else v = along(base, first + l31, (FR / 2) * part + 2 * s + h);    // 8-bit: the lane's half takes 16-byte slots h and h + 2
                o[4 * s] = v.x; o[4 * s + 1] = v.y; o[4 * s + 2] = v.z; o[4 * s + 3] = v.w;
            }
        };
        if (n < J) side(Bool<BX>(), lds + NSA * SA::BYTES + (c % NSB) * SB::BYTES, wj + n * 32, SB::LINE, SB::SWZ, f.b[n < J ? n : 0]);
        else side(Bool<AX>(), lds + (c % NSA) * SA::BYTES, wi + (n - J) * 32, SA::LINE, SA::SWZ, f.a[n < J ? 0 : n - J]);
    };
    auto four = [](const unsigned (&r)[FR], int s) { return make_uint4(r[4 * s], r[4 * s + 1], r[4 * s + 2], r[4 * s + 3]); };
    // group g of the STEPS * I groups of J matrix instructions that multiply a part
    constexpr int STEPS = ES == 4 || WIDEN ? 4 : 1, GROUPS = STEPS * I;
    constexpr int EARLY = GROUPS >= 4 ? GROUPS * 3 / 4 : 1;     // the groups that the next part's reads go between
    auto multiply = [&](const Frag& f, int g) {
        const int s = g / I, i = g % I;
        auto eight = [](const unsigned (&r)[FR]) {
            return lin_i32x8{(int)r[0], (int)r[1], (int)r[2], (int)r[3], (int)r[4], (int)r[5], (int)r[6], (int)r[7]};
        };
        // 8-bit operands of a result in fp32 or fp16: the 8-bit matrix instruction adds 8 neighbouring products to 2^-13 of the largest of them
        // (measured: linear.hip), which is more than those types' own rounding (2^-24, 2^-11) where a group's 7 others lose it each.  e4m3 is exact
        // in bf16: widened here, at half the rate.  A result in bf16, whose rounding is 2^-8 of it, takes the 8-bit instruction: what it
        // leaves out shows where sums cancel to less than about 2^-3 of their terms' magnitudes
        auto wide = [&](const unsigned (&r)[FR]) {
            return __builtin_bit_cast(lin_bf16x8, make_uint4(widen2(r[2 * s], false), widen2(r[2 * s], true), widen2(r[2 * s + 1], false),
                                                             widen2(r[2 * s + 1], true)));
        };
#pragma unroll
        for (int j = 0; j < J; ++j) {
            if constexpr (T::code == SCENERF_T_BF16)
                acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(lin_bf16x8, four(f.b[j], s)),
                                                                    __builtin_bit_cast(lin_bf16x8, four(f.a[i], s)), acc[i][j], 0, 0, 0);
            else if constexpr (T::code == SCENERF_T_F16)
                acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(lin_f16x8, four(f.b[j], s)),
                                                                   __builtin_bit_cast(lin_f16x8, four(f.a[i], s)), acc[i][j], 0, 0, 0);
            else if constexpr (WIDEN)
                acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(wide(f.b[j]), wide(f.a[i]), acc[i][j], 0, 0, 0);
            else if constexpr (ES == 1)         // 64 k in one instruction; every scale is 1 (127 as an exponent)
                acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(eight(f.b[j]), eight(f.a[i]), acc[i][j], 0, 0, 0, 0x7f7f7f7f, 0, 0x7f7f7f7f);
            else                                // the lane's half holds k = 4 h + s
                acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(f.b[j][s]), __uint_as_float(f.a[i][s]), acc[i][j], 0, 0, 0);
        }
    };

    // ---- the loop.  A part is multiplied from registers while the next one is read from LDS and loads of further chunks are issued, a few of
    // each between the groups of matrix instructions: in a burst, the loads kept both waves of a SIMD from their products.  What the next part
    // needs first, B's fragments and A's first, is read first, and nothing in the last quarter: 1 to 2 percent.  (Four waves of 128 x 128, a
    // third less to read, in the whole accumulator file: 1,037 against 880 us at 8,192^3, results twice as slow.)
    // Loads run in the order A(0) B(0) .. , B(c + NSB) behind the barrier in front of chunk c's last part, A(c + NSA) behind the chunk.
    auto turn = [&](const Frag& now, int c, int part, Frag& next, auto load, int first, int last) {
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) {
#pragma unroll
            for (int t = min(g, EARLY) * READS / EARLY; t < min(g + 1, EARLY) * READS / EARLY; ++t) fetch(c, part, next, t);
#pragma unroll
            for (int u = first + g * (last - first) / GROUPS; u < first + (g + 1) * (last - first) / GROUPS; ++u) load(u);
            multiply(now, g);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    // Chunks whose loads end inside the split go through a loop of their own, without the loads' comparisons, selections and 64-bit sums
    // (1.7 vector instructions a matrix instruction else; before and behind it on one box): 153,600 x 2,480 x 1,536 bf16 1,165 -> 1,140 us and its dx 1,111 -> 1,075, 8 bits 677 ->
    // 669, 4,800 x 512 x 512 fp32 with its gradients 71 -> 67.  Small tiles of 16 and 8 bits have few chunks and lose by the longer code (29.8 -> 30.4).
    constexpr bool FAST = ES == 4 || BM * BN >= 128 * 128;
    constexpr bool TWICE = ES == 2 && BX && BM * BN < 256 * 256;       // (LinArgs.A2; the large tiles have no registers for it)
    Frag f0, f1;
    bool again = TWICE && p.A2;
#pragma unroll 1
    while (chunks > 0) {
#pragma unroll
        for (int c = 0; c < NSA; ++c) {
#pragma unroll
            for (int u = 0; u < LA; ++u)
                if (c < NSA - 1) loadA(c, u, Bool<false>());
#pragma unroll
            for (int u = 0; u < LB; ++u)
                if (c < NSB) loadB(c, u, Bool<false>());
        }
        // chunk 0 has landed: what was issued behind it may be outstanding
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"((NSA - 2) * LA + (NSB - 1) * LB) : "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
#pragma unroll
        for (int t = 0; t < READS; ++t) fetch(0, 0, f0, t);
        auto chunk = [&](int c, auto inside) {
#pragma unroll
            for (int part = 0; part < PARTS - 1; ++part)
                turn(part % 2 ? f1 : f0, c, part + 1, part % 2 ? f0 : f1, [&](int u) { loadA(c + NSA - 1, u, inside); }, part * LA / (PARTS - 1),
                     (part + 1) * LA / (PARTS - 1));
            // this wave's loads of chunk c + 1 have landed, its reads of chunk c are done; behind the barrier that holds for every wave:
            // the stages of chunk c are free
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((NSA - 2) * LA + (NSB - 2) * LB) : "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            turn(f1, c + 1, 0, f0, [&](int u) { loadB(c + NSB, u, inside); }, 0, LB);
        };
        // as long as what is loaded is inside the split, and the last few
        int c = 0;
        if constexpr (FAST) {
            const int last = (ke - kb) / BK - (NSB > NSA - 1 ? NSB : NSA - 1);
#pragma unroll 1
            for (; c < last; ++c) chunk(c, Bool<true>());
        }
#pragma unroll 1
        for (; c < chunks; ++c) chunk(c, Bool<false>());
        if (!TWICE || !again) break;
        if constexpr (TWICE) {
            again = false;
            baseA = (const char*)p.A2 + i0 * p.a_i * ES;
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();           // the rings are free again
            asm volatile("" ::: "memory");
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();       // the ring is free: it becomes the waves' store slabs
    asm volatile("" ::: "memory");

    // ---- results: 32 rows of the wave at a time through a slab of [32][BN / WN] floats (rows 16 bytes apart in the banks)
    constexpr int WCOLS = BN / WN, PITCH = WCOLS + 4, W = 16 / (int)sizeof(typename O::raw), LANES_ROW = WCOLS / W, ROWS_PASS = 64 / LANES_ROW;
    static_assert(WAVES * 32 * PITCH * 4 <= NSA * SA::BYTES + NSB * SB::BYTES, "the slabs fit the rings");
    float* slab = (float*)lds + wv * 32 * PITCH;
    // (a lane's columns are the same in every row: their bias and scales are read once; the residual of the next 32 rows is under way
    // while these leave, which a load per row and its wait cost 8 us a tile)
    constexpr int PASSES = 32 / ROWS_PASS;
    const int c = (lane % LANES_ROW) * W, col = j0 + wj + c, lrow = lane / LANES_ROW;
    const int in = p.N - col;
    // (WHOLE: no lane's piece reaches over the row's end)
    {
        EpilogueCols<O, W, WHOLE> ec;
        uint4 res[PASSES];
        auto residual = [&](int i) {
#pragma unroll
            for (int t = 0; t < PASSES; ++t) {
                const long row = i0 + wi + i * 32 + lrow + t * ROWS_PASS;
                if (row < p.M) res[t] = residual_piece<O, W, WHOLE>(p, row, col, in);
            }
        };
        if (!p.part && in > 0) {
            ec.load(p, col, in);
            if (p.residual) residual(0);
        }
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
#pragma unroll 4
                for (int r = 0; r < 32; ++r)
                    for (int k = lane; k < WCOLS; k += 64)
                        if (row0 + r < p.M && j0 + wj + k < p.N) part[(size_t)(row0 + r) * p.N + j0 + wj + k] = slab[r * PITCH + k];
            } else if (in > 0) {
                uint4 now[PASSES];
#pragma unroll
                for (int t = 0; t < PASSES; ++t) now[t] = res[t];
                if (p.residual && i + 1 < I) residual(i + 1);
#pragma unroll
                for (int t = 0; t < PASSES; ++t) {
                    const int r = lrow + t * ROWS_PASS;
                    float v[W];
#pragma unroll
                    for (int e = 0; e < W; e += 4) {
                        const float4 q = *(const float4*)(slab + r * PITCH + c + e);
                        v[e] = q.x; v[e + 1] = q.y; v[e + 2] = q.z; v[e + 3] = q.w;
                    }
                    if (row0 + r < p.M) epilogue_vec<O, W, WHOLE>(p, ec, row0 + r, col, in, now[t], v);
                }
            }
            wave_sync();
        }
    }
}

template <typename T, typename O, bool AX, bool BX, int BM, int BN, int WM, int WN, int NSA, int NSB, bool WHOLE>
__global__ __launch_bounds__(64 * WM * WN) void linear_tile_kernel(LinArgs p) {
    linear_tile<T, O, AX, BX, BM, BN, WM, WN, NSA, NSB, WHOLE>(p, blockIdx.x, gridDim.x);
}
// dx and dw of a layer in one launch: workgroups before `first` make dw, whose contraction is the longer one
template <typename T, int BM, int BN, int WM, int WN, int NSA, int NSB, bool WHOLE>
__global__ __launch_bounds__(64 * WM * WN) void linear_pair_kernel(LinArgs dx, LinArgs dw, int first) {
    if ((int)blockIdx.x < first) linear_tile<T, T, true, true, BM, BN, WM, WN, NSA, NSB, WHOLE>(dw, blockIdx.x, first);
    else linear_tile<T, T, false, true, BM, BN, WM, WN, NSA, NSB, WHOLE>(dx, blockIdx.x - first, gridDim.x - first);
}

template <typename T, typename O, bool AX, bool BX, int BM, int BN, int WM, int WN, int NSA, int NSB, bool WHOLE>
static int lin_tile_start(const LinArgs& a, hipStream_t s) {
    constexpr int LDS = (NSA * BM + NSB * BN) * LIN_CHUNK_BYTES;
    auto kernel = linear_tile_kernel<T, O, AX, BX, BM, BN, WM, WN, NSA, NSB, WHOLE>;
    SRF_ONCE_PER_DEVICE(SRF_HIP(hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, LDS)));
    const long blocks = (long)a.tiles_i * a.tiles_j * a.splits;
    SRF_CHECK(blocks < (1L << 32) / (64 * WM * WN), "linear: %ld tiles are more than one launch holds", blocks);
    kernel<<<(unsigned)blocks, 64 * WM * WN, LDS, s>>>(a);
    SRF_LAUNCH_CHECK("linear_tile_kernel");
    return 0;
}
template <typename T, typename O, bool AX, bool BX, int BM, int BN, int WM, int WN, int NSA, int NSB> static int lin_tile_launch(const LinArgs& a, hipStream_t s) {
    if (a.N % (16 / (int)sizeof(typename O::raw)) == 0) return lin_tile_start<T, O, AX, BX, BM, BN, WM, WN, NSA, NSB, true>(a, s);
    return lin_tile_start<T, O, AX, BX, BM, BN, WM, WN, NSA, NSB, false>(a, s);
}
template <typename T, typename O, bool AX, bool BX> static int lin_tile_pick(const LinArgs& a, LinTile tile, hipStream_t s) {
    switch (tile) {
        case LIN_256x256:
            if constexpr (T::code != SCENERF_T_F32) return lin_tile_launch<T, O, AX, BX, 256, 256, 2, 4, 3, 2>(a, s);
            break;
        case LIN_128x128: return lin_tile_launch<T, O, AX, BX, 128, 128, 2, 2, 3, 2>(a, s);
        case LIN_64x64: return lin_tile_launch<T, O, AX, BX, 64, 64, 2, 2, 3, 3>(a, s);
        case LIN_128x32: return lin_tile_launch<T, O, AX, BX, 128, 32, 4, 1, 3, 3>(a, s);
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
template <typename T, int BM, int BN, int WM, int WN, int NSA, int NSB, bool WHOLE> static int lin_pair_start(const LinArgs& dx, const LinArgs& dw, hipStream_t s) {
    constexpr int LDS = (NSA * BM + NSB * BN) * LIN_CHUNK_BYTES;
    auto kernel = linear_pair_kernel<T, BM, BN, WM, WN, NSA, NSB, WHOLE>;
    SRF_ONCE_PER_DEVICE(SRF_HIP(hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, LDS)));
    const long first = (long)dw.tiles_i * dw.tiles_j * dw.splits, blocks = first + (long)dx.tiles_i * dx.tiles_j * dx.splits;
    SRF_CHECK(blocks < (1L << 32) / (64 * WM * WN), "linear: %ld tiles are more than one launch holds", blocks);
    kernel<<<(unsigned)blocks, 64 * WM * WN, LDS, s>>>(dx, dw, (int)first);
    SRF_LAUNCH_CHECK("linear_pair_kernel");
    return 0;
}
template <typename T, int BM, int BN, int WM, int WN, int NSA, int NSB> static int lin_pair_launch(const LinArgs& dx, const LinArgs& dw, hipStream_t s) {
    // (both have k columns)
    if (dx.N % (16 / (int)sizeof(typename T::raw)) == 0) return lin_pair_start<T, BM, BN, WM, WN, NSA, NSB, true>(dx, dw, s);
    return lin_pair_start<T, BM, BN, WM, WN, NSA, NSB, false>(dx, dw, s);
}
template <typename T> static int lin_pair(const LinArgs& dx, const LinArgs& dw, LinTile tile, hipStream_t s) {
    switch (tile) {
        case LIN_128x128: return lin_pair_launch<T, 128, 128, 2, 2, 3, 2>(dx, dw, s);
        case LIN_64x64: return lin_pair_launch<T, 64, 64, 2, 2, 3, 3>(dx, dw, s);
        case LIN_128x32: return lin_pair_launch<T, 128, 32, 4, 1, 3, 3>(dx, dw, s);
        default: break;
    }
    srf_set_error("linear: no such tile for this type");
    return 1;
}
