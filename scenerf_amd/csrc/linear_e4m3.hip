// The staged product (linear_tile.h) of e4m3 operands: forward only, results in fp32, bf16 or fp16.
#include "linear_tile.h"

int linear_tile_e4m3(const LinArgs& a, LinTile tile, int out_type, hipStream_t s) {
    if (out_type == SCENERF_T_F32) return lin_tile_pick<TypeE4M3, TypeF32, false, false>(a, tile, s);
    if (out_type == SCENERF_T_BF16) return lin_tile_pick<TypeE4M3, TypeBF16, false, false>(a, tile, s);
    return lin_tile_pick<TypeE4M3, TypeF16, false, false>(a, tile, s);
}
