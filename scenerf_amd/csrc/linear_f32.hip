// The staged product (linear_tile.h) of f32 operands.
#include "linear_tile.h"

int linear_tile_f32(const LinArgs& a, LinTile tile, hipStream_t s) { return lin_tile_layout<TypeF32>(a, tile, s); }
int linear_pair_f32(const LinArgs& dx, const LinArgs& dw, LinTile tile, hipStream_t s) { return lin_pair<TypeF32>(dx, dw, tile, s); }
