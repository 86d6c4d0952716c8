// The staged product (linear_tile.h) of f32 operands.
#include "linear_tile.h"

int linear_tile_f32(const LinArgs& a, LinTile tile, hipStream_t s) { return lin_tile_layout<TypeF32>(a, tile, s); }
