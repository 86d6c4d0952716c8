// The staged product (linear_tile.h) of bf16 operands.
#include "linear_tile.h"

int linear_tile_bf16(const LinArgs& a, LinTile tile, hipStream_t s) { return lin_tile_layout<TypeBF16>(a, tile, s); }
int linear_pair_bf16(const LinArgs& dx, const LinArgs& dw, LinTile tile, hipStream_t s) { return lin_pair<TypeBF16>(dx, dw, tile, s); }
