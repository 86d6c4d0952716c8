// The staged product (linear_tile.h) of f16 operands.
#include "linear_tile.h"

int linear_tile_f16(const LinArgs& a, LinTile tile, hipStream_t s) { return lin_tile_layout<TypeF16>(a, tile, s); }
int linear_pair_f16(const LinArgs& dx, const LinArgs& dw, LinTile tile, hipStream_t s) { return lin_pair<TypeF16>(dx, dw, tile, s); }
