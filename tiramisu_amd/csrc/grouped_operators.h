// What expert_operators.hip (the entry points) and grouped_tiles.hip (the kernels on tiles, compiled once for each operand type) share.
#ifndef TIRAMISU_AMD_GROUPED_OPERATORS_H
#define TIRAMISU_AMD_GROUPED_OPERATORS_H
#include "operators.h"

#include "kernels/grouped_products.hip.h"

namespace tgroups {

// Tiles of `height` rows that the rows of so many groups, and those ahead of them and behind them, can need at most
inline long most_row_tiles(long rows, long groups, long height, long others = 2) { return rows / height + (groups + others < rows ? groups + others : rows); }

// Forward; y: element type of the results
void launch_grouped_F16(product_tile, int epilogue, int y, const grouped_arguments &, hipStream_t stream);
void launch_grouped_BF16(product_tile, int epilogue, int y, const grouped_arguments &, hipStream_t stream);
void launch_grouped_F8(product_tile, int epilogue, int y, const grouped_arguments &, hipStream_t stream);
// The gradients of the rows and of the weights on the same tiles, in one launch; one without a place for its result (p.y) is not computed
void launch_grouped_gradients_F16(product_tile, const grouped_arguments &rows, const grouped_arguments &weights, hipStream_t stream);
void launch_grouped_gradients_BF16(product_tile, const grouped_arguments &rows, const grouped_arguments &weights, hipStream_t stream);

}  // namespace tgroups
#endif
