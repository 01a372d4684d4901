// What operators.hip (the entry points), linear_tiles.hip (the matrix products' kernels, compiled once for each operand type) and
// hip_wrappers.hip (the runtime's state) share.
#ifndef TIRAMISU_AMD_OPERATORS_H
#define TIRAMISU_AMD_OPERATORS_H
#include <hip/hip_runtime.h>

#include <cstdint>

namespace tops {

struct product_arguments;
struct column_sums;

// How a product's operands lie: k along the rows of both (forward), of A alone (gradient of the input), of neither (gradient of the weights).
enum product_layout { FORWARD, INPUT_GRADIENT, WEIGHT_GRADIENT };

// The tiles, by rows and columns of the product (a gated layer's columns count twice).
enum product_tile { TILE_256, TILE_256x128, TILE_128, TILE_128x64, TILE_64 };

// Launches on `stream`; splits > 1: partial sums to arguments.partial, without the epilogue.  y: element type of the outputs.
void launch_tiles_F16(product_tile, product_layout, int epilogue, int y, const product_arguments &, int splits, hipStream_t stream);
void launch_tiles_BF16(product_tile, product_layout, int epilogue, int y, const product_arguments &, int splits, hipStream_t stream);
void launch_tiles_F8(product_tile, product_layout, int epilogue, int y, const product_arguments &, int splits, hipStream_t stream);

// The gradient of the input (p) and of the weights (q) in one launch, on the same tiles; `q_first`: the longer one begins; and behind them `sums`.
void launch_gradients_F16(product_tile, bool q_first, const product_arguments &p, const product_arguments &q, const column_sums &sums,
                          hipStream_t stream);
void launch_gradients_BF16(product_tile, bool q_first, const product_arguments &p, const product_arguments &q, const column_sums &sums,
                          hipStream_t stream);

}  // namespace tops

namespace tiramisu_runtime {

// The calling thread's stream, the failure model of the runtime, and a record of what lies between construction and destruction for
// tiramisu_hip_profile_start / _stop.
hipStream_t stream();
void check(hipError_t e, const char *function);
class timed {
public:
    explicit timed(const char *name);
    ~timed();
private:
    hipEvent_t stop;
};
// Scratch of one operator call on the thread's stream, at least `bytes` large; null where the memory cannot be had.  It comes from the thread's source where
// it has one (tiramisu_hip_exchange_scratch_source).  Else the next call there gets the same block or a larger one, in the stream's order; a block that
// a call was given while its stream recorded a graph stays where it is.
void *operator_scratch(uint64_t bytes);

}  // namespace tiramisu_runtime
#endif
