// The kernels of linear_tiles.hip.h for operands of one type (TIRAMISU_OPERAND: F16, BF16 or F8; compiled once for each), and the choice among them by
// the tile, how the operands lie and the epilogue.
#include "operators.h"

#include <atomic>

#include "kernels/linear_tiles.hip.h"

namespace tops {
namespace {

// more LDS than a launch gets unasked: asked for once on every device
void allow_lds(const void *kernel, int bytes, std::atomic<unsigned long long> &asked) {
    int device = 0;
    tiramisu_runtime::check(hipGetDevice(&device), "tiramisu_hip_linear");
    const unsigned long long bit = 1ull << (device & 63);
    if (asked.load() & bit) return;
    tiramisu_runtime::check(hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes), "tiramisu_hip_linear");
    asked.fetch_or(bit);
}

template <class C>
int tiles_of(const product_arguments &p) {
    return ((p.M + C::BM - 1) / C::BM) * ((p.N + C::COLUMNS - 1) / C::COLUMNS);
}

template <class C, int Y>
void launch(const product_arguments &p, int splits, hipStream_t stream) {
    auto kernel = product_kernel<C, Y>;
    static std::atomic<unsigned long long> asked{0};
    allow_lds((const void *)kernel, C::LDS_BYTES, asked);
    hipLaunchKernelGGL(kernel, dim3((unsigned)tiles_of<C>(p), (unsigned)splits), dim3(C::NT), C::LDS_BYTES, stream, p);
    tiramisu_runtime::check(hipGetLastError(), "tiramisu_hip_linear");
}

template <class C, class D, int Y>
void launch_pair(const product_arguments &p, const product_arguments &q, const column_sums &sums, hipStream_t stream) {
    auto kernel = product_pair_kernel<C, D, Y>;
    constexpr int LDS = C::LDS_BYTES > D::LDS_BYTES ? C::LDS_BYTES : D::LDS_BYTES;
    static std::atomic<unsigned long long> asked{0};
    allow_lds((const void *)kernel, LDS, asked);
    const int tiles = tiles_of<C>(p), start = (tiles + XCDS - 1) / XCDS * XCDS, end = start + tiles_of<D>(q);
    const int of_sums = sums.parts ? (int)((sums.columns + SUM_COLUMNS - 1) / SUM_COLUMNS) : 0;
    hipLaunchKernelGGL(kernel, dim3((unsigned)(end + of_sums)), dim3(C::NT), LDS, stream, p, q, sums, tiles, start, end);
    tiramisu_runtime::check(hipGetLastError(), "tiramisu_hip_linear");
}

// Wavefronts, stages and matrix instructions of each tile.  Of those measured, the fastest for the launches that choose the tile; us for bf16 with 2 x 2
// wavefronts and 32 x 32 blocks / as here: 256 x 256 (4096^3) 117 / 102 (4 x 2: 133, registers spilled); 256 x 128 (4096^3) 123 / 115; 128 x 128 in
// one round (4096 x 1024 x 4096) 43 with two stages, 37.4 with four / 35.1; 64 x 64 (1024^3) 7.7 / 7.0;
// gated 64 x 128 (e4m3, 1000 x 1500 x 700) with 2 x 2 wavefronts 12.2, with 2 x 4 10.3.  8 bits: 256 x 256 (4096^3) 68 / 62, where 16 x 16 blocks
// do not leave registers for two sets of fragments (150); 256 x 128 74 / 67; 128 x 128 (4096 x 1024 x 4096) 26 / 23; 64 x 64 (512 x 2048 x 2048) 8.2 / 7.0.
template <int E, bool A_ROWS, bool B_ROWS, int EPILOGUE> struct tiles_for {
    typedef tile_config<E, 256, 256, 2, 4, 2, A_ROWS, B_ROWS, EPILOGUE, E == F8 ? 32 : 16> tile_256;
    typedef tile_config<E, 256, 128, 4, 2, 3, A_ROWS, B_ROWS, EPILOGUE, 16> tile_256x128;
    typedef tile_config<E, 128, 128, 4, 2, 4, A_ROWS, B_ROWS, EPILOGUE, 16> tile_128;
    typedef tile_config<E, 128, EPILOGUE == GATED ? 128 : 64, 4, 2, EPILOGUE == GATED ? 4 : 3, A_ROWS, B_ROWS, EPILOGUE, 16> tile_128x64;      // (gated: the one before)
    typedef tile_config<E, 64, EPILOGUE == GATED ? 128 : 64, 2, EPILOGUE == GATED ? 4 : 2, 3, A_ROWS, B_ROWS, EPILOGUE, 16> tile_64;
};
template <int E, int Y, bool A_ROWS, bool B_ROWS, int EPILOGUE>
void launch_tile(product_tile tile, const product_arguments &p, int splits, hipStream_t stream) {
    typedef tiles_for<E, A_ROWS, B_ROWS, EPILOGUE> T;
    if (tile == TILE_256) launch<typename T::tile_256, Y>(p, splits, stream);
    else if (tile == TILE_256x128) launch<typename T::tile_256x128, Y>(p, splits, stream);
    else if (tile == TILE_128) launch<typename T::tile_128, Y>(p, splits, stream);
    else if (tile == TILE_128x64) launch<typename T::tile_128x64, Y>(p, splits, stream);
    else launch<typename T::tile_64, Y>(p, splits, stream);
}

// (P, Q: how the operands of the two products lie)
template <int E, class P, class Q>
void launch_pair_of(product_tile tile, const product_arguments &p, const product_arguments &q, const column_sums &sums, hipStream_t stream) {
    if (tile == TILE_256) launch_pair<typename P::tile_256, typename Q::tile_256, E>(p, q, sums, stream);
    else if (tile == TILE_256x128) launch_pair<typename P::tile_256x128, typename Q::tile_256x128, E>(p, q, sums, stream);
    else if (tile == TILE_128) launch_pair<typename P::tile_128, typename Q::tile_128, E>(p, q, sums, stream);
    else if (tile == TILE_128x64) launch_pair<typename P::tile_128x64, typename Q::tile_128x64, E>(p, q, sums, stream);
    else launch_pair<typename P::tile_64, typename Q::tile_64, E>(p, q, sums, stream);
}

}  // namespace

#define JOIN_NAMES(name, element) name##element
#define NAME_OF(name, element) JOIN_NAMES(name, element)
void NAME_OF(launch_tiles_, TIRAMISU_OPERAND)(product_tile tile, product_layout layout, int epilogue, int y, const product_arguments &p, int splits, hipStream_t stream) {
    constexpr int E = TIRAMISU_OPERAND;
    if constexpr (E == F8) {                // with k along the rows, to either 16-bit type
        if (epilogue == GATED) y == BF16 ? launch_tile<E, BF16, true, true, GATED>(tile, p, splits, stream) : launch_tile<E, F16, true, true, GATED>(tile, p, splits, stream);
        else y == BF16 ? launch_tile<E, BF16, true, true, LINEAR>(tile, p, splits, stream) : launch_tile<E, F16, true, true, LINEAR>(tile, p, splits, stream);
    } else if (epilogue == GATED) launch_tile<E, E, true, true, GATED>(tile, p, splits, stream);
    else if (layout == FORWARD) launch_tile<E, E, true, true, LINEAR>(tile, p, splits, stream);
    else if (layout == INPUT_GRADIENT) launch_tile<E, E, true, false, LINEAR>(tile, p, splits, stream);
    else launch_tile<E, E, false, false, LINEAR>(tile, p, splits, stream);
}

#ifndef TIRAMISU_OPERAND_HAS_NO_GRADIENTS
void NAME_OF(launch_gradients_, TIRAMISU_OPERAND)(product_tile tile, bool q_first, const product_arguments &p, const product_arguments &q, const column_sums &sums, hipStream_t stream) {
    constexpr int E = TIRAMISU_OPERAND;
    typedef tiles_for<E, true, false, LINEAR> of_input;
    typedef tiles_for<E, false, false, LINEAR> of_weights;
    if (q_first) launch_pair_of<E, of_weights, of_input>(tile, q, p, sums, stream);
    else launch_pair_of<E, of_input, of_weights>(tile, p, q, sums, stream);
}
#endif

}  // namespace tops
