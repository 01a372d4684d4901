// The kernels of linear_tiles.hip.h for operands of one type (TIRAMISU_OPERAND: F16, BF16 or F8; compiled once for each), and the choice among them by
// the edge of the tile, how the operands lie and the epilogue.
#include "operators.h"

#include <atomic>

#include "kernels/linear_tiles.hip.h"

namespace tops {
namespace {

template <class C, int Y>
void launch(const product_arguments &p, int splits, hipStream_t stream) {
    auto kernel = product_kernel<C, Y>;
    // more LDS than a launch gets unasked: asked for once on every device
    static std::atomic<unsigned long long> asked{0};
    int device = 0;
    tiramisu_runtime::check(hipGetDevice(&device), "tiramisu_hip_linear");
    const unsigned long long bit = 1ull << (device & 63);
    if (!(asked.load() & bit)) {
        tiramisu_runtime::check(hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, C::LDS_BYTES), "tiramisu_hip_linear");
        asked.fetch_or(bit);
    }
    const unsigned tiles = (unsigned)(((p.M + C::BM - 1) / C::BM) * ((p.N + C::COLUMNS - 1) / C::COLUMNS));
    hipLaunchKernelGGL(kernel, dim3(tiles, (unsigned)splits), dim3(C::NT), C::LDS_BYTES, stream, p);
    tiramisu_runtime::check(hipGetLastError(), "tiramisu_hip_linear");
}

template <int E, int Y, bool A_ROWS, bool B_ROWS>
void launch_linear(int edge, const product_arguments &p, int splits, hipStream_t stream) {
    if (edge == 256) launch<tile_config<E, 256, 256, 4, 2, 2, A_ROWS, B_ROWS, LINEAR>, Y>(p, splits, stream);
    else if (edge == 128) launch<tile_config<E, 128, 128, 2, 2, 2, A_ROWS, B_ROWS, LINEAR>, Y>(p, splits, stream);
    else launch<tile_config<E, 64, 64, 2, 2, 3, A_ROWS, B_ROWS, LINEAR>, Y>(p, splits, stream);
}

template <int E, int Y>
void launch_gated(int edge, const product_arguments &p, int splits, hipStream_t stream) {
    if (edge == 256) launch<tile_config<E, 256, 256, 4, 2, 2, true, true, GATED>, Y>(p, splits, stream);
    else if (edge == 128) launch<tile_config<E, 128, 128, 2, 2, 2, true, true, GATED>, Y>(p, splits, stream);
    else launch<tile_config<E, 64, 128, 2, 2, 2, true, true, GATED>, Y>(p, splits, stream);
}

}  // namespace

#define LAUNCH_TILES_OF(element) launch_tiles_##element
#define LAUNCH_TILES(element) LAUNCH_TILES_OF(element)
void LAUNCH_TILES(TIRAMISU_OPERAND)(int edge, product_layout layout, int epilogue, int y, const product_arguments &p, int splits, hipStream_t stream) {
    constexpr int E = TIRAMISU_OPERAND;
    if constexpr (E == F8) {                // with k along the rows, to either 16-bit type
        if (epilogue == GATED) y == BF16 ? launch_gated<E, BF16>(edge, p, splits, stream) : launch_gated<E, F16>(edge, p, splits, stream);
        else y == BF16 ? launch_linear<E, BF16, true, true>(edge, p, splits, stream) : launch_linear<E, F16, true, true>(edge, p, splits, stream);
    } else if (epilogue == GATED) launch_gated<E, E>(edge, p, splits, stream);
    else if (layout == FORWARD) launch_linear<E, E, true, true>(edge, p, splits, stream);
    else if (layout == INPUT_GRADIENT) launch_linear<E, E, true, false>(edge, p, splits, stream);
    else launch_linear<E, E, false, false>(edge, p, splits, stream);
}

}  // namespace tops
