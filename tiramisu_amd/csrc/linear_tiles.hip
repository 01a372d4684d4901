// The kernels of linear_tiles.hip.h for operands of one type (TIRAMISU_OPERAND: F16, BF16 or F8; compiled once for each), and the choice among them by
// the tile, how the operands lie and the epilogue.
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

// Wavefronts, stages and matrix instructions of each tile.  Of those measured, the fastest for the launches that choose the tile; us for bf16 with 2 x 2
// wavefronts and 32 x 32 blocks / as here: 256 x 256 (4096^3) 117 / 102 (4 x 2: 133, registers spilled); 256 x 128 (4096^3) 123 / 115; 128 x 128 in
// one round (4096 x 1024 x 4096) 43 with two stages, 37.4 with four / 35.1; 64 x 64 (1024^3) 7.7 / 7.0.  8 bits: 256 x 256 (4096^3) 68 / 62, where 16 x 16 blocks
// do not leave registers for two sets of fragments (150); 256 x 128 74 / 67; 128 x 128 (4096 x 1024 x 4096) 26 / 23; 64 x 64 (512 x 2048 x 2048) 8.2 / 7.0.
template <int E, int Y, bool A_ROWS, bool B_ROWS, int EPILOGUE>
void launch_tile(product_tile tile, const product_arguments &p, int splits, hipStream_t stream) {
    if (tile == TILE_256) launch<tile_config<E, 256, 256, 2, 4, 2, A_ROWS, B_ROWS, EPILOGUE, E == F8 ? 32 : 16>, Y>(p, splits, stream);
    else if (tile == TILE_256x128) launch<tile_config<E, 256, 128, 4, 2, 3, A_ROWS, B_ROWS, EPILOGUE, 16>, Y>(p, splits, stream);
    else if (tile == TILE_128) launch<tile_config<E, 128, 128, 4, 2, 4, A_ROWS, B_ROWS, EPILOGUE, 16>, Y>(p, splits, stream);
    else if constexpr (EPILOGUE == GATED) launch<tile_config<E, 64, 128, 2, 2, 3, A_ROWS, B_ROWS, EPILOGUE, 16>, Y>(p, splits, stream);
    else launch<tile_config<E, 64, 64, 2, 2, 3, A_ROWS, B_ROWS, EPILOGUE, 16>, Y>(p, splits, stream);
}

}  // namespace

#define LAUNCH_TILES_OF(element) launch_tiles_##element
#define LAUNCH_TILES(element) LAUNCH_TILES_OF(element)
void LAUNCH_TILES(TIRAMISU_OPERAND)(product_tile tile, product_layout layout, int epilogue, int y, const product_arguments &p, int splits, hipStream_t stream) {
    constexpr int E = TIRAMISU_OPERAND;
    if constexpr (E == F8) {                // with k along the rows, to either 16-bit type
        if (epilogue == GATED) y == BF16 ? launch_tile<E, BF16, true, true, GATED>(tile, p, splits, stream) : launch_tile<E, F16, true, true, GATED>(tile, p, splits, stream);
        else y == BF16 ? launch_tile<E, BF16, true, true, LINEAR>(tile, p, splits, stream) : launch_tile<E, F16, true, true, LINEAR>(tile, p, splits, stream);
    } else if (epilogue == GATED) launch_tile<E, E, true, true, GATED>(tile, p, splits, stream);
    else if (layout == FORWARD) launch_tile<E, E, true, true, LINEAR>(tile, p, splits, stream);
    else if (layout == INPUT_GRADIENT) launch_tile<E, E, true, false, LINEAR>(tile, p, splits, stream);
    else launch_tile<E, E, false, false, LINEAR>(tile, p, splits, stream);
}

}  // namespace tops
