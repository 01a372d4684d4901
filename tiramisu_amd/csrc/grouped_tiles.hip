// The kernels of grouped_products.hip.h on tiles, for operands of one type (TIRAMISU_OPERAND: F16, BF16 or F8; compiled once for each), and the choice among
// them by the tile, how the operands lie and the epilogue.
#include "grouped_operators.h"

#include <atomic>

#include "kernels/target_gfx950.h"

namespace tgroups {
namespace {

using tiramisu_runtime::check;

// more LDS than a launch gets unasked: asked for once on every device
void allow_lds(const void *kernel, int bytes, std::atomic<unsigned long long> &asked) {
    int device = 0;
    check(hipGetDevice(&device), "tiramisu_hip_grouped_linear");
    const unsigned long long bit = 1ull << (device & 63);
    if (asked.load() & bit) return;
    check(hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes), "tiramisu_hip_grouped_linear");
    asked.fetch_or(bit);
}

template <class C>
long tiles_of(const grouped_arguments &a, long others = 2) {
    const long across = (a.p.N + C::COLUMNS - 1) / C::COLUMNS;
    if (C::A_ROWS) return most_row_tiles(a.rows, a.groups, C::BM, others) * across;
    return ((a.p.M + C::BM - 1L) / C::BM * across + XCDS - 1) / XCDS * XCDS * a.groups * a.splits;
}
// Whether tiles are two to a compute unit: by those of a launch for all groups, whose rows none are ahead of
bool more_than_a_round(long tiles) { return tiles > ttarget::COMPUTE_UNITS; }
template <class C, class D, int Y>
void launch(const grouped_arguments &a, hipStream_t stream) {
    auto kernel = grouped_rows_kernel<C, D, Y>;
    constexpr int LDS = C::LDS_BYTES > D::LDS_BYTES ? C::LDS_BYTES : D::LDS_BYTES;
    static std::atomic<unsigned long long> asked{0};
    allow_lds((const void *)kernel, LDS, asked);
    hipLaunchKernelGGL(kernel, dim3((unsigned)tiles_of<C>(a)), dim3(C::NT), LDS, stream, a);
    check(hipGetLastError(), "tiramisu_hip_grouped_linear");
}
template <class C, class D, class G, int Y>
void launch_gradients(const grouped_arguments &a, const grouped_arguments &b, hipStream_t stream) {
    auto kernel = grouped_gradients_kernel<C, D, G, Y>;
    constexpr int ROWS = C::LDS_BYTES > D::LDS_BYTES ? C::LDS_BYTES : D::LDS_BYTES, RING = G::STAGES * G::STAGE + 4 * PICKS, WEIGHTS = RING > G::LDS_BYTES ? RING : G::LDS_BYTES,
                  LDS = ROWS > WEIGHTS ? ROWS : WEIGHTS;
    static_assert(LDS <= 160 * 1024, "LDS of a compute unit");
    static std::atomic<unsigned long long> asked{0};
    allow_lds((const void *)kernel, LDS, asked);
    const long start = a.p.y ? (tiles_of<C>(a) + XCDS - 1) / XCDS * XCDS : 0, tiles = start + (b.p.y ? tiles_of<G>(b) : 0);
    hipLaunchKernelGGL(kernel, dim3((unsigned)tiles), dim3(C::NT), b.picked.index ? LDS : ROWS > G::LDS_BYTES ? ROWS : G::LDS_BYTES, stream, a, b, (int)start);
    check(hipGetLastError(), "tiramisu_hip_grouped_linear");
}

template <int E, bool A_ROWS, bool B_ROWS, int EPILOGUE> struct tiles_for {
    static constexpr int F = E == F8 ? 32 : 16, SMALL_N = EPILOGUE == GATED ? 128 : 64;
    typedef tile_config<E, 256, 256, 2, 4, 2, A_ROWS, B_ROWS, EPILOGUE, F> tile_256;
    typedef tile_config<E, 128, 256, 2, 4, 3, A_ROWS, B_ROWS, EPILOGUE, 16> tile_256_end;
    typedef tile_config<E, 256, 128, 4, 2, 3, A_ROWS, B_ROWS, EPILOGUE, 16> tile_256x128;
    typedef tile_config<E, 128, 128, 4, 2, 4, A_ROWS, B_ROWS, EPILOGUE, 16> tile_128;
    // (two stages: two workgroups to a compute unit, which cover each other's beginnings and ends where there is more than a round of tiles; us with four / with two, bf16:
    // 8192 rows in 64 groups, gated 1024 x 2048 154 / 145, gradient of 16384 rows in 32 groups of 2048 x 2048 200 / 186, one round of 1500 x 700 19.7 / 23.7; 8 bits, 32768 rows 259 / 315)
    typedef tile_config<E, 128, 128, 4, 2, 2, A_ROWS, B_ROWS, EPILOGUE, 16> tile_128_pair;
    typedef tile_config<E, 64, 128, 2, 4, 4, A_ROWS, B_ROWS, EPILOGUE, 16> tile_128_end;
    typedef tile_config<E, 64, 128, 2, 4, 2, A_ROWS, B_ROWS, EPILOGUE, 16> tile_128_pair_end;
    // Two to a compute unit, whose LDS they fill, four wavefronts of 96 x 64 each: they read LDS as little as those of 256 x 128 and cover each other's beginnings and ends
    // (8192 rows in 8 groups bf16, 2048 x 2048, as 256 x 256 / 256 x 128 / 128 x 128 / so: 89 / 81 / 80 / 65 us, gated, which the rule leaves on the first, 158 / 151 / 157 / 131).
    typedef tile_config<E, 192, 128, 2, 2, 2, A_ROWS, B_ROWS, EPILOGUE, 16> tile_192x128;
    typedef tile_config<E, 96, 128, 1, 4, 2, A_ROWS, B_ROWS, EPILOGUE, 16> tile_192x128_end;
    typedef tile_config<E, 64, SMALL_N, 2, EPILOGUE == GATED ? 4 : 2, 3, A_ROWS, B_ROWS, EPILOGUE, 16> tile_64;
};
template <int E, int Y, int EPILOGUE>
void launch_tile(product_tile tile, const grouped_arguments &a, hipStream_t stream) {
    typedef tiles_for<E, true, true, EPILOGUE> T;
    if (tile == TILE_256) launch<typename T::tile_256, typename T::tile_256_end, Y>(a, stream);
    else if (tile == TILE_256x128) launch<typename T::tile_256x128, typename T::tile_128, Y>(a, stream);
    else if (tile == TILE_128) {
        if constexpr (E != F8)
            if (more_than_a_round(tiles_of<typename T::tile_128>(a, 1))) return launch<typename T::tile_128_pair, typename T::tile_128_pair_end, Y>(a, stream);
        launch<typename T::tile_128, typename T::tile_128_end, Y>(a, stream);
    } else if (tile == TILE_192x128) {
        if constexpr (E != F8) launch<typename T::tile_192x128, typename T::tile_192x128_end, Y>(a, stream);
    } else launch<typename T::tile_64, typename T::tile_64, Y>(a, stream);
}

}  // namespace

#define JOIN_NAMES(name, element) name##element
#define NAME_OF(name, element) JOIN_NAMES(name, element)
void NAME_OF(launch_grouped_, TIRAMISU_OPERAND)(product_tile tile, int epilogue, int y, const grouped_arguments &a, hipStream_t stream) {
    constexpr int E = TIRAMISU_OPERAND;
    if constexpr (E == F8) {                // to either 16-bit type
        if (epilogue == GATED) y == BF16 ? launch_tile<E, BF16, GATED>(tile, a, stream) : launch_tile<E, F16, GATED>(tile, a, stream);
        else y == BF16 ? launch_tile<E, BF16, LINEAR>(tile, a, stream) : launch_tile<E, F16, LINEAR>(tile, a, stream);
    } else if (epilogue == GATED) launch_tile<E, E, GATED>(tile, a, stream);
    else launch_tile<E, E, LINEAR>(tile, a, stream);
}

#ifndef TIRAMISU_OPERAND_HAS_NO_GRADIENTS
void NAME_OF(launch_grouped_gradients_, TIRAMISU_OPERAND)(product_tile tile, const grouped_arguments &a, const grouped_arguments &b, hipStream_t stream) {
    constexpr int E = TIRAMISU_OPERAND;
    typedef tiles_for<E, true, false, LINEAR> R;
    typedef tiles_for<E, false, false, LINEAR> W;
    if (tile == TILE_256) launch_gradients<typename R::tile_256, typename R::tile_256_end, typename W::tile_256, E>(a, b, stream);
    else if (tile == TILE_256x128) launch_gradients<typename R::tile_256x128, typename R::tile_128, typename W::tile_256x128, E>(a, b, stream);
    else if (tile == TILE_128) {
        if (more_than_a_round((a.p.y ? tiles_of<typename R::tile_128>(a, 1) : 0) + (b.p.y ? tiles_of<typename W::tile_128>(b) : 0)))
            launch_gradients<typename R::tile_128_pair, typename R::tile_128_pair_end, typename W::tile_128_pair, E>(a, b, stream);
        else launch_gradients<typename R::tile_128, typename R::tile_128_end, typename W::tile_128, E>(a, b, stream);
    } else launch_gradients<typename R::tile_64, typename R::tile_64, typename W::tile_64, E>(a, b, stream);
}
#endif

}  // namespace tgroups
