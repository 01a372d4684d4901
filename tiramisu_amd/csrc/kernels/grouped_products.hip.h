// Matrix products of rows that are grouped, every group with a weight of its own: y[s] = x[s] W[g]^T for offsets[g] <= s < offsets[g + 1], and its gradients, on the
// tiles of linear_tiles.hip.h and the wavefronts of linear_few_tokens.hip.h.  How many rows a group has stands in GPU memory and the host never asks: a launch
// has as many workgroups as the groups could need at most, every workgroup looks up which tile of which group is its own, and those left over end at once.
//
// Looking up is a sum over the groups' tiles, 64 groups at a time across the lanes of a wavefront, and each wavefront does it for itself: no barrier, no
// launch ahead that would plan, and no table.  Rows ahead of the first group's (of a launch for some of the experts) and behind the last one's are rows of zeros: two more
// groups, whose products have no terms.
// Offsets are bounded by the number of rows before they are used, so that no offsets whatever lead outside of the operands.
#ifndef TIRAMISU_AMD_GROUPED_PRODUCTS_HIP_H
#define TIRAMISU_AMD_GROUPED_PRODUCTS_HIP_H
#include "linear_few_tokens.hip.h"
#include "wave_reduce.hip.h"

namespace tgroups {

using namespace tops;

struct grouped_arguments {
    product_arguments p;                    // addresses of the first group's; M: rows in all (gradient of the weights: rows of a group's result)
    const int *offsets;                     // groups + 1
    int groups, rows;                       // rows in all
    picked_rows picked;                     // forward: x's rows (index null: x holds the grouped rows themselves, from the caller or moved)
    long b_step, b2_step;                   // elements from group to group of the weights (input's gradient, gated: b2 is the second pair's)
    long y_step;                            // gradient of the weights: elements from group to group of the result
    int splits;                             // ... workgroups that share the terms of a tile: sums to p.partial, [group][split][M][N]
};

struct group_span { int first, rows; };
__device__ __forceinline__ group_span span_of(const int *offsets, int g, int all) {
    const int first = min(max(offsets[g], 0), all), end = min(max(offsets[g + 1], first), all);
    return {first, end - first};
}
__device__ __forceinline__ int sum_up_to(int v) { return twave::wave_group_sum<64>(v); }       // (its steps leave in every lane the sum over the lanes up to it)
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// Consecutive workgroups go to the eight XCDs in turn: every XCD gets a run of consecutive tiles (as in tile_of).
__device__ __forceinline__ int tile_in_runs(int id, int tiles) {
    const int x = id % XCDS, each = tiles / XCDS, rest = tiles % XCDS;
    return x * each + min(x, rest) + id / XCDS;
}
// Tile t of a product of `rows` x `columns` tiles: down BAND rows of tiles before a column on (as in tile_of)
__device__ __forceinline__ void tile_in_bands(int t, int rows, int columns, int &row, int &column) {
    constexpr int BAND = 4;
    const int band = t / (BAND * columns), in = t - band * BAND * columns, height = min(rows - band * BAND, BAND);
    column = in / height;
    row = band * BAND + in - column * height;
}

// Whose tile workgroup `id` computes, of tiles that are HEIGHT rows high and `across` to a row: group < 0: nobody's; group == groups: the rows' ahead of the groups or behind them.
struct found_tile { int group, first, rows, tile; };
template <int HEIGHT>
__device__ __forceinline__ found_tile find_tile(const int *offsets, int groups, int all, int across, int id, int lane) {
    const int chunks = (groups + 63) / 64, head = uniform(min(max(offsets[0], 0), all)), last = uniform(min(max(offsets[groups], 0), all));
    auto of_lane = [&](int chunk) {
        const int g = chunk * 64 + lane;
        return g < groups ? span_of(offsets, g, all) : group_span{0, 0};
    };
    auto tiles_of = [&](const group_span &s) { return (s.rows + HEIGHT - 1) / HEIGHT * across; };
    group_span s = of_lane(0);
    int tiles = tiles_of(s), upto = sum_up_to(tiles), total = __builtin_amdgcn_readlane(upto, 63);
    for (int c = 1; c < chunks; c++) total += __builtin_amdgcn_readlane(sum_up_to(tiles_of(of_lane(c))), 63);
    const int ahead = (head + HEIGHT - 1) / HEIGHT * across, everything = total + ahead + (all - last + HEIGHT - 1) / HEIGHT * across;
    if (id >= everything) return {-1, 0, 0, 0};
    int t = tile_in_runs(id, everything);
    if (t >= total + ahead) return {groups, last, all - last, t - total - ahead};
    if (t >= total) return {groups, 0, head, t - total};
    int c = 0;
    for (int here; t >= (here = __builtin_amdgcn_readlane(upto, 63)) && c + 1 < chunks;) {
        t -= here;
        s = of_lane(++c);
        tiles = tiles_of(s);
        upto = sum_up_to(tiles);
    }
    const int owner = __builtin_ctzll(__ballot(upto > t) | 1ull << 63);
    return {c * 64 + owner, __builtin_amdgcn_readlane(s.first, owner), __builtin_amdgcn_readlane(s.rows, owner),
            t - (__builtin_amdgcn_readlane(upto, owner) - __builtin_amdgcn_readlane(tiles, owner))};
}

// The product of one group's rows, from `first` on: forward and gradient of the input.  BYTES: of an operand's element, YB: of a result's.
template <int BYTES>
__device__ __forceinline__ product_arguments product_of_rows(const grouped_arguments &a, int group, int first, int rows, picked_rows &picked) {
    product_arguments p = a.p;
    picked = a.picked;
    const long f = first;
    if (picked.given) picked.given += f;
    if (picked.index) picked.index += f;
    else {
        p.a = (const char *)p.a + f * p.lda * BYTES;
        picked.all = rows;
        if (p.a_scale) p.a_scale += f;
    }
    if (p.a_more) p.a_more = (const char *)p.a_more + f * p.lda * BYTES;
    p.y = (char *)p.y + f * p.N * 2;
    if (p.pre) {
        p.pre = (char *)p.pre + f * p.N * 2;
        p.pre2 = (char *)p.pre2 + f * p.N * 2;
    }
    p.M = p.rows_above = p.split_row = rows;
    if (group >= a.groups) {                               // rows of zeros
        p.K = 0;
        p.a_scale = nullptr;
        return p;
    }
    const long g = group;
    p.b = (const char *)p.b + g * a.b_step * BYTES;
    if (p.b2) p.b2 = (const char *)p.b2 + g * a.b2_step * BYTES;
    if (p.b_more) p.b_more = (const char *)p.b_more + g * a.b2_step * BYTES;
    if (p.b_scale) p.b_scale += g * p.N;
    if (p.b2_scale) p.b2_scale += g * p.N;
    return p;
}

// D: the tile for the last rows of a group that are no more than it is high, of C's width and half of its height or less (of 256 x 256 tiles a third would be half empty
// where groups have some hundred rows).
#ifdef __HIP_DEVICE_COMPILE__               // (the host's compilation needs no body)
template <class C, class D, int Y>
__device__ __forceinline__ void rows_tile(const grouped_arguments &a, int id, lds_char *lds) {
    static_assert(C::NT == D::NT && C::COLUMNS == D::COLUMNS && C::BM % D::BM == 0, "one workgroup's size and width");
    const int across = (a.p.N + C::COLUMNS - 1) / C::COLUMNS;
    const found_tile f = find_tile<C::BM>(a.offsets, a.groups, a.rows, across, id, threadIdx.x & 63);
    const int group = uniform(f.group), rows = uniform(f.rows);
    if (group < 0) return;
    picked_rows picked;
    const product_arguments p = product_of_rows<C::BYTES>(a, group, uniform(f.first), rows, picked);
    int row, column;
    tile_in_bands(uniform(f.tile), (rows + C::BM - 1) / C::BM, across, row, column);
    constexpr int PICK = C::A_ROWS && C::B_ROWS ? ROWS_OF_A : NOTHING;
    if (C::BM != D::BM && rows - row * C::BM <= D::BM) compute_tile_at<D, Y, PICK>(p, row * (C::BM / D::BM), column, 0, lds, picked);
    else compute_tile_at<C, Y, PICK>(p, row, column, 0, lds, picked);
}

// Tiles of a group's gradient are dealt to all eight XCDs, so that each has its share of every group however many rows that has (a run of whole groups to each
// left some with half as much again as others); where eight does not divide them, groups begin at different XCDs.
template <class C, int Y>
__device__ __forceinline__ void weights_tile(const grouped_arguments &a, int id, lds_char *lds) {
    const int down = (a.p.M + C::BM - 1) / C::BM, across = (a.p.N + C::COLUMNS - 1) / C::COLUMNS, tiles = down * across, each = (tiles + XCDS - 1) / XCDS;
    const int split = id / (XCDS * each * a.groups), in = id - split * XCDS * each * a.groups;
    const int group = in / XCDS / each, tile = (in + group) % XCDS * each + in / XCDS % each;
    if (tile >= tiles) return;
    const group_span s = span_of(a.offsets, group, a.rows);
    product_arguments p = a.p;
    const long first = uniform(s.first), g = group;
    p.K = uniform(s.rows);
    if (a.splits > 1) {
        p.partial += g * a.splits * p.M * p.N;
        p.slices_per_split = ((p.K + 63) / 64 + a.splits - 1) / a.splits;
    }
    p.a = (const char *)p.a + first * p.lda * C::BYTES;
    p.y = (char *)p.y + g * a.y_step * 2;
    if (p.y_below) p.y_below = (char *)p.y_below + g * a.y_step * 2;
    int row, column;
    tile_in_bands(tile, down, across, row, column);
    if (a.picked.index) return compute_tile_at<C, Y, K_OF_B>(p, row, column, split, lds, {a.picked.index + first, a.picked.all});
    p.b = (const char *)p.b + first * p.ldb * C::BYTES;
    compute_tile_at<C, Y>(p, row, column, split, lds);
}
#endif

// (192 rows: registers for two workgroups to a compute unit, which the LDS has room for)
template <class C, class D, int Y>
__global__ __launch_bounds__(C::NT, C::BM == 192 ? 2 : 1) void grouped_rows_kernel(grouped_arguments a) {
#ifdef __HIP_DEVICE_COMPILE__
    extern __shared__ __attribute__((aligned(16))) char shared_bytes[];
    rows_tile<C, D, Y>(a, blockIdx.x, (lds_char *)shared_bytes);
#endif
}

// Both gradients in one launch: of the rows (a: C, and D for the last ones of a group), a.p.M x a.p.N of every group's weights behind them (b: G, the rows its terms; a
// group without rows has zeros).  `start`: b's first workgroup, a multiple of the XCDs.
template <class C, class D, class G, int Y>
__global__ __launch_bounds__(C::NT) void grouped_gradients_kernel(grouped_arguments a, grouped_arguments b, int start) {
#ifdef __HIP_DEVICE_COMPILE__
    static_assert(C::NT == G::NT, "one workgroup's size");
    extern __shared__ __attribute__((aligned(16))) char shared_bytes[];
    const int id = blockIdx.x;
    if (id < start) rows_tile<C, D, Y>(a, id, (lds_char *)shared_bytes);
    else weights_tile<G, Y>(b, id - start, (lds_char *)shared_bytes);
#endif
}

// Few rows to a group: bound by the bytes of the weights of the groups that have rows.  grid: (columns in sixteens, groups that may have rows and one): workgroups
// of the last row of the grid write the rows ahead of the groups and behind them.  A group's weights are read once for each TILES x 16 of its rows.
template <int E, int Y, int EPILOGUE, int TILES, int SPLIT>
__global__ __launch_bounds__(64 * FEW_WAVES) void grouped_few_kernel(grouped_arguments a) {
    constexpr int BYTES = E == F8 ? 1 : 2, COLUMNS = FEW_ROWS * (FEW_WAVES / SPLIT);
    const int lane = threadIdx.x & 63, wanted = blockIdx.y;
    const long n0 = (long)blockIdx.x * COLUMNS;
    if (wanted == (int)gridDim.y - 1) {
        const int head = min(max(a.offsets[0], 0), a.rows), last = min(max(a.offsets[a.groups], 0), a.rows), some = (int)min((long)COLUMNS, a.p.N - n0);
        for (long i = threadIdx.x; i < (long)(head + a.rows - last) * COLUMNS; i += 64 * FEW_WAVES) {
            const long row = i / COLUMNS, at = (row < head ? row : last + row - head) * a.p.N + n0 + i % COLUMNS;
            if (i % COLUMNS >= some) continue;
            ((uint16_t *)a.p.y)[at] = 0;
            if (a.p.pre) ((uint16_t *)a.p.pre)[at] = ((uint16_t *)a.p.pre2)[at] = 0;
        }
        return;
    }
    int group = -1, first = 0, rows = 0;
    for (int c = 0, seen = 0; c * 64 < a.groups && group < 0; c++) {
        const int g = c * 64 + lane;
        const group_span s = g < a.groups ? span_of(a.offsets, g, a.rows) : group_span{0, 0};
        const unsigned long long some = __ballot(s.rows > 0);
        const int before = __popcll(some & ((1ull << lane) - 1));
        const unsigned long long mine = __ballot(s.rows > 0 && seen + before == wanted);
        if (mine) {
            const int owner = __builtin_ctzll(mine);
            group = c * 64 + owner;
            first = __builtin_amdgcn_readlane(s.first, owner);
            rows = __builtin_amdgcn_readlane(s.rows, owner);
        }
        seen += __popcll(some);
    }
    if (group < 0) return;
    for (int from = 0; from < rows; from += 16 * TILES) {
        if (from > 0) __syncthreads();                     // (the sums of the rows before have been read)
        picked_rows picked;
        const product_arguments p = product_of_rows<BYTES>(a, group, first + from, min(rows - from, 16 * TILES), picked);
        few_tokens<E, Y, EPILOGUE, TILES, true, SPLIT>(p, n0, picked);
    }
}

// The sums of the gradient of the weights, added in order: 8 columns of a row of a group to a thread
template <int Y>
__global__ __launch_bounds__(256) void grouped_weights_finish_kernel(grouped_arguments a) {
    const long across = (a.p.N + 7) / 8, id = (long)blockIdx.x * 256 + threadIdx.x, all = across * a.p.M;
    if (id >= all * a.groups) return;
    const long g = id / all, m = (id - g * all) / across, n = 8 * (id - g * all - m * across);
    const int some = (int)min(8L, a.p.N - n);
    product_arguments p = a.p;
    p.y = (char *)p.y + g * a.y_step * 2;
    if (p.y_below) p.y_below = (char *)p.y_below + g * a.y_step * 2;
    float z[8];
#pragma unroll
    for (int i = 0; i < 8; i++) z[i] = 0.f;
    for (int s = 0; s < a.splits; s++) {
        float v[8];
        load_some<F32>(p.partial + ((g * a.splits + s) * p.M + m) * p.N + n, some, v);
#pragma unroll
        for (int i = 0; i < 8; i++) z[i] += v[i];
    }
    store_linear<Y, true>(p, z, m, n, some);
}

// Rows to where the tiles can load them, 16 bytes at a time, `to` bytes apart (a multiple of 16; the rest of a row is zero): in their order, or those that an index picks, zeros where it picks
// none of x's.  Up to three operands in one launch, blockIdx.y.
struct row_move { const char *in; char *out; const int *index; long rows, all, bytes, from, to; };
struct row_moves { row_move of[3]; };
template <int BYTES>
__global__ __launch_bounds__(256) void move_operands_kernel(row_moves moves) {
    const row_move m = moves.of[blockIdx.y];
    const long across = m.to / 16, all = across * m.rows;
    for (long id = (long)blockIdx.x * 256 + threadIdx.x; id < all; id += (long)gridDim.x * 256) {
        const long r = id / across, c = 16 * (id - r * across), row = m.index ? m.index[r] : r;
        u32x4 w = {0, 0, 0, 0};
        if (row >= 0 && row < m.all) w = load_to_end<BYTES>(m.in + row * m.from + c, m.bytes - c, m.bytes);
        *reinterpret_cast<u32x4 *>(m.out + r * m.to + c) = w;
    }
}

// ... and their scales
static __global__ __launch_bounds__(256) void pick_scales_kernel(const float *in, float *out, const int *index, long rows, long all) {
    const long m = (long)blockIdx.x * 256 + threadIdx.x;
    if (m >= rows) return;
    const long row = index[m];
    out[m] = row >= 0 && row < all ? in[row] : 1.f;
}

}  // namespace tgroups
#endif
