// Entry points of the operators of a feed-forward sublayer with experts and of 4-bit weights (include/tiramisu_hip_wrappers.h): what they refuse, which kernel a
// call goes to, and the launches.  As in operators.hip: all launches of a call are planned first, then its scratch is asked for, as one block.
#include "operator_calls.h"

#include <algorithm>
#include <atomic>
#include <cstdint>

#include "../../include/tiramisu_hip_wrappers.h"
#include "grouped_operators.h"
#include "kernels/combine.hip.h"
#include "kernels/four_bit.hip.h"
#include "kernels/operator_backward.hip.h"
#include "kernels/route.hip.h"
#include "kernels/target_gfx950.h"

using namespace tops;
using tiramisu_runtime::check;
using tiramisu_runtime::stream;
using tiramisu_runtime::timed;

namespace {

typedef unsigned long long ull;

// ---- route
using troute::ROUTE_FEW_THREADS;
using troute::ROUTE_THREADS;
using troute::route_arguments;
using troute::route_backward_arguments;

// (lanes of a token and values of a lane, by the number of experts)
template <class F>
void by_experts(int experts, F f) {
    if (experts <= 16) f(std::integral_constant<int, 16>(), std::integral_constant<int, 1>());
    else if (experts <= 32) f(std::integral_constant<int, 16>(), std::integral_constant<int, 2>());
    else if (experts <= 64) f(std::integral_constant<int, 16>(), std::integral_constant<int, 4>());
    else if (experts <= 128) f(std::integral_constant<int, 16>(), std::integral_constant<int, 8>());
    else if (experts <= 256) f(std::integral_constant<int, 16>(), std::integral_constant<int, 16>());
    else if (experts <= 512) f(std::integral_constant<int, 64>(), std::integral_constant<int, 8>());
    else f(std::integral_constant<int, 64>(), std::integral_constant<int, 16>());
}

// Tokens that one workgroup routes; with more, blocks of tokens do, in two launches (us as one / as blocks, 8 of 64 experts: 32 tokens 5.7 / 9.5, 64 7.7 / 10.0, 128 12.9 / 10.1; of 600, a wavefront to a
// token: 16 tokens 14 / 16, 32 24 / 16.5).
long experts_lanes(int experts) { return experts <= 256 ? 16 : 64; }
long route_few(int experts) { return experts_lanes(experts) == 16 ? 80 : 24; }
template <int E>
int route(const char *fn, route_arguments a) {
    if (a.tokens <= route_few(a.experts)) {
        const size_t lds = troute::route_lds_bytes(a.experts, ROUTE_FEW_THREADS);
        by_experts(a.experts, [&](auto lanes, auto values) {
            hipLaunchKernelGGL((troute::route_few_kernel<E, decltype(lanes)::value, decltype(values)::value>), dim3(1), dim3(ROUTE_FEW_THREADS), lds, stream(), a);
        });
        check(hipGetLastError(), fn);
        return 0;
    }
    const size_t lds = troute::route_lds_bytes(a.experts, ROUTE_THREADS);
    a.block = (int)std::max(experts_lanes(a.experts) == 16 ? 64L : 16L, (a.tokens + ttarget::COMPUTE_UNITS - 1) / ttarget::COMPUTE_UNITS);
    const unsigned blocks = (unsigned)((a.tokens + a.block - 1) / a.block);
    call_scratch s;
    const uint64_t counts = s.want((uint64_t)blocks * a.experts * 4);
    if (s.take(fn)) return 1;
    a.counts = (int *)s.at(counts);
    by_experts(a.experts, [&](auto lanes, auto values) {
        hipLaunchKernelGGL((troute::route_choose_kernel<E, decltype(lanes)::value, decltype(values)::value>), dim3(blocks), dim3(ROUTE_THREADS), lds, stream(), a);
    });
    hipLaunchKernelGGL(troute::route_place_kernel, dim3(blocks), dim3(ROUTE_THREADS), lds, stream(), a);
    check(hipGetLastError(), fn);
    return 0;
}
template <int E>
void route_backward(const char *fn, const route_backward_arguments &a) {
    by_experts(a.experts, [&](auto lanes, auto values) {
        constexpr int TOKENS = 256 / decltype(lanes)::value;
        hipLaunchKernelGGL((troute::route_backward_kernel<E, decltype(lanes)::value, decltype(values)::value>), dim3((unsigned)((a.tokens + TOKENS - 1) / TOKENS)), dim3(256), 0, stream(), a);
    });
    check(hipGetLastError(), fn);
}
int refuse_route(const char *fn, uint64_t tokens, uint64_t experts, uint64_t k, int type) {
    if (!known_type(type, true)) return refuse(fn, "element type %d: float32, float16 or bfloat16", type);
    if (experts < 1 || experts > troute::MOST_EXPERTS) return refuse(fn, "%llu experts: 1 to %d", (ull)experts, troute::MOST_EXPERTS);
    if (k < 1 || k > experts || k > troute::MOST_CHOSEN) return refuse(fn, "%llu of %llu experts: 1 to all of them, and to %d", (ull)k, (ull)experts, troute::MOST_CHOSEN);
    if (tokens > (1 << 24)) return refuse(fn, "%llu tokens: at most 2^24", (ull)tokens);
    return 0;
}

// ---- products of grouped rows
using tgroups::grouped_arguments;

constexpr uint64_t MOST_GROUPS = 1024;
int refuse_grouped(const char *fn, uint64_t S, uint64_t T, uint64_t groups, uint64_t N, uint64_t K, int activation, int type, int y) {
    if (groups < 1 || groups > MOST_GROUPS) return refuse(fn, "%llu groups: 1 to %llu", (ull)groups, (ull)MOST_GROUPS);
    if (S > MOST || T > MOST) return refuse(fn, "%llu rows of %llu: at most 2^30 - 1", (ull)S, (ull)T);
    if (const int rc = refuse_product(fn, std::min<uint64_t>(S, 64), N, K, activation, type, y)) return rc;
    if ((uint64_t)tgroups::most_row_tiles((long)S, (long)groups, 64) * ((N + 63) / 64) > MOST_TILES) return refuse(fn, "%llu rows of %llu in %llu groups: more tiles than a launch holds", (ull)S, (ull)N, (ull)groups);
    return 0;
}

// ---- which tile, by the launch's model (operators.hip) for the tiles that the groups have if the rows are spread as routers spread them, a tenth more than evenly, a
// group's last tile half empty where it has several; what the model says is multiplied by `factor`, as groups bring weights of their own, whose bytes come at 4.6 TB/s.  192 x 128 are 16 bits' and forward.  Of 585
// launches of 16 bits and 135 of 8 (2 to 128 groups, 64 to 32768 rows, groups uneven) the choice is 5 % and 3 % behind the fastest tile in the geometric mean (16 bits without 192 x 128: 6 %), a third to a half at worst:
// few tiles of few rows, or a round that begins with a few tiles, as the groups' sizes are not known here (4096 rows in 16 groups, 2048 x 6144: 175 us on the 256 x 256 that this takes, 146 on 192 x 128).
constexpr struct { product_tile tile; int rows, columns; double factor; } GROUPED_TILES[] = {{TILE_256, 256, 256, 1.0}, {TILE_256x128, 256, 128, 1.1}, {TILE_192x128, 192, 128, 1.05}, {TILE_128, 128, 128, 1.0},
                                                                                             {TILE_64, 64, 64, 1.25}};
double rows_tiles(const grouped_arguments &a, int rows, int columns, bool gated) {
    const double active = (double)std::min(a.groups, a.rows);
    return 1.1 * active * std::max(1.0, a.rows / active / rows + 0.5) * (double)(((gated ? 2L : 1L) * a.p.N + columns - 1) / columns);
}
product_tile grouped_tile(const grouped_arguments &a, int bytes, bool gated) {
    const double weights = (gated ? 2.0 : 1.0) * std::min(a.groups, a.rows) * a.p.N * a.p.K * bytes / 4.6e6 + 3.0;
    product_tile best = TILE_64;
    double best_cost = 0;
    for (const auto &t : GROUPED_TILES) {
        if (t.tile == TILE_192x128 && bytes == 1) continue;
        const long tiles = std::max(1L, (long)rows_tiles(a, t.rows, gated && t.tile == TILE_64 ? 128 : t.columns, gated)), slices = std::max(1L, ((long)a.p.K * bytes + 127) / 128);
        const double launch = t.factor * tile_launch_cost(t.tile, tiles, slices, bytes, gated), cost = std::max(launch, weights) + 0.2 * std::min(launch, weights);
        if (best_cost == 0 || cost < best_cost) { best = t.tile; best_cost = cost; }
    }
    return best;
}
// Both gradients: as one launch of as many tiles as they have together, whose slices are theirs in the mean; where there are few rounds, those of a group of twice the
// mean's rows, whose tiles the launch waits for (6720 rows in 14 groups, 140 x 1053: 256 x 256 tiles 45 us, 128 x 128 34).  The terms of the weights' tiles may be shared by several workgroups, whose
// sums, written and read again at 5 TB/s, a launch more adds (14252 rows in 3 groups, 192 x 103: 50 us, so 28).
struct gradients_plan { product_tile tile; int splits; };
gradients_plan plan_gradients(const grouped_arguments &a, const grouped_arguments &b, int pairs) {
    gradients_plan best = {TILE_64, 1};
    double best_cost = 0;
    for (const auto &t : GROUPED_TILES)
        for (int splits = 1; splits <= 16 && t.tile != TILE_192x128; splits *= 2) {
            const double of_rows = pairs * ((a.p.K + 63) / 64), of_weights = (double)b.rows / b.groups / 64 / splits;
            const double down = a.p.y ? rows_tiles(a, t.rows, t.columns, false) : 0;
            const double across = b.p.y ? (double)((b.p.M + t.rows - 1L) / t.rows) * ((b.p.N + t.columns - 1L) / t.columns) * b.groups * splits : 0, tiles = std::max(1.0, down + across);
            if (splits > 1 && (!b.p.y || of_weights < 2.0 || tiles > 4 * ttarget::COMPUTE_UNITS)) break;
            double slices = (down * of_rows + across * (of_weights + 0.5)) / tiles;
            if (tiles <= 2 * ttarget::COMPUTE_UNITS) slices = std::max(slices, std::max(down ? of_rows : 0.0, across ? 2 * of_weights : 0.0));
            double cost = t.factor * tile_launch_cost(t.tile, (long)tiles, std::max(1L, (long)(slices + 0.5)), 2, false);
            if (splits > 1) cost += 4.0 + 2.0 * splits * b.groups * b.p.M * b.p.N * 4 / 5e6;
            if (best_cost == 0 || cost < best_cost) { best = {t.tile, splits}; best_cost = cost; }
        }
    return best;
}
struct planned_gradients {
    gradients_plan plan;
    uint64_t partial;
};
planned_gradients plan_gradients(grouped_arguments &a, grouped_arguments &b, int pairs, call_scratch &s) {
    planned_gradients g = {plan_gradients(a, b, pairs), call_scratch::NOWHERE};
    b.splits = g.plan.splits;
    if (b.splits > 1) g.partial = s.want((uint64_t)b.splits * b.groups * b.p.M * b.p.N * 4);
    return g;
}
void launch_gradients(const char *fn, int type, const planned_gradients &g, const grouped_arguments &a, grouped_arguments &b, const call_scratch &s) {
    if (!a.p.y && !b.p.y) return;
    b.p.partial = (float *)s.at(g.partial);
    (type == BF16 ? tgroups::launch_grouped_gradients_BF16 : tgroups::launch_grouped_gradients_F16)(g.plan.tile, a, b, stream());
    if (b.splits == 1) return;
    const unsigned blocks = (unsigned)(((b.p.N + 7L) / 8 * b.p.M * b.groups + 255) / 256);
    if (type == BF16) hipLaunchKernelGGL(tgroups::grouped_weights_finish_kernel<BF16>, dim3(blocks), dim3(256), 0, stream(), b);
    else hipLaunchKernelGGL(tgroups::grouped_weights_finish_kernel<F16>, dim3(blocks), dim3(256), 0, stream(), b);
    check(hipGetLastError(), fn);
}

template <int E, int Y, int EPILOGUE>
void launch_few(const char *fn, const grouped_arguments &a) {
    const int active = std::min(a.groups, a.rows);
    auto go = [&](auto kernel, int split) {
        const long columns = FEW_ROWS * (FEW_WAVES / split);
        hipLaunchKernelGGL(kernel, dim3((unsigned)((a.p.N + columns - 1) / columns), (unsigned)active + 1), dim3(64 * FEW_WAVES), few_lds_bytes(1, EPILOGUE == GATED), stream(), a);
        check(hipGetLastError(), fn);
    };
    // Wavefronts that share the k of 16 columns: half or a quarter of a workgroup's where rows are short (of up to 4 KB, 2 KB) and workgroups of as many more columns still are two to a
    // compute unit: each then reads more for its look-up, launch and sums.  us with 8 / 4 / 2, bf16: 128 rows in 64 groups, 2048 x 1024 61 / 46 / 41, gated 1024 x 2048 87 / 79 / 86;
    // 8 rows in 8 groups 10.9 / 8.9 / 9.2 and 14.4 / 14.8 / 19.6.
    const long bytes = (long)a.p.K * bytes_of(E), workgroups = (a.p.N + FEW_ROWS - 1L) / FEW_ROWS * active;
    if constexpr (EPILOGUE == LINEAR)
        if (bytes <= 2048 && workgroups >= 8 * ttarget::COMPUTE_UNITS) return go(tgroups::grouped_few_kernel<E, Y, EPILOGUE, 1, 2>, 2);
    if (bytes <= 4096 && workgroups >= 4 * ttarget::COMPUTE_UNITS) return go(tgroups::grouped_few_kernel<E, Y, EPILOGUE, 1, 4>, 4);
    go(tgroups::grouped_few_kernel<E, Y, EPILOGUE, 1, 8>, 8);
}
template <int EPILOGUE>
void launch_few(const char *fn, int type, int y, const grouped_arguments &a) {
    if (type == BF16) launch_few<BF16, BF16, EPILOGUE>(fn, a);
    else if (type == F16) launch_few<F16, F16, EPILOGUE>(fn, a);
    else if (y == BF16) launch_few<F8, BF16, EPILOGUE>(fn, a);
    else launch_few<F8, F16, EPILOGUE>(fn, a);
}

// (rows are picked at offsets of 31 bits)
bool can_pick(const operand &x, long rows, long columns, int bytes) { return rows > 0 && loadable(x, bytes, true) && ((rows - 1) * x.ld + columns) * bytes < 0x7ffffff0L; }

// Operands that have to be moved ahead of a call's product: up to three, all in one launch (gated gradients at odd sizes had five launches, so three: 552 rows in 29 groups, 443 x 131, 28 -> 23 us).
class operand_moves {
public:
    explicit operand_moves(int bytes_) : bytes(bytes_) {}
    // An operand in its order: its address, and where it has to be moved what will be there
    const void *settle(const placed_operand &q, const call_scratch &s) {
        if (q.place == call_scratch::NOWHERE) return q.from.p;
        return add({(const char *)q.from.p, (char *)s.at(q.place), nullptr, q.rows, q.rows, q.columns * bytes, q.from.ld * bytes, q.ld * bytes});
    }
    // Rows of x in the groups' order
    const void *settle(const void *x, const int *index, long ldx, long tokens, long rows, long columns, long ld, uint64_t place, const call_scratch &s) {
        return add({(const char *)x, (char *)s.at(place), index, rows, tokens, columns * bytes, ldx * bytes, ld * bytes});
    }
    void launch(const char *fn) const {
        if (count == 0) return;
        long blocks = 1;
        for (int i = 0; i < count; i++) blocks = std::max(blocks, (moves.of[i].to / 16 * moves.of[i].rows + 255) / 256);
        auto kernel = bytes == 1 ? tgroups::move_operands_kernel<1> : tgroups::move_operands_kernel<2>;
        hipLaunchKernelGGL(kernel, dim3((unsigned)std::min(blocks, 1L << 20), (unsigned)count), dim3(256), 0, stream(), moves);
        check(hipGetLastError(), fn);
    }

private:
    const void *add(const tgroups::row_move &m) {
        moves.of[count++] = m;
        return m.out;
    }
    int bytes, count = 0;
    tgroups::row_moves moves = {};
};
// Rows of x where a product cannot pick them itself: a place for them, rows at multiples of 16 bytes
struct planned_rows { uint64_t place; long ld; };
planned_rows plan_rows(long rows, long columns, int bytes, call_scratch &s) {
    const long ld = (columns * bytes + 15) / 16 * 16 / bytes;
    return {rows > 0 && columns > 0 ? s.want((uint64_t)ld * bytes * rows) : call_scratch::NOWHERE, ld};
}
// Rows of x as the gradient of the weights takes them, down whose columns k runs: picked there, or moved
struct planned_weight_rows {
    const void *x;
    const int *rows;
    long ldx, places, tokens, columns;
    bool pick;
    planned_rows moved;
    placed_operand in_order;
};
planned_weight_rows plan_weight_rows(const void *x, const int *rows, long ldx, long S, long T, long K, call_scratch &s) {
    planned_weight_rows q = {x, rows, ldx, S, T, K, rows && can_pick({x, ldx}, T, K, 2) && ldx <= MOST_STEP, {call_scratch::NOWHERE, 0}, {}};
    q.in_order.place = call_scratch::NOWHERE;
    if (rows && !q.pick) q.moved = plan_rows(S, K, 2, s);
    else q.in_order = place_operand({x, ldx}, rows ? 0 : S, K, 2, false, s);
    return q;
}
void settle_weight_rows(const planned_weight_rows &q, grouped_arguments &b, operand_moves &moves, const call_scratch &s) {
    if (q.moved.place != call_scratch::NOWHERE) {
        b.p.b = moves.settle(q.x, q.rows, q.ldx, q.tokens, q.places, q.columns, q.moved.ld, q.moved.place, s);
        b.p.ldb = q.moved.ld;
        return;
    }
    b.p.b = moves.settle(q.in_order, s);
    b.p.ldb = q.in_order.ld;
    if (q.pick) b.picked = {q.rows, q.tokens};
}

// Rows that a group has in the mean, up to which wavefronts that load weights straight into registers are faster than tiles, which read each weight once for all rows of a group (us as
// few / as tiles, 64 groups of 2, 4, 8, 16 rows: gated 1024 x 2048 bf16 83 / 94, 99 / 103, 121 / 111, 176 / 111, e4m3 42 / 43, 50 / 51, 62 / 59; 2048 x 1024 bf16 41 / 41, 50 / 48, 65 / 53).
constexpr long FEW_ROWS_OF_A_GROUP = 3;

int grouped_forward(const char *fn, int type, int y, int epilogue, grouped_arguments a, const int *rows, long tokens) {
    if (a.rows == 0 || a.p.N == 0) return 0;
    const int bytes = bytes_of(type);
    const bool gated = epilogue == GATED;
    const long K = a.p.K, all = (long)a.groups * a.p.N;
    a.picked = {rows, rows ? tokens : a.rows, rows, tokens};
    a.b_step = (long)a.p.N * a.p.ldb;
    a.b2_step = (long)a.p.N * a.p.ldb2;
    if (K > 0 && a.p.N <= MOST_FEW_COLUMNS && a.rows <= FEW_ROWS_OF_A_GROUP * std::min(a.groups, a.rows)) {
        gated ? launch_few<GATED>(fn, type, y, a) : launch_few<LINEAR>(fn, type, y, a);
        return 0;
    }
    call_scratch s;
    const operand x = {a.p.a, a.p.lda};
    const bool pick = rows && can_pick(x, tokens, K, bytes);
    planned_rows moved = {call_scratch::NOWHERE, 0};
    placed_operand in_order = {};
    in_order.place = call_scratch::NOWHERE;
    if (rows && !pick) moved = plan_rows(a.rows, K, bytes, s);
    else if (!rows) in_order = place_operand(x, a.rows, K, bytes, true, s);
    const uint64_t scales = rows && !pick && a.p.a_scale ? s.want((uint64_t)a.rows * 4) : call_scratch::NOWHERE;
    const placed_operand b = place_operand({a.p.b, a.p.ldb}, all, K, bytes, true, s), b2 = place_operand({a.p.b2, a.p.ldb2}, gated ? all : 0, K, bytes, true, s);
    if (s.take(fn)) return 1;
    operand_moves moves(bytes);
    if (rows && !pick) {
        if (moved.place != call_scratch::NOWHERE) a.p.a = moves.settle(a.p.a, rows, a.p.lda, tokens, a.rows, K, moved.ld, moved.place, s);
        a.p.lda = moved.ld;
        a.picked = {nullptr, a.rows, rows, tokens};
        if (a.p.a_scale) {
            hipLaunchKernelGGL(tgroups::pick_scales_kernel, dim3((unsigned)((a.rows + 255L) / 256)), dim3(256), 0, stream(), a.p.a_scale, (float *)s.at(scales), rows, (long)a.rows, tokens);
            check(hipGetLastError(), fn);
            a.p.a_scale = (const float *)s.at(scales);
        }
    } else if (!rows) {
        a.p.a = moves.settle(in_order, s);
        a.p.lda = in_order.ld;
    }
    a.p.b = moves.settle(b, s);
    a.p.b2 = moves.settle(b2, s);
    moves.launch(fn);
    a.p.ldb = b.ld;
    a.p.ldb2 = b2.ld;
    a.b_step = (long)a.p.N * b.ld;
    a.b2_step = (long)a.p.N * b2.ld;
    const product_tile tile = grouped_tile(a, bytes, gated);
    (type == BF16 ? tgroups::launch_grouped_BF16 : type == F16 ? tgroups::launch_grouped_F16 : tgroups::launch_grouped_F8)(tile, epilogue, y, a, stream());
    return 0;
}

grouped_arguments grouped_of(uint64_t S, uint64_t groups, uint64_t N, uint64_t K, const int32_t *offsets) {
    grouped_arguments a = {};
    a.p = product_of((long)S, (long)N, (long)K);
    a.offsets = offsets;
    a.groups = (int)groups;
    a.rows = (int)S;
    a.splits = 1;
    return a;
}

// ---- 4-bit weights
using tfour::four_bit_arguments;

// more LDS than a launch gets unasked: asked for once on every device
void allow_lds(const char *fn, const void *kernel, int bytes, std::atomic<unsigned long long> &asked) {
    int device = 0;
    check(hipGetDevice(&device), fn);
    const unsigned long long bit = 1ull << (device & 63);
    if (asked.load() & bit) return;
    check(hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes), fn);
    asked.fetch_or(bit);
}
// LDS of x: whole units of k, up to a chunk
long four_bit_chunk_bytes(long K, int tiles) { return std::min(K / 128 * 128, (long)tfour::four_bit_chunk(tiles)) * 16 * tiles * 2; }

// Wavefronts that share the k of 16 columns: as few as leave a workgroup to each compute unit, as x is read once by each (us with 8 / 4 / 2: one token, 16384 x 4096 19 / 14 / 20; 64 tokens 51 / 31 /
// 21; 128 tokens, 4096 x 4096 26 / 16 / 20)
int four_bit_split(long M, long N, bool gated) {
    const long tiles = (N + FEW_ROWS - 1) / FEW_ROWS * ((M + 63) / 64);
    return tiles <= ttarget::COMPUTE_UNITS ? 8 : gated || M <= 16 || tiles <= 2 * ttarget::COMPUTE_UNITS ? 4 : 2;
}
// What the kernel of few tokens takes, for every round of its workgroups a beginning and an end and the bytes of x and weights at what a compute unit takes in, and what widening the weights ahead of a product on tiles
// does, in microseconds (few / widened: 4096 x 4096 with 128, 256 and 512 tokens 16 / 32, 21 / 37, 39 / 38; gated 8192 x 2048 with 128 and 256 23 / 45, 44 / 47).
double four_bit_few_cost(long M, long N, long K, bool gated) {
    const long teams = FEW_WAVES / four_bit_split(M, N, gated), workgroups = (N + FEW_ROWS * teams - 1) / (FEW_ROWS * teams) * ((M + 63) / 64);
    const double rounds = (double)((workgroups + ttarget::COMPUTE_UNITS - 1) / ttarget::COMPUTE_UNITS);
    return 3.0 + (rounds - 1) * 4.0 + rounds * (double)K * (2.0 * std::min(M, 64L) + 8.5 * (double)teams * (gated ? 2 : 1)) / 33e3;
}
double four_bit_widened_cost(const planned_forward &f, long N, long K, bool gated) { return 7.0 + (gated ? 2.0 : 1.0) * N * K * 2.53 / 5e6 + f.q.plan.cost; }
template <int E, int EPILOGUE, int TILES, int SPLIT>
void launch_four_few(const char *fn, const four_bit_arguments &a) {
    constexpr int TEAMS = FEW_WAVES / SPLIT;
    auto kernel = tfour::four_bit_few_kernel<E, EPILOGUE, TILES, SPLIT>;
    static std::atomic<unsigned long long> asked{0};
    allow_lds(fn, (const void *)kernel, 16 * TILES * 2 * tfour::four_bit_chunk(TILES), asked);
    const long columns = FEW_ROWS * TEAMS, lds = std::max(four_bit_chunk_bytes(a.p.K, TILES), (long)few_lds_bytes(TILES, EPILOGUE == GATED));
    hipLaunchKernelGGL(kernel, dim3((unsigned)((a.p.N + columns - 1) / columns), (unsigned)((a.p.M + 16 * TILES - 1) / (16 * TILES))), dim3(64 * FEW_WAVES), (size_t)lds, stream(), a);
    check(hipGetLastError(), fn);
}
template <int E, int EPILOGUE, int TILES>
void launch_four_few(const char *fn, const four_bit_arguments &a) {
    const int split = four_bit_split(a.p.M, a.p.N, EPILOGUE == GATED);
    if (split == 8) return launch_four_few<E, EPILOGUE, TILES, 8>(fn, a);
    if constexpr (EPILOGUE == LINEAR && TILES > 1)
        if (split == 2) return launch_four_few<E, EPILOGUE, TILES, 2>(fn, a);
    launch_four_few<E, EPILOGUE, TILES, 4>(fn, a);
}
template <int E, int EPILOGUE>
void launch_four_few(const char *fn, const four_bit_arguments &a) {
    if (a.p.M <= 16) launch_four_few<E, EPILOGUE, 1>(fn, a);
    else if (a.p.M <= 32) launch_four_few<E, EPILOGUE, 2>(fn, a);
    else launch_four_few<E, EPILOGUE, 4>(fn, a);
}
constexpr long MOST_PARTS = 65535;          // workgroups of a launch in a direction other than the first
// Few tokens in parts of 64, or the weights widened ahead of a product on tiles
template <int E>
int four_bit(const char *fn, int epilogue, four_bit_arguments a) {
    if (a.p.M == 0 || a.p.N == 0) return 0;
    const bool gated = epilogue == GATED;
    const long N = a.p.N, K = a.p.K, to = (K + 7) / 8 * 8;
    call_scratch s;
    const uint64_t wide[2] = {s.want((uint64_t)to * N * 2), gated ? s.want((uint64_t)to * N * 2) : call_scratch::NOWHERE};
    product_arguments p = a.p;
    p.b = p.b2 = nullptr;
    p.ldb = p.ldb2 = to;
    planned_forward f = plan_forward(E, E, epilogue, p, s);
    if (K > 0 && N <= MOST_FEW_COLUMNS && a.p.M <= 64 * MOST_PARTS && (a.p.M <= 64 || four_bit_few_cost(a.p.M, N, K, gated) <= four_bit_widened_cost(f, N, K, gated))) {
        call_scratch few;
        const placed_operand x = place_operand({a.p.a, a.p.lda}, a.p.M, K, 2, true, few);
        if (few.take(fn)) return 1;
        a.p.a = settle(fn, x, few);
        a.p.lda = x.ld;
        gated ? launch_four_few<E, GATED>(fn, a) : launch_four_few<E, LINEAR>(fn, a);
        return 0;
    }
    if (s.take(fn)) return 1;
    f.b.from.p = s.at(wide[0]);
    f.b2.from.p = s.at(wide[1]);
    for (int i = 0; i < (gated ? 2 : 1) && K > 0; i++)
        for (long first = 0, most = std::max(1L, MOST_PIECES_A_LAUNCH / (to / 8)); first < N; first += most) {
            const long n = std::min(most, N - first), ldq = i ? a.p.ldb2 : a.p.ldb, lds = i ? a.lds_2 : a.lds;
            hipLaunchKernelGGL((tfour::widen_rows_kernel<E>), dim3((unsigned)((to / 8 * n + 255) / 256)), dim3(256), 0, stream(), (const char *)(i ? a.p.b2 : a.p.b) + first * ldq,
                               (i ? a.scale_2 : a.scale) + first * lds, ldq, lds, n, K, (char *)s.at(wide[i]) + first * to * 2, to);
        }
    check(hipGetLastError(), fn);
    launch_forward(fn, f, s);
    return 0;
}

}  // namespace

extern "C" {

int tiramisu_hip_route(const void *logits, int32_t *experts, float *weights, int32_t *offsets, int32_t *rows, int32_t *places, uint64_t tokens, uint64_t count, uint64_t k,
                       uint64_t ldl, int32_t normalise, int32_t type) {
    if (const int rc = refuse_route(__FUNCTION__, tokens, count, k, type)) return rc;
    if (!offsets || (tokens && (!logits || !experts || !weights || !rows || !places))) return refuse(__FUNCTION__, "logits and a place for every result are needed");
    timed record(__FUNCTION__);
    const route_arguments a = {logits, ldl ? (long)ldl : (long)count, (long)tokens, (int)count, (int)k, normalise != 0, experts, weights, offsets, rows, places, nullptr, 0};
    return type == F32 ? route<F32>(__FUNCTION__, a) : type == F16 ? route<F16>(__FUNCTION__, a) : route<BF16>(__FUNCTION__, a);
}

int tiramisu_hip_route_backward(const float *dweights, const void *logits, const int32_t *experts, void *dlogits, uint64_t tokens, uint64_t count, uint64_t k, uint64_t ldl,
                                int32_t normalise, int32_t type) {
    if (const int rc = refuse_route(__FUNCTION__, tokens, count, k, type)) return rc;
    if (tokens == 0) return 0;
    if (!dweights || !logits || !experts || !dlogits) return refuse(__FUNCTION__, "dweights, logits, experts and dlogits are needed");
    timed record(__FUNCTION__);
    const route_backward_arguments a = {dweights, logits, experts, dlogits, ldl ? (long)ldl : (long)count, (long)tokens, (int)count, (int)k, normalise != 0};
    type == F32 ? route_backward<F32>(__FUNCTION__, a) : type == F16 ? route_backward<F16>(__FUNCTION__, a) : route_backward<BF16>(__FUNCTION__, a);
    return 0;
}

int tiramisu_hip_grouped_linear(const void *x, const void *weight, const int32_t *offsets, const int32_t *rows, const float *x_scale, const float *weight_scale, void *y,
                                uint64_t S, uint64_t T, uint64_t groups, uint64_t N, uint64_t K, uint64_t ldx, uint64_t ldw, int32_t type, int32_t y_type) {
    if (const int rc = refuse_grouped(__FUNCTION__, S, T, groups, N, K, NONE, type, y_type)) return rc;
    if (S == 0 || N == 0) return 0;
    if (!offsets || !y || (K && ((T && !x) || !weight))) return refuse(__FUNCTION__, "x, weight, offsets and y are needed");
    if (!rows && T != S) return refuse(__FUNCTION__, "%llu rows of x for %llu places", (ull)T, (ull)S);
    if ((type == F8) != (x_scale != nullptr) || (type == F8) != (weight_scale != nullptr)) return refuse(__FUNCTION__, "8-bit operands and their scales belong together");
    timed record(__FUNCTION__);
    grouped_arguments a = grouped_of(S, groups, N, K, offsets);
    a.p.a = x;
    a.p.lda = ldx ? (long)ldx : (long)K;
    a.p.b = weight;
    a.p.ldb = ldw ? (long)ldw : (long)K;
    a.p.a_scale = x_scale;
    a.p.b_scale = weight_scale;
    a.p.y = y;
    return grouped_forward(__FUNCTION__, type, y_type, LINEAR, a, rows, (long)T);
}

int tiramisu_hip_grouped_gated_linear(const void *x, const void *gate_weight, const void *up_weight, const int32_t *offsets, const int32_t *rows, const float *x_scale,
                                      const float *gate_scale, const float *up_scale, void *h, void *gate, void *up, uint64_t S, uint64_t T, uint64_t groups, uint64_t N, uint64_t K,
                                      uint64_t ldx, uint64_t ldg, uint64_t ldu, int32_t activation, int32_t type, int32_t h_type) {
    if (const int rc = refuse_grouped(__FUNCTION__, S, T, groups, 2 * std::min(N, MOST), K, activation, type, h_type)) return rc;
    if (S == 0 || N == 0) return 0;
    if (!offsets || !h || (K && ((T && !x) || !gate_weight || !up_weight))) return refuse(__FUNCTION__, "x, both weights, offsets and h are needed");
    if (!rows && T != S) return refuse(__FUNCTION__, "%llu rows of x for %llu places", (ull)T, (ull)S);
    if ((gate != nullptr) != (up != nullptr)) return refuse(__FUNCTION__, "gate and up are kept together");
    if ((type == F8) != (x_scale != nullptr) || (type == F8) != (gate_scale != nullptr) || (type == F8) != (up_scale != nullptr))
        return refuse(__FUNCTION__, "8-bit operands and their scales belong together");
    timed record(__FUNCTION__);
    grouped_arguments a = grouped_of(S, groups, N, K, offsets);
    a.p.a = x;
    a.p.lda = ldx ? (long)ldx : (long)K;
    a.p.b = gate_weight;
    a.p.ldb = ldg ? (long)ldg : (long)K;
    a.p.b2 = up_weight;
    a.p.ldb2 = ldu ? (long)ldu : (long)K;
    a.p.a_scale = x_scale;
    a.p.b_scale = gate_scale;
    a.p.b2_scale = up_scale;
    a.p.y = h;
    a.p.pre = gate;
    a.p.pre2 = up;
    a.p.activation = activation;
    return grouped_forward(__FUNCTION__, type, h_type, GATED, a, rows, (long)T);
}

int tiramisu_hip_grouped_linear_backward(const void *dy, const void *x, const void *weight, const int32_t *offsets, const int32_t *rows, void *dx, void *dweight, uint64_t S,
                                         uint64_t T, uint64_t groups, uint64_t N, uint64_t K, uint64_t ldy, uint64_t ldx, uint64_t ldw, int32_t type) {
    if (const int rc = refuse_grouped(__FUNCTION__, S, T, groups, std::max(N, K), K, NONE, type, type)) return rc;
    if ((int64_t)N * 2 > MOST_ROW_BYTES) return refuse(__FUNCTION__, "N of %llu: rows of at most %lld bytes", (ull)N, (long long)MOST_ROW_BYTES);
    if (refuse_result(__FUNCTION__, N * groups + 64 * groups, K)) return 1;
    if (type == F8) return refuse(__FUNCTION__, "gradients are of float16 or bfloat16 operands");
    if (!rows && T != S) return refuse(__FUNCTION__, "%llu rows of x for %llu places", (ull)T, (ull)S);
    if (refuse_overlap(__FUNCTION__, "dy", S, N, ldy) || refuse_overlap(__FUNCTION__, "x", T, K, ldx) || refuse_overlap(__FUNCTION__, "weight", N * groups, K, ldw)) return 1;
    if (!offsets || (S && N && !dy) || (T && S && K && dweight && !x) || (N && K && dx && !weight)) return refuse(__FUNCTION__, "dy, x, weight and offsets are needed");
    if (K == 0) return 0;
    timed record(__FUNCTION__);
    call_scratch s;
    const placed_operand d = place_operand({dy, ldy ? (long)ldy : (long)N}, (long)S, (long)N, 2, true, s);
    const placed_operand w = place_operand({weight, ldw ? (long)ldw : (long)K}, dx && S ? (long)(N * groups) : 0, (long)K, 2, false, s);
    const bool gradient = dweight && N > 0;
    const planned_weight_rows xs = plan_weight_rows(x, rows, ldx ? (long)ldx : (long)K, gradient ? (long)S : 0, (long)T, (long)K, s);
    grouped_arguments a = grouped_of(S, groups, K, N, offsets), b = grouped_of(N, groups, K, 0, offsets);
    a.p.y = S > 0 ? dx : nullptr;
    b.p.y = gradient ? dweight : nullptr;
    b.p.past = groups * N * K * 2 >= PAST_THE_CACHES;
    b.rows = (int)S;
    const planned_gradients g = plan_gradients(a, b, 1, s);
    if (s.take(__FUNCTION__)) return 1;
    operand_moves moves(2);
    a.p.a = b.p.a = moves.settle(d, s);
    a.p.lda = b.p.lda = d.ld;
    a.p.b = moves.settle(w, s);
    a.p.ldb = w.ld;
    a.b_step = (long)N * w.ld;
    settle_weight_rows(xs, b, moves, s);
    b.y_step = (long)N * (long)K;
    moves.launch(__FUNCTION__);
    launch_gradients(__FUNCTION__, type, g, a, b, s);
    return 0;
}

int tiramisu_hip_grouped_gated_linear_backward(const void *dh, const void *x, const void *gate_weight, const void *up_weight, const void *gate, const void *up, const int32_t *offsets,
                                               const int32_t *rows, void *dx, void *dgate_weight, void *dup_weight, uint64_t S, uint64_t T, uint64_t groups, uint64_t N, uint64_t K,
                                               uint64_t ldh, uint64_t ldx, uint64_t ldg, uint64_t ldu, uint64_t ld_gate, uint64_t ld_up, int32_t activation, int32_t type) {
    if (const int rc = refuse_grouped(__FUNCTION__, S, T, groups, std::max(N, K), K, activation, type, type)) return rc;
    if ((int64_t)(2 * N + 16) * 2 > MOST_ROW_BYTES) return refuse(__FUNCTION__, "N of %llu: rows of at most %lld bytes", (ull)N, (long long)MOST_ROW_BYTES);
    if (refuse_result(__FUNCTION__, (2 * N + 80) * groups, K)) return 1;
    if (type == F8) return refuse(__FUNCTION__, "gradients are of float16 or bfloat16 operands");
    if (!rows && T != S) return refuse(__FUNCTION__, "%llu rows of x for %llu places", (ull)T, (ull)S);
    if (refuse_overlap(__FUNCTION__, "x", T, K, ldx) || refuse_overlap(__FUNCTION__, "gate_weight", N * groups, K, ldg) || refuse_overlap(__FUNCTION__, "up_weight", N * groups, K, ldu)) return 1;
    if (!offsets || (S && N && (!dh || !gate || !up)) || (T && S && K && N && dgate_weight && !x) || (N && K && dx && (!gate_weight || !up_weight)))
        return refuse(__FUNCTION__, "dh, x, both weights, gate, up and offsets are needed");
    if ((dgate_weight != nullptr) != (dup_weight != nullptr)) return refuse(__FUNCTION__, "gradients of both weights, or of neither");
    if (K == 0) return 0;
    timed record(__FUNCTION__);
    const long m = (long)S, n = (long)N, k = (long)K, half = (n + 7) / 8 * 8, ld = 2 * half;        // [dgate | dup] in rows of 2 x `half` elements
    // (dgate and dup are operands of two products, of 16 bits as the matrix instructions take them: kept in 32 they would be two operands each, at twice the products' work.  Gradients are off by
    // 0.0024 of their size, 0.0017 with 32 bits.)
    call_scratch s;
    const uint64_t gradient = s.want((uint64_t)std::max(1L, m) * std::max(1L, ld) * 2);
    const long of_weights = dx && m ? n * (long)groups : 0;
    const placed_operand wg = place_operand({gate_weight, ldg ? (long)ldg : k}, of_weights, k, 2, false, s), wu = place_operand({up_weight, ldu ? (long)ldu : k}, of_weights, k, 2, false, s);
    const bool weights = dgate_weight && n > 0;
    const planned_weight_rows xs = plan_weight_rows(x, rows, ldx ? (long)ldx : k, weights ? m : 0, (long)T, k, s);
    // rows of the weights' product: those of gate, up to `half` nothing, those of up
    grouped_arguments a = grouped_of(S, groups, K, N, offsets), b = grouped_of((uint64_t)(half + n), groups, K, 0, offsets);
    a.p.y = m > 0 ? dx : nullptr;
    b.p.y = weights ? dgate_weight : nullptr;
    b.p.y_below = weights ? dup_weight : nullptr;
    b.p.past = 2 * groups * N * K * 2 >= PAST_THE_CACHES;
    b.p.rows_above = (int)n;
    b.p.split_row = (int)half;
    b.rows = (int)m;
    const planned_gradients g = plan_gradients(a, b, 2, s);
    if (s.take(__FUNCTION__)) return 1;
    char *const d = (char *)s.at(gradient);
    if (m > 0 && n > 0) launch_gated_gradients(__FUNCTION__, type, {dh, gate, up, d, d + 2 * half, m, n, ldh ? (long)ldh : n, ld_gate ? (long)ld_gate : n, ld_up ? (long)ld_up : n, ld, activation});
    operand_moves moves(2);
    a.p.a = b.p.a = d;
    a.p.a_more = d + 2 * half;
    a.p.lda = b.p.lda = ld;
    a.p.b = moves.settle(wg, s);
    a.p.b_more = moves.settle(wu, s);
    a.p.ldb = wg.ld;
    a.p.ldb_more = wu.ld;
    a.b_step = n * wg.ld;
    a.b2_step = n * wu.ld;
    settle_weight_rows(xs, b, moves, s);
    b.y_step = n * k;
    moves.launch(__FUNCTION__);
    launch_gradients(__FUNCTION__, type, g, a, b, s);
    return 0;
}

int tiramisu_hip_combine_rows(const void *x, const int32_t *places, const float *weights, const void *residual, void *y, uint64_t tokens, uint64_t k, uint64_t rows, uint64_t columns,
                              uint64_t ldx, uint64_t ldr, int32_t type) {
    if (tokens > MOST || rows > MOST || columns > MOST_COLUMNS) return refuse(__FUNCTION__, "%llu tokens of %llu columns: at most 2^30 - 1 of at most 2^26", (ull)tokens, (ull)columns);
    if (k > 1024) return refuse(__FUNCTION__, "%llu rows of a token: at most 1024", (ull)k);
    if (!known_type(type, false)) return refuse(__FUNCTION__, "element type %d: float16 or bfloat16", type);
    if (tokens == 0 || columns == 0) return 0;
    if (!y || (k && !places) || (k && rows && !x)) return refuse(__FUNCTION__, "x, places and y are needed");
    timed record(__FUNCTION__);
    const long n = (long)columns, across = (n + 7) / 8, most = std::max(1L, MOST_PIECES_A_LAUNCH / across);
    for (long first = 0; first < (long)tokens; first += most) {
        const long t = std::min(most, (long)tokens - first), step = ldr ? (long)ldr : n;
        const tcombine::combine_arguments a = {x, residual ? (const char *)residual + first * step * 2 : nullptr, places + first * (long)k, weights ? weights + first * (long)k : nullptr,
                                               (char *)y + first * n * 2, t, (long)rows, n, ldx ? (long)ldx : n, step, (int)k};
        auto kernel = type == F16 ? tcombine::combine_kernel<F16> : tcombine::combine_kernel<BF16>;
        hipLaunchKernelGGL(kernel, dim3((unsigned)((across * t + 255) / 256)), dim3(256), 0, stream(), a);
        check(hipGetLastError(), __FUNCTION__);
    }
    return 0;
}

int tiramisu_hip_combine_rows_backward(const void *dy, const void *x, const int32_t *places, const int32_t *owners, const float *weights, void *dx, float *dweights, uint64_t tokens,
                                       uint64_t k, uint64_t rows, uint64_t columns, uint64_t ldy, uint64_t ldx, int32_t type) {
    if (rows > MOST || columns > MOST_COLUMNS) return refuse(__FUNCTION__, "%llu rows of %llu columns: at most 2^30 - 1 of at most 2^26", (ull)rows, (ull)columns);
    if (k > 1024) return refuse(__FUNCTION__, "%llu rows of a token: at most 1024", (ull)k);
    if (tokens > MOST || tokens * k > 1 << 25) return refuse(__FUNCTION__, "%llu tokens of %llu rows: at most 2^25 rows of all", (ull)tokens, (ull)k);
    if (!known_type(type, false)) return refuse(__FUNCTION__, "element type %d: float16 or bfloat16", type);
    // (the kernel reads places whether or not the rows have columns)
    if ((tokens && k && (!places || (columns && !dy))) || (rows && columns && dx && !owners) || (rows && columns && dweights && !x)) return refuse(__FUNCTION__, "dy, x, places and owners are needed");
    if (dweights && !weights) return refuse(__FUNCTION__, "a gradient of weights that are not given");
    const long n = (long)columns;
    if (!dweights && !(dx && n)) return 0;
    const bool wide = n > 256;
    const long choices = wide ? 4 : 16, choice_blocks = ((long)tokens * (long)k + choices - 1) / choices, blocks = choice_blocks + (dx && n ? ((long)rows + 63) / 64 : 0);
    if (blocks == 0) return 0;
    if (blocks >= 1L << 24) return refuse(__FUNCTION__, "%llu rows and %llu choices: more workgroups than a launch holds", (ull)rows, (ull)(tokens * k));
    timed record(__FUNCTION__);
    const tcombine::combine_backward_arguments a = {dy, x, places, owners, weights, n ? dx : nullptr, dweights, (long)tokens, (long)rows, n, ldy ? (long)ldy : n, ldx ? (long)ldx : n, (int)k, choice_blocks};
    auto kernel = type == F16 ? (wide ? tcombine::combine_backward_kernel<F16, 64> : tcombine::combine_backward_kernel<F16, 16>)
                              : (wide ? tcombine::combine_backward_kernel<BF16, 64> : tcombine::combine_backward_kernel<BF16, 16>);
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(256), 0, stream(), a);
    check(hipGetLastError(), __FUNCTION__);
    return 0;
}

int tiramisu_hip_quantize_groups(const void *x, void *q, uint8_t *scale, uint64_t rows, uint64_t columns, uint64_t ldx, int32_t type) {
    if (rows > MOST || columns > MOST_COLUMNS) return refuse(__FUNCTION__, "%llu rows of %llu: at most 2^30 - 1 of at most 2^26", (ull)rows, (ull)columns);
    if (!known_type(type, true)) return refuse(__FUNCTION__, "element type %d: float32, float16 or bfloat16", type);
    if (rows == 0 || columns == 0) return 0;
    if (!x || !q || !scale) return refuse(__FUNCTION__, "x, q and scale are needed");
    timed record(__FUNCTION__);
    const long n = (long)columns, step = ldx ? (long)ldx : n, groups = (n + tfour::GROUP - 1) / tfour::GROUP, most = std::max(1L, MOST_PIECES_A_LAUNCH / groups);
    auto kernel = type == F32 ? tfour::quantize_groups_kernel<F32> : type == F16 ? tfour::quantize_groups_kernel<F16> : tfour::quantize_groups_kernel<BF16>;
    for (long first = 0; first < (long)rows; first += most) {
        const long m = std::min(most, (long)rows - first);
        hipLaunchKernelGGL(kernel, dim3((unsigned)((groups * m + 255) / 256)), dim3(256), 0, stream(), (const void *)((const char *)x + first * step * bytes_of(type)), step, m, n,
                           (char *)q + first * ((n + 1) / 2), scale + first * groups);
        check(hipGetLastError(), __FUNCTION__);
    }
    return 0;
}

int tiramisu_hip_four_bit_linear(const void *x, const void *q, const uint8_t *scale, const void *bias, const void *residual, void *y, uint64_t M, uint64_t N, uint64_t K, uint64_t ldx,
                                 uint64_t ldq, uint64_t lds, uint64_t ldr, int32_t activation, int32_t type) {
    if (const int rc = refuse_product(__FUNCTION__, M, N, K, activation, type, type)) return rc;
    if (type == F8) return refuse(__FUNCTION__, "4-bit weights are multiplied with float16 or bfloat16");
    if (M == 0 || N == 0) return 0;
    if (!y || (K && (!x || !q || !scale))) return refuse(__FUNCTION__, "x, the weight, its scales and y are needed");
    timed record(__FUNCTION__);
    four_bit_arguments a = {};
    a.p = product_of((long)M, (long)N, (long)K);
    a.p.a = x;
    a.p.lda = ldx ? (long)ldx : (long)K;
    a.p.b = q;
    a.p.ldb = ldq ? (long)ldq : (long)(K + 1) / 2;
    a.scale = scale;
    a.lds = lds ? (long)lds : (long)(K + tfour::GROUP - 1) / tfour::GROUP;
    a.p.bias = bias;
    a.p.residual = residual;
    a.p.ldr = ldr ? (long)ldr : (long)N;
    a.p.y = y;
    a.p.activation = activation;
    return type == F16 ? four_bit<F16>(__FUNCTION__, LINEAR, a) : four_bit<BF16>(__FUNCTION__, LINEAR, a);
}

int tiramisu_hip_four_bit_gated_linear(const void *x, const void *gate_q, const void *up_q, const uint8_t *gate_scale, const uint8_t *up_scale, void *h, uint64_t M, uint64_t N,
                                       uint64_t K, uint64_t ldx, uint64_t ldg, uint64_t ldu, uint64_t ldgs, uint64_t ldus, int32_t activation, int32_t type) {
    if (const int rc = refuse_product(__FUNCTION__, M, N, K, activation, type, type)) return rc;
    if (type == F8) return refuse(__FUNCTION__, "4-bit weights are multiplied with float16 or bfloat16");
    if (M == 0 || N == 0) return 0;
    if (!h || (K && (!x || !gate_q || !up_q || !gate_scale || !up_scale))) return refuse(__FUNCTION__, "x, both weights, their scales and h are needed");
    timed record(__FUNCTION__);
    const long dense = (long)(K + 1) / 2, groups = (long)(K + tfour::GROUP - 1) / tfour::GROUP;
    four_bit_arguments a = {};
    a.p = product_of((long)M, (long)N, (long)K);
    a.p.a = x;
    a.p.lda = ldx ? (long)ldx : (long)K;
    a.p.b = gate_q;
    a.p.ldb = ldg ? (long)ldg : dense;
    a.p.b2 = up_q;
    a.p.ldb2 = ldu ? (long)ldu : dense;
    a.scale = gate_scale;
    a.scale_2 = up_scale;
    a.lds = ldgs ? (long)ldgs : groups;
    a.lds_2 = ldus ? (long)ldus : groups;
    a.p.y = h;
    a.p.activation = activation;
    return type == F16 ? four_bit<F16>(__FUNCTION__, GATED, a) : four_bit<BF16>(__FUNCTION__, GATED, a);
}

}  // extern "C"
