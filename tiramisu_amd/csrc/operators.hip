// Entry points of the transformer operators (include/tiramisu_hip_wrappers.h): what they refuse, which kernel a call goes to, and the launches.
// Every launch goes to the calling thread's stream.  A call plans all of its launches first, then asks for the scratch that they need, as one block, and
// launches only when it has it.
#include "operators.h"

#include <algorithm>
#include <atomic>
#include <cstdarg>
#include <cstdint>
#include <cstdio>
#include <cstdlib>

#include "../../include/tiramisu_hip_wrappers.h"
#include "kernels/linear_few_tokens.hip.h"
#include "kernels/linear_tiles.hip.h"
#include "kernels/operator_backward.hip.h"
#include "kernels/rms_norm.hip.h"
#include "kernels/target_gfx950.h"

namespace tops {
namespace {

using tiramisu_runtime::check;
using tiramisu_runtime::stream;
using tiramisu_runtime::timed;

__attribute__((format(printf, 2, 3))) int refuse(const char *fn, const char *format, ...) {
    fprintf(stderr, "Error at %s: ", fn);
    va_list args;
    va_start(args, format);
    vfprintf(stderr, format, args);
    va_end(args);
    fprintf(stderr, "\n");
    return 1;
}

constexpr uint64_t MOST = 0x3fffffff;                    // rows and columns are counted in 31 bits, with room for a tile
constexpr int64_t MOST_ROWS_A_LAUNCH = (1 << 22) - 4;    // of a workgroup of up to 1024 threads each: a launch holds fewer than 2^32 threads
constexpr int64_t MOST_PIECES_A_LAUNCH = 1LL << 31;      // of a thread each
constexpr uint64_t MOST_TILES = (1 << 23) - 1;           // of 64 x 64: the same
constexpr uint64_t MOST_COLUMNS = 1 << 26;               // of a norm: the same for the sums of the columns
constexpr long MOST_FEW_COLUMNS = 1 << 26;               // of a product of few tokens
constexpr int64_t MOST_ROW_BYTES = 1 << 22;              // of an operand with k along its rows: a tile's offsets stay below 2^31
constexpr int64_t MOST_STEP = 1 << 23;                   // elements from k to k of one with k down its columns: the same

bool known_type(int type, bool with_f32) { return type == F16 || type == BF16 || (with_f32 && type == F32); }
int bytes_of(int type) { return type == F32 ? 4 : type == F8 ? 1 : 2; }

// ---- scratch of one call: places are given out while its launches are planned, and become addresses when the block is taken.
class call_scratch {
public:
    static constexpr uint64_t NOWHERE = ~0ull;
    uint64_t want(uint64_t bytes) {
        const uint64_t place = total;
        total += (bytes + 255) / 256 * 256;
        return place;
    }
    // 0, or 1 and a message where the memory cannot be had
    int take(const char *fn) {
        if (total == 0 || (base = (char *)tiramisu_runtime::operator_scratch(total))) return 0;
        return refuse(fn, "no memory for %llu bytes of scratch", (unsigned long long)total);
    }
    void *at(uint64_t place) const { return place == NOWHERE ? nullptr : base + place; }

private:
    uint64_t total = 0;
    char *base = nullptr;
};

// ---- operands as the tiles can load them: rows that begin at multiples of 4 bytes, and strides within the limits above.  Others are
// moved to scratch, rows at multiples of 16 bytes.
struct operand { const void *p; long ld; };
bool loadable(const operand &o, int bytes, bool k_along_rows) {
    return (uintptr_t)o.p % 4 == 0 && (o.ld * bytes) % 4 == 0 && (k_along_rows ? o.ld * bytes <= MOST_ROW_BYTES : o.ld <= MOST_STEP);
}
struct placed_operand {
    operand from;
    long rows, columns;
    int bytes;
    uint64_t place;                         // NOWHERE: stays where it is
    long ld;
};
placed_operand place_operand(const operand &o, long rows, long columns, int bytes, bool k_along_rows, call_scratch &s) {
    placed_operand q = {o, rows, columns, bytes, call_scratch::NOWHERE, o.ld};
    if (rows <= 0 || columns <= 0 || loadable(o, bytes, k_along_rows)) return q;
    const long to = (columns * bytes + 15) / 16 * 16;
    q.ld = to / bytes;
    q.place = s.want((uint64_t)to * (uint64_t)rows);
    return q;
}
// its address, and the launch that moves it there
const void *settle(const char *fn, const placed_operand &q, const call_scratch &s) {
    if (q.place == call_scratch::NOWHERE) return q.from.p;
    const long to = q.ld * q.bytes;
    char *out = (char *)s.at(q.place);
    for (long first = 0, most = std::max(1L, MOST_PIECES_A_LAUNCH / (to / 16)); first < q.rows; first += most) {
        const long n = std::min(most, q.rows - first);
        const unsigned blocks = (unsigned)((to / 16 * n + 255) / 256);
        const char *in = (const char *)q.from.p + first * q.from.ld * q.bytes;
        auto kernel = q.bytes == 1 ? move_rows_kernel<1> : move_rows_kernel<2>;
        hipLaunchKernelGGL(kernel, dim3(blocks), dim3(256), 0, stream(), in, out + first * to, n, q.columns * q.bytes, q.from.ld * q.bytes, to);
    }
    check(hipGetLastError(), fn);
    return out;
}

// ---- which tile, and how many workgroups share the k of one.  A launch is modelled in microseconds: `fixed`, for every slice of 128 bytes of k `first` for the first
// round of tiles over the compute units (and `full` as far as it fills them), and for every further round `round` and `further` a slice.
// Splitting k adds a launch and the partial sums' bytes, which caches hold in part, at 5 TB/s.  Fitted to launches of 16 ... 4096 tiles of 8 ... 64 slices (tables of
// 29 configurations; rms error 6 %); us with 256 x 256, 256 x 128, 128 x 128 and 64 x 64 tiles, bf16: 4096^3 102, 115, 149, 190; 4096 x 1024 x 4096 74, 48, 35, 50;
// 1024^3 24, 15.5, 11, 7.0; 128 x 4096 x 4096 70, 45, 29, 18.  128 x 64 tiles lie between (128 x 128, 128 x 64, 64 x 64): 1024 x 2048 x 1024 bf16 10.3, 8.2, 9.4,
// 512 x 4096 x 2048 16.3, 12.9, 16.0, 2000 x 1500 x 1000 12.8, 15.8, 17.8; e4m3 9.2, 7.0, 7.2, 11.5, 8.8, 10.7 and 11.0, 11.0, 11.3.
struct tile_model { product_tile tile; int rows, columns; double fixed, first, full, round, further, pair_round, pair_slice; };
constexpr tile_model TILES_16_BITS[] = {{TILE_256, 256, 256, 9.0, 0.94, 0.5, 4.0, 1.44, 4.0, 1.44}, {TILE_256x128, 256, 128, 5.8, 0.6, 0.15, 7.0, 0.75, 3.0, 0.75},
                                        {TILE_128, 128, 128, 4.8, 0.38, 0.09, 0.8, 0.58, 0.8, 0.58}, {TILE_128x64, 128, 64, 4.0, 0.24, 0.03, 0.8, 0.32, 0.8, 0.32},
                                        {TILE_64, 64, 64, 3.5, 0.2, 0.03, 0.7, 0.155, 0.7, 0.18}};
constexpr tile_model TILES_8_BITS[] = {{TILE_256, 256, 256, 13.8, 0.8, 0.6, 9.0, 1.4, 0, 0}, {TILE_256x128, 256, 128, 9.6, 0.44, 0.24, 13.5, 0.69, 0, 0},
                                       {TILE_128, 128, 128, 7.0, 0.26, 0.24, 4.7, 0.467, 0, 0}, {TILE_128x64, 128, 64, 5.2, 0.15, 0.07, 0.9, 0.4, 0, 0},
                                       {TILE_64, 64, 64, 4.8, 0.13, 0.02, 0.7, 0.19, 0, 0}};
// (a gated layer's smallest tile is 64 x 128: 64 columns of gate and the same of up)
constexpr tile_model GATED_64_16_BITS = {TILE_64, 64, 128, 3.9, 0.27, 0.08, 0.7, 0.31, 0, 0}, GATED_64_8_BITS = {TILE_64, 64, 128, 5.4, 0.13, 0.05, 0.7, 0.3, 0, 0};
struct tile_plan { product_tile tile; int splits, slices; double cost; };
tile_plan plan_for(long M, long N, long K, int bytes, bool gated) {
    const long slices = std::max(1L, (K * bytes + 127) / 128);
    tile_plan best = {TILE_64, 0, 0, 0.0};
    double best_cost = 0;
    auto consider = [&](const tile_model &t) {
        if (gated && t.tile == TILE_128x64) return;
        const long tiles = ((M + t.rows - 1) / t.rows) * ((N * (gated ? 2 : 1) + t.columns - 1) / t.columns);
        for (long splits = 1; splits <= 16 && splits <= slices; splits++) {
            const long each = (slices + splits - 1) / splits;
            if (splits > 1 && tiles * splits > 2 * ttarget::COMPUTE_UNITS) break;
            if ((slices + each - 1) / each != splits) continue;            // (the same slices to each as with fewer)
            const double busy = (double)(tiles * splits) / ttarget::COMPUTE_UNITS, more = (double)((tiles * splits - 1) / ttarget::COMPUTE_UNITS);
            double cost = t.fixed + (double)each * (t.first + std::min(1.0, busy) * t.full) + more * (t.round + (double)each * t.further);
            if (splits > 1) cost += 5.5 + (gated ? 2.0 : 1.0) * M * N * 4 * 2 * splits / 5e6;
            if (!best.splits || cost < best_cost) { best = {t.tile, (int)splits, (int)each, cost}; best_cost = cost; }
        }
    };
    for (const tile_model &t : TILES_16_BITS)
        if (bytes == 2) consider(gated && t.tile == TILE_64 ? GATED_64_16_BITS : t);
    for (const tile_model &t : TILES_8_BITS)
        if (bytes == 1) consider(gated && t.tile == TILE_64 ? GATED_64_8_BITS : t);
    return best;
}

// Both gradients in one launch: tiles of the longer product first, then those of the other on compute units as they become free.  Modelled like one
// product, with `pair_slice` and `pair_round` for tiles of more than a round (slices of the two kinds take their time together; over 23 pairs the choices are 2 %
// behind the best ones in the mean), against the two launches one after the other (about 2 us more than their sum).  us as 256 x 256, 256 x 128, 128 x 128,
// 128 x 64, 64 x 64 tiles and apart: 4096 x 4096 x 1024 86, 62, 77, 85, 107, 73; 1024 x 4096 x 1024 73, 44, 31, 27, 31, 35; 2048^3 47, 34, 41, 46, 56, 44;
// 1000 x 700 x 500 25, 16, 11, 9.4, 7.8, 13.5.
struct pair_plan { product_tile tile; bool together, q_first; };
pair_plan plan_for_pair(long M, long N, long K, long M2, long N2, long K2) {
    pair_plan best = {TILE_64, false, false};
    double best_cost = plan_for(M, N, K, 2, false).cost + plan_for(M2, N2, K2, 2, false).cost + 2.0;
    for (const tile_model &t : TILES_16_BITS) {
        auto tiles_of = [&](long m, long n) { return ((m + t.rows - 1) / t.rows) * ((n + t.columns - 1) / t.columns); };
        const long units = ttarget::COMPUTE_UNITS, tiles[2] = {tiles_of(M, N), tiles_of(M2, N2)};
        if (tiles[0] + tiles[1] > (long)MOST_TILES / 2) continue;          // (workgroups of up to 512 threads, and those of sums)
        const double busy = std::min(1.0, (double)(tiles[0] + tiles[1]) / units);
        double each[2];
        const double slice = tiles[0] + tiles[1] <= units ? t.first + busy * t.full : t.pair_slice;
        for (int i = 0; i < 2; i++) each[i] = (double)(((i ? K2 : K) + 63) / 64) * slice + t.pair_round;
        const int a = each[0] >= each[1] ? 0 : 1, b = 1 - a;
        // whole rounds of the first kind, its last tiles, and how many of the second are done when
        const long rounds = tiles[a] / units, last = tiles[a] % units;
        const double free_at[2] = {rounds * each[a], (rounds + (last > 0)) * each[a]};
        // the earliest moment, a whole number of the second kind's tiles behind either, at which all of them are finished
        double done = 0;
        for (int from = 0; from < 2; from++)
            for (long k = 0;; k++) {
                const double when = free_at[from] + k * each[b];
                const auto finished_since = [&](double begin) { return when < begin ? 0L : (long)((when - begin) / each[b] + 1e-6); };
                if ((units - last) * finished_since(free_at[0]) + last * finished_since(free_at[1]) < tiles[b]) continue;
                done = from == 0 ? when : std::min(done, when);
                break;
            }
        done = std::max(done, free_at[1]);
        const double cost = t.fixed + done;
        if (cost < best_cost) { best = {t.tile, true, a == 1}; best_cost = cost; }
    }
    return best;
}

// A product as it will be launched; its operands' addresses and `a_more` may still be missing.  `pairs`: 2 where a second pair of operands will be added.
struct planned_product {
    int type, epilogue, y;
    product_layout layout;
    product_arguments p;
    tile_plan plan;
    uint64_t partial;
};
planned_product plan_product(int type, product_layout layout, int epilogue, int y, const product_arguments &p, int pairs, call_scratch &s) {
    planned_product q = {type, epilogue, y, layout, p, {TILE_64, 1, 0, 0.0}, call_scratch::NOWHERE};
    if (p.M == 0 || p.N == 0) return q;
    const bool gated = epilogue == GATED;
    q.plan = plan_for(p.M, p.N, (long)pairs * p.K, bytes_of(type), gated);
    if (pairs == 2 && q.plan.splits > 1) {
        // (the slices are those of both pairs, and each workgroup takes its part of either)
        q.plan.slices = (q.plan.slices + 1) / 2;
        q.plan.splits = (int)std::max(1L, ((long)p.K + 64L * q.plan.slices - 1) / (64L * q.plan.slices));
    }
    q.p.slices_per_split = q.plan.slices;
    if (q.plan.splits > 1) q.partial = s.want((uint64_t)q.plan.splits * (gated ? 2 : 1) * p.M * p.N * 4);
    return q;
}
void launch_product(const char *fn, planned_product &q, const call_scratch &s) {
    product_arguments &p = q.p;
    if (p.M == 0 || p.N == 0) return;
    p.partial = (float *)s.at(q.partial);
    if (q.type == BF16) launch_tiles_BF16(q.plan.tile, q.layout, q.epilogue, q.y, p, q.plan.splits, stream());
    else if (q.type == F16) launch_tiles_F16(q.plan.tile, q.layout, q.epilogue, q.y, p, q.plan.splits, stream());
    else launch_tiles_F8(q.plan.tile, q.layout, q.epilogue, q.y, p, q.plan.splits, stream());
    if (q.plan.splits > 1) {
        const unsigned blocks = (unsigned)(((p.N + 7L) / 8 * p.M + 255) / 256);
        auto kernel = q.epilogue == GATED ? (q.y == BF16 ? finish_kernel<BF16, GATED> : finish_kernel<F16, GATED>) : (q.y == BF16 ? finish_kernel<BF16, LINEAR> : finish_kernel<F16, LINEAR>);
        hipLaunchKernelGGL(kernel, dim3(blocks), dim3(256), 0, stream(), p, q.plan.splits);
        check(hipGetLastError(), fn);
    }
}

template <int E>
void launch_sums(const char *fn, const column_sums &a) {
    hipLaunchKernelGGL(sum_parts_kernel<E>, dim3((unsigned)((a.columns + SUM_COLUMNS - 1) / SUM_COLUMNS)), dim3(1024), 0, stream(), a);
    check(hipGetLastError(), fn);
}

// p: gradient of the input, q: of the weights; what is not asked for has no place for its result.  sums: the bias's gradient, which the one launch of both
// gradients takes along (4096 x 4096 x 1024: 64 us; as a launch of their own ahead of it 63 and 4.7).
struct planned_gradients {
    int type;
    pair_plan pair;
    planned_product p, q;
};
planned_gradients plan_gradients(int type, const product_arguments &p, int pairs, const product_arguments &q, call_scratch &s) {
    planned_gradients g = {type, {TILE_64, false, false}, {}, {}};
    g.p.p = p;
    g.q.p = q;
    if (p.y && q.y && p.M && p.N && q.M && q.N) g.pair = plan_for_pair(p.M, p.N, (long)pairs * p.K, q.M, q.N, q.K);
    if (g.pair.together) return g;
    if (p.y) g.p = plan_product(type, INPUT_GRADIENT, LINEAR, type, p, pairs, s);
    if (q.y) g.q = plan_product(type, WEIGHT_GRADIENT, LINEAR, type, q, 1, s);
    return g;
}
int launch_gradients(const char *fn, planned_gradients &g, const column_sums &sums, const call_scratch &s) {
    if (g.pair.together) {
        (g.type == BF16 ? launch_gradients_BF16 : launch_gradients_F16)(g.pair.tile, g.pair.q_first, g.p.p, g.q.p, sums, stream());
        return 0;
    }
    if (sums.parts) g.type == BF16 ? launch_sums<BF16>(fn, sums) : launch_sums<F16>(fn, sums);
    if (g.p.p.y) launch_product(fn, g.p, s);
    if (g.q.p.y) launch_product(fn, g.q, s);
    return 0;
}

// Rows of x that the kernel of few tokens (linear_few_tokens.hip.h) takes at most, and what a call of it takes: the weights' bytes at what memory gives, or what a
// compute unit takes in of weights and x for the workgroups it runs, the other hidden but for a part.  The tiles are held to the weights' bytes too, at
// the rates they reached.  us as the kernel of few tokens / as tiles, for 1, 16 and 64 rows: bf16 4096 x 4096 8.7, 9.9, 20.6 / 11.2,
// 11.7, 13.1; 8192 x 2048 9.1, 10.5, 20.7 / 10.8, 10.7, 11.2; 16384 x 4096 25, 37, 83 / 33, 33, 34; gated 4096 x 4096 14.3, 14.6, 24.6 / 16.3, 16.9, 19.5,
// 8192 x 2048 15.1, 16.6, 25.8 / 13.1, 13.4, 14.0; e4m3 4096 x 4096 6.6, 7.6, 12.0 / 11.2, 11.0, 11.6, 16384 x 4096 17.7, 20.2, 38.3 / 12.8, 12.7, 14.0.
constexpr long FEW_TOKENS = 64;
double few_tokens_cost(long M, long N, long K, int bytes, bool gated) {
    const double parts = gated ? 2 : 1, row = (double)K * bytes, rounds = (double)((N + 16L * ttarget::COMPUTE_UNITS - 1) / (16L * ttarget::COMPUTE_UNITS));
    const double memory = parts * N * row / 5.4e6, unit = rounds * (16 * parts + M) * row / 39e3;
    return 2.5 + std::max(memory, unit) + 0.1 * std::min(memory, unit) + (rounds - 1);
}
double tiles_cost(const tile_plan &plan, long N, long K, int bytes, bool gated, int moved) {
    const double rate = !gated && bytes == 2 ? 4.4e6 : gated && N < 64L * ttarget::COMPUTE_UNITS / 2 ? 5.0e6 : 6.2e6;
    return std::max(plan.cost, 3.0 + (gated ? 2.0 : 1.0) * N * K * bytes / rate) + 3.5 * moved;
}

template <int E, int Y, int EPILOGUE, int TILES>
void launch_few(const char *fn, const product_arguments &p) {
    auto kernel = few_tokens_kernel<E, Y, EPILOGUE, TILES>;
    hipLaunchKernelGGL(kernel, dim3((unsigned)((p.N + FEW_ROWS - 1L) / FEW_ROWS)), dim3(64 * FEW_WAVES), few_lds_bytes(TILES, EPILOGUE == GATED), stream(), p);
    check(hipGetLastError(), fn);
}
template <int E, int Y, int EPILOGUE>
void launch_few(const char *fn, const product_arguments &p) {
    if (p.M <= 16) launch_few<E, Y, EPILOGUE, 1>(fn, p);
    else if (p.M <= 32) launch_few<E, Y, EPILOGUE, 2>(fn, p);
    else launch_few<E, Y, EPILOGUE, 4>(fn, p);
}
template <int EPILOGUE>
void launch_few(const char *fn, int type, int y, const product_arguments &p) {
    if (type == BF16) launch_few<BF16, BF16, EPILOGUE>(fn, p);
    else if (type == F16) launch_few<F16, F16, EPILOGUE>(fn, p);
    else if (y == BF16) launch_few<F8, BF16, EPILOGUE>(fn, p);
    else launch_few<F8, F16, EPILOGUE>(fn, p);
}

// A forward product: few tokens, or tiles
int forward(const char *fn, int type, int y, int epilogue, product_arguments p) {
    if (p.M == 0 || p.N == 0) return 0;
    const int bytes = bytes_of(type);
    const bool gated = epilogue == GATED;
    if (p.M <= FEW_TOKENS && p.K > 0 && p.N <= MOST_FEW_COLUMNS) {
        const int moved = !loadable({p.a, p.lda}, bytes, true) + !loadable({p.b, p.ldb}, bytes, true) + (gated && !loadable({p.b2, p.ldb2}, bytes, true));
        if (few_tokens_cost(p.M, p.N, p.K, bytes, gated) <= tiles_cost(plan_for(p.M, p.N, p.K, bytes, gated), p.N, p.K, bytes, gated, moved)) {
            gated ? launch_few<GATED>(fn, type, y, p) : launch_few<LINEAR>(fn, type, y, p);
            return 0;
        }
    }
    call_scratch s;
    const placed_operand a = place_operand({p.a, p.lda}, p.M, p.K, bytes, true, s), b = place_operand({p.b, p.ldb}, p.N, p.K, bytes, true, s),
                         b2 = place_operand({p.b2, p.ldb2}, gated ? p.N : 0, p.K, bytes, true, s);
    p.lda = a.ld;
    p.ldb = b.ld;
    p.ldb2 = b2.ld;
    planned_product q = plan_product(type, FORWARD, epilogue, y, p, 1, s);
    if (s.take(fn)) return 1;
    q.p.a = settle(fn, a, s);
    q.p.b = settle(fn, b, s);
    q.p.b2 = settle(fn, b2, s);
    launch_product(fn, q, s);
    return 0;
}

// ---- rows
template <int E, int Y>
void launch_norm(const char *fn, const norm_arguments &a) {
    constexpr int N = E == F32 ? 4 : 8;
    const long pieces = (a.columns + N - 1) / N;
    auto go = [&](auto kernel, int threads, int rows) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)((a.rows + rows - 1) / rows)), dim3(threads), 0, stream(), a);
    };
    // (A wavefront to a row of up to 256 pieces, without a barrier, is no faster: 2000 x 1430 float16 10.5 us, with 256 threads 9.2.)
    if (pieces <= 64) go(rms_norm_kernel<E, Y, 64, 1, true>, 256, 4);
    else if (pieces <= 256) go(rms_norm_kernel<E, Y, 256, 1, true>, 256, 1);
    else if (pieces <= 512) go(rms_norm_kernel<E, Y, 256, 2, true>, 256, 1);
    else if (pieces <= 1024) go(rms_norm_kernel<E, Y, 256, 4, true>, 256, 1);
    else if (pieces <= 4096) go(rms_norm_kernel<E, Y, 1024, 4, true>, 1024, 1);
    else go(rms_norm_kernel<E, Y, 1024, 1, false>, 1024, 1);
    check(hipGetLastError(), fn);
}
int norm(const char *fn, int type, int y, norm_arguments a) {
    const long all = a.rows, step = bytes_of(type), step_y = bytes_of(y);
    auto moved = [](auto *p, long bytes) { return p ? (decltype(p))((uintptr_t)p + bytes) : p; };
    for (long first = 0; first < all; first += MOST_ROWS_A_LAUNCH) {
        norm_arguments part = a;
        part.rows = std::min(MOST_ROWS_A_LAUNCH, all - first);
        part.x = moved(a.x, first * a.ldx * step);
        part.residual = moved(a.residual, first * a.ldr * step);
        part.y = moved(a.y, first * a.columns * step_y);
        part.sum = moved(a.sum, first * a.columns * step);
        part.scale = moved(a.scale, first * 4);
        part.rstd = moved(a.rstd, first * 4);
        if (type == F32) y == F8 ? launch_norm<F32, F8>(fn, part) : launch_norm<F32, F32>(fn, part);
        else if (type == F16) y == F8 ? launch_norm<F16, F8>(fn, part) : launch_norm<F16, F16>(fn, part);
        else y == F8 ? launch_norm<BF16, F8>(fn, part) : launch_norm<BF16, BF16>(fn, part);
    }
    return 0;
}

template <int E>
int launch_norm_backward(const char *fn, norm_backward_arguments a, void *dweight) {
    constexpr int N = E == F32 ? 4 : 8;
    const long pieces = (a.columns + N - 1) / N;
    call_scratch s;
    auto sums_of = [&](long parts) {
        a.parts = (int)std::max(1L, parts);
        const uint64_t place = s.want((uint64_t)a.parts * a.columns * 4);
        if (s.take(fn)) return false;
        a.partial = (float *)s.at(place);
        return true;
    };
    // workgroups: enough to cover the way to memory, few enough that their sums are little beside the rows
    auto go = [&](auto kernel, int threads, int teams, long most) {
        if (!sums_of(std::min((a.rows + teams - 1) / teams, most))) return false;
        hipLaunchKernelGGL(kernel, dim3((unsigned)a.parts), dim3(threads), 0, stream(), a);
        return true;
    };
    auto go_long = [&] {
        if (!sums_of(std::min(a.rows, 64L))) return false;
        for (a.first = 0; a.first < a.rows; a.first += MOST_ROWS_A_LAUNCH)
            hipLaunchKernelGGL(rms_norm_backward_long_rows_kernel<E>, dim3((unsigned)std::min(MOST_ROWS_A_LAUNCH, a.rows - a.first)), dim3(1024), 0, stream(), a);
        hipLaunchKernelGGL(rms_norm_backward_long_columns_kernel<E>, dim3((unsigned)((a.columns + 255) / 256), (unsigned)a.parts), dim3(256), 0, stream(), a);
        return true;
    };
    const bool launched = pieces <= 64    ? go(rms_norm_backward_kernel<E, 64, 1>, 512, 8, 512)
                          : pieces <= 128  ? go(rms_norm_backward_kernel<E, 64, 2>, 512, 8, 512)
                          : pieces <= 192  ? go(rms_norm_backward_kernel<E, 64, 3>, 512, 8, 256)
                          : pieces <= 256  ? go(rms_norm_backward_kernel<E, 64, 4>, 512, 8, 256)
                          : pieces <= 512  ? go(rms_norm_backward_kernel<E, 256, 2>, 256, 1, 768)
                          : pieces <= 1024 ? go(rms_norm_backward_kernel<E, 256, 4>, 256, 1, 512)
                          : pieces <= 2048 ? go(rms_norm_backward_kernel<E, 512, 4>, 512, 1, 256)
                                           : go_long();
    if (!launched) return 1;
    check(hipGetLastError(), fn);
    launch_sums<E>(fn, {a.partial, dweight, a.columns, a.parts});
    return 0;
}

// How the launch of dz is divided: `across` threads along a row and columns of workgroups, rows of a chunk and chunks
struct activation_backward_plan { int across; long columns, rows; int chunks; };
activation_backward_plan plan_activation_backward(long M, long N) {
    activation_backward_plan plan = {1, 0, 0, 0};
    while (plan.across < 64 && plan.across * 8 < N) plan.across *= 2;
    plan.columns = (N + 8L * plan.across - 1) / (8L * plan.across);
    // workgroups: one row to a thread where there are few, and few enough that their sums are little beside the rows
    const long down = 256 / plan.across, chunks = std::max(1L, std::min((M + down - 1) / down, std::min(256L, std::max(1L, 1024 / plan.columns))));
    plan.rows = std::max(1L, (M + chunks - 1) / chunks);
    plan.chunks = (int)std::max(1L, (M + plan.rows - 1) / plan.rows);
    return plan;
}
// dz, and what the bias's gradient is the sums of; what is null is not computed
template <int E>
column_sums launch_activation_backward(const char *fn, activation_backward_arguments a, const activation_backward_plan &plan, void *dbias) {
    a.across = plan.across;
    a.rows = plan.rows;
    hipLaunchKernelGGL(activation_backward_kernel<E>, dim3((unsigned)plan.columns, (unsigned)plan.chunks), dim3(256), 0, stream(), a);
    check(hipGetLastError(), fn);
    return {a.partial, dbias, a.N, dbias ? plan.chunks : 0};
}

product_arguments product_of(long M, long N, long K) {
    product_arguments p = {};
    p.M = (int)M;
    p.N = (int)N;
    p.K = (int)K;
    p.rows_above = p.split_row = p.M;
    return p;
}

int refuse_result(const char *fn, uint64_t rows, uint64_t columns) {
    if (((rows + 63) / 64) * ((columns + 63) / 64) <= MOST_TILES) return 0;
    return refuse(fn, "result of %llu x %llu: more tiles than a launch holds", (unsigned long long)rows, (unsigned long long)columns);
}
// An operand whose rows overlap has no end behind its last row that the tiles could stop at where k runs down its columns.
int refuse_overlap(const char *fn, const char *name, uint64_t rows, uint64_t columns, uint64_t ld) {
    if (rows <= 1 || ld == 0 || ld >= columns) return 0;
    return refuse(fn, "%s: rows of %llu are %llu apart", name, (unsigned long long)columns, (unsigned long long)ld);
}
// What both products refuse alike
int refuse_product(const char *fn, uint64_t M, uint64_t N, uint64_t K, int activation, int type, int y) {
    if (M > MOST || N > MOST || K > MOST) return refuse(fn, "product of %llu x %llu x %llu: dimensions of at most 2^30 - 1", (unsigned long long)M, (unsigned long long)N, (unsigned long long)K);
    if ((int64_t)K * bytes_of(type) > MOST_ROW_BYTES) return refuse(fn, "K of %llu: rows of at most %lld bytes", (unsigned long long)K, (long long)MOST_ROW_BYTES);
    if (activation < NONE || activation > SILU) return refuse(fn, "activation %d is not known", activation);
    if (!known_type(type, false) && type != F8) return refuse(fn, "element type %d: float16, bfloat16 or float8_e4m3", type);
    if (type == F8 ? !known_type(y, false) : y != type) return refuse(fn, "results of type %d from operands of type %d", y, type);
    return refuse_result(fn, M, N);
}

}  // namespace
}  // namespace tops

using namespace tops;

extern "C" {

int tiramisu_hip_rms_norm(const void *x, const void *residual, const void *weight, void *y, void *sum, float *scale, float *rstd, uint64_t rows,
                          uint64_t columns, uint64_t ldx, uint64_t ldr, float eps, int32_t type, int32_t y_type) {
    if (rows > MOST || columns > MOST_COLUMNS) return refuse(__FUNCTION__, "%llu rows of %llu: at most 2^30 - 1 of at most 2^26", (unsigned long long)rows, (unsigned long long)columns);
    if (!known_type(type, true)) return refuse(__FUNCTION__, "element type %d: float32, float16 or bfloat16", type);
    if (y_type != type && y_type != F8) return refuse(__FUNCTION__, "results of type %d from rows of type %d", y_type, type);
    if (rows == 0) return 0;
    if (columns && (!x || !weight || !y)) return refuse(__FUNCTION__, "x, weight and y are needed");
    if ((residual != nullptr) != (sum != nullptr)) return refuse(__FUNCTION__, "a residual and a place for the sum belong together");
    if ((y_type == F8) != (scale != nullptr)) return refuse(__FUNCTION__, "8-bit results and a place for their scales belong together");
    if (columns == 0) {
        if (!scale && !rstd) return 0;
        weight = scale ? scale : rstd;                       // (of no elements, and not read)
    }
    timed record(__FUNCTION__);
    const norm_arguments a = {x, residual, weight, y, sum, scale, rstd, (long)rows, (long)columns, ldx ? (long)ldx : (long)columns, ldr ? (long)ldr : (long)columns, eps};
    return norm(__FUNCTION__, type, y_type, a);
}

int tiramisu_hip_quantize_rows(const void *x, void *q, float *scale, uint64_t rows, uint64_t columns, uint64_t ldx, int32_t type) {
    if (rows > MOST || columns > MOST_COLUMNS) return refuse(__FUNCTION__, "%llu rows of %llu: at most 2^30 - 1 of at most 2^26", (unsigned long long)rows, (unsigned long long)columns);
    if (!known_type(type, true)) return refuse(__FUNCTION__, "element type %d: float32, float16 or bfloat16", type);
    if (rows == 0) return 0;
    if ((columns && (!x || !q)) || !scale) return refuse(__FUNCTION__, "x, q and scale are needed");
    timed record(__FUNCTION__);
    const norm_arguments a = {x, nullptr, nullptr, q, nullptr, scale, nullptr, (long)rows, (long)columns, ldx ? (long)ldx : (long)columns, 0, 0.f};
    return norm(__FUNCTION__, type, F8, a);
}

int tiramisu_hip_rms_norm_backward(const void *dy, const void *sum, const void *weight, const float *rstd, const void *dsum, void *dx, void *dweight,
                                   uint64_t rows, uint64_t columns, uint64_t ldy, uint64_t lds, uint64_t ldd, int32_t type) {
    if (rows > MOST || columns > MOST_COLUMNS) return refuse(__FUNCTION__, "%llu rows of %llu: at most 2^30 - 1 of at most 2^26", (unsigned long long)rows, (unsigned long long)columns);
    if (!known_type(type, true)) return refuse(__FUNCTION__, "element type %d: float32, float16 or bfloat16", type);
    if (columns == 0) return 0;
    if (!dweight || !weight || (rows && (!dy || !sum || !rstd || !dx))) return refuse(__FUNCTION__, "dy, sum, weight, rstd, dx and dweight are needed");
    timed record(__FUNCTION__);
    const norm_backward_arguments a = {dy, sum, weight, dsum, rstd, dx, nullptr, (long)rows, (long)columns, ldy ? (long)ldy : (long)columns,
                                       lds ? (long)lds : (long)columns, ldd ? (long)ldd : (long)columns, 0, 0};
    return type == F32 ? launch_norm_backward<F32>(__FUNCTION__, a, dweight) : type == F16 ? launch_norm_backward<F16>(__FUNCTION__, a, dweight) : launch_norm_backward<BF16>(__FUNCTION__, a, dweight);
}

int tiramisu_hip_linear(const void *x, const void *weight, const void *bias, const void *residual, const float *x_scale, const float *weight_scale, void *y,
                        void *pre, uint64_t M, uint64_t N, uint64_t K, uint64_t ldx, uint64_t ldw, uint64_t ldr, int32_t activation, int32_t type,
                        int32_t y_type) {
    if (const int rc = refuse_product(__FUNCTION__, M, N, K, activation, type, y_type)) return rc;
    if (M == 0 || N == 0) return 0;
    if (!y || (K && (!x || !weight))) return refuse(__FUNCTION__, "x, weight and y are needed");
    if ((type == F8) != (x_scale != nullptr) || (type == F8) != (weight_scale != nullptr)) return refuse(__FUNCTION__, "8-bit operands and their scales belong together");
    timed record(__FUNCTION__);
    product_arguments p = product_of((long)M, (long)N, (long)K);
    p.a = x;
    p.lda = ldx ? (long)ldx : (long)K;
    p.b = weight;
    p.ldb = ldw ? (long)ldw : (long)K;
    p.bias = bias;
    p.residual = residual;
    p.ldr = ldr ? (long)ldr : (long)N;
    p.a_scale = x_scale;
    p.b_scale = weight_scale;
    p.y = y;
    p.pre = pre;
    p.activation = activation;
    return forward(__FUNCTION__, type, y_type, LINEAR, p);
}

int tiramisu_hip_gated_linear(const void *x, const void *gate_weight, const void *up_weight, const float *x_scale, const float *gate_scale,
                              const float *up_scale, void *h, void *gate, void *up, uint64_t M, uint64_t N, uint64_t K, uint64_t ldx, uint64_t ldg,
                              uint64_t ldu, int32_t activation, int32_t type, int32_t h_type) {
    if (const int rc = refuse_product(__FUNCTION__, M, N, K, activation, type, h_type)) return rc;
    if (M == 0 || N == 0) return 0;
    if (!h || (K && (!x || !gate_weight || !up_weight))) return refuse(__FUNCTION__, "x, both weights and h are needed");
    if ((gate != nullptr) != (up != nullptr)) return refuse(__FUNCTION__, "gate and up are kept together");
    if ((type == F8) != (x_scale != nullptr) || (type == F8) != (gate_scale != nullptr) || (type == F8) != (up_scale != nullptr))
        return refuse(__FUNCTION__, "8-bit operands and their scales belong together");
    timed record(__FUNCTION__);
    product_arguments p = product_of((long)M, (long)N, (long)K);
    p.a = x;
    p.lda = ldx ? (long)ldx : (long)K;
    p.b = gate_weight;
    p.ldb = ldg ? (long)ldg : (long)K;
    p.b2 = up_weight;
    p.ldb2 = ldu ? (long)ldu : (long)K;
    p.a_scale = x_scale;
    p.b_scale = gate_scale;
    p.b2_scale = up_scale;
    p.y = h;
    p.pre = gate;
    p.pre2 = up;
    p.activation = activation;
    return forward(__FUNCTION__, type, h_type, GATED, p);
}

int tiramisu_hip_linear_backward(const void *dy, const void *x, const void *weight, const void *pre, void *dx, void *dweight, void *dbias, uint64_t M,
                                 uint64_t N, uint64_t K, uint64_t ldy, uint64_t ldx, uint64_t ldw, uint64_t ldp, int32_t activation, int32_t type) {
    if (const int rc = refuse_product(__FUNCTION__, M, N, K, activation, type, type)) return rc;
    if ((int64_t)N * 2 > MOST_ROW_BYTES) return refuse(__FUNCTION__, "N of %llu: rows of at most %lld bytes", (unsigned long long)N, (long long)MOST_ROW_BYTES);
    if (refuse_result(__FUNCTION__, M, K) || refuse_result(__FUNCTION__, N, K)) return 1;
    if (type == F8) return refuse(__FUNCTION__, "gradients are of float16 or bfloat16 operands");
    if (refuse_overlap(__FUNCTION__, "dy", M, N, ldy) || refuse_overlap(__FUNCTION__, "x", M, K, ldx) || refuse_overlap(__FUNCTION__, "weight", N, K, ldw)) return 1;
    if ((activation != NONE) != (pre != nullptr)) return refuse(__FUNCTION__, "an activation and the sums ahead of it belong together");
    if ((M && N && !dy) || (M && K && dweight && !x) || (N && K && dx && !weight)) return refuse(__FUNCTION__, "dy, x and weight are needed");
    timed record(__FUNCTION__);
    const long m = (long)M, n = (long)N, k = (long)K;
    const bool activated = activation != NONE && n > 0, elementwise = n > 0 && (activated || dbias);
    call_scratch s;
    // the gradient ahead of the activation; without one it is dy, moved only where the tiles cannot load it
    const long ldz = (n + 7) / 8 * 8;
    const uint64_t gradient = activated ? s.want((uint64_t)std::max(1L, m) * ldz * 2) : call_scratch::NOWHERE;
    const placed_operand moved_dy = place_operand({dy, ldy ? (long)ldy : n}, activated ? 0 : m, n, 2, true, s);
    const activation_backward_plan rows = elementwise ? plan_activation_backward(m, n) : activation_backward_plan();
    const uint64_t partial = elementwise && dbias ? s.want((uint64_t)rows.chunks * n * 4) : call_scratch::NOWHERE;
    const placed_operand w = place_operand({weight, ldw ? (long)ldw : k}, dx ? n : 0, k, 2, false, s), xs = place_operand({x, ldx ? (long)ldx : k}, dweight ? m : 0, k, 2, false, s);
    product_arguments p = product_of(m, k, n), q = product_of(n, k, m);
    p.lda = q.lda = activated ? ldz : moved_dy.ld;
    p.ldb = w.ld;
    q.ldb = xs.ld;
    p.y = dx;
    q.y = dweight;
    planned_gradients g = plan_gradients(type, p, 1, q, s);
    if (s.take(__FUNCTION__)) return 1;
    column_sums sums = {};
    if (elementwise) {
        const activation_backward_arguments a = {dy, activated ? pre : nullptr, s.at(gradient), (float *)s.at(partial), m, n, ldy ? (long)ldy : n, ldp ? (long)ldp : n, ldz, 0, activation, 0};
        sums = type == F16 ? launch_activation_backward<F16>(__FUNCTION__, a, rows, dbias) : launch_activation_backward<BF16>(__FUNCTION__, a, rows, dbias);
    }
    g.p.p.a = g.q.p.a = activated ? s.at(gradient) : settle(__FUNCTION__, moved_dy, s);
    g.p.p.b = settle(__FUNCTION__, w, s);
    g.q.p.b = settle(__FUNCTION__, xs, s);
    return launch_gradients(__FUNCTION__, g, sums, s);
}

int tiramisu_hip_gated_linear_backward(const void *dh, const void *x, const void *gate_weight, const void *up_weight, const void *gate, const void *up,
                                       void *dx, void *dgate_weight, void *dup_weight, uint64_t M, uint64_t N, uint64_t K, uint64_t ldh, uint64_t ldx,
                                       uint64_t ldg, uint64_t ldu, uint64_t ld_gate, uint64_t ld_up, int32_t activation, int32_t type) {
    if (const int rc = refuse_product(__FUNCTION__, M, N, K, activation, type, type)) return rc;
    if ((int64_t)(2 * N + 16) * 2 > MOST_ROW_BYTES) return refuse(__FUNCTION__, "N of %llu: rows of at most %lld bytes", (unsigned long long)N, (long long)MOST_ROW_BYTES);
    if (refuse_result(__FUNCTION__, M, K) || refuse_result(__FUNCTION__, 2 * N + 16, K)) return 1;
    if (type == F8) return refuse(__FUNCTION__, "gradients are of float16 or bfloat16 operands");
    if (refuse_overlap(__FUNCTION__, "x", M, K, ldx) || refuse_overlap(__FUNCTION__, "gate_weight", N, K, ldg) || refuse_overlap(__FUNCTION__, "up_weight", N, K, ldu)) return 1;
    if ((M && N && (!dh || !gate || !up)) || (M && K && N && !x) || (N && K && (!gate_weight || !up_weight))) return refuse(__FUNCTION__, "dh, x, both weights, gate and up are needed");
    if ((dgate_weight != nullptr) != (dup_weight != nullptr)) return refuse(__FUNCTION__, "gradients of both weights, or of neither");
    timed record(__FUNCTION__);
    const long m = (long)M, n = (long)N, k = (long)K;
    // [dgate | dup] in rows of 2 x `half` elements
    const long half = (n + 7) / 8 * 8, ld = 2 * half;
    call_scratch s;
    const uint64_t gradient = s.want((uint64_t)std::max(1L, m) * std::max(1L, ld) * 2);
    const placed_operand wg = place_operand({gate_weight, ldg ? (long)ldg : k}, dx ? n : 0, k, 2, false, s), wu = place_operand({up_weight, ldu ? (long)ldu : k}, dx ? n : 0, k, 2, false, s),
                         xs = place_operand({x, ldx ? (long)ldx : k}, dgate_weight && n > 0 ? m : 0, k, 2, false, s);
    product_arguments p = product_of(m, k, n), q = product_of(half + n, k, m);
    p.lda = q.lda = ld;
    p.ldb = wg.ld;
    p.ldb_more = wu.ld;
    p.y = dx;
    if (dgate_weight && n > 0) {
        // rows of the product: those of gate, up to `half` nothing, those of up
        q.ldb = xs.ld;
        q.y = dgate_weight;
        q.y_below = dup_weight;
        q.rows_above = (int)n;
        q.split_row = (int)half;
    }
    planned_gradients g = plan_gradients(type, p, 2, q, s);
    if (s.take(__FUNCTION__)) return 1;
    char *d = (char *)s.at(gradient);
    if (m > 0 && n > 0) {
        const gated_backward_arguments a = {dh, gate, up, d, d + 2 * half, m, n, ldh ? (long)ldh : n, ld_gate ? (long)ld_gate : n, ld_up ? (long)ld_up : n, ld, activation};
        const unsigned blocks = (unsigned)((half / 8 * m + 255) / 256);
        if (type == F16) hipLaunchKernelGGL(gated_backward_kernel<F16>, dim3(blocks), dim3(256), 0, stream(), a);
        else hipLaunchKernelGGL(gated_backward_kernel<BF16>, dim3(blocks), dim3(256), 0, stream(), a);
        check(hipGetLastError(), __FUNCTION__);
    }
    g.p.p.a = g.q.p.a = d;
    g.p.p.a_more = d + 2 * half;
    g.p.p.b = settle(__FUNCTION__, wg, s);
    g.p.p.b_more = settle(__FUNCTION__, wu, s);
    g.q.p.b = settle(__FUNCTION__, xs, s);
    return launch_gradients(__FUNCTION__, g, {}, s);
}

float *tiramisu_hip_no_buffer(void) { return nullptr; }       // (a pointer that is also one to scales)

int tiramisu_hip_require(int32_t status) {
    if (status != 0) exit(1);
    return 0;
}

}  // extern "C"
