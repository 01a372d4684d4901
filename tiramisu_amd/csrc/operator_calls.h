// What the entry points of the operators share on the host (operators.hip, expert_operators.hip): refusals, limits, the scratch of a call, operands that
// have to be moved, and what operators.hip plans and launches for the others.
#ifndef TIRAMISU_AMD_OPERATOR_CALLS_H
#define TIRAMISU_AMD_OPERATOR_CALLS_H
#include "operators.h"

#include <cstdarg>
#include <cstdint>
#include <cstdio>

#include "kernels/linear_tiles.hip.h"

namespace tops {

__attribute__((format(printf, 2, 3))) inline int refuse(const char *fn, const char *format, ...) {
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

// Gradients of weights of so many bytes in all go past the caches: smaller ones are still there for the optimiser that reads them next (backward pass and its reader, which adds them
// to 32-bit weights, us past the caches / through them, bf16: 4 MB 32.2 / 30.3, 17 MB 85.7 / 84.8, 34 MB 93.1 / 91.3, copied instead 78.1 / 75.8, 67 MB copied 227.9 / 223.8), larger ones only
// put operands out of them (134 MB 511.9 / 521.5, 268 MB 657.0 / 679.5, those of 32 groups without a reader 356 / 369).
constexpr uint64_t PAST_THE_CACHES = 1 << 27;

inline bool known_type(int type, bool with_f32) { return type == F16 || type == BF16 || (with_f32 && type == F32); }
inline int bytes_of(int type) { return type == F32 ? 4 : type == F8 ? 1 : 2; }

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
inline bool loadable(const operand &o, int bytes, bool k_along_rows) {
    return (uintptr_t)o.p % 4 == 0 && (o.ld * bytes) % 4 == 0 && (k_along_rows ? o.ld * bytes <= MOST_ROW_BYTES : o.ld <= MOST_STEP);
}
struct placed_operand {
    operand from;
    long rows, columns;
    int bytes;
    uint64_t place;                         // NOWHERE: stays where it is
    long ld;
};
inline placed_operand place_operand(const operand &o, long rows, long columns, int bytes, bool k_along_rows, call_scratch &s) {
    placed_operand q = {o, rows, columns, bytes, call_scratch::NOWHERE, o.ld};
    if (rows <= 0 || columns <= 0 || loadable(o, bytes, k_along_rows)) return q;
    const long to = (columns * bytes + 15) / 16 * 16;
    q.ld = to / bytes;
    q.place = s.want((uint64_t)to * (uint64_t)rows);
    return q;
}
// its address, and the launch that moves it there
const void *settle(const char *fn, const placed_operand &q, const call_scratch &s);

// ---- a product on tiles
struct tile_plan { product_tile tile; int splits, slices; double cost; };
// A product as it will be launched; its operands' addresses and `a_more` may still be missing.  `pairs`: 2 where a second pair of operands will be added.
struct planned_product {
    int type, epilogue, y;
    product_layout layout;
    product_arguments p;
    tile_plan plan;
    uint64_t partial;
};
inline product_arguments product_of(long M, long N, long K) {
    product_arguments p = {};
    p.M = (int)M;
    p.N = (int)N;
    p.K = (int)K;
    p.rows_above = p.split_row = p.M;
    return p;
}


// A forward product on tiles: its operands, moved where they have to be, and the launch (p.a, p.b and p.b2 may be scratch, which has its address later: f.a.from.p ... then).
struct planned_forward {
    placed_operand a, b, b2;
    planned_product q;
};
planned_forward plan_forward(int type, int y, int epilogue, product_arguments p, call_scratch &s);
void launch_forward(const char *fn, planned_forward &f, const call_scratch &s);
// What a launch of so many tiles is modelled to take, in microseconds; slices: of 128 bytes of k
double tile_launch_cost(product_tile tile, long tiles, long slices, int bytes, bool gated);
// dgate and dup of a gated layer, next to each other in rows of a.ld elements
void launch_gated_gradients(const char *fn, int type, const struct gated_backward_arguments &a);

// ---- refusals
inline int refuse_result(const char *fn, uint64_t rows, uint64_t columns) {
    if (((rows + 63) / 64) * ((columns + 63) / 64) <= MOST_TILES) return 0;
    return refuse(fn, "result of %llu x %llu: more tiles than a launch holds", (unsigned long long)rows, (unsigned long long)columns);
}
// An operand whose rows overlap has no end behind its last row that the tiles could stop at where k runs down its columns.
inline int refuse_overlap(const char *fn, const char *name, uint64_t rows, uint64_t columns, uint64_t ld) {
    if (rows <= 1 || ld == 0 || ld >= columns) return 0;
    return refuse(fn, "%s: rows of %llu are %llu apart", name, (unsigned long long)columns, (unsigned long long)ld);
}
// What both products refuse alike
inline int refuse_product(const char *fn, uint64_t M, uint64_t N, uint64_t K, int activation, int type, int y) {
    if (M > MOST || N > MOST || K > MOST) return refuse(fn, "product of %llu x %llu x %llu: dimensions of at most 2^30 - 1", (unsigned long long)M, (unsigned long long)N, (unsigned long long)K);
    if ((int64_t)K * bytes_of(type) > MOST_ROW_BYTES) return refuse(fn, "K of %llu: rows of at most %lld bytes", (unsigned long long)K, (long long)MOST_ROW_BYTES);
    if (activation < NONE || activation > SILU) return refuse(fn, "activation %d is not known", activation);
    if (!known_type(type, false) && type != F8) return refuse(fn, "element type %d: float16, bfloat16 or float8_e4m3", type);
    if (type == F8 ? !known_type(y, false) : y != type) return refuse(fn, "results of type %d from operands of type %d", y, type);
    return refuse_result(fn, M, N);
}

}  // namespace tops
#endif
