// attend_rows_plan.hpp — how attend_rows (attend_rows.hpp) cuts a call into
// blocks, and the layout of an 8-bit KV state. Plain host arithmetic (tests
// build it without HIP).
#pragma once

#include <algorithm>
#include <cstdint>

namespace syn {

// ---- 8-bit KV states --------------------------------------------------------
// A KV head's positions in tiles of 64; a tile's record holds its K bytes, V
// bytes, K steps and V steps. Bytes are value + 128 (attend_rows.hpp turns
// them into halves by placing them in a mantissa).
constexpr uint32_t kv8_tile = 64;

struct kv8_shape {
    uint32_t n_kv, hd;
    uint32_t hdp;         // hd rounded up to whole 32s, the matrix core's k
    uint32_t tiles;       // tiles of one KV head
    uint32_t v_at;        // V bytes in a record (K bytes are at 0)
    uint32_t ks_at;       // K steps
    uint32_t vs_at;       // V steps
    uint32_t tile_bytes;  // a record
};

inline kv8_shape kv8_shape_of(uint32_t max_ctx, uint32_t n_kv, uint32_t hd) {
    kv8_shape s{};
    s.n_kv = n_kv;
    s.hd = hd;
    s.hdp = (hd + 31) / 32 * 32;
    s.tiles = max_ctx / kv8_tile + (max_ctx % kv8_tile != 0);
    s.v_at = kv8_tile * s.hdp;
    s.ks_at = 2 * kv8_tile * s.hdp;
    s.vs_at = s.ks_at + kv8_tile * 4;
    s.tile_bytes = s.vs_at + kv8_tile * 4;
    return s;
}

inline uint64_t kv8_bytes(const kv8_shape& s) {
    return uint64_t{s.n_kv} * s.tiles * s.tile_bytes;
}

// Where position key (of its tile), dim d has its K byte. A wave's load of a
// score operand (16 keys x 64 dims, lane 16 G + m: 16 dims of key row m) is
// 1 KiB in lane order; an odd last 32 dims take 8 bytes a lane. Row m = 4 G'
// + r of operand (c, a) is key 32 c + 8 G' + 4 a + r, so that a lane's eight
// scores of operands (c, 0) and (c, 1) are eight neighbouring keys, which is
// how the output product wants its probabilities.
inline constexpr uint32_t kv8_k_at(uint32_t hdp, uint32_t key, uint32_t d) {
    const uint32_t c = key / 32, g = key / 8 % 4, a = key / 4 % 2, r = key % 4;
    const uint32_t m = 4 * g + r;
    const uint32_t base = (2 * c + a) * 16 * hdp;
    const uint32_t pairs = hdp / 64 * 64;  // dims in whole 64s
    if (d < pairs) {
        return base + d / 64 * 1024 + (d % 64 / 16 * 16 + m) * 16 + d % 16;
    }
    const uint32_t e = d - pairs;
    return base + pairs * 16 + (e / 8 * 16 + m) * 8 + e % 8;
}
// Its V byte: 16 dims x 64 keys are 1 KiB in lane order, lane 16 G + d % 16
// holding keys 8 G .. + 7 and 32 + 8 G .. + 7.
inline constexpr uint32_t kv8_v_at(uint32_t key, uint32_t d) {
    return d / 16 * 1024 + (key / 8 % 4 * 16 + d % 16) * 16 + key / 32 * 8 + key % 8;
}

// ---- blocks of attend_rows --------------------------------------------------
constexpr uint32_t attend_tile = 64;        // keys of a step
constexpr uint32_t attend_waves = 4;        // waves of a block
constexpr uint32_t attend_max_splits = 256;
// Splits are added up to this many waves: two on each of 256 CUs' four SIMDs.
constexpr uint32_t attend_cus = 256;
constexpr uint32_t attend_split_waves = attend_cus * 4 * 2;

enum attend_kernel : uint32_t {
    attend_few,     // one block has the rows, its waves share out the keys
    attend_many16,  // four waves of 16 rows
    attend_many32,  // four waves of 32 rows
    attend_turns,   // eight waves of 32 rows, half of them in their products at a time
};

constexpr uint32_t attend_max_group = 32768;       // a block's rows of one token more times it stay below 2^32
constexpr uint32_t attend_max_row_blocks = 65535;  // a grid dimension

struct attend_plan {
    attend_kernel kernel;
    uint32_t block_rows;   // query rows per block
    uint32_t row_blocks;   // blocks over the query rows of one KV head
    uint32_t chunk;        // key tiles per split
    uint32_t splits;
};

// The most splits a plan of these row blocks may have on up to len keys:
// four tiles each at least, one per wave or per staged row block.
inline uint32_t attend_max_splits_of(const attend_plan& p, uint32_t n_kv, uint32_t len) {
    const uint64_t units = uint64_t{p.row_blocks} * n_kv;
    const uint32_t tiles = len / attend_tile + (len % attend_tile != 0);
    const uint32_t blocks = attend_split_waves / (p.kernel == attend_turns ? 8 : 4);
    const uint64_t few = units < blocks ? blocks / units : 1;
    return static_cast<uint32_t>(std::min<uint64_t>(
        {few, std::max(1u, tiles / attend_waves + (tiles % attend_waves != 0)), attend_max_splits}));
}

// Up to 16 rows of a KV head go to attend_few, but over a binary16 state of
// more than 192 dims, whose tile spills its registers: 16 rows of 4 heads of
// 256 behind 12000 keys 26.0 us, by attend_many16 22.0 (of 192 18.1 and 18.8; over
// an 8-bit state of 256 18.9 and 20.5).
inline bool attend_takes_few(uint64_t rows, uint32_t hd, bool halves) {
    return rows <= 16 && !(halves && hd > 192);
}
// The kernels for other rows.
inline void set_attend_kernel(attend_plan& p, attend_kernel kernel, uint64_t rows) {
    p.kernel = kernel;
    p.block_rows = kernel == attend_turns ? 256 : kernel == attend_many32 ? 128 : 64;
    p.row_blocks = static_cast<uint32_t>((rows + p.block_rows - 1) / p.block_rows);
}
inline bool attend_takes(attend_kernel kernel, uint64_t rows, uint32_t hd, bool by_pairs) {
    switch (kernel) {
    case attend_turns:  // over 128 dims a wave's rows leave no second wave on a SIMD
        return rows > 128 && hd <= 128 && !by_pairs;
    case attend_many32:
        return rows > 64 && !by_pairs;
    default:
        return true;
    }
}

// n tokens of `group` query heads per KV head attend up to len keys. halves: a
// binary16 state; by_pairs: one whose K rows are off 16 bytes; its tiles go
// through registers, which 32 rows a wave do not leave.
//
// The more rows a block has, the less of its tiles' cost each bears: 509
// tokens of 4 heads behind 7683 (8 KV heads of 128) take the turns kernel 102
// us and attend_many32 113. But where the blocks of all splits do not reach
// the CUs' count, the time is one block's way through its few tiles, and
// smaller blocks go it sooner: 29 tokens of 7 heads behind 171 took the turns
// kernel 22.8 us and take attend_many16 11.2; 95 tokens of 4 heads behind 8,
// 19.4 and 8.3. And where the last block's half would go without rows, which
// leaves the turns kernel's other half no one to take turns with, the blocks
// of attend_many32, at 1.1 times the time a row, can win.
inline attend_plan plan_attend_rows(uint32_t n, uint32_t group, uint32_t n_kv, uint32_t hd, uint32_t len,
                                    bool halves, bool by_pairs) {
    attend_plan p{};
    const uint64_t rows = uint64_t{n} * group;
    if (attend_takes_few(rows, hd, halves)) {
        p.kernel = attend_few;
        p.block_rows = 16;
        p.row_blocks = 1;
    } else {
        for (const attend_kernel kernel : {attend_turns, attend_many32, attend_many16}) {
            if (!attend_takes(kernel, rows, hd, by_pairs)) {
                continue;
            }
            set_attend_kernel(p, kernel, rows);
            const bool halved = kernel == attend_turns && (rows + 127) / 128 * 11 < uint64_t{p.row_blocks} * 2 * 10;
            if (!halved && uint64_t{p.row_blocks} * n_kv * attend_max_splits_of(p, n_kv, len) >= attend_cus) {
                break;
            }
        }
    }
    const uint32_t tiles = len / attend_tile + (len % attend_tile != 0);
    const uint32_t splits = attend_max_splits_of(p, n_kv, len);
    p.chunk = std::max(1u, (tiles + splits - 1) / splits);
    p.splits = std::max(1u, (tiles + p.chunk - 1) / p.chunk);
    return p;
}

// Scratch a plan needs: per split, KV head and query row an output and its
// (max, sum); none for a single split.
inline uint64_t attend_scratch_floats(const attend_plan& p, uint32_t n_kv, uint64_t rows, uint32_t hd) {
    return p.splits > 1 ? uint64_t{p.splits} * n_kv * rows * (hd + 2) : 0;
}

// The most any call of up to max_n tokens on up to max_len keys needs: each
// kernel's splits only grow with the keys, and there are none from some count
// of rows on.
inline uint64_t attend_scratch_bound(uint32_t max_n, uint32_t group, uint32_t n_kv, uint32_t hd, uint32_t max_len,
                                     bool halves, bool by_pairs) {
    uint64_t most = 0;
    for (uint32_t n = 1; n <= max_n; ++n) {
        const uint64_t rows = uint64_t{n} * group;
        if (rows * n_kv > attend_split_waves * 64) {  // a wave's most rows: no splits from here on
            break;
        }
        attend_plan p{attend_few, 16, 1, 0, 0};
        const bool few = attend_takes_few(rows, hd, halves);
        uint32_t splits = few ? attend_max_splits_of(p, n_kv, max_len) : 1;
        for (const attend_kernel kernel : {attend_turns, attend_many32, attend_many16}) {
            if (!few && attend_takes(kernel, rows, hd, by_pairs)) {
                set_attend_kernel(p, kernel, rows);
                splits = std::max(splits, attend_max_splits_of(p, n_kv, max_len));
            }
        }
        if (splits > 1) {
            most = std::max(most, splits * n_kv * rows * (hd + 2));
        }
    }
    return most;
}

}  // namespace syn
