// attend_rows.hpp — attention of a run's query rows over a KV state, for the
// states and masks the decode and prefill kernels do not take: 8-bit states
// (attend_kv8.hip), and drafted trees over either kind (attend_tree.hip).
//
//   out_r = sum_t p_rt v_t / sum_t p_rt,  p_rt = exp(scale q_r . k_t - m_r)
//
// over the keys t that row r sees, in one pass with a running maximum m.
//
// Rows. The query rows of a KV head are (token, head) pairs, r = token *
// group + head: a key or value byte serves all of them. Three kernels share
// the arithmetic here (plan_attend_rows chooses; 32 query heads on 8 KV heads
// of 128 unless said otherwise):
//  - up to 16 rows (a decode step), attend_few: a wave takes all of them and
//    every fourth tile of 64 keys of the block's split, straight from memory
//    into operand registers, and the block's four waves meet in LDS at the
//    end. Bound by HBM, so nothing is shared and no barrier is in the loop:
//    100001 keys in 39.7 us (5.3 TB/s); 4097 in 6.3, which is the launch and a
//    chain of four trips to memory (q and tile, then three tiles).
//  - more rows, attend_many: each of the four waves has 16 or 32 of its own,
//    and the tiles of keys, which they all need, come through LDS as operands
//    (two buffers, one barrier a tile). 26 tokens behind 4096: 15.3 us.
//  - many rows, attend_turns: eight waves of 32, whose halves take turns at
//    the matrix cores. 509 tokens behind 7683: 100.5 us (659 TFLOP/s counted,
//    988 issued, as P V goes twice); 61 behind 20000: 42.2 us. The matrix
//    units are 44 % busy and the vector units 48 %.
// Splits of one row block meet in a second, small kernel (attend_merge.hip).
//
// Products. S^T = K Q^T and O^T += V^T P^T on v_mfma_f32_16x16x32_f16: a
// lane holds one query (column) of every tile, so its maximum, sum and
// rescaling are its own, and the scores of its keys are the P^T operand as
// they stand (keys are dealt to the score operand's rows so that a lane gets
// eight neighbouring ones). 8-bit values become halves exactly: the byte b =
// value + 128 under 0x64 is the half 1024 + b, less 1152.
//
// Numbers. Scores, maxima, sums and outputs are f32. q is rounded to
// binary16 as the other attention kernels round it. Probabilities go to the
// matrix core as two halves, p = hi + lo, which keeps 22 bits: a single half
// alone is 2e-4 off in the output. They are scaled by 2^6 (and at most 2^8
// above that, before the running maximum follows), so that lo is a normal
// number wherever it counts. With an 8-bit state p carries its key's V step,
// held against the power of two above the largest step so far that the row
// sees (`vexp`), so steps of any size keep that range.
#pragma once

#include "attend_rows_plan.hpp"
#include "device.hpp"
#include "kernels.hpp"

#include <type_traits>

namespace syn {

namespace attend {

constexpr float p_shift = 6.0f;  // probabilities are 2^6 exp2(s - m)
constexpr float lazy = 8.0f;     // a maximum follows once a score is 2^8 above it
constexpr int no_vexp = -1000;   // no step but zeros so far
constexpr float no_max = -3.0e38f;  // before any score (finite: a score of -inf is 0, not NaN, over it)

typedef unsigned int u2 __attribute__((ext_vector_type(2)));
typedef float f2 __attribute__((ext_vector_type(2)));
typedef int i2 __attribute__((ext_vector_type(2)));

// Eight bytes (value + 128) as halves, exactly.
__device__ __forceinline__ h8 bytes_h8(unsigned lo, unsigned hi) {
    constexpr unsigned one_k = 0x64646464u;
    const h2 bias = {static_cast<_Float16>(1152.0f), static_cast<_Float16>(1152.0f)};
    const h2 a = __builtin_bit_cast(h2, __builtin_amdgcn_perm(one_k, lo, 0x04010400u)) - bias;
    const h2 b = __builtin_bit_cast(h2, __builtin_amdgcn_perm(one_k, lo, 0x04030402u)) - bias;
    const h2 c = __builtin_bit_cast(h2, __builtin_amdgcn_perm(one_k, hi, 0x04010400u)) - bias;
    const h2 d = __builtin_bit_cast(h2, __builtin_amdgcn_perm(one_k, hi, 0x04030402u)) - bias;
    return h8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// x - h[0] and x - h[1], in one instruction each (the compiler converts first
// and then subtracts).
__device__ __forceinline__ float less_low(float x, h2 h) {
    float r;
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(r) : "v"(h), "v"(x));
    return r;
}
__device__ __forceinline__ float less_high(float x, h2 h) {
    float r;
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r) : "v"(h), "v"(x));
    return r;
}

__device__ __forceinline__ bool any_lane(bool x) {
    return __builtin_amdgcn_ballot_w64(x) != 0;
}

// First dim of a lane's eight in k-step dc of the score product. An 8-bit
// state's loads give a lane 16 neighbouring dims, for two k-steps.
template <int DC, bool EIGHT>
__device__ __forceinline__ uint32_t k_dim(int dc, uint32_t G) {
    return EIGHT && dc < DC / 2 * 2 ? dc / 2 * 64 + G * 16 + dc % 2 * 8 : dc * 32 + G * 8;
}

// The key (of its tile) of a lane's score j, and of score operand st's row m.
__device__ __forceinline__ uint32_t score_key(int j, uint32_t G) {
    return j / 8 * 32 + G * 8 + j % 8;
}
__device__ __forceinline__ uint32_t operand_key(int st, uint32_t m) {
    return st / 2 * 32 + m / 4 * 8 + st % 2 * 4 + m % 4;
}

// Eight halves of a binary16 K row from dim d on; zeros past the head's last
// one (what follows is the next head's, and could be NaN).
template <bool WHOLE8>
__device__ __forceinline__ h8 k_halves(const _Float16* p, uint32_t d, uint32_t hd) {
    if constexpr (WHOLE8) {
        const bool in = d < hd;
        const u4 x = load16(p + (in ? d : 0));
        return as_h8(in ? x : zero_u4());
    } else {
        h8 x;
#pragma unroll
        for (int e = 0; e < 8; e += 2) {  // hd is even: pairs are 4-byte aligned
            const bool in = d + e < hd;
            const h2 y = *reinterpret_cast<const h2*>(p + (in ? d + e : 0));
            x[e] = in ? y[0] : static_cast<_Float16>(0);
            x[e + 1] = in ? y[1] : static_cast<_Float16>(0);
        }
        return x;
    }
}

// Of eight keys of a binary16 V^T row, the first `left` (all ones for theirs).
__device__ __forceinline__ u4 first_halves(uint32_t left) {
    u4 keep;
#pragma unroll
    for (uint32_t e = 0; e < 4; ++e) {
        keep[e] = left >= 2 * e + 2 ? 0xffffffffu : left == 2 * e + 1 ? 0xffffu : 0u;
    }
    return keep;
}
// The larger magnitudes of x's halves and top's, as bits.
__device__ __forceinline__ uint32_t top_halves(uint32_t top, u4 x) {
    typedef unsigned short us2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const uint32_t y = x[e] & 0x7fff7fffu;
        top = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(us2, top), __builtin_bit_cast(us2, y)));
    }
    return top;
}
// Whether one of them is infinite or NaN.
__device__ __forceinline__ bool wild_halves(uint32_t top) {
    return (top & 0xffffu) >= 0x7c00u || top >> 16 >= 0x7c00u;
}

// Weight of a part (max, sum) of a row whose maximum is top.
__device__ __forceinline__ float part_weight(float m, float l, float top) {
    return l == 0.0f ? 0.0f : l * fast_exp2(m - top);  // (l == 0: nothing seen, m may be -inf)
}

// The exponent of the power of two above the largest of a tile's V steps, or
// no_vexp.
__device__ __forceinline__ int step_exp(float top) {
    return top > 0.0f ? __builtin_amdgcn_frexp_expf(top) : no_vexp;
}

// x / group for x below 2^32 / group (a row of the block, counted from its
// first token's first head).
__device__ __forceinline__ uint32_t div_group(const attend_rows_args& a, uint32_t x) {
    return a.group == 1 ? x : __umulhi(x, a.inv_group);
}

// A block's place: KV heads fastest (with 8 of them each XCD keeps to one,
// whose L2 then serves all row blocks), then splits, the last row blocks
// first (a causal run's longest). A grid of three dimensions, and one division
// for the block's first row: a launch finds its instructions in neither cache
// (other kernels and the keys have gone through both), and starting with four
// divisions to fetch took 2 to 12 us.
struct block_place {
    uint32_t g, split, row0, len, t_begin, t_end;
    uint32_t token0, head0;  // of row0
};
template <bool TREE>
__device__ __forceinline__ block_place place_block(const attend_rows_args& a) {
    block_place b;
    b.g = blockIdx.x;
    b.split = blockIdx.y;
    b.row0 = (a.row_blocks - 1 - blockIdx.z) * a.block_rows;
    b.token0 = b.row0 / a.group;
    b.head0 = b.row0 - b.token0 * a.group;
    const uint32_t rows = a.n * a.group;
    const uint32_t last = min(a.block_rows, rows - b.row0) - 1;
    // Up to the last row's last key.
    b.len = TREE ? a.pos + a.n : a.pos + b.token0 + div_group(a, b.head0 + last) + 1;
    const uint32_t tiles = (b.len + attend_tile - 1) / attend_tile;
    b.t_begin = b.split * a.chunk;
    b.t_end = min(tiles, b.t_begin + a.chunk);
    return b;
}

// Where the output of row r of all, at q's place `at`, goes: the output
// itself, or its split's part.
__device__ __forceinline__ float* row_out(const attend_rows_args& a, const block_place& b, uint32_t r, size_t at) {
    return a.splits == 1 ? a.out + at : a.part + ((size_t{b.split} * a.n_kv + b.g) * (a.n * a.group) + r) * a.hd;
}
__device__ __forceinline__ void store_part(const attend_rows_args& a, const block_place& b, uint32_t r, float m,
                                           float l) {
    *reinterpret_cast<f2*>(a.part_ml + ((size_t{b.split} * a.n_kv + b.g) * (a.n * a.group) + r) * 2) = f2{m, l};
}

// The order of stream_operands for the scheduler: a pair's products, two reads.
template <int AHEAD, int N, int O, class PRODUCTS>
__device__ __forceinline__ void sched_pairs() {
    if constexpr (O < N) {
        __builtin_amdgcn_sched_group_barrier(0x008, PRODUCTS::at(O), 0);
        if constexpr (O + AHEAD < N) {
            __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
        }
        sched_pairs<AHEAD, N, O + 2, PRODUCTS>();
    }
}

// N operands from LDS, used in pairs: AHEAD reads are in flight before the
// first use, and each pair's use is followed by two more. Left to itself the
// compiler reads a pair, waits for it, and only then reads the next one, which
// left the matrix units idle for as long as they worked. PRODUCTS: how many
// the pair at o has.
template <int AHEAD, int N, class PRODUCTS, class READ, class USE>
__device__ __forceinline__ void stream_operands(READ read, USE use) {
    static_assert(AHEAD % 2 == 0 && N % 2 == 0 && AHEAD <= N);
    h8 f[AHEAD];
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
        f[i] = read(i);
    }
#pragma unroll
    for (int o = 0; o < N; o += 2) {
        const h8 x = f[o % AHEAD], y = f[o % AHEAD + 1];
        if (o + AHEAD < N) {
            f[o % AHEAD] = read(o + AHEAD);
            f[o % AHEAD + 1] = read(o + AHEAD + 1);
        }
        use(o, x, y);
    }
    __builtin_amdgcn_sched_group_barrier(0x100, AHEAD, 0);  // LDS reads
    sched_pairs<AHEAD, N, 0, PRODUCTS>();
    __builtin_amdgcn_sched_barrier(0);
}

// RT tiles of 16 query rows that one wave holds: lane 16 G + col has column
// col of every tile.
template <int DC, int RT, bool EIGHT, bool TREE>
struct wave_rows {
    static constexpr int DT = 2 * DC;
    static_assert(RT <= 2);
    uint32_t G, col, row0;
    uint32_t from;              // row0, counted from the first head of the block's first token
    h8 q[RT][DC];
    f4 acc[RT][DT];             // O^T: dims 16 dt + 4 G .. + 3
    // The running maximum less p_shift; the sum of this lane's keys. Vectors:
    // as arrays the compiler kept them in LDS by work-item, and finding that
    // place read the dispatch packet in host memory (1 to 13 us of a start).
    f2 mref, l;
    h8 hi[RT][2], lo[RT][2];    // the last step's probabilities
    uint32_t seen[RT];          // the keys of a masked tile that the row sees, by score
    i2 vexp;                    // 8-bit states: the exponent that the row's V steps are held against

    struct raw_q {
        f4 x[RT][DC][2];
    };
    // Rows from row `skip` of the block's on.
    __device__ __forceinline__ void place(const block_place& b, uint32_t skip, uint32_t lane) {
        G = lane / 16;
        col = lane % 16;
        row0 = b.row0 + skip;
        from = b.head0 + skip;
        vexp = i2{no_vexp, no_vexp};
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            mref[rt] = no_max;
            l[rt] = 0.0f;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                acc[rt][dt] = f4{0, 0, 0, 0};
            }
        }
    }
    // A row's place in q and in the output (0: no row).
    __device__ __forceinline__ size_t at(const attend_rows_args& a, const block_place& b, int rt) const {
        const uint32_t x = from + rt * 16 + col, later = div_group(a, x);
        return row0 + rt * 16 + col < a.n * a.group
                   ? size_t{b.token0 + later} * a.q_row + (b.g * a.group + x - later * a.group) * a.hd
                   : 0;
    }
    // Starts the rows' loads, 32 bytes for eight dims (of which binary16 rows
    // use the first 16), with no branch on the type: at a join the compiler
    // waited for what each side had loaded, one operand after the other (8 us
    // of a block's start). Heads of no whole eights are loaded by take_q.
    __device__ __forceinline__ void load_q(const attend_rows_args& a, const block_place& b, raw_q& raw) const {
        if (a.hd % 8 == 0) {
            const uint32_t size = a.q_f16 ? 2 : 4, half = a.q_f16 ? 0 : 16;
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                const size_t i = at(a, b, rt);
#pragma unroll
                for (int dc = 0; dc < DC; ++dc) {
                    const uint32_t d = k_dim<DC, EIGHT>(dc, G);
                    const char* p = static_cast<const char*>(a.q) + (i + (d < a.hd ? d : 0)) * size;
                    raw.x[rt][dc][0] = *reinterpret_cast<const f4*>(p);
                    raw.x[rt][dc][1] = *reinterpret_cast<const f4*>(p + half);
                }
            }
        }
    }
    // Rounds them to binary16; zeros past the head's last dim.
    __device__ __forceinline__ void take_q(const attend_rows_args& a, const block_place& b, const raw_q& raw) {
        if (a.hd % 8 == 0) {
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
                for (int dc = 0; dc < DC; ++dc) {
                    const f4 x = raw.x[rt][dc][0], y = raw.x[rt][dc][1];
                    h8 h = a.q_f16 ? __builtin_bit_cast(h8, x)
                                   : h8{to_h(x[0]), to_h(x[1]), to_h(x[2]), to_h(x[3]), to_h(y[0]), to_h(y[1]),
                                        to_h(y[2]), to_h(y[3])};
                    q[rt][dc] = k_dim<DC, EIGHT>(dc, G) < a.hd ? h : as_h8(zero_u4());
                }
            }
            return;
        }
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const size_t row = at(a, b, rt);
#pragma unroll
            for (int dc = 0; dc < DC; ++dc) {
                const uint32_t d = k_dim<DC, EIGHT>(dc, G);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const size_t i = row + (d + e < a.hd ? d + e : 0);
                    const _Float16 x = a.q_f16 ? static_cast<const _Float16*>(a.q)[i]
                                               : to_h(static_cast<const float*>(a.q)[i]);
                    q[rt][dc][e] = d + e < a.hd ? x : static_cast<_Float16>(0);
                }
            }
        }
    }

    // Row rt's V steps go up to 2^e: what is summed already goes with them.
    __device__ __forceinline__ void raise_vexp(int rt, int e) {
        if (any_lane(e > vexp[rt])) {
            const int to = e > vexp[rt] ? e : vexp[rt];
            const float f = vexp[rt] == no_vexp ? 0.0f : ldexpf(1.0f, vexp[rt] - to);
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                acc[rt][dt] *= f;
            }
            vexp[rt] = to;
        }
    }
    // The same for a tile that all rows see.
    __device__ __forceinline__ void raise_vexp(int e) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            raise_vexp(rt, e);
        }
    }

    // Which keys of the tile at key0 the rows see. A lane's two eights of keys,
    // 32 apart, lie in three words of its row's mask, loaded without branches
    // (with them each was waited for before the next: 4 us a tile), words
    // outside the row from its first. Rows' tokens and limits are found again
    // for each of the few masked tiles: kept, they took the other tiles'
    // registers (a tree of 61: 50 us, 46).
    __device__ __forceinline__ void take_mask(const attend_rows_args& a, const block_place& b, uint32_t key0) {
        const int w = static_cast<int>(key0 + G * 8 - a.pos) >> 5, words = static_cast<int>(a.mask_words);
        uint32_t word[RT][3];
        if constexpr (TREE) {
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                const bool in = row0 + rt * 16 + col < a.n * a.group;
                const uint32_t token = in ? b.token0 + div_group(a, from + rt * 16 + col) : 0;
#pragma unroll
                for (int i = 0; i < 3; ++i) {
                    word[rt][i] = a.mask[size_t{token} * a.mask_words + (w + i >= 0 && w + i < words ? w + i : 0)];
                }
            }
        }
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const bool in = row0 + rt * 16 + col < a.n * a.group;
            const uint32_t all = !in ? 0 : TREE ? a.pos : a.pos + b.token0 + div_group(a, from + rt * 16 + col) + 1;
            uint32_t bits = 0;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const uint32_t k0 = key0 + score_key(8 * c, G);
                const uint32_t open = all > k0 ? all - k0 : 0;
                uint32_t eight = open >= 8 ? 0xffu : (1u << open) - 1u;
                if constexpr (TREE) {
                    const int j = static_cast<int>(k0 - a.pos);  // (the first before or behind the drafted tokens: none)
                    const uint32_t lo = w + c >= 0 && w + c < words ? word[rt][c] : 0u;
                    const uint32_t hi = w + c + 1 >= 0 && w + c + 1 < words ? word[rt][c + 1] : 0u;
                    const uint32_t drafted = static_cast<uint32_t>((uint64_t{hi} << 32 | lo) >> (j & 31));
                    const int left = static_cast<int>(a.n) - j;  // bits past the last token are ignored
                    eight |= in ? drafted & (left >= 8 ? 0xffu : left > 0 ? (1u << left) - 1u : 0u) : 0u;
                }
                bits |= eight << (8 * c);
            }
            seen[rt] = bits;
        }
    }

    // Scores of the tile at key0 to probabilities, split into hi and lo. ks: the
    // keys' K steps times the scale in exp2's units (or that scale alone); vm:
    // their V steps over 2^vexp. MASKED: some row may not see some of the
    // tile's keys (take_mask); vm are the steps themselves then, and each row's
    // vexp comes from those that it sees (against a large one that it does not see, its
    // own would leave the halves' range). While no lane has a score more than `lazy` above its row's
    // maximum, lanes need nothing from each other.
    template <bool MASKED, class KS, class VM>
    __device__ __forceinline__ void softmax(const f4 (&s)[RT][4], KS ks, VM vm) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const uint32_t bits = MASKED ? seen[rt] : 0xffffu;
            if constexpr (EIGHT && MASKED) {
                float top = 0.0f;
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    top = fmaxf(top, bits >> j & 1 ? vm(j) : 0.0f);
                }
                raise_vexp(rt, step_exp(max32(max16(top))));
            }
            float p[16];  // over the maximum, in exp2's units
            const auto over = [&](float m) {
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    p[j] = __builtin_fmaf(s[rt][j / 4][j % 4], ks(j), -m);
                }
                if constexpr (MASKED) {
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        p[j] = bits >> j & 1 ? p[j] : -INFINITY;
                    }
                }
                float top = p[0];
#pragma unroll
                for (int j = 1; j < 16; ++j) {
                    top = fmaxf(top, p[j]);
                }
                return top;
            };
            float top = over(mref[rt]);
            if (any_lane(top > p_shift + lazy)) {
                top = max32(max16(over(0.0f))) - p_shift;
                const float m = top > mref[rt] + lazy ? top : mref[rt];
                const float f = fast_exp2(mref[rt] - m);
                mref[rt] = m;
                l[rt] *= f;
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) {
                    acc[rt][dt] *= f;
                }
                over(m);
            }
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                p[j] = fast_exp2(p[j]);
            }
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                l[rt] += p[j];
                if constexpr (EIGHT && MASKED) {  // a masked key's step may be anything
                    p[j] = bits >> j & 1 ? p[j] * ldexpf(vm(j), -vexp[rt]) : 0.0f;
                } else if constexpr (EIGHT) {
                    p[j] *= vm(j);
                }
            }
#pragma unroll
            for (int j = 0; j < 16; j += 2) {
                const h2 h = __builtin_convertvector((f2{p[j], p[j + 1]}), h2);
                hi[rt][j / 8][j % 8] = h[0];
                hi[rt][j / 8][j % 8 + 1] = h[1];
                const h2 r = __builtin_convertvector((f2{less_low(p[j], h), less_high(p[j + 1], h)}), h2);
                lo[rt][j / 8][j % 8] = r[0];
                lo[rt][j / 8][j % 8 + 1] = r[1];
            }
        }
    }

    // The products of a tile, its operands in LDS in lane order: V (dt, c) at
    // v_from, then K (st, dc) of the next tile at k_from. Operand o of V is dims
    // o % DT of key half o / DT, of K score tile o % 4 of k-step o / 4: what
    // neighbouring products add to lies apart.
    static constexpr int v_ops = 4 * DC, k_ops = 4 * DC;
    template <int FIRST_K>  // operands from FIRST_K on are K's
    struct products {
        static constexpr int at(int o) { return o < FIRST_K ? 4 * RT : 2 * RT; }
    };
    __device__ static __forceinline__ h8 read_v(const h8* v_from, int o) {
        return v_from[(o % DT * 2 + o / DT) * 64];
    }
    __device__ static __forceinline__ h8 read_k(const h8* k_from, int o) {
        return k_from[(o % 4 * DC + o / 4) * 64];
    }
    __device__ __forceinline__ void use_v(int o, h8 x, h8 y) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            acc[rt][o % DT] = mfma16(x, hi[rt][o / DT], acc[rt][o % DT]);
            acc[rt][o % DT + 1] = mfma16(y, hi[rt][o / DT], acc[rt][o % DT + 1]);
        }
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            acc[rt][o % DT] = mfma16(x, lo[rt][o / DT], acc[rt][o % DT]);
            acc[rt][o % DT + 1] = mfma16(y, lo[rt][o / DT], acc[rt][o % DT + 1]);
        }
    }
    // k_in: the lane's last eight dims are the head's (else a binary16 state's
    // operand has the next head's there, which could be NaN).
    __device__ __forceinline__ void use_k(int o, h8 x, h8 y, f4 (&s)[RT][4], bool k_in) const {
        if (!EIGHT && o / 4 == DC - 1) {
            x = as_h8(k_in ? as_u4(x) : zero_u4());
            y = as_h8(k_in ? as_u4(y) : zero_u4());
        }
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const f4 zero = {0, 0, 0, 0};
            s[rt][o % 4] = mfma16(x, q[rt][o / 4], o < 4 ? zero : s[rt][o % 4]);
            s[rt][o % 4 + 1] = mfma16(y, q[rt][o / 4], o < 4 ? zero : s[rt][o % 4 + 1]);
        }
    }
    template <int AHEAD>
    __device__ __forceinline__ void stream_k(const h8* k_from, f4 (&s)[RT][4], bool k_in) {
        stream_operands<AHEAD, k_ops, products<0>>([&](int o) { return read_k(k_from, o); },
                                                   [&](int o, h8 x, h8 y) { use_k(o, x, y, s, k_in); });
    }
    template <int AHEAD>
    __device__ __forceinline__ void stream_v(const h8* v_from) {
        stream_operands<AHEAD, v_ops, products<v_ops>>([&](int o) { return read_v(v_from, o); },
                                                       [&](int o, h8 x, h8 y) { use_v(o, x, y); });
    }
    template <int AHEAD>
    __device__ __forceinline__ void stream_vk(const h8* v_from, const h8* k_from, f4 (&s)[RT][4], bool k_in) {
        stream_operands<AHEAD, v_ops + k_ops, products<v_ops>>(
            [&](int o) { return o < v_ops ? read_v(v_from, o) : read_k(k_from, o - v_ops); },
            [&](int o, h8 x, h8 y) {
                if (o < v_ops) {
                    use_v(o, x, y);
                } else {
                    use_k(o - v_ops, x, y, s, k_in);
                }
            });
    }

    // O^T += V^T P^T for 16 dims and 32 keys.
    __device__ __forceinline__ void add_v(int dt, int c, h8 v) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            acc[rt][dt] = mfma16(v, hi[rt][c], acc[rt][dt]);
            acc[rt][dt] = mfma16(v, lo[rt][c], acc[rt][dt]);
        }
    }
    // The same in a masked tile of a binary16 state that holds infinities or
    // NaN, which as an operand would reach the rows that do not see them (0
    // times one is NaN). They get products of their own: a row has +inf added
    // where it sees a +inf or NaN among the 32 keys, and -inf where it sees a
    // -inf or NaN (so NaN where both).
    __device__ __forceinline__ void add_wild_v(int dt, int c, h8 v) {
        h8 finite, up, down;
        bool any = false;
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e) {
            const _Float16 x = v[e];  // (a bit cast of the element itself casts element 0)
            const unsigned short b = __builtin_bit_cast(unsigned short, x);
            const bool wild = (b & 0x7c00u) == 0x7c00u, nan = (b & 0x3ffu) != 0;
            finite[e] = wild ? static_cast<_Float16>(0) : x;
            up[e] = static_cast<_Float16>(wild && (nan || b >> 15 == 0) ? 1.0f : 0.0f);
            down[e] = static_cast<_Float16>(wild && (nan || b >> 15 != 0) ? 1.0f : 0.0f);
            any = any || wild;
        }
        add_v(dt, c, finite);
        if (any_lane(any)) {
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                h8 sees;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    sees[e] = static_cast<_Float16>(seen[rt] >> (8 * c + e) & 1 ? 1.0f : 0.0f);
                }
                const f4 ups = mfma16(up, sees, f4{0, 0, 0, 0}), downs = mfma16(down, sees, f4{0, 0, 0, 0});
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    acc[rt][dt][e] += ups[e] > 0.0f ? INFINITY : 0.0f;
                    acc[rt][dt][e] -= downs[e] > 0.0f ? INFINITY : 0.0f;
                }
            }
        }
    }
    template <class V>
    __device__ __forceinline__ void add_wild(V v) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                add_wild_v(dt, c, v(dt, c));
                __builtin_amdgcn_sched_barrier(0);  // (the next operand's read would take registers)
            }
        }
    }

    // Rows as (maximum, sum, output over sum).
    __device__ __forceinline__ void finish() {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            l[rt] = sum32(sum16(l[rt]));
            const float inv = l[rt] == 0.0f ? 0.0f : 1.0f / l[rt];
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                acc[rt][dt] *= inv;
                if constexpr (EIGHT) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        acc[rt][dt][e] = ldexpf(acc[rt][dt][e], vexp[rt] == no_vexp ? 0 : vexp[rt]);
                    }
                }
            }
        }
    }

    // The finished rows to the output, or to their split's part.
    __device__ __forceinline__ void store(const attend_rows_args& a, const block_place& b) const {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const uint32_t r = row0 + rt * 16 + col;
            if (r < a.n * a.group) {
                float* out = row_out(a, b, r, at(a, b, rt));
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) {
                    const uint32_t d = dt * 16 + G * 4;
                    const f4 o = acc[rt][dt];
                    if (a.hd % 4 == 0) {
                        if (d < a.hd) {
                            *reinterpret_cast<f4*>(out + d) = o;
                        }
                    } else {
                        if (d < a.hd) {
                            *reinterpret_cast<f2*>(out + d) = f2{o[0], o[1]};
                        }
                        if (d + 2 < a.hd) {
                            *reinterpret_cast<f2*>(out + d + 2) = f2{o[2], o[3]};
                        }
                    }
                }
                if (a.splits > 1 && G == 0) {
                    store_part(a, b, r, mref[rt], l[rt]);
                }
            }
        }
    }
};

// A wave's V operands of a masked tile (every fourth), in LDS: keys past the
// last one to zeros (what is there could be NaN). Whether some of the rest is
// infinite or NaN.
template <int DC>
__device__ __forceinline__ bool clean_v(h8* v, uint32_t w, uint32_t lane, uint32_t tile, uint32_t len) {
    uint32_t top = 0;
    const uint32_t key = tile * attend_tile + w % 2 * 32 + lane / 16 * 8;  // (operand 2 dt + c, w and c of one parity)
    const u4 keep = first_halves(len > key ? len - key : 0);
#pragma unroll
    for (int i = 0; i < DC; ++i) {
        h8* at = v + (i * 4 + w) * 64 + lane;
        const u4 x = as_u4(*at) & keep;
        top = top_halves(top, x);
        *at = as_h8(x);
    }
    return any_lane(wild_halves(top));
}
__device__ __forceinline__ bool any_wild(const int (&wild)[attend_waves]) {
    return __builtin_amdgcn_readfirstlane(wild[0] | wild[1] | wild[2] | wild[3]) != 0;
}

// ---- up to 16 rows: each wave its own tiles, from memory to operands ---------
template <int DC>
struct kv8_source {
    static constexpr bool eight = true;
    static constexpr int KQ = DC / 2;      // K loads of 16 bytes per score operand
    static constexpr bool odd = DC % 2;    // and one of 8
    const uint8_t* head;                   // the KV head's records
    size_t tile_bytes;
    uint32_t v_at, ks_at, vs_at;
    u4 kq[4][KQ > 0 ? KQ : 1];
    u2 ko[4];
    u4 vq[2 * DC];
    f4 ks[4], vs[4];

    __device__ __forceinline__ kv8_source(const attend_rows_args& a, uint32_t g, uint32_t)
        : head(a.kv8 + size_t{g} * a.tiles_per_head * a.tile_bytes), tile_bytes(a.tile_bytes),
          v_at(a.v_at), ks_at(a.ks_at), vs_at(a.vs_at) {}

    __device__ __forceinline__ void load(uint32_t tile, uint32_t lane) {
        const uint8_t* t = head + tile * tile_bytes;
#pragma unroll
        for (int st = 0; st < 4; ++st) {
#pragma unroll
            for (int p = 0; p < KQ; ++p) {
                kq[st][p] = *reinterpret_cast<const u4*>(t + (st * DC * 512 + p * 1024) + lane * 16);
            }
            if constexpr (odd) {
                ko[st] = *reinterpret_cast<const u2*>(t + (st * DC * 512 + KQ * 1024) + lane * 8);
            }
        }
        const uint32_t G = lane / 16;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            ks[j] = *reinterpret_cast<const f4*>(t + ks_at + score_key(4 * j, G) * 4);
            vs[j] = *reinterpret_cast<const f4*>(t + vs_at + score_key(4 * j, G) * 4);
        }
#pragma unroll
        for (int dt = 0; dt < 2 * DC; ++dt) {
            vq[dt] = *reinterpret_cast<const u4*>(t + v_at + dt * 1024 + lane * 16);
        }
    }
    __device__ __forceinline__ h8 k(int st, int dc) const {
        if (dc < 2 * KQ) {
            const u4 x = kq[st][dc / 2];
            return dc % 2 ? bytes_h8(x[2], x[3]) : bytes_h8(x[0], x[1]);
        }
        return bytes_h8(ko[st][0], ko[st][1]);
    }
    __device__ __forceinline__ h8 v(int dt, int c) const {
        const u4 x = vq[dt];
        return c ? bytes_h8(x[2], x[3]) : bytes_h8(x[0], x[1]);
    }
};

template <int DC, bool WHOLE8>
struct f16_source {
    static constexpr bool eight = false;
    const _Float16* kh;    // the KV head's column of K rows
    const _Float16* vh;    // its V^T rows
    size_t row, ctx_stride;
    uint32_t hd, len;
    h8 kq[4][DC];
    h8 vq[2 * DC][2];

    __device__ __forceinline__ f16_source(const attend_rows_args& a, uint32_t g, uint32_t length)
        : kh(a.k + size_t{g} * a.hd), vh(a.vt + size_t{g} * a.hd * a.ctx_stride), row(a.row),
          ctx_stride(a.ctx_stride), hd(a.hd), len(length) {}

    // Keys past the last one are read from the last one (their scores are
    // masked). ctx_stride is a multiple of 8, so eight keys are in the V^T row
    // or past it; dims past the head's are read from its last one and not
    // written out.
    __device__ __forceinline__ void load(uint32_t tile, uint32_t lane) {
        const uint32_t G = lane / 16, m = lane % 16;
#pragma unroll
        for (int st = 0; st < 4; ++st) {
            const uint32_t key = tile * attend_tile + operand_key(st, m);
            const _Float16* p = kh + (key < len ? key : len - 1) * row;
#pragma unroll
            for (int dc = 0; dc < DC; ++dc) {
                kq[st][dc] = k_halves<WHOLE8>(p, dc * 32 + G * 8, hd);
            }
        }
#pragma unroll
        for (int dt = 0; dt < 2 * DC; ++dt) {
            const uint32_t d = dt * 16 + m;
            const _Float16* p = vh + (d < hd ? d : hd - 1) * ctx_stride;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const uint32_t key = tile * attend_tile + c * 32 + G * 8;
                vq[dt][c] = as_h8(load16(p + (key < ctx_stride ? key : 0)));
            }
        }
    }
    // V past the last key to zeros (what is there could be NaN); whether some
    // of the rest is infinite or NaN.
    __device__ __forceinline__ bool clean(uint32_t tile, uint32_t lane) {
        uint32_t top = 0;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const uint32_t key = tile * attend_tile + c * 32 + lane / 16 * 8;
            const u4 keep = first_halves(len > key ? len - key : 0);
#pragma unroll
            for (int dt = 0; dt < 2 * DC; ++dt) {
                const u4 x = as_u4(vq[dt][c]) & keep;
                top = top_halves(top, x);
                vq[dt][c] = as_h8(x);
            }
        }
        return any_lane(wild_halves(top));
    }
    __device__ __forceinline__ h8 k(int st, int dc) const {
        return kq[st][dc];
    }
    __device__ __forceinline__ h8 v(int dt, int c) const {
        return vq[dt][c];
    }
};

}  // namespace attend

// grid: KV heads x splits (one row block); block 256. Two waves per SIMD where
// the registers allow it (8-bit heads of up to 128: 100001 keys of 8 x 128 in
// 39.7 us; one wave 47.6).
template <int DC, class SRC, bool TREE>
__global__ __launch_bounds__(256, SRC::eight && DC <= 4 ? 2 : 1) void attend_few_kernel(const attend_rows_args a) {
    using namespace attend;
    constexpr int DT = 2 * DC;
    constexpr uint32_t pitch = DC * 32 + 4;
    __shared__ float lds_o[attend_waves][16][pitch];
    __shared__ float lds_m[attend_waves][16], lds_l[attend_waves][16];

    const uint32_t lane = threadIdx.x % 64;
    const uint32_t w = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const block_place b = place_block<TREE>(a);
    const uint32_t open = TREE ? a.pos : a.pos + 1;  // keys that every row sees

    wave_rows<DC, 1, SRC::eight, TREE> rows;
    typename decltype(rows)::raw_q raw;
    rows.place(b, 0, lane);
    rows.load_q(a, b, raw);
    SRC src(a, b.g, b.len);
    uint32_t tile = b.t_begin + w;
    if (tile < b.t_end) {
        src.load(tile, lane);
    }
    rows.take_q(a, b, raw);

    const auto step = [&](auto masked) {
        constexpr bool MASKED = decltype(masked)::value;
        f4 s[1][4];
#pragma unroll
        for (int st = 0; st < 4; ++st) {
            s[0][st] = f4{0, 0, 0, 0};
#pragma unroll
            for (int dc = 0; dc < DC; ++dc) {
                s[0][st] = mfma16(src.k(st, dc), rows.q[0][dc], s[0][st]);
            }
        }
        if constexpr (MASKED) {
            rows.take_mask(a, b, tile * attend_tile);
        }
        if constexpr (SRC::eight) {
            float vm[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                vm[j] = src.vs[j / 4][j % 4];
            }
            if constexpr (!MASKED) {
                float top = 0.0f;
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    top = fmaxf(top, vm[j]);
                }
                rows.raise_vexp(step_exp(max32(max16(top))));
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    vm[j] = ldexpf(vm[j], -rows.vexp[0]);
                }
            }
            rows.template softmax<MASKED>(s, [&](int j) { return src.ks[j / 4][j % 4] * a.scale_log2e; },
                                          [&](int j) { return vm[j]; });
        } else {
            rows.template softmax<MASKED>(s, [&](int) { return a.scale_log2e; }, [](int) { return 1.0f; });
        }
        bool wild = false;
        if constexpr (!SRC::eight) {
            if constexpr (MASKED) {
                wild = src.clean(tile, lane);
            }
        }
        if (wild) {
            rows.add_wild([&](int dt, int c) { return src.v(dt, c); });
        } else {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) {
                    rows.add_v(dt, c, src.v(dt, c));
                }
            }
        }
    };
    // Tiles that every row sees whole, then the others, in loops of their own:
    // the masks would take the first one's registers.
    const auto run = [&](uint32_t to, auto masked) {
        while (tile < to) {
            step(masked);
            tile += attend_waves;
            if (tile < b.t_end) {
                src.load(tile, lane);
            }
        }
    };
    run(min(b.t_end, open / attend_tile), std::false_type{});
    run(b.t_end, std::true_type{});

    // The waves' rows meet in LDS as a weighted mean.
    rows.finish();
    if (rows.G == 0) {
        lds_m[w][rows.col] = rows.mref[0];
        lds_l[w][rows.col] = rows.l[0];
    }
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
        *reinterpret_cast<f4*>(&lds_o[w][rows.col][dt * 16 + rows.G * 4]) = rows.acc[0][dt];
    }
    __syncthreads();
    const uint32_t pairs = a.hd / 2, all = a.n * a.group * pairs;
    for (uint32_t i = threadIdx.x; i < all; i += 256) {
        const uint32_t r = i / pairs, d = i % pairs * 2;
        float top = -INFINITY, sum = 0.0f;
#pragma unroll
        for (uint32_t x = 0; x < attend_waves; ++x) {
            top = fmaxf(top, lds_m[x][r]);
        }
        f2 o = {0.0f, 0.0f};
#pragma unroll
        for (uint32_t x = 0; x < attend_waves; ++x) {
            const float wx = part_weight(lds_m[x][r], lds_l[x][r], top);
            sum += wx;
            const f2 ox = *reinterpret_cast<const f2*>(&lds_o[x][r][d]);
            o[0] += wx == 0.0f ? 0.0f : wx * ox[0];
            o[1] += wx == 0.0f ? 0.0f : wx * ox[1];
        }
        o *= sum == 0.0f ? 0.0f : 1.0f / sum;
        const uint32_t token = div_group(a, r);
        const size_t at = size_t{token} * a.q_row + (b.g * a.group + r - token * a.group) * a.hd;
        *reinterpret_cast<f2*>(row_out(a, b, r, at) + d) = o;
        if (a.splits > 1 && d == 0) {
            store_part(a, b, r, top, sum);
        }
    }
}

// ---- more rows: waves own rows, tiles come through LDS -------------------------
// grid: KV heads x splits x row blocks; block 256. A buffer holds a tile as
// operands in lane order: K (st, dc), then V (dt, c), 1 KiB each, so every
// LDS access is 64 neighbouring 16-byte units.
template <int DC, int RT, bool EIGHT, bool WHOLE8, bool TREE>
__global__ __launch_bounds__(256, DC <= 4 ? 2 : 1) void attend_many_kernel(const attend_rows_args a) {
    using namespace attend;
    constexpr int KQ = DC / 2;
    constexpr uint32_t v_frag = 4 * DC;          // first V operand
    constexpr bool COPY = !EIGHT && WHOLE8;      // binary16 operands, copied to LDS as they are
    constexpr int LOADS = EIGHT ? DC : 2 * DC;   // 16-byte units of a tile per thread
    __shared__ h8 tiles[2][8 * DC][64];
    __shared__ float ks_lds[2][attend_tile], vs_lds[2][attend_tile];
    __shared__ int vexp_lds[2];
    __shared__ int wild_lds[2][attend_waves];

    const uint32_t lane = threadIdx.x % 64;
    const uint32_t w = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const block_place b = place_block<TREE>(a);
    const uint32_t n_rows = a.n * a.group;
    const uint32_t row0 = b.row0 + w * (RT * 16);
    const bool has_rows = row0 < n_rows;
    const uint32_t open = TREE ? a.pos : a.pos + b.token0 + 1;  // keys that all the block's rows see
    // Keys that any of this wave's rows sees.
    const uint32_t reach = !has_rows ? 0
                           : TREE    ? b.len
                                     : a.pos + b.token0 + div_group(a, b.head0 + min(w * RT * 16 + RT * 16, n_rows - b.row0) - 1) + 1;

    const uint8_t* head = EIGHT ? a.kv8 + size_t{b.g} * a.tiles_per_head * a.tile_bytes : nullptr;
    const _Float16* kh = EIGHT ? nullptr : a.k + size_t{b.g} * a.hd;
    const _Float16* vh = EIGHT ? nullptr : a.vt + size_t{b.g} * a.hd * a.ctx_stride;
    u4 next[COPY ? 1 : LOADS];
    float next_ks = 0.0f, next_vs = 0.0f;
    int run_vexp = no_vexp;  // wave 0's: the power of two of the steps staged for all rows
    const uint32_t whole = max(b.t_begin, min(b.t_end, open / attend_tile));  // from here on tiles are masked

    // A tile's loads into registers, or (binary16) copies to buffer buf.
    const auto load = [&](uint32_t tile, uint32_t buf) {
        if constexpr (EIGHT) {
            const uint8_t* t = head + size_t{tile} * a.tile_bytes;
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                next[i] = load16(t + (i * 256 + threadIdx.x) * 16);
            }
            if (w == 0) {
                next_ks = *reinterpret_cast<const float*>(t + a.ks_at + lane * 4);
                next_vs = *reinterpret_cast<const float*>(t + a.vs_at + lane * 4);
            }
        } else {
            const uint32_t G = lane / 16, m = lane % 16;
#pragma unroll
            for (int i = 0; i < DC; ++i) {
                const int f = i * 4 + w, st = f / DC, dc = f % DC;
                const uint32_t key = tile * attend_tile + operand_key(st, m), d = dc * 32 + G * 8;
                const _Float16* p = kh + size_t{key < b.len ? key : b.len - 1} * a.row;
                if constexpr (COPY) {
                    load16_lds(p + (d < a.hd ? d : 0), &tiles[buf][f][0]);  // (dims past the head's: k_left)
                } else {
                    next[i] = as_u4(k_halves<false>(p, d, a.hd));
                }
            }
#pragma unroll
            for (int i = 0; i < DC; ++i) {
                const int f = i * 4 + w, dt = f / 2, c = f % 2;
                const uint32_t d = dt * 16 + m, key = tile * attend_tile + c * 32 + G * 8;
                const _Float16* p = vh + size_t{d < a.hd ? d : a.hd - 1} * a.ctx_stride + (key < a.ctx_stride ? key : 0);
                if constexpr (COPY) {
                    load16_lds(p, &tiles[buf][v_frag + f][0]);
                } else {
                    next[DC + i] = load16(p);
                }
            }
        }
    };
    // What load started, to buffer buf (and waited for).
    const auto stage = [&](uint32_t tile, uint32_t buf) {
        h8* to = &tiles[buf][0][0];
        if constexpr (COPY) {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        } else if constexpr (!EIGHT) {
#pragma unroll
            for (int i = 0; i < DC; ++i) {
                to[(i * 4 + w) * 64 + lane] = as_h8(next[i]);
                to[(v_frag + i * 4 + w) * 64 + lane] = as_h8(next[DC + i]);
            }
        }
        if constexpr (!EIGHT) {
            if (tile >= whole) {
                const bool wild = clean_v<DC>(&tiles[buf][v_frag][0], w, lane, tile, b.len);
                if (lane == 0) {
                    wild_lds[buf][w] = wild;
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                const uint32_t u = i * 256 + threadIdx.x;
                uint32_t at, then = 64;
                if (u < 128 * DC) {  // K: 16 dims of a key, or (an odd last 32) 8 dims of two keys
                    const uint32_t st = u / (32 * DC), rest = u % (32 * DC);
                    if (rest < 64 * KQ) {
                        at = (st * DC + rest / 64 * 2) * 64 + rest % 64;
                    } else {
                        at = (st * DC + DC - 1) * 64 + (rest - 64 * KQ) * 2;
                        then = 1;
                    }
                } else {  // V: 16 keys of a dim
                    const uint32_t r = u - 128 * DC;
                    at = (v_frag + r / 64 * 2) * 64 + r % 64;
                }
                to[at] = bytes_h8(next[i][0], next[i][1]);
                to[at + then] = bytes_h8(next[i][2], next[i][3]);
            }
            if (w == 0) {
                if (tile < whole) {
                    const int e = step_exp(wave_reduce_max(next_vs));
                    run_vexp = e > run_vexp ? e : run_vexp;
                    next_vs = ldexpf(next_vs, -run_vexp);
                }
                ks_lds[buf][lane] = next_ks * a.scale_log2e;
                vs_lds[buf][lane] = next_vs;
                if (lane == 0) {
                    vexp_lds[buf] = run_vexp;
                }
            }
        }
    };

    wave_rows<DC, RT, EIGHT, TREE> rows;
    {
        typename decltype(rows)::raw_q raw;
        rows.place(b, w * (RT * 16), lane);
        rows.load_q(a, b, raw);
        if (b.t_begin < b.t_end) {
            load(b.t_begin, 0);
            stage(b.t_begin, 0);
        }
        rows.take_q(a, b, raw);
    }
    __syncthreads();
    const bool k_in = !COPY || (DC - 1) * 32 + rows.G * 8 < a.hd;
    const auto step = [&](uint32_t buf, auto masked) {
        constexpr bool MASKED = decltype(masked)::value;
        const h8* from = &tiles[buf][0][lane];
        f4 s[RT][4];
        rows.template stream_k<4>(from, s, k_in);
        if constexpr (EIGHT) {
            if constexpr (!MASKED) {
                rows.raise_vexp(__builtin_amdgcn_readfirstlane(vexp_lds[buf]));
            }
            f4 ks[4], vm[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                ks[j] = *reinterpret_cast<const f4*>(&ks_lds[buf][score_key(4 * j, rows.G)]);
                vm[j] = *reinterpret_cast<const f4*>(&vs_lds[buf][score_key(4 * j, rows.G)]);
            }
            rows.template softmax<MASKED>(s, [&](int j) { return ks[j / 4][j % 4]; },
                                          [&](int j) { return vm[j / 4][j % 4]; });
        } else {
            rows.template softmax<MASKED>(s, [&](int) { return a.scale_log2e; }, [](int) { return 1.0f; });
        }
        if (!EIGHT && MASKED && any_wild(wild_lds[buf])) {
            rows.add_wild([&](int dt, int c) { return from[(v_frag + dt * 2 + c) * 64]; });
        } else {
            rows.template stream_v<4>(from + v_frag * 64);
        }
    };
    // Tiles that every row of the block sees whole, then the others, in loops
    // of their own: the masks would take the first one's registers.
    const auto run = [&](uint32_t from, uint32_t to, auto masked) {
        for (uint32_t tile = from; tile < to; ++tile) {
            const uint32_t buf = (tile - b.t_begin) & 1;
            const bool more = tile + 1 < b.t_end;
            if (masked.value) {  // (before the next loads: a wait for the words would wait for those too)
                rows.take_mask(a, b, tile * attend_tile);
            }
            if (more) {
                load(tile + 1, buf ^ 1);
            }
            if (tile * attend_tile < reach) {
                step(buf, masked);
            }
            if (more) {
                stage(tile + 1, buf ^ 1);
            }
            __syncthreads();
        }
    };
    run(b.t_begin, whole, std::false_type{});
    run(whole, b.t_end, std::true_type{});

    rows.finish();
    rows.store(a, b);
}

// ---- many rows: two groups of waves that take turns -----------------------------
// Eight waves of 32 rows; waves w and w + 4 share a SIMD. Between two barriers
// one group is in its matrix products (P V of a tile and K Q of the next), the
// other in its exponentials and in bringing tiles, so that a SIMD's matrix and
// vector units work at the same time; waves left to themselves were found in
// the same phase (matrix units 39 % busy, vector units 47 %, and hardly ever
// both). In interval 2 i group 0 takes the softmax of tile i, in 2 i + 1 its
// products; group 1 is one interval behind. The products of tile i read V(i)
// and K(i + 1), in buffers of their parity, in intervals 2 i + 1 and 2 i + 2.
// With the softmax of tile i, group 0 brings K(i + 1), in 2 i, and group 1
// V(i + 1), in 2 i + 1: each after the last read of what was there (K(i - 1)
// in 2 i - 2, V(i - 1) in 2 i) and before the first of what comes (2 i + 1, 2 i
// + 3). An 8-bit tile's steps(i + 2) come with group 1's products of tile i, in
// 2 i + 2; a group reads steps(i + 1) into registers at the end of its products
// of tile i, in 2 i + 1 and 2 i + 2, those of i being in registers by 2 i.
template <int DC, bool EIGHT, bool TREE>
__global__ __launch_bounds__(512, 2) void attend_turns_kernel(const attend_rows_args a) {
    using namespace attend;
    constexpr int RT = 2, KQ = DC / 2;
    constexpr int LOADS = (DC + 1) / 2;  // 16-byte units of an 8-bit tile's K or V per thread of a group
    typedef wave_rows<DC, RT, EIGHT, TREE> wave_rows_t;
    __shared__ h8 k_lds[2][4 * DC][64], v_lds[2][4 * DC][64];
    __shared__ float ks_lds[2][attend_tile], vs_lds[2][attend_tile];
    __shared__ int vexp_lds[2];
    __shared__ int wild_lds[2][attend_waves];  // with V

    const uint32_t lane = threadIdx.x % 64, in_group = threadIdx.x % 256;
    const uint32_t w = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const bool k_group = w < 4;  // group 0: brings K
    const block_place b = place_block<TREE>(a);
    const uint32_t n_rows = a.n * a.group;
    const uint32_t row0 = b.row0 + w * (RT * 16);
    const uint32_t open = TREE ? a.pos : a.pos + b.token0 + 1;  // keys that all the block's rows see
    // Keys that any of this wave's rows sees.
    const uint32_t reach = row0 >= n_rows ? 0
                           : TREE         ? b.len
                                          : a.pos + b.token0 + div_group(a, b.head0 + min(w * RT * 16 + RT * 16, n_rows - b.row0) - 1) + 1;

    const uint8_t* head = EIGHT ? a.kv8 + size_t{b.g} * a.tiles_per_head * a.tile_bytes : nullptr;
    const _Float16* kh = EIGHT ? nullptr : a.k + size_t{b.g} * a.hd;
    const _Float16* vh = EIGHT ? nullptr : a.vt + size_t{b.g} * a.hd * a.ctx_stride;
    u4 next[LOADS];
    float next_ks = 0.0f, next_vs = 0.0f;
    int run_vexp = no_vexp;  // wave 4's: the power of two of the steps staged for all rows
    const uint32_t whole = max(b.t_begin, min(b.t_end, open / attend_tile));  // from here on tiles are masked

    // This group's part (K or V) of a tile: 8-bit loads into registers, to be
    // staged; binary16 copies straight to their buffer.
    const auto load = [&](uint32_t tile) {
        if constexpr (EIGHT) {
            const uint8_t* t = head + size_t{tile} * a.tile_bytes + (k_group ? 0 : a.v_at);
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                const uint32_t u = i * 256 + in_group;
                next[i] = load16(t + (DC % 2 == 0 || u < 128 * DC ? u : 0) * 16);
            }
        } else {
            const uint32_t w4 = w % 4, G = lane / 16, m = lane % 16;
#pragma unroll
            for (int i = 0; i < DC; ++i) {
                const uint32_t f = i * 4 + w4;
                if (k_group) {
                    const uint32_t key = tile * attend_tile + operand_key(f / DC, m), d = f % DC * 32 + G * 8;
                    load16_lds(kh + size_t{key < b.len ? key : b.len - 1} * a.row + (d < a.hd ? d : 0),
                               &k_lds[tile & 1][f][0]);
                } else {
                    const uint32_t d = f / 2 * 16 + m, key = tile * attend_tile + f % 2 * 32 + G * 8;
                    load16_lds(vh + size_t{d < a.hd ? d : a.hd - 1} * a.ctx_stride + (key < a.ctx_stride ? key : 0),
                               &v_lds[tile & 1][f][0]);
                }
            }
        }
    };
    // What load started, to its buffer (and waited for).
    const auto stage = [&](uint32_t tile) {
        if constexpr (EIGHT) {
            h8* to = k_group ? &k_lds[tile & 1][0][0] : &v_lds[tile & 1][0][0];
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                const uint32_t u = i * 256 + in_group;
                uint32_t at = u / 64 * 128 + u % 64, then = 64;  // V, and K of whole 64s of dims
                if (DC % 2 != 0 && k_group) {
                    const uint32_t st = u / (32 * DC), rest = u % (32 * DC);
                    if (rest < 64 * KQ) {
                        at = (st * DC + rest / 64 * 2) * 64 + rest % 64;
                    } else {  // an odd last 32: 8 dims of two keys
                        at = (st * DC + DC - 1) * 64 + (rest - 64 * KQ) * 2;
                        then = 1;
                    }
                }
                if (DC % 2 == 0 || u < 128 * DC) {
                    to[at] = bytes_h8(next[i][0], next[i][1]);
                    to[at + then] = bytes_h8(next[i][2], next[i][3]);
                }
            }
        } else {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            if (!k_group && tile >= whole) {
                const bool wild = clean_v<DC>(&v_lds[tile & 1][0][0], w % 4, lane, tile, b.len);
                if (lane == 0) {
                    wild_lds[tile & 1][w % 4] = wild;
                }
            }
        }
    };
    const auto load_steps = [&](uint32_t tile) {
        if (EIGHT && w == 4 && tile < b.t_end) {
            const uint8_t* t = head + size_t{tile} * a.tile_bytes;
            next_ks = *reinterpret_cast<const float*>(t + a.ks_at + lane * 4);
            next_vs = *reinterpret_cast<const float*>(t + a.vs_at + lane * 4);
        }
    };
    const auto stage_steps = [&](uint32_t tile) {
        if (EIGHT && w == 4 && tile < b.t_end) {
            float vs = next_vs;
            if (tile < whole) {
                const int e = step_exp(wave_reduce_max(vs));
                run_vexp = e > run_vexp ? e : run_vexp;
                vs = ldexpf(vs, -run_vexp);
            }
            ks_lds[tile & 1][lane] = next_ks * a.scale_log2e;
            vs_lds[tile & 1][lane] = vs;
            if (lane == 0) {
                vexp_lds[tile & 1] = run_vexp;
            }
        }
    };
    const auto turn = [] {
        __builtin_amdgcn_sched_barrier(0);
        lds_barrier();
        __builtin_amdgcn_sched_barrier(0);
    };

    wave_rows_t rows;
    rows.place(b, w * (RT * 16), lane);
    f4 s[RT][4];
    f4 ks[4], vm[4];  // the steps of this lane's keys in the next softmax's tile
    int vexp = no_vexp;
    const auto read_steps = [&](uint32_t tile) {
        if constexpr (EIGHT) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                ks[j] = *reinterpret_cast<const f4*>(&ks_lds[tile & 1][score_key(4 * j, rows.G)]);
                vm[j] = *reinterpret_cast<const f4*>(&vs_lds[tile & 1][score_key(4 * j, rows.G)]);
            }
            vexp = vexp_lds[tile & 1];
        }
    };
    const bool k_in = (DC - 1) * 32 + lane / 16 * 8 < a.hd;
    const uint32_t t0 = b.t_begin, t1 = b.t_end;
    if (t0 < t1) {  // (a split of a causal run may lie behind all keys of these rows)
        // Before the turns: the first tile, its steps and the second one's; the
        // first scores; the loads that the first softmax stages.
        typename wave_rows_t::raw_q raw;
        rows.load_q(a, b, raw);
        load(t0);
        load_steps(t0);
        stage(t0);
        stage_steps(t0);
        load_steps(t0 + 1);
        stage_steps(t0 + 1);
        if (EIGHT && t0 + 1 < t1) {
            load(t0 + 1);
        }
        load_steps(t0 + 2);
        rows.take_q(a, b, raw);
        turn();
        read_steps(t0);
        if (t0 * attend_tile < reach) {
            rows.template stream_k<4>(&k_lds[t0 & 1][0][lane], s, k_in);
        }
        turn();
        if (!k_group) {
            turn();
        }
        const auto run = [&](uint32_t from, uint32_t to, auto masked) {
            constexpr bool MASKED = decltype(masked)::value;
            for (uint32_t tile = from; tile < to; ++tile) {
                const uint32_t key0 = tile * attend_tile;
                const bool more = tile + 1 < t1;
                if (MASKED) {  // (before the next loads: a wait for the words would wait for those too)
                    rows.take_mask(a, b, key0);
                }
                if (!EIGHT && more) {
                    load(tile + 1);
                }
                if (key0 < reach) {
                    if constexpr (EIGHT) {
                        if constexpr (!MASKED) {
                            rows.raise_vexp(__builtin_amdgcn_readfirstlane(vexp));
                        }
                        rows.template softmax<MASKED>(s, [&](int j) { return ks[j / 4][j % 4]; },
                                                      [&](int j) { return vm[j / 4][j % 4]; });
                    } else {
                        rows.template softmax<MASKED>(s, [&](int) { return a.scale_log2e; },
                                                      [](int) { return 1.0f; });
                    }
                }
                if (more) {
                    stage(tile + 1);
                }
                if (EIGHT && tile + 2 < t1) {
                    load(tile + 2);
                }
                turn();
                __builtin_amdgcn_s_setprio(1);
                if (key0 < reach) {  // (behind the last tile the scores are not used)
                    const h8* v_from = &v_lds[tile & 1][0][lane];
                    const h8* k_from = &k_lds[(tile + 1) & 1][0][lane];
                    if (!EIGHT && MASKED && any_wild(wild_lds[tile & 1])) {
                        rows.add_wild([&](int dt, int c) { return v_from[(dt * 2 + c) * 64]; });
                        rows.template stream_k<4>(k_from, s, k_in);
                    } else {
                        rows.template stream_vk<6>(v_from, k_from, s, k_in);
                    }
                }
                if constexpr (EIGHT) {
                    stage_steps(tile + 2);
                    load_steps(tile + 3);
                    read_steps(tile + 1);
                }
                __builtin_amdgcn_s_setprio(0);
                turn();
            }
        };
        run(t0, whole, std::false_type{});
        run(whole, t1, std::true_type{});
        if (k_group) {
            turn();
        }
    }
    rows.finish();
    rows.store(a, b);
}

template <class KERNEL>
hipError_t launch_attend_blocks(KERNEL kernel, uint32_t threads, const attend_rows_args& a, hipStream_t stream) {
    if (a.row_blocks > attend_max_row_blocks || a.group > attend_max_group) {
        return hipErrorInvalidValue;
    }
    kernel<<<dim3(a.n_kv, a.splits, a.row_blocks), threads, 0, stream>>>(a);
    if (hipError_t e = hipGetLastError(); e != hipSuccess || a.splits == 1) {
        return e;
    }
    return launch_attend_merge(a, stream);
}

}  // namespace syn
