// attend_rows.hpp — attention of a run's query rows over a KV state, for the
// states and masks the decode and prefill kernels do not take: 8-bit states
// (attend_kv8.hip), and drafted trees over either kind (attend_tree.hip).
//
//   out_r = sum_t p_rt v_t / sum_t p_rt,  p_rt = exp(scale q_r . k_t - m_r)
//
// over the keys t that row r sees, in one pass with a running maximum m.
//
// Rows. The query rows of a KV head are (token, head) pairs, r = token *
// group + head: a key or value byte serves all of them. Two kernels share the
// arithmetic here:
//  - up to 16 rows (a decode step): a wave takes all of them and every fourth
//    tile of 64 keys of the block's split, straight from memory into operand
//    registers, and the block's four waves meet in LDS at the end. Bound by
//    HBM, so nothing is shared and no barrier is in the loop.
//  - more rows: each of the four waves has 16 or 32 of its own, and the tiles
//    of keys, which they all need, come through LDS as operands (two buffers,
//    one barrier a tile). Bound by the matrix cores, the exponentials and
//    LDS, which are about even at 32 rows a wave.
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
// held against the power of two above the largest step so far (`vexp`), so
// steps of any size keep that range.
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

// Bits 0..7 of draft row `bits` from drafted token j on (j may start before
// the first or end past the last): whole words in range, so no read is
// outside the row's `words` words.
__device__ __forceinline__ uint32_t mask_bits8(const uint32_t* bits, uint32_t words, uint32_t n, int j) {
    const int w = j >> 5;  // rounds down
    const uint32_t lo = w >= 0 && w < static_cast<int>(words) ? bits[w] : 0u;
    const uint32_t hi = w + 1 >= 0 && w + 1 < static_cast<int>(words) ? bits[w + 1] : 0u;
    const uint64_t both = (uint64_t{hi} << 32 | lo) >> (j & 31);
    const int left = static_cast<int>(n) - j;  // bits past the last token are ignored
    return static_cast<uint32_t>(both) & (left >= 8 ? 0xffu : left > 0 ? (1u << left) - 1u : 0u);
}

// Weight of a part (max, sum) of a row whose maximum is top.
__device__ __forceinline__ float part_weight(float m, float l, float top) {
    return l == 0.0f ? 0.0f : l * fast_exp2(m - top);  // (l == 0: nothing seen, m may be -inf)
}

// The exponent of the power of two above the largest of a tile's V steps
// (`top`, the same in every lane), or no_vexp.
__device__ __forceinline__ int step_exp(float top) {
    return __builtin_amdgcn_readfirstlane(top > 0.0f ? __builtin_amdgcn_frexp_expf(top) : no_vexp);
}

// RT tiles of 16 query rows that one wave holds: lane 16 G + col has column
// col of every tile.
template <int DC, int RT, bool EIGHT, bool TREE>
struct wave_rows {
    static constexpr int DT = 2 * DC;
    uint32_t G, col, row0;
    uint32_t limit[RT];         // keys seen without the mask (0: no row)
    const uint32_t* draft[RT];  // the row's mask
    h8 q[RT][DC];
    f4 acc[RT][DT];             // O^T: dims 16 dt + 4 G .. + 3
    float mref[RT], l[RT];      // the running maximum less p_shift; the sum of this lane's keys
    h8 hi[RT][2], lo[RT][2];    // the last step's probabilities
    uint32_t seen[RT];          // its keys that the row sees, by score
    int vexp;

    // Starts the rows' loads (f32 rows raw, to be rounded by take_q).
    struct raw_q {
        f4 x[RT][DC][2];
    };
    __device__ __forceinline__ void place(const attend_rows_args& a, uint32_t g, uint32_t first, uint32_t lane,
                                          raw_q& raw) {
        G = lane / 16;
        col = lane % 16;
        row0 = first;
        vexp = no_vexp;
        const uint32_t rows = a.n * a.group;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const uint32_t r = row0 + rt * 16 + col;
            const bool in = r < rows;
            const uint32_t token = in ? r / a.group : 0, head = in ? g * a.group + r % a.group : 0;
            limit[rt] = !in ? 0 : TREE ? a.pos : a.pos + token + 1;
            if constexpr (TREE) {
                draft[rt] = a.mask + size_t{token} * a.mask_words;
            }
            mref[rt] = no_max;
            l[rt] = 0.0f;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                acc[rt][dt] = f4{0, 0, 0, 0};
            }
            const size_t at = size_t{token} * a.q_row + head * a.hd;
#pragma unroll
            for (int dc = 0; dc < DC; ++dc) {
                const uint32_t d = k_dim<DC, EIGHT>(dc, G);
                if (a.hd % 8 == 0) {
                    const size_t i = d < a.hd ? at + d : 0;
                    if (a.q_f16) {
                        raw.x[rt][dc][0] = __builtin_bit_cast(f4, load16(static_cast<const _Float16*>(a.q) + i));
                    } else {
                        raw.x[rt][dc][0] = *reinterpret_cast<const f4*>(static_cast<const float*>(a.q) + i);
                        raw.x[rt][dc][1] = *reinterpret_cast<const f4*>(static_cast<const float*>(a.q) + i + 4);
                    }
                } else {
                    h8 x;
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const size_t i = d + e < a.hd ? at + d + e : 0;
                        x[e] = a.q_f16 ? static_cast<const _Float16*>(a.q)[i] : to_h(static_cast<const float*>(a.q)[i]);
                        x[e] = d + e < a.hd ? x[e] : static_cast<_Float16>(0);
                    }
                    raw.x[rt][dc][0] = __builtin_bit_cast(f4, x);
                }
            }
        }
    }
    __device__ __forceinline__ void take_q(const attend_rows_args& a, const raw_q& raw) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
            for (int dc = 0; dc < DC; ++dc) {
                const f4 x = raw.x[rt][dc][0], y = raw.x[rt][dc][1];
                h8 h = __builtin_bit_cast(h8, x);
                if (a.hd % 8 == 0) {
                    if (!a.q_f16) {
                        h = h8{to_h(x[0]), to_h(x[1]), to_h(x[2]), to_h(x[3]), to_h(y[0]), to_h(y[1]), to_h(y[2]),
                               to_h(y[3])};
                    }
                    if (k_dim<DC, EIGHT>(dc, G) >= a.hd) {
                        h = as_h8(zero_u4());
                    }
                }
                q[rt][dc] = h;
            }
        }
    }

    // The steps' power of two is now e: what is summed already goes with it.
    __device__ __forceinline__ void raise_vexp(int e) {
        if (e > vexp) {
            const float f = vexp == no_vexp ? 0.0f : ldexpf(1.0f, vexp - e);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) {
                    acc[rt][dt] *= f;
                }
            }
            vexp = e;
        }
    }

    // Scores of the tile at key0 to probabilities, split into hi and lo. ks: the
    // keys' K steps times the scale in exp2's units (or that scale alone); vm:
    // their V steps over 2^vexp. MASKED: some row may not see some of the
    // tile's keys. While no lane has a score more than `lazy` above its row's
    // maximum, lanes need nothing from each other.
    template <bool MASKED, class KS, class VM>
    __device__ __forceinline__ void softmax(const attend_rows_args& a, const f4 (&s)[RT][4], uint32_t key0, KS ks,
                                            VM vm) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            uint32_t bits = 0xffffu;
            if constexpr (MASKED) {
                bits = 0;
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const uint32_t k0 = key0 + score_key(8 * c, G);
                    const uint32_t left = limit[rt] > k0 ? limit[rt] - k0 : 0;
                    uint32_t b = left >= 8 ? 0xffu : (1u << left) - 1u;
                    if constexpr (TREE) {
                        if (row0 + rt * 16 + col < a.n * a.group) {
                            b |= mask_bits8(draft[rt], a.mask_words, a.n, static_cast<int>(k0 - a.pos));
                        }
                    }
                    bits |= b << (8 * c);
                }
            }
            seen[rt] = bits;
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
                if constexpr (EIGHT) {
                    p[j] *= vm(j);
                }
            }
            if constexpr (EIGHT && MASKED) {  // a masked key's step may be NaN
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    p[j] = bits >> j & 1 ? p[j] : 0.0f;
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

    // O^T += V^T P^T for 16 dims and 32 keys.
    __device__ __forceinline__ void add_v(int dt, int c, h8 v) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            acc[rt][dt] = mfma16(v, hi[rt][c], acc[rt][dt]);
            acc[rt][dt] = mfma16(v, lo[rt][c], acc[rt][dt]);
        }
    }
    // The same in a tile of a binary16 state that holds drafted rows, or ends
    // before its end: of v's keys the first `left` are there, and a value that
    // is infinite or NaN, which as an operand would reach the rows that do not
    // see it (0 times it is NaN), gets products of its own: a row has +inf
    // added where it sees a +inf or NaN among the 32 keys, and -inf where it
    // sees a -inf or NaN (so NaN where both).
    __device__ __forceinline__ void add_v_tail(int dt, int c, h8 v, uint32_t left) {
        h8 finite;
        bool any = false;
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e) {
            const _Float16 x = v[e];  // (a bit cast of the element itself casts element 0)
            const unsigned short b = __builtin_bit_cast(unsigned short, x);
            const bool wild = (b & 0x7c00u) == 0x7c00u;
            finite[e] = e < left && !wild ? x : static_cast<_Float16>(0);
            any = any || (e < left && wild);
        }
        add_v(dt, c, finite);
        if (any_lane(any)) {
            h8 up, down;
#pragma unroll
            for (uint32_t e = 0; e < 8; ++e) {
                const _Float16 x = v[e];
                const unsigned short b = __builtin_bit_cast(unsigned short, x);
                const bool wild = e < left && (b & 0x7c00u) == 0x7c00u, nan = (b & 0x3ffu) != 0;
                up[e] = static_cast<_Float16>(wild && (nan || b >> 15 == 0) ? 1.0f : 0.0f);
                down[e] = static_cast<_Float16>(wild && (nan || b >> 15 != 0) ? 1.0f : 0.0f);
            }
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
                    if (vexp != no_vexp) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            acc[rt][dt][e] = ldexpf(acc[rt][dt][e], vexp);
                        }
                    }
                }
            }
        }
    }
};

// Where a row's output goes: the output itself, or its split's part.
__device__ __forceinline__ float* row_out(const attend_rows_args& a, uint32_t g, uint32_t split, uint32_t r) {
    if (a.splits == 1) {
        return a.out + size_t{r / a.group} * a.q_row + (g * a.group + r % a.group) * a.hd;
    }
    return a.part + ((size_t{split} * a.n_kv + g) * (a.n * a.group) + r) * a.hd;
}
__device__ __forceinline__ void store_part(const attend_rows_args& a, uint32_t g, uint32_t split, uint32_t r, float m,
                                           float l) {
    *reinterpret_cast<f2*>(a.part_ml + ((size_t{split} * a.n_kv + g) * (a.n * a.group) + r) * 2) = f2{m, l};
}

// A block's place: KV heads fastest (with 8 of them each XCD keeps to one,
// whose L2 then serves all row blocks), then splits, the last row blocks
// first (a causal run's longest).
struct block_place {
    uint32_t g, split, row0, len, t_begin, t_end;
};
template <bool TREE>
__device__ __forceinline__ block_place place_block(const attend_rows_args& a) {
    block_place b;
    b.g = blockIdx.x % a.n_kv;
    b.split = blockIdx.x / a.n_kv % a.splits;
    b.row0 = (a.row_blocks - 1 - blockIdx.x / a.n_kv / a.splits) * a.block_rows;
    const uint32_t rows = a.n * a.group;
    const uint32_t last = min(b.row0 + a.block_rows, rows) - 1;
    b.len = TREE ? a.pos + a.n : a.pos + last / a.group + 1;  // up to the last row's last key
    const uint32_t tiles = (b.len + attend_tile - 1) / attend_tile;
    b.t_begin = b.split * a.chunk;
    b.t_end = min(tiles, b.t_begin + a.chunk);
    return b;
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
    __device__ __forceinline__ h8 k(int st, int dc) const {
        return kq[st][dc];
    }
    __device__ __forceinline__ h8 v(int dt, int c) const {
        return vq[dt][c];
    }
};

}  // namespace attend

// grid: splits x KV heads (one row block); block 256.
template <int DC, class SRC, bool TREE>
__global__ __launch_bounds__(256) void attend_few_kernel(const attend_rows_args a) {
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
    rows.place(a, b.g, 0, lane, raw);
    SRC src(a, b.g, b.len);
    uint32_t tile = b.t_begin + w;
    if (tile < b.t_end) {
        src.load(tile, lane);
    }
    rows.take_q(a, raw);

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
        const uint32_t key0 = tile * attend_tile;
        if constexpr (SRC::eight) {
            float vm[16];
            float top = 0.0f;
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                vm[j] = src.vs[j / 4][j % 4];
                if constexpr (MASKED) {  // past the last key the steps may be anything
                    vm[j] = key0 + score_key(j, rows.G) < b.len ? vm[j] : 0.0f;
                }
                top = fmaxf(top, vm[j]);
            }
            rows.raise_vexp(step_exp(max32(max16(top))));
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                vm[j] = ldexpf(vm[j], -rows.vexp);
            }
            rows.template softmax<MASKED>(a, s, key0, [&](int j) { return src.ks[j / 4][j % 4] * a.scale_log2e; },
                                          [&](int j) { return vm[j]; });
        } else {
            rows.template softmax<MASKED>(a, s, key0, [&](int) { return a.scale_log2e; }, [](int) { return 1.0f; });
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const uint32_t key = key0 + score_key(8 * c, rows.G);
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                if constexpr (!SRC::eight && MASKED) {
                    rows.add_v_tail(dt, c, src.v(dt, c), b.len > key ? b.len - key : 0);
                } else {
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
        *reinterpret_cast<f2*>(row_out(a, b.g, b.split, r) + d) = o;
        if (a.splits > 1 && d == 0) {
            store_part(a, b.g, b.split, r, top, sum);
        }
    }
}

// ---- more rows: waves own rows, tiles come through LDS -------------------------
// grid: splits x row blocks x KV heads; block 256. A buffer holds a tile as
// operands in lane order: K (st, dc), then V (dt, c), 1 KiB each, so every
// LDS access is 64 neighbouring 16-byte units.
template <int DC, int RT, bool EIGHT, bool WHOLE8, bool TREE>
__global__ __launch_bounds__(256, DC <= 4 ? 2 : 1) void attend_many_kernel(const attend_rows_args a) {
    using namespace attend;
    constexpr int DT = 2 * DC;
    constexpr int KQ = DC / 2;
    constexpr uint32_t v_frag = 4 * DC;          // first V operand
    constexpr bool COPY = !EIGHT && WHOLE8;      // binary16 operands, copied to LDS as they are
    constexpr int LOADS = EIGHT ? DC : 2 * DC;   // 16-byte units of a tile per thread
    __shared__ h8 tiles[2][8 * DC][64];
    __shared__ float ks_lds[2][attend_tile], vs_lds[2][attend_tile];
    __shared__ int vexp_lds[2];

    const uint32_t lane = threadIdx.x % 64;
    const uint32_t w = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const block_place b = place_block<TREE>(a);
    const uint32_t n_rows = a.n * a.group;
    const uint32_t row0 = b.row0 + w * (RT * 16);
    const bool has_rows = row0 < n_rows;
    const uint32_t open = TREE ? a.pos : a.pos + b.row0 / a.group + 1;  // keys that all the block's rows see
    // Keys that any of this wave's rows sees.
    const uint32_t reach = !has_rows ? 0 : TREE ? b.len : a.pos + (min(row0 + RT * 16, n_rows) - 1) / a.group + 1;

    const uint8_t* head = EIGHT ? a.kv8 + size_t{b.g} * a.tiles_per_head * a.tile_bytes : nullptr;
    const _Float16* kh = EIGHT ? nullptr : a.k + size_t{b.g} * a.hd;
    const _Float16* vh = EIGHT ? nullptr : a.vt + size_t{b.g} * a.hd * a.ctx_stride;
    u4 next[COPY ? 1 : LOADS];
    float next_ks = 0.0f, next_vs = 0.0f;
    int run_vexp = no_vexp;  // wave 0's: the steps' power of two up to the staged tile

    // A tile's loads into registers, or (binary16) copies to buffer buf.
    const auto load = [&](uint32_t tile, uint32_t buf) {
        if constexpr (EIGHT) {
            const uint8_t* t = head + size_t{tile} * a.tile_bytes;
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                next[i] = load16(t + (i * 256 + threadIdx.x) * 16);
            }
            if (w == 0) {
                const bool in = tile * attend_tile + lane < b.len;  // past the last key the steps may be anything
                const float x = *reinterpret_cast<const float*>(t + a.ks_at + lane * 4);
                const float y = *reinterpret_cast<const float*>(t + a.vs_at + lane * 4);
                next_ks = in ? x : 0.0f;
                next_vs = in ? y : 0.0f;
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
    const auto stage = [&](uint32_t buf) {
        h8* to = &tiles[buf][0][0];
        if constexpr (COPY) {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        } else if constexpr (!EIGHT) {
#pragma unroll
            for (int i = 0; i < DC; ++i) {
                to[(i * 4 + w) * 64 + lane] = as_h8(next[i]);
                to[(v_frag + i * 4 + w) * 64 + lane] = as_h8(next[DC + i]);
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
                const int e = step_exp(wave_reduce_max(next_vs));
                run_vexp = e > run_vexp ? e : run_vexp;
                ks_lds[buf][lane] = next_ks * a.scale_log2e;
                vs_lds[buf][lane] = ldexpf(next_vs, -run_vexp);
                if (lane == 0) {
                    vexp_lds[buf] = run_vexp;
                }
            }
        }
    };

    wave_rows<DC, RT, EIGHT, TREE> rows;
    {
        typename decltype(rows)::raw_q raw;
        rows.place(a, b.g, row0, lane, raw);
        if (b.t_begin < b.t_end) {
            load(b.t_begin, 0);
            stage(0);
        }
        rows.take_q(a, raw);
    }
    __syncthreads();
    const bool k_in = (DC - 1) * 32 + rows.G * 8 < a.hd;  // the lane's last eight dims are the head's
    const auto step = [&](uint32_t key0, uint32_t buf, auto masked) {
        constexpr bool MASKED = decltype(masked)::value;
        const h8* from = &tiles[buf][0][lane];
        f4 s[RT][4];
#pragma unroll
        for (int st = 0; st < 4; ++st) {
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                s[rt][st] = f4{0, 0, 0, 0};
            }
#pragma unroll
            for (int dc = 0; dc < DC; ++dc) {
                h8 k = from[(st * DC + dc) * 64];
                if constexpr (COPY) {
                    if (dc == DC - 1) {  // (what follows is the next head's, and could be NaN)
                        k = as_h8(k_in ? as_u4(k) : zero_u4());
                    }
                }
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    s[rt][st] = mfma16(k, rows.q[rt][dc], s[rt][st]);
                }
            }
        }
        if constexpr (EIGHT) {
            rows.raise_vexp(__builtin_amdgcn_readfirstlane(vexp_lds[buf]));
            f4 ks[4], vm[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                ks[j] = *reinterpret_cast<const f4*>(&ks_lds[buf][score_key(4 * j, rows.G)]);
                vm[j] = *reinterpret_cast<const f4*>(&vs_lds[buf][score_key(4 * j, rows.G)]);
            }
            rows.template softmax<MASKED>(a, s, key0, [&](int j) { return ks[j / 4][j % 4]; },
                                          [&](int j) { return vm[j / 4][j % 4]; });
        } else {
            rows.template softmax<MASKED>(a, s, key0, [&](int) { return a.scale_log2e; }, [](int) { return 1.0f; });
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const uint32_t key = key0 + score_key(8 * c, rows.G);
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                const h8 v = from[(v_frag + dt * 2 + c) * 64];
                if constexpr (!EIGHT && MASKED) {
                    rows.add_v_tail(dt, c, v, b.len > key ? b.len - key : 0);
                } else {
                    rows.add_v(dt, c, v);
                }
            }
        }
    };
    // Tiles that every row of the block sees whole, then the others, in loops
    // of their own: the masks would take the first one's registers.
    const auto run = [&](uint32_t from, uint32_t to, auto masked) {
        for (uint32_t tile = from; tile < to; ++tile) {
            const uint32_t buf = (tile - b.t_begin) & 1;
            const bool more = tile + 1 < b.t_end;
            if (more) {
                load(tile + 1, buf ^ 1);
            }
            if (tile * attend_tile < reach) {
                step(tile * attend_tile, buf, masked);
            }
            if (more) {
                stage(buf ^ 1);
            }
            __syncthreads();
        }
    };
    const uint32_t whole = max(b.t_begin, min(b.t_end, open / attend_tile));
    run(b.t_begin, whole, std::false_type{});
    run(whole, b.t_end, std::true_type{});

    rows.finish();
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const uint32_t r = row0 + rt * 16 + rows.col;
        if (r < n_rows) {
            float* out = row_out(a, b.g, b.split, r);
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                const uint32_t d = dt * 16 + rows.G * 4;
                const f4 o = rows.acc[rt][dt];
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
            if (a.splits > 1 && rows.G == 0) {
                store_part(a, b.g, b.split, r, rows.mref[rt], rows.l[rt]);
            }
        }
    }
}

template <class KERNEL>
hipError_t launch_attend_blocks(KERNEL kernel, const attend_rows_args& a, hipStream_t stream) {
    const uint64_t blocks = uint64_t{a.row_blocks} * a.n_kv * a.splits;
    if (blocks > 0x7fffffffu) {
        return hipErrorInvalidValue;
    }
    kernel<<<static_cast<uint32_t>(blocks), 256, 0, stream>>>(a);
    if (hipError_t e = hipGetLastError(); e != hipSuccess || a.splits == 1) {
        return e;
    }
    return launch_attend_merge(a, stream);
}

}  // namespace syn
