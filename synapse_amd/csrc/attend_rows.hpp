// attend_rows.hpp — attention of a run's query rows over a KV state, for the
// states and masks the decode and prefill kernels do not take: 8-bit states
// (attend_kv8.hip), and drafted trees over either kind (attend_tree.hip).
//
//   out_r = sum_t p_rt v_t / sum_t p_rt,  p_rt = exp(scale q_r . k_t - m_r)
//
// over the keys t that row r sees, in one pass with a running maximum m.
//
// Rows. The query rows of a KV head are (token, head) pairs, r = token *
// group + head: a key or value byte serves all of them. A block takes up to
// 64 rows (RT tiles of 16) and a split of the keys; its 4 waves take every
// fourth tile of 64 keys each and meet in LDS at the end. Splits of one row
// block meet in a second, small kernel (attend_merge). Nothing is shared
// while the keys go by, so there is no barrier in the loop.
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

namespace syn {

namespace attend {

constexpr float p_shift = 6.0f;  // probabilities are 2^6 exp2(s - m)
constexpr float lazy = 8.0f;     // a maximum follows once a score is 2^8 above it

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

__device__ __forceinline__ bool any_lane(bool x) {
    return __builtin_amdgcn_ballot_w64(x) != 0;
}

// The keys of one wave's step as matrix-core operands. K operand (st, dc): 16
// keys of score operand st, dims k_dim(dc) of each lane; V operand (dt, c):
// 16 dims, keys 32 c + 8 G .. + 7 of each lane.
template <int DC>
struct kv8_source {
    static constexpr bool steps = true;
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

    // First dim of a lane's eight in k-step dc.
    __device__ static __forceinline__ uint32_t k_dim(int dc, uint32_t G) {
        return dc < 2 * KQ ? dc / 2 * 64 + G * 16 + dc % 2 * 8 : dc * 32 + G * 8;
    }
    __device__ __forceinline__ void load_k(uint32_t tile, uint32_t lane) {
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
        for (int j = 0; j < 4; ++j) {  // keys 32 (j / 2) + 8 G + 4 (j % 2) .. + 3
            ks[j] = *reinterpret_cast<const f4*>(t + ks_at + (j / 2 * 32 + G * 8 + j % 2 * 4) * 4);
        }
    }
    __device__ __forceinline__ void load_v(uint32_t tile, uint32_t lane) {
        const uint8_t* t = head + tile * tile_bytes;
        const uint32_t G = lane / 16;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            vs[j] = *reinterpret_cast<const f4*>(t + vs_at + (j / 2 * 32 + G * 8 + j % 2 * 4) * 4);
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
    static constexpr bool steps = false;
    const _Float16* kh;    // the KV head's column of K rows
    const _Float16* vh;    // its V^T rows
    size_t row, ctx_stride;
    uint32_t hd, len;
    h8 kq[4][DC];
    h8 vq[2 * DC][2];

    __device__ __forceinline__ f16_source(const attend_rows_args& a, uint32_t g, uint32_t length)
        : kh(a.k + size_t{g} * a.hd), vh(a.vt + size_t{g} * a.hd * a.ctx_stride), row(a.row),
          ctx_stride(a.ctx_stride), hd(a.hd), len(length) {}

    __device__ static __forceinline__ uint32_t k_dim(int dc, uint32_t G) {
        return dc * 32 + G * 8;
    }
    // Keys past the last one are read from the last one (their scores are
    // masked); dims past the head's are zeros (the next head's could be NaN).
    __device__ __forceinline__ void load_k(uint32_t tile, uint32_t lane) {
        const uint32_t G = lane / 16, m = lane % 16;
#pragma unroll
        for (int st = 0; st < 4; ++st) {
            const uint32_t key = tile * attend_tile + st / 2 * 32 + m / 4 * 8 + st % 2 * 4 + m % 4;
            const _Float16* p = kh + (key < len ? key : len - 1) * row;
#pragma unroll
            for (int dc = 0; dc < DC; ++dc) {
                const uint32_t d = k_dim(dc, G);
                if constexpr (WHOLE8) {
                    const bool in = dc < DC - 1 || d < hd;
                    const u4 x = load16(p + (in ? d : 0));
                    kq[st][dc] = as_h8(in ? x : zero_u4());
                } else {
#pragma unroll
                    for (int e = 0; e < 8; e += 2) {  // hd is even: pairs are 4-byte aligned
                        const bool in = d + e < hd;
                        const h2 x = *reinterpret_cast<const h2*>(p + (in ? d + e : 0));
                        kq[st][dc][e] = in ? x[0] : static_cast<_Float16>(0);
                        kq[st][dc][e + 1] = in ? x[1] : static_cast<_Float16>(0);
                    }
                }
            }
        }
    }
    // ctx_stride is a multiple of 8, so eight keys are in the row or past it;
    // dims past the head's are read from its last one and not written out.
    __device__ __forceinline__ void load_v(uint32_t tile, uint32_t lane) {
        const uint32_t G = lane / 16, m = lane % 16;
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
    // Zeroes the values of keys past the last one, and says whether those
    // left hold an infinity or NaN anywhere in the wave.
    __device__ __forceinline__ bool clear_past(uint32_t tile, uint32_t lane) {
        const uint32_t G = lane / 16;
        bool wild = false;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const uint32_t key = tile * attend_tile + c * 32 + G * 8;
            const uint32_t left = len > key ? len - key : 0;
#pragma unroll
            for (int dt = 0; dt < 2 * DC; ++dt) {
#pragma unroll
                for (uint32_t e = 0; e < 8; ++e) {
                    const _Float16 x = vq[dt][c][e];  // (a bit cast of the element itself casts element 0)
                    const unsigned short b = __builtin_bit_cast(unsigned short, x);
                    vq[dt][c][e] = e < left ? x : static_cast<_Float16>(0);
                    wild = wild || (e < left && (b & 0x7c00u) == 0x7c00u);
                }
            }
        }
        return any_lane(wild);
    }
};

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

}  // namespace attend

// grid: splits x row blocks x KV heads, KV heads fastest (with 8 of them each
// XCD keeps to one, whose L2 then serves all row blocks), then splits, the
// last row blocks first (a causal run's longest); block 256.
template <int DC, int RT, class SRC, bool TREE>
__global__ __launch_bounds__(256) void attend_rows_kernel(const attend_rows_args a) {
    using namespace attend;
    constexpr int DT = 2 * DC;
    constexpr uint32_t pitch = DC * 32 + 4;
    __shared__ float lds_o[attend_waves][16][pitch];
    __shared__ float lds_m[attend_waves][RT * 16], lds_l[attend_waves][RT * 16];

    const uint32_t lane = threadIdx.x % 64, G = lane / 16, col = lane % 16;
    const uint32_t w = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const uint32_t g = blockIdx.x % a.n_kv;
    const uint32_t split = blockIdx.x / a.n_kv % a.splits;
    const uint32_t row0 = (a.row_blocks - 1 - blockIdx.x / a.n_kv / a.splits) * (RT * 16);
    const uint32_t rows = a.n * a.group;

    // The block's keys: up to the last row's last one.
    const uint32_t last = (row0 + RT * 16 < rows ? row0 + RT * 16 : rows) - 1;
    const uint32_t len = TREE ? a.pos + a.n : a.pos + last / a.group + 1;
    const uint32_t open = TREE ? a.pos : a.pos + row0 / a.group + 1;  // keys that every row sees
    const uint32_t tiles = (len + attend_tile - 1) / attend_tile;
    const uint32_t t_end = min(tiles, (split + 1) * a.chunk);

    // Q operands and each lane's rows.
    h8 q[RT][DC];
    uint32_t limit[RT];              // keys seen without the mask
    const uint32_t* draft[RT];       // the row's mask
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const uint32_t r = row0 + rt * 16 + col;
        const bool in = r < rows;
        const uint32_t token = in ? r / a.group : 0, head = in ? g * a.group + r % a.group : 0;
        limit[rt] = !in ? 0 : TREE ? a.pos : a.pos + token + 1;
        draft[rt] = a.mask + size_t{token} * a.mask_words;
        const size_t at = size_t{token} * a.q_row + head * a.hd;
#pragma unroll
        for (int dc = 0; dc < DC; ++dc) {
            const uint32_t d0 = SRC::k_dim(dc, G);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const bool has = in && d0 + e < a.hd;
                const size_t i = has ? at + d0 + e : 0;
                const _Float16 x = a.q_f16 ? static_cast<const _Float16*>(a.q)[i]
                                           : to_h(static_cast<const float*>(a.q)[i]);
                q[rt][dc][e] = has ? x : static_cast<_Float16>(0);
            }
        }
    }

    f4 acc[RT][DT];
    float mref[RT], l[RT];  // the running maximum less p_shift; the sum of this lane's keys
    int vexp = -1000;       // 2^vexp is over every V step so far
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        mref[rt] = -INFINITY;
        l[rt] = 0.0f;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
            acc[rt][dt] = f4{0, 0, 0, 0};
        }
    }

    SRC src(a, g, len);
    for (uint32_t tile = split * a.chunk + w; tile < t_end; tile += attend_waves) {
        src.load_k(tile, lane);
        src.load_v(tile, lane);
        f4 s[RT][4];
#pragma unroll
        for (int st = 0; st < 4; ++st) {
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                s[rt][st] = f4{0, 0, 0, 0};
            }
#pragma unroll
            for (int dc = 0; dc < DC; ++dc) {
                const h8 k = src.k(st, dc);
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    s[rt][st] = mfma16(k, q[rt][dc], s[rt][st]);
                }
            }
        }
        const uint32_t key0 = tile * attend_tile;
        const bool masked = key0 + attend_tile > open;
        bool wild = false;
        float vmul[16];  // a key's V step over 2^vexp
        if constexpr (SRC::steps) {
            float top = 0.0f;
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const uint32_t key = key0 + j / 8 * 32 + G * 8 + j % 8;
                vmul[j] = key < len ? src.vs[j / 4][j % 4] : 0.0f;  // (past the last key the steps may be anything)
                top = fmaxf(top, vmul[j]);
            }
            top = max32(max16(top));
            const int e = __builtin_amdgcn_readfirstlane(top > 0.0f ? __builtin_amdgcn_frexp_expf(top) : -1000);
            if (e > vexp) {
                const float f = vexp == -1000 ? 0.0f : ldexpf(1.0f, vexp - e);
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt) {
                        acc[rt][dt] *= f;
                    }
                }
                vexp = e;
            }
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                vmul[j] = ldexpf(vmul[j], -vexp);
            }
        } else if (masked) {
            wild = src.clear_past(tile, lane);
        }
        h8 hi[RT][2], lo[RT][2];
        uint32_t seen[RT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            float p[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) {  // key 32 (j / 8) + 8 G + j % 8
                const float x = s[rt][j / 4][j % 4];
                if constexpr (SRC::steps) {
                    p[j] = x * (src.ks[j / 4][j % 4] * a.scale_log2e);
                } else {
                    p[j] = x * a.scale_log2e;
                }
            }
            seen[rt] = 0xffffu;
            if (masked) {
                uint32_t bits = 0;
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const uint32_t k0 = key0 + c * 32 + G * 8;
                    const uint32_t left = limit[rt] > k0 ? limit[rt] - k0 : 0;
                    uint32_t b = left >= 8 ? 0xffu : (1u << left) - 1u;
                    if constexpr (TREE) {
                        if (row0 + rt * 16 + col < rows) {
                            b |= mask_bits8(draft[rt], a.mask_words, a.n, static_cast<int>(k0 - a.pos));
                        }
                    }
                    bits |= b << (8 * c);
                }
                seen[rt] = bits;
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
            top = max32(max16(top));
            const bool follow = top - p_shift > mref[rt] + lazy;
            if (any_lane(follow)) {
                const float m = follow ? top - p_shift : mref[rt];
                const float f = follow ? fast_exp2(mref[rt] - m) : 1.0f;
                mref[rt] = m;
                l[rt] *= f;
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) {
                    acc[rt][dt] *= f;
                }
            }
            const float m = mref[rt] == -INFINITY ? 0.0f : mref[rt];
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                p[j] = fast_exp2(p[j] - m);
                l[rt] += p[j];
                if constexpr (SRC::steps) {
                    // A masked key's step may be NaN.
                    p[j] = seen[rt] >> j & 1 ? p[j] * vmul[j] : 0.0f;
                }
                const _Float16 h = to_h(p[j]);
                hi[rt][j / 8][j % 8] = h;
                lo[rt][j / 8][j % 8] = to_h(p[j] - static_cast<float>(h));
                s[rt][j / 4][j % 4] = p[j];
            }
        }
        if constexpr (!SRC::steps) {
            if (wild) {
                // Some value among the drafted rows is infinite or NaN: on
                // the matrix core it would reach the rows that do not see
                // it. Key by key, each row's own keys only.
                for (int j = 0; j < 16; ++j) {
                    for (uint32_t G2 = 0; G2 < 4; ++G2) {
#pragma unroll
                        for (int rt = 0; rt < RT; ++rt) {
                            float mine = 0.0f;
#pragma unroll
                            for (int i = 0; i < 16; ++i) {
                                mine = i == j ? s[rt][i / 4][i % 4] : mine;
                            }
                            const float pj = __shfl(mine, static_cast<int>(G2 * 16 + col));
                            const uint32_t sees = __shfl(static_cast<int>(seen[rt]), static_cast<int>(G2 * 16 + col));
                            const uint32_t key = key0 + j / 8 * 32 + G2 * 8 + j % 8;
                            if (sees >> j & 1) {
#pragma unroll
                                for (int dt = 0; dt < DT; ++dt) {
#pragma unroll
                                    for (int e = 0; e < 4; ++e) {
                                        const uint32_t d = dt * 16 + G * 4 + e;
                                        const _Float16 x = src.vh[(d < a.hd ? d : a.hd - 1) * src.ctx_stride + key];
                                        acc[rt][dt][e] += pj * static_cast<float>(x);
                                    }
                                }
                            }
                        }
                    }
                }
                continue;
            }
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                const h8 v = src.v(dt, c);
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    acc[rt][dt] = mfma16(v, hi[rt][c], acc[rt][dt]);
                    acc[rt][dt] = mfma16(v, lo[rt][c], acc[rt][dt]);
                }
            }
        }
    }

    // Each wave's rows as (maximum, sum, output over sum); the four meet in
    // LDS, a 16-row tile at a time, as a weighted mean.
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        l[rt] = sum32(sum16(l[rt]));
        if (G == 0) {
            lds_m[w][rt * 16 + col] = mref[rt];
            lds_l[w][rt * 16 + col] = l[rt];
        }
        const float inv = l[rt] == 0.0f ? 0.0f : 1.0f / l[rt];
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
            f4 o = acc[rt][dt] * inv;
            if constexpr (SRC::steps) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    o[e] = vexp == -1000 ? o[e] : ldexpf(o[e], vexp);
                }
            }
            acc[rt][dt] = o;
        }
    }
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        if (rt > 0) {
            __syncthreads();
        }
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
            *reinterpret_cast<f4*>(&lds_o[w][col][dt * 16 + G * 4]) = acc[rt][dt];
        }
        __syncthreads();
        const uint32_t pairs = a.hd / 2;
        for (uint32_t i = threadIdx.x; i < 16 * pairs; i += 256) {
            const uint32_t rr = i / pairs, d = i % pairs * 2;
            const uint32_t r = row0 + rt * 16 + rr;
            if (r >= rows) {
                break;  // (later ones are further rows)
            }
            float top = -INFINITY, sum = 0.0f;
#pragma unroll
            for (uint32_t x = 0; x < attend_waves; ++x) {
                top = fmaxf(top, lds_m[x][rt * 16 + rr]);
            }
            f2 o = {0.0f, 0.0f};
#pragma unroll
            for (uint32_t x = 0; x < attend_waves; ++x) {
                const float wx = part_weight(lds_m[x][rt * 16 + rr], lds_l[x][rt * 16 + rr], top);
                sum += wx;
                const f2 ox = *reinterpret_cast<const f2*>(&lds_o[x][rr][d]);
                o[0] += wx == 0.0f ? 0.0f : wx * ox[0];
                o[1] += wx == 0.0f ? 0.0f : wx * ox[1];
            }
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
            o *= inv;
            if (a.splits == 1) {
                const size_t at = size_t{r / a.group} * a.q_row + (g * a.group + r % a.group) * a.hd + d;
                *reinterpret_cast<f2*>(a.out + at) = o;
            } else {
                const size_t slot = (size_t{split} * a.n_kv + g) * rows + r;
                *reinterpret_cast<f2*>(a.part + slot * a.hd + d) = o;
                if (d == 0) {
                    *reinterpret_cast<f2*>(a.part_ml + slot * 2) = f2{top, sum};
                }
            }
        }
    }
}

template <int DC, int RT, class SRC, bool TREE>
hipError_t launch_attend_rows_as(const attend_rows_args& a, hipStream_t stream) {
    const uint64_t blocks = uint64_t{a.row_blocks} * a.n_kv * a.splits;
    if (blocks > 0x7fffffffu) {
        return hipErrorInvalidValue;
    }
    attend_rows_kernel<DC, RT, SRC, TREE><<<static_cast<uint32_t>(blocks), 256, 0, stream>>>(a);
    if (hipError_t e = hipGetLastError(); e != hipSuccess || a.splits == 1) {
        return e;
    }
    return launch_attend_merge(a, stream);
}

}  // namespace syn
