// kv8.hip — 8-bit KV states: rows quantized as they are written, read back,
// and moved together after a drafted tree; the move for binary16 states too.
//
// A row (position, KV head) of hd values x has one step d = max|x| / 127,
// rounded to f32, and bytes q = x / d, rounded to the nearest whole number
// with ties to even -- of the quotient itself, not of its f32 rounding: the
// remainder x - q d is exact in one fused multiply-add, and says on which
// side of a half the quotient lies. A row of zeros has step 0; a row that
// holds an infinity or NaN has step NaN and reads back as NaN.
//
// Append and read move bytes (rows of 4 or 2 bytes a value one way, 1 the
// other) and are bound by HBM: a block takes one tile of 64 positions of one
// KV head, a part-wave of hd / 4 lanes takes one row at a time, four values a
// lane, and LDS turns rows into the tile's record and back, so that both
// sides of the copy are whole lines. 16384 rows of 8 x 128 f32: append 41.5 us
// and read 34.1 us for 169 MB (4.1 and 5.0 TB/s); 100000 rows appended in 224 us
// (4.6 TB/s); one row 3.7 and 2.8 us, the launch and a trip each way.

#include "kernels.hpp"

namespace syn {

namespace {

constexpr uint32_t threads = 512;
constexpr uint32_t max_record = kv8_tile * 256;  // K or V bytes of a tile at hd 256

// Four values of a row, from dim d0 on (zeros past the last one).
template <typename T>
__device__ __forceinline__ f4 load_four(const T* row, uint32_t d0, uint32_t hd, bool vec) {
    typedef T t4 __attribute__((ext_vector_type(4)));
    f4 x = {0, 0, 0, 0};
    if (vec) {
        if (d0 < hd) {
            const t4 y = *reinterpret_cast<const t4*>(row + d0);
            x = f4{static_cast<float>(y[0]), static_cast<float>(y[1]), static_cast<float>(y[2]),
                   static_cast<float>(y[3])};
        }
        return x;
    }
#pragma unroll
    for (uint32_t e = 0; e < 4; ++e) {
        if (d0 + e < hd) {
            x[e] = static_cast<float>(row[d0 + e]);
        }
    }
    return x;
}
template <typename T>
__device__ __forceinline__ void store_four(T* row, uint32_t d0, uint32_t hd, bool vec, f4 x) {
    typedef T t4 __attribute__((ext_vector_type(4)));
    if (vec) {
        if (d0 < hd) {
            *reinterpret_cast<t4*>(row + d0) =
                t4{static_cast<T>(x[0]), static_cast<T>(x[1]), static_cast<T>(x[2]), static_cast<T>(x[3])};
        }
        return;
    }
#pragma unroll
    for (uint32_t e = 0; e < 4; ++e) {
        if (d0 + e < hd) {
            row[d0 + e] = static_cast<T>(x[e]);
        }
    }
}

// The largest of u over aligned groups of LANES lanes.
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_max(uint32_t u) {
    const uint32_t v = static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(u), CTRL, 0xF, 0xF, false));
    return u > v ? u : v;
}
template <int LANES>
__device__ __forceinline__ uint32_t group_max(uint32_t u) {
    u = dpp_max<dpp_quad_xor1>(u);
    u = dpp_max<dpp_quad_xor2>(u);
    u = dpp_max<dpp_row_half_mirror>(u);
    u = dpp_max<dpp_row_mirror>(u);
    if constexpr (LANES >= 32) {
        const uint32_t v = __builtin_bit_cast(uint32_t, partner16(__builtin_bit_cast(float, u)));
        u = u > v ? u : v;
    }
    if constexpr (LANES >= 64) {
        const uint32_t v = __builtin_bit_cast(uint32_t, partner32(__builtin_bit_cast(float, u)));
        u = u > v ? u : v;
    }
    return u;
}

// A row's four values of this lane over its step: whole numbers + 128, a byte
// each. inv is next to 1 / d, so x inv is off by some 2^-22: rounded, it is the
// quotient's nearest whole number or, next to a half, that number's neighbour.
// The remainder tells which, exactly (a multiple of half an ulp of d, not over
// d, so the fused multiply-add does not round it); only where some lane's
// reaches half a step is there anything to put right.
__device__ __forceinline__ uint32_t quotients(f4 x, float step) {
#pragma clang fp contract(off)
    float d = step;
    const bool small = step < 0x1p-100f;  // its inverse may be out of range: row and step times 2^64, exactly
    if (__builtin_amdgcn_ballot_w64(small && step != 0.0f) != 0) {
        const float up = small ? 0x1p64f : 1.0f;
        d *= up;
        x *= up;
    }
    const float inv = __builtin_amdgcn_rcpf(d), half = 0.5f * d;
    float q[4], r[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        q[e] = rintf(x[e] * inv);
        r[e] = __builtin_fmaf(-q[e], d, x[e]);
    }
    const float most = fmaxf(fmaxf(fabsf(r[0]), fabsf(r[1])), fmaxf(fabsf(r[2]), fabsf(r[3])));
    if (__builtin_amdgcn_ballot_w64(most >= half) != 0) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const bool odd = (static_cast<int>(q[e]) & 1) != 0;
            const float ar = fabsf(r[e]);
            q[e] += ar > half || (ar == half && odd) ? copysignf(1.0f, r[e]) : 0.0f;
        }
    }
    uint32_t bytes = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        bytes = __builtin_amdgcn_cvt_pk_u8_f32(__builtin_amdgcn_fmed3f(q[e], -127.0f, 127.0f) + 128.0f, e, bytes);
    }
    return bytes;
}

// grid: tiles of the run x KV heads, KV heads fastest; block 512. LANES: hd /
// 4 rounded up to a power of two. A group of LANES lanes takes K or V of four
// neighbouring keys at a time, so that a lane has a word of each key's K and
// of each dim's V. Tiles that are the run's whole go through LDS as whole
// lines; of the first and last, K's words are written straight to the record,
// and V's through LDS, by words where all four keys are the run's. Up to four
// keys (a decode step) write V's bytes straight too: no barrier.
template <typename T, int LANES>
__global__ __launch_bounds__(threads) void kv8_append_kernel(const kv8_rows_args a, uint32_t tile0, bool vec) {
    __shared__ __align__(16) uint8_t lds[2][max_record];
    const kv8_shape& s = a.shape;
    const uint32_t g = blockIdx.x % s.n_kv, tile = tile0 + blockIdx.x / s.n_kv;
    const uint32_t key0 = tile * kv8_tile, end = a.pos0 + a.n;
    const uint32_t from = key0 < a.pos0 ? a.pos0 - key0 : 0;             // the tile's keys that the run writes
    const uint32_t to = end - key0 < kv8_tile ? end - key0 : kv8_tile;
    const bool whole = from == 0 && to == kv8_tile, few = to - from <= 4;
    const uint32_t in_group = threadIdx.x % LANES, d0 = in_group * 4;
    constexpr uint32_t per_wave = 64 / LANES, groups = threads / LANES / 2;  // for K, and as many for V
    const uint32_t w = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const uint32_t which = w % 2;                                            // 0 K, 1 V
    const uint32_t group = w / 2 * per_wave + threadIdx.x % 64 / LANES;
    const size_t row = size_t{s.n_kv} * s.hd;
    const T* in = static_cast<const T*>(which ? a.v_in : a.k_in) + size_t{g} * s.hd;
    uint8_t* rec = a.kv8 + (size_t{g} * s.tiles + tile) * s.tile_bytes;
    float* steps = reinterpret_cast<float*>(rec + (which ? s.vs_at : s.ks_at));

#pragma unroll 1
    for (uint32_t key4 = from / 4 * 4 + group * 4; key4 < to; key4 += groups * 4) {
        f4 x[4];
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            if (key4 + i >= from && key4 + i < to) {
                x[i] = load_four(in + (key0 + key4 + i - a.pos0) * row, d0, s.hd, vec);
            }
        }
        uint32_t bytes[4];
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            uint32_t top = 0;  // of the magnitudes' bits, which are in their order, NaN above all
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float xe = x[i][e];  // (a bit cast of the element itself casts element 0)
                const uint32_t b = __builtin_bit_cast(uint32_t, xe) & 0x7fffffffu;
                top = b > top ? b : top;
            }
            top = group_max<LANES>(top);
            const bool wild = top >= 0x7f800000u;
            const float step = __builtin_bit_cast(float, top) / 127.0f;
            const uint32_t q = quotients(x[i], step);
            bytes[i] = wild || step == 0.0f ? 0x80808080u : q;
            if (in_group == 0 && key4 + i >= from && key4 + i < to) {
                steps[key4 + i] = wild ? __builtin_nanf("") : step;
            }
        }
        if (d0 >= s.hdp) {
            continue;
        }
        if (which == 0) {
            uint8_t* k = whole ? lds[0] : rec;
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                if (key4 + i >= from && key4 + i < to) {
                    *reinterpret_cast<uint32_t*>(k + kv8_k_at(s.hdp, key4 + i, d0)) = bytes[i];
                }
            }
        } else if (!few) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t v = (bytes[0] >> (8 * e) & 0xff) | (bytes[1] >> (8 * e) & 0xff) << 8 |
                                   (bytes[2] >> (8 * e) & 0xff) << 16 | (bytes[3] >> (8 * e) & 0xff) << 24;
                *reinterpret_cast<uint32_t*>(lds[1] + kv8_v_at(key4, d0 + e)) = v;
            }
        } else {
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                if (key4 + i >= from && key4 + i < to) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        rec[s.v_at + kv8_v_at(key4 + i, d0 + e)] = static_cast<uint8_t>(bytes[i] >> (8 * e));
                    }
                }
            }
        }
    }
    if (whole) {
        __syncthreads();
        const uint32_t bytes = kv8_tile * s.hdp;
        for (uint32_t i = threadIdx.x * 16; i < 2 * bytes; i += threads * 16) {
            const uint32_t in_v = i >= bytes, b = i - in_v * bytes;
            store16(rec + i, *reinterpret_cast<const u4*>(&lds[in_v][b]));
        }
    } else if (!few) {
        __syncthreads();
        for (uint32_t b = threadIdx.x * 4; b < kv8_tile * s.hdp; b += threads * 4) {
            const uint32_t key = b % 16 / 8 * 32 + b % 1024 / 256 * 8 + b % 8;  // (kv8_v_at the other way)
            const uint32_t x = *reinterpret_cast<const uint32_t*>(&lds[1][b]);
            if (key >= from && key + 3 < to) {
                *reinterpret_cast<uint32_t*>(rec + s.v_at + b) = x;
            } else {
#pragma unroll
                for (uint32_t e = 0; e < 4; ++e) {
                    if (key + e >= from && key + e < to) {
                        rec[s.v_at + b + e] = static_cast<uint8_t>(x >> (8 * e));
                    }
                }
            }
        }
    }
}

// The same grid and groups, the other way.
template <typename T, int LANES>
__global__ __launch_bounds__(threads) void kv8_read_kernel(const kv8_rows_args a, uint32_t tile0, bool vec) {
    __shared__ __align__(16) uint8_t lds[2][max_record];
    __shared__ float steps[2][kv8_tile];
    const kv8_shape& s = a.shape;
    const uint32_t g = blockIdx.x % s.n_kv, tile = tile0 + blockIdx.x / s.n_kv;
    const uint32_t key0 = tile * kv8_tile, end = a.pos0 + a.n;
    const uint32_t from = key0 < a.pos0 ? a.pos0 - key0 : 0;
    const uint32_t to = end - key0 < kv8_tile ? end - key0 : kv8_tile;
    const uint8_t* rec = a.kv8 + (size_t{g} * s.tiles + tile) * s.tile_bytes;
    const uint32_t bytes = kv8_tile * s.hdp;
    constexpr uint32_t most = 2 * kv8_tile * 4 * LANES / (threads * 16);
    u4 x[most];
#pragma unroll
    for (uint32_t i = 0; i < most; ++i) {
        const uint32_t at = (i * threads + threadIdx.x) * 16;
        if (at < 2 * bytes) {
            x[i] = load16(rec + at);
        }
    }
    if (threadIdx.x < 2 * kv8_tile) {
        const uint32_t which = threadIdx.x / kv8_tile, key = threadIdx.x % kv8_tile;
        steps[which][key] = *reinterpret_cast<const float*>(rec + (which ? s.vs_at : s.ks_at) + key * 4);
    }
#pragma unroll
    for (uint32_t i = 0; i < most; ++i) {
        const uint32_t at = (i * threads + threadIdx.x) * 16;
        if (at < 2 * bytes) {
            const uint32_t which = at >= bytes;
            *reinterpret_cast<u4*>(&lds[which][at - which * bytes]) = x[i];
        }
    }
    __syncthreads();
    const uint32_t d0 = threadIdx.x % LANES * 4;
    if (d0 >= s.hd) {
        return;
    }
    constexpr uint32_t per_wave = 64 / LANES, groups = threads / LANES / 2;
    const uint32_t w = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const uint32_t which = w % 2;
    const uint32_t group = w / 2 * per_wave + threadIdx.x % 64 / LANES;
    const size_t row = size_t{s.n_kv} * s.hd;
    T* out = static_cast<T*>(which ? a.v_out : a.k_out) + size_t{g} * s.hd;
    for (uint32_t key4 = from / 4 * 4 + group * 4; key4 < to; key4 += groups * 4) {
        uint32_t b[4];  // K: of key i, V: of dim i
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            b[i] = *reinterpret_cast<const uint32_t*>(which ? &lds[1][kv8_v_at(key4, d0 + i)]
                                                            : &lds[0][kv8_k_at(s.hdp, key4 + i, d0)]);
        }
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            if (key4 + i >= from && key4 + i < to) {
                const float d = steps[which][key4 + i];
                f4 x;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t q = which ? b[e] >> (8 * i) & 0xff : b[i] >> (8 * e) & 0xff;
                    x[e] = static_cast<float>(static_cast<int>(q) - 128) * d;
                }
                store_four(out + (key0 + key4 + i - a.pos0) * row, d0, s.hd, vec, x);
            }
        }
    }
}

// Four-value accesses: whole fours of dims on four-element offsets.
bool fours(const kv8_rows_args& a, const void* k, const void* v) {
    const uintptr_t to = a.f16 ? 8 : 16;
    return a.shape.hd % 4 == 0 && reinterpret_cast<uintptr_t>(k) % to == 0 && reinterpret_cast<uintptr_t>(v) % to == 0;
}

template <template <typename, int> class K>
hipError_t launch_rows(const kv8_rows_args& a, bool vec, hipStream_t stream) {
    const uint32_t tile0 = a.pos0 / kv8_tile, tile1 = (a.pos0 + a.n - 1) / kv8_tile;
    const uint64_t blocks = uint64_t{tile1 - tile0 + 1} * a.shape.n_kv;
    if (blocks > 0x7fffffffu) {
        return hipErrorInvalidValue;
    }
    const dim3 grid(static_cast<uint32_t>(blocks));
    if (a.f16) {
        if (a.shape.hd <= 64) {
            K<_Float16, 16>::run(grid, stream, a, tile0, vec);
        } else if (a.shape.hd <= 128) {
            K<_Float16, 32>::run(grid, stream, a, tile0, vec);
        } else {
            K<_Float16, 64>::run(grid, stream, a, tile0, vec);
        }
    } else if (a.shape.hd <= 64) {
        K<float, 16>::run(grid, stream, a, tile0, vec);
    } else if (a.shape.hd <= 128) {
        K<float, 32>::run(grid, stream, a, tile0, vec);
    } else {
        K<float, 64>::run(grid, stream, a, tile0, vec);
    }
    return hipGetLastError();
}
template <typename T, int LANES>
struct append_rows {
    static void run(dim3 grid, hipStream_t stream, const kv8_rows_args& a, uint32_t tile0, bool vec) {
        kv8_append_kernel<T, LANES><<<grid, threads, 0, stream>>>(a, tile0, vec);
    }
};
template <typename T, int LANES>
struct read_rows {
    static void run(dim3 grid, hipStream_t stream, const kv8_rows_args& a, uint32_t tile0, bool vec) {
        kv8_read_kernel<T, LANES><<<grid, threads, 0, stream>>>(a, tile0, vec);
    }
};

// ---- keep: rows moved to the front -------------------------------------------
// Position pos + first + i <- pos + row[i], the rows rising, so row[i] >=
// first + i: every source is read before it is written over when a thread
// owns its column (one word of K, one feature of V^T, one byte or step) and
// goes through the rows in order, `batch` loads ahead of their stores. A
// handful of rows of a few KB: bound by the launch and two dependent trips to
// memory (6 rows: 3.3 us, of an 8-bit state 4.3).
constexpr uint32_t batch = 8;

// A launch of up to `batch` rows (an accepted path) carries them in an argument
// block of 16 bytes, read with the other arguments.
struct few_rows {
    uint16_t row[batch];
};

template <typename T, class ROWS, class AT>
__device__ __forceinline__ void move_column(AT at, uint32_t first, uint32_t count, const ROWS& r) {
    constexpr uint32_t most = sizeof(r.row) / sizeof(r.row[0]);
    for (uint32_t i0 = 0; i0 < (most == batch ? 1 : count); i0 += batch) {
        T x[batch];
#pragma unroll
        for (uint32_t i = 0; i < batch; ++i) {
            if (i0 + i < count) {
                x[i] = *at(r.row[i0 + i]);
            }
        }
#pragma unroll
        for (uint32_t i = 0; i < batch; ++i) {
            if (i0 + i < count) {
                *at(first + i0 + i) = x[i];
            }
        }
    }
}

template <class ROWS>
__global__ __launch_bounds__(256) void kv_keep_kernel(const kv_layout c, uint32_t pos, uint32_t first, uint32_t count,
                                                      const ROWS r) {
    const uint32_t row = c.n_kv * c.hd;  // even, as hd is
    const uint32_t i = blockIdx.x * 256 + threadIdx.x;
    if (i < row / 2) {
        uint32_t* k = reinterpret_cast<uint32_t*>(c.k) + i;
        move_column<uint32_t>([=](uint32_t t) { return k + (size_t{pos} + t) * (row / 2); }, first, count, r);
    } else if (i - row / 2 < row) {
        _Float16* v = c.vt + size_t{i - row / 2} * c.ctx_stride + pos;
        move_column<_Float16>([=](uint32_t t) { return v + t; }, first, count, r);
    }
}

template <class ROWS>
__global__ __launch_bounds__(256) void kv8_keep_kernel(uint8_t* kv8, const kv8_shape s, uint32_t pos, uint32_t first,
                                                       uint32_t count, const ROWS r) {
    const uint32_t words = s.hdp / 4, columns = words + s.hd + 2;  // a KV head's: K words, V bytes, steps
    const uint32_t j = blockIdx.y * 256 + threadIdx.x;
    if (j >= columns) {
        return;
    }
    uint8_t* head = kv8 + size_t{blockIdx.x} * s.tiles * s.tile_bytes;
    const auto rec = [=](uint32_t t) { return head + size_t{(pos + t) / kv8_tile} * s.tile_bytes; };
    if (j < words) {
        move_column<uint32_t>(
            [=](uint32_t t) {
                return reinterpret_cast<uint32_t*>(rec(t) + kv8_k_at(s.hdp, (pos + t) % kv8_tile, j * 4));
            },
            first, count, r);
    } else if (j - words < s.hd) {
        move_column<uint8_t>(
            [=](uint32_t t) { return rec(t) + s.v_at + kv8_v_at((pos + t) % kv8_tile, j - words); }, first, count, r);
    } else {
        const uint32_t at = j == columns - 2 ? s.ks_at : s.vs_at;
        move_column<float>(
            [=](uint32_t t) { return reinterpret_cast<float*>(rec(t) + at + (pos + t) % kv8_tile * 4); }, first, count,
            r);
    }
}

few_rows few_of(const keep_rows& rows) {
    few_rows f{};
    for (uint32_t i = 0; i < batch; ++i) {
        f.row[i] = rows.row[i];
    }
    return f;
}

}  // namespace

hipError_t launch_kv8_append(const kv8_rows_args& a, hipStream_t stream) {
    return launch_rows<append_rows>(a, fours(a, a.k_in, a.v_in), stream);
}

hipError_t launch_kv8_read(const kv8_rows_args& a, hipStream_t stream) {
    return launch_rows<read_rows>(a, fours(a, a.k_out, a.v_out), stream);
}

hipError_t launch_kv_keep(const kv_layout& c, uint32_t pos, uint32_t first, uint32_t count, const keep_rows& rows,
                          hipStream_t stream) {
    const uint64_t columns = uint64_t{c.n_kv} * c.hd / 2 * 3;
    const uint32_t blocks = static_cast<uint32_t>((columns + 255) / 256);
    if (count <= batch) {
        kv_keep_kernel<<<blocks, 256, 0, stream>>>(c, pos, first, count, few_of(rows));
    } else {
        kv_keep_kernel<<<blocks, 256, 0, stream>>>(c, pos, first, count, rows);
    }
    return hipGetLastError();
}

hipError_t launch_kv8_keep(uint8_t* kv8, const kv8_shape& s, uint32_t pos, uint32_t first, uint32_t count,
                           const keep_rows& rows, hipStream_t stream) {
    const dim3 blocks(s.n_kv, (s.hdp / 4 + s.hd + 2 + 255) / 256);
    if (count <= batch) {
        kv8_keep_kernel<<<blocks, 256, 0, stream>>>(kv8, s, pos, first, count, few_of(rows));
    } else {
        kv8_keep_kernel<<<blocks, 256, 0, stream>>>(kv8, s, pos, first, count, rows);
    }
    return hipGetLastError();
}

}  // namespace syn
