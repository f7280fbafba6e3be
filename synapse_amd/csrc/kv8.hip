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
// sides of the copy are whole lines.

#include "kernels.hpp"

namespace syn {

namespace {

constexpr uint32_t threads = 512;
constexpr uint32_t max_record = kv8_tile * 256;  // K or V bytes of a tile at hd 256

// The key whose value is in byte b of a tile's K block, and likewise V.
__device__ __forceinline__ uint32_t k_key(uint32_t b, uint32_t hdp) {
    const uint32_t op = b / (16 * hdp), rest = b % (16 * hdp), pairs = hdp / 64 * 64;
    const uint32_t m = rest < pairs * 16 ? rest / 16 % 16 : (rest - pairs * 16) / 8 % 16;
    return op / 2 * 32 + m / 4 * 8 + op % 2 * 4 + m % 4;
}
__device__ __forceinline__ uint32_t v_key(uint32_t b) {
    return b % 16 / 8 * 32 + b % 1024 / 256 * 8 + b % 8;
}

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

// x / d to the nearest whole number, ties to even, for |x| up to 127.5 d.
__device__ __forceinline__ int quotient(float x, float d) {
#pragma clang fp contract(off)
    float q = rintf(x / d);
    const float r = __builtin_fmaf(-q, d, x);  // exact: a multiple of half an ulp of d, not over d
    const float twice = 2.0f * fabsf(r);
    const bool odd = (static_cast<int>(q) & 1) != 0;
    if (twice > d || (twice == d && odd)) {
        q += copysignf(1.0f, r);
    }
    return static_cast<int>(fminf(fmaxf(q, -127.0f), 127.0f));
}

// grid: tiles of the run x KV heads, KV heads fastest; block 512. LANES: hd /
// 4 rounded up to a power of two.
template <typename T, int LANES>
__global__ __launch_bounds__(threads) void kv8_append_kernel(const kv8_rows_args a, uint32_t tile0, bool vec) {
    __shared__ __align__(16) uint8_t lds[2][max_record];
    __shared__ float steps[2][kv8_tile];
    const kv8_shape& s = a.shape;
    const uint32_t g = blockIdx.x % s.n_kv, tile = tile0 + blockIdx.x / s.n_kv;
    const uint32_t key0 = tile * kv8_tile, end = a.pos0 + a.n;
    const uint32_t from = key0 < a.pos0 ? a.pos0 - key0 : 0;             // the tile's keys that the run writes
    const uint32_t to = end - key0 < kv8_tile ? end - key0 : kv8_tile;
    const uint32_t in_group = threadIdx.x % LANES, d0 = in_group * 4;
    const size_t row = size_t{s.n_kv} * s.hd;
    constexpr uint32_t groups = threads / LANES;

    // Rows 2 key + (0 K, 1 V); each group takes every groups-th.
    for (uint32_t i = 2 * from + threadIdx.x / LANES; i < 2 * to; i += groups) {
        const uint32_t key = i / 2, which = i % 2;
        const T* src = static_cast<const T*>(which ? a.v_in : a.k_in) + (key0 + key - a.pos0) * row + size_t{g} * s.hd;
        const f4 x = load_four(src, d0, s.hd, vec);
        uint32_t top = 0;  // of the magnitudes' bits, which are in their order, NaN above all
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float xe = x[e];  // (a bit cast of the element itself casts element 0)
            const uint32_t b = __builtin_bit_cast(uint32_t, xe) & 0x7fffffffu;
            top = b > top ? b : top;
        }
        top = group_max<LANES>(top);
        const bool wild = top >= 0x7f800000u;
        const float d = __builtin_bit_cast(float, top) / 127.0f;
        uint32_t bytes = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int q = wild || d == 0.0f ? 0 : quotient(x[e], d);
            bytes |= static_cast<uint32_t>(q + 128) << (8 * e);
        }
        if (d0 < s.hdp) {
            if (which == 0) {
                *reinterpret_cast<uint32_t*>(&lds[0][kv8_k_at(s.hdp, key, d0)]) = bytes;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    lds[1][kv8_v_at(key, d0 + e)] = static_cast<uint8_t>(bytes >> (8 * e));
                }
            }
        }
        if (in_group == 0) {
            steps[which][key] = wild ? __builtin_nanf("") : d;
        }
    }
    __syncthreads();

    uint8_t* rec = a.kv8 + (size_t{g} * s.tiles + tile) * s.tile_bytes;
    const uint32_t bytes = kv8_tile * s.hdp;
    if (from == 0 && to == kv8_tile) {
        for (uint32_t i = threadIdx.x * 16; i < 2 * bytes; i += threads * 16) {
            const uint32_t which = i >= bytes, b = i - which * bytes;
            store16(rec + i, *reinterpret_cast<const u4*>(&lds[which][b]));
        }
    } else {
        // Only the run's keys: a word of K is one key's, a word of V four
        // keys', stored by the byte where some of them are not the run's.
        for (uint32_t i = threadIdx.x * 4; i < 2 * bytes; i += threads * 4) {
            const uint32_t which = i >= bytes, b = i - which * bytes;
            const uint32_t key = which ? v_key(b) : k_key(b, s.hdp);
            const uint32_t x = *reinterpret_cast<const uint32_t*>(&lds[which][b]);
            if (key >= from && key + (which ? 3 : 0) < to) {
                *reinterpret_cast<uint32_t*>(rec + i) = x;
            } else if (which) {
#pragma unroll
                for (uint32_t e = 0; e < 4; ++e) {
                    if (key + e >= from && key + e < to) {
                        rec[i + e] = static_cast<uint8_t>(x >> (8 * e));
                    }
                }
            }
        }
    }
    if (threadIdx.x < 2 * kv8_tile) {
        const uint32_t which = threadIdx.x / kv8_tile, key = threadIdx.x % kv8_tile;
        if (key >= from && key < to) {
            *reinterpret_cast<float*>(rec + (which ? s.vs_at : s.ks_at) + key * 4) = steps[which][key];
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
    for (uint32_t i = threadIdx.x * 16; i < 2 * bytes; i += threads * 16) {
        const uint32_t which = i >= bytes;
        *reinterpret_cast<u4*>(&lds[which][i - which * bytes]) = load16(rec + i);
    }
    if (threadIdx.x < 2 * kv8_tile) {
        const uint32_t which = threadIdx.x / kv8_tile, key = threadIdx.x % kv8_tile;
        steps[which][key] = *reinterpret_cast<const float*>(rec + (which ? s.vs_at : s.ks_at) + key * 4);
    }
    __syncthreads();
    const uint32_t d0 = threadIdx.x % LANES * 4;
    const size_t row = size_t{s.n_kv} * s.hd;
    if (d0 >= s.hd) {
        return;
    }
    constexpr uint32_t groups = threads / LANES;
    for (uint32_t i = 2 * from + threadIdx.x / LANES; i < 2 * to; i += groups) {
        const uint32_t key = i / 2, which = i % 2;
        uint32_t b;
        if (which == 0) {
            b = *reinterpret_cast<const uint32_t*>(&lds[0][kv8_k_at(s.hdp, key, d0)]);
        } else {
            b = lds[1][kv8_v_at(key, d0)] | lds[1][kv8_v_at(key, d0 + 1)] << 8 |
                lds[1][kv8_v_at(key, d0 + 2)] << 16 | static_cast<uint32_t>(lds[1][kv8_v_at(key, d0 + 3)]) << 24;
        }
        const float d = steps[which][key];
        f4 x;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            x[e] = static_cast<float>(static_cast<int>(b >> (8 * e) & 0xff) - 128) * d;
        }
        store_four(static_cast<T*>(which ? a.v_out : a.k_out) + (key0 + key - a.pos0) * row + size_t{g} * s.hd, d0,
                   s.hd, vec, x);
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
// handful of rows of a few KB: bound by two dependent trips to memory.
constexpr uint32_t batch = 8;

template <typename T, class AT>
__device__ __forceinline__ void move_column(AT at, uint32_t first, uint32_t count, const keep_rows& r) {
    for (uint32_t i0 = 0; i0 < count; i0 += batch) {
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

__global__ __launch_bounds__(256) void kv_keep_kernel(const kv_layout c, uint32_t pos, uint32_t first, uint32_t count,
                                                      const keep_rows r) {
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

__global__ __launch_bounds__(256) void kv8_keep_kernel(uint8_t* kv8, const kv8_shape s, uint32_t pos, uint32_t first,
                                                       uint32_t count, const keep_rows r) {
    const uint32_t words = s.hdp / 4, columns = words + s.hd + 2;  // a KV head's: K words, V bytes, steps
    const uint32_t i = blockIdx.x * 256 + threadIdx.x;
    const uint32_t g = i / columns, j = i % columns;
    if (g >= s.n_kv) {
        return;
    }
    uint8_t* head = kv8 + size_t{g} * s.tiles * s.tile_bytes;
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
    kv_keep_kernel<<<static_cast<uint32_t>((columns + 255) / 256), 256, 0, stream>>>(c, pos, first, count, rows);
    return hipGetLastError();
}

hipError_t launch_kv8_keep(uint8_t* kv8, const kv8_shape& s, uint32_t pos, uint32_t first, uint32_t count,
                           const keep_rows& rows, hipStream_t stream) {
    const uint64_t columns = uint64_t{s.n_kv} * (s.hdp / 4 + s.hd + 2);
    kv8_keep_kernel<<<static_cast<uint32_t>((columns + 255) / 256), 256, 0, stream>>>(kv8, s, pos, first, count, rows);
    return hipGetLastError();
}

}  // namespace syn
