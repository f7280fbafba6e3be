// attend_merge.hip — joins the splits of attend_rows: each query row's parts
// are outputs already divided by their sums, so the row is their mean,
// weighted by sum * exp2(maximum - largest maximum).
//
// One wave per (KV head, query row); where rows are few and one wave would
// take its splits in several rounds of loads (a decode step), four, each a
// quarter of the head's dims (32 rows of 17 splits 3.7 us, one wave 4.8; but 14
// rows of 2 splits 3.8 and 3.1, and 3904 rows of 32 splits 8.4 and 7.4). Every
// wave makes all the weights itself, four splits a lane, with no barrier; a
// lane then sums every parts-th split of its quad of dims in order, and the
// parts meet in a fixed tree, so results do not depend on timing. A few
// hundred KB to some MB from L2: bound by the launch and two dependent trips;
// 16288 rows of 4 splits, 34 MB, take 10.9 us, 3.1 TB/s.

#include "attend_rows.hpp"

namespace syn {

namespace {

// block 256: WPR waves per row. quads: power of two, the quads of dims a wave
// takes; parts = 64 / quads.
template <int WPR>
__global__ __launch_bounds__(256) void attend_merge_kernel(const attend_rows_args a, uint32_t quads) {
    using namespace attend;
    const uint32_t rows = a.n * a.group;
    const uint32_t lane = threadIdx.x % 64;
    const uint32_t wv = blockIdx.x * 4 + threadIdx.x / 64;  // one wave of all
    const uint32_t unit = wv / WPR, quarter = wv % WPR;
    const uint32_t g = unit % a.n_kv, r = unit / a.n_kv;
    if (r >= rows) {
        return;
    }
    const size_t slot0 = size_t{g} * rows + r, stride = size_t{a.n_kv} * rows;  // from split to split
    float weight[4], m[4], l[4];
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
        const uint32_t s = i * 64 + lane;
        const bool has = s < a.splits;
        const f2 ml = *reinterpret_cast<const f2*>(a.part_ml + (slot0 + (has ? s : 0) * stride) * 2);
        m[i] = has ? ml[0] : -INFINITY;
        l[i] = has ? ml[1] : 0.0f;
    }
    const float top = wave_reduce_max(fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])));
    float sum = 0.0f;
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
        weight[i] = part_weight(m[i], l[i], top);
        sum += weight[i];
    }
    sum = wave_reduce_sum(sum);
    const uint32_t quad = lane % quads, part = lane / quads, parts = 64 / quads;
    const uint32_t d = (quarter * quads + quad) * 4;
    const bool in = d < a.hd;
    const bool two = d + 2 < a.hd;  // hd is even: the quad is whole or half
    f4 o = {0, 0, 0, 0};
    for (uint32_t s0 = 0; s0 < a.splits; s0 += parts * 4) {
        f2 x[4], y[4];
        float ws[4];
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            const uint32_t s = s0 + i * parts + part;
            const float* p = a.part + (slot0 + (s < a.splits ? s : 0) * stride) * a.hd + (in ? d : 0);
            x[i] = *reinterpret_cast<const f2*>(p);
            y[i] = *reinterpret_cast<const f2*>(p + (two ? 2 : 0));
            const uint32_t k = s / 64;
            const float mine0 = __shfl(weight[0], static_cast<int>(s % 64)), mine1 = __shfl(weight[1], static_cast<int>(s % 64));
            const float mine2 = __shfl(weight[2], static_cast<int>(s % 64)), mine3 = __shfl(weight[3], static_cast<int>(s % 64));
            ws[i] = s >= a.splits ? 0.0f : k == 0 ? mine0 : k == 1 ? mine1 : k == 2 ? mine2 : mine3;
        }
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            if (ws[i] != 0.0f) {  // (a part without weight may hold anything)
                o[0] += ws[i] * x[i][0];
                o[1] += ws[i] * x[i][1];
                o[2] += ws[i] * y[i][0];
                o[3] += ws[i] * y[i][1];
            }
        }
    }
    for (uint32_t step = quads; step < 64; step *= 2) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            o[e] += __shfl_xor(o[e], static_cast<int>(step));
        }
    }
    if (part == 0 && in) {
        o *= sum == 0.0f ? 0.0f : 1.0f / sum;
        float* out = a.out + size_t{r / a.group} * a.q_row + (g * a.group + r % a.group) * a.hd + d;
        *reinterpret_cast<f2*>(out) = f2{o[0], o[1]};
        if (two) {
            *reinterpret_cast<f2*>(out + 2) = f2{o[2], o[3]};
        }
    }
}

}  // namespace

hipError_t launch_attend_merge(const attend_rows_args& a, hipStream_t stream) {
    const uint64_t units = uint64_t{a.n} * a.group * a.n_kv;
    uint32_t quads = 1;
    while (quads * 4 < a.hd) {
        quads *= 2;
    }
    const uint32_t round = 64 / quads * 4;  // splits that one wave loads at once
    const uint32_t wpr = units < 1024 && a.splits > round && quads >= 4 ? 4 : 1;
    quads /= wpr;
    const uint64_t blocks = (units * wpr + 3) / 4;
    if (blocks > 0x7fffffffu) {
        return hipErrorInvalidValue;
    }
    if (wpr == 4) {
        attend_merge_kernel<4><<<static_cast<uint32_t>(blocks), 256, 0, stream>>>(a, quads);
    } else {
        attend_merge_kernel<1><<<static_cast<uint32_t>(blocks), 256, 0, stream>>>(a, quads);
    }
    return hipGetLastError();
}

}  // namespace syn
