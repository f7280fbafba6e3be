// attend_kv8.hip — attend_rows over 8-bit KV states: causal runs and drafted
// trees.

#include "attend_rows.hpp"

namespace syn {

namespace {

template <int DC, bool TREE>
hipError_t by_rows(const attend_rows_args& a, hipStream_t stream) {
    switch (a.kernel) {
    case attend_few:
        return launch_attend_blocks(attend_few_kernel<DC, attend::kv8_source<DC>, TREE>, 256, a, stream);
    case attend_many16:
        return launch_attend_blocks(attend_many_kernel<DC, 1, true, true, TREE>, 256, a, stream);
    case attend_many32:
        return launch_attend_blocks(attend_many_kernel<DC, 2, true, true, TREE>, 256, a, stream);
    case attend_turns:
        if constexpr (DC <= 4) {
            return launch_attend_blocks(attend_turns_kernel<DC, true, TREE>, 512, a, stream);
        }
        [[fallthrough]];
    default:
        return hipErrorInvalidValue;
    }
}

template <int DC>
hipError_t by_mask(const attend_rows_args& a, hipStream_t stream) {
    return a.mask != nullptr ? by_rows<DC, true>(a, stream) : by_rows<DC, false>(a, stream);
}

}  // namespace

hipError_t launch_attend_kv8(const attend_rows_args& a, hipStream_t stream) {
    switch ((a.hd + 31) / 32) {
    case 1:
        return by_mask<1>(a, stream);
    case 2:
        return by_mask<2>(a, stream);
    case 3:
        return by_mask<3>(a, stream);
    case 4:
        return by_mask<4>(a, stream);
    case 5:
        return by_mask<5>(a, stream);
    case 6:
        return by_mask<6>(a, stream);
    case 7:
        return by_mask<7>(a, stream);
    case 8:
        return by_mask<8>(a, stream);
    default:
        return hipErrorInvalidValue;
    }
}

}  // namespace syn
