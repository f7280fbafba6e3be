// attend_tree.hip — attend_rows over binary16 KV states: drafted trees.

#include "attend_rows.hpp"

namespace syn {

namespace {

// WHOLE8: K rows on 16 bytes; other head sizes load them by pairs.
template <int DC, bool WHOLE8>
hipError_t by_rows(const attend_rows_args& a, hipStream_t stream) {
    switch (a.kernel) {
    case attend_few:
        if constexpr (DC <= 6) {
            return launch_attend_blocks(attend_few_kernel<DC, attend::f16_source<DC, WHOLE8>, true>, 256, a, stream);
        }
        return hipErrorInvalidValue;
    case attend_many16:
        return launch_attend_blocks(attend_many_kernel<DC, 1, false, WHOLE8, true>, 256, a, stream);
    case attend_many32:
        if constexpr (WHOLE8) {
            return launch_attend_blocks(attend_many_kernel<DC, 2, false, true, true>, 256, a, stream);
        }
        return hipErrorInvalidValue;
    case attend_turns:
        if constexpr (WHOLE8 && DC <= 4) {
            return launch_attend_blocks(attend_turns_kernel<DC, false, true>, 512, a, stream);
        }
        [[fallthrough]];
    default:
        return hipErrorInvalidValue;
    }
}

template <int DC>
hipError_t by_size(const attend_rows_args& a, hipStream_t stream) {
    return a.hd % 8 == 0 ? by_rows<DC, true>(a, stream) : by_rows<DC, false>(a, stream);
}

}  // namespace

hipError_t launch_attend_tree(const attend_rows_args& a, hipStream_t stream) {
    switch ((a.hd + 31) / 32) {
    case 1:
        return by_size<1>(a, stream);
    case 2:
        return by_size<2>(a, stream);
    case 3:
        return by_size<3>(a, stream);
    case 4:
        return by_size<4>(a, stream);
    case 5:
        return by_size<5>(a, stream);
    case 6:
        return by_size<6>(a, stream);
    case 7:
        return by_size<7>(a, stream);
    case 8:
        return by_size<8>(a, stream);
    default:
        return hipErrorInvalidValue;
    }
}

}  // namespace syn
