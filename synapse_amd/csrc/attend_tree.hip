// attend_tree.hip — attend_rows over binary16 KV states: drafted trees.

#include "attend_rows.hpp"

namespace syn {

namespace {

template <int DC, int RT>
hipError_t whole(const attend_rows_args& a, hipStream_t stream) {
    return launch_attend_rows_as<DC, RT, attend::f16_source<DC, true>, true>(a, stream);
}

template <int DC>
hipError_t by_rows(const attend_rows_args& a, hipStream_t stream) {
    if (a.hd % 8 != 0) {  // K rows off 16 bytes: loads by pairs, in 16-row blocks
        return a.row_tiles == 1 ? launch_attend_rows_as<DC, 1, attend::f16_source<DC, false>, true>(a, stream)
                                : hipErrorInvalidValue;
    }
    switch (a.row_tiles) {
    case 1:
        return whole<DC, 1>(a, stream);
    case 2:
        return whole<DC, 2>(a, stream);
    case 4:
        if constexpr (DC <= 4) {
            return whole<DC, 4>(a, stream);
        }
        [[fallthrough]];
    default:
        return hipErrorInvalidValue;
    }
}

}  // namespace

hipError_t launch_attend_tree(const attend_rows_args& a, hipStream_t stream) {
    switch ((a.hd + 31) / 32) {
    case 1:
        return by_rows<1>(a, stream);
    case 2:
        return by_rows<2>(a, stream);
    case 3:
        return by_rows<3>(a, stream);
    case 4:
        return by_rows<4>(a, stream);
    case 5:
        return by_rows<5>(a, stream);
    case 6:
        return by_rows<6>(a, stream);
    case 7:
        return by_rows<7>(a, stream);
    case 8:
        return by_rows<8>(a, stream);
    default:
        return hipErrorInvalidValue;
    }
}

}  // namespace syn
