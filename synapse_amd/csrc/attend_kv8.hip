// attend_kv8.hip — attend_rows over 8-bit KV states: causal runs and drafted
// trees.

#include "attend_rows.hpp"

namespace syn {

namespace {

template <int DC, int RT>
hipError_t by_mask(const attend_rows_args& a, hipStream_t stream) {
    return a.mask != nullptr ? launch_attend_rows_as<DC, RT, attend::kv8_source<DC>, true>(a, stream)
                             : launch_attend_rows_as<DC, RT, attend::kv8_source<DC>, false>(a, stream);
}

template <int DC>
hipError_t by_rows(const attend_rows_args& a, hipStream_t stream) {
    switch (a.row_tiles) {
    case 1:
        return by_mask<DC, 1>(a, stream);
    case 2:
        return by_mask<DC, 2>(a, stream);
    case 4:
        if constexpr (DC <= 4) {
            return by_mask<DC, 4>(a, stream);
        }
        [[fallthrough]];
    default:
        return hipErrorInvalidValue;
    }
}

}  // namespace

hipError_t launch_attend_kv8(const attend_rows_args& a, hipStream_t stream) {
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
